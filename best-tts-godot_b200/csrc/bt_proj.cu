// bt_proj.cu -- quantised projections: symmetric 8-bit row quantisation
// (bt_quantize_rows) and the int8 x int8 product with a scale for each token
// and each output channel (bt_matmul_int8).
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include "bt_ops.h"
#include "bt_internal.h"
#include "bt_tc.h"

namespace bt {
namespace {

// ---- row quantisation ------------------------------------------------------
//   a = max(max_k |x_k|, 2^-100);  scale = a / 127;  q_k = rint(x_k (127 / a))
// in float32, each step rounded once; |x_k| <= a keeps |q_k| <= 127 without
// a clip, the 2^-100 floor keeps 127 / a finite.  A NaN makes the row's scale
// NaN (fmaxf would drop it, so it is carried in a flag), an infinity makes it
// infinite; products that are NaN become 0.
constexpr int kQuantThreads = 128;

template <typename T>
__device__ __forceinline__ float ld1(const T* p, int64_t i) {
  if constexpr (sizeof(T) == 2) return __half2float(p[i]);
  else return p[i];
}

template <typename T>
__global__ void __launch_bounds__(kQuantThreads) quantize_rows_kernel(const T* x, int64_t ldx, int64_t rows, int64_t K,
                                                                      int8_t* q, int64_t ldq, float* scale,
                                                                      int64_t lds) {
  __shared__ float part[kQuantThreads / 32];
  __shared__ int nan_seen;
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* xr = x + r * ldx;
    if (threadIdx.x == 0) nan_seen = 0;
    __syncthreads();
    float a = 0x1p-100f;
    bool nan = false;
    for (int64_t i = threadIdx.x; i < K; i += kQuantThreads) {
      const float v = ld1(xr, i);
      nan |= v != v;
      a = fmaxf(a, fabsf(v));
    }
    for (int o = 16; o > 0; o >>= 1) a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = a;
    if (nan) nan_seen = 1;
    __syncthreads();
    for (int w = 0; w < kQuantThreads / 32; ++w) a = fmaxf(a, part[w]);
    if (nan_seen) a = __int_as_float(0x7fffffff);
    const float inv = __fdiv_rn(127.0f, a);
    if (threadIdx.x == 0) scale[r * lds] = __fdiv_rn(a, 127.0f);
    for (int64_t i = threadIdx.x; i < K; i += kQuantThreads) {
      const float v = __fmul_rn(ld1(xr, i), inv);
      q[r * ldq + i] = v == v ? (int8_t)__float2int_rn(v) : (int8_t)0;
    }
    __syncthreads();
  }
}

// Rows on 16-byte boundaries, read once: the TPR threads of a row (a warp, or
// the CTA) hold it in registers as V 16-byte vectors each, up to
// TPR * V * 16 bytes; the at most seven values past the last whole vector
// are one more value on each of the first lanes.  HBM-bound: 32640 rows of
// 2048 float32 (334 MB) take 52 us of device time, of float16 (201 MB) 30 us,
// the rate of a copy (82 us for the float32 rows by the kernel above, which
// reads them twice and serves longer and unaligned rows).
template <typename T>
__device__ __forceinline__ void vec_floats(const uint4 v, float (&f)[16 / sizeof(T)]) {
  if constexpr (sizeof(T) == 2) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 x = __half22float2(h[i]);
      f[2 * i] = x.x;
      f[2 * i + 1] = x.y;
    }
  } else {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
  }
}

// The bits of |v| order like the values, with NaN above infinity, so one
// integer maximum finds the largest magnitude and keeps a NaN.
__device__ __forceinline__ unsigned mag_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The same for the values of a vector (a NaN anywhere gives a NaN); halves
// are compared two at a time, as halves.
template <typename T>
__device__ __forceinline__ unsigned vec_mag(const uint4 v) {
  if constexpr (sizeof(T) == 2) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
    const __half2 m = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
    const float2 f = __half22float2(m);
    return max(mag_bits(f.x), mag_bits(f.y));
  } else {
    return max(max(v.x & 0x7fffffffu, v.y & 0x7fffffffu), max(v.z & 0x7fffffffu, v.w & 0x7fffffffu));
  }
}

__device__ __forceinline__ unsigned q8_sym(float v, float inv) {
  const float p = __fmul_rn(v, inv);
  return (unsigned)(p == p ? __float2int_rn(p) : 0) & 0xffu;
}

template <typename T, int TPR, int V>
__global__ void __launch_bounds__(256, V <= 8 ? 4 : 2) quantize_rows_vec_kernel(const T* x, int64_t ldx, int64_t rows, int K, int8_t* q,
                                                                int64_t ldq, float* scale, int64_t lds) {
  constexpr int N = 16 / sizeof(T), kRows = 256 / TPR;
  __shared__ unsigned part[8];
  const int t = threadIdx.x % TPR, nv = K / N, rest = K - nv * N;
  for (int64_t r = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR; r < rows; r += (int64_t)gridDim.x * kRows) {
    const uint4* xv = reinterpret_cast<const uint4*>(x + r * ldx);
    uint4 v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = t + i * TPR < nv ? __ldcs(xv + t + i * TPR) : make_uint4(0, 0, 0, 0);
    const float tail = t < rest ? ld1(x + r * ldx, nv * N + t) : 0.0f;
    unsigned a = max(mag_bits(tail), 0x0d800000u);   // 2^-100
#pragma unroll
    for (int i = 0; i < V; ++i) a = max(a, vec_mag<T>(v[i]));
    a = __reduce_max_sync(0xffffffffu, a);
    if constexpr (TPR > 32) {
      __syncthreads();   // (the previous row's reads of part)
      if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = a;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < 8; ++w) a = max(a, part[w]);
    }
    const float top = __uint_as_float(a > 0x7f800000u ? 0x7fffffffu : a), inv = __fdiv_rn(127.0f, top);
    if (t == 0) scale[r * lds] = __fdiv_rn(top, 127.0f);
    int8_t* qr = q + r * ldq;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (t + i * TPR < nv) {
        float f[N];
        vec_floats<T>(v[i], f);
        unsigned w[N / 4];
#pragma unroll
        for (int j = 0; j < N / 4; ++j)
          w[j] = q8_sym(f[4 * j], inv) | q8_sym(f[4 * j + 1], inv) << 8 | q8_sym(f[4 * j + 2], inv) << 16 |
                 q8_sym(f[4 * j + 3], inv) << 24;
        if constexpr (N == 4) *reinterpret_cast<unsigned*>(qr + (t + i * TPR) * 4) = w[0];
        else *reinterpret_cast<uint2*>(qr + (t + i * TPR) * 8) = make_uint2(w[0], w[1]);
      }
    if (t < rest) qr[nv * N + t] = (int8_t)q8_sym(tail, inv);
  }
}

template <typename T>
void quantize_run(const T* x, int64_t ldx, int64_t rows, int64_t K, int8_t* q, int64_t ldq, float* scale, int64_t lds,
                  int sms) {
  const int64_t row_bytes = K * (int64_t)sizeof(T);
  const bool one = rows == 1;
  const int64_t qa = 16 / sizeof(T);   // q is written as 4 or 8 bytes at a time
  const bool vec = ((uintptr_t)x & 15) == 0 && (one || ldx * (int64_t)sizeof(T) % 16 == 0) && (uintptr_t)q % qa == 0 &&
                   (one || ldq % qa == 0) && row_bytes <= 256 * 16 * 16;
  cudaStream_t s = cur_stream();
  if (!vec) {
    const int64_t cap = (int64_t)sms * 16;
    quantize_rows_kernel<T><<<(int)(rows < cap ? rows : cap), kQuantThreads, 0, s>>>(x, ldx, rows, K, q, ldq, scale, lds);
    return;
  }
  // a warp a row where its registers hold the row and there are rows enough
  // for eight CTAs on every SM; else a CTA a row (rows of 2048 float32, us of
  // device time by warps / CTAs: 510 rows 3.2 / 2.8, 2400 rows 6.3 / 7.1, 32640
  // rows 52 / 77).  Of the kernels whose registers hold the row, the one with the
  // fewest vectors a thread: 32640 rows of 256 float32 with 2 / 6 vectors 9.2 /
  // 11.7 us, of 768 with 6 / 8 / 16 17.7 / 18.6 / 28.8, of 1024 with 8 / 16 22.6 /
  // 30.2; by CTAs 510 rows of 768 with 1 / 4 2.3 / 2.6, 2000 rows of 4096 with
  // 4 / 8 / 16 7.9 / 8.9 / 14.9.
  const bool warp = row_bytes <= 32 * 16 * 16 && rows > 8 * sms;
  const int tpr = warp ? 32 : 256, per = (int)((row_bytes + tpr * 16 - 1) / (tpr * 16));
  const int64_t want = warp ? (rows + 7) / 8 : rows, cap = (int64_t)sms * 8;
  const int grid = (int)(want < cap ? want : cap);
  auto go = [&](auto kern) { kern<<<grid, 256, 0, s>>>(x, ldx, rows, (int)K, q, ldq, scale, lds); };
  if (warp) {
    if (per <= 2) go(quantize_rows_vec_kernel<T, 32, 2>);
    else if (per <= 6) go(quantize_rows_vec_kernel<T, 32, 6>);
    else if (per <= 8) go(quantize_rows_vec_kernel<T, 32, 8>);
    else go(quantize_rows_vec_kernel<T, 32, 16>);
  } else {
    if (per <= 1) go(quantize_rows_vec_kernel<T, 256, 1>);
    else if (per <= 4) go(quantize_rows_vec_kernel<T, 256, 4>);
    else if (per <= 8) go(quantize_rows_vec_kernel<T, 256, 8>);
    else go(quantize_rows_vec_kernel<T, 256, 16>);
  }
}

// ---- int8 product ----------------------------------------------------------
//   y[m, n] = float(sum_k a[m, k] w[n, k]) * (a_scale[m] * w_scale[n]) (+ bias[n])
// the sum in int32, exact for K <= 131071 (|a w| <= 2^14).
struct MmArgs {
  const int8_t* a;
  const int8_t* w;
  const float* a_scale;
  const float* w_scale;
  const float* bias;   // may be null
  void* out;
  int64_t M, N, K, lda, ldw, ldo;
  int64_t sa, sw, sb;  // strides of the scales and the bias
};

// K = 0: the sum is empty, and no scale makes anything of it.
template <typename TO>
__global__ void __launch_bounds__(256) matmul_empty_kernel(MmArgs A) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < A.M * A.N; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / A.N, n = i % A.N;
    const float y = A.bias ? A.bias[n * A.sb] : 0.0f;
    if constexpr (sizeof(TO) == 2) ((__half*)A.out)[m * A.ldo + n] = __float2half_rn(y);
    else ((float*)A.out)[m * A.ldo + n] = y;
  }
}

// The product on the tensor cores.  Output channels lie along the 128 lanes
// of tensor memory and tokens along its columns: one token is enough to use
// the instruction (a tile of 16 columns), a thread owns one channel, so its
// scale and bias sit in registers, and the 32 lanes of a warp store 32
// neighbouring channels of one token.
//
// A unit -- one CTA (CG = 1), or a pair whose instruction spans both SMs
// (CG = 2) -- walks tiles of 128 * CG channels x NT tokens.  Warp 0 loads
// 128-byte-wide blocks of both operands by TMA into a ring of stages (the
// pair splits the tokens, so each SM loads and reads half of them), warp 1
// issues the matrix instructions, sixteen further warps scale and store from
// one of two accumulators while the next tile fills the other.  What bounds a
// batched projection (32640 x 2048 x 768, us of device time, float16 / float32
// results): loads and products alone take 36 / 36, with the sums read and
// scaled but not stored 43 / 43, with the stores (134, 267 MB) 60 / 74: they
// overlap the rest only in part, and the storing warps wait longest at the
// release of an accumulator, which comes after its stores.  With eight storing
// warps instead of sixteen float16 took 69 us; whole-row and TMA stores from
// shared memory were measured with those eight only (67-71 us).
//
// Where a product has fewer tiles than the GPU has SMs, S CTAs form a cluster
// that splits the summed axis of one tile; each sends its int32 partial sums
// to the CTA that owns the column (shared memory of the cluster), which adds
// and stores them.  Integer sums do not depend on the order.
constexpr int kMmStore = 16, kMmThreads = 64 + 32 * kMmStore;   // storing warps: four for each quarter of the lanes

template <int NT, int CG>
struct MmShape {
  static constexpr int kA = 128 * 128;              // bytes of one stage: channels
  static constexpr int kB = NT / CG * 128;          // and tokens
  static constexpr int kStage = kA + kB;
  static constexpr int kStages = 200 * 1024 / kStage > 8 ? 8 : 200 * 1024 / kStage;
  static constexpr int kCols = 2 * NT;              // tensor memory: two accumulators
  static constexpr int kChunk = NT < 64 ? 16 : 32;  // columns a storing warp takes at a time
  static constexpr int kTok = NT <= 128 ? 32 : NT / 4;   // scales it keeps for its tokens
  static constexpr int kScales = kMmStore * kTok * 4;
  static constexpr int kSmem = 1024 + kStages * kStage + kScales + 512;
};


template <typename TO>
__device__ __forceinline__ void mm_store(TO* p, float v) {
  if constexpr (sizeof(TO) == 2) *p = __float2half_rn(v);
  else *p = v;
}

// Two values of neighbouring tokens, rounded to float16 as a pair (two clocks
// a warp; one value alone takes eight).
template <typename TO>
__device__ __forceinline__ void mm_store2(TO* p, TO* q, float v, float w) {
  if constexpr (sizeof(TO) == 2) {
    const __half2 h = __floats2half2_rn(v, w);
    *p = __low2half(h);
    *q = __high2half(h);
  } else {
    *p = v;
    *q = w;
  }
}

// kChunk columns of an accumulator.
template <int kChunk>
__device__ __forceinline__ void mm_ld(uint32_t at, uint32_t (&r)[kChunk]) {
  if constexpr (kChunk == 16) tmem_ld16(at, r);
  else tmem_ld32(at, r);
}

__device__ __forceinline__ void mm_tile(unsigned t, unsigned tiles_n, unsigned tiles_m, int* tn, int* tm) {
  // bands of eight channel tiles, so that the tiles in flight share both
  // operands' rows in L2
  const unsigned band = t / (8 * tiles_m), r = t - band * 8 * tiles_m;
  const unsigned width = tiles_n - band * 8 < 8 ? tiles_n - band * 8 : 8, m = r / width;
  *tm = (int)m;
  *tn = (int)(band * 8 + r - m * width);
}

// Where a storing warp's part of a tile lies and the scales it needs: its
// channel's, and its tokens' spread over the lanes.  Chunk i of warp group g
// is tokens [(4 i + g) kChunk, + kChunk) of the tile.
template <int NT, int CG>
struct MmTile {
  static constexpr int kTok = MmShape<NT, CG>::kTok / 32, kChunk = MmShape<NT, CG>::kChunk;
  int64_t m0, n0;
  float sw, b, tok[kTok];
  __device__ __forceinline__ void load(const MmArgs& A, unsigned t, unsigned tiles_n, unsigned tiles_m, unsigned rank,
                                       int quad, int group, int lane) {
    int tn, tm;
    mm_tile(t, tiles_n, tiles_m, &tn, &tm);
    m0 = (int64_t)tm * NT;
    n0 = (int64_t)tn * 128 * CG + (CG == 2 ? 128 * (int)rank : 0) + quad * 32;
    const int64_t n = n0 + lane;
    sw = n < A.N ? A.w_scale[n * A.sw] : 0.0f;
    b = n < A.N && A.bias ? A.bias[n * A.sb] : 0.0f;
#pragma unroll
    for (int k = 0; k < kTok; ++k) {
      const int i = lane + 32 * k, c = (i / kChunk * 4 + group) * kChunk + i % kChunk;
      tok[k] = c < NT && m0 + c < A.M ? A.a_scale[(m0 + c) * A.sa] : 0.0f;
    }
  }
};

template <int NT, int CG, typename TO>
__global__ void __launch_bounds__(kMmThreads, 1) matmul_tc_kernel(const __grid_constant__ CUtensorMap map_w,
                                                           const __grid_constant__ CUtensorMap map_a,
                                                           MmArgs A, int S) {
  using Sh = MmShape<NT, CG>;
  extern __shared__ uint8_t smem_raw[];
  const unsigned base = (smem_u32(smem_raw) + 1023) & ~1023u;
  uint8_t* ring = smem_raw + (base - smem_u32(smem_raw));
  uint64_t* full = (uint64_t*)(ring + Sh::kStages * Sh::kStage + Sh::kScales);
  uint64_t* empty = full + Sh::kStages;
  uint64_t* acc_full = empty + Sh::kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* slot = (uint32_t*)(acc_empty + 2);
  volatile int* aborted = (volatile int*)(slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned csize = CG == 2 ? 2 : (unsigned)S;
  const unsigned rank = csize > 1 ? cluster_rank() : 0;
  const bool leader = CG == 1 || rank == 0;
  const unsigned unit = blockIdx.x / csize, units = gridDim.x / csize;
  const unsigned tiles_n = (unsigned)((A.N + 128 * CG - 1) / (128 * CG)), tiles_m = (unsigned)((A.M + NT - 1) / NT);
  const unsigned tiles = tiles_n * tiles_m;   // (the host keeps tiles + units below 2^31)
  const int kblocks = (int)((A.K + 127) / 128);
  const int kb0 = CG == 1 ? (int)((int64_t)kblocks * rank / S) : 0;
  const int kb1 = CG == 1 ? (int)((int64_t)kblocks * (rank + 1) / S) : kblocks;

  if (threadIdx.x == 0) {
    *aborted = 0;
    for (int i = 0; i < Sh::kStages; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full + i, 1);
      mbar_init(acc_empty + i, kMmStore * CG);
    }
    tma_prefetch(&map_w);
    tma_prefetch(&map_a);
  }
  if (warp == 1) tmem_alloc<CG>(slot, Sh::kCols);
  tc_fence_before();
  __syncthreads();
  if (csize > 1) {
    cluster_arrive();
    cluster_wait();
  }
  tc_fence_after();
  const uint32_t tmem = *slot;

  if (warp == 0) {
    if (lane == 0) {
      int st = 0;
      unsigned ph = 0;
      for (unsigned t = unit; t < tiles; t += units) {
        int tn, tm;
        mm_tile(t, tiles_n, tiles_m, &tn, &tm);
        const int n0 = tn * 128 * CG + (CG == 2 ? 128 * (int)rank : 0);
        const int m0 = tm * NT + (CG == 2 ? NT / 2 * (int)rank : 0);
        for (int kb = kb0; kb < kb1; ++kb) {
          tc_wait(empty + st, ph ^ 1, aborted);
          const unsigned dst = base + st * Sh::kStage;
          if (leader) mbar_arrive_expect_tx(full + st, Sh::kStage * CG);
          if constexpr (CG == 1) {
            tma_load2(dst, &map_w, smem_u32(full + st), kb * 128, n0);
            tma_load2(dst + Sh::kA, &map_a, smem_u32(full + st), kb * 128, m0);
          } else {
            const unsigned bar = cluster_addr(smem_u32(full + st), 0);
            tma_load2_pair(dst, &map_w, bar, kb * 128, n0);
            tma_load2_pair(dst + Sh::kA, &map_a, bar, kb * 128, m0);
          }
          if (++st == Sh::kStages) st = 0, ph ^= 1;
        }
      }
      // every stage drained: no arrival is under way when the CTA ends
      for (int i = 0; i < Sh::kStages; ++i) {
        tc_wait(empty + st, ph ^ 1, aborted);
        if (++st == Sh::kStages) st = 0, ph ^= 1;
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      // int32 accumulator, signed 8-bit operands, both K-major
      constexpr uint32_t idesc = 2u << 4 | 1u << 7 | 1u << 10 | (NT / 8u) << 17 | (128u * CG / 16u) << 24;
      int st = 0, buf = 0;
      unsigned ph = 0, aph = 0;
      for (unsigned t = unit; t < tiles; t += units) {
        tc_wait(acc_empty + buf, aph ^ 1, aborted);
        tc_fence_after();
        const uint32_t d = tmem + buf * NT;
        for (int kb = kb0; kb < kb1; ++kb) {
          tc_wait(full + st, ph, aborted);
          tc_fence_after();
          const unsigned sa = base + st * Sh::kStage, sb = sa + Sh::kA;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_i8<CG>(d, smem_desc(sa + 32 * k, 16, 1024), smem_desc(sb + 32 * k, 16, 1024), idesc, kb > kb0 || k > 0);
          if constexpr (CG == 1) mma_commit(empty + st);
          else mma_commit_pair(empty + st);
          if (++st == Sh::kStages) st = 0, ph ^= 1;
        }
        if constexpr (CG == 1) mma_commit(acc_full + buf);
        else mma_commit_pair(acc_full + buf);
        if (++buf == 2) buf = 0, aph ^= 1;
      }
    }
  } else {
    const int quad = warp & 3, group = (warp - 2) >> 2;
    constexpr int kChunk = Sh::kChunk, kTok = MmTile<NT, CG>::kTok;
    float* ts = (float*)(ring + Sh::kStages * Sh::kStage) + (warp - 2) * Sh::kTok;
    int buf = 0;
    unsigned aph = 0;
    MmTile<NT, CG> next;
    if ((CG == 2 || S == 1) && unit < tiles) next.load(A, unit, tiles_n, tiles_m, rank, quad, group, lane);
    for (unsigned t = unit; t < tiles; t += units) {
      if (CG == 1 && S > 1) {
        tc_wait(acc_full + buf, aph, aborted);   // (the cluster finishes below)
        continue;
      }
      // this tile's scales were asked for a tile ago; the next one's are now
      const MmTile<NT, CG> now = next;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kTok; ++i) ts[lane + 32 * i] = now.tok[i];
      __syncwarp();
      if (t + units < tiles) next.load(A, t + units, tiles_n, tiles_m, rank, quad, group, lane);
      const int cols = A.M - now.m0 < NT ? (int)(A.M - now.m0) : NT;
      const bool live = now.n0 + lane < A.N, biased = A.bias != nullptr;
      const float sw = now.sw, b = now.b;
      tc_wait(acc_full + buf, aph, aborted);
      tc_fence_after();
      const uint32_t acc = tmem + buf * NT + ((uint32_t)(quad * 32) << 16);
      TO* out = (TO*)A.out + now.m0 * A.ldo + now.n0 + lane;
      uint32_t r[kChunk];
      int c0 = group * kChunk;
      if (c0 < cols) mm_ld<kChunk>(acc + c0, r);
#pragma unroll 1
      for (int i = 0; c0 < cols; ++i, c0 += 4 * kChunk) {
        tc_loaded(r);
        float y[kChunk];
        const float4* t4 = reinterpret_cast<const float4*>(ts + i * kChunk);
#pragma unroll
        for (int j = 0; j < kChunk; j += 4) {
          const float4 f = t4[j / 4];
          y[j] = __fmul_rn(__int2float_rn((int)r[j]), __fmul_rn(f.x, sw));
          y[j + 1] = __fmul_rn(__int2float_rn((int)r[j + 1]), __fmul_rn(f.y, sw));
          y[j + 2] = __fmul_rn(__int2float_rn((int)r[j + 2]), __fmul_rn(f.z, sw));
          y[j + 3] = __fmul_rn(__int2float_rn((int)r[j + 3]), __fmul_rn(f.w, sw));
        }
        if (biased) {
#pragma unroll
          for (int j = 0; j < kChunk; ++j) y[j] = __fadd_rn(y[j], b);
        }
        // the next chunk's sums are on their way while this one is stored
        if (c0 + 4 * kChunk < cols) mm_ld<kChunk>(acc + c0 + 4 * kChunk, r);
        TO* op = out + c0 * A.ldo;
        if (c0 + kChunk <= cols) {
          if (live) {
#pragma unroll
            for (int j = 0; j < kChunk; j += 2, op += 2 * A.ldo) mm_store2(op, op + A.ldo, y[j], y[j + 1]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < kChunk; ++j, op += A.ldo)
            if (live && c0 + j < cols) mm_store(op, y[j]);
        }
      }
      tc_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 1) mbar_arrive(acc_empty + buf);
        else mbar_arrive_cluster(cluster_addr(smem_u32(acc_empty + buf), 0));
      }
      if (++buf == 2) buf = 0, aph ^= 1;
    }
  }
  __syncwarp();
  if constexpr (CG == 1) {
    if (S > 1) {
      // every CTA of the cluster has its partial sums; the rings are free
      tc_fence_before();
      __syncthreads();
      cluster_arrive();
      cluster_wait();
      tc_fence_after();
      const int per = (NT + S - 1) / S;
      int tn, tm;
      mm_tile(unit, tiles_n, tiles_m, &tn, &tm);
      const int64_t m0 = (int64_t)tm * NT;
      const int cols = A.M - m0 < NT ? (int)(A.M - m0) : NT;
      if (warp >= 2) {
        const int quad = warp & 3;
        constexpr int CH = 16;
#pragma unroll 1
        for (int c0 = ((warp - 2) >> 2) * CH; c0 < cols; c0 += 4 * CH) {
          uint32_t r[CH];
          tmem_ld16(tmem + c0 + ((uint32_t)(quad * 32) << 16), r);
          tc_loaded(r);
#pragma unroll
          for (int j = 0; j < CH; ++j) {
            const int c = c0 + j, owner = c % S;
            if (c < cols) {
              const unsigned a = cluster_addr(base + ((rank * per + c / S) * 128 + quad * 32 + lane) * 4, owner);
              asm volatile("st.shared::cluster.u32 [%0], %1;\n" ::"r"(a), "r"(r[j]) : "memory");
            }
          }
        }
      }
      __syncwarp();
      cluster_arrive();
      cluster_wait();
      if (warp >= 2) {
        const int ch = (threadIdx.x - 64) & 127, first = (warp - 2) >> 2;
        const int64_t n = (int64_t)tn * 128 + ch;
        if (n < A.N) {
          const float sw = A.w_scale[n * A.sw], b = A.bias ? A.bias[n * A.sb] : 0.0f;
          const int* red = (const int*)ring;
          for (int i = first, c = rank + first * S; c < cols; c += 4 * S, i += 4) {
            int acc = 0;
            for (int s = 0; s < S; ++s) acc += red[(s * per + i) * 128 + ch];
            float y = __fmul_rn(__int2float_rn(acc), __fmul_rn(A.a_scale[(m0 + c) * A.sa], sw));
            if (A.bias) y = __fadd_rn(y, b);
            mm_store((TO*)A.out + (m0 + c) * A.ldo + n, y);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*aborted) {   // copies may still be in flight: give them time to land
    const long long t0 = clock64();
    while (clock64() - t0 < 4000000ll) {}
  }
  __syncwarp();
  if constexpr (CG == 2) {   // the pair's last instructions and arrivals are done on both sides
    cluster_arrive();
    cluster_wait();
  }
  if (warp == 1) tmem_free<CG>(tmem, Sh::kCols);
}

template <int NT, int CG, typename TO>
int mm_launch(const MmArgs& A, int S, int sms, const char* what) {
  using Sh = MmShape<NT, CG>;
  CUtensorMap mw, ma;
  const uint64_t dw[2] = {(uint64_t)A.K, (uint64_t)A.N}, da[2] = {(uint64_t)A.K, (uint64_t)A.M};
  const uint64_t sw[1] = {(uint64_t)A.ldw}, sa[1] = {(uint64_t)A.lda};
  const uint32_t bw[2] = {128, 128}, ba[2] = {128, (uint32_t)(NT / CG)};
  int rc;
  if ((rc = tma_map(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, A.w, dw, sw, bw)) ||
      (rc = tma_map(&ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, A.a, da, sa, ba)))
    return rc;
  auto kern = matmul_tc_kernel<NT, CG, TO>;
  static int raised[64] = {};   // per device: the limit only has to be raised once
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !raised[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem);
    if (e != cudaSuccess) return set_error(BT_ECUDA, "%s: shared memory: %s", what, cudaGetErrorString(e));
    if (dev < 64) raised[dev] = 1;
  }
  const int64_t tiles = (A.N + 128 * CG - 1) / (128 * CG) * ((A.M + NT - 1) / NT);
  const int csize = CG == 2 ? 2 : S;
  const int64_t cap = S > 1 ? tiles : sms / CG;
  const int64_t units = tiles < cap ? tiles : cap;
  if (tiles + sms > INT32_MAX || units * csize > INT32_MAX) return set_error(BT_ETOOBIG, "%s: too many output values", what);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * csize));
  cfg.blockDim = dim3(kMmThreads);
  cfg.dynamicSmemBytes = Sh::kSmem;
  cfg.stream = cur_stream();
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)csize, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, mw, ma, A, S);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(BT_ECUDA, "%s: launch failed: %s", what, cudaGetErrorString(e));
  }
  return BT_OK;
}

// The tile and the split with the least estimated time, in SM clocks: a block
// of 128 along the summed axis takes the longer of its matrix instructions
// (8192 products a clock) and its loads (64 bytes a clock); a tile adds its
// stores, a launch its start, a split its exchange.  The estimates are there to
// be compared: they leave out most of what loads from cold and stores take, and
// come to half the time that is measured.  Their choice against every other
// tile and split, us of device time, as tokens of a tile / split (p: a pair):
//   M x N x K              chosen           the others' best
//   1 x 2048 x 768         16/1     5.3     16/6    6.4
//   1 x 8192 x 8192        16/2    18.1     16/1   22.3
//   16 x 768 x 768         16/1     5.3     16/6    7.5
//   64 x 4096 x 4096       64/4    11.1     64/3   12.1    (without a split 12.7)
//   77 x 5001 x 1000       32/1     6.3     64/1    7.0    (with a split 12.3)
//   300 x 3001 x 5120      64/1    16.0     128/1  16.9    (with a split 20.8)
//   510 x 768 x 2048       32/1     8.1     64/1    8.9    (with a split 12.4)
//   510 x 2048 x 768       64/1     6.1     128/1   6.9
//   2048 x 2048 x 512      256p     8.7     256/1   8.0
//   4096 x 4096 x 4096     256p    55       256/1  60
//   8160 x 768 x 2048      256p    19.8     256/1  20.3
//   32640 x 2048 x 768     256p    60       256/1  59      (float32 results: 75, 72)
struct MmChoice {
  int64_t M, N, K;
  int sms, nt, cg, split;
};

void mm_choose(MmChoice& c) {
  const int kblocks = (int)((c.K + 127) / 128);
  double best = 1e300;
  auto consider = [&](int nt, int cg, int s) {
    const double tiles = (double)((c.N + 128 * cg - 1) / (128 * cg)) * (double)((c.M + nt - 1) / nt);
    const double units = cg == 2 ? c.sms / 2 : c.sms / s;
    const double waves = ceil(tiles / units);
    const double mma = 2.0 * nt, load = (16384 + nt * 128 / cg) / 64.0;
    const double per = ceil((double)kblocks / s) * (mma > load ? mma : load);
    const double store = nt * 8.0;
    const double t = 3000 + waves * (per > store ? per : store) + store + (s > 1 ? 2500 + 20.0 * nt : 0);
    if (t < best) best = t, c.nt = nt, c.cg = cg, c.split = s;
  };
  for (int nt = 16; nt <= 256; nt *= 2) {
    if (nt > 16 && c.M <= nt / 2) break;
    consider(nt, 1, 1);
    if (nt <= 128)
      for (int s = 2; s <= 8 && s <= kblocks; ++s) consider(nt, 1, s);
  }
  consider(256, 2, 1);
}

template <typename TO>
int mm_run(const MmArgs& A, int sms, const char* what) {
  // (a thread's products mostly repeat a few sizes)
  static thread_local MmChoice seen[8] = {};
  MmChoice& c = seen[(A.M * 31 + A.N * 7 + A.K) & 7];
  if (c.M != A.M || c.N != A.N || c.K != A.K || c.sms != sms) {
    c.M = A.M, c.N = A.N, c.K = A.K, c.sms = sms;
    mm_choose(c);
  }
  if (c.cg == 2) return mm_launch<256, 2, TO>(A, 1, sms, what);
  switch (c.nt) {
    case 16: return mm_launch<16, 1, TO>(A, c.split, sms, what);
    case 32: return mm_launch<32, 1, TO>(A, c.split, sms, what);
    case 64: return mm_launch<64, 1, TO>(A, c.split, sms, what);
    case 128: return mm_launch<128, 1, TO>(A, c.split, sms, what);
    default: return mm_launch<256, 1, TO>(A, c.split, sms, what);
  }
}

// The rows of a view: all leading axes as one axis of constant stride, the
// last axis of unit stride.
int rows_of(const bt_tensor* t, const char* what, const char* name, int64_t* rows, int64_t* cols, int64_t* ld) {
  if (t->rank < 1) return set_error(BT_ESHAPE, "%s: %s needs at least one axis", what, name);
  const int last = t->rank - 1;
  *cols = t->shape[last];
  if (*cols > 1 && t->strides[last] != 1)
    return set_error(BT_EUNSUPPORTED, "%s: the last axis of %s must have unit stride", what, name);
  int64_t n = 1, stride = 0;
  for (int d = last - 1; d >= 0; --d) {
    if (t->shape[d] != 1) {
      if (n == 1) stride = t->strides[d];
      else if (t->strides[d] != stride * n && n > 0)
        return set_error(BT_EUNSUPPORTED, "%s: the rows of %s must have one stride", what, name);
    }
    n *= t->shape[d];
  }
  *rows = n;
  *ld = stride;
  return BT_OK;
}

int vec_of(const bt_tensor* t, const char* what, const char* name, int64_t n, const float** p, int64_t* stride) {
  int rc = check_tensor(t, name, false);
  if (rc) return rc;
  if (t->dtype != BT_F32) return set_error(BT_EDTYPE, "%s: %s must be float32", what, name);
  if (t->rank != 1 || t->shape[0] != n)
    return set_error(BT_ESHAPE, "%s: %s must have shape [%lld]", what, name, (long long)n);
  *p = (const float*)t->data;
  *stride = t->strides[0];
  return BT_OK;
}

}  // namespace

cudaError_t proj_timeouts(unsigned int* sum) { return take_timeouts(sum); }

}  // namespace bt

using namespace bt;

extern "C" int bt_quantize_rows(const bt_tensor* x, const bt_tensor* q, const bt_tensor* scale) {
  const char* what = "bt_quantize_rows";
  int rc;
  if ((rc = check_tensor(x, "x", false)) || (rc = check_tensor(q, "q", false))) return rc;
  if (x->dtype != BT_F32 && x->dtype != BT_F16) return set_error(BT_EDTYPE, "%s: x must be float32 or float16", what);
  if (q->dtype != BT_I8) return set_error(BT_EDTYPE, "%s: q must be int8", what);
  int64_t rows, K, ldx, qrows, qk, ldq;
  if ((rc = rows_of(x, what, "x", &rows, &K, &ldx)) || (rc = rows_of(q, what, "q", &qrows, &qk, &ldq))) return rc;
  if (qrows != rows || qk != K) return set_error(BT_ESHAPE, "%s: x and q must have the same rows", what);
  if (K == 0) return set_error(BT_ESHAPE, "%s: rows without values have no largest value", what);
  const float* sp;
  int64_t lds;
  if ((rc = vec_of(scale, what, "scale", rows, &sp, &lds))) return rc;
  if (rows == 0) return BT_OK;
  DevInfo di;
  if ((rc = dev_info(&di))) return rc;
  if (x->dtype == BT_F32)
    quantize_run((const float*)x->data, ldx, rows, K, (int8_t*)q->data, ldq, (float*)sp, lds, di.sm_count);
  else
    quantize_run((const __half*)x->data, ldx, rows, K, (int8_t*)q->data, ldq, (float*)sp, lds, di.sm_count);
  return check_launch(what);
}

extern "C" int bt_matmul_int8(const bt_tensor* a, const bt_tensor* a_scale, const bt_tensor* w,
                              const bt_tensor* w_scale, const bt_tensor* bias, const bt_tensor* out) {
  const char* what = "bt_matmul_int8";
  int rc;
  if ((rc = check_tensor(a, "a", false)) || (rc = check_tensor(w, "w", false)) ||
      (rc = check_tensor(out, "out", false)))
    return rc;
  if (a->dtype != BT_I8 || w->dtype != BT_I8) return set_error(BT_EDTYPE, "%s: a and w must be int8", what);
  if (out->dtype != BT_F32 && out->dtype != BT_F16)
    return set_error(BT_EDTYPE, "%s: out must be float32 or float16", what);
  MmArgs A;
  int64_t k2, m2, n2;
  if ((rc = rows_of(a, what, "a", &A.M, &A.K, &A.lda)) || (rc = rows_of(w, what, "w", &A.N, &k2, &A.ldw)) ||
      (rc = rows_of(out, what, "out", &m2, &n2, &A.ldo)))
    return rc;
  if (w->rank != 2) return set_error(BT_ESHAPE, "%s: w must have two axes", what);
  if (k2 != A.K) return set_error(BT_ESHAPE, "%s: a has %lld values a row, w %lld", what, (long long)A.K, (long long)k2);
  if (m2 != A.M || n2 != A.N) return set_error(BT_ESHAPE, "%s: out must have a's rows of w's row count", what);
  if (A.K > 131071) return set_error(BT_ETOOBIG, "%s: more than 131071 values a row could overflow the int32 sum", what);
  if ((rc = vec_of(a_scale, what, "a_scale", A.M, &A.a_scale, &A.sa)) ||
      (rc = vec_of(w_scale, what, "w_scale", A.N, &A.w_scale, &A.sw)))
    return rc;
  A.bias = nullptr;
  A.sb = 0;
  if (bias && (rc = vec_of(bias, what, "bias", A.N, &A.bias, &A.sb))) return rc;
  if (A.M == 0 || A.N == 0) return BT_OK;
  A.a = (const int8_t*)a->data;
  A.w = (const int8_t*)w->data;
  A.out = out->data;
  DevInfo di;
  if (A.K == 0) {
    if ((rc = dev_info(&di))) return rc;
    const int64_t want = (A.M * A.N + 255) / 256, cap = (int64_t)di.sm_count * 8;
    const int grid = (int)(want < cap ? want : cap);
    if (out->dtype == BT_F32) matmul_empty_kernel<float><<<grid, 256, 0, cur_stream()>>>(A);
    else matmul_empty_kernel<__half><<<grid, 256, 0, cur_stream()>>>(A);
    return check_launch(what);
  }
  if (A.M > INT32_MAX - 256 || A.N > INT32_MAX - 256) return set_error(BT_ETOOBIG, "%s: more than 2^31 rows", what);
  // one row has no stride to speak of: any that a tensor map takes
  if (A.M == 1) A.lda = (A.K + 15) / 16 * 16;
  if (A.N == 1) A.ldw = (A.K + 15) / 16 * 16;
  if ((((uintptr_t)A.a | (uintptr_t)A.w) & 15) || A.lda <= 0 || A.ldw <= 0 || (A.lda & 15) || (A.ldw & 15))
    return set_error(BT_EUNSUPPORTED, "%s: the rows of a and w must start on 16-byte boundaries", what);
  if ((rc = dev_info(&di))) return rc;
  return out->dtype == BT_F32 ? mm_run<float>(A, di.sm_count, what) : mm_run<__half>(A, di.sm_count, what);
}

// bt_attn.cu -- attention of queries over keys and values of another length
// (bt_attention): out = softmax(scale q k^T) v, row by row over the keys that
// take part.
//
// Per query row, one pass over the keys with the running maximum m, the
// running sum l and the unnormalised output o, all float32:
//   m' = max(m, s_j),  l' = l e^(m - m') + e^(s_j - m'),
//   o' = o e^(m - m') + e^(s_j - m') v_j
// and out = o / l, or 0 where no key takes part.  A key outside lengths or
// the mask is never looked at: its score is replaced, not added to, and its
// value row is left out, so NaN or infinities stored there have no effect.
// Where every key that takes part scores -inf, l is 0 and the row 0 / 0: a
// maximum of -inf does not mean that no key took part, so that is kept apart.
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <type_traits>
#include "bt_ops.h"
#include "bt_internal.h"
#include "bt_pk.h"
#include "bt_tc.h"

namespace bt {
namespace {

constexpr int kMaxHeadDim = 128;

struct AttnArgs {
  const void *q, *k, *v;
  void* out;
  const void* lengths;      // [B] int32 / int64, may be null
  const uint8_t* mask;      // [B, Tk] bool, may be null
  int64_t B, H, G, Tq, Tk;  // G = query heads per key head
  int32_t D, len64;
  int64_t qs[4], ks[4], vs[4], os[4];   // element strides of [B, H, T, D]
  int64_t len_stride, mask_sb, mask_sk;
  float scale;
};

__device__ __forceinline__ int64_t keys_of(const AttnArgs& A, int64_t b) {
  int64_t n = A.Tk;
  if (A.lengths) {
    n = A.len64 ? ((const int64_t*)A.lengths)[b * A.len_stride] : ((const int32_t*)A.lengths)[b * A.len_stride];
    n = n < 0 ? 0 : n > A.Tk ? A.Tk : n;
  }
  return n;
}

template <typename T>
__device__ __forceinline__ float ldf(const T* p) {
  if constexpr (sizeof(T) == 2) return __half2float(*p);
  else return *p;
}

// 2^x by the special-function unit (relative error 2^-22.5; results below
// 2^-126 become 0).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A row's result is a mean of float16 values, so never larger than they are;
// but rounded weights over an unrounded sum (up to 2^-11 of it) or a long
// float32 sum may put it past the largest one's rounding range.  Only an
// infinity among the values is one in the result.
__device__ __forceinline__ __half half_mean(float y) {
  const float a = fabsf(y);
  return __float2half_rn(a > 65504.0f && a < INFINITY ? copysignf(65504.0f, y) : y);
}

// One warp per query row, any strides: a lane scores one key of 32, then the
// lanes share the output's dimensions.
constexpr int kRowWarps = 4;

template <typename T>
__global__ void __launch_bounds__(32 * kRowWarps) attn_rows_kernel(AttnArgs A, int64_t rows) {
  __shared__ float qsh[kRowWarps][kMaxHeadDim];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  for (int64_t r = (int64_t)blockIdx.x * kRowWarps + w; r < rows; r += (int64_t)gridDim.x * kRowWarps) {
    const int64_t t = r % A.Tq, h = r / A.Tq % A.H, b = r / A.Tq / A.H, hk = h / A.G;
    const T* qp = (const T*)A.q + b * A.qs[0] + h * A.qs[1] + t * A.qs[2];
    const T* kp = (const T*)A.k + b * A.ks[0] + hk * A.ks[1];
    const T* vp = (const T*)A.v + b * A.vs[0] + hk * A.vs[1];
    __syncwarp();
    for (int d = lane; d < A.D; d += 32) qsh[w][d] = ldf(qp + d * A.qs[3]);
    __syncwarp();
    const int64_t n = keys_of(A, b);
    float m = -INFINITY, l = 0.0f, o[kMaxHeadDim / 32] = {};
    bool any = false;   // a key took part
    for (int64_t j0 = 0; j0 < n; j0 += 32) {
      const int64_t j = j0 + lane;
      const bool in = j < n && (!A.mask || A.mask[b * A.mask_sb + j * A.mask_sk]);
      unsigned live = __ballot_sync(0xffffffffu, in);
      if (!live) continue;
      any = true;
      float s = -INFINITY;
      if (in) {
        float dot = 0.0f;
        for (int d = 0; d < A.D; ++d) dot = __fmaf_rn(qsh[w][d], ldf(kp + j * A.ks[2] + d * A.ks[3]), dot);
        s = dot;   // (scaled as a difference to the maximum: the product alone may overflow)
      }
      float mx = s;
      for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float mn = fmaxf(m, mx), base = mn == -INFINITY ? 0.0f : mn;
      const float keep = expf((m - base) * A.scale), p = in ? expf((s - base) * A.scale) : 0.0f;
      m = mn;
      float sum = p;
      for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      l = l * keep + sum;
#pragma unroll
      for (int i = 0; i < kMaxHeadDim / 32; ++i) o[i] *= keep;
      while (live) {
        const int x = __ffs(live) - 1;
        live &= live - 1;
        const float px = __shfl_sync(0xffffffffu, p, x);
        const T* vr = vp + (j0 + x) * A.vs[2];
#pragma unroll
        for (int i = 0; i < kMaxHeadDim / 32; ++i)
          if (lane + 32 * i < A.D) o[i] = __fmaf_rn(px, ldf(vr + (lane + 32 * i) * A.vs[3]), o[i]);
      }
    }
    T* op = (T*)A.out + b * A.os[0] + h * A.os[1] + t * A.os[2];
#pragma unroll
    for (int i = 0; i < kMaxHeadDim / 32; ++i)
      if (lane + 32 * i < A.D) {
        const float y = any ? __fdiv_rn(o[i], l) : 0.0f;
        if constexpr (sizeof(T) == 2) op[(lane + 32 * i) * A.os[3]] = half_mean(y);
        else op[(lane + 32 * i) * A.os[3]] = y;
      }
  }
}


// ---- float16 on the tensor cores --------------------------------------------
// A work item is two tiles of 128 queries of one head (256 rows, so that a
// key tile read once serves both); CTAs walk the items.  Tensor memory holds
// for each tile the 128 x 128 float32 scores S of the current key tile, the
// float16 weights P (D <= 64: beside S; else over S) and the 128 x D output O.
//   warps 0-3, 4-7  softmax of tile 0, 1: a thread owns a query row, reads its
//                   128 scores into registers (216 of them: the other warps
//                   give theirs up), writes its weights
//   warps 8, 9      issue tile 0's, 1's S = Q K^T and O += P V (P read from
//                   tensor memory)
//   warp 10         TMA loads: the item's Q tiles, a ring of K and V tiles
//   warp 11         zeroes the rows of V whose keys take no part (only where
//                   there are lengths or a mask: a weight of 0 times NaN
//                   would not be 0)
// With P beside S the next scores are computed while the softmax still works
// on these; else the tiles overlap each other.  The softmax bounds it: its
// exponentials alone take 1024 clocks a 128 x 128 tile, the tensor cores 512
// (D = 64) or 1024 (D = 128), and with two warps a scheduler the latencies
// between them show.  So tile 0 and 1 take turns at the exponentials (each
// then has the special-function unit to itself while the other waits, reads
// and compares: 134 -> 120 us at 16 heads of 4096 x 4096 x 64).  Measured
// beside those 120 us and not taken: blocks of 64 keys with two score buffers a
// tile (174 us: each block has a fixed part), two threads a row (144 us),
// scores read twice instead of kept (157 us), the maximum found along with the
// weights and these redone where it grew (162 us).  There it takes 111 us now,
// 617 TFLOP/s, and at D = 128 136 us, 1.01 PFLOP/s, at 1965 MHz (149 us after
// seconds at the power limit, at 1790 MHz).
//
// Softmax: with c = scale log2(e) and a reference value m per row,
// p = 2^(s c - m c + 7).  m is the row's running maximum, but it moves (and O
// and the sum are rescaled) only when the maximum has grown by more than 2^8
// in p: rescaling O costs a pass over tensor memory, and p <= 2^15 stays in
// float16's range.  The 2^7 lifts small weights off float16's subnormals: a
// weight loses precision only below 2^-21 of the reference.  The exponent is
// one fma of the score with 7 - m c, whose rounding is an error of up to 2^-14
// while m c is below 2^11, and grows with it: to a factor past float16's range
// at 2^24.  A row beyond 2^11 subtracts m from its scores first: a vote a key
// tile (4096 queries of 16 heads over 16384 keys of 128: 489 -> 496 us), and in
// warps with such a row a pass over the scores (590 us if every warp made it,
// as a part of the exponents).  P is rounded to
// float16 (the tensor cores' operand; relative error 2^-11 a weight, as a
// float16 result has anyway); the row's sum is of the float32 weights.
constexpr int kTile = 128;
constexpr int kAttnThreads = 384;
constexpr float kGrow = 8.0f, kLift = 7.0f, kFar = 2048.0f;

struct AttnTc {
  AttnArgs a;
  int32_t q_mul[2], k_mul[2], v_mul[2];   // 0 where an axis (head, batch) is broadcast
  int32_t q_tiles;                        // items of a head
  int32_t step_t, step_h, step_b;         // the grid's size in items, heads and batch entries
  uint32_t items;
  int32_t wide;                           // out: 2 by TMA stores, 1 rows of 16-byte pieces, 0 neither
};

template <int DP>
struct AttnShape {
  static constexpr int kPanel = kTile * 128;               // 128 rows of 64 values
  static constexpr int kPanels = DP / 64;
  static constexpr int kRows = kPanel * kPanels;           // one tile of Q, K or V
  static constexpr int kSlots = DP == 64 ? 8 : 4;          // ring of K and V tiles
  static constexpr bool kBeside = DP == 64;                // P beside S
  static constexpr int kP = kBeside ? 256 : 0;             // tensor memory: S at 0, 128
  static constexpr int kPStep = kBeside ? 64 : 128;
  static constexpr int kO = kBeside ? 384 : 256;
  static constexpr bool kStage = DP == 64;                 // room for results on their way out
  static constexpr int kSmem = 1024 + (2 + kSlots + (kStage ? 2 : 0)) * kRows + 512;
};

// The valid keys of a key tile as four words; all ones where every key is.
__device__ __forceinline__ unsigned tail_word(int left, int i) {   // keys left from the tile's start
  const int n = left - 32 * i;
  return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
}

// The scores of keys that take no part become -inf.
__device__ __forceinline__ void only(uint32_t (&s)[32], unsigned w) {
#pragma unroll
  for (int j = 0; j < 32; ++j) s[j] = w >> j & 1 ? s[j] : 0xff800000u;
}

// The largest of three, NaN if one of them is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// The same operations where they are written: the order is the schedule.
__device__ __forceinline__ float2 pk_fma_v(float2 a, float2 b, float2 c) {
  float2 d;
  asm volatile("{\n\t.reg .b64 ra, rb, rc, rd;\n\tmov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
               "mov.b64 rc, {%6, %7};\n\tfma.rn.f32x2 rd, ra, rb, rc;\n\tmov.b64 {%0, %1}, rd;\n\t}"
               : "=f"(d.x), "=f"(d.y)
               : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ void ex2_v(float& x) { asm volatile("ex2.approx.ftz.f32 %0, %0;" : "+f"(x)); }
__device__ __forceinline__ uint32_t cvt_v(float2 x) {
  uint32_t h;
  asm volatile("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(h) : "f"(x.y), "f"(x.x));
  return h;
}

// The walk of a CTA over its items: item it is query tile pair t of head h of
// batch entry b; the next one is gridDim.x on, in steps that the host has
// split the same way, so that a step is three sums with carries.  The keys of
// the next item are asked for an item ahead: the load's latency would stand
// before each item.
struct Items {
  uint32_t it;
  int t, h, b, n;
  int t0;   // first query
  __device__ __forceinline__ explicit Items(const AttnTc& A) : it(blockIdx.x) {
    const uint32_t head = it / (uint32_t)A.q_tiles;
    t = (int)(it - head * (uint32_t)A.q_tiles);
    b = (int)(head / (uint32_t)A.a.H);
    h = (int)(head - (uint32_t)b * (uint32_t)A.a.H);
    n = (int)keys_of(A.a, b);   // (a CTA has an item)
    t0 = t * 2 * kTile;
    ask(A);
  }
  __device__ __forceinline__ bool live(const AttnTc& A) const { return it < A.items; }
  __device__ __forceinline__ void next(const AttnTc& A) {
    it += gridDim.x;
    t = t2, h = h2, b = b2, n = n_next;
    t0 = t * 2 * kTile;
    ask(A);
  }

 private:
  int t2, h2, b2, n_next;
  __device__ __forceinline__ void ask(const AttnTc& A) {
    t2 = t + A.step_t, h2 = h + A.step_h, b2 = b + A.step_b;
    if (t2 >= A.q_tiles) t2 -= A.q_tiles, ++h2;
    if (h2 >= (int)A.a.H) h2 -= (int)A.a.H, ++b2;
    n_next = it + gridDim.x < A.items ? (int)keys_of(A.a, b2) : 0;
  }
};

// A warp's rows again, where a result overflowed (see half_mean): into `at`,
// `step` apart, or, with swizzle >= 0, a staged row whose 16-byte pieces lie
// at their index xor swizzle.  A call, so that it costs the walk of the items
// next to nothing (inlined, 64 x 12 heads over 510 keys took 88.0 us against
// 86.8, and 86.1 without the test for overflows).
__device__ __noinline__ void store_overflows(uint32_t op, float inv, bool mine, int D, __half* at, int64_t step, int swizzle) {
#pragma unroll 1
  for (int i = 0; i < D; ++i) {
    const float y = tmem_ld1(op + i) * inv;
    if (mine && fabsf(y) > 65504.0f && fabsf(y) < INFINITY) at[swizzle < 0 ? i * step : i ^ swizzle << 3] = half_mean(y);
  }
}

template <int DP>
__global__ void __launch_bounds__(kAttnThreads, 1)
    attn_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                   const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_out,
                   const __grid_constant__ AttnTc A) {
  using Sh = AttnShape<DP>;
  extern __shared__ uint8_t smem_raw[];
  const unsigned base = (smem_u32(smem_raw) + 1023) & ~1023u;
  uint8_t* smem = smem_raw + (base - smem_u32(smem_raw));
  const unsigned ring = base + 2 * Sh::kRows;
  uint64_t* bars = (uint64_t*)(smem + (2 + Sh::kSlots + (Sh::kStage ? 2 : 0)) * Sh::kRows);
  uint64_t *q_full = bars, *q_empty = bars + 2, *s_full = bars + 4, *s_free = bars + 6, *p_full = bars + 8;
  uint64_t* pv_done = bars + 10;   // [tile][key tile's parity]: two, so that a phase may pass unwaited for
  uint64_t *kv_full = bars + 14, *kv_empty = kv_full + Sh::kSlots, *v_ok = kv_empty + Sh::kSlots;
  uint32_t* slot = (uint32_t*)(v_ok + Sh::kSlots);
  volatile int* aborted = (volatile int*)(slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const AttnArgs& a = A.a;
  const bool fix_v = a.lengths || a.mask;
  if (threadIdx.x == 0) {
    *aborted = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + i, 1);
      mbar_init(q_empty + i, 1);
      mbar_init(pv_done + 2 * i, 1);
      mbar_init(pv_done + 2 * i + 1, 1);
      mbar_init(s_full + i, 1);
      mbar_init(s_free + i, 4);
      mbar_init(p_full + i, 4);
    }
    for (int i = 0; i < Sh::kSlots; ++i) {
      mbar_init(kv_full + i, 1);
      mbar_init(kv_empty + i, 2);
      mbar_init(v_ok + i, 1);
    }
    tma_prefetch(&map_q);
    tma_prefetch(&map_k);
    tma_prefetch(&map_v);
  }
  if (warp == 8) tmem_alloc<1>(slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *slot;

  if (warp < 8) {
    const int tile = warp >> 2;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;\n");   // 256 x 216 + 128 x 72 = 384 x 168
    const uint32_t sp = tmem + tile * kTile + lanes, pp = tmem + Sh::kP + tile * Sh::kPStep + lanes;
    const uint32_t op = tmem + Sh::kO + tile * DP + lanes;
    const float c = a.scale * 1.4426950408889634f;   // log2(e)
    // Tile 0 and 1 take turns at the exponentials (see above): a warpgroup
    // waits for its turn and then passes it on, tile 0 first.
    auto my_turn = [&]() { asm volatile("bar.sync %0, 256;\n" ::"r"(1 + tile) : "memory"); };
    auto your_turn = [&]() { asm volatile("bar.arrive %0, 256;\n" ::"r"(2 - tile) : "memory"); };
    if (tile == 1) your_turn();
    uint32_t g = 0;   // key tiles this query tile has worked on
    for (Items pos(A); pos.live(A); pos.next(A)) {
      const int n = pos.n;
      const int64_t t = pos.t0 + tile * kTile + (warp & 3) * 32 + lane;
      if (pos.t0 + tile * kTile >= a.Tq) continue;
      const bool turns = pos.t0 + kTile < a.Tq;   // both tiles have work
      const uint8_t* mask = a.mask ? a.mask + pos.b * a.mask_sb : nullptr;
      float m = -INFINITY;          // the reference (-inf: no key yet)
      float off = 0.0f, ref = 0.0f;   // p = 2^((s - ref) c + off)
      float2 l = {0.0f, 0.0f};
      bool any = false;   // a key took part
      uint8_t mb[4] = {1, 1, 1, 1};
      if (mask)
#pragma unroll
        for (int i = 0; i < 4; ++i) mb[i] = 32 * i + lane < n ? mask[(int64_t)(32 * i + lane) * a.mask_sk] : 0;
      for (int k0 = 0; k0 < n; k0 += kTile, ++g) {
        unsigned w[4] = {~0u, ~0u, ~0u, ~0u};
        bool part = n - k0 < kTile;
        if (mask) {
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = __ballot_sync(0xffffffffu, mb[i] != 0);
          part = (w[0] & w[1] & w[2] & w[3]) != ~0u;
          any |= (w[0] | w[1] | w[2] | w[3]) != 0;
          // the next tile's bytes, while this one is computed
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int k = k0 + kTile + 32 * i + lane;
            mb[i] = k < n ? mask[(int64_t)k * a.mask_sk] : 0;
          }
        } else if (part) {
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = tail_word(n - k0, i);
        }
        tc_wait(s_full + tile, g & 1, aborted);
        tc_fence_after();
        uint32_t s[4][32];
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld32(sp + 32 * i, s[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) tc_loaded(s[i]);
        if constexpr (Sh::kBeside) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(s_free + tile);
        }
        if (part) {
#pragma unroll
          for (int i = 0; i < 4; ++i) only(s[i], w[i]);
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < 32; j += 2)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx[i] = max3(mx[i], __uint_as_float(s[i][j]), __uint_as_float(s[i][j + 1]));
        float top = max3(max3(mx[0], mx[1], mx[2]), mx[3], -INFINITY);
        // a NaN among the scores, or +inf (inf - inf), makes the row NaN by
        // way of its reference; the comparisons below are true for NaN
        const bool grow = !(top <= m) && (m == -INFINITY || !((top - m) * c <= kGrow));
        // (asked for here, needed below)
        const bool p_free = !Sh::kBeside || k0 == 0 || mbar_try(smem_u32(pv_done + 2 * tile + ((g - 1) & 1)), (g - 1) >> 1 & 1);
        if (__any_sync(0xffffffffu, grow)) {
          if (top == INFINITY) top = NAN;
          // where there was no key before, O and l are 0 or not yet written
          const float keep = grow ? (m == -INFINITY ? 0.0f : exp2f((m - top) * c)) : 1.0f;
          if (grow) {
            m = top;
            off = fmaf(top, -c, kLift);
            const bool far = fabsf(off) > kFar;
            ref = far ? top : 0.0f;
            off = far ? kLift : off;
            l.x *= keep;
            l.y *= keep;
          }
          if (k0 > 0) {
            tc_wait(pv_done + 2 * tile + ((g - 1) & 1), (g - 1) >> 1 & 1, aborted);   // O holds every key tile before
            tc_fence_after();
            // (a few columns at a time: the 128 scores stay in registers)
#pragma unroll 1
            for (int i = 0; i < DP; i += 16) {
              uint32_t o[16];
              tmem_ld16(op + i, o);
              tc_loaded(o);
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * keep);
              tmem_st16(op + i, o);
            }
          }
        }
        if (__any_sync(0xffffffffu, ref != 0.0f)) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 32; ++j) s[i][j] = __float_as_uint(__uint_as_float(s[i][j]) - ref);
        }
        if (turns) my_turn();
        const float2 c2 = {c, c}, off2 = {off, off};
        float2 part_l[2] = {};
        // Pair x is scaled in step x, exponentiated in step x + 1, summed and
        // rounded in step x + 3, in this order (volatile): the special-function
        // unit takes eight clocks an instruction, and what is issued between
        // two of its instructions is free.  (A quarter of the exponentials as
        // polynomials on the FMA pipe instead measured slower: 126 against
        // 120 us at 16 heads of 4096 x 4096 x 64.)
        float2 e[64];
        uint32_t p[4][16];
#pragma unroll
        for (int x = 0; x < 64 + 3; ++x) {
          if (x < 64)
            e[x] = pk_fma_v(make_float2(__uint_as_float(s[x / 16][x % 16 * 2]), __uint_as_float(s[x / 16][x % 16 * 2 + 1])), c2, off2);
          if (x >= 1 && x <= 64) ex2_v(e[x - 1].x);
          if (x >= 3) part_l[x & 1] = pk_add(part_l[x & 1], e[x - 3]);
          if (x >= 1 && x <= 64) ex2_v(e[x - 1].y);
          if (x >= 3) {
            const int y = x - 3;
            p[y / 16][y % 16] = cvt_v(e[y]);
            if (y % 16 == 15) {
              // (P beside S: the last product has read its weights by now)
              if (y == 15 && !p_free) tc_wait(pv_done + 2 * tile + ((g - 1) & 1), (g - 1) >> 1 & 1, aborted);
              tmem_st16(pp + y / 16 * 16, p[y / 16]);   // column j: keys 2 j and 2 j + 1
            }
          }
        }
        if (turns) your_turn();
        l = pk_add(l, pk_add(part_l[0], part_l[1]));
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + tile);
      }
      // the result: O / l
      const float sum = l.x + l.y;
      const bool none = mask ? !any : n == 0;
      const float inv = 1.0f / sum;
      __half* out = (__half*)a.out + pos.b * a.os[0] + pos.h * a.os[1] + t * a.os[2];
      if (n > 0) {
        // (s_full of the last key tile came after the product two before it,
        // so only the last two are open, one on each barrier)
        tc_wait(pv_done + 2 * tile + ((g - 1) & 1), (g - 1) >> 1 & 1, aborted);
        tc_fence_after();
      }
      uint32_t over[2] = {};   // NaN once a result is not finite (infinity times 0)
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) {
        if (32 * i >= a.D) break;
        uint32_t o[32];
        if (n > 0) {
          tmem_ld32(op + 32 * i, o);
          tc_loaded(o);
        }
        uint32_t y[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          // (the select keeps a row without keys 0 whatever O holds)
          const __half2 h = none ? __floats2half2_rn(0.0f, 0.0f)
                                        : __floats2half2_rn(__uint_as_float(o[2 * j]) * inv, __uint_as_float(o[2 * j + 1]) * inv);
          y[j] = *reinterpret_cast<const uint32_t*>(&h);
          asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(over[j & 1]) : "r"(y[j]), "r"(0u));
        }
        if (Sh::kStage && A.wide == 2) {
          // a row of 128 bytes, its 16-byte pieces where the store's swizzle
          // has them
          const int row = (warp & 3) * 32 + lane;
          if (i == 0) {   // (the last item's store has read the tile: its issuer waited, all wait for the issuer)
            if (row == 0) bulk_wait_read<0>();
            asm volatile("bar.sync %0, 128;\n" ::"r"(3 + tile) : "memory");
          }
          uint8_t* at = smem + (2 + Sh::kSlots + tile) * Sh::kRows + row * 128;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<uint4*>(at + (((4 * i + j) ^ (row & 7)) << 4)) =
                make_uint4(y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]);
        } else if (t < a.Tq) {
          const int left = a.D - 32 * i;
          if (A.wide) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (8 * j < left)
                *reinterpret_cast<uint4*>(out + 32 * i + 8 * j) = make_uint4(y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]);
          } else {
            const __half* e = reinterpret_cast<const __half*>(y);
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j < left) out[(int64_t)(32 * i + j) * a.os[3]] = e[j];
          }
        }
      }
      if (__any_sync(0xffffffffu, ((over[0] | over[1]) & 0x7fff7fffu) != 0)) {
        const int row = (warp & 3) * 32 + lane;
        const bool staged = Sh::kStage && A.wide == 2;
        store_overflows(op, inv, !none && (staged || t < a.Tq), a.D,
                        staged ? reinterpret_cast<__half*>(smem + (2 + Sh::kSlots + tile) * Sh::kRows + row * 128) : out,
                        a.os[3], staged ? row & 7 : -1);
      }
      if (Sh::kStage && A.wide == 2) {
        fence_async_shared();
        asm volatile("bar.sync %0, 128;\n" ::"r"(3 + tile) : "memory");
        if ((warp & 3) == 0 && lane == 0) {
          tma_store4(&map_out, base + (2 + Sh::kSlots + tile) * Sh::kRows, 0, pos.t0 + tile * kTile, pos.h, pos.b);
          bulk_commit();
        }
      }
      tc_fence_before();   // (O is read before this warp's next arrival lets it be written)
    }
  } else if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;\n");
  }
  if (warp == 8 || warp == 9) {
    // The whole warp walks the loop and one elected lane issues: the operands
    // are then known to be uniform (with the loop on one lane, issuing sixteen
    // products took 3300 clocks).
    constexpr uint32_t id_s = 1u << 4 | (kTile / 8u) << 17 | (kTile / 16u) << 24;
    constexpr uint32_t id_o = 1u << 4 | 1u << 16 | (DP / 8u) << 17 | (kTile / 16u) << 24;   // V: rows along the sum
    const int i = warp - 8;
    const uint32_t ts = tmem + i * kTile, tp = tmem + Sh::kP + i * Sh::kPStep, to = tmem + Sh::kO + i * DP;
    const uint64_t dq = smem_desc(base + i * Sh::kRows, 16, 1024);   // (the low bits are the address / 16)
    unsigned q_ph = 0;
    uint32_t g = 0, r = 0;   // key tiles scored; K and V tiles used so far: K tile j of an item is r + 2 j, its V the one after
    auto score = [&](uint32_t kt, bool first, bool last) {
      const uint32_t slot_k = kt % Sh::kSlots;
      if (first) {
        tc_wait(q_full + i, q_ph, aborted);
        q_ph ^= 1;
      }
      tc_wait(kv_full + slot_k, kt / Sh::kSlots & 1, aborted);
      if (Sh::kBeside && g > 0) tc_wait(s_free + i, (g - 1) & 1, aborted);
      tc_fence_after();
      const uint64_t dk = smem_desc(ring + slot_k * Sh::kRows, 16, 1024);
      if (elect_one()) {
#pragma unroll
        for (int x = 0; x < DP / 16; ++x) {
          constexpr int kStep = Sh::kPanel / 16;
          mma_f16_ss(ts, dq + (x / 4 * kStep + x % 4 * 2), dk + (x / 4 * kStep + x % 4 * 2), id_s, x > 0);
        }
        mma_commit(s_full + i);
        mma_commit(kv_empty + slot_k);
        if (last) mma_commit(q_empty + i);
      }
      __syncwarp();
      ++g;
    };
    for (Items pos(A); pos.live(A); pos.next(A)) {
      const int nb = (pos.n + kTile - 1) / kTile;
      if (pos.t0 + i * kTile >= a.Tq) {   // no such tile in this item: pass its keys on
        for (int j = 0; j < 2 * nb; ++j, ++r) {
          tc_wait(kv_full + r % Sh::kSlots, r / Sh::kSlots & 1, aborted);
          if (lane == 0) mbar_arrive(kv_empty + r % Sh::kSlots);
          __syncwarp();
        }
        continue;
      }
      if (nb > 0) score(r, true, nb == 1);
      for (int j = 0; j < nb; ++j, r += 2) {
        const bool last = j == nb - 1;
        const uint32_t slot_v = (r + 1) % Sh::kSlots, b = g - 1;
        if (Sh::kBeside && !last) score(r + 2, false, j + 1 == nb - 1);
        tc_wait((fix_v ? v_ok : kv_full) + slot_v, (r + 1) / Sh::kSlots & 1, aborted);
        tc_wait(p_full + i, b & 1, aborted);
        tc_fence_after();
        const uint64_t dv = smem_desc(ring + slot_v * Sh::kRows, Sh::kPanel, 1024);
        if (elect_one()) {
#pragma unroll
          for (int x = 0; x < kTile / 16; ++x) mma_f16_ts(to, tp + 8 * x, dv + 128 * x, id_o, j > 0 || x > 0);
          mma_commit(pv_done + 2 * i + (b & 1));
          mma_commit(kv_empty + slot_v);
        }
        __syncwarp();
        if (!Sh::kBeside && !last) score(r + 2, false, j + 1 == nb - 1);
      }
    }
  } else if (warp == 10) {
    if (lane == 0) {
      unsigned q_ph[2] = {1, 1};
      uint32_t g = 0;
      for (Items pos(A); pos.live(A); pos.next(A)) {
        const int nb = (pos.n + kTile - 1) / kTile;
        if (nb == 0) continue;
        const int tiles = pos.t0 + kTile < a.Tq ? 2 : 1, b = pos.b, hk = pos.h / (int)a.G;
        auto load = [&](const CUtensorMap* m, unsigned dst, uint64_t* bar, int t0, int h, int bb) {
          mbar_arrive_expect_tx(bar, Sh::kRows);
#pragma unroll
          for (int x = 0; x < Sh::kPanels; ++x) tma_load4(dst + x * Sh::kPanel, m, smem_u32(bar), 64 * x, t0, h, bb);
        };
        for (int i = 0; i < tiles; ++i) {
          tc_wait(q_empty + i, q_ph[i], aborted);
          q_ph[i] ^= 1;
          load(&map_q, base + i * Sh::kRows, q_full + i, pos.t0 + i * kTile, pos.h * A.q_mul[0], b * A.q_mul[1]);
        }
        for (int j = 0; j < nb; ++j) {
          for (int y = 0; y < 2; ++y, ++g) {
            const int sl = (int)(g % Sh::kSlots);
            tc_wait(kv_empty + sl, (g / Sh::kSlots & 1) ^ 1, aborted);
            load(y ? &map_v : &map_k, ring + sl * Sh::kRows, kv_full + sl, j * kTile, hk * (y ? A.v_mul : A.k_mul)[0],
                 b * (y ? A.v_mul : A.k_mul)[1]);
          }
        }
      }
      for (int i = 0; i < Sh::kSlots; ++i, ++g)   // every tile used: no arrival is under way when the CTA ends
        tc_wait(kv_empty + g % Sh::kSlots, (g / Sh::kSlots & 1) ^ 1, aborted);
      for (int i = 0; i < 2; ++i) tc_wait(q_empty + i, q_ph[i], aborted);
    }
  } else if (warp == 11 && fix_v) {
    uint32_t g = 1;
    for (Items pos(A); pos.live(A); pos.next(A)) {
      const int n = pos.n;
      const uint8_t* mask = a.mask ? a.mask + pos.b * a.mask_sb : nullptr;
      // which of this lane's four rows of a key tile take no part
      auto look = [&](int k0) {
        unsigned out = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int k = k0 + 32 * i + lane;
          if (!(k < n && (!mask || mask[(int64_t)k * a.mask_sk]))) out |= 1u << i;
        }
        return out;
      };
      unsigned next = look(0);
      for (int k0 = 0; k0 < n; k0 += kTile, g += 2) {
        const unsigned out = next;
        next = look(k0 + kTile);
        const int sl = (int)(g % Sh::kSlots);
        tc_wait(kv_full + sl, g / Sh::kSlots & 1, aborted);
        if (__any_sync(0xffffffffu, out != 0)) {
          // a lane clears its row's 128 bytes piece by piece, each lane
          // beginning at another one, so that no two meet in a bank
          uint8_t* at = smem + (2 + sl) * Sh::kRows + lane * 128;
#pragma unroll 1
          for (int i = 0; i < 4; ++i, at += 32 * 128)
            if (out >> i & 1) {
#pragma unroll
              for (int x = 0; x < Sh::kPanels; ++x)
#pragma unroll
                for (int y = 0; y < 8; ++y)
                  *reinterpret_cast<uint4*>(at + x * Sh::kPanel + ((y + lane & 7) << 4)) = make_uint4(0, 0, 0, 0);
            }
          fence_async_shared();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(v_ok + sl);
      }
    }
  }
  if (Sh::kStage && warp < 8 && (warp & 3) == 0 && lane == 0) bulk_wait_all();
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (*aborted) {   // copies may still be in flight: give them time to land
    const long long t0 = clock64();
    while (clock64() - t0 < 4000000ll) {}
  }
  if (warp == 8) tmem_free<1>(tmem, 512);
}

// ---- few queries ---------------------------------------------------------------
// A step of generation: the queries that share a key head (Tq of each of its
// G query heads) are rows of one or a few 16-row tiles, and the time is that
// of reading K and V once.  A warp takes 16 keys at a time, fetched a step or
// two ahead into a ring of its own (cp.async), as operands of 16 x 8 x 16
// products (far below the tensor cores' rate here):
//   S = Q K^T  the order of the summed dims is free, so a lane's 16 bytes of a
//              key row are dims 8c..8c+7 of two products, Q permuted alike;
//   O += P V   a lane holds dims 8q..8q+7 of the four keys its weights belong
//              to, and pairs the keys' values register by register; the
//              order of the result's columns is free as well.
// Warps, and the CTAs of a cluster, share the keys out and join their
// (maximum, sum, O) at the end, in a fixed order: through shared memory, and
// the cluster's shared memory.  No workspace, one launch.
constexpr int kFewRows = 16, kFewRows32 = 4;

__device__ __forceinline__ void mma_16x8x16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A part of the result in shared memory: ROWS rows of partial O, each with its
// maximum and sum behind it; one for each warp.
template <int DP, int ROWS, int W>
struct FewShape {
  static constexpr int kO = DP / 8;                           // 8-column tiles of O
  static constexpr int kPitch = DP + 4;
  static constexpr int kPart = ROWS * kPitch;                 // floats
  static constexpr int kSmem = W * kPart * 4;
  // the float16 form's ring: 16 rows of K, then of V, for each step; the parts
  // lie over it at the end.  32 x 16 heads, one query, 2000 keys of 64: 46 us
  // with two steps (5.7 TB/s), 52 with three, 62 with four; 8 x 8 key heads,
  // 8192 keys of 128: 72 us with two, 62 with three
  static constexpr int kSteps = DP == 64 ? 2 : 3, kRow = DP * 2, kStep = 2 * 16 * kRow;
  static constexpr int kRing = W * kSteps * kStep;
};

// Joins the parts of all warps of the CTA, or of the cluster (each CTA then
// takes the rows r = rank mod S), and stores the outputs.  The parts' O are
// lifted by `lift` against their sums.  A part whose keys all scored -inf has
// that maximum and a sum of NaN, one without keys a sum of 0.
template <int DP, int ROWS, int W, typename T>
__device__ __forceinline__ void few_join(const AttnArgs& A, float* sm, int S, int rank, int64_t b, int64_t hk, int64_t row0,
                                         float cs, float lift) {
  using Sh = FewShape<DP, ROWS, W>;
  __syncthreads();
  if (S > 1) {
    cluster_arrive();
    cluster_wait();
  }
  const unsigned sm_addr = smem_u32(sm);
  const int64_t rows = A.G * A.Tq;
  for (int i = threadIdx.x; i < ROWS * DP; i += 32 * W) {
    const int r = i / DP, d = i % DP;
    const int64_t gr = row0 + r;
    if (d >= A.D || gr >= rows || r % S != rank) continue;
    auto at = [&](int k, int w, int col) {
      const int off = w * Sh::kPart + r * Sh::kPitch + col;
      if (S == 1) return sm[off];
      float v;
      asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(cluster_addr(sm_addr + off * 4, k)) : "memory");
      return v;
    };
    float mx = -INFINITY;
    for (int k = 0; k < S; ++k)
      for (int w = 0; w < W; ++w) mx = max3(mx, at(k, w, DP), -INFINITY);
    float num = 0.0f, den = 0.0f;
    for (int k = 0; k < S; ++k)
      for (int w = 0; w < W; ++w) {
        const float pm = at(k, w, DP);
        if (pm == -INFINITY) {
          if (mx == -INFINITY) den += at(k, w, DP + 1);
          continue;
        }
        const float f = exp2f((pm - mx) * cs);
        num = fmaf(at(k, w, d), f, num);
        den = fmaf(at(k, w, DP + 1), f, den);
      }
    const float y = mx == -INFINITY ? den : num / (den * lift);
    T* out = (T*)A.out + b * A.os[0] + (hk * A.G + gr / A.Tq) * A.os[1] + gr % A.Tq * A.os[2];
    if constexpr (sizeof(T) == 2) out[d * A.os[3]] = half_mean(y);
    else out[d * A.os[3]] = y;
  }
  if (S > 1) {   // no CTA of the cluster leaves while its shared memory is read
    __syncwarp();
    cluster_arrive();
    cluster_wait();
  }
}

template <int DP, int W>
__global__ void __launch_bounds__(32 * W) attn_few_kernel(const __grid_constant__ AttnArgs A, int S, int row_tiles) {
  using Sh = FewShape<DP, kFewRows, W>;
  extern __shared__ __align__(16) float few_sm[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, q = lane >> 2, c = lane & 3;
  const unsigned part = S > 1 ? cluster_rank() : 0;
  uint32_t u = blockIdx.x / (unsigned)S;
  const int rt = (int)(u % (unsigned)row_tiles);
  u /= (unsigned)row_tiles;
  const int64_t Hk = A.H / A.G, b = u / (uint32_t)Hk, hk = u - b * Hk;
  const int64_t rows = A.G * A.Tq;
  const int n = (int)keys_of(A, b);
  const uint8_t* mask = A.mask ? A.mask + b * A.mask_sb : nullptr;
  const __half* kp = (const __half*)A.k + b * A.ks[0] + hk * A.ks[1];
  const __half* vp = (const __half*)A.v + b * A.vs[0] + hk * A.vs[1];

  // Q: rows q and q + 8 of the tile, dims 32 x + 8 c ..
  uint32_t qa[DP / 16][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t r = (int64_t)rt * kFewRows + q + 8 * h;
    const __half* qp = (const __half*)A.q + b * A.qs[0] + (hk * A.G + r / A.Tq) * A.qs[1] + r % A.Tq * A.qs[2];
#pragma unroll
    for (int x = 0; x < DP / 32; ++x) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (r < rows && 32 * x + 8 * c < A.D) v = *reinterpret_cast<const uint4*>(qp + 32 * x + 8 * c);
      qa[2 * x][h] = v.x;
      qa[2 * x][2 + h] = v.y;
      qa[2 * x + 1][h] = v.z;
      qa[2 * x + 1][2 + h] = v.w;
    }
  }
  float o[Sh::kO][4] = {};
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  bool any = false;   // a key took part
  const float cs = A.scale * 1.4426950408889634f;   // log2(e)

  // this CTA's keys: whole steps of 16, as even as they go
  const int steps = (n + 15) / 16;
  const int s0 = (int)((int64_t)steps * part / S), s1 = (int)((int64_t)steps * (part + 1) / S);
  // the ring: a row's 16-byte pieces are permuted so that the reads below meet
  // no bank twice (K: eight lanes read four pieces of two neighbouring rows;
  // V: two pieces of every other row)
  const unsigned ring = smem_u32(few_sm) + warp * (Sh::kSteps * Sh::kStep);
  auto fetch = [&](int st, int slot) {
    if (st < s1) {
      constexpr int kPieces = DP / 8;
#pragma unroll
      for (int i = 0; i < 16 * kPieces / 32; ++i) {
        const int piece = lane + 32 * i, row = piece / kPieces, ch = piece % kPieces, key = 16 * st + row;
        const int bytes = key < n && 8 * ch < A.D ? 16 : 0;
        const int64_t ko = bytes ? key * A.ks[2] + 8 * ch : 0, vo = bytes ? key * A.vs[2] + 8 * ch : 0;
        const unsigned at = ring + slot * Sh::kStep + row * Sh::kRow;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(at + ((ch ^ ((row & 1) << 2 | (row >> 1 & 3))) << 4)),
                     "l"(kp + ko), "r"(bytes)
                     : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(at + 16 * Sh::kRow + ((ch ^ (row & 7)) << 4)),
                     "l"(vp + vo), "r"(bytes)
                     : "memory");
      }
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  };
  auto piece = [&](unsigned at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
  };
#pragma unroll
  for (int i = 0; i < Sh::kSteps - 1; ++i) fetch(s0 + warp + i * W, i);
  for (int st = s0 + warp, slot = 0; st < s1; st += W, slot = slot + 1 == Sh::kSteps ? 0 : slot + 1) {
    const int k0 = 16 * st;
    fetch(st + (Sh::kSteps - 1) * W, slot == 0 ? Sh::kSteps - 1 : slot - 1);
    asm volatile("cp.async.wait_group %0;\n" ::"n"(Sh::kSteps - 1) : "memory");
    __syncwarp();
    const unsigned kt = ring + slot * Sh::kStep, vt = kt + 16 * Sh::kRow;
    uint4 kr[2][DP / 32], vr[4][DP / 64];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int x = 0; x < DP / 32; ++x)
        kr[h][x] = piece(kt + (8 * h + q) * Sh::kRow + (((4 * x + c) ^ ((q & 1) << 2 | (q >> 1 & 3))) << 4));
    bool in[4] = {true, true, true, true};   // keys 2 c, 2 c + 1 of each eight
    if (mask || k0 + 16 > n) {
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int key = k0 + 2 * c + (y & 1) + 8 * (y >> 1);
        in[y] = key < n && (!mask || mask[key * A.mask_sk]);
      }
    }
    any |= in[0] | in[1] | in[2] | in[3];
    float s[2][4] = {};
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int x = 0; x < DP / 32; ++x) {
        mma_16x8x16(s[h], qa[2 * x], kr[h][x].x, kr[h][x].y);
        mma_16x8x16(s[h], qa[2 * x + 1], kr[h][x].z, kr[h][x].w);
      }
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int row = 2 * c + (y & 1) + 8 * (y >> 1);
#pragma unroll
      for (int x = 0; x < DP / 64; ++x) vr[y][x] = piece(vt + row * Sh::kRow + (((8 * x + q) ^ (row & 7)) << 4));
    }
    __syncwarp();   // (the step is read: its place may be filled)
    // scores of rows q (s[.][0, 1]) and q + 8 (s[.][2, 3]), keys 2 c, 2 c + 1 of each eight
    if (mask || k0 + 16 > n) {
#pragma unroll
      for (int y = 0; y < 4; ++y)
        if (!in[y]) {
          s[y >> 1][y & 1] = s[y >> 1][2 + (y & 1)] = -INFINITY;
#pragma unroll
          for (int x = 0; x < DP / 64; ++x) vr[y][x] = make_uint4(0, 0, 0, 0);   // whatever V holds there
        }
    }
    uint32_t pa[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {   // row q + 8 h
      // (a NaN score makes the maximum, and so the row, NaN)
      float top = max3(max3(s[0][2 * h], s[0][2 * h + 1], s[1][2 * h]), s[1][2 * h + 1], m[h]);
      top = max3(top, __shfl_xor_sync(0xffffffffu, top, 1), -INFINITY);
      const float mn = max3(top, __shfl_xor_sync(0xffffffffu, top, 2), -INFINITY);
      // (the reference is subtracted before the scaling: as a scaled and rounded
      // product of a large score it would lift a weight past float16's range)
      const float base = mn == -INFINITY ? 0.0f : mn;
      if (__any_sync(0xffffffffu, !(mn <= m[h]))) {
        const float keep = ex2((m[h] - base) * cs);   // (m = -inf: 0)
        m[h] = mn;
        l[h] *= keep;
#pragma unroll
        for (int i = 0; i < Sh::kO; ++i) {
          o[i][2 * h] *= keep;
          o[i][2 * h + 1] *= keep;
        }
      }
      float p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[e] = ex2((s[e >> 1][2 * h + (e & 1)] - base) * cs);
        l[h] += p[e];
      }
      // weights as float16, lifted by 2^7 off its subnormals (the sum is of
      // the unrounded ones, lifted alike where the parts are joined)
      const __half2 h0 = __floats2half2_rn(p[0] * 128.0f, p[1] * 128.0f), h1 = __floats2half2_rn(p[2] * 128.0f, p[3] * 128.0f);
      pa[h] = *reinterpret_cast<const uint32_t*>(&h0);
      pa[2 + h] = *reinterpret_cast<const uint32_t*>(&h1);
    }
#pragma unroll
    for (int x = 0; x < DP / 64; ++x) {
      const uint32_t* v0 = &vr[0][x].x;
      const uint32_t* v1 = &vr[1][x].x;
      const uint32_t* v2 = &vr[2][x].x;
      const uint32_t* v3 = &vr[3][x].x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {   // dims 64 x + 8 q + 2 i and + 1
        mma_16x8x16(o[8 * x + 2 * i], pa, __byte_perm(v0[i], v1[i], 0x5410), __byte_perm(v2[i], v3[i], 0x5410));
        mma_16x8x16(o[8 * x + 2 * i + 1], pa, __byte_perm(v0[i], v1[i], 0x7632), __byte_perm(v2[i], v3[i], 0x7632));
      }
    }
  }
  any = __any_sync(0xffffffffu, any);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    if (any && m[h] == -INFINITY) l[h] = NAN;
  }
  asm volatile("cp.async.wait_group 0;\n" ::: "memory");
  __syncthreads();   // every warp is done with its ring
  // the warp's part: O[row][dim], then the maximum and the sum.  Column 2 c + e
  // of 8-column tile 8 x + j is dim 64 x + 8 (2 c + e) + j.
  float* mine = few_sm + warp * Sh::kPart;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float* row = mine + (q + 8 * h) * Sh::kPitch;
#pragma unroll
    for (int i = 0; i < Sh::kO; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) row[64 * (i / 8) + 8 * (2 * c + e) + i % 8] = o[i][2 * h + e];
    if (c == 0) {
      row[DP] = m[h];
      row[DP + 1] = l[h];
    }
  }
  few_join<DP, kFewRows, W, __half>(A, few_sm, S, (int)part, b, hk, (int64_t)rt * kFewRows, cs, 128.0f);
}

// The float32 form, for rows of up to 4 queries at a time: eight lanes share a
// key (a lane holds dims 4 (x + 8 y) .. of Q, K, V and O), four keys a warp
// step, each of the four lane groups with its own maximum, sum and O.
template <int DP, int W>
__global__ void __launch_bounds__(32 * W) attn_few32_kernel(const __grid_constant__ AttnArgs A, int S, int row_tiles) {
  using Sh = FewShape<DP, kFewRows32, W>;
  constexpr int R = kFewRows32, Y = DP / 32, kAhead = DP == 64 ? 4 : 2;   // steps of four keys loaded together
  extern __shared__ __align__(16) float few_sm[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, x = lane & 7, grp = lane >> 3;
  const unsigned part = S > 1 ? cluster_rank() : 0;
  uint32_t u = blockIdx.x / (unsigned)S;
  const int rt = (int)(u % (unsigned)row_tiles);
  u /= (unsigned)row_tiles;
  const int64_t Hk = A.H / A.G, b = u / (uint32_t)Hk, hk = u - b * Hk;
  const int64_t rows = A.G * A.Tq;
  const int n = (int)keys_of(A, b);
  const uint8_t* mask = A.mask ? A.mask + b * A.mask_sb : nullptr;
  const float* kp = (const float*)A.k + b * A.ks[0] + hk * A.ks[1];
  const float* vp = (const float*)A.v + b * A.vs[0] + hk * A.vs[1];
  const float cs = A.scale * 1.4426950408889634f;   // log2(e)
  auto ld4 = [&](const float* p, int y, bool in) {
    const int d = 4 * (x + 8 * y);
    return in && d < A.D ? __ldg(reinterpret_cast<const float4*>(p + d)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  };
  float4 q[R][Y], o[R][Y] = {};
  float m[R], l[R] = {};
  bool any = false;   // a key took part
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t gr = (int64_t)rt * R + r;
    m[r] = -INFINITY;
#pragma unroll
    for (int y = 0; y < Y; ++y)
      q[r][y] = ld4((const float*)A.q + b * A.qs[0] + (hk * A.G + gr / A.Tq) * A.qs[1] + gr % A.Tq * A.qs[2], y, gr < rows);
  }
  // this CTA's keys: whole steps
  constexpr int kStep = 4 * kAhead;
  const int steps = (n + kStep - 1) / kStep;
  const int s0 = (int)((int64_t)steps * part / S), s1 = (int)((int64_t)steps * (part + 1) / S);
  for (int st = s0 + warp; st < s1; st += W) {
    float4 k[kAhead][Y], v[kAhead][Y];
    bool in[kAhead];
#pragma unroll
    for (int t = 0; t < kAhead; ++t) {
      const int key = kStep * st + 4 * t + grp;
      in[t] = key < n && (!mask || mask[key * A.mask_sk]);
      any |= in[t];
#pragma unroll
      for (int y = 0; y < Y; ++y) {
        k[t][y] = ld4(kp + key * A.ks[2], y, key < n);
        v[t][y] = ld4(vp + key * A.vs[2], y, key < n);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if ((int64_t)rt * R + r >= rows) break;
      float s[kAhead], mn = m[r];
#pragma unroll
      for (int t = 0; t < kAhead; ++t) {
        float a = 0.0f;
#pragma unroll
        for (int y = 0; y < Y; ++y) {
          a = fmaf(q[r][y].x, k[t][y].x, a);
          a = fmaf(q[r][y].y, k[t][y].y, a);
          a = fmaf(q[r][y].z, k[t][y].z, a);
          a = fmaf(q[r][y].w, k[t][y].w, a);
        }
        a += __shfl_xor_sync(0xffffffffu, a, 1);
        a += __shfl_xor_sync(0xffffffffu, a, 2);
        a += __shfl_xor_sync(0xffffffffu, a, 4);
        s[t] = in[t] ? a : -INFINITY;
        mn = max3(mn, s[t], -INFINITY);
      }
      const float base = mn == -INFINITY ? 0.0f : mn;
      const float keep = ex2((m[r] - base) * cs);
      m[r] = mn;
      l[r] *= keep;
#pragma unroll
      for (int y = 0; y < Y; ++y) o[r][y] = make_float4(o[r][y].x * keep, o[r][y].y * keep, o[r][y].z * keep, o[r][y].w * keep);
#pragma unroll
      for (int t = 0; t < kAhead; ++t) {
        const float p = ex2((s[t] - base) * cs);
        l[r] += p;
        if (!in[t]) continue;   // whatever V holds there
#pragma unroll
        for (int y = 0; y < Y; ++y) {
          o[r][y].x = fmaf(p, v[t][y].x, o[r][y].x);
          o[r][y].y = fmaf(p, v[t][y].y, o[r][y].y);
          o[r][y].z = fmaf(p, v[t][y].z, o[r][y].z);
          o[r][y].w = fmaf(p, v[t][y].w, o[r][y].w);
        }
      }
    }
  }
  // the four lane groups of the warp become one part
  float* mine = few_sm + warp * Sh::kPart;
  any = __any_sync(0xffffffffu, any);
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int z = 8; z <= 16; z *= 2) {
      const float om = __shfl_xor_sync(0xffffffffu, m[r], z), mn = max3(m[r], om, -INFINITY);
      const float keep = m[r] == -INFINITY ? 0.0f : exp2f((m[r] - mn) * cs);
      m[r] = mn;
      l[r] *= keep;
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], z);
#pragma unroll
      for (int y = 0; y < Y; ++y) {
        float* e = &o[r][y].x;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          e[w] *= keep;
          e[w] += __shfl_xor_sync(0xffffffffu, e[w], z);
        }
      }
    }
    if (grp == 0) {
#pragma unroll
      for (int y = 0; y < Y; ++y) *reinterpret_cast<float4*>(mine + r * Sh::kPitch + 4 * (x + 8 * y)) = o[r][y];
      if (x == 0) {
        mine[r * Sh::kPitch + DP] = m[r];
        mine[r * Sh::kPitch + DP + 1] = any && m[r] == -INFINITY ? NAN : l[r];
      }
    }
  }
  few_join<DP, R, W, float>(A, few_sm, S, (int)part, b, hk, (int64_t)rt * R, cs, 1.0f);
}

// ---- float32 --------------------------------------------------------------------
// A CTA holds 128 query rows of a head and walks the keys 64 at a time, all
// arithmetic float32 on the FMA pipe.  Thread (rg, kg) of 16 x 16 owns rows
// rg + 16 i: of S the keys kg + 16 j, of O the dims 4 kg .. + 3 (+ 64), so a
// row's maximum is a reduction over sixteen lanes and its rescaling stays with
// its owner.  Products run two lanes at a time (fma.f32x2): S along pairs of
// the summed dims, added at the end; O along pairs of dims, with each weight
// stored twice.  So Q, K and V lie in shared memory as they come, rows of
// dims, 16 bytes a read.  P is exchanged inside the half-warp that owns its
// rows.  K and V tiles arrive by cp.async (16 bytes, or 4 for any strides;
// rows of keys that take no part are filled with zeros), for dims up to 64
// the next tile while this one is worked on.  Bound by the FMA pipe.
// Measured: 37 TFLOP/s at 8 x 16 heads of 1024 x 1024 x 64, half of the FMA
// pipe's rate, and 172 us at 8 x 12 heads of up to 510 x 510 x 64 (three rounds
// of CTAs); 8 x 8 sums a thread with two CTAs of 128 threads on an SM came to
// the same (36 TFLOP/s, 175 us).
constexpr int kRows32 = 128, kKeys32 = 64, kThreads32 = 256;

template <int DP>
struct Shape32 {
  static constexpr int kD = DP + 4;                     // pitch: 16-byte reads of 8 rows fall into different banks
  static constexpr int kP = 2 * kKeys32 + 4;            // a row of weights, each twice
  static constexpr int kQ = kRows32 * kD, kKt = kKeys32 * kD, kPt = kRows32 * kP;
  static constexpr int kBufs = DP == 64 ? 2 : 1;
  static constexpr int kSmem = (kQ + kPt + kBufs * 2 * kKt) * 4;
};

template <int N>
__device__ __forceinline__ void cp_async_or_zero(unsigned dst, const float* src, bool in) {
  if constexpr (N == 4) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(in ? 4 : 0) : "memory");
}

template <int DP, int N>   // N: values a copy (4 where every row is 16-byte pieces)
__global__ void __launch_bounds__(kThreads32, 1) attn_f32_kernel(const __grid_constant__ AttnArgs A, int q_tiles, int S) {
  using Sh = Shape32<DP>;
  constexpr int J = DP / 64;
  extern __shared__ __align__(16) float sm32[];
  float* qs = sm32;
  float* ps = qs + Sh::kQ;
  float* kv = ps + Sh::kPt;
  const int tid = threadIdx.x, lane = tid & 31, kg = lane & 15, rg = tid >> 4;
  const unsigned rank = S > 1 ? cluster_rank() : 0;
  const uint32_t cta = blockIdx.x / (unsigned)S, u = cta / (unsigned)q_tiles;
  const int64_t t0 = (int64_t)(cta % (unsigned)q_tiles) * kRows32;
  const int64_t b = u / (uint32_t)A.H, h = u - b * A.H, hk = h / A.G;
  const int n = (int)keys_of(A, b), D = A.D;
  const uint8_t* mask = A.mask ? A.mask + b * A.mask_sb : nullptr;
  const float* qp = (const float*)A.q + b * A.qs[0] + h * A.qs[1] + t0 * A.qs[2];
  const float* kp = (const float*)A.k + b * A.ks[0] + hk * A.ks[1];
  const float* vp = (const float*)A.v + b * A.vs[0] + hk * A.vs[1];
  const int rows = A.Tq - t0 < kRows32 ? (int)(A.Tq - t0) : kRows32;
  const float cs = A.scale * 1.4426950408889634f;   // log2(e)

  // a thread copies the same dims of every (kThreads32 / kCols)-th row
  constexpr int kCols = DP / N, kStep = kThreads32 / kCols;
  const int d0 = tid % kCols * N, r0 = tid / kCols;
  const bool dim = d0 < D;
  for (int r = r0; r < kRows32; r += kStep) {
    const bool in = r < rows && dim;
    cp_async_or_zero<N>(smem_u32(qs + r * Sh::kD + d0), in ? qp + r * A.qs[2] + d0 * A.qs[3] : qp, in);
  }
  auto fetch = [&](int k0, int buf) {
    float* ks = kv + buf * 2 * Sh::kKt;
#pragma unroll 4
    for (int r = r0; r < kKeys32; r += kStep) {
      const int key = k0 + r;
      const bool in = key < n && dim, live = in && (!mask || mask[key * A.mask_sk]);
      cp_async_or_zero<N>(smem_u32(ks + r * Sh::kD + d0), in ? kp + key * A.ks[2] + d0 * A.ks[3] : kp, in);
      cp_async_or_zero<N>(smem_u32(ks + Sh::kKt + r * Sh::kD + d0), live ? vp + key * A.vs[2] + d0 * A.vs[3] : vp, live);
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  };

  float2 o[8][2 * J] = {};
  float m[8], l[8] = {};
  bool any = false;   // a key took part
#pragma unroll
  for (int i = 0; i < 8; ++i) m[i] = -INFINITY;
  // this CTA's keys: whole tiles
  const int key_tiles = (n + kKeys32 - 1) / kKeys32;
  const int first = (int)((int64_t)key_tiles * rank / S) * kKeys32, end = (int)((int64_t)key_tiles * (rank + 1) / S) * kKeys32;
  if (first < end) fetch(first, 0);
  for (int k0 = first, buf = 0; k0 < end; k0 += kKeys32) {
    const float* ks = kv + buf * 2 * Sh::kKt;
    const float* vs = ks + Sh::kKt;
    asm volatile("cp.async.wait_group 0;\n" ::: "memory");
    __syncthreads();   // this tile is there, and the last one is read by nobody any more
    if (Sh::kBufs == 2 && k0 + kKeys32 < end) fetch(k0 + kKeys32, buf ^ 1);
    bool in[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int key = k0 + kg + 16 * j;
      in[j] = key < n && (!mask || mask[key * A.mask_sk]);
      any |= in[j];
    }
    const int left = n - k0 < kKeys32 ? n - k0 : kKeys32;
    float2 s2[8][4] = {};
    auto score = [&](auto groups) {   // of every sixteen keys, the first `groups`
      constexpr int kGroups = decltype(groups)::value;
#pragma unroll(DP == 64 ? 2 : 1)
      for (int d = 0; d < D; d += 4) {
        float4 kk[kGroups];
#pragma unroll
        for (int j = 0; j < kGroups; ++j) kk[j] = *reinterpret_cast<const float4*>(ks + (kg + 16 * j) * Sh::kD + d);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 qq = *reinterpret_cast<const float4*>(qs + (rg + 16 * i) * Sh::kD + d);
#pragma unroll
          for (int j = 0; j < kGroups; ++j) {
            s2[i][j] = pk_fma(make_float2(qq.x, qq.y), make_float2(kk[j].x, kk[j].y), s2[i][j]);
            s2[i][j] = pk_fma(make_float2(qq.z, qq.w), make_float2(kk[j].z, kk[j].w), s2[i][j]);
          }
        }
      }
    };
    if (left > 16) score(std::integral_constant<int, 4>());
    else score(std::integral_constant<int, 1>());
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float s[4], mn = m[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[j] = in[j] ? s2[i][j].x + s2[i][j].y : -INFINITY;
        mn = max3(mn, s[j], -INFINITY);
      }
#pragma unroll
      for (int z = 1; z < 16; z *= 2) mn = max3(mn, __shfl_xor_sync(0xffffffffu, mn, z), -INFINITY);
      const float base = mn == -INFINITY ? 0.0f : mn;
      if (mn != m[i]) {   // (a NaN maximum too)
        const float keep = ex2((m[i] - base) * cs);
        m[i] = mn;
        l[i] *= keep;
#pragma unroll
        for (int j = 0; j < 2 * J; ++j) o[i][j] = make_float2(o[i][j].x * keep, o[i][j].y * keep);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float p = ex2((s[j] - base) * cs);
        l[i] += p;
        *reinterpret_cast<float2*>(ps + (rg + 16 * i) * Sh::kP + 2 * (kg + 16 * j)) = make_float2(p, p);
      }
    }
    __syncwarp();
#pragma unroll 2
    for (int k = 0; k < left; k += 2) {   // (weights past the last key are 0, value rows zeros)
      float4 v0[J], v1[J];
#pragma unroll
      for (int j = 0; j < J; ++j) {
        v0[j] = *reinterpret_cast<const float4*>(vs + k * Sh::kD + 4 * kg + 64 * j);
        v1[j] = *reinterpret_cast<const float4*>(vs + (k + 1) * Sh::kD + 4 * kg + 64 * j);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 pp = *reinterpret_cast<const float4*>(ps + (rg + 16 * i) * Sh::kP + 2 * k);
#pragma unroll
        for (int j = 0; j < J; ++j) {
          o[i][2 * j] = pk_fma(make_float2(pp.x, pp.y), make_float2(v0[j].x, v0[j].y), o[i][2 * j]);
          o[i][2 * j + 1] = pk_fma(make_float2(pp.x, pp.y), make_float2(v0[j].z, v0[j].w), o[i][2 * j + 1]);
          o[i][2 * j] = pk_fma(make_float2(pp.z, pp.w), make_float2(v1[j].x, v1[j].y), o[i][2 * j]);
          o[i][2 * j + 1] = pk_fma(make_float2(pp.z, pp.w), make_float2(v1[j].z, v1[j].w), o[i][2 * j + 1]);
        }
      }
    }
    if (Sh::kBufs == 2) {
      buf ^= 1;
    } else {
      __syncthreads();
      if (k0 + kKeys32 < end) fetch(k0 + kKeys32, 0);
    }
  }
  if (S > 1) {
    // the cluster's parts -- O, then a row's maximum and sum behind it, where Q
    // was -- are joined by the CTA that owns the row (r mod S), in a fixed order
    asm volatile("cp.async.wait_all;\n" ::: "memory");   // (a CTA without keys still has Q on its way)
    __syncthreads();
  }
  any = __any_sync(0xffffffffu, any);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = rg + 16 * i;
#pragma unroll
    for (int z = 1; z < 16; z *= 2) l[i] += __shfl_xor_sync(0xffffffffu, l[i], z);
    if (any && m[i] == -INFINITY) l[i] = NAN;
    if (S > 1) {
#pragma unroll
      for (int j = 0; j < J; ++j)
        *reinterpret_cast<float4*>(qs + r * Sh::kD + 4 * kg + 64 * j) =
            make_float4(o[i][2 * j].x, o[i][2 * j].y, o[i][2 * j + 1].x, o[i][2 * j + 1].y);
      if (kg == 0) {
        qs[r * Sh::kD + DP] = m[i];
        qs[r * Sh::kD + DP + 1] = l[i];
      }
      continue;
    }
    if (r >= rows) continue;
    float* out = (float*)A.out + b * A.os[0] + h * A.os[1] + (t0 + r) * A.os[2];
#pragma unroll
    for (int j = 0; j < 4 * J; ++j) {
      const int d = 4 * kg + 64 * (j / 4) + j % 4;
      const float num = j & 1 ? o[i][j / 2].y : o[i][j / 2].x;
      if (d < D) out[d * A.os[3]] = m[i] == -INFINITY ? l[i] : __fdiv_rn(num, l[i]);
    }
  }
  if (S > 1) {
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    const unsigned part = smem_u32(qs);
    auto at = [&](int k, int r, int col) {
      float v;
      asm volatile("ld.shared::cluster.f32 %0, [%1];\n"
                   : "=f"(v)
                   : "r"(cluster_addr(part + (unsigned)(r * Sh::kD + col) * 4, k))
                   : "memory");
      return v;
    };
    for (int i = tid; i < kRows32 / S * DP; i += kThreads32) {
      const int r = i / DP * S + (int)rank, d = i % DP;
      if (r >= rows || d >= D) continue;
      float mx = -INFINITY, num = 0.0f, den = 0.0f;
      for (int k = 0; k < S; ++k) mx = max3(mx, at(k, r, DP), -INFINITY);
      for (int k = 0; k < S; ++k) {   // (a part without weights: its sum is 0, or NaN where it had keys)
        const float pm = at(k, r, DP);
        if (pm == -INFINITY) {
          if (mx == -INFINITY) den += at(k, r, DP + 1);
          continue;
        }
        const float f = ex2((pm - mx) * cs);
        num = fmaf(at(k, r, d), f, num);
        den = fmaf(at(k, r, DP + 1), f, den);
      }
      ((float*)A.out)[b * A.os[0] + h * A.os[1] + (t0 + r) * A.os[2] + d * A.os[3]] =
          mx == -INFINITY ? den : __fdiv_rn(num, den);
    }
    __syncwarp();   // no CTA of the cluster leaves while its shared memory is read
    cluster_arrive();
    cluster_wait();
  }
}

template <int DP, int N>
int attn_f32_launch(const AttnArgs& A, int64_t ctas, int q_tiles, int S) {
  auto kern = attn_f32_kernel<DP, N>;
  static bool raised[64];
  if (const int rc = raise_smem(kern, Shape32<DP>::kSmem, raised)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(ctas * S));
  cfg.blockDim = dim3(kThreads32);
  cfg.dynamicSmemBytes = Shape32<DP>::kSmem;
  cfg.stream = cur_stream();
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)S, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, A, q_tiles, S);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(BT_ECUDA, "bt_attention: launch failed: %s", cudaGetErrorString(e));
  }
  return BT_OK;
}

// Rows of 16-byte pieces (`per` values each) that the loads above can take.
bool rows16(const void* p, const int64_t* st, int64_t B, int64_t H, int64_t T, int64_t D, int per) {
  return ((uintptr_t)p & 15) == 0 && (D == 1 || st[3] == 1) && D % per == 0 && (B == 1 || st[0] % per == 0) &&
         (H == 1 || st[1] % per == 0) && (T == 1 || st[2] % per == 0);
}

// Raises a kernel's shared-memory limit, once per device.
template <typename K>
int raise_smem(K kern, int bytes, bool (&done)[64]) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !done[dev])) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 64) done[dev] = true;
  }
  return e == cudaSuccess ? BT_OK : set_error(BT_ECUDA, "bt_attention: shared memory: %s", cudaGetErrorString(e));
}

template <int W, auto kern>
int few_launch(int smem, const AttnArgs& A, int64_t units, int S, int row_tiles) {
  if (smem > 48 * 1024) {
    static bool raised[64];
    if (const int rc = raise_smem(kern, smem, raised)) return rc;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * S));
  cfg.blockDim = dim3(32 * W);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = cur_stream();
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)S, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, A, S, row_tiles);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return set_error(BT_ECUDA, "bt_attention: launch failed: %s", cudaGetErrorString(e));
  }
  return BT_OK;
}

template <int DP, int W>
int few_run(const AttnArgs& A, bool half, int64_t units, int S, int row_tiles) {
  using F16 = FewShape<DP, kFewRows, W>;
  static_assert(F16::kSmem <= F16::kRing, "the parts lie over the ring");
  if (half) return few_launch<W, attn_few_kernel<DP, W>>(F16::kRing, A, units, S, row_tiles);
  return few_launch<W, attn_few32_kernel<DP, W>>(FewShape<DP, kFewRows32, W>::kSmem, A, units, S, row_tiles);
}

// A tensor map over [B, H, T, D] (innermost D), 64 x 128 boxes; false where
// the strides or the base do not suit one.  mul: 0 for a broadcast head or
// batch axis, whose extent in the map is 1.
bool attn_map(CUtensorMap* m, const void* p, const int64_t* st, int64_t B, int64_t H, int64_t T, int64_t D, int32_t* mul,
              int* rc) {
  *rc = BT_OK;
  if (((uintptr_t)p & 15) || (D > 1 && st[3] != 1) || T < 1) return false;
  const int64_t ext[3] = {T, H, B}, str[3] = {st[2], st[1], st[0]};
  uint64_t dims[4] = {(uint64_t)D, 1, 1, 1}, bytes[3];
  for (int i = 0; i < 3; ++i) {
    bytes[i] = (uint64_t)(D * 2 + 15) / 16 * 16;
    if (i) mul[i - 1] = 0;
    if (ext[i] == 1) continue;
    if (str[i] == 0 && i) continue;
    if (str[i] <= 0 || str[i] % 8 || str[i] >= (int64_t)1 << 38) return false;
    dims[i + 1] = (uint64_t)ext[i];
    bytes[i] = (uint64_t)str[i] * 2;
    if (i) mul[i - 1] = 1;
  }
  const uint32_t box[4] = {64, kTile, 1, 1};
  *rc = tma_map(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, p, dims, bytes, box);
  return *rc == BT_OK;
}

template <int DP>
int attn_tc_launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const CUtensorMap& mo, AttnTc& A,
                   int sms) {
  auto kern = attn_tc_kernel<DP>;
  constexpr int smem = AttnShape<DP>::kSmem;
  static bool raised[64];
  if (const int rc = raise_smem(kern, smem, raised)) return rc;
  const int grid = (int)(A.items < (uint32_t)sms ? A.items : (uint32_t)sms);
  A.step_t = grid % A.q_tiles;
  A.step_h = grid / A.q_tiles % (int)A.a.H;
  A.step_b = grid / A.q_tiles / (int)A.a.H;
  kern<<<grid, kAttnThreads, smem, cur_stream()>>>(mq, mk, mv, mo, A);
  return check_launch("bt_attention");
}

}  // namespace

cudaError_t attn_timeouts(unsigned int* sum) { return take_timeouts(sum); }

}  // namespace bt

using namespace bt;

extern "C" int bt_attention(const bt_tensor* q, const bt_tensor* k, const bt_tensor* v, const bt_tensor* lengths,
                            const bt_tensor* key_mask, float scale, const bt_tensor* out) {
  const char* what = "bt_attention";
  int rc;
  if ((rc = check_tensor(q, "q", false)) || (rc = check_tensor(k, "k", false)) || (rc = check_tensor(v, "v", false)) ||
      (rc = check_tensor(out, "out", false)))
    return rc;
  if (q->dtype != BT_F32 && q->dtype != BT_F16) return set_error(BT_EDTYPE, "%s: q must be float32 or float16", what);
  if (k->dtype != q->dtype || v->dtype != q->dtype || out->dtype != q->dtype)
    return set_error(BT_EDTYPE, "%s: q, k, v and out must have one dtype", what);
  if (q->rank != 4 || k->rank != 4 || v->rank != 4 || out->rank != 4)
    return set_error(BT_ESHAPE, "%s: q, k, v and out must be [batch, heads, length, dim]", what);
  AttnArgs A{};
  A.B = q->shape[0];
  A.H = q->shape[1];
  A.Tq = q->shape[2];
  const int64_t Hk = k->shape[1], D = q->shape[3];
  A.Tk = k->shape[2];
  for (int d = 0; d < 4; ++d) {
    if (k->shape[d] != v->shape[d]) return set_error(BT_ESHAPE, "%s: k and v must have the same shape", what);
    if (out->shape[d] != q->shape[d]) return set_error(BT_ESHAPE, "%s: out must have q's shape", what);
    A.qs[d] = q->strides[d];
    A.ks[d] = k->strides[d];
    A.vs[d] = v->strides[d];
    A.os[d] = out->strides[d];
  }
  if (k->shape[0] != A.B || k->shape[3] != D)
    return set_error(BT_ESHAPE, "%s: q and k must have the same batch and dim", what);
  if (Hk < 1 ? A.H != 0 : A.H % Hk != 0)
    return set_error(BT_ESHAPE, "%s: %lld query heads cannot share %lld key heads", what, (long long)A.H, (long long)Hk);
  if (D < 1 || D > kMaxHeadDim) return set_error(BT_ETOOBIG, "%s: dim %lld outside 1..%d", what, (long long)D, kMaxHeadDim);
  if (!(scale > 0.0f) || isinf(scale * 1.4426950408889634f))   // (the kernels' scale log2(e))
    return set_error(BT_EINVAL, "%s: scale must be positive and scale log2(e) finite", what);
  if (A.Tk > INT32_MAX / 2 || A.Tq > INT32_MAX / 2) return set_error(BT_ETOOBIG, "%s: more than 2^30 positions", what);
  if (lengths) {
    if ((rc = check_tensor(lengths, "lengths", false))) return rc;
    if (lengths->dtype != BT_I32 && lengths->dtype != BT_I64)
      return set_error(BT_EDTYPE, "%s: lengths must be int32 or int64", what);
    if (lengths->rank != 1 || lengths->shape[0] != A.B) return set_error(BT_ESHAPE, "%s: lengths must be [batch]", what);
    A.lengths = lengths->data;
    A.len64 = lengths->dtype == BT_I64;
    A.len_stride = lengths->strides[0];
  }
  if (key_mask) {
    if ((rc = check_tensor(key_mask, "key_mask", false))) return rc;
    if (key_mask->dtype != BT_BOOL) return set_error(BT_EDTYPE, "%s: key_mask must be bool", what);
    if (key_mask->rank != 2 || key_mask->shape[0] != A.B || key_mask->shape[1] != A.Tk)
      return set_error(BT_ESHAPE, "%s: key_mask must be [batch, keys]", what);
    A.mask = (const uint8_t*)key_mask->data;
    A.mask_sb = key_mask->strides[0];
    A.mask_sk = key_mask->strides[1];
  }
  A.D = (int32_t)D;
  A.scale = scale;
  const int64_t rows = A.B * A.H * A.Tq;
  if (rows == 0) return BT_OK;
  A.G = A.H / Hk;
  A.q = q->data;
  A.k = k->data;
  A.v = v->data;
  A.out = out->data;
  DevInfo di;
  if ((rc = dev_info(&di))) return rc;
  const bool half = q->dtype == BT_F16;
  const int per = half ? 8 : 4, few_rows = half ? kFewRows : kFewRows32;
  const int64_t group = A.G * A.Tq, row_tiles = (group + few_rows - 1) / few_rows, units = A.B * Hk * row_tiles;
  const bool pieces = rows16(A.q, A.qs, A.B, A.H, A.Tq, D, per) && rows16(A.k, A.ks, A.B, Hk, A.Tk, D, per) &&
                      rows16(A.v, A.vs, A.B, Hk, A.Tk, D, per);
  // The form with the least estimated time (us; measured with 1 to 64 batch
  // entries, 1 to 16 heads, 1 to 4000 queries over 6 to 4096 keys): rows
  // straight from global memory pay for every tile of rows (a CTA's start and
  // join) and step of 16 keys; the tiled forms for every round of CTAs and its
  // tiles of keys.
  //   float16, 1 x 1 head,   256 queries, 4096 keys of 64: 21 against 54 us
  //            4 x 8 heads,  256 queries, 1000 keys of 64: 46 against 20 us
  //   float32, 2 x 4 heads,  256 queries, 1000 keys of 64: 61 against 135 us
  //            4 x 32 heads, 4249 queries, 6 keys of 32: 1540 against 180 us
  const int q_rows = half ? 2 * kTile : kRows32, k_rows = half ? kTile : kKeys32;
  const double waves = ceil((double)(A.B * A.H * ((A.Tq + q_rows - 1) / q_rows)) / di.sm_count);
  const double steps = (double)(A.Tk / 16 + 1), tiles = (double)((A.Tk + k_rows - 1) / k_rows);
  const double few_us = 17 + (double)units * (10e-3 + steps * (half ? (D <= 64 ? 0.7e-3 : 2.5e-3) : (D <= 64 ? 1.0e-3 : 3.5e-3)));
  // (float32 tiles: the keys split over a cluster while that still fits one round)
  const int64_t ctas32 = A.B * A.H * ((A.Tq + kRows32 - 1) / kRows32);
  int split32 = 1;
  while (split32 < 8 && ctas32 * split32 * 2 <= di.sm_count && tiles >= 4 * split32) split32 *= 2;
  const double tile_us =
      9 + waves * (half ? 2.5 + tiles * (D <= 64 ? 1.5 : 1.9) : 3 + 2 * (split32 > 1) + tiles / split32 * (D <= 64 ? 8.8 : 16.5));
  if (A.Tk > 0 && pieces && (row_tiles == 1 || few_us < tile_us)) {
    // the keys split over a cluster, then over more warps, until the GPU is
    // full or a warp is down to four steps of 16 keys (32 x 16 heads, one
    // query over 2000 keys, before the ring: 54 us in 512 CTAs, 61 in 1024, 74
    // in 2048).  Eight warps where a cluster of eight still leaves SMs idle, us
    // with eight / four: one row tile of 4 key heads over 16384 keys, float16 dims
    // of 128 30.4 / 35.9, of 64 20.0 / 23.0; float32 dims of 128 67 / 108
    int S = 1;
    while (S < 8 && units * S < 3 * (int64_t)di.sm_count && A.Tk >= (int64_t)2 * S * 4 * 64) S *= 2;
    if (units * S < INT32_MAX)
      return D <= 64 ? (S == 8 && units * S < di.sm_count ? few_run<64, 8>(A, half, units, S, (int)row_tiles)
                                                          : few_run<64, 4>(A, half, units, S, (int)row_tiles))
                     : (S == 8 && units * S < di.sm_count ? few_run<128, 8>(A, half, units, S, (int)row_tiles)
                                                          : few_run<128, 4>(A, half, units, S, (int)row_tiles));
  }
  if (!half && A.Tk > 0) {
    const int64_t q_tiles = (A.Tq + kRows32 - 1) / kRows32, ctas = ctas32;
    if (ctas < INT32_MAX && pieces)
      return D <= 64 ? attn_f32_launch<64, 4>(A, ctas, (int)q_tiles, split32) : attn_f32_launch<128, 4>(A, ctas, (int)q_tiles, split32);
    if (ctas < INT32_MAX)
      return D <= 64 ? attn_f32_launch<64, 1>(A, ctas, (int)q_tiles, split32) : attn_f32_launch<128, 1>(A, ctas, (int)q_tiles, split32);
  }
  if (half && A.Tk > 0) {
    AttnTc P{};
    CUtensorMap mq, mk, mv;
    const int64_t q_tiles = (A.Tq + 2 * kTile - 1) / (2 * kTile), items = A.B * A.H * q_tiles;
    if (items < INT32_MAX && attn_map(&mq, A.q, A.qs, A.B, A.H, A.Tq, D, P.q_mul, &rc) &&
        attn_map(&mk, A.k, A.ks, A.B, Hk, A.Tk, D, P.k_mul, &rc) && attn_map(&mv, A.v, A.vs, A.B, Hk, A.Tk, D, P.v_mul, &rc)) {
      P.a = A;
      P.q_tiles = (int32_t)q_tiles;
      P.items = (uint32_t)items;
      CUtensorMap mo = {};
      int32_t o_mul[2];
      // (a TMA store needs every axis of its own: no two rows of out overlap)
      P.wide = !rows16(A.out, A.os, A.B, A.H, A.Tq, D, 8) ? 0
               : attn_map(&mo, A.out, A.os, A.B, A.H, A.Tq, D, o_mul, &rc) && (A.B == 1 || o_mul[1]) && (A.H == 1 || o_mul[0])
                   ? 2
                   : 1;
      if (rc) return rc;
      return D <= 64 ? attn_tc_launch<64>(mq, mk, mv, mo, P, di.sm_count) : attn_tc_launch<128>(mq, mk, mv, mo, P, di.sm_count);
    }
    if (rc) return rc;
  }
  const int64_t want = (rows + kRowWarps - 1) / kRowWarps, cap = (int64_t)di.sm_count * 16;
  const int grid = (int)(want < cap ? want : cap);
  if (q->dtype == BT_F32) attn_rows_kernel<float><<<grid, 32 * kRowWarps, 0, cur_stream()>>>(A, rows);
  else attn_rows_kernel<__half><<<grid, 32 * kRowWarps, 0, cur_stream()>>>(A, rows);
  return check_launch(what);
}

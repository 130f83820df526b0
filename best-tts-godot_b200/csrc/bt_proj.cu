// bt_proj.cu -- quantised projections: symmetric 8-bit row quantisation
// (bt_quantize_rows) and the int8 x int8 product with a scale for each token
// and each output channel (bt_matmul_int8).
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include "bt_ops.h"
#include "bt_internal.h"

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

template <typename TO>
__global__ void __launch_bounds__(256) matmul_int8_kernel(MmArgs A) {
  __shared__ int8_t as[16][33], ws[16][33];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int64_t n_tiles = (A.N + 15) / 16;
  const int64_t m0 = (int64_t)blockIdx.x / n_tiles * 16, n0 = (int64_t)blockIdx.x % n_tiles * 16;
  int acc = 0;
  for (int64_t k0 = 0; k0 < A.K; k0 += 32) {
    for (int i = threadIdx.x; i < 512; i += 256) {
      const int r = i >> 5, c = i & 31;
      as[r][c] = m0 + r < A.M && k0 + c < A.K ? A.a[(m0 + r) * A.lda + k0 + c] : (int8_t)0;
      ws[r][c] = n0 + r < A.N && k0 + c < A.K ? A.w[(n0 + r) * A.ldw + k0 + c] : (int8_t)0;
    }
    __syncthreads();
    for (int c = 0; c < 32; ++c) acc += (int)as[ty][c] * (int)ws[tx][c];
    __syncthreads();
  }
  const int64_t m = m0 + ty, n = n0 + tx;
  if (m >= A.M || n >= A.N) return;
  float y = __fmul_rn(__int2float_rn(acc), __fmul_rn(A.a_scale[m * A.sa], A.w_scale[n * A.sw]));
  if (A.bias) y = __fadd_rn(y, A.bias[n * A.sb]);
  if constexpr (sizeof(TO) == 2) ((__half*)A.out)[m * A.ldo + n] = __float2half_rn(y);
  else ((float*)A.out)[m * A.ldo + n] = y;
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
  const int64_t cap = (int64_t)di.sm_count * 16;
  const int grid = (int)(rows < cap ? rows : cap);
  if (x->dtype == BT_F32)
    quantize_rows_kernel<float><<<grid, kQuantThreads, 0, cur_stream()>>>((const float*)x->data, ldx, rows, K,
                                                                          (int8_t*)q->data, ldq, (float*)sp, lds);
  else
    quantize_rows_kernel<__half><<<grid, kQuantThreads, 0, cur_stream()>>>((const __half*)x->data, ldx, rows, K,
                                                                           (int8_t*)q->data, ldq, (float*)sp, lds);
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
  const int64_t tiles = (A.M + 15) / 16 * ((A.N + 15) / 16);
  if (tiles > INT32_MAX) return set_error(BT_ETOOBIG, "%s: too many output values", what);
  if (out->dtype == BT_F32) matmul_int8_kernel<float><<<(int)tiles, 256, 0, cur_stream()>>>(A);
  else matmul_int8_kernel<__half><<<(int)tiles, 256, 0, cur_stream()>>>(A);
  return check_launch(what);
}

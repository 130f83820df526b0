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
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include "bt_ops.h"
#include "bt_internal.h"

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
    for (int64_t j0 = 0; j0 < n; j0 += 32) {
      const int64_t j = j0 + lane;
      const bool in = j < n && (!A.mask || A.mask[b * A.mask_sb + j * A.mask_sk]);
      unsigned live = __ballot_sync(0xffffffffu, in);
      if (!live) continue;
      float s = -INFINITY;
      if (in) {
        float dot = 0.0f;
        for (int d = 0; d < A.D; ++d) dot = __fmaf_rn(qsh[w][d], ldf(kp + j * A.ks[2] + d * A.ks[3]), dot);
        s = dot * A.scale;
      }
      float mx = s;
      for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float mn = fmaxf(m, mx), base = mn == -INFINITY ? 0.0f : mn;
      const float keep = expf(m - base), p = in ? expf(s - base) : 0.0f;
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
        const float y = l == 0.0f ? 0.0f : __fdiv_rn(o[i], l);
        if constexpr (sizeof(T) == 2) op[(lane + 32 * i) * A.os[3]] = __float2half_rn(y);
        else op[(lane + 32 * i) * A.os[3]] = y;
      }
  }
}

}  // namespace
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
  if (!(scale > 0.0f) || isinf(scale)) return set_error(BT_EINVAL, "%s: scale must be positive and finite", what);
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
  const int64_t want = (rows + kRowWarps - 1) / kRowWarps, cap = (int64_t)di.sm_count * 16;
  const int grid = (int)(want < cap ? want : cap);
  if (q->dtype == BT_F32) attn_rows_kernel<float><<<grid, 32 * kRowWarps, 0, cur_stream()>>>(A, rows);
  else attn_rows_kernel<__half><<<grid, 32 * kRowWarps, 0, cur_stream()>>>(A, rows);
  return check_launch(what);
}

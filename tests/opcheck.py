"""64-bit forms of the projection and attention operators, with error bounds
counted from their roundings (used by the GPU tests)."""
import numpy as np
import torch

EPS32 = 2.0 ** -24    # half a step, relative
EPS16 = 2.0 ** -11


def quantize_rows_np(x):
    """The definition in numpy float32 steps: exact for the kernels."""
    x = np.asarray(x).astype(np.float32)
    with np.errstate(all="ignore"):
        a = np.maximum(np.abs(x).max(-1, keepdims=True), np.float32(2.0 ** -100))   # np.max carries a NaN
        v = x * (np.float32(127) / a)
        q = np.where(np.isnan(v), np.float32(0), np.rint(v)).astype(np.int8)
        return q, (a / np.float32(127))[..., 0]


def matmul_int8_64(a, a_scale, w, w_scale, bias, out_dtype):
    """(value, bound): float64 result and the most a kernel may be off."""
    acc = a.double() @ w.double().t()
    y0 = acc * a_scale.double()[..., None] * w_scale.double()
    y = y0 if bias is None else y0 + bias.double()
    # int -> float, the scales' product, the scaling: 3 roundings; the bias add: one
    tol = 3.01 * EPS32 * y0.abs() + 1.01 * EPS32 * y.abs() + 2.0 ** -148
    if out_dtype == torch.float16:
        tol = tol + EPS16 * (y.abs() + tol) + 2.0 ** -25
    return y, tol


def attention_64(q, k, v, lengths=None, key_mask=None, scale=None):
    """(value, bound).  Per row with scores s_j, p_j = e^(s_j - m):
    a score is a D-term float32 dot product and a scaling, off by at most
    (D + 3) eps scale |q||k|; p_j then by that (and the row maximum's, which
    cancels), by exp's own 2 ulp and the rounded argument (|s - m| <= 104
    where p_j counts, one rounding each of the scaled argument and log2(e):
    2 * 104 eps); sums of n terms by n eps.  float16 adds p_j rounded to 11
    bits (or to multiples of 2^-25 below 2^-14; the largest p_j of a row is
    at least 2^-8 of the running reference), and the result's rounding."""
    B, H, Tq, D = q.shape
    Hk, Tk = k.shape[1], k.shape[2]
    G = H // Hk
    half = q.dtype == torch.float16
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros((B, H, Tq, D), dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for b in range(B):
        n = Tk if lengths is None else min(max(int(lengths[b]), 0), Tk)
        keep = torch.arange(n, device=q.device)
        if key_mask is not None:
            keep = keep[key_mask[b, :n]]
        if keep.numel() == 0:
            continue
        for h in range(H):
            qq, kk, vv = q[b, h].double(), k[b, h // G].double()[keep], v[b, h // G].double()[keep]
            s = qq @ kk.t() * scale
            p = torch.softmax(s, -1)
            o = p @ vv
            mag = p @ vv.abs()
            ds = (D + 3) * EPS32 * scale * (qq.abs() @ kk.abs().t()).amax(-1, keepdim=True)
            rel = 2 * ds + (208 + 8 + 2 * keep.numel()) * EPS32
            t = rel * mag + 2.0 ** -140
            if half:
                t = t + EPS16 * mag + keep.numel() * 2.0 ** -25 * vv.abs().amax(0)
                t = t + EPS16 * (o.abs() + t) + 2.0 ** -25
            out[b, h], tol[b, h] = o, t
    return out, tol


def assert_within(got, want, tol, what=""):
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)} != {tuple(want.shape)}"
    bad = ~((got.double() - want).abs() <= tol)
    if bad.any():
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside the bound, first at {i}: "
                             f"{got[i].item()} for {want[i].item()} +- {tol[i].item()}")

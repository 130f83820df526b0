"""Attention (bt_attention) at the ends of its range: scores of any size.

The scores here are sums that float32 holds without a rounding (small whole
numbers times powers of two), so a bound need not allow for theirs."""
import pytest
import torch

from opcheck import EPS16, EPS32, assert_within

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32

# (batch, heads, key heads, queries, keys, dim): few queries; tiles of queries, in
# float32 with the keys split and not; float16 rows that are read as they lie
FORMS = [(2, 4, 2, 1, 700, 64), (2, 4, 2, 1, 700, 128), (2, 4, 2, 3, 100, 64), (2, 4, 2, 3, 100, 128), (2, 4, 2, 1, 700, 36),
         (4, 8, 4, 256, 700, 64), (4, 8, 4, 256, 700, 128), (4, 8, 4, 256, 700, 36), (8, 8, 4, 256, 300, 64), (8, 8,
         4, 256, 300, 128), (8, 8, 4, 256, 300, 36), (2, 4, 2, 3, 100, 36)]


def attention_of_exact_scores(q, k, v, scale=None):
    """(value, bound) in 64 bits.  A weight's argument carries three roundings
    (log2(e) scale, the difference to the reference, their product) of at most
    104 where the weight counts, exp 2 ulp, sums of n terms n; a form that
    multiplies the reference first does so below 2^11 only, which rounds the
    weights of one reference alike, those of another one otherwise.  float16
    rounds the weights (or takes multiples of 2^-25 of the reference's) and
    the result."""
    G, D, n = q.shape[1] // k.shape[1], q.shape[-1], k.shape[2]
    scale = float(torch.tensor(D ** -0.5 if scale is None else scale, dtype=torch.float32))
    kk, vv = (t.double().repeat_interleave(G, 1) for t in (k, v))
    s = q.double() @ kk.transpose(-1, -2)
    assert torch.equal(s.float().double(), s), "scores that float32 does not hold"
    far = min(float(s.abs().max()) * scale * 1.4427, 2.0 ** 11)
    p = torch.softmax((s - s.amax(-1, keepdim=True)) * scale, -1)
    o, mag = p @ vv, p @ vv.abs()
    tol = (312 + 8 + 2 * n + 2 * far) * EPS32 * mag + 2.0 ** -140
    if q.dtype == F16:
        tol = tol + EPS16 * mag + n * 2.0 ** -25 * vv.abs().amax(-2, keepdim=True)
        tol = tol + EPS16 * (o.abs() + tol) + 2.0 ** -25
    return o, tol


def _check(rt, q, k, v, what, **kw):
    o = rt.attention(q, k, v, **kw)
    assert_within(o, *attention_of_exact_scores(q, k, v, **kw), what)


def _whole(g, most, shape, dtype):
    return torch.randint(-most, most + 1, shape, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("B,H,Hk,Tq,Tk,D", FORMS)
def test_large_scales(gpu_runtime, B, H, Hk, Tq, Tk, D, dtype):
    """Up to a softmax that is one key, or the keys that tie for the largest score."""
    g = torch.Generator("cuda").manual_seed(Tq + Tk + D)
    q, k = _whole(g, 2, (B, H, Tq, D), dtype), _whole(g, 2, (B, Hk, Tk, D), dtype)
    v = torch.randn(B, Hk, Tk, D, generator=g, device="cuda").to(dtype)
    for scale in (0.5, 10.0, 1e3, 1e5, 1e8, 1e9, 1e20, 2.35e38):
        _check(gpu_runtime, q, k, v, f"scale {scale}", scale=scale)


@pytest.mark.parametrize("B,H,Hk,Tq,Tk,D", FORMS)
def test_large_half_operands(gpu_runtime, B, H, Hk, Tq, Tk, D):
    g = torch.Generator("cuda").manual_seed(Tq + Tk + D)
    v = torch.randn(B, Hk, Tk, D, generator=g, device="cuda").half()
    for step in (512, 2048, 8192, 32768):
        q, k = step * _whole(g, 1, (B, H, Tq, D), F16), step * _whole(g, 1, (B, Hk, Tk, D), F16)
        _check(gpu_runtime, q, k, v, f"multiples of {step}")
        _check(gpu_runtime, q.abs(), -k.abs(), v, f"multiples of {step}, no score above 0")


@pytest.mark.parametrize("B,H,Hk,Tq,Tk,D", FORMS)
def test_equal_keys(gpu_runtime, B, H, Hk, Tq, Tk, D):
    """All keys alike, whatever their score: the mean of the values."""
    g = torch.Generator("cuda").manual_seed(Tk + D)
    v = torch.randn(B, Hk, Tk, D, generator=g, device="cuda").half()
    flat = torch.zeros(B, H, Tq, D, device="cuda").half(), torch.zeros(B, Hk, Tk, D, device="cuda").half()
    want, tol = attention_of_exact_scores(*flat, v)
    for a in (300.0, 2500.0, 5000.0, 8000.0, 20000.0, 30000.0, 60000.0):
        for sign in (1, -1):
            o = gpu_runtime.attention(torch.full_like(flat[0], a), torch.full_like(flat[1], sign * a), v)
            assert_within(o, want, tol, f"{sign} x {a}")


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("B,H,Hk,Tq,Tk,D", FORMS)
def test_large_scores_that_grow_along_the_keys(gpu_runtime, B, H, Hk, Tq, Tk, D, dtype):
    """Near 2e8, and 4 or 8 more after scaling every 128 keys, or 4 every 37 (for
    dims of 64; growth that a form may leave its reference behind by)."""
    g = torch.Generator("cuda").manual_seed(Tk + D)
    v = torch.randn(B, Hk, Tk, D, generator=g, device="cuda").to(dtype)
    for sign in (1, -1):
        for every, step in ((128, 1), (128, 2), (37, 1)):
            q = torch.full((B, H, Tq, D), 2048.0, device="cuda").to(dtype)
            k = torch.zeros(B, Hk, Tk, D, device="cuda").to(dtype)
            k[..., :48] = sign * 2048.0
            q[..., D - 1] = 32.0
            k[..., D - 1] = (step * (torch.arange(Tk, device="cuda") // every)).to(dtype)
            _check(gpu_runtime, q, k, v, f"{sign} {every} {step}")


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("B,H,Hk,Tq,Tk,D", FORMS + [(4, 2, 2, Tq, 2500, D) for Tq in (1, 900) for D in (64, 128, 36)])
def test_scores_of_minus_infinity(gpu_runtime, B, H, Hk, Tq, Tk, D, dtype):
    """A key that scores -inf has no weight, wherever it lies; where every key
    that takes part does, the softmax is 0 / 0 and the row NaN; a row no key
    takes part in stays 0."""
    rt, g = gpu_runtime, torch.Generator("cuda").manual_seed(Tk + D)
    q, k, v = (torch.randn(B, h, t, D, generator=g, device="cuda").to(dtype) for h, t in ((H, Tq), (Hk, Tk), (Hk, Tk)))
    q[..., 0] = 1.0
    some = torch.rand(B, Tk, generator=g, device="cuda") < 0.5
    some[:, :Tk // 2] = True     # whole parts of the keys, the first ones too
    some[:, -1] = False
    low = k.clone()
    low[..., 0] = torch.where(some[:, None, :].expand(B, Hk, Tk), float("-inf"), k[..., 0].float()).to(dtype)
    assert torch.equal(rt.attention(q, low, v), rt.attention(q, k, v, key_mask=~some))
    assert rt.attention(q, low, v, key_mask=some).isnan().all()
    n = torch.full((B,), Tk, dtype=torch.int32, device="cuda")
    n[0], n[1] = Tk // 2, 0
    o = rt.attention(q, low, v, lengths=n)
    assert o[0].isnan().all() and (o[1] == 0).all() and torch.isfinite(o[2:]).all()
    assert (rt.attention(q, low, v, key_mask=torch.zeros_like(some)) == 0).all()
    # one row of queries
    row = q.clone()
    row[0, H - 1, Tq - 1, 0] = float("inf")
    o = rt.attention(row, torch.cat([-k[..., :1].abs() - 1, k[..., 1:]], -1), v)
    same = rt.attention(q, torch.cat([-k[..., :1].abs() - 1, k[..., 1:]], -1), v)
    assert o[0, H - 1, Tq - 1].isnan().all()
    o[0, H - 1, Tq - 1] = same[0, H - 1, Tq - 1]
    assert torch.equal(o, same)


@pytest.mark.parametrize("B,H,Hk,Tq,Tk,D", FORMS)
def test_largest_half_values(gpu_runtime, B, H, Hk, Tq, Tk, D):
    """A mean of values at the type's largest stays there, also where fifteen
    weights of sixteen are rounded up by nearly half a step: 2^7 e^-0.6926 =
    64.035, which float16 holds as 64.0625."""
    q = torch.zeros(B, H, Tq, D, device="cuda").half()
    k = torch.zeros(B, Hk, Tk, D, device="cuda").half()
    q[..., 0], k[..., 0] = 1.0, -1.0
    k[:, :, ::16, 0] = 0.0
    v = torch.full_like(k, torch.finfo(F16).max)
    v[..., 1] *= -1
    v[..., 2] = 1.0
    _check(gpu_runtime, q, k, v, "largest values", scale=0.6926)
    v[:, :, Tk // 2, 3] = float("inf")
    o = gpu_runtime.attention(q, k, v, scale=0.6926)
    assert (o[..., 3] == float("inf")).all() and torch.isfinite(o[..., :3]).all()
    v[:, :, Tk // 2, 3] = float("-inf")
    o = gpu_runtime.attention(q, k, v, scale=0.6926)
    assert (o[..., 3] == float("-inf")).all() and torch.isfinite(o[..., :3]).all()


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("B,H,Hk,Tq,Tk,D", FORMS)
def test_large_scores_under_masks(gpu_runtime, B, H, Hk, Tq, Tk, D, dtype):
    """Rows near 2e8 beside rows of small scores, over the keys that take part."""
    rt, g = gpu_runtime, torch.Generator("cuda").manual_seed(Tq + Tk + D)
    q, k = _whole(g, 2, (B, H, Tq, D), dtype), _whole(g, 2, (B, Hk, Tk, D), dtype)
    q[:, ::2] *= 8192
    q[:, :, ::3] *= 0.125
    k *= 16
    v = torch.randn(B, Hk, Tk, D, generator=g, device="cuda").to(dtype)
    keep = torch.rand(Tk, generator=g, device="cuda") < 0.6
    keep[:min(Tk // 3, 140)] = False
    n = Tk - 13
    live = keep.nonzero()[:, 0]
    live = live[live < n]
    want = attention_of_exact_scores(q, k[:, :, live], v[:, :, live])
    out = torch.ones(Tk, dtype=torch.bool, device="cuda")
    out[live] = False
    k, v = (t.masked_fill(out[:, None], float("nan")) for t in (k, v))
    o = rt.attention(q, k, v, lengths=torch.full((B,), n, dtype=torch.int32, device="cuda"), key_mask=keep.expand(B, Tk))
    assert_within(o, *want)

"""Attention over keys of another length (bt_attention) against 64 bits, and
one attention block of the operators together."""
import threading

import pytest
import torch

from opcheck import EPS16, EPS32, assert_within, attention_64, matmul_int8_64

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


def _states(g, B, H, T, D, dtype, layout="head", gain=1.0):
    if layout == "token":
        return (gain * torch.randn(B, T, H, D, generator=g, device="cuda")).to(dtype).permute(0, 2, 1, 3)
    return (gain * torch.randn(B, H, T, D, generator=g, device="cuda")).to(dtype)


def _run(rt, q, k, v, what="", **kw):
    o = rt.attention(q, k, v, **kw)
    torch.cuda.synchronize()
    assert o.dtype == q.dtype
    want, tol = attention_64(q, k, v, **kw)
    assert_within(o, want, tol, what)
    return o


SIZES = [(1, 1, 1, 1, 1, 64), (1, 2, 1, 1, 33, 64), (2, 3, 3, 5, 7, 32), (1, 12, 12, 510, 510, 64), (2, 4, 2, 128, 128, 64),
         (1, 2, 2, 129, 127, 128), (2, 2, 1, 255, 129, 96), (1, 3, 3, 256, 256, 128), (1, 1, 1, 257, 1, 64),
         (3, 2, 2, 300, 65, 80), (1, 4, 4, 64, 1000, 40), (2, 8, 2, 1, 700, 128), (4, 6, 6, 1, 2000, 64), (1, 16, 2, 3, 300, 64),
         (1, 8, 1, 1, 5000, 128), (2, 2, 2, 17, 2049, 8), (1, 1, 1, 1000, 3000, 128), (1, 2, 2, 700, 1, 16),
         (1, 2, 2, 4, 9, 20), (1, 2, 1, 30, 50, 7), (1, 1, 1, 3, 3, 1), (2, 2, 2, 140, 200, 36), (5, 1, 1, 2, 31, 72),
         (1, 32, 4, 2, 640, 64), (1, 4, 1, 40, 200, 64), (2, 12, 1, 2, 150, 128), (1, 5, 1, 9, 1500, 56)]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("B,H,Hk,Tq,Tk,D", SIZES)
def test_sizes(gpu_runtime, B, H, Hk, Tq, Tk, D, dtype):
    g = torch.Generator("cuda").manual_seed(B + H + Tq + Tk + D)
    for layout in ("head", "token"):
        q, k, v = (_states(g, B, h, t, D, dtype, layout) for h, t in ((H, Tq), (Hk, Tk), (Hk, Tk)))
        o = _run(gpu_runtime, q, k, v, f"{layout}")
        assert layout == "head" or o.permute(0, 2, 1, 3).is_contiguous()


# (batch, heads, queries, keys, dim): enough heads and queries that the tiled
# forms run, with more items than the GPU has SMs, a second query tile of a few
# rows or none, and key tiles that wrap the ring of tiles
MANY = [(40, 8, 130, 260, 64), (40, 8, 130, 260, 128), (25, 12, 100, 600, 64), (25, 12, 100, 600, 40), (20, 10, 300, 1500, 96),
        (10, 16, 513, 1000, 64), (9, 20, 257, 129, 128), (3, 64, 128, 2100, 64)]


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("B,H,Tq,Tk,D", MANY)
def test_many_items(gpu_runtime, B, H, Tq, Tk, D, dtype):
    g = torch.Generator("cuda").manual_seed(B + Tk)
    q, k, v = (_states(g, B, h, t, D, dtype, "token") for h, t in ((H, Tq), (H // 2, Tk), (H // 2, Tk)))
    lengths = torch.randint(0, Tk + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    lengths[1], lengths[2], lengths[B - 1] = 0, Tk, 0
    mask = torch.rand(B, Tk, generator=g, device="cuda") < 0.8
    mask[0, :128] = False
    _run(gpu_runtime, q, k, v, "all")
    _run(gpu_runtime, q, k, v, "lengths", lengths=lengths)
    _run(gpu_runtime, q, k, v, "mask", key_mask=mask)
    o = _run(gpu_runtime, q, k, v, "both", key_mask=mask, lengths=lengths)
    out = ~(mask & (torch.arange(Tk, device="cuda") < lengths[:, None]))
    k2, v2 = (t.masked_fill(out[:, None, :, None], float("nan")) for t in (k, v))
    assert torch.equal(gpu_runtime.attention(q, k2, v2, key_mask=mask, lengths=lengths), o)
    for _ in range(3):
        assert torch.equal(gpu_runtime.attention(q, k, v, key_mask=mask, lengths=lengths), o)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D", [64, 128, 36])
def test_few_tiles_over_long_keys(gpu_runtime, D, dtype):
    """Fewer tiles of queries than SMs, so that the keys are split: lengths that
    leave whole parts without keys, and NaN in one part."""
    rt, g = gpu_runtime, torch.Generator("cuda").manual_seed(D)
    B, H, Tq, Tk = 4, 2, 900, 2500
    q, k, v = (_states(g, B, H, t, D, dtype, "token") for t in (Tq, Tk, Tk))
    lengths = torch.tensor([0, 1, 70, Tk], dtype=torch.int32, device="cuda")
    _run(rt, q, k, v, "all")
    o = _run(rt, q, k, v, "lengths", lengths=lengths)
    assert (o[0] == 0).all()
    mask = torch.zeros(B, Tk, dtype=torch.bool, device="cuda")
    mask[1, 2400:] = True
    mask[2, 1200] = True
    mask[3, ::3] = True
    o = _run(rt, q, k, v, "mask", key_mask=mask)
    k2 = k.clone()
    k2[3, 1, 2490, 0] = float("nan")
    full = rt.attention(q, k, v)
    bad = rt.attention(q, k2, v)
    assert bad[3, 1].isnan().all()
    bad[3, 1] = full[3, 1]
    assert torch.equal(bad, full)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("D", [64, 128])
def test_many_items_growing_and_non_finite(gpu_runtime, D, dtype):
    """Rows whose reference moves in every key tile, beside rows where it never
    does; NaN and infinite scores in some rows of the tiled forms."""
    rt, g = gpu_runtime, torch.Generator("cuda").manual_seed(D)
    B, H, Tq, Tk = 6, 30, 300, 900
    q, k, v = (_states(g, B, H, t, D, dtype) for t in (Tq, Tk, Tk))
    ramp = torch.linspace(0, 60, Tk, device="cuda")
    k[..., 0] = ramp.to(dtype)
    q[..., 0] = torch.where(torch.rand(B, H, Tq, generator=g, device="cuda") < 0.3, 30.0, 0.1).to(dtype)
    o = _run(rt, q, k, v, "ramp")
    q2, k2 = q.clone(), k.clone()
    q2[0, 0, 5, 3] = float("nan")
    q2[1, 2, 299, 0] = float("inf")
    k2[2, 3, 700, 1] = float("nan")      # every row of head (2, 3)
    o2 = rt.attention(q2, k2, v)
    assert o2[0, 0, 5].isnan().all() and o2[1, 2, 299].isnan().all() and o2[2, 3].isnan().all()
    o2[0, 0, 5], o2[1, 2, 299], o2[2, 3] = o[0, 0, 5], o[1, 2, 299], o[2, 3]
    assert torch.equal(o2, o)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("Tq", [1, 6, 130, 400])
def test_lengths_and_masks(gpu_runtime, Tq, dtype):
    """Lengths 0, 1, inside and at tile ends, beyond Tk and negative; masks
    that leave some rows empty, whole tiles, single keys; both together."""
    rt, g = gpu_runtime, torch.Generator("cuda").manual_seed(Tq)
    B, H, Hk, Tk, D = 9, 4, 2, 300, 64
    q, k, v = (_states(g, B, h, t, D, dtype, "token") for h, t in ((H, Tq), (Hk, Tk), (Hk, Tk)))
    lengths = torch.tensor([0, 1, 127, 128, 129, 256, 300, 999, -5], device="cuda")
    mask = torch.rand(B, Tk, generator=g, device="cuda") < 0.5
    mask[0] = False
    mask[1] = False
    mask[1, 299] = True
    mask[2, :200] = False
    mask[3, 130:] = False
    mask[4] = True
    for dt in (torch.int32, torch.int64):
        o = _run(rt, q, k, v, f"lengths {dt}", lengths=lengths.to(dt))
        assert (o[0] == 0).all() and (o[8] == 0).all()
    o = _run(rt, q, k, v, "mask", key_mask=mask)
    assert (o[0] == 0).all()
    _run(rt, q, k, v, "both", key_mask=mask, lengths=lengths.int())
    _run(rt, q, k, v, "strided mask and lengths", key_mask=mask.t().contiguous().t(),
         lengths=lengths.repeat_interleave(2)[::2])
    _run(rt, q, k, v, "one mask for the batch", key_mask=mask[2:3].expand(B, Tk))


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("Tq", [1, 5, 200])
@pytest.mark.parametrize("D", [64, 128, 20])
def test_what_masked_keys_hold_has_no_effect(gpu_runtime, Tq, D, dtype):
    rt, g = gpu_runtime, torch.Generator("cuda").manual_seed(Tq + D)
    B, H, Hk, Tk = 3, 4, 2, 290
    q, k, v = (_states(g, B, h, t, D, dtype) for h, t in ((H, Tq), (Hk, Tk), (Hk, Tk)))
    lengths = torch.tensor([290, 131, 17], dtype=torch.int32, device="cuda")
    mask = torch.rand(B, Tk, generator=g, device="cuda") < 0.7
    out = ~(mask & (torch.arange(Tk, device="cuda") < lengths[:, None]))
    want = rt.attention(q, k, v, lengths=lengths, key_mask=mask)
    for bad in (float("nan"), float("inf"), float("-inf"), torch.finfo(dtype).max, torch.finfo(dtype).min):
        k2, v2 = (t.masked_fill(out[:, None, :, None], bad) for t in (k, v))
        assert torch.equal(rt.attention(q, k2, v2, lengths=lengths, key_mask=mask), want), bad
    o2 = ~(torch.arange(Tk, device="cuda") < lengths[:, None])
    want = rt.attention(q, k, v, lengths=lengths)
    k2, v2 = (t.masked_fill(o2[:, None, :, None], float("nan")) for t in (k, v))
    assert torch.equal(rt.attention(q, k2, v2, lengths=lengths), want)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("Tq", [1, 150])
def test_growing_scores(gpu_runtime, Tq, dtype):
    """Scores that rise along the keys, so that the running maximum moves in
    every tile by little and by much; scores far below the maximum; equal
    scores; large negative scores only."""
    rt, g = gpu_runtime, torch.Generator("cuda").manual_seed(Tq)
    B, H, Tk, D = 2, 3, 700, 64
    v = _states(g, B, H, Tk, D, dtype)
    for slope in (0.002, 0.02, 0.2, -0.1):
        q = torch.full((B, H, Tq, D), 1.0, device="cuda").to(dtype)
        k = (slope * torch.arange(Tk, device="cuda")[None, None, :, None].expand(B, H, Tk, D)).to(dtype)
        _run(rt, q, k, v, f"slope {slope}")
    _run(rt, q, torch.zeros_like(k), v, "equal scores")
    _run(rt, q, torch.full_like(k, -30.0), v, "negative scores")
    _run(rt, 3 * _states(g, B, H, Tq, D, dtype), 3 * _states(g, B, H, Tk, D, dtype), v, "wide scores")


@pytest.mark.parametrize("scale", [1.0, 0.01, 2.5])
def test_scale(gpu_runtime, scale):
    g = torch.Generator("cuda").manual_seed(1)
    for dtype in (F16, F32):
        for Tq in (1, 140):
            q, k, v = (_states(g, 2, 2, t, 64, dtype, gain=0.7) for t in (Tq, 210, 210))
            _run(gpu_runtime, q, k, v, f"{scale}", scale=scale)


@pytest.mark.parametrize("Hk", [4, 1])
def test_half_rows_off_16_bytes(gpu_runtime, Hk):
    """Views that are copied to aligned rows first: the aligned call's bits,
    in q's axis order; a row that stands for all keys; a captured call."""
    rt, g = gpu_runtime, torch.Generator("cuda").manual_seed(13)
    n = torch.tensor([400, 33], dtype=torch.int32, device="cuda")
    for Tq, D in ((1, 64), (300, 64), (300, 128)):
        q, k, v = _states(g, 2, 4, Tq, D, F16, "token"), _states(g, 2, Hk, 400, D, F16), _states(g, 2, Hk, 400, D, F16)
        want = rt.attention(q, k, v, lengths=n)

        def off(t):
            room = torch.full(tuple(t.shape[:-1]) + (D + 3,), float("nan"), dtype=F16, device="cuda")
            room[..., 1:D + 1].copy_(t)
            return room[..., 1:D + 1]
        for args in ((off(q), k, v), (q, off(k), v), (q, k, off(v)), (off(q), off(k), off(v))):
            assert torch.equal(rt.attention(*args, lengths=n), want)
        p = torch.empty(2 * Tq * 4 * D + 1, dtype=F16, device="cuda")[1:].view(2, Tq, 4, D).permute(0, 2, 1, 3)
        p.copy_(q)
        o = rt.attention(p, k, v, lengths=n)
        assert torch.equal(o, want) and o.stride() == want.stride()
        same = k[:, :, 7:8].expand(2, Hk, 400, D)
        assert torch.equal(rt.attention(q, same, v, lengths=n), rt.attention(q, same.contiguous(), v, lengths=n))
        args, s = (off(q), off(k), off(v)), torch.cuda.Stream()
        with torch.cuda.stream(s):
            rt.attention(*args, lengths=n)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            o = rt.attention(*args, lengths=n)
        args[0].neg_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, rt.attention(-q, k, v, lengths=n))


@pytest.mark.parametrize("B,H,Hk,Tq,Tk,D", [(2, 4, 2, 300, 300, 36), (1, 2, 1, 150, 700, 7), (2, 2, 2, 260, 500, 100),
                                            (1, 2, 2, 1, 900, 1), (1, 3, 3, 140, 400, 65)])
def test_half_dims_off_16_bytes(gpu_runtime, B, H, Hk, Tq, Tk, D):
    g = torch.Generator("cuda").manual_seed(14)
    mask = torch.rand(B, Tk, generator=g, device="cuda") < 0.7
    mask[-1] = False
    for layout in ("head", "token"):
        q, k, v = (_states(g, B, h, t, D, F16, layout) for h, t in ((H, Tq), (Hk, Tk), (Hk, Tk)))
        _run(gpu_runtime, q, k, v, layout)
        _run(gpu_runtime, q, k, v, layout, key_mask=mask)


def test_scale_is_taken_by_value(gpu_runtime):
    """One scalar tensor whose value changes between two calls."""
    g = torch.Generator("cuda").manual_seed(12)
    q, k, v = (_states(g, 1, 2, t, 64, F32) for t in (3, 50, 50))
    s = torch.tensor(0.1)
    for x in (0.1, 0.7):
        s.fill_(x)
        assert torch.equal(gpu_runtime.attention(q, k, v, scale=s), gpu_runtime.attention(q, k, v, scale=float(s)))


def test_non_finite_values_stay_in_their_rows(gpu_runtime):
    g = torch.Generator("cuda").manual_seed(2)
    for dtype in (F16, F32):
        for Tq in (7, 200):
            q, k, v = (_states(g, 1, 2, t, 64, dtype) for t in (Tq, 150, 150))
            want = gpu_runtime.attention(q, k, v)
            q2 = q.clone()
            q2[0, 1, 3, 5] = float("nan")
            o = gpu_runtime.attention(q2, k, v)
            assert o[0, 1, 3].isnan().all()
            o[0, 1, 3] = want[0, 1, 3]
            assert torch.equal(o, want)
            v2 = v.clone()
            v2[0, 0, 149, 9] = float("inf")
            o = gpu_runtime.attention(q, k, v2)
            assert torch.isinf(o[0, 0, :, 9]).all() and torch.isfinite(o[0, 0, :, :9]).all()
            assert torch.equal(o[0, 1], want[0, 1])


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("Tq", [1, 4, 190])
def test_views(gpu_runtime, Tq, dtype):
    rt, g = gpu_runtime, torch.Generator("cuda").manual_seed(Tq)
    B, H, D, Tk = 2, 3, 64, 170
    qkv = torch.randn(B, max(Tq, Tk), 3, H, D, generator=g, device="cuda").to(dtype)   # one fused projection
    q, k, v = qkv[:, :Tq, 0].permute(0, 2, 1, 3), qkv[:, :Tk, 1].permute(0, 2, 1, 3), qkv[:, :Tk, 2].permute(0, 2, 1, 3)
    want = _run(rt, q, k, v, "fused projection")
    assert torch.equal(rt.attention(q.contiguous(), k.contiguous(), v.contiguous()), want)
    off = torch.randn(B, H, Tk, D + 3, generator=g, device="cuda").to(dtype)
    _run(rt, q, off[..., 3:], off[..., :D], "rows off 16 bytes")
    _run(rt, q, off[..., 3:].transpose(2, 3).contiguous().transpose(2, 3), v, "dim-major keys")
    _run(rt, q, k[:, :, ::2], v[:, :, ::2], "every other key")
    _run(rt, q[:, :, ::3], k, v, "every third query")
    _run(rt, q, k[:1].expand(B, H, Tk, D), v[:, :1].expand(B, H, Tk, D), "broadcast batch and heads")
    _run(rt, q[:, :1].expand(B, 5, Tq, D), k[:, :1], v[:, :1], "broadcast query heads")
    _run(rt, q, k.flip(2)[:, :, :Tk], v, "a reversed copy")
    one = torch.randn(1 + H * Tk * D, generator=g, device="cuda").to(dtype)[1:].view(1, H, Tk, D)
    _run(rt, q[:1], one, one, "a base off 16 bytes")


def test_empty(gpu_runtime):
    rt = gpu_runtime
    for dtype in (F16, F32):
        for Tq in (1, 200):
            q = torch.randn(2, 4, Tq, 64, device="cuda").to(dtype)
            none = torch.empty(2, 2, 0, 64, device="cuda", dtype=dtype)
            assert (rt.attention(q, none, none) == 0).all()
            assert rt.attention(q[:, :, :0], q, q).shape == (2, 4, 0, 64)
            assert rt.attention(q[:0], q[:0], q[:0]).shape == (0, 4, Tq, 64)


def test_refusals(gpu_runtime):
    rt = gpu_runtime
    q = torch.randn(2, 4, 5, 64, device="cuda")
    k = torch.randn(2, 2, 7, 64, device="cuda")
    n = torch.ones(2, dtype=torch.int32, device="cuda")
    m = torch.ones(2, 7, dtype=torch.bool, device="cuda")
    for args, kw, err in (((q.double(), k.double(), k.double()), {}, TypeError), ((q, k.half(), k), {}, TypeError),
                          ((q[0], k, k), {}, ValueError), ((q, k, k[:, :, :3]), {}, ValueError),
                          ((q[:, :3], k, k), {}, ValueError), ((q[..., :32], k, k), {}, ValueError),
                          ((q, k, k), {"lengths": n.float()}, TypeError), ((q, k, k), {"lengths": n[:1]}, ValueError),
                          ((q, k, k), {"key_mask": m.int()}, TypeError), ((q, k, k), {"key_mask": m[:, :3]}, ValueError),
                          ((q, k, k), {"lengths": n.cpu()}, ValueError), ((q, k, k), {"lengths": [1, 2]}, TypeError),
                          ((q, k, k), {"scale": 0.0}, RuntimeError), ((q.cpu(), k, k), {}, ValueError),
                          ((torch.cat([q, q, q], 3), torch.cat([k, k, k], 3), torch.cat([k, k, k], 3)), {}, RuntimeError)):
        with pytest.raises(err):
            rt.attention(*args, **kw)


def test_offsets_past_32_bits(gpu_runtime):
    """A key buffer whose second batch entry starts 2^31 elements on."""
    g = torch.Generator("cuda").manual_seed(3)
    far = (1 << 31) + 64
    buf = torch.empty(far + 2 * 400 * 64, dtype=F16, device="cuda")
    kv = buf.as_strided((2, 2, 400, 64), (far, 400 * 64, 64, 1))
    kv.copy_(torch.randn(2, 2, 400, 64, generator=g, device="cuda").half())
    for Tq in (1, 140):
        q = torch.randn(2, 2, Tq, 64, generator=g, device="cuda").half()
        _run(gpu_runtime, q, kv, kv, f"Tq={Tq}")
    del buf, kv
    torch.cuda.empty_cache()


def test_rows_around_the_result_are_left_alone(gpu_runtime):
    """bt_attention into the middle of a larger buffer."""
    import ctypes
    from bt_b200._lib import check
    from bt_b200.runtime import tensor_desc
    rt, g = gpu_runtime, torch.Generator("cuda").manual_seed(4)
    for dtype, Tq, D, left, wide in ((dt, t, d, left, wide) for dt in (F16, F32) for t in (1, 130, 300)
                                     for d in (64, 128, 40) for left, wide in ((8, 144), (3, 141), (1, 144))):
        q, k, v = (_states(g, 2, 16, t, D, dtype) for t in (Tq, 90, 90))
        room = torch.full((2, 18, Tq + 5, wide), 7.0, dtype=dtype, device="cuda")
        out = room[:, 1:17, 2:2 + Tq, left:left + D]
        rt._stream()
        check(rt.lib.bt_attention(ctypes.byref(tensor_desc(q)), ctypes.byref(tensor_desc(k)), ctypes.byref(tensor_desc(v)),
                                  None, None, 0.125, ctypes.byref(tensor_desc(out))), "bt_attention")
        torch.cuda.synchronize()
        assert torch.equal(out, rt.attention(q, k, v, scale=0.125))
        rest = room.clone()
        rest[:, 1:17, 2:2 + Tq, left:left + D] = 7.0
        assert (rest == 7.0).all()


def test_repeats_bit_for_bit_on_streams_threads_and_graphs(gpu_runtime):
    rt, g = gpu_runtime, torch.Generator("cuda").manual_seed(5)
    cases = [tuple(_states(g, 2, 4, t, 64, dt) for t in (Tq, 800, 800)) for dt, Tq in ((F16, 1), (F16, 333), (F32, 100), (F32, 2))]
    want = [rt.attention(*c) for c in cases]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got[i] = rt.attention(*cases[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:   # noqa: BLE001
            errors.append(e)
    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not errors
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    s, graphs, outs = torch.cuda.Stream(), [], []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            outs.append(rt.attention(*c))
        graphs.append(graph)
    for q, k, v in cases:
        q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
        k.copy_(torch.randn(k.shape, generator=g, device="cuda"))
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for c, o in zip(cases, outs):
        assert torch.equal(o, rt.attention(*c))


# ---- the operators together --------------------------------------------------------
@pytest.mark.parametrize("T,S", [(1, 40), (50, 77), (510, 510)])
def test_attention_block(gpu_runtime, T, S):
    """Frames [2, T, 768] attend to encoder states [2, S, 768] through int8
    projections of 12 heads: each step against 64 bits on its own inputs."""
    rt, g = gpu_runtime, torch.Generator("cuda").manual_seed(T)
    B, C, H = 2, 768, 12

    def weight():
        return rt.quantize_rows(0.03 * torch.randn(C, C, generator=g, device="cuda"))

    x, enc = torch.randn(B, T, C, generator=g, device="cuda"), torch.randn(B, S, C, generator=g, device="cuda")
    lengths = torch.tensor([S, (S + 1) // 2], dtype=torch.int32, device="cuda")
    bias = torch.randn(C, generator=g, device="cuda")

    def project(t, w, out=F32):
        q, s = rt.quantize_rows(t)
        y = rt.matmul_int8(q, s, *w, bias=bias, out_dtype=out)
        assert_within(y, *matmul_int8_64(q, s, *w, bias, out), "projection")
        # the quantised product of normal rows stays near the full product
        full = t.double() @ (w[0].double() * w[1].double()[:, None]).t() + bias.double()
        step = (s.double()[..., None] / 2) * (w[0].double().abs() * w[1].double()[:, None]).sum(-1)
        lim = step * 1.0001 + 4 * EPS32 * full.abs() + EPS32 * 1000
        assert_within(y, full, lim + (2 * EPS16 * (full.abs() + lim) if out == F16 else 0), "quantised")
        return y

    for out in (F32, F16):
        wq, wk, wv, wo = (weight() for _ in range(4))
        heads = [project(t, w, out).view(B, -1, H, C // H).permute(0, 2, 1, 3) for t, w in ((x, wq), (enc, wk), (enc, wv))]
        o = _run(rt, *heads, "block", lengths=lengths)
        y = project(o.permute(0, 2, 1, 3).reshape(B, T, C), wo)
        assert y.shape == (B, T, C) and torch.isfinite(y).all()


def test_no_wait_gave_up(gpu_runtime):
    """Every bounded wait of the runs above ended by what it waited for."""
    import ctypes
    from bt_b200._lib import check
    n = ctypes.c_uint32(99)
    check(gpu_runtime.lib.bt_wait_timeouts(ctypes.byref(n)), "bt_wait_timeouts")
    assert n.value == 0

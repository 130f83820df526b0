"""Row quantisation (bt_quantize_rows) against its float32 definition, bit for
bit, and the int8 product (bt_matmul_int8) against 64 bits."""
import threading

import numpy as np
import pytest
import torch

from opcheck import assert_within, matmul_int8_64, quantize_rows_np
from parity import assert_same

pytestmark = pytest.mark.gpu


# ---- quantize_rows ---------------------------------------------------------------
def _quant(rt, x, what=""):
    q, s = rt.quantize_rows(x)
    torch.cuda.synchronize()
    wq, ws = quantize_rows_np(x.cpu().numpy())
    assert q.shape == x.shape and q.dtype == torch.int8
    assert_same(q.cpu().numpy(), wq, f"values {what}")
    assert_same(s.cpu().numpy(), ws, f"scale {what}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("rows,K", [(1, 1), (1, 768), (3, 2), (5, 7), (7, 16), (33, 31), (2, 100), (64, 510), (9, 512),
                                    (17, 1023), (300, 1024), (4, 2047), (40, 4096), (3, 5000), (2, 16384), (2, 70001),
                                    (20001, 24)])
def test_quantize_sizes(gpu_runtime, rows, K, dtype):
    g = torch.Generator("cuda").manual_seed(rows * 100 + K)
    _quant(gpu_runtime, (torch.randn(rows, K, generator=g, device="cuda") * 2.5).to(dtype), f"{rows}x{K}")


def test_quantize_special_rows(gpu_runtime):
    x = np.random.default_rng(0).standard_normal((14, 600)).astype(np.float32)
    x[0] = 0
    x[1] = -0.0
    x[2, 5] = np.nan
    x[3, 599] = np.inf
    x[4, 0], x[4, 1] = -np.inf, np.nan
    x[5] *= 1e-38
    x[6] *= 1e-44
    x[7] *= 3e38 / np.abs(x[7]).max()
    x[8] = 1.0
    x[9] = np.arange(600) / 2 - 149.75 + 0.25      # ties and near-ties of the rounding
    x[9, 0] = 127.0 * 2
    x[10, :] = np.float32(2.0 ** -100)
    x[11, :] = np.float32(2.0 ** -101)
    x[12, 3:] = 0
    x[13, 100] = 1e30
    for K in (600, 599, 64, 1):
        for dt in (np.float32, np.float16):
            with np.errstate(over="ignore"):
                _quant(gpu_runtime, torch.from_numpy(np.ascontiguousarray(x[:, :K].astype(dt))).cuda(), f"K={K} {dt}")


def test_quantize_views(gpu_runtime):
    base = torch.randn(6, 40, 72, device="cuda")
    _quant(gpu_runtime, base[:, :, :50], "rows of a wider buffer")
    _quant(gpu_runtime, base[:, ::2, 3:], "every other row, off 16 bytes")
    _quant(gpu_runtime, base[:, 3:9], "a gap between the leading axes")
    _quant(gpu_runtime, base.transpose(1, 2), "transposed")
    _quant(gpu_runtime, base[0, 0], "one row, no leading axes")
    _quant(gpu_runtime, base.half()[1:, :, 1:], "half, off 4 bytes")
    _quant(gpu_runtime, base[:1, :1].expand(3, 4, 72), "broadcast rows")


def test_quantize_empty_and_refusals(gpu_runtime):
    q, s = gpu_runtime.quantize_rows(torch.empty(0, 32, device="cuda"))
    assert q.shape == (0, 32) and s.shape == (0,)
    with pytest.raises(ValueError):
        gpu_runtime.quantize_rows(torch.empty(4, 0, device="cuda"))
    with pytest.raises(TypeError):
        gpu_runtime.quantize_rows(torch.ones(4, 8, device="cuda", dtype=torch.int32))
    with pytest.raises(ValueError):
        gpu_runtime.quantize_rows(torch.ones(4, 8))


# ---- matmul_int8 -----------------------------------------------------------------
def _codes(g, rows, K, full=False):
    v = torch.randint(-128 if full else -127, 128, (rows, (K + 15) // 16 * 16), generator=g, device="cuda", dtype=torch.int8)
    return v[:, :K]


def _case(seed, M, N, K, bias, full=False):
    g = torch.Generator("cuda").manual_seed(seed)
    a, w = _codes(g, M, K, full), _codes(g, N, K, full)
    sa = torch.rand(M, generator=g, device="cuda") * 0.02 + 0.001
    sw = torch.rand(N, generator=g, device="cuda") * 0.002 + 0.0001
    b = torch.randn(N, generator=g, device="cuda") if bias else None
    return a, sa, w, sw, b


def _mm(rt, a, sa, w, sw, b, out, what=""):
    y = rt.matmul_int8(a, sa, w, sw, bias=b, out_dtype=out)
    torch.cuda.synchronize()
    assert y.dtype == out
    want, tol = matmul_int8_64(a, sa, w, sw, b, out)
    assert_within(y, want, tol, what)
    return y


SIZES = [(1, 1, 1), (1, 2048, 768), (1, 5, 16), (2, 128, 128), (3, 7, 5), (8, 130, 64), (16, 256, 2048), (17, 129, 200),
         (31, 1000, 33), (33, 64, 4096), (64, 768, 768), (77, 5001, 1000), (100, 100, 100), (127, 127, 127), (128, 128, 128),
         (129, 257, 129), (200, 768, 2048), (255, 384, 640), (256, 256, 256), (257, 513, 1025), (510, 768, 2048),
         (511, 2048, 768), (1000, 1000, 96), (1025, 300, 17), (2048, 2048, 512), (3000, 2500, 1100), (4096, 128, 128),
         (5, 9000, 64), (32640, 96, 32), (300, 3001, 5120)]


@pytest.mark.parametrize("out", [torch.float32, torch.float16])
@pytest.mark.parametrize("M,N,K", SIZES)
def test_matmul_sizes(gpu_runtime, M, N, K, out):
    for bias in (True, False):
        _mm(gpu_runtime, *_case(M + N + K, M, N, K, bias), out, f"{M}x{N}x{K} {out} bias={bias}")


def test_matmul_extreme_sum_and_infinite_scales(gpu_runtime):
    """K = 131071 values of -128 on both sides: the largest int32 sum."""
    K = 131071
    a = torch.full((3, 131072), -128, dtype=torch.int8, device="cuda")[:, :K]
    w = torch.full((130, 131072), -128, dtype=torch.int8, device="cuda")[:, :K]
    w[5] = 127
    sa, sw = torch.ones(3, device="cuda"), torch.ones(130, device="cuda")
    _mm(gpu_runtime, a, sa, w, sw, None, torch.float32, "largest sums")
    with pytest.raises(ValueError):
        gpu_runtime.matmul_int8(torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), sa[:1],
                                torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), sw[:1])
    a, sa, w, sw, b = _case(3, 40, 70, 96, True)
    sa[3], sa[7], sw[9] = float("nan"), float("inf"), float("inf")
    y = gpu_runtime.matmul_int8(a, sa, w, sw, bias=b)
    want = matmul_int8_64(a, sa, w, sw, b, torch.float32)[0]
    assert torch.equal(y.isnan(), want.isnan()) and y[3].isnan().all()
    rows = [i for i in range(40) if i not in (3, 7)]
    cols = [i for i in range(70) if i != 9]
    clean = y[rows][:, cols]
    assert torch.isfinite(clean).all()


def test_matmul_half_overflow_is_infinity(gpu_runtime):
    a, sa, w, sw, b = _case(4, 20, 30, 64, False)
    y = gpu_runtime.matmul_int8(a, sa * 1e6, w, sw * 1e6, out_dtype=torch.float16)
    want = matmul_int8_64(a, sa * 1e6, w, sw * 1e6, None, torch.float32)[0]
    big = want.abs() > 65536
    assert big.any() and torch.isinf(y[big]).all()


def test_matmul_layouts(gpu_runtime):
    rt = gpu_runtime
    a, sa, w, sw, b = _case(5, 60, 90, 160, True)
    want = _mm(rt, a, sa, w, sw, b, torch.float32)
    for name, a2, w2 in (("rows off 16 bytes", torch.empty(60, 161, dtype=torch.int8, device="cuda")[:, 1:], w),
                         ("pitch not a multiple of 16", torch.empty(60, 170, dtype=torch.int8, device="cuda")[:, :160], w),
                         ("column-major a", torch.empty(160, 60, dtype=torch.int8, device="cuda").t(), w),
                         ("column-major w", a, torch.empty(160, 90, dtype=torch.int8, device="cuda").t()),
                         ("every other row", torch.empty(120, 160, dtype=torch.int8, device="cuda")[::2], w)):
        if a2 is not a:
            a2.copy_(a)
        if w2 is not w:
            w2.copy_(w)
        assert torch.equal(rt.matmul_int8(a2, sa, w2, sw, bias=b), want), name
    s2 = torch.empty(120, device="cuda")[::2]
    s2.copy_(sa)
    w3, b3 = torch.empty(180, device="cuda")[::2], torch.empty(270, device="cuda")[::3]
    w3.copy_(sw)
    b3.copy_(b)
    assert torch.equal(rt.matmul_int8(a, s2, w, w3, bias=b3), want)
    y = rt.matmul_int8(a.reshape(3, 20, 160), sa.reshape(3, 20), w, sw, bias=b)
    assert torch.equal(y.reshape(60, 90), want)
    one = rt.matmul_int8(a[7], sa[7], w, sw, bias=b)       # a vector: no leading axes
    assert one.shape == (90,) and torch.equal(one, want[7])
    rep = rt.matmul_int8(a[7:8].expand(50, 160), sa[7:8].expand(50), w, sw, bias=b)
    assert torch.equal(rep, want[7:8].expand(50, 90))


def test_matmul_empty(gpu_runtime):
    rt = gpu_runtime
    a, sa, w, sw, b = _case(6, 4, 8, 32, True)
    assert rt.matmul_int8(a[:0], sa[:0], w, sw).shape == (0, 8)
    assert rt.matmul_int8(a, sa, w[:0], sw[:0]).shape == (4, 0)
    assert torch.equal(rt.matmul_int8(a[:, :0], sa, w[:, :0], sw, bias=b), b.expand(4, 8))
    assert torch.equal(rt.matmul_int8(a[:, :0], sa, w[:, :0], sw), torch.zeros(4, 8, device="cuda"))


def test_matmul_and_quantize_empty_in_any_layout(gpu_runtime):
    """Operands without values: allocated as such, or seen through odd strides."""
    rt = gpu_runtime
    a, w = torch.empty(4, 0, dtype=torch.int8, device="cuda"), torch.empty(8, 0, dtype=torch.int8, device="cuda")
    sa, sw, b = torch.ones(4, device="cuda"), torch.ones(8, device="cuda"), torch.arange(8.0, device="cuda")
    assert torch.equal(rt.matmul_int8(a, sa, w, sw, bias=b), b.expand(4, 8))
    a3 = torch.empty(3, 2, 0, dtype=torch.int8, device="cuda").transpose(0, 1)
    assert torch.equal(rt.matmul_int8(a3, torch.ones(2, 3, device="cuda"), w, sw, bias=b), b.expand(2, 3, 8))
    none, rows = torch.empty(3, 0, 16, device="cuda"), torch.empty(3, 0, device="cuda")
    assert rt.matmul_int8(none.char(), rows, torch.ones(8, 16, dtype=torch.int8, device="cuda"), sw).shape == (3, 0, 8)
    q, s = rt.quantize_rows(none)
    assert q.shape == (3, 0, 16) and s.shape == (3, 0)


def test_matmul_refusals(gpu_runtime):
    rt = gpu_runtime
    a, sa, w, sw, b = _case(7, 4, 8, 32, True)
    for args, kw, err in (((a.float(), sa, w, sw), {}, TypeError), ((a, sa, w.short(), sw), {}, TypeError),
                          ((a, sa.double(), w, sw), {}, TypeError), ((a, sa, w, sw), {"bias": b.half()}, TypeError),
                          ((a, sa, w, sw), {"out_dtype": torch.bfloat16}, TypeError), ((a, sa, w[:, :16], sw), {}, ValueError),
                          ((a, sa[:3], w, sw), {}, ValueError), ((a, sa, w, sw[:3]), {}, ValueError),
                          ((a, sa, w, sw), {"bias": b[:5]}, ValueError), ((a.cpu(), sa, w, sw), {}, ValueError),
                          ((a, sa, w.reshape(2, 4, 32), sw), {}, ValueError), ((a, 0.5, w, sw), {}, TypeError)):
        with pytest.raises(err):
            rt.matmul_int8(*args, **kw)


def test_matmul_repeats_bit_for_bit(gpu_runtime):
    for M, N, K in ((1, 300, 4096), (50, 700, 3000), (600, 768, 2048)):
        args = _case(M, M, N, K, True)
        y = gpu_runtime.matmul_int8(*args[:4], bias=args[4])
        for _ in range(5):
            assert torch.equal(gpu_runtime.matmul_int8(*args[:4], bias=args[4]), y)


def test_streams_threads_and_graphs(gpu_runtime):
    """Two streams and two threads at once; a captured pass replayed on new inputs."""
    rt = gpu_runtime
    cases = [_case(i, 70 + i, 200, 520, True) for i in range(4)]
    want = [rt.matmul_int8(*c[:4], bias=c[4]) for c in cases]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i] = rt.matmul_int8(*cases[i][:4], bias=cases[i][4])
                torch.cuda.current_stream().synchronize()
        except Exception as e:   # noqa: BLE001
            errors.append(e)
    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not errors
    for g, w in zip(got, want):
        assert torch.equal(g, w)
    x = torch.randn(70, 520, device="cuda")
    w, sw, b = cases[0][2], cases[0][3], cases[0][4]
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        rt.matmul_int8(*rt.quantize_rows(x), w, sw, bias=b)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        y = rt.matmul_int8(*rt.quantize_rows(x), w, sw, bias=b)
    for i in range(3):
        x.copy_(torch.randn(70, 520, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, rt.matmul_int8(*rt.quantize_rows(x), w, sw, bias=b))


def test_no_wait_gave_up(gpu_runtime):
    """Every bounded wait of the runs above ended by what it waited for."""
    import ctypes
    from bt_b200._lib import check
    n = ctypes.c_uint32(99)
    check(gpu_runtime.lib.bt_wait_timeouts(ctypes.byref(n)), "bt_wait_timeouts")
    assert n.value == 0

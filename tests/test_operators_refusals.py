"""Refusals of bt_quantize_rows, bt_matmul_int8 and bt_attention: bad
arguments return a status with a message before any launch (no GPU)."""
import ctypes

import numpy as np
import pytest

from bt_b200 import _lib

F32, F16, I8, I32, BOOL = np.float32, np.float16, np.int8, np.int32, np.bool_


def T(dt, *shape, strides=None, ptr=1 << 20):
    return _lib.make_tensor(ptr, dt, shape, strides)


def _ref(t):
    return None if t is None else ctypes.byref(t)


def _refused(lib, rc, code, word):
    assert rc == code, (rc, lib.bt_last_error())
    assert word in lib.bt_last_error(), lib.bt_last_error()


@pytest.mark.parametrize("x,q,s,code,word", [
    (T(I8, 4, 8), T(I8, 4, 8), T(F32, 4), -3, b"float32 or float16"),
    (T(F32, 4, 8), T(np.uint8, 4, 8), T(F32, 4), -3, b"int8"),
    (T(F32, 4, 8), T(I8, 4, 9), T(F32, 4), -2, b"same rows"),
    (T(F32, 4, 0), T(I8, 4, 0), T(F32, 4), -2, b"without values"),
    (T(F32, 4, 8), T(I8, 4, 8), T(F32, 5), -2, b"scale"),
    (T(F32, 4, 8), T(I8, 4, 8), T(F16, 4), -3, b"scale"),
    (T(F32, 4, 8, strides=(16, 2)), T(I8, 4, 8), T(F32, 4), -5, b"unit stride"),
    (T(F32, 2, 4, 8, strides=(100, 8, 1)), T(I8, 8, 8), T(F32, 8), -5, b"one stride"),
    (T(F32, 4, 8, ptr=None), T(I8, 4, 8), T(F32, 4), -1, b"null data"),
    (T(F32), T(I8, 1), T(F32, 1), -2, b"at least one axis"),
])
def test_quantize_rows(lib, x, q, s, code, word):
    _refused(lib, lib.bt_quantize_rows(_ref(x), _ref(q), _ref(s)), code, word)


@pytest.mark.parametrize("change,code,word", [
    ({"a": T(np.uint8, 4, 32)}, -3, b"int8"),
    ({"w": T(F32, 8, 32)}, -3, b"int8"),
    ({"out": T(np.float64, 4, 8)}, -3, b"float32 or float16"),
    ({"w": T(I8, 8, 48)}, -2, b"values a row"),
    ({"w": T(I8, 2, 4, 32)}, -2, b"two axes"),
    ({"out": T(F32, 4, 9)}, -2, b"row count"),
    ({"a_scale": T(F32, 5)}, -2, b"a_scale"),
    ({"a_scale": None}, -1, b"a_scale"),
    ({"w_scale": T(F16, 8)}, -3, b"w_scale"),
    ({"bias": T(F32, 4)}, -2, b"bias"),
    ({"a": T(I8, 4, 131072), "w": T(I8, 8, 131072)}, -6, b"131071"),
    ({"a": T(I8, 4, 32, strides=(64, 2))}, -5, b"unit stride"),
    ({"a": T(I8, 4, 32, ptr=None)}, -1, b"null data"),
])
def test_matmul_int8(lib, change, code, word):
    t = {"a": T(I8, 4, 32), "a_scale": T(F32, 4), "w": T(I8, 8, 32), "w_scale": T(F32, 8), "bias": T(F32, 8),
         "out": T(F32, 4, 8)}
    t.update(change)
    _refused(lib, lib.bt_matmul_int8(*(_ref(t[n]) for n in ("a", "a_scale", "w", "w_scale", "bias", "out"))), code, word)


@pytest.mark.parametrize("change,code,word", [
    ({"q": T(I8, 2, 4, 5, 64)}, -3, b"float32 or float16"),
    ({"k": T(F32, 2, 2, 7, 64)}, -3, b"one dtype"),
    ({"q": T(F16, 8, 5, 64), "out": T(F16, 8, 5, 64)}, -2, b"[batch, heads, length, dim]"),
    ({"v": T(F16, 2, 2, 8, 64)}, -2, b"same shape"),
    ({"out": T(F16, 2, 4, 6, 64)}, -2, b"q's shape"),
    ({"k": T(F16, 3, 2, 7, 64), "v": T(F16, 3, 2, 7, 64)}, -2, b"batch and dim"),
    ({"k": T(F16, 2, 3, 7, 64), "v": T(F16, 2, 3, 7, 64)}, -2, b"cannot share"),
    ({"k": T(F16, 2, 0, 7, 64), "v": T(F16, 2, 0, 7, 64)}, -2, b"cannot share"),
    ({n: T(F16, 2, 4, 5, 136) for n in ("q", "k", "v", "out")}, -6, b"outside 1..128"),
    ({"lengths": T(F32, 2)}, -3, b"lengths"),
    ({"lengths": T(I32, 3)}, -2, b"lengths"),
    ({"key_mask": T(np.uint8, 2, 7)}, -3, b"key_mask"),
    ({"key_mask": T(BOOL, 2, 8)}, -2, b"key_mask"),
    ({"scale": 0.0}, -1, b"scale"),
    ({"scale": -1.0}, -1, b"scale"),
    ({"scale": float("nan")}, -1, b"scale"),
    ({"scale": float("inf")}, -1, b"scale"),
    ({"q": T(F16, 2, 4, 5, 64, ptr=None)}, -1, b"null data"),
    ({"out": None}, -1, b"out"),
])
def test_attention(lib, change, code, word):
    t = {"q": T(F16, 2, 4, 5, 64), "k": T(F16, 2, 2, 7, 64), "v": T(F16, 2, 2, 7, 64), "lengths": None,
         "key_mask": None, "scale": 0.125, "out": T(F16, 2, 4, 5, 64)}
    t.update(change)
    rc = lib.bt_attention(_ref(t["q"]), _ref(t["k"]), _ref(t["v"]), _ref(t["lengths"]), _ref(t["key_mask"]), t["scale"],
                          _ref(t["out"]))
    _refused(lib, rc, code, word)


def test_empty_results_need_no_gpu(lib):
    x, q, s = T(F32, 0, 8), T(I8, 0, 8), T(F32, 0)
    assert lib.bt_quantize_rows(_ref(x), _ref(q), _ref(s)) == 0
    a, sa, w, sw, o = T(I8, 0, 32), T(F32, 0), T(I8, 8, 32), T(F32, 8), T(F32, 0, 8)
    assert lib.bt_matmul_int8(_ref(a), _ref(sa), _ref(w), _ref(sw), None, _ref(o)) == 0
    q, k, o = T(F16, 2, 4, 0, 64), T(F16, 2, 2, 7, 64), T(F16, 2, 4, 0, 64)
    assert lib.bt_attention(_ref(q), _ref(k), _ref(k), None, None, 0.125, _ref(o)) == 0


@pytest.mark.parametrize("shape", [(4, 0), (2, 3, 0), (3, 0, 16), (0, 5)])
def test_operands_without_values_need_no_copy(shape):
    torch = pytest.importorskip("torch")
    from bt_b200.runtime import _one_row_stride, _row_pitch_ok
    for t in (torch.empty(shape, dtype=torch.int8), torch.empty(shape[::-1], dtype=torch.int8).permute(
            *reversed(range(len(shape))))):
        assert _one_row_stride(t) and _row_pitch_ok(t)


@pytest.mark.parametrize("scale,rc", [(2.35e38, 0), (1e-30, 0), (2.37e38, -1), (3.4e38, -1)])
def test_attention_scales_that_overflow(lib, scale, rc):
    """scale * log2(e) has to be finite in float32."""
    q, k = T(F16, 2, 4, 0, 64), T(F16, 2, 2, 7, 64)
    assert lib.bt_attention(_ref(q), _ref(k), _ref(k), None, None, scale, _ref(q)) == rc
    if rc:
        assert b"scale" in lib.bt_last_error()

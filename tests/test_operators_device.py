"""The device of the launches of quantize_rows, matmul_int8 and attention where
another one is current: a stand-in library records it (no GPU)."""
import threading

import pytest
import torch

from bt_b200 import runtime

CURRENT, OWN = 0, -1     # (get_device() of a CPU tensor is -1)


class Library:
    """Every entry returns BT_OK and notes its name and the current device."""

    def __init__(self, state):
        self.state, self.calls = state, []

    def __getattr__(self, name):
        def entry(*args):
            self.calls.append((name, self.state["current"]))
            return 0
        return entry


@pytest.fixture
def rt(monkeypatch):
    state = {"current": CURRENT}

    class device:
        def __init__(self, d):
            assert d == torch.device("cpu")

        def __enter__(self):
            self.before, state["current"] = state["current"], OWN

        def __exit__(self, *exc):
            state["current"] = self.before

    monkeypatch.setattr(runtime.torch.cuda, "device", device)
    monkeypatch.setattr(runtime, "_get_device", lambda: state["current"])
    monkeypatch.setattr(runtime, "_raw_stream", lambda index: 0)
    r = runtime.BtRuntime.__new__(runtime.BtRuntime)
    r.device, r._index, r.launches, r._local = torch.device("cpu"), OWN, 0, threading.local()
    r.lib, r.state = Library(state), state
    return r


def _launches(rt):
    calls = [c for c in rt.lib.calls if c[0] != "bt_set_stream"]
    assert all(d == OWN for _, d in calls), calls
    assert rt.state["current"] == CURRENT and rt.launches == len(calls)
    names = [n for n, _ in calls]
    rt.lib.calls.clear()
    rt.launches = 0
    return names


def test_operands_read_in_place(rt):
    x, w = torch.randn(6, 32), torch.ones(5, 32, dtype=torch.int8)
    q, s = rt.quantize_rows(x)
    rt.matmul_int8(q, s, w, torch.ones(5))
    h = torch.zeros(2, 4, 300, 64, dtype=torch.float16)
    rt.attention(h, h, h)
    assert _launches(rt) == ["bt_quantize_rows", "bt_matmul_int8", "bt_attention"]


def test_operands_that_are_copied_first(rt):
    rt.quantize_rows(torch.randn(6, 32).t())
    assert _launches(rt) == ["bt_elementwise", "bt_quantize_rows"]
    a, w = torch.ones(6, 33, dtype=torch.int8)[:, 1:], torch.ones(5, 40, dtype=torch.int8)[:, :32]
    rt.matmul_int8(a, torch.ones(12)[::2], w, torch.ones(5))
    assert _launches(rt) == ["bt_elementwise"] * 3 + ["bt_matmul_int8"]
    h = torch.zeros(2, 4, 300, 68, dtype=torch.float16)[..., 1:65]
    rt.attention(h, h, h)
    assert _launches(rt) == ["bt_elementwise"] * 3 + ["bt_attention"]

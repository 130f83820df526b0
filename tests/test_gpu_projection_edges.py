"""The int8 product (bt_matmul_int8) where its summed axis is empty."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out", [torch.float32, torch.float16])
def test_an_empty_sum_is_0_whatever_the_scales(gpu_runtime, out):
    """quantize_rows gives rows with an infinity or a NaN such scales."""
    rt = gpu_runtime
    sa = torch.tensor([1.0, float("inf"), float("nan"), -float("inf"), 0.0], device="cuda")
    sw = torch.tensor([1.0, float("nan"), float("inf")], device="cuda")
    b = torch.tensor([0.5, -2.0, float("inf")], device="cuda")
    a, w = (torch.empty(n, 0, dtype=torch.int8, device="cuda") for n in (5, 3))
    assert torch.equal(rt.matmul_int8(a, sa, w, sw, out_dtype=out), torch.zeros(5, 3, device="cuda", dtype=out))
    assert torch.equal(rt.matmul_int8(a, sa, w, sw, bias=b, out_dtype=out), b.to(out).expand(5, 3))

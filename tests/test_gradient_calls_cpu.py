"""What the gradient operators and their autograd forms do around a launch, as far as it needs no GPU."""
import pytest
import torch

from sinkattn_amd import ops


def odd_views(dtype):
    """Dense [B, H, N, D] tensors whose dims of size 1 have strides that no kernel takes, and one on an address that
    no 16-byte load takes."""
    return {"one row": torch.zeros(1, 3, 64, 1, dtype=dtype).transpose(2, 3),
            "one batch": torch.zeros(3, 40, 64, 1, dtype=dtype).permute(3, 0, 1, 2),
            "one head": torch.zeros(2, 40, 64, 1, dtype=dtype).permute(0, 3, 1, 2),
            "one row, no stride": torch.zeros(2, 3, 1, 64, dtype=dtype).as_strided((2, 3, 1, 64), (192, 64, 0, 1)),
            "odd address": torch.zeros(2 * 3 * 40 * 64 + 1, dtype=dtype)[1:].view(2, 3, 40, 64)}


def addressable(t):
    return t.stride(3) == 1 and not any(s % 8 for s in t.stride()[:3]) and t.data_ptr() % 16 == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("what", list(odd_views(torch.float32)))
def test_operands_and_gradients_of_odd_strides(dtype, what):
    t = odd_views(dtype)[what]
    t.copy_(torch.arange(t.numel()).view(t.shape) % 100)
    for kept in (ops._kernel_operand(t), ops._grad_operand(t)):
        assert addressable(kept) and torch.equal(kept, t)
    for out_dtype in (dtype, torch.float32):
        grad = ops._grad_output(t, out_dtype)
        assert grad.shape == t.shape and grad.dtype == out_dtype
        assert addressable(grad) and grad.stride(2) >= 64


@pytest.mark.parametrize("layout", ["bhnd", "bnhd"])
def test_gradients_keep_the_order_of_dims(layout):
    t = torch.zeros(2, 3, 40, 64) if layout == "bhnd" else torch.zeros(2, 40, 3, 64).transpose(1, 2)
    assert ops._grad_output(t, torch.float32).stride() == t.stride()

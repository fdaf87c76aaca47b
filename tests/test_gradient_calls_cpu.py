"""What the gradient operators and their autograd forms do around a launch, as far as it needs no GPU."""
import pytest
import torch
from torch.autograd import forward_ad

from sinkattn_amd import autograd, ops


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


class _Twice(torch.autograd.Function):
    """A step whose saved tensors are gone after its backward pass."""

    @staticmethod
    def forward(ctx, x):
        ctx.save_for_backward(x)
        return 2 * x

    @staticmethod
    def backward(ctx, g):
        return 2 * g + 0 * ctx.saved_tensors[0]


def test_copy_into_a_buffer_used_again():
    """A buffer that every call writes: no call's graph holds an earlier one's."""
    x = torch.ones(2, 3, requires_grad=True)
    out = torch.empty(2, 3)
    for i in range(3):
        assert autograd.copy_into(out, _Twice.apply(x)) is out
        edges = out.grad_fn.next_functions
        assert [e[0] for e in edges].count(None) == len(edges) - 1
        (g,) = torch.autograd.grad(out.sum(), x)
        assert torch.equal(g, torch.full((2, 3), 2.0))
    # without a backward pass between the calls, and where something still reads the earlier result
    first = autograd.copy_into(out, _Twice.apply(x)) * 3
    autograd.copy_into(out, _Twice.apply(x))
    assert torch.equal(torch.autograd.grad(first.sum(), x)[0], torch.full((2, 3), 6.0))
    assert torch.equal(torch.autograd.grad(out.sum(), x)[0], torch.full((2, 3), 2.0))


def test_copy_into_parts_of_a_buffer():
    """Views of one buffer, written one after the other: each part's gradient arrives."""
    x, y = (torch.ones(3, requires_grad=True) for _ in range(2))
    base = torch.zeros(2, 3)
    for i, t in enumerate((x, y)):
        autograd.copy_into(base[i], _Twice.apply(t))
    for g in torch.autograd.grad(base.sum(), (x, y)):
        assert torch.equal(g, torch.full((3,), 2.0))


def test_tangents_are_seen():
    x = torch.ones(1, 1, 8, 64)
    assert not autograd.has_tangent(x, None)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, x)
        assert autograd.has_tangent(None, d) and autograd.needs_grad(x, d)
        assert not autograd.has_tangent(x, torch.zeros(2, dtype=torch.bool)) and not autograd.needs_grad(x)
        with torch.no_grad():
            assert autograd.needs_grad(d)  # forward mode goes on without recorded gradients
    assert not autograd.needs_grad(x)

"""Calls of the gradient operators and their autograd forms that a program may make around the usual ones: operands of
unusual strides, buffers used again, masks that change, streams, other ways of differentiation."""
import math

import pytest
import torch
from torch.autograd import forward_ad

from sinkattn_amd import ops
from sinkattn_amd import sparse_attention as sa
from sinkattn_amd import timing
from sinkattn_amd import wan_runtime as wr
from sinkattn_amd import zimage_runtime as zr

from backward_bars import check, formula, make, make_mask, plans

pytestmark = pytest.mark.gpu


def odd_view(t, what):
    """t's values with strides in its dims of size 1, or on an address, that no kernel takes."""
    B, H, N, D = t.shape
    if what == "one row":
        x = torch.empty(B, H, D, 1, dtype=t.dtype, device=t.device).transpose(2, 3)
    elif what == "one batch":
        x = torch.empty(H, N, D, 1, dtype=t.dtype, device=t.device).permute(3, 0, 1, 2)
    else:
        x = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape)
    return x.copy_(t)


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 32)])
@pytest.mark.parametrize("what,B,Nq,Nk", [("one row", 2, 1, 1), ("one batch", 1, 200, 300), ("odd address", 2, 130, 70)])
def test_odd_strides(dtype, D, what, B, Nq, Nk):
    """Dims of size 1 with odd strides and odd addresses: the plain layout's results, in the op and through autograd."""
    ts = make(B, 3, Nq, Nk, D, dtype, layout="bhnd", seed=71)
    mask = make_mask(B, 3, Nq, Nk, 1.0)
    plan, kplan = plans(mask)
    q, k, v, do = ts
    out, lse = ops.block_sparse_attention(q, k, v, plan)
    want = ops.block_sparse_attention_backward(do, q, k, v, out, lse, plan, kplan)
    q, k, v, do, o = (odd_view(t, what) for t in (*ts, out))
    got = ops.block_sparse_attention_backward(do, q, k, v, o, lse, plan, kplan)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    y, _ = sa._block_sparse_attn(*leaves, mask)
    assert torch.equal(y, out)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, leaves, do), want))


@pytest.mark.parametrize("what,B,N", [("one row", 2, 25), ("one batch", 1, 100), ("odd address", 2, 100)])
def test_pool_odd_strides(what, B, N):
    """The pooling's gradient from an output gradient of such strides."""
    gap = 30
    x = make(B, 2, N, N, 64, torch.bfloat16, layout="bhnd", seed=72)[0]
    rows = -(-N // gap)
    d = make(B, 2, rows, rows, 64, torch.bfloat16, layout="bhnd", seed=73)[0]
    want = ops.mean_pool_tokens_backward(d, N, gap)
    got = ops.mean_pool_tokens_backward(odd_view(d, what), N, gap, add=None)
    assert torch.equal(got, want)
    leaf = x.clone().requires_grad_()
    y = sa._mean_pool_sequence(leaf, gap)
    assert torch.equal(torch.autograd.grad(y, leaf, odd_view(d, what))[0], want)
    if what != "one row":
        more = odd_view(x, what)
        assert torch.equal(ops.mean_pool_tokens_backward(d, N, gap, add=more), ops.mean_pool_tokens_backward(d, N, gap, add=x))


def test_compensation_into_a_buffer_used_again():
    """The compensated call's `out` as a buffer that every step writes."""
    N, gap = 400, 30
    mask = make_mask(1, 2, N, N, 0.6, seed=74)
    out = torch.empty(1, 2, N, 128, dtype=torch.bfloat16, device="cuda")
    for seed in range(3):
        q, k, v, do = make(1, 2, N, N, 128, torch.bfloat16, seed=80 + seed)
        kd, vd = ops.mean_pool_kv(k, v, gap)
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        fresh = sa._block_sparse_attn_with_compensation(*leaves, mask, kd, vd, gap)
        want = torch.autograd.grad(fresh, leaves, do)
        got = sa._block_sparse_attn_with_compensation(*leaves, mask, kd, vd, gap, out=out)
        assert got is out and torch.equal(got, fresh)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, leaves, do), want))


def op_gradients(q, k, v, do, mask):
    plan, kplan = plans(mask)
    out, lse = ops.block_sparse_attention(q, k, v, plan)
    return [out, *ops.block_sparse_attention_backward(do, q, k, v, out, lse, plan, kplan)]


def call_gradients(leaves, do, mask):
    out, _ = sa._block_sparse_attn(*leaves, mask)
    return [out.detach(), *torch.autograd.grad(out, leaves, do)]


def same(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_mask_written_by_a_graph():
    """A mask buffer that a replayed graph fills, which torch does not count as a change of the tensor: each call takes
    the mask as it is."""
    N, D = 700, 64
    q, k, v, do = make(1, 2, N, N, D, torch.bfloat16, seed=75)
    masks = [make_mask(1, 2, N, N, 0.5, seed=s) for s in (75, 76)]
    want = [op_gradients(q, k, v, do, m) for m in masks]
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    source, mask = masks[0].clone(), torch.zeros_like(masks[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mask.copy_(source)
    for turn in (0, 1, 1, 0):
        source.copy_(masks[turn])
        version = mask._version
        graph.replay()
        assert mask._version == version
        for _ in range(2):
            assert same(call_gradients(leaves, do, mask), want[turn])


def test_mask_changed_before_the_backward_pass():
    """The backward pass takes the mask that the forward saw."""
    q, k, v, do = make(1, 2, 500, 600, 64, torch.float16, seed=77)
    masks = [make_mask(1, 2, 500, 600, 0.5, seed=s) for s in (77, 78)]
    want = op_gradients(q, k, v, do, masks[0])
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    mask = masks[0].clone()
    out, _ = sa._block_sparse_attn(*leaves, mask)
    mask.copy_(masks[1])
    for _ in range(2):
        assert same(torch.autograd.grad(out, leaves, do, retain_graph=True), want[1:])
    del mask
    assert same(torch.autograd.grad(out, leaves, do), want[1:])


def test_mask_made_in_inference_mode():
    q, k, v, do = make(1, 2, 300, 300, 64, torch.bfloat16, seed=79)
    mask = make_mask(1, 2, 300, 300, 0.6, seed=79)
    with torch.inference_mode():
        kept = mask.clone()
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    assert same(call_gradients(leaves, do, kept), op_gradients(q, k, v, do, mask))


def test_one_mask_on_two_streams():
    """Differentiable calls on two streams at once that share one mask: the bits of calls one by one."""
    N, D = 1500, 128
    mask = make_mask(1, 3, N, N, 0.4, seed=81)
    sets = [make(1, 3, N, N, D, torch.bfloat16, seed=81 + i) for i in range(2)]
    want = [op_gradients(*s, mask) for s in sets]
    leaves = [[t.clone().requires_grad_() for t in s[:3]] for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        fresh = mask.clone()
        got = []
        for stream, ls, s in zip(streams, leaves, sets):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                got.append(call_gradients(ls, s[3], fresh))
        torch.cuda.synchronize()
        assert all(same(g, w) for g, w in zip(got, want))


@pytest.mark.parametrize("comp", [False, True])
def test_more_query_blocks_than_a_key_plan_takes(comp):
    """Such calls run where an input asks for a gradient, with the results of a call without; their backward passes raise."""
    N, D, gap = 8192 * 128 + 5, 128 if comp else 32, 30
    g = torch.Generator(device="cuda").manual_seed(86)
    q, k, v = (torch.randn(1, 1, n, D, device="cuda", generator=g).bfloat16() for n in (N, 200, 200))
    mask = torch.ones(1, 1, 8193, 2, dtype=torch.bool, device="cuda")
    kd, vd = ops.mean_pool_kv(k, v, gap)

    def call(q, k, v):
        if comp:
            return sa._block_sparse_attn_with_compensation(q, k, v, mask, kd, vd, gap)
        return sa._block_sparse_attn(q, k, v, mask)[0]

    plain = call(q, k, v)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = call(*leaves)
    assert torch.equal(out, plain)
    with pytest.raises(RuntimeError, match="8193 blocks of queries"):
        torch.autograd.grad(out, leaves, torch.zeros_like(out))


def test_forward_mode():
    """The attention refuses tangents instead of dropping them; pooling and QK norms carry them."""
    N, gap = 260, 30
    q, k, v, t = make(1, 2, N, N, 128, torch.bfloat16, layout="bhnd", seed=87)
    mask = make_mask(1, 2, N, N, 1.0)
    kd, vd = ops.mean_pool_kv(k, v, gap)
    with forward_ad.dual_level():
        for i in range(3):
            args = [q, k, v]
            args[i] = forward_ad.make_dual(args[i], t)
            for grad in (torch.enable_grad, torch.no_grad):
                with grad():
                    with pytest.raises(NotImplementedError):
                        sa._block_sparse_attn(*args, mask)
                    with pytest.raises(NotImplementedError):
                        sa._block_sparse_attn_with_compensation(*args, mask, kd, vd, gap)
                    with pytest.raises(NotImplementedError):
                        wr.WanSinkSparseInnerAttention(0, mask[0], sa.SinkSparseConfig(sample_gap=gap))(*args)
        x = forward_ad.make_dual(k, t)
        for prefix in (0, 17):
            y = sa._mean_pool_sequence_preserve_prefix(x, gap, prefix_tokens=prefix)
            tangent = forward_ad.unpack_dual(y).tangent
            # the pooling is linear: the tangent is the pooled tangent, a sum of `gap` terms and two roundings apart
            # from the kernel's
            want = ops.mean_pool_tokens(t, gap, prefix).double()
            bound = 2 * torch.finfo(t.dtype).eps * ops.mean_pool_tokens(t.abs(), gap, prefix).double() * 1.05
            assert ((tangent.double() - want).abs() <= bound).all()

    class Norms:
        heads = 2
        norm_q, norm_k = (torch.nn.RMSNorm(256, eps=1e-6, device="cuda", dtype=torch.bfloat16) for _ in range(2))

    rows = [u.transpose(1, 2).flatten(2) for u in (q, k, t)]
    assert wr._fused_qk_prep(Norms, rows[0], rows[1], None) is not None
    with forward_ad.dual_level():
        assert wr._fused_qk_prep(Norms, forward_ad.make_dual(rows[0], rows[2]), rows[1], None) is None


def timed():
    state = sa.SinkRuntimeState()
    state.timing = timing.AttentionTimingCollector(label="sink", enabled=True)
    return state


def sections(state):
    return {name: entry["count"] for name, entry in state.summarize_timing()["by_section"].items()}


def test_timing_sections_with_gradients():
    """A layer call records the same sections and pooled lengths whether an input asks for a gradient or not."""
    N, text = 700, 40
    q, k, v, _ = make(1, 2, N, N, 128, torch.bfloat16, seed=88)
    mask = make_mask(1, 2, N, N, 0.5, seed=88)
    seen = []
    for grad in (False, True):
        state = timed()
        layer = wr.WanSinkSparseInnerAttention(0, mask[0], sa.SinkSparseConfig(sample_gap=30, text_length=text), runtime_state=state)
        layer(*(t.clone().requires_grad_(grad) for t in (q, k, v)))
        seen.append((sections(state), state.sparsity_events))
    assert "comp_pool" in seen[0][0] and seen[0] == seen[1]


def test_timing_sections_of_an_image_layer_with_gradients():
    H, D, side, text = 2, 128, 16, 20
    cfg = zr.build_zimg_sink_config(config_overrides=dict(token_width=side, token_height=side, dynamic_mode="pooled_kv",
                                                          sample_gap=30))
    nb = zr._fixed_block_shape(cfg)[2]

    class Layer(torch.nn.Module):
        heads = H

        def __init__(self):
            super().__init__()
            self.to_q, self.to_k, self.to_v = (torch.nn.Linear(H * D, H * D) for _ in range(3))
            self.to_out = torch.nn.ModuleList([torch.nn.Linear(H * D, H * D)])
            self.norm_q, self.norm_k = (torch.nn.RMSNorm(D, eps=1e-6) for _ in range(2))

    layer = Layer().bfloat16().cuda()
    x = torch.randn(1, side * side + text, H * D, device="cuda").bfloat16()
    seen = []
    for grad in (False, True):
        state = timed()
        proc = zr.ZImageStaticSinkProcessor(layer_idx=0, total_layers=2, sink_mask=torch.ones(H, nb, nb, dtype=torch.bool),
                                            config=cfg, runtime_state=state)
        with torch.set_grad_enabled(grad):
            proc(layer, x)
        seen.append((sections(state), state.sparsity_events))
    assert "comp_pool" in seen[0][0] and seen[0] == seen[1]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_more_heads_than_launch_chunks(dtype):
    """More heads than a plan deals to the XCDs in chunks (4096): the launch order without a chunk table."""
    B, H, N, D = 65, 64, 200, 32
    q, k, v, do = make(B, H, N, N, D, dtype, seed=89)
    mask = make_mask(B, H, N, N, 0.7, seed=89)
    plan, kplan = plans(mask)
    out, lse = ops.block_sparse_attention(q, k, v, plan)
    grads = ops.block_sparse_attention_backward(do, q, k, v, out, lse, plan, kplan)
    for b in (0, 31, 64):
        at = slice(b, b + 1)
        want, off = formula(q[at], k[at], v[at], do[at], out[at], lse[at], mask[at], 1 / math.sqrt(D))
        check([g[at] for g in grads], want, off)
    assert all(torch.isfinite(g).all() for g in grads)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,H,N", [(1, 1, 5000), (1, 6, 3300)])
def test_long_lists_of_head_dim_32(dtype, B, H, N):
    """Lists that are cut into parts at the smallest head dim."""
    q, k, v, do = make(B, H, N, N, 32, dtype, seed=90)
    mask = make_mask(B, H, N, N, 0.05, seed=90)
    mask[..., 0] = mask[..., 17] = True
    mask[:, :, 3] = True
    plan, kplan = plans(mask)
    out, lse = ops.block_sparse_attention(q, k, v, plan)
    grads = ops.block_sparse_attention_backward(do, q, k, v, out, lse, plan, kplan)
    want, off = formula(q, k, v, do, out, lse, mask, 1 / math.sqrt(32))
    check(grads, want, off)
    assert same(grads, ops.block_sparse_attention_backward(do, q, k, v, out, lse, plan, kplan))

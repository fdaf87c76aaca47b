"""Differentiable forms of the layer's kernels.

The names of `sinkattn_amd.sparse_attention` and the two runtimes call these where gradients are
recorded and an input asks for one; without gradients they call `ops` directly.  Forward results
are the same bits either way.  What a forward saves is what torch's own attention saves: its
operands, its output and the fp32 log-sum-exp; probabilities are recomputed in the backward pass,
which runs on the forward's stream, allocates through torch and can be captured into a graph with it.
Second derivatives and forward-mode differentiation are refused.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import ops


def has_tangent(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether one of the tensors carries a tangent of forward-mode differentiation."""
    if getattr(forward_ad, "_current_level", 0) < 0:  # outside every dual level
        return False
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def needs_grad(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether gradients are recorded and one of the tensors asks for one, or one carries a tangent (which the forms
    below refuse, and a kernel's plain call would drop)."""
    return (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)) or has_tangent(*tensors)


def copy_into(out: torch.Tensor, res: torch.Tensor) -> torch.Tensor:
    """res copied into `out`, which takes res's place in the graph.  All of `out` is overwritten, so a whole
    tensor's own history ends here: torch's copy_ keeps it, and a buffer used again would hold every earlier call's
    graph and run through it.  (Of a view only a part of its base is overwritten: the base's history stays.)"""
    if out.grad_fn is not None and not out._is_view():
        out.detach_()
    return out.copy_(res)


def _plan(mask: torch.Tensor) -> ops.BlockSparsePlan:
    """A plan of the mask as it is now, made on the current stream and kept by nothing but the call's graph: no write
    to the mask, from wherever it comes, is missed.  Its launch order comes from the stream's cache of orders by tile
    counts, but not in a capture, whose replays may run beside that stream."""
    with torch.cuda.device(mask.device):
        captured = torch.cuda.is_current_stream_capturing()
    if captured or mask.dim() != 4 or mask.numel() == 0:
        return ops.block_sparse_plan(mask)
    return ops.block_sparse_plan(mask, ops.PLAN_CACHE.order_cache(mask), ops.PLAN_CACHE.ORDER_CACHE_ENTRIES)


MAX_QUERY_BLOCKS = 8192  # of the transposed mask's plan


def _plans(mask: torch.Tensor) -> Tuple[ops.BlockSparsePlan, Optional[ops.BlockSparsePlan]]:
    """The mask's plan and key plan; no key plan where the mask has more query blocks than one takes: the forward
    runs all the same, and a backward pass says so."""
    plan = _plan(mask)
    return plan, _plan(mask.transpose(2, 3)) if plan.shape[2] <= MAX_QUERY_BLOCKS else None


def _key_plan(ctx) -> ops.BlockSparsePlan:
    if ctx.key_plan is None:
        raise RuntimeError(f"block-sparse attention gradient: {ctx.plan.shape[2]} blocks of queries, at most {MAX_QUERY_BLOCKS} "
                           "are supported")
    return ctx.key_plan


class _BlockSparseAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, mask, return_lse):
        ctx.plan, ctx.key_plan = _plans(mask)
        out, lse = ops.block_sparse_attention(q, k, v, ctx.plan)
        ctx.save_for_backward(q, k, v, out, lse)
        ctx.set_materialize_grads(False)
        return (out, lse.to(q.dtype).unsqueeze(-1)) if return_lse else (out, None)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, dlse):
        q, k, v, out, lse = ctx.saved_tensors
        if dout is None and dlse is None:
            return None, None, None, None, None
        if dout is None:
            dout = torch.zeros_like(out)
        if dlse is not None:
            dlse = dlse.squeeze(-1).float()
        return (*ops.block_sparse_attention_backward(dout, q, k, v, out, lse, ctx.plan, _key_plan(ctx), dlse=dlse),
                None, None)


def block_sparse_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: torch.Tensor,
                           return_lse: bool) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """out [B, H, Nq, D] and the lse [B, H, Nq, 1] in q.dtype (or None) of `_block_sparse_attn`."""
    return _BlockSparseAttention.apply(q, k, v, mask, return_lse)


class _BlockSparseAttentionComp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, kd, vd, mask, gap, comp_rows):
        ctx.plan, ctx.key_plan = _plans(mask)
        ctx.gap, ctx.comp_rows = gap, comp_rows
        out, lse = ops.block_sparse_attention_comp(q, k, v, ctx.plan, kd, vd, gap, comp_rows=comp_rows, return_lse=True)
        ctx.save_for_backward(q, k, v, kd, vd, out, lse)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, kd, vd, out, lse = ctx.saved_tensors
        grads = ops.block_sparse_attention_comp_backward(dout, q, k, v, out, lse, ctx.plan, _key_plan(ctx), kd, vd, ctx.gap,
                                                         comp_rows=ctx.comp_rows)
        return (*grads, None, None, None)


def block_sparse_attention_comp(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: torch.Tensor,
                                kd: torch.Tensor, vd: torch.Tensor, gap: int,
                                comp_rows: Optional[int]) -> torch.Tensor:
    """`_block_sparse_attn_with_compensation` on pooled keys of the caller's."""
    return _BlockSparseAttentionComp.apply(q, k, v, kd, vd, mask, gap, comp_rows)


class _BlockSparseAttentionPooled(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, kd, vd, mask, gap, prefix, pool_end, comp_rows):
        ctx.plan, ctx.key_plan = _plans(mask)
        ctx.pool, ctx.comp_rows = (gap, prefix, pool_end), comp_rows
        out, lse = ops.block_sparse_attention_comp(q, k, v, ctx.plan, kd, vd, gap, comp_rows=comp_rows, return_lse=True)
        ctx.save_for_backward(q, k, v, kd, vd, out, lse)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, kd, vd, out, lse = ctx.saved_tensors
        gap, prefix, pool_end = ctx.pool
        dq, dk, dv, dkd, dvd = ops.block_sparse_attention_comp_backward(
            dout, q, k, v, out, lse, ctx.plan, _key_plan(ctx), kd, vd, gap, comp_rows=ctx.comp_rows,
            key_grad_dtype=torch.float32)
        # the pooled keys' share joins the attention's in fp32: one rounding of the whole gradient
        dk, dv = ops.mean_pool_kv_backward(dkd, dvd, int(k.shape[2]), gap, prefix, pool_end, add=(dk, dv), out_dtype=k.dtype)
        return dq, dk, dv, None, None, None, None, None, None, None


def block_sparse_attention_pooled(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, mask: torch.Tensor, gap: int,
                                  prefix: int = 0, pool_end: Optional[int] = None,
                                  comp_rows: Optional[int] = None,
                                  pooled: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> torch.Tensor:
    """`ops.mean_pool_kv` and the compensated attention over its rows as one step of the graph, so that K
    and V get one gradient each.  `pooled`: that call's rows of these K and V, where the caller has made them."""
    kd, vd = ops.mean_pool_kv(k, v, gap, prefix, pool_end) if pooled is None else pooled
    return _BlockSparseAttentionPooled.apply(q, k, v, kd, vd, mask, gap, prefix, pool_end, comp_rows)


class _MeanPoolTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gap, prefix):
        ctx.n, ctx.gap, ctx.prefix = int(x.shape[2]), gap, prefix
        return ops.mean_pool_tokens(x, gap, prefix)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        return ops.mean_pool_tokens_backward(dout, ctx.n, ctx.gap, ctx.prefix), None, None


def mean_pool_tokens(x: torch.Tensor, gap: int, prefix: int = 0) -> torch.Tensor:
    """`ops.mean_pool_tokens` with its gradient."""
    return _MeanPoolTokens.apply(x, gap, prefix)


class _QkNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, wk, eps_q, eps_k, head_dim, freq_real, freq_imag, rows_per_pos):
        ctx.scalars = (eps_q, eps_k, head_dim)
        ctx.rows_per_pos = rows_per_pos
        ctx.save_for_backward(q, k, wq, wk, freq_real, freq_imag)
        ctx.set_materialize_grads(False)
        return ops.qk_norm_rotary(q, k, wq, wk, eps_q, eps_k, head_dim, freq_real, freq_imag, rows_per_pos=rows_per_pos)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, wq, wk, freq_real, freq_imag = ctx.saved_tensors
        if dq_out is None and dk_out is None:
            return (None,) * 10
        dq_out = torch.zeros_like(q) if dq_out is None else dq_out
        dk_out = torch.zeros_like(k) if dk_out is None else dk_out
        dq, dk, dwq, dwk = ops.qk_norm_rotary_backward(dq_out, dk_out, q, k, wq, wk, *ctx.scalars, freq_real, freq_imag,
                                                       rows_per_pos=ctx.rows_per_pos)
        return dq, dk, dwq.to(wq), dwk.to(wk), None, None, None, None, None, None


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, wq: torch.Tensor, wk: torch.Tensor, eps_q: float, eps_k: float,
                   head_dim: int, freq_real: Optional[torch.Tensor] = None, freq_imag: Optional[torch.Tensor] = None,
                   rows_per_pos: int = 1) -> Tuple[torch.Tensor, torch.Tensor]:
    """`ops.qk_norm_rotary` with the gradients of q, k and both weights (the tables are constants)."""
    return _QkNormRotary.apply(q, k, wq, wk, eps_q, eps_k, head_dim, freq_real, freq_imag, rows_per_pos)

"""Varlen attention with a learned bias by relative position, on the gfx950 kernels (esa_rel_attn_fwd / _bwd).

``relative_attention`` is ``varlen_attention`` without a mask whose scores get
``bias[bucket(d), head]``, d the key's position minus the query's in their
segment: what tells the tokens of a chain (residues, bases, edges in chain
order) apart in the unmasked layers.  The reference has no counterpart: its
layers see a set.  ``bucket_starts`` says which distances share a bucket.
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .attention import _SEED_MASK, _check_dropout, _check_index, _check_tokens, draw_dropout_seed
from .eager import EXACT, FITS, ordinary

MAX_REACH, MAX_BUCKETS = 768, 256
_TABLE = (torch.float32, torch.bfloat16)


@functools.lru_cache(maxsize=64)
def bucket_starts(num_buckets: int, max_distance: int = 128, bidirectional: bool = True) -> tuple[int, ...]:
    """The distances at which the buckets of one side begin.

    ``bidirectional``: half of the buckets for keys up to the query, half for keys after it; else all of them for keys
    up to the query, every later key in bucket 0.  The first half of a side's buckets hold one distance each
    (0, 1, ...), the others grow by a constant factor: with n buckets on the side and e = n // 2, bucket e + t begins
    at the least distance x with (x / e) ** (n - e) >= (max_distance / e) ** t, compared in whole numbers.  The last
    bucket has no end; where several begin at one distance, the last of them holds it.
    """
    num_buckets, max_distance = int(num_buckets), int(max_distance)
    side = num_buckets // 2 if bidirectional else num_buckets
    if bidirectional and num_buckets % 2:
        raise ValueError(f"num_buckets must be even for both sides (got {num_buckets})")
    if side < 2 or num_buckets > MAX_BUCKETS or side > MAX_BUCKETS // 2:
        raise ValueError(f"num_buckets must give a side 2 to {MAX_BUCKETS // 2} buckets (got {num_buckets}, "
                         f"{'two sides' if bidirectional else 'one side'})")
    exact = side // 2
    if max_distance <= exact:
        raise ValueError(f"max_distance must exceed the {exact} distances with a bucket of their own (got {max_distance})")
    wide, starts, x = side - exact, list(range(exact)), exact
    for t in range(wide):
        while x ** wide * exact ** t < max_distance ** t * exact ** wide:
            x += 1
            if x > MAX_REACH:
                raise ValueError(f"the last bucket would begin beyond distance {MAX_REACH} (num_buckets {num_buckets}, "
                                 f"max_distance {max_distance})")
        starts.append(x)
    return tuple(starts)


@functools.lru_cache(maxsize=64)
def _start_bytes(starts: tuple[int, ...]) -> bytes:
    return bytes((ctypes.c_int * len(starts))(*starts))


def _call(starts, scale, dropout_p, seed):
    """What the host module takes of a call besides its tensors."""
    return (_lib.address("esa_rel_attn_fwd"), _lib.address("esa_rel_attn_bwd"), _lib.address("esa_rel_attn_workspace_size"),
            _start_bytes(starts), scale, dropout_p, seed)


class _RelativeAttention(torch.autograd.Function):
    """The call where torch has to see it as a function (under transforms, tracing and dispatch modes, over subclasses);
    ordinary eager calls are a node of the host module's."""

    @staticmethod
    def forward(ctx, q, k, v, bias, cu_q, cu_k, q_start, starts, scale, dropout_p, seed):
        # kept for a backward: what the rounding of a bf16 out leaves, so that its row statistic has none
        call = _call(starts, scale, dropout_p, seed)
        rc, out, low, lse, table = _lib.tensors().relative_forward(*call, q, k, v, bias, q_start, cu_q, cu_k,
                                                                   any(ctx.needs_input_grad))
        _lib.check(rc, "esa_rel_attn_fwd")
        ctx.save_for_backward(q, k, v, table, out, low, lse, cu_q, cu_k, q_start)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(lse)
        ctx.call = call
        return out, lse

    @staticmethod
    @once_differentiable
    def backward(ctx, g, _):
        q, k, v, table, out, low, lse, cu_q, cu_k, q_start = ctx.saved_tensors
        if g is None:
            return (None,) * 11
        rc, dq, dk, dv, dtable = _lib.tensors().relative_backward(*ctx.call, q, k, v, table, q_start, cu_q, cu_k, out, low, lse, g)
        _lib.check(rc, "esa_rel_attn_bwd")
        return dq, dk, dv, dtable, None, None, None, None, None, None, None


def _check(q, k, v, bias, cu_seqlens_q, cu_seqlens_k, q_start):
    """Says what is wrong with a call that the host module found not to fit."""
    _check_tokens("q", q)
    heads, hd = q.shape[1], q.shape[2]
    _check_tokens("k", k, heads, q.dtype, hd)
    _check_tokens("v", v, heads, q.dtype, hd)
    if k.shape[0] != v.shape[0]:
        raise ValueError("k and v must have the same number of tokens")
    if bias.dtype not in _TABLE:
        raise TypeError(f"bias must be float32 or bfloat16 (got {bias.dtype})")
    if bias.dim() != 2 or bias.shape[1] != heads:
        raise ValueError(f"bias must be [num_buckets, heads = {heads}] (got {tuple(bias.shape)})")
    _check_index("cu_seqlens_q", cu_seqlens_q)
    batch = cu_seqlens_q.numel() - 1
    if batch < 1:
        raise ValueError("cu_seqlens_q must have at least two entries")
    _check_index("cu_seqlens_k", cu_seqlens_k, batch + 1)
    _check_index("q_start", q_start, batch)


def relative_attention(q, k, v, bias, cu_seqlens_q, cu_seqlens_k, max_seqlen_q=None, max_seqlen_k=None, max_distance=128,
                       bidirectional=True, q_start=None, dropout_p=0.0, softmax_scale=None, return_lse=False,
                       dropout_seed=None):
    """Unmasked varlen attention with the learned bias ``bias[bucket(d), head]`` added to the scaled scores.

    q: [Tq, H, hd]; k, v: [Tk, H, hd] (hd 16, 24, 32 or 64), contiguous, all bfloat16 or all float32; cu_seqlens_*:
    int32 [B + 1].  max_seqlen_* are taken as ``varlen_attention`` takes them and never change a result.
    bias: [num_buckets, H], float32 or bfloat16, with the buckets of
    ``bucket_starts(num_buckets, max_distance, bidirectional)``.
    d = (key's index in its segment) - (query's index in its segment) - q_start[segment]: q_start (int32 [B]) is the
    position of a segment's first query, where the queries are a later part of their chain (default 0).
    A table entry of -inf leaves its pairs out; finite entries beyond +-1e4 count as +-1e4.  A query without a key, or a
    token of no segment, gets 0 (lse -inf) and no gradient.
    dropout_p, dropout_seed, softmax_scale (positive), return_lse: as ``varlen_attention``'s; the lse has no gradient.
    Gradients reach q, k, v and bias (in its dtype, summed in float32 in a fixed order), once: they cannot be
    differentiated again.
    """
    dropout_p = _check_dropout(dropout_p)
    if dropout_p > 0.0 and dropout_seed is None:
        dropout_seed = draw_dropout_seed()
    flags = _lib.tensors().relative_fits(q, k, v, bias, cu_seqlens_q, cu_seqlens_k, q_start)
    if not flags & FITS:
        _check(q, k, v, bias, cu_seqlens_q, cu_seqlens_k, q_start)
    starts = bucket_starts(bias.shape[0], max_distance, bool(bidirectional))
    scale = 1.0 / math.sqrt(q.shape[2]) if softmax_scale is None else float(softmax_scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"softmax_scale must be positive and finite (got {softmax_scale})")
    if not flags & FITS:
        _lib.require_on_one_gpu(q, k, v, bias, cu_seqlens_q, cu_seqlens_k, q_start)
        q, k, v, bias = (t.resolve_neg() for t in (q, k, v, bias))
    seed = int(dropout_seed or 0) & _SEED_MASK
    if flags & EXACT and ordinary():
        rc, out, lse = _lib.tensors().relative(*_call(starts, scale, dropout_p, seed), q, k, v, bias, q_start, cu_seqlens_q,
                                               cu_seqlens_k)
        _lib.check(rc, "esa_rel_attn_fwd")
    else:
        out, lse = _RelativeAttention.apply(q, k, v, bias, cu_seqlens_q, cu_seqlens_k, q_start, starts, scale, dropout_p, seed)
    return (out, lse) if return_lse else out

"""Norms of queries and keys per head with the rotation of positions in the same pass (esa_qk_norm_fwd / _bwd).

``qk_norm_rotary`` takes projected query and key rows to what attention over
ordered tokens uses: each head's row divided by its root mean square, scaled
by weights shared by the heads, and its first dimensions rotated in pairs by
the token's position.  The reference has no counterpart: its layers see a set.
"""
from __future__ import annotations

import math

import torch
from torch.autograd.function import once_differentiable

from .. import _lib
from .attention import HEAD_DIMS
from .eager import EXACT, FITS, ordinary

_CODES = {torch.float32: _lib.ESA_F32, torch.bfloat16: _lib.ESA_BF16}
MAX_HEADS = 2048


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, device=None) -> torch.Tensor:
    """The radians per position of each pair, base ** (-2 i / rotary_dim), float64 [rotary_dim / 2]."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive (got {rotary_dim})")
    return float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)


def _call(eps, interleaved):
    """What the host module takes of a call besides its tensors."""
    return (_lib.address("esa_qk_norm_fwd"), _lib.address("esa_qk_norm_bwd"), _lib.address("esa_qk_norm_bwd_workspace_size"),
            eps, interleaved)


class _QkNorm(torch.autograd.Function):
    """The call where torch has to see it as a function (under transforms, tracing and dispatch modes, over subclasses);
    ordinary eager calls are a node of the host module's."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, frequencies, eps, interleaved):
        ctx.call = _call(eps, interleaved)
        rc, q_out, k_out, q, k = _lib.tensors().qk_norm_forward(*ctx.call, q, k, q_weight, k_weight, positions, frequencies)
        _lib.check(rc, "esa_qk_norm_fwd")
        ctx.save_for_backward(q, k, q_weight, k_weight, positions, frequencies)
        return (q_out, k_out) if k is not None else q_out

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk=None):
        rc, *grads = _lib.tensors().qk_norm_backward(*ctx.call, *ctx.saved_tensors, gq, gk, *ctx.needs_input_grad[2:4])
        _lib.check(rc, "esa_qk_norm_bwd")
        return *grads, None, None, None, None


def _check_rows(name: str, x: torch.Tensor, like: torch.Tensor | None = None) -> None:
    if x.dtype not in _CODES:
        raise TypeError(f"{name} must be float32 or bfloat16 (got {x.dtype})")
    if x.dim() != 3 or x.shape[2] not in HEAD_DIMS or not 1 <= x.shape[1] <= MAX_HEADS:
        raise ValueError(f"{name} must be [total, heads, head_dim] with 1 to {MAX_HEADS} heads and head_dim in {HEAD_DIMS} "
                         f"(got {tuple(x.shape)})")
    if like is not None and (x.dtype != like.dtype or x.shape[0] != like.shape[0] or x.shape[2] != like.shape[2]):
        raise ValueError(f"{name} must have the tokens, head_dim and dtype of q (got {tuple(x.shape)}, {x.dtype})")


def _check(q, k, q_weight, k_weight, positions, frequencies):
    """Says what is wrong with a call that the host module found not to fit."""
    _check_rows("q", q)
    if k is not None:
        _check_rows("k", k, q)
    elif k_weight is not None:
        raise ValueError("k_weight without k")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (tuple(w.shape) != (q.shape[2],) or w.dtype not in _CODES):
            raise ValueError(f"{name} must be a float32 or bfloat16 [{q.shape[2]}] (got {w.dtype}, {tuple(w.shape)})")
    if (positions is None) != (frequencies is None):
        raise ValueError("positions and frequencies must be given together")
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64) or positions.dim() != 1 or not positions.is_contiguous():
            raise TypeError(f"positions must be a contiguous 1-D int32 or int64 tensor (got {positions.dtype}, "
                            f"{tuple(positions.shape)})")
        if positions.numel() != q.shape[0]:
            raise ValueError(f"positions has {positions.numel()} entries, expected {q.shape[0]}")
        if frequencies.dtype != torch.float64 or frequencies.dim() != 1 or not frequencies.is_contiguous():
            raise TypeError(f"frequencies must be a contiguous 1-D float64 tensor (got {frequencies.dtype}, "
                            f"{tuple(frequencies.shape)})")
        r = 2 * frequencies.numel()
        if r % 8 or not 8 <= r <= q.shape[2]:
            raise ValueError(f"frequencies must rotate a multiple of 8 dimensions up to head_dim {q.shape[2]} (got {r})")


def qk_norm_rotary(q, k=None, q_weight=None, k_weight=None, positions=None, frequencies=None, eps=1e-6, interleaved=False):
    """(q', k') of query rows q [T, Hq, hd] and key rows k [T, Hk, hd] (k None: q' alone); hd 16, 24, 32 or 64, float32
    or bfloat16 with float32 arithmetic, rounded once.

    y = x / sqrt(mean(x ** 2) + eps) * weight over each head's row; q_weight / k_weight: [hd] or None (ones).  With
    ``positions`` (int32 or int64 [T], any values) and ``frequencies`` (float64 [r / 2], ``rotary_frequencies``; r a
    multiple of 8 up to hd), the first r dimensions are rotated in pairs (i, i + r / 2), or (2i, 2i + 1) with
    ``interleaved``, by positions * frequencies[i], worked out in 64 bits (an angle is off by at most 2^-51 of itself).

    q and k may be views (of one projection's output, say): rows of hd consecutive elements on 16-byte boundaries are
    read where they are, others from a copy.  The outputs are contiguous.  Gradients reach q, k and the weights (summed
    in float32 in a fixed order), once: they cannot be differentiated again.
    """
    flags = _lib.tensors().qk_norm_fits(q, k, q_weight, k_weight, positions, frequencies)
    if not flags & FITS:
        _check(q, k, q_weight, k_weight, positions, frequencies)
    eps = float(eps)
    if not (eps >= 0.0 and math.isfinite(eps)):
        raise ValueError(f"eps must be finite and not negative (got {eps})")
    if not flags & FITS:
        _lib.require_on_one_gpu(q, k, q_weight, k_weight, positions, frequencies)
        q, k, q_weight, k_weight, frequencies = (None if t is None else t.resolve_neg()
                                                 for t in (q, k, q_weight, k_weight, frequencies))
    if flags & EXACT and ordinary():
        rc, q_out, k_out = _lib.tensors().qk_norm(*_call(eps, bool(interleaved)), q, k, q_weight, k_weight, positions, frequencies)
        _lib.check(rc, "esa_qk_norm_fwd")
        return q_out if k is None else (q_out, k_out)
    return _QkNorm.apply(q, k, q_weight, k_weight, positions, frequencies, eps, bool(interleaved))

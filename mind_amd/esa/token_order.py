"""Blocks over tokens that have an order: what the encoder's self-attention layers take from ``token_order``.

The reference's layers see a set: nothing tells residue 5 of a chain from residue 50.  With a ``TokenOrder`` a layer's
queries and keys are normalised per head and rotated by their index in their graph (``qk_norm_rotary``), and its
unmasked attention adds a learned bias by relative position (``relative_attention``).  A masked layer's attention keeps
its mask and takes the norms and the rotation alone.  Without one nothing changes, the state dict's keys included.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch
from torch import nn

from .attention import HEAD_DIMS, varlen_attention
from .qk_norm import qk_norm_rotary, rotary_frequencies
from .relative import bucket_starts, relative_attention


@dataclass(frozen=True)
class TokenOrder:
    """rotary_dim: the dimensions of a head that are rotated, a multiple of 8 (None: all, 0: none), rotary_base their
    slowest pair's; num_buckets (0: no bias), max_distance, bidirectional: as in ``relative_attention``."""

    rotary_dim: int | None = None
    rotary_base: float = 10000.0
    num_buckets: int = 32
    max_distance: int = 128
    bidirectional: bool = True


class OrderedHeads(nn.Module):
    """The parameters of one layer's token order, and its attention: weights of ones, a bias table of zeros."""

    def __init__(self, order: TokenOrder, heads: int, head_dim: int, masked: bool):
        super().__init__()
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim {head_dim} is not supported by the kernels {HEAD_DIMS}")
        rotary = head_dim if order.rotary_dim is None else order.rotary_dim
        if rotary % 8 or not 0 <= rotary <= head_dim:
            raise ValueError(f"rotary_dim must be a multiple of 8 up to head_dim {head_dim} (got {rotary})")
        self.settings = order
        # no buffer: a module moved to another type keeps its angles in 64 bits
        self.frequencies = rotary_frequencies(rotary, order.rotary_base) if rotary else None
        self.q_weight, self.k_weight = nn.Parameter(torch.ones(head_dim)), nn.Parameter(torch.ones(head_dim))
        self.bias = None
        if order.num_buckets and not masked:
            bucket_starts(order.num_buckets, order.max_distance, order.bidirectional)   # its checks
            self.bias = nn.Parameter(torch.zeros(order.num_buckets, heads))

    def forward(self, q, k, v, positions, cu, longest, dropout_p=0.0, dropout_seed=None, **mask):
        """Self-attention of q, k, v [T, H, hd] by the segments cu; positions [T] (int64), mask: a masked layer's."""
        if self.frequencies is not None and self.frequencies.device != q.device:
            self.frequencies = self.frequencies.to(q.device)
        turned = self.frequencies is not None
        q, k = qk_norm_rotary(q, k, self.q_weight, self.k_weight, positions if turned else None, self.frequencies)
        if self.bias is None:
            return varlen_attention(q, k, v, cu, cu, longest, longest, dropout_p=dropout_p, dropout_seed=dropout_seed, **mask)
        return relative_attention(q, k, v, self.bias, cu, cu, longest, longest, self.settings.max_distance,
                                  self.settings.bidirectional, dropout_p=dropout_p, dropout_seed=dropout_seed)

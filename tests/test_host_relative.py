"""Relative position buckets and the refusals of the biased attention (no GPU needed)."""
import ctypes
import math

import pytest
import torch

from mind_amd import _lib
from mind_amd.esa.relative import bucket_starts, relative_attention


@pytest.mark.parametrize("n,distance,two", [(32, 128, True), (32, 128, False), (64, 512, True), (8, 20, True), (16, 40, False)])
def test_starts_against_the_logarithm(n, distance, two):
    """Bucket e + t holds the distances whose e + floor(log(x / e) / log(max / e) (n - e)) is that (64 bits, quotients
    within 1e-9 of a whole number taken as it), the last everything beyond."""
    starts = bucket_starts(n, distance, two)
    side = n // 2 if two else n
    e = side // 2
    assert len(starts) == side and list(starts[:e]) == list(range(e)) and starts[e] == e
    for x in range(1, 2 * distance):
        want = x if x < e else min(side - 1, e + math.floor(math.log(x / e) / math.log(distance / e) * (side - e) + 1e-9))
        assert max(i for i, s in enumerate(starts) if s <= x) == want


def test_known_starts():
    assert bucket_starts(32, 128) == (0, 1, 2, 3, 4, 5, 6, 7, 8, 12, 16, 23, 32, 46, 64, 91)
    assert bucket_starts(4, 2) == (0, 1)


@pytest.mark.parametrize("args", [(31, 128, True), (2, 128, True), (1, 10, False), (258, 700, True), (129, 600, False),
                                  (32, 8, True), (32, 7, True), (32, 4096, True)])
def test_starts_refused(args):
    with pytest.raises(ValueError):
        bucket_starts(*args)


def _args(t=6, h=2, hd=16, dtype=torch.bfloat16):
    x = torch.zeros(t, h, hd, dtype=dtype)
    cu = torch.tensor([0, t], dtype=torch.int32)
    return dict(q=x, k=x, v=x, bias=torch.zeros(32, h), cu_seqlens_q=cu, cu_seqlens_k=cu)


@pytest.mark.parametrize("change,error", [
    (dict(q=torch.zeros(6, 2, 20, dtype=torch.bfloat16)), ValueError), (dict(q=torch.zeros(6, 2, 16)), TypeError),
    (dict(k=torch.zeros(6, 3, 16, dtype=torch.bfloat16)), ValueError),
    (dict(v=torch.zeros(5, 2, 16, dtype=torch.bfloat16)), ValueError),
    (dict(q=torch.zeros(6, 2, 32, dtype=torch.bfloat16)[..., ::2]), ValueError),
    (dict(bias=torch.zeros(32, 3)), ValueError), (dict(bias=torch.zeros(32, 2, dtype=torch.float16)), TypeError),
    (dict(bias=torch.zeros(33, 2)), ValueError), (dict(max_distance=4), ValueError), (dict(dropout_p=1.0), ValueError),
    (dict(softmax_scale=0.0), ValueError), (dict(softmax_scale=math.inf), ValueError),
    (dict(softmax_scale=math.nan), ValueError), (dict(cu_seqlens_q=torch.tensor([0, 6])), TypeError),
    (dict(cu_seqlens_k=torch.tensor([0, 3, 6], dtype=torch.int32)), ValueError),
    (dict(cu_seqlens_q=torch.zeros(1, dtype=torch.int32)), ValueError),
    (dict(q_start=torch.zeros(2, dtype=torch.int32)), ValueError), (dict(q_start=torch.zeros(1)), TypeError),
    (dict(), _lib.EsaError)])   # host tensors
def test_refused(change, error):
    with pytest.raises(error):
        relative_attention(**{**_args(), **change})


def test_entry_points_refuse_before_launch():
    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    lib, n = _lib.load(), ctypes.c_size_t(0)
    bf16 = _lib.ESA_BF16

    def size(batch=2, tq=100, tk=90, h=4, hd=16, dt=bf16, nb=4, starts=(0, 3), ns=None, bwd=1):
        s = (ctypes.c_int * max(len(starts), 1))(*starts)
        return lib.esa_rel_attn_workspace_size(batch, tq, tk, h, hd, dt, nb, s, len(starts) if ns is None else ns, bwd,
                                               ctypes.byref(n))
    assert size() == 0 and n.value > 0
    assert size(hd=48) == -3 and size(dt=5) == -5 and size(batch=0) == -2 and size(h=0) == -2 and size(tq=-1) == -2
    assert size(tk=1 << 28) == -2 and size(nb=5) == -2 and size(nb=0) == -2 and size(starts=(1, 3)) == -2
    assert size(starts=(0, 769)) == -2 and size(starts=(0, 4, 3), nb=3) == -2 and size(ns=0) == -2
    assert size(nb=300, starts=range(150)) == -2
    assert lib.esa_rel_attn_workspace_size(2, 100, 90, 4, 16, bf16, 4, None, 2, 1, ctypes.byref(n)) == -1
    s = (ctypes.c_int * 2)(0, 3)

    def fwd(q=16, table=16, tdt=0, scale=0.25, p=0.0, ws=16, nbytes=1 << 24, tq=100):
        return lib.esa_rel_attn_fwd(q, 16, 16, table, tdt, 4, s, 2, None, 16, 16, 2, tq, 90, 4, 16, bf16, scale, p, 0, 16, None,
                                    16, ws, nbytes, None)
    assert fwd(q=None) == -1 and fwd(table=None) == -1 and fwd(q=8) == -6 and fwd(tdt=3) == -5 and fwd(scale=0.0) == -2
    assert fwd(scale=float("nan")) == -2 and fwd(p=1.0) == -9 and fwd(nbytes=256) == -4 and fwd(ws=None) == -1
    assert fwd(tq=0, q=None) == 0   # no queries: nothing to do

    def bwd(g=16, dtable=16, nbytes=1 << 24, low=None):
        return lib.esa_rel_attn_bwd(g, 16, 16, 16, 16, low, 16, 16, 0, 4, s, 2, None, 16, 16, 2, 100, 90, 4, 16, bf16, 0.25, 0.0,
                                    0, 16, 16, 16, dtable, 16, nbytes, None)
    assert bwd(g=None) == -1 and bwd(dtable=None) == -1 and bwd(g=24) == -6 and bwd(low=24) == -6 and bwd(nbytes=64) == -4

"""Varlen attention with a learned bias by relative position against the formula in 64 bits: head dims, types, lengths
from none to long, segments without keys, query offsets, one- and two-sided buckets, -inf entries, dropout, gradients.

Tolerances.  bf16 calls: the inputs are exact in 64 bits; P and dS enter their products rounded to bf16 (at most half a
step, torch.finfo(torch.bfloat16).eps / 2 = 2^-8 of a value) and the result is rounded once more, so an output's error is
at most 2^-7 of its sum of absolute terms.  Norm-wise, roundings are independent and spread evenly over half a step either
way, 2^-8 / sqrt 3 in the root of their mean square at most: three of them make 2^-8, held as 6e-3.  The backward takes
D = sum(dO O) from the rounded O, one more of the same size.  The table's gradient sums dS, whose terms cancel (over all
of a row's keys to nothing), and roundings are relative to the terms: D's error e, about 2^-8 sqrt(sum of (P dP)^2) for a
row, enters a bucket's sum as e times the row's P in the bucket, at most 2^-8 of sqrt(sum dS^2) where the bucket holds
the whole row.  Its error is therefore held against the larger of its norm and the norm of the buckets' sqrt(sum dS^2),
the size such a sum has when its terms do not happen to cancel.  float32: products and sums
in 24 bits, exponentials within a few units of 2^-24 times |score| (up to about 20 here): 1e-5 norm-wise, as for the
other float32 attention kernels."""
import math

import numpy as np
import pytest
import torch

from mind_amd import _lib
from mind_amd.esa.relative import bucket_starts, relative_attention
from oracle.dropout import keep_mask, params
from tests._util import cu_from_lengths, seeded_normal

pytestmark = pytest.mark.gpu


def buckets_of(d, num_buckets, max_distance, bidirectional):
    starts = torch.tensor(bucket_starts(num_buckets, max_distance, bidirectional))
    far = d.abs() if bidirectional else (-d).clamp(min=0)
    b = torch.searchsorted(starts, far.contiguous(), right=True) - 1
    return b + (d > 0).long() * len(starts) if bidirectional else b


def oracle(q, k, v, bias, lens_q, lens_k, max_distance=128, bidirectional=True, starts=None, g=None, scale=None, keep=None):
    """(out, lse, dq, dk, dv, dbias, sqrt(sum dS^2) by bucket, what an error of D makes of dq, dk and dbias) in 64 bits on
    the CPU; keep: [H, Tq, Tk] scaled mask."""
    q, k, v, bias = (x.detach().double().cpu() for x in (q, k, v, bias))
    h, hd, nb = q.shape[1], q.shape[2], bias.shape[0]
    scale = 1 / math.sqrt(hd) if scale is None else scale
    out, dq, dk, dv = (torch.zeros_like(x) for x in (q, q, k, v))
    lse = torch.full((h, q.shape[0]), -math.inf, dtype=torch.float64)
    db, sq, qs, ks = torch.zeros_like(bias), torch.zeros_like(bias), 0, 0
    by_d = [torch.zeros_like(x) for x in (q, k, bias)]
    for s, (lq, lk) in enumerate(zip(lens_q, lens_k)):
        a, b = slice(qs, qs + lq), slice(ks, ks + lk)
        qs, ks = qs + lq, ks + lk
        if lq == 0 or lk == 0:
            continue
        d = torch.arange(lk)[None, :] - torch.arange(lq)[:, None] - (0 if starts is None else starts[s])
        bk = buckets_of(d, nb, max_distance, bidirectional)
        x = torch.einsum("ihd,jhd->hij", q[a], k[b]) * scale + bias[bk].permute(2, 0, 1)
        lse[:, a] = torch.logsumexp(x, 2)
        p = torch.exp(x - lse[:, a, None])
        p[torch.isneginf(lse[:, a])] = 0
        z = 1.0 if keep is None else keep[:, a, b]
        out[a] = torch.einsum("hij,jhd->ihd", p * z, v[b])
        if g is None:
            continue
        gx = g.detach().double().cpu()[a]
        dp = torch.einsum("ihd,jhd->hij", gx, v[b]) * z
        ds = p * (dp - (p * dp).sum(2, keepdim=True))
        dq[a] = torch.einsum("hij,jhd->ihd", ds, k[b]) * scale
        dk[b] = torch.einsum("hij,ihd->jhd", ds, q[a]) * scale
        dv[b] = torch.einsum("hij,ihd->jhd", p * z, gx)
        db.index_add_(0, bk.reshape(-1), ds.permute(1, 2, 0).reshape(-1, h))
        sq.index_add_(0, bk.reshape(-1), ds.square().permute(1, 2, 0).reshape(-1, h))
        e = p * (gx * out[a]).abs().sum(2).t()[:, :, None]   # P times D's terms
        by_d[0][a] = torch.einsum("hij,jhd->ihd", e, k[b].abs()) * scale
        by_d[1][b] = torch.einsum("hij,ihd->jhd", e, q[a].abs()) * scale
        by_d[2].index_add_(0, bk.reshape(-1), e.permute(1, 2, 0).reshape(-1, h))
    return out, lse, dq, dk, dv, db, sq.sqrt(), by_d


def case(device, dtype, h, hd, lens_q, lens_k=None, buckets=32, seed=0, table=torch.float32, extra=0):
    same = lens_k is None
    lens_k = lens_q if same else lens_k
    tq, tk = sum(lens_q) + extra, sum(lens_k) + extra
    q, k, v, g = (seeded_normal((t, h, hd), seed + i, dtype).to(device) for i, t in enumerate((tq, tk, tk, tq)))
    bias = seeded_normal((buckets, h), seed + 9, torch.float32).to(table).to(device)
    cu_q = torch.as_tensor(cu_from_lengths(lens_q)).to(device)
    cu_k = cu_q if same else torch.as_tensor(cu_from_lengths(lens_k)).to(device)
    return q, k, v, g, bias, cu_q, cu_k


def scaled_keep(p, seed, h, tq, tk):
    return torch.as_tensor(keep_mask(p, seed, h, np.arange(tq), np.arange(tk))).double() * params(p, seed)[3]


def rel_err(got, ref, more=0.0):
    got, ref = got.detach().double().cpu(), ref.double()
    assert torch.isfinite(got).all()
    return float((got - ref).norm()) / (float(ref.norm()) + more) if ref.norm() > 0 else float(got.abs().sum())


def check(device, dtype, h, hd, lens_q, lens_k=None, buckets=32, max_distance=128, bidirectional=True, starts=None, seed=0,
          table=torch.float32, extra=0, dropout=0.0, bias=None, peaked=False):
    """``peaked``: nearly all of a row's weight may lie on one key, whose dS = P (dP - D) then cancels to nothing, while
    D = sum(dO O) keeps what the rounding of O (half a step each) does to its terms.  Such an error of D reaches dq, dk
    and dbias times P, so that 2^-8 (2^-24) of ``by_d`` is allowed beside the bar."""
    q, k, v, g, b, cu_q, cu_k = case(device, dtype, h, hd, lens_q, lens_k, buckets, seed, table, extra)
    if bias is not None:
        b = bias(b)
    q0 = None if starts is None else torch.tensor(starts, dtype=torch.int32, device=device)
    leaves = [x.requires_grad_(True) for x in (q, k, v, b)]
    out, lse = relative_attention(*leaves, cu_q, cu_k, max_distance=max_distance, bidirectional=bidirectional, q_start=q0,
                                  return_lse=True, dropout_p=dropout, dropout_seed=77)
    grads = torch.autograd.grad(out, leaves, g)
    keep = None
    if dropout:
        keep = scaled_keep(dropout, 77, h, q.shape[0], k.shape[0])
    ref = oracle(q, k, v, b, lens_q, lens_k or lens_q, max_distance, bidirectional, starts, g, keep=keep)
    bar = 1e-5 if dtype == torch.float32 else 6e-3
    assert grads[3].dtype == table
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    allow = [half * float(x.norm()) / bar if peaked else 0.0 for x in ref[7]]
    errs = [rel_err(x, r, s) for x, r, s in zip((out, *grads), (ref[0], *ref[2:5]), (0.0, *allow[:2], 0.0))]
    size = max(float(ref[5].norm()), float(ref[6].norm())) + allow[2]
    errs.append(float((grads[3].detach().double().cpu() - ref[5]).norm()) / size if size else float(grads[3].abs().max()))
    assert all(e <= bar for e in errs[:4]), errs
    assert errs[4] <= (max(bar, 4e-3) if table == torch.bfloat16 else bar), errs
    assert torch.isfinite(grads[3]).all()
    dead = torch.isneginf(ref[1])
    assert torch.equal(torch.isneginf(lse.cpu()), dead)
    # the lse of a bf16 call is of exact products too; its row sum adds probabilities rounded to bf16, each off by at
    # most 2^-8 of itself: the logarithm by at most that and a little
    off = (lse.cpu().double() - ref[1])[~dead].abs()
    assert not off.numel() or float(off.max()) <= (2.0 ** -7 if dtype == torch.bfloat16 else 2e-5)
    return q, k, v, b, out, grads


LENGTHS = ([1], [2, 1, 31], [33, 0, 64, 65], [127, 128, 129], [1, 300, 17], [700])


@pytest.mark.parametrize("hd", [16, 24, 32, 64])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens", LENGTHS, ids=str)
def test_self_attention(device, dtype, hd, lens):
    check(device, dtype, 3, hd, lens)


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 16), (torch.bfloat16, 64), (torch.float32, 16), (torch.float32, 64)])
@pytest.mark.parametrize("buckets,distance,two", [(32, 128, False), (4, 2, True), (8, 20, True), (2, 900, False),
                                                  (64, 512, True), (256, 768, True), (128, 700, False), (12, 7, True)])
def test_buckets(device, dtype, hd, buckets, distance, two):
    check(device, dtype, 2, hd, [450, 5, 901], buckets=buckets, max_distance=distance, bidirectional=two, seed=3)


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 16), (torch.bfloat16, 32), (torch.float32, 16), (torch.float32, 64)])
@pytest.mark.parametrize("lens_q,lens_k,starts", [
    ([1, 1, 1], [500, 1, 77], [499, 0, 76]), ([3, 0, 40], [200, 30, 0], None), ([130, 5], [70, 300], [-40, 295]),
    ([64, 64], [64, 64], [2 ** 31 - 1, -2 ** 31]), ([0, 0], [5, 40], None), ([33], [257], [1000])], ids=str)
def test_query_chunks(device, dtype, hd, lens_q, lens_k, starts):
    check(device, dtype, 2, hd, lens_q, lens_k, starts=starts, seed=5)


@pytest.mark.parametrize("hd", [16, 24, 32, 64])
@pytest.mark.parametrize("lens_q,lens_k", [
    ([1], [5000]), ([1], [512]), ([3, 1, 2], [4097, 12, 900]), ([32, 33, 1], [1500, 700, 2000]), ([0, 5, 0, 1], [900, 1800, 0, 1111]),
    ([2, 7], [0, 3000]), ([70, 1, 1], [2000, 1, 33])], ids=str)
def test_few_queries_over_many_keys(device, hd, lens_q, lens_k):
    """The forward whose keys are cut into groups (bf16, at most 32 queries a segment on average, 512 keys and more)."""
    check(device, torch.bfloat16, 3, hd, lens_q, lens_k, starts=[k - q for q, k in zip(lens_q, lens_k)], seed=51, extra=2)
    check(device, torch.bfloat16, 2, hd, lens_q, lens_k, dropout=0.3, seed=52, bias=lambda b: b * 30,
          peaked=True)


def test_few_queries_masked_and_not_finite(device):
    """A row whose every key a table of -inf leaves out, keys of infinite score beside it, a neighbour full of NaN."""
    lens_q, lens_k = [2, 1, 1], [1300, 800, 700]
    q, k, v, g, b, cu_q, cu_k = case(device, torch.bfloat16, 2, 32, lens_q, lens_k, seed=53)
    b[:, 1] = -math.inf
    out, lse = relative_attention(q, k, v, b, cu_q, cu_k, return_lse=True)
    ref = oracle(q, k, v, b, lens_q, lens_k)
    assert not out[:, 1].any() and bool(torch.isneginf(lse[1]).all()) and rel_err(out[:, 0], ref[0][:, 0]) <= 6e-3
    bad_k, bad_v = k.clone(), v.clone()
    bad_k[1300:2100], bad_v[1300:2100] = math.nan, math.inf
    got = relative_attention(q, bad_k, bad_v, b, cu_q, cu_k)
    assert rel_err(got[:2, 0], ref[0][:2, 0]) <= 6e-3 and rel_err(got[3:, 0], ref[0][3:, 0]) <= 6e-3
    assert bool(torch.isnan(got[2, 0]).all())


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 16), (torch.bfloat16, 24), (torch.float32, 32)])
def test_dropout(device, dtype, hd):
    check(device, dtype, 2, hd, [33, 150, 1, 200], dropout=0.25, seed=7)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_bf16_table_and_tokens_in_no_segment(device, dtype):
    q, k, v, b, out, grads = check(device, dtype, 4, 16, [50, 200], table=torch.bfloat16, extra=37, seed=11)
    assert not out[250:].any() and not any(x[250:].any() for x in grads[:3])


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 16), (torch.float32, 16), (torch.bfloat16, 64)])
def test_masking_entries(device, dtype, hd):
    """-inf entries leave their pairs out, also where that leaves a row empty; entries of the type's lowest value leave a
    row of nothing else its plain softmax; a large spread takes the running maximum."""
    lens = [300, 40]

    def ahead(b):   # keys after the query left out, and in head 1 everything
        b = b.clone()
        b[16:] = -math.inf
        b[:, 1] = -math.inf
        return b

    def lowest(b):
        b = b.clone()
        b[:, 0] = torch.finfo(torch.float32).min
        return b

    def wide(b):
        return b * 40
    check(device, dtype, 3, hd, lens, bias=ahead, seed=13)
    check(device, dtype, 3, hd, lens, bias=wide, seed=15)
    q, k, v, g, b, cu, _ = case(device, dtype, 3, hd, lens, seed=17)
    got = relative_attention(q, k, v, lowest(b), cu, cu)
    plain = b.clone()
    plain[:, 0] = 0
    ref = oracle(q, k, v, plain, lens, lens)[0]
    # |bias| log2(e) is 14,427, one unit of whose last place is 2^-10: the exponents are off by at most that much
    assert rel_err(got, ref) <= 6e-3


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 16), (torch.bfloat16, 32), (torch.float32, 16)])
def test_other_segments_values_do_not_leak(device, dtype, hd):
    """A graph with infinities and NaN leaves its neighbours' outputs and gradients as they are: the same bits in float32;
    in bf16 the forward's reference point (fixed or running maximum) goes by key norms of 32-token tiles, which may hold
    a neighbour's, so both results are within the bar of the formula, and of each other within twice that."""
    lens = [45, 70, 33]
    q, k, v, g, b, cu, _ = case(device, dtype, 2, hd, lens, seed=19)

    def run(q, k, v, g):
        leaves = [x.detach().clone().requires_grad_(True) for x in (q, k, v)]
        out = relative_attention(*leaves, b, cu, cu)
        return (out, *torch.autograd.grad(out, leaves, g))
    good = run(q, k, v, g)
    bad = [x.clone() for x in (q, k, v, g)]
    for x, bad_value in zip(bad, (math.nan, math.inf, math.nan, -math.inf)):
        x[45:115] = bad_value
    for x, y in zip(good, run(*bad)):
        for s in (slice(0, 45), slice(115, None)):
            assert torch.equal(x[s], y[s]) if dtype == torch.float32 else rel_err(y[s], x[s].detach().cpu()) <= 1.2e-2


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 16), (torch.float32, 32)])
def test_gradients_against_differences(device, dtype, hd):
    """The table's and v's gradients against central differences of the 64-bit formula."""
    lens = [60, 5]
    q, k, v, g, b, cu, _ = case(device, dtype, 2, hd, lens, seed=23)
    vv, bb = v.detach().requires_grad_(True), b.detach().requires_grad_(True)
    out = relative_attention(q, k, vv, bb, cu, cu)
    dv, db = torch.autograd.grad(out, (vv, bb), g)
    gen, eps = torch.Generator().manual_seed(5), 1e-4
    tb, tv = torch.randn(b.shape, generator=gen).double(), torch.randn(v.shape, generator=gen).double()

    def f(e, f_):
        o = oracle(q, k, v.cpu().double() + f_ * tv, b.cpu().double() + e * tb, lens, lens)[0]
        return float((o * g.cpu().double()).sum())
    bar = 6e-3 if dtype == torch.bfloat16 else 2e-5   # a gradient off by bar * |gradient| moves its product with t by this
    for grad, t, diff in ((db, tb, f(eps, 0) - f(-eps, 0)), (dv, tv, f(0, eps) - f(0, -eps))):
        diff /= 2 * eps
        assert abs(float((grad.cpu().double() * t).sum()) - diff) <= bar * float(grad.double().norm().cpu() * t.norm())


def test_same_bits_twice_and_on_another_stream(device):
    q, k, v, g, b, cu, _ = case(device, torch.bfloat16, 8, 16, [700, 33, 512], seed=29)

    def run():
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v, b)]
        out = relative_attention(*leaves, cu, cu)
        return (out, *torch.autograd.grad(out, leaves, g))
    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(first, second))


def test_captured_and_replayed(device):
    """Forward and backward in one graph, replayed with other inputs between eager calls."""
    q, k, v, g, b, cu, _ = case(device, torch.bfloat16, 4, 16, [200, 77], seed=31)

    def step():
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v, b)]
        out = relative_attention(*leaves, cu, cu)
        return (out, *torch.autograd.grad(out, leaves, g))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (1, 2, 3):
        for x in (q, k, v, g, b):
            x.copy_(seeded_normal(tuple(x.shape), 100 * seed + x.shape[0], torch.float32))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(held, step()))


def test_longest_line_and_many_buckets(device):
    """The largest reach and the largest table, whose sums need most of a CU's LDS."""
    check(device, torch.float32, 1, 64, [1800], buckets=256, max_distance=768, seed=37)
    check(device, torch.bfloat16, 2, 64, [1800, 3], buckets=256, max_distance=768, seed=37)


def test_larger_than_one_group(device):
    check(device, torch.bfloat16, 16, 16, [900, 1500, 64, 3], seed=41)
    check(device, torch.float32, 8, 16, [340] * 5, seed=43)


def test_no_tokens(device):
    for lens_q, lens_k in (([0], [0]), ([0], [9]), ([9], [0])):
        check(device, torch.bfloat16, 2, 16, lens_q, lens_k)
        check(device, torch.float32, 2, 16, lens_q, lens_k)


def test_output_gradient_off_a_boundary_and_strided(device):
    q, k, v, g, b, cu, _ = case(device, torch.bfloat16, 2, 16, [50, 20], seed=47)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v, b)]
    out = relative_attention(*leaves, cu, cu)
    want = torch.autograd.grad(out, leaves, g, retain_graph=True)
    off = torch.empty(g.numel() + 1, dtype=g.dtype, device=device)[1:].view(g.shape).copy_(g)
    turned = g.transpose(0, 1).contiguous().transpose(0, 1)
    for other in (off, turned):
        assert all(torch.equal(x, y) for x, y in zip(want, torch.autograd.grad(out, leaves, other, retain_graph=True)))


def test_refused_on_the_device(device):
    q, k, v, g, b, cu, _ = case(device, torch.bfloat16, 2, 16, [8])
    with pytest.raises(_lib.EsaError, match="ALIGN"):
        flat = torch.empty(q.numel() + 1, dtype=q.dtype, device=device)
        relative_attention(flat[1:].view(q.shape).copy_(q), k, v, b, cu, cu)
    leaf = q.detach().requires_grad_(True)
    out = relative_attention(leaf, k, v, b, cu, cu)
    (grad,) = torch.autograd.grad(out.float().square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.float().sum().backward()


@pytest.mark.parametrize("hd", [16, 24, 32, 64])
@pytest.mark.parametrize("dropout", [0.0, 0.2])
def test_many_blocks_in_single_precision(device, hd, dropout):
    """The fp32 kernels' groups of 128 tokens (more than 2,048 blocks of them; the other tests' few blocks take 64)."""
    lens = [1 + (7 * i) % 19 for i in range(290)] + [0, 260, 129]
    check(device, torch.float32, 7, hd, lens, dropout=dropout, seed=61, extra=3)


@pytest.mark.parametrize("lens_q,lens_k", [([3, 0, 40], [900, 30, 0]), ([2, 1], [700, 1500])], ids=str)
def test_split_forward_then_backward_with_rows_left_out(device, lens_q, lens_k):
    """A segment without keys and a head whose table leaves everything out, after the forward that writes neither's
    rounding residue: no gradient there, and none of the other rows is touched."""
    q, k, v, g, b, cu_q, cu_k = case(device, torch.bfloat16, 2, 16, lens_q, lens_k, seed=63, extra=2)
    b[:, 1] = -math.inf
    junk = torch.full((1 << 22,), math.nan, device=device)   # what a fresh allocation finds
    del junk
    leaves = [x.requires_grad_(True) for x in (q, k, v, b)]
    grads = torch.autograd.grad(relative_attention(*leaves, cu_q, cu_k), leaves, g)
    ref = oracle(q, k, v, b.masked_fill(torch.isinf(b), -1e4), lens_q, lens_k, g=g)   # its head 1 is not compared
    for got, want in zip(grads[:3], ref[2:5]):
        assert not got[:, 1].any() and rel_err(got[:, 0], want[:, 0]) <= 6e-3
    assert not grads[3][:, 1].any() and torch.isfinite(grads[3]).all()


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 16), (torch.bfloat16, 32), (torch.float32, 16)])
@pytest.mark.parametrize("lens_q,lens_k", [([40, 90], [40, 90]), ([2, 1], [900, 700])], ids=["whole", "few"])
def test_segments_that_begin_behind_the_first_token(device, dtype, hd, lens_q, lens_k):
    """Tokens before the first segment belong to none, as those behind the last."""
    q, k, v, g, b, cu_q, cu_k = case(device, dtype, 2, hd, lens_q, lens_k, seed=71)
    around = lambda x, n, v=math.nan: torch.cat([x.new_full((n, *x.shape[1:]), v), x, x.new_full((2, *x.shape[1:]), v)])
    junk = [torch.full((1 << 20,), math.nan, device=device) for _ in range(4)]   # what fresh allocations find
    del junk
    plain = [x.requires_grad_(True) for x in (q, k, v, b)]
    out, lse = relative_attention(*plain, cu_q, cu_k, return_lse=True)
    grads = torch.autograd.grad(out, plain, g)
    moved = [around(q.detach(), 5), around(k.detach(), 3), around(v.detach(), 3), b.detach().clone()]
    moved = [x.requires_grad_(True) for x in moved]
    out2, lse2 = relative_attention(*moved, cu_q + 5, cu_k + 3, return_lse=True)
    grads2 = torch.autograd.grad(out2, moved, around(g, 5, 1.0))
    assert torch.equal(out2[5:-2], out) and not out2[:5].any() and not out2[-2:].any()
    assert torch.equal(lse2[:, 5:-2], lse) and bool(torch.isneginf(lse2[:, :5]).all())
    for x, y, n in zip(grads2[:3], grads[:3], (5, 3, 3)):
        assert torch.equal(x[n:-2], y) and not x[:n].any() and not x[-2:].any()
    assert torch.equal(grads2[3], grads[3])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_no_keys_and_negative_views(device, dtype):
    q, k, v, g, b, cu_q, _ = case(device, dtype, 2, 32, [3, 70], seed=73)
    leaves = [x.requires_grad_(True) for x in (q, k[:0].clone(), v[:0].clone(), b)]
    out, lse = relative_attention(*leaves, cu_q, torch.zeros_like(cu_q), return_lse=True)
    grads = torch.autograd.grad(out, leaves, g)
    assert not out.any() and bool(torch.isneginf(lse).all()) and not any(x.any() for x in grads)
    with torch.no_grad():
        want = relative_attention(-q, k, v, b, cu_q, cu_q)
        assert torch.equal(relative_attention(torch._neg_view(q), k, v, b, cu_q, cu_q), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_two_graphs_in_turn_with_few_queries(device, dtype):
    """Two captured forwards over keys cut into groups (bf16; one launch in fp32), replayed in turn with new inputs and
    lengths between eager calls."""
    made = [case(device, dtype, 3, 32, lens_q, lens_k, seed=81 + i) for i, (lens_q, lens_k) in
            enumerate((([3, 1], [900, 1100]), ([2, 2, 5], [2000, 40, 700])))]
    graphs, held = [], []
    for q, k, v, _, b, cu_q, cu_k in made:
        with torch.no_grad():
            relative_attention(q, k, v, b, cu_q, cu_k)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                held.append(relative_attention(q, k, v, b, cu_q, cu_k, return_lse=True))
            graphs.append(graph)
    for seed in (1, 2, 3):
        for q, k, v, _, b, cu_q, cu_k in made:
            for x in (q, k, v, b):
                x.copy_(seeded_normal(tuple(x.shape), 100 * seed + x.shape[0], torch.float32))
            cu_q[1] += 1 if seed == 2 else 0   # the lengths are read on the device
        for graph in graphs:
            graph.replay()
        for (q, k, v, _, b, cu_q, cu_k), (out, lse) in zip(made, held):
            with torch.no_grad():
                want = relative_attention(q, k, v, b, cu_q, cu_k, return_lse=True)
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 16), (torch.bfloat16, 64), (torch.float32, 24)])
def test_two_calls_at_once(device, dtype, hd):
    made = [case(device, dtype, 4, hd, lens, seed=91 + i) for i, lens in enumerate(([300, 77, 512], [64, 700]))]

    def step(i):
        q, k, v, g, b, cu, _ = made[i]
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v, b)]
        out = relative_attention(*leaves, cu, cu)
        return (out, *torch.autograd.grad(out, leaves, g))
    want = [step(0), step(1)]
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in sides:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(sides):
            with torch.cuda.stream(s):
                got[i].append(step(i))
    for s in sides:
        torch.cuda.current_stream().wait_stream(s)
    for i in (0, 1):
        assert all(torch.equal(x, y) for run in got[i] for x, y in zip(run, want[i]))


def test_one_tensor_for_all(device):
    """q, k and v the same tensor: its gradient is the three together."""
    q, _, _, g, b, cu, _ = case(device, torch.float32, 3, 32, [70, 9], seed=95)
    x = q.clone().requires_grad_(True)
    parts = [q.clone().requires_grad_(True) for _ in range(3)]
    whole, = torch.autograd.grad(relative_attention(x, x, x, b, cu, cu), (x,), g)
    split = torch.autograd.grad(relative_attention(*parts, b, cu, cu), parts, g)
    assert float((whole - sum(split)).norm()) <= 2.0 ** -22 * sum(float(y.norm()) for y in split)


@pytest.mark.parametrize("dtype,hd", [(torch.bfloat16, 16), (torch.bfloat16, 32), (torch.float32, 16)])
def test_table_gradient_of_many_equal_segments(device, dtype, hd):
    """Segments of equal length are planned in any order; the table's gradient adds them in the tokens'."""
    q, k, v, g, b, cu, _ = case(device, dtype, 2, hd, [33] * 900 + [0, 170] * 40, seed=97)
    leaves = [x.requires_grad_(True) for x in (q, k, v, b)]
    grads = [torch.autograd.grad(relative_attention(*leaves, cu, cu), leaves, g) for _ in range(6)]
    assert all(torch.equal(x, y) for run in grads[1:] for x, y in zip(run, grads[0]))


@pytest.mark.parametrize("hd", [16, 24, 32])
@pytest.mark.parametrize("dropout", [0.0, 0.2])
def test_blocks_between_in_single_precision(device, hd, dropout):
    """The fp32 kernels' groups of 64 tokens with more blocks than the forward's halved walk takes."""
    check(device, torch.float32, 7, hd, [100] * 150, dropout=dropout, seed=67)


MANY = [1, 31, 32, 33, 64, 65] * 12 + [300, 0, 257, 512]   # with 16 heads more than 1,024 blocks


@pytest.mark.parametrize("change", [None, lambda b: b * 30, lambda b: torch.where(b > 1.0, torch.full_like(b, -math.inf), b),
                                    lambda b: b.index_fill(1, torch.tensor([3, 7], device=b.device), -math.inf)],
                         ids=["plain", "wide", "left out", "heads left out"])
def test_many_blocks_at_head_dim_16(device, change):
    """The bf16 forward of many blocks (few take the other head dims' kernel)."""
    check(device, torch.bfloat16, 16, 16, MANY, seed=101, extra=5, bias=change, peaked=change is not None)


def test_many_blocks_at_head_dim_16_of_chunks(device):
    lens_q = [max(n - 20, 0) for n in MANY]
    check(device, torch.bfloat16, 24, 16, lens_q, MANY, starts=[n - m for n, m in zip(MANY, lens_q)], seed=103)


def test_many_blocks_at_head_dim_16_beside_what_is_not_finite(device):
    q, k, v, _, b, cu, _ = case(device, torch.bfloat16, 16, 16, MANY, seed=105)
    want = relative_attention(q, k, v, b, cu, cu)
    bad = slice(int(cu[40]), int(cu[41]))
    k[bad], v[bad] = math.nan, math.inf
    got = relative_attention(q, k, v, b, cu, cu)
    rest = torch.ones(q.shape[0], dtype=torch.bool, device=device)
    rest[bad] = False
    # key norms are by 32 tokens of the whole tensor: the neighbours' softmax may take another reference point
    assert rel_err(got[rest], want[rest].double().cpu()) <= 6e-3 and bool(torch.isnan(got[bad]).all())

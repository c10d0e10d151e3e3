"""Query and key norms with the rotation of positions, against the formula in 64 bits.

Tolerances.  Arithmetic is float32 on exact inputs: a row's sum of squares, the root, two products and the rotation's two
products and sum are a dozen roundings of 2^-24 of the row's size at most, and the cosines and sines are those of an angle
exact to 2^-24 of a half turn: 2e-6 norm-wise for float32, and for bf16 the one rounding of the result on top, at most
half a step, torch.finfo(torch.bfloat16).eps / 2 = 2^-8 of each value.  The weights' gradients are float32 sums of float32 terms in short chains: 2e-6 of the sum of the
terms' sizes' root of squares, held here as 5e-6 of sqrt(sum of squares) or the gradient's norm, the larger."""
import math

import pytest
import torch

from mind_amd.esa.qk_norm import qk_norm_rotary, rotary_frequencies
from tests._util import seeded_normal

pytestmark = pytest.mark.gpu


def oracle(x, w, positions, frequencies, eps, interleaved, g=None):
    """(y, dx, dw, size of dw's sum) in 64 bits."""
    x = x.detach().double().cpu()
    w = torch.ones(x.shape[2], dtype=torch.float64) if w is None else w.detach().double().cpu()
    rms = (x.square().mean(-1, keepdim=True) + eps).sqrt()

    def turn(y, sign):
        if frequencies is None:
            return y
        f = frequencies.cpu()
        angle = sign * (positions.cpu().double()[:, None] * f)[:, None]
        r, y = 2 * f.numel(), y.clone()
        i = torch.arange(f.numel())
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
        ya, yb = y[..., a].clone(), y[..., b].clone()
        y[..., a], y[..., b] = ya * angle.cos() - yb * angle.sin(), ya * angle.sin() + yb * angle.cos()
        return y
    unit = x / rms
    if g is None:
        return turn(unit * w, 1), None, None, None
    back = turn(g.detach().double().cpu(), -1)
    gw = back * w
    dx = (gw - unit * (gw * unit).mean(-1, keepdim=True)) / rms
    return turn(unit * w, 1), dx, (back * unit).sum((0, 1)), (back * unit).square().sum((0, 1)).sqrt()


def rel(got, ref):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape and torch.isfinite(got).all()
    return float((got - ref).norm() / ref.norm().clamp(min=1e-30))


def check(device, dtype, t, hq, hk, hd, rotary=0, interleaved=False, weights=torch.float32, first=0, wide=False, seed=0,
          eps=1e-6, make=None, scale=1.0):
    make = make or (lambda t, h, i: seeded_normal((t, h, hd), seed + i, dtype).to(device))
    q, k = make(t, hq, 0).mul(scale), make(t, hk, 1).mul(scale) if hk else None
    wq, wk = ((1 + 0.3 * seeded_normal((hd,), seed + 2 + i, torch.float32)).to(weights).to(device) if weights else None
              for i in (0, 1))
    wk = wk if hk else None
    pos = freq = None
    if rotary:
        pos = (torch.arange(t, dtype=torch.int64 if wide else torch.int32, device=device) * 7) % 1013 + first
        freq = rotary_frequencies(rotary, device=device)
    leaves = [x for x in (q, k, wq, wk) if x is not None]
    for x in leaves:
        x.requires_grad_(True)
    out = qk_norm_rotary(q, k, wq, wk, pos, freq, eps, interleaved)
    outs = out if hk else (out,)
    gs = [seeded_normal(tuple(y.shape), seed + 20 + i, dtype).to(device) for i, y in enumerate(outs)]
    grads = list(torch.autograd.grad(outs, leaves, gs))
    bar = (2e-6 if dtype == torch.float32 else 2.0 ** -8 + 2e-6) + (abs(first) + 1013) * 2.0 ** -51
    dxs = [grads.pop(0) for _ in outs]
    for x, w, y, g, dx in zip((q, k), (wq, wk), outs, gs, dxs):
        ref = oracle(x, w, pos, freq, eps, interleaved, g)
        assert y.is_contiguous() and rel(y, ref[0]) <= bar and rel(dx, ref[1]) <= bar
        if w is not None:
            dw = grads.pop(0)
            size = max(float(ref[2].norm()), float(ref[3].norm()))
            err = float((dw.double().cpu() - ref[2]).norm()) / max(size, 1e-30)
            assert dw.dtype == w.dtype and err <= (5e-6 if weights == torch.float32 else 2.0 ** -8) + bar, err


@pytest.mark.parametrize("hd,rotary", [(16, 16), (16, 8), (24, 24), (24, 16), (24, 8), (32, 32), (32, 24), (64, 64), (64, 8),
                                       (64, 40), (16, 0), (24, 0), (64, 0)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_head_dims_and_rotations(device, dtype, interleaved, hd, rotary):
    check(device, dtype, 77, 3, 5, hd, rotary, interleaved)


@pytest.mark.parametrize("t,hq,hk", [(1, 1, 0), (1, 1, 1), (3, 1, 0), (2, 33, 1), (513, 16, 16), (2049, 3, 0), (4100, 8, 2),
                                     (40000, 1, 0), (1, 2048, 2048), (35000, 5, 4)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tokens_and_heads(device, dtype, t, hq, hk):
    check(device, dtype, t, hq, hk, 16, 16, seed=t)


@pytest.mark.parametrize("first,wide", [(0, True), (2 ** 31 - 2000, False), (-2 ** 31, False), (10 ** 12, True), (-77, True)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions(device, first, wide, interleaved):
    check(device, torch.float32, 300, 2, 2, 32, 32, interleaved, first=first, wide=wide)


@pytest.mark.parametrize("weights", [None, torch.bfloat16])
def test_weights(device, weights):
    check(device, torch.bfloat16, 200, 4, 4, 16, 16, weights=weights)
    check(device, torch.float32, 200, 4, 4, 24, 0, weights=weights)


def test_no_tokens(device):
    for dtype in (torch.float32, torch.bfloat16):
        q, k = (torch.empty(0, 4, 16, dtype=dtype, device=device, requires_grad=True) for _ in range(2))
        w = torch.ones(16, device=device, requires_grad=True)
        y, z = qk_norm_rotary(q, k, w, w, torch.empty(0, dtype=torch.int32, device=device), rotary_frequencies(16, device=device))
        dw, dq = torch.autograd.grad((y, z), (w, q), (torch.zeros_like(y), torch.zeros_like(z)))
        assert y.shape == z.shape == dq.shape == (0, 4, 16) and not dw.any()


@pytest.mark.parametrize("scale", [0.0, 1e-12, 1e12])
def test_sizes_of_rows(device, scale):
    """Rows of zeros give zeros (eps holds the root), tiny ones are held by eps, large ones by nothing."""
    if scale:
        check(device, torch.float32, 50, 2, 2, 16, 16, scale=scale)
    else:
        q = torch.zeros(9, 2, 16, device=device, requires_grad=True)
        y = qk_norm_rotary(q, None, positions=torch.arange(9, device=device), frequencies=rotary_frequencies(16, device=device))
        (dq,) = torch.autograd.grad(y, q, torch.ones_like(y))
        assert not y.any() and torch.isfinite(dq).all()


def test_a_row_that_is_not_finite_stays_alone(device):
    for hd, h in ((24, 3), (16, 3), (64, 2)):
        x = seeded_normal((30, h, hd), 3, torch.float32).to(device)
        good = qk_norm_rotary(x)
        x[7, 1, 5] = math.nan
        x[8, 0, 2] = math.inf
        bad = qk_norm_rotary(x)
        keep = torch.ones(30, h, dtype=torch.bool, device=device)
        keep[7, 1] = keep[8, 0] = False
        assert torch.equal(good[keep], bad[keep]) and torch.isnan(bad[7, 1]).all()


def test_views(device):
    """Rows of one projection's output, read where they are, and layouts that are copied first, give the same bits."""
    for dtype in (torch.float32, torch.bfloat16):
        qkv = seeded_normal((120, 3, 4, 32), 5, dtype).to(device)
        w = torch.ones(32, device=device)
        pos, freq = torch.arange(120, device=device), rotary_frequencies(32, device=device)
        want = qk_norm_rotary(qkv[:, 0].contiguous(), qkv[:, 1].contiguous(), w, w, pos, freq)
        off = torch.empty(120 * 4 * 32 + 1, dtype=dtype, device=device)[1:].view(120, 4, 32).copy_(qkv[:, 0])
        by_head = qkv[:, 0].transpose(0, 1).contiguous().transpose(0, 1)
        strided = torch.empty(120, 4, 64, dtype=dtype, device=device)[..., ::2].copy_(qkv[:, 0])
        for q in (qkv[:, 0], off, by_head, strided):
            got = qk_norm_rotary(q, qkv[:, 1], w, w, pos, freq)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        one = qkv[:1, 0].expand(120, 4, 32)   # every token the same row
        leaf = qkv[:1, 0].clone().requires_grad_(True)
        y = qk_norm_rotary(leaf.expand(120, 4, 32), None, w, None, pos, freq)
        assert torch.equal(y, qk_norm_rotary(one.contiguous(), None, w, None, pos, freq))
        (d,) = torch.autograd.grad(y.float().sum(), leaf)
        assert d.shape == leaf.shape and torch.isfinite(d).all()


def test_gradients_against_differences(device):
    q, g = (seeded_normal((6, 2, 24), i, torch.float32).to(device) for i in (1, 2))
    w = (1 + 0.2 * seeded_normal((24,), 3, torch.float32)).to(device)
    pos, freq = torch.arange(6, device=device) * 1000, rotary_frequencies(16, device=device)
    leaf, wl = q.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dq, dw = torch.autograd.grad(qk_norm_rotary(leaf, None, wl, None, pos, freq), (leaf, wl), g)
    gen, e = torch.Generator().manual_seed(9), 1e-5
    tq, tw = torch.randn(q.shape, generator=gen).double(), torch.randn(24, generator=gen).double()

    def f(a, b):
        return float((oracle(q.cpu().double() + a * tq, w.cpu().double() + b * tw, pos, freq, 1e-6, False)[0] * g.cpu().double()).sum())
    for grad, t, diff in ((dq, tq, f(e, 0) - f(-e, 0)), (dw, tw, f(0, e) - f(0, -e))):
        assert abs(float((grad.cpu().double() * t).sum()) - diff / (2 * e)) <= 1e-5 * float(grad.double().norm().cpu() * t.norm())


def test_same_bits_on_a_stream_and_replayed(device):
    x = seeded_normal((700, 3, 4, 16), 11, torch.bfloat16).to(device)
    w = torch.ones(16, device=device)
    pos, freq = torch.arange(700, device=device), rotary_frequencies(16, device=device)
    g = seeded_normal((700, 4, 16), 12, torch.bfloat16).to(device)

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (x[:, 0], x[:, 1], w, w.clone())]
        outs = qk_norm_rotary(*leaves, pos, freq)
        return (*outs, *torch.autograd.grad(outs, leaves, (g, g)))
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (1, 2, 3):
        x.copy_(seeded_normal(tuple(x.shape), seed, torch.bfloat16))
        pos.add_(1000)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step()))


def test_differentiated_again_is_refused(device):
    leaf = seeded_normal((5, 2, 16), 1, torch.float32).to(device).requires_grad_(True)
    (d,) = torch.autograd.grad(qk_norm_rotary(leaf).square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        d.sum().backward()

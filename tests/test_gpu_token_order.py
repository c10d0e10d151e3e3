"""An ESA whose layers know their tokens' order: query/key norms with rotation, attention with a bias by relative
position and gradient clipping together, as a training step and a served forward use them.

The oracle restates the stack in 64 bits on the CPU from the module's own state dict, with its gradients from autograd
and, along one direction, from differences.  fp32: every operator's results are within 1e-5 of their norm (their own
tests); a stack of four blocks with residuals adds up less than one such error per operator, fewer than 16 in a chain,
so outputs and gradients are held to 16e-5 of their norm.  Under autocast each block's input, weights, projections,
normed queries and keys, probabilities, attention output and epilogue are rounded to bf16, 2^-9 rms at most each
(half a step is at most 2^-8, its rms over a binade less than half of that): about 8 in a block, 4 blocks, forward and
backward, added as independent errors sqrt(64) 2^-9 = 1.6e-2 of a norm; held to 4 times that, 6e-2.
"""
import copy
import math
import threading

import numpy as np
import pytest
import torch
from torch.nn import functional as F
from torch.utils.checkpoint import checkpoint

from mind_amd import generators
from mind_amd.esa import masked_layers as ML
from mind_amd.esa.gradients import clip_grad_norm_
from mind_amd.esa.graphs import GraphedForward
from mind_amd.esa.packing import EdgeAdjacency
from mind_amd.esa.qk_norm import qk_norm_rotary, rotary_frequencies
from mind_amd.esa.relative import relative_attention
from mind_amd.esa.token_order import TokenOrder
from tests.test_gpu_relative import buckets_of

pytestmark = pytest.mark.gpu

D, H = 64, 4
ORDER = TokenOrder(rotary_dim=8, num_buckets=8, max_distance=20)


def build(device, order=ORDER, layers=("S", "M", "S", "P"), dropout=0.0, seed=0):
    torch.manual_seed(seed)
    m = ML.ESA(4, 16, [D] * len(layers), [H] * len(layers), list(layers), xformers_or_torch_attn="hip", token_order=order,
               sab_dropout=dropout)
    with torch.no_grad():
        for name, p in m.named_parameters():
            if name.endswith(("order.bias", "order.q_weight", "order.k_weight")):
                p.add_(torch.randn(p.shape) * 0.5)
    return m.to(device)


def batch(device, num_graphs=6, seed=0):
    gb, _ = generators.small_molecules(seed=seed, num_graphs=num_graphs)
    n = int(gb.edge_counts.max())
    tokens = EdgeAdjacency.from_edge_index(torch.as_tensor(gb.edge_index).to(device), torch.as_tensor(gb.batch).to(device),
                                           gb.num_graphs, n)
    x = torch.randn(tokens.num_tokens, D, generator=torch.Generator().manual_seed(seed + 1))
    g = torch.randn(gb.num_graphs, 16, generator=torch.Generator().manual_seed(seed + 2))
    return gb, tokens, x, g


def mish(x):
    return x * torch.tanh(F.softplus(x))


def oracle_block(p, x, allowed, lens, order):
    """One encoder block: p(name) its parameters, allowed [T, T] pairs."""
    t, hd = x.shape[0], D // H
    x = F.layer_norm(x, (D,), p("norm.ln.weight"), p("norm.ln.bias"))
    q, k, v = (F.linear(x, p(f"sab.mab.fc_{n}.weight"), p(f"sab.mab.fc_{n}.bias")).view(t, H, hd) for n in "qkv")
    at = torch.cat([torch.arange(n) for n in lens])
    r = hd if order.rotary_dim is None else order.rotary_dim
    angle = at.double()[:, None] * order.rotary_base ** (-torch.arange(0, r, 2, dtype=torch.float64) / max(r, 1))
    c, s = (y[:, None, :] for y in (angle.cos(), angle.sin()))

    def turn(y, w):
        y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
        a, b = y[..., :r // 2], y[..., r // 2:r]
        return torch.cat([a * c - b * s, b * c + a * s, y[..., r:]], -1)
    q, k = turn(q, p("sab.mab.order.q_weight")), turn(k, p("sab.mab.order.k_weight"))
    a = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(hd)
    table = p("sab.mab.order.bias")
    if table is not None:
        bk = buckets_of(at[None, :] - at[:, None], order.num_buckets, order.max_distance, order.bidirectional)
        a = a + table[bk].permute(2, 0, 1)
    alive = allowed.any(1)[None, :, None]   # a query with no admissible key gets 0
    w = torch.softmax(torch.where(alive, a.masked_fill(~allowed, -math.inf), torch.zeros_like(a)), -1) * alive
    o = torch.einsum("hij,jhd->ihd", w, v).reshape(t, D)
    return x + o + mish(F.linear(o, p("sab.mab.fc_o.weight"), p("sab.mab.fc_o.bias")))


def oracle(params, x, gb, order, layers):
    """(graph embeddings, token embeddings) from a dict of 64-bit parameters."""
    graph = torch.as_tensor(np.repeat(np.arange(gb.num_graphs), gb.edge_counts))
    same = graph[:, None] == graph[None, :]
    s, d = torch.as_tensor(gb.edge_index)
    share = (s[:, None] == s) | (s[:, None] == d) | (d[:, None] == s) | (d[:, None] == d)
    share = share & same & ~torch.eye(len(s), dtype=torch.bool)
    h = x
    for i, kind in enumerate(layers[:-1]):
        h = oracle_block(lambda n, i=i: params.get(f"encoder.{i}.{n}"), h, share if kind == "M" else same,
                         gb.edge_counts, order)
    enc = h + x
    p = lambda n: params[f"decoder.0.{n}"]
    y = F.layer_norm(enc, (D,), p("norm.ln.weight"), p("norm.ln.bias"))
    hd, seeds = D // H, p("pma.S")[0]
    q = F.linear(seeds, p("pma.mab.fc_q.weight"), p("pma.mab.fc_q.bias")).view(-1, H, hd)
    k, v = (F.linear(y, p(f"pma.mab.fc_{n}.weight"), p(f"pma.mab.fc_{n}.bias")).view(-1, H, hd) for n in "kv")
    a = torch.einsum("ihd,jhd->hij", q, k)[None] / math.sqrt(hd)
    member = (graph[None, :] == torch.arange(gb.num_graphs)[:, None])[:, None, None, :]
    o = torch.einsum("bhij,jhd->bihd", torch.softmax(a.masked_fill(~member, -math.inf), -1), v).reshape(gb.num_graphs, -1, D)
    o = o + mish(F.linear(o, p("pma.mab.fc_o.weight"), p("pma.mab.fc_o.bias")))
    return mish(F.linear(o.mean(1), params["decoder_linear.weight"], params["decoder_linear.bias"])), enc


def off(got, ref):
    got = got.detach().double().cpu()
    assert torch.isfinite(got).all()
    return float((got - ref).norm() / ref.norm())


@pytest.mark.parametrize("order", [ORDER, TokenOrder(num_buckets=0), TokenOrder(rotary_dim=0, num_buckets=5, bidirectional=False)],
                         ids=["both", "rotation", "bias"])
def test_training_step(device, order):
    layers = ("S", "M", "S", "P")
    m = build(device, order, layers)
    gb, tokens, x, g = batch(device)
    xd = x.to(device).requires_grad_()
    out, enc = m.forward_packed(xd, tokens)
    (out * g.to(device)).sum().backward()
    params = {k: v.detach().double().cpu().requires_grad_() for k, v in m.state_dict().items()}
    x64 = x.double().requires_grad_()
    ref, ref_enc = oracle(params, x64, gb, order, layers)
    loss = (ref * g.double()).sum()
    loss.backward()
    assert off(out, ref.detach()) <= 16e-5 and off(enc, ref_enc.detach()) <= 16e-5 and off(xd.grad, x64.grad) <= 16e-5
    grads = {n: p.grad.clone() for n, p in m.named_parameters() if p.grad is not None}   # no MLPs: their norms have none
    whole = math.sqrt(sum(float(params[n].grad.square().sum()) for n in grads))
    for n, got in grads.items():   # small gradients (a key bias's is 0 but for rounding) against the whole
        d = float((got.double().cpu() - params[n].grad).norm())
        assert d <= 16e-5 * float(params[n].grad.norm()) + 1e-6 * whole, n
    # a difference along one direction of the order's own parameters: third-order error 1e-10, cancellation 1e-16 / 1e-5
    own = [n for n in grads if ".order." in n]
    u = {n: torch.randn(params[n].shape, dtype=torch.float64, generator=torch.Generator().manual_seed(i)) for i, n in enumerate(own)}
    with torch.no_grad():
        side = [float((oracle({n: v + e * u[n] if n in u else v for n, v in params.items()}, x.double(), gb, order, layers)[0]
                       * g.double()).sum()) for e in (1e-5, -1e-5)]
    along = sum(float((grads[n].double().cpu() * u[n]).sum()) for n in own)
    size = math.sqrt(sum(float(params[n].grad.square().sum()) for n in own) * sum(float(y.square().sum()) for y in u.values()))
    assert abs((side[0] - side[1]) / 2e-5 - along) <= 17e-5 * size
    # the step's clipping
    norm = clip_grad_norm_(m.parameters(), whole / 3)
    assert abs(float(norm) - whole) <= 17e-5 * whole
    for n, p in ((n, p) for n, p in m.named_parameters() if n in grads):
        assert float((p.grad.double().cpu() - params[n].grad * (1 / 3)).norm()) <= (
            34e-5 * float(params[n].grad.norm()) + 1e-6 * whole), n


def test_training_step_under_autocast(device):
    m = build(device)
    gb, tokens, x, g = batch(device, seed=3)
    with torch.autocast("cuda", torch.bfloat16):
        out, _ = m.forward_packed(x.to(device), tokens)
        loss = (out.float() * g.to(device)).sum()
    loss.backward()
    params = {k: v.detach().double().cpu().requires_grad_() for k, v in m.state_dict().items()}
    ref, _ = oracle(params, x.double(), gb, ORDER, ("S", "M", "S", "P"))
    (ref * g.double()).sum().backward()
    assert off(out, ref.detach()) <= 6e-2
    got = torch.cat([p.grad.double().cpu().reshape(-1) for p in m.parameters() if p.grad is not None])
    want = torch.cat([params[n].grad.reshape(-1) for n, p in m.named_parameters() if p.grad is not None])
    assert off(got, want) <= 6e-2
    norm = clip_grad_norm_(m.parameters(), 1.0)
    assert abs(float(norm) - float(got.norm())) <= 1e-6 * float(got.norm())


def test_padded_entry_and_dropout(device):
    """ESA.forward on padded input is forward_packed's; dropout draws one seed a layer and repeats with it."""
    m = build(device, dropout=0.2).eval()
    gb, tokens, x, _ = batch(device, seed=5)
    out, enc = m.forward_packed(x.to(device), tokens)
    padded = tokens.pad(x.to(device))
    out2, enc2 = m(padded, torch.as_tensor(gb.edge_index).to(device), torch.as_tensor(gb.batch).to(device), tokens.max_items)
    assert torch.equal(out, out2) and torch.equal(tokens.unpad(enc2), enc)
    blk = m.encoder[0]
    y = blk((padded, None, None, tokens.max_items, tokens))[0]
    assert torch.equal(tokens.unpad(y), ML._sab_forward_packed(blk, x.to(device), tokens))
    m.train()
    torch.manual_seed(9)
    a = m.forward_packed(x.to(device), tokens)[0]
    torch.manual_seed(9)
    b = m.forward_packed(x.to(device), tokens)[0]
    assert torch.equal(a, b) and not torch.equal(a, out)


def test_served_from_a_graph(device):
    m = build(device).to(torch.bfloat16).eval()
    gb, tokens, x, _ = batch(device, seed=6)
    x = x.to(device, torch.bfloat16)
    served = GraphedForward(lambda y: m.forward_packed(y, tokens)[0], x)
    for i in range(3):
        y = torch.randn(x.shape, device=device).to(torch.bfloat16)
        with torch.no_grad():
            eager = m.forward_packed(y, tokens)[0]
        assert torch.equal(served(y).clone(), eager)


def test_without_an_order_nothing_changes(device):
    torch.manual_seed(1)
    a = ML.ESA(4, 16, [D] * 3, [H] * 3, ["S", "M", "P"], xformers_or_torch_attn="hip").to(device)
    assert not any(".order." in n for n in a.state_dict())
    b = build(device, ORDER, ("S", "M", "P"))
    own = [n for n in b.state_dict() if ".order." in n]
    assert own == ["encoder.0.sab.mab.order.q_weight", "encoder.0.sab.mab.order.k_weight", "encoder.0.sab.mab.order.bias",
                   "encoder.1.sab.mab.order.q_weight", "encoder.1.sab.mab.order.k_weight"]
    c = copy.deepcopy(b)
    _, tokens, x, _ = batch(device)
    assert torch.equal(b.forward_packed(x.to(device), tokens)[0], c.forward_packed(x.to(device), tokens)[0])
    # the order matters: the same graph's tokens in reverse are another input
    flat = ML.ESA(4, 16, [D] * 2, [H] * 2, ["S", "P"], xformers_or_torch_attn="hip", token_order=ORDER).to(device)
    with torch.no_grad():
        flat.encoder[0].sab.mab.order.bias[1:4] += 1.0
    one = EdgeAdjacency.from_edge_index(torch.arange(40, device=device).reshape(2, 20), torch.zeros(40, dtype=torch.long, device=device), 1, 20)
    z = torch.randn(20, D, device=device)
    with torch.no_grad():
        e, r = flat.forward_packed(z, one)[1], flat.forward_packed(z.flip(0).contiguous(), one)[1].flip(0)
    assert float((e - r).norm() / e.norm()) > 1e-3


def _both(device, dtype=torch.float32):
    """A chain of both operators: (leaves, function of them)."""
    gen = torch.Generator(device).manual_seed(11)
    q, k, v = (torch.randn(120, 3, 16, device=device, dtype=dtype, generator=gen) for _ in range(3))
    w, bias = torch.rand(16, device=device, generator=gen) + 0.5, torch.randn(8, 3, device=device, generator=gen)
    cu = torch.tensor([0, 50, 120], dtype=torch.int32, device=device)
    at, f = torch.arange(120, device=device), rotary_frequencies(8, device=device)
    leaves = [x.requires_grad_(True) for x in (q, k, v, w, bias)]

    def run(q, k, v, w, bias):
        a, b = qk_norm_rotary(q, k, w, w, positions=at, frequencies=f)
        return relative_attention(a, b, v, bias, cu, cu, max_distance=20)
    return leaves, run


def test_as_any_recorded_operation(device):
    """Graphs kept and used again, checkpoints, saved tensors on the host, leaves without gradients, outputs left out."""
    leaves, run = _both(device)
    out = run(*leaves)
    g = torch.randn_like(out)
    want = torch.autograd.grad(out, leaves, g, retain_graph=True)
    same = lambda got: all(torch.equal(x, y) for x, y in zip(got, want))
    assert same(torch.autograd.grad(out, leaves, g))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out, leaves, g)   # the graph is gone
    assert same(torch.autograd.grad(checkpoint(run, *leaves, use_reentrant=False), leaves, g))
    with torch.autograd.graph.save_on_cpu():
        out = run(*leaves)
    assert same(torch.autograd.grad(out, leaves, g))
    for i, leaf in enumerate(leaves):   # one at a time
        rest = [x if j == i else x.detach() for j, x in enumerate(leaves)]
        assert torch.equal(torch.autograd.grad(run(*rest), leaf, g)[0], want[i])
    with torch.no_grad():
        assert not run(*leaves).requires_grad
    assert not run(*[x.detach() for x in leaves]).requires_grad
    a, _ = qk_norm_rotary(leaves[0], leaves[1])
    assert not torch.autograd.grad(a.sum(), leaves[1])[0].any()   # the other output's gradient counts as zeros
    out = run(*leaves)
    with torch.no_grad():
        leaves[2].add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, leaves, g)


def test_differentiated_again_is_refused(device):
    leaves, run = _both(device)
    first = torch.autograd.grad(run(*leaves).sum(), leaves, create_graph=True)
    assert all(x.requires_grad for x in first)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first[0].sum(), leaves[0])


def test_backward_in_other_threads_and_on_a_stream(device):
    leaves, run = _both(device, torch.bfloat16)
    out = run(*leaves)
    g = torch.ones_like(out)
    want = torch.autograd.grad(out, leaves, g)
    got = [None] * 4

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            got[i] = torch.autograd.grad(run(*leaves), leaves, g)
            torch.cuda.current_stream().synchronize()
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(x, y) for run_ in got for x, y in zip(run_, want))


def test_out_of_memory_is_torchs(device):
    q = torch.zeros(1 << 20, 8, 32, device=device)   # 1 GiB; its outputs as much again
    cu = torch.tensor([0, 10], dtype=torch.int32, device=device)
    bias = torch.zeros(8, 8, device=device)
    torch.cuda.empty_cache()
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_allocated() + (256 << 20)) / torch.cuda.mem_get_info()[1])
    try:
        with pytest.raises(torch.cuda.OutOfMemoryError):
            relative_attention(q, q, q, bias, cu, cu, max_distance=20)
        with pytest.raises(torch.cuda.OutOfMemoryError):
            qk_norm_rotary(q)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert not relative_attention(q[:64], q[:64], q[:64], bias, cu, cu, max_distance=20).any()

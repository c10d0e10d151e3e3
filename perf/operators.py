"""Operators for models over ordered tokens, as cases: attention with a learned bias by relative position, norms of
queries and keys with the rotation of positions, and the global gradient norm with clipping.

``run`` computes a case in elementary torch operations (``own`` false) or through this framework's operators (``own``
true).  Three kinds:

  relative  varlen attention over packed graphs whose scores get ``bias[bucket(key position - query position), head]``;
            ``rows`` > 0 takes the last ``rows`` tokens of every graph as the queries (a chunk whose positions begin
            at ``q_start``), else every token; ``train`` adds the gradients of q, k, v and the bias
  qk_norm   the RMS norm of every query and key head row, its weights, and the rotation of its first ``rotary``
            dimensions by the token's position, on rows taken from one [T, 3, H, hd] projection
  clip      the norm over all gradients of a model and their clipped values; ``ragged`` gradients lie one behind
            another in a flat buffer, so that most begin off a 16-byte boundary

Which graphs or tensor sizes a case has is the case's; order, features and weights come from the seed.
"""
from __future__ import annotations

import functools
import math

import numpy as np
import torch

from mind_amd import generators

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
DEV = "cuda"
EPS = 1e-6


def _relative(graphs, size, heads, head_dim, dtype, train, buckets=32, distance=128, rows=0, two_sided=True, pick=0):
    return {"kind": "relative", "graphs": graphs, "size": size, "pick": pick, "heads": heads, "head_dim": head_dim,
            "dtype": dtype, "train": train, "buckets": buckets, "distance": distance, "rows": rows,
            "two_sided": two_sided}


def _qk_norm(tokens, heads, head_dim, dtype, train, rotary, interleaved=False, first=0):
    return {"kind": "qk_norm", "tokens": tokens, "heads": heads, "head_dim": head_dim, "dtype": dtype, "train": train,
            "rotary": rotary, "interleaved": interleaved, "first": first}


def _clip(dim, mlp, layers, dtype, out, ragged=False):
    return {"kind": "clip", "dim": dim, "mlp": mlp, "layers": layers, "dtype": dtype, "out": out, "ragged": ragged}


def listed():
    return [
        # A property server's small request, eight molecules through an fp32 layer: latency.
        dict(_relative("molecules", 8, 8, 16, "fp32", False), name="relative-molecules-infer-fp32"),
        # The fp32 model's layer on an ordinary training batch.
        dict(_relative("molecules", 64, 8, 16, "fp32", True, pick=1), name="relative-molecules-train-fp32"),
        # The pretraining model's unmasked layer (16 heads of 16) on protein-like chains.
        dict(_relative("proteins", 32, 16, 16, "bf16", True), name="relative-proteins-16x16-bf16"),
        # The wide models' layer (8 heads of 64), finer buckets that reach further along the chain.
        dict(_relative("proteins", 24, 8, 64, "bf16", True, 64, 512, pick=1), name="relative-proteins-8x64-bf16"),
        # The last tokens of every chain against the whole chain, as a service that extends its inputs asks for.
        dict(_relative("proteins", 16, 16, 32, "bf16", False, rows=3, pick=2), name="relative-last-rows-bf16"),
        # The encoder stack's layer on the largest token budget (32 heads of 16).
        dict(_relative("budget", 131072, 32, 16, "bf16", True), name="relative-budget-32x16-bf16"),
        # One graph's queries and keys in inference.
        dict(_qk_norm(1013, 16, 16, "bf16", False, 16), name="qk-norm-one-graph-infer-bf16"),
        # A training batch of the largest token budget (32 heads of 16).
        dict(_qk_norm(129850, 32, 16, "bf16", True, 16), name="qk-norm-budget-train-bf16"),
        # fp32 training with wide heads, half of the dimensions rotated in neighbouring pairs, far positions.
        dict(_qk_norm(43670, 8, 64, "fp32", True, 32, True, 1000000), name="qk-norm-8x64-train-fp32"),
        # The small-molecule model's gradients: fifty small tensors, launches and latency.
        dict(_clip(128, 256, 3, "fp32", "fp32"), name="clip-small-fp32"),
        # The encoder stack's gradients (512 wide, MLP 2048, nine blocks).
        dict(_clip(512, 2048, 9, "fp32", "fp32"), name="clip-stack-fp32"),
        # bf16 gradients of a deep model in one flat buffer, clipped into fp32 master gradients.
        dict(_clip(256, 1000, 48, "bf16", "fp32", True), name="clip-ragged-bf16-to-fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["relative", "relative", "qk_norm", "clip"])
    if kind == "relative":
        pick, train = rng.randrange(1 << 20), rng.random() < 0.7
        heads, head_dim = rng.choice([(16, 16), (8, 16), (32, 16), (8, 24), (16, 32), (8, 32), (8, 64), (5, 16)])
        buckets, distance = rng.choice([(32, 128), (32, 128), (16, 40), (64, 512), (8, 20), (32, 800)])
        rows = rng.choice([0, 0, 0, 1, 17, 200])
        two_sided = rng.random() < 0.8
        if rng.random() < 0.35:
            return _relative("molecules", _log(rng, 1, 128), heads, head_dim, "fp32", train, buckets, distance, rows,
                             two_sided, pick)
        graphs = rng.choice(["molecules", "proteins", "budget"])
        size = {"molecules": _log(rng, 1, 256), "proteins": _log(rng, 1, 32), "budget": _log(rng, 4000, 65536)}[graphs]
        return _relative(graphs, size, heads, head_dim, "bf16", train, buckets, distance, rows, two_sided, pick)
    if kind == "qk_norm":
        heads, head_dim = rng.choice([(16, 16), (8, 16), (32, 16), (8, 24), (16, 32), (8, 64), (3, 32)])
        rotary = rng.choice([head_dim, head_dim, 8, 0])
        return _qk_norm(_log(rng, 1, 130000), heads, head_dim, rng.choice(["bf16", "fp32"]), rng.random() < 0.6, rotary,
                        rng.random() < 0.4, rng.choice([0, 0, 70001, 2000000]))
    dtype = rng.choice(["bf16", "fp32"])
    return _clip(rng.choice([64, 128, 192, 256, 300]), _log(rng, 64, 2048), _log(rng, 1, 16), dtype,
                 dtype if rng.random() < 0.5 else "fp32", rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ the inputs

@functools.lru_cache(maxsize=64)
def _lengths(graphs, size, pick):
    """Tokens of each graph in the generator's order."""
    if graphs == "molecules":
        gb = generators.small_molecules(seed=pick, num_graphs=size)[0]
    elif graphs == "proteins":
        gb = generators.protein_like(seed=pick, num_graphs=size)
    else:
        gb = generators.protein_budget(seed=pick, token_budget=size)
    return tuple(int(n) for n in gb.edge_counts)


def _shapes(case):
    """The parameters of ``layers`` pre-norm blocks: two norms, four projections and the MLP, with their biases."""
    d, m = case["dim"], case["mlp"]
    block = [(d,), (d,)] + [(d, d), (d,)] * 4 + [(d,), (d,), (m, d), (m,), (d, m), (d,)]
    return block * case["layers"]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, device=DEV, generator=gen).to(dtype)

    dt = DTYPES[case["dtype"]]
    if case["kind"] == "relative":
        lens = np.random.default_rng(int(seed)).permutation(_lengths(case["graphs"], case["size"], case["pick"]))
        rows = np.minimum(lens, case["rows"]) if case["rows"] else lens
        h, hd, tq, tk = case["heads"], case["head_dim"], int(rows.sum()), int(lens.sum())

        def cu(n):
            return torch.as_tensor(np.concatenate([[0], np.cumsum(n)]).astype(np.int32)).to(DEV)

        s = {"case": case, "len_q": [int(n) for n in rows], "len_k": [int(n) for n in lens], "cu_k": cu(lens)}
        s["cu_q"] = cu(rows) if case["rows"] else s["cu_k"]
        s["q_start"] = torch.as_tensor((lens - rows).astype(np.int32)).to(DEV) if case["rows"] else None
        s["q"], s["k"], s["v"] = randn(tq, h, hd, dtype=dt), randn(tk, h, hd, dtype=dt), randn(tk, h, hd, dtype=dt)
        s["bias"] = randn(case["buckets"], h).mul_(0.5).to(dt)   # a trained table's spread, in the layer's type
        if case["train"]:
            s["g"] = randn(tq, h, hd, dtype=dt)
            for name in ("q", "k", "v", "bias"):
                s[name].requires_grad_(True)
        return s
    if case["kind"] == "qk_norm":
        t, h, hd = case["tokens"], case["heads"], case["head_dim"]
        qkv = randn(t, 3, h, hd, dtype=dt)   # one projection's output, whose queries and keys are views
        s = {"case": case, "q": qkv[:, 0], "k": qkv[:, 1]}
        s["wq"], s["wk"] = randn(hd).mul_(0.2).add_(1), randn(hd).mul_(0.2).add_(1)
        s["positions"] = s["frequencies"] = None
        if case["rotary"]:
            length = np.random.default_rng(int(seed)).integers(1, 2000)   # positions begin again with every graph
            s["positions"] = (torch.arange(t, device=DEV, dtype=torch.int32) % int(length)) + case["first"]
            s["frequencies"] = 10000.0 ** (-torch.arange(0, case["rotary"], 2, device=DEV, dtype=torch.float64)
                                           / case["rotary"])
        if case["train"]:
            s["gq"], s["gk"] = randn(t, h, hd, dtype=dt), randn(t, h, hd, dtype=dt)
            for name in ("q", "k", "wq", "wk"):
                s[name] = s[name].detach().requires_grad_(True)
        return s
    shapes = _shapes(case)
    sizes = [math.prod(x) for x in shapes]
    scale = torch.exp(randn(len(sizes)))   # layers differ in the size of their gradients
    flat = randn(sum(sizes)).mul_(torch.repeat_interleave(scale, torch.tensor(sizes, device=DEV))).mul_(1e-2).to(dt)
    out = torch.empty(sum(sizes), device=DEV, dtype=DTYPES[case["out"]])
    grads = [g.view(x) if case["ragged"] else g.view(x).clone() for g, x in zip(flat.split(sizes), shapes)]
    return {"case": case, "grads": grads, "flat": out, "out": [o.view(x) for o, x in zip(out.split(sizes), shapes)],
            "max_norm": 1.0}


# ------------------------------------------------------------------------------------------------ one pass

def run(s):
    case = s["case"]
    if case["kind"] == "relative":
        return _run_relative(s, case)
    if case["kind"] == "qk_norm":
        return _run_qk_norm(s, case)
    return _run_clip(s)


def _run_relative(s, case):
    if own:
        from mind_amd.esa.relative import relative_attention
        out = relative_attention(s["q"], s["k"], s["v"], s["bias"], s["cu_q"], s["cu_k"], max(s["len_q"]),
                                 max(s["len_k"]), max_distance=case["distance"], bidirectional=case["two_sided"],
                                 q_start=s["q_start"])
        if not case["train"]:
            return {"out": out}
        dq, dk, dv, db = torch.autograd.grad(out, (s["q"], s["k"], s["v"], s["bias"]), s["g"])
        return {"out": out, "dq": dq, "dk": dk, "dv": dv, "dbias": db}
    with torch.no_grad():
        return _plain_relative(s, case)


def _run_qk_norm(s, case):
    if own:
        from mind_amd.esa.qk_norm import qk_norm_rotary
        q, k = qk_norm_rotary(s["q"], s["k"], s["wq"], s["wk"], positions=s["positions"],
                              frequencies=s["frequencies"], eps=EPS, interleaved=case["interleaved"])
    else:
        turn = _plain_angles(s, case)
        q, k = (_plain_norm(s[x], s["w" + x], turn, case) for x in ("q", "k"))
    if not case["train"]:
        return {"q": q, "k": k}
    dq, dk, dwq, dwk = torch.autograd.grad((q, k), (s["q"], s["k"], s["wq"], s["wk"]), (s["gq"], s["gk"]))
    return {"q": q, "k": k, "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}


def _run_clip(s):
    if own:
        from mind_amd.esa.gradients import clip_gradients
        norm = clip_gradients(s["grads"], s["max_norm"], out=s["out"])
        return {"norm": norm, "clipped": s["flat"]}
    flat = torch.cat([g.reshape(-1) for g in s["grads"]]).float()
    norm = flat.square().sum().sqrt()
    s["flat"].copy_(flat * torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0))
    return {"norm": norm, "clipped": s["flat"]}


# ------------------------------------------------------------------------------------------------ plain forms

_BUDGET = 1 << 27   # scores of one group of graphs in the plain form


def _starts(buckets, distance, two_sided):
    """The distance at which each bucket of a side begins, in whole numbers: bucket exact + t from the least n with
    (n / exact)^wide >= (distance / exact)^t."""
    side = buckets // 2 if two_sided else buckets
    exact = side // 2
    wide, starts, n = side - exact, list(range(exact)), exact
    for t in range(wide):
        while n ** wide * exact ** t < distance ** t * exact ** wide:
            n += 1
        starts.append(n)
    return starts


def _groups(s, heads):
    """Runs of graphs whose padded scores fit the budget, each with its number of heads at a time."""
    lq, lk, first = s["len_q"], s["len_k"], 0
    while first < len(lq):
        last, a, b = first, 0, 0
        while last < len(lq):
            a2, b2 = max(a, lq[last]), max(b, lk[last])
            if last > first and (last + 1 - first) * a2 * b2 * heads > _BUDGET:
                break
            last, a, b = last + 1, a2, b2
        yield first, last, max(1, min(heads, _BUDGET // ((last - first) * a * b)))
        first = last


def _plain_relative(s, case):
    q, k, v, g = s["q"], s["k"], s["v"], s.get("g")
    h, hd, nb, train = case["heads"], case["head_dim"], case["buckets"], case["train"]
    scale = 1.0 / math.sqrt(hd)
    starts = torch.tensor(_starts(nb, case["distance"], case["two_sided"]), device=DEV)
    out = torch.zeros(q.shape, device=DEV)
    if train:
        dq, dk, dv, db = (torch.zeros(x.shape, device=DEV) for x in (q, k, v, s["bias"]))
    for first, last, step in _groups(s, h):
        n, lq, lk = last - first, max(s["len_q"][first:last]), max(s["len_k"][first:last])
        i, j = torch.arange(lq, device=DEV), torch.arange(lk, device=DEV)
        bq, bk = s["cu_q"][first:last, None].long(), s["cu_k"][first:last, None].long()
        in_q = i < s["cu_q"][first + 1:last + 1, None] - bq   # [n, lq]
        in_k = j < s["cu_k"][first + 1:last + 1, None] - bk
        at_q, at_k = (bq + i).clamp_(max=q.shape[0] - 1), (bk + j).clamp_(max=k.shape[0] - 1)
        d = (j - i[:, None])[None]
        if s["q_start"] is not None:
            d = d - s["q_start"][first:last, None, None]   # [n, lq, lk], else [1, lq, lk]
        far = (d.abs() if case["two_sided"] else (-d).clamp_(min=0)).contiguous()
        bucket = torch.searchsorted(starts, far, right=True) - 1
        if case["two_sided"]:
            bucket += (d > 0) * (nb // 2)
        kinds = (bucket.reshape(-1, 1) == torch.arange(nb, device=DEV)).float() if train else None
        for h0 in range(0, h, step):
            hs = slice(h0, min(h0 + step, h))

            def rows(x, at):   # [n, heads, length, hd]
                return x[:, hs][at].float().permute(0, 2, 1, 3).contiguous()

            qp, kp, vp = rows(q, at_q), rows(k, at_k), rows(v, at_k)
            p = torch.matmul(qp, kp.transpose(2, 3)).mul_(scale)
            p += s["bias"][:, hs].float()[bucket].permute(0, 3, 1, 2)
            p.masked_fill_(~in_k[:, None, None, :], -math.inf)
            p -= p.amax(3, keepdim=True)
            p.exp_()
            p /= p.sum(3, keepdim=True)
            o = torch.matmul(p, vp)
            out[:, hs][at_q[in_q]] = o.permute(0, 2, 1, 3)[in_q]
            if not train:
                continue
            gp = rows(g, at_q) * in_q[:, None, :, None]
            dvp = torch.matmul(p.transpose(2, 3), gp)
            ds = torch.matmul(gp, vp.transpose(2, 3))
            ds -= (gp * o).sum(3, keepdim=True)
            ds *= p
            dqp, dkp = torch.matmul(ds, kp).mul_(scale), torch.matmul(ds.transpose(2, 3), qp).mul_(scale)
            dq[:, hs][at_q[in_q]] = dqp.permute(0, 2, 1, 3)[in_q]
            dk[:, hs][at_k[in_k]] = dkp.permute(0, 2, 1, 3)[in_k]
            dv[:, hs][at_k[in_k]] = dvp.permute(0, 2, 1, 3)[in_k]
            pairs = ds.sum(0) if d.shape[0] == 1 else ds.permute(1, 0, 2, 3)
            db[:, hs] += torch.matmul(pairs.reshape(pairs.shape[0], -1), kinds).t()
    res = {"out": out.to(q.dtype)}
    if train:
        res |= {"dq": dq.to(q.dtype), "dk": dk.to(q.dtype), "dv": dv.to(q.dtype), "dbias": db.to(s["bias"].dtype)}
    return res


def _plain_angles(s, case):
    """(cos, sin) [T, 1, rotary / 2] of the tokens' angles; far positions need 64 bits."""
    if not case["rotary"]:
        return None
    angle = s["positions"].double()[:, None, None] * s["frequencies"]
    return torch.cos(angle).float(), torch.sin(angle).float()


def _plain_norm(x, w, turn, case):
    y = x.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w
    if turn is not None:
        r, (cos, sin) = case["rotary"], turn
        a, b = (y[..., 0:r:2], y[..., 1:r:2]) if case["interleaved"] else (y[..., :r // 2], y[..., r // 2:r])
        u, v = a * cos - b * sin, a * sin + b * cos
        turned = torch.stack((u, v), -1).flatten(-2) if case["interleaved"] else torch.cat((u, v), -1)
        y = torch.cat((turned, y[..., r:]), -1)
    return y.to(x.dtype)


# ------------------------------------------------------------------------------------------------ what it takes

def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "relative":
        lens = np.asarray(_lengths(case["graphs"], case["size"], case["pick"]), dtype=np.int64)
        rows = np.minimum(lens, case["rows"]) if case["rows"] else lens
        d, tq, tk = case["heads"] * case["head_dim"], int(rows.sum()), int(lens.sum())
        table = case["buckets"] * case["heads"] * size
        pairs = int((rows * lens).sum())
        if case["train"]:   # q, k, v, the output and its gradient read or written once, the gradients written
            return {"bytes": (4 * tq + 4 * tk) * d * size + 2 * table, "flops": 14 * d * pairs}
        return {"bytes": (2 * tq + 2 * tk) * d * size + table, "flops": 4 * d * pairs}
    if case["kind"] == "qk_norm":
        n, hd = 2 * case["tokens"] * case["heads"] * case["head_dim"], case["head_dim"]
        extra = (4 * case["tokens"] + 4 * case["rotary"] if case["rotary"] else 0) + 8 * hd
        # forward: read x, write y; training: x, y, and in the backward g and dx
        return {"bytes": (4 if case["train"] else 2) * n * size + extra, "flops": (24 if case["train"] else 8) * n}
    n = sum(math.prod(x) for x in _shapes(case))
    return {"bytes": n * (size + (4 if case["out"] == "fp32" else 2)) + 4, "flops": 3 * n}


# ------------------------------------------------------------------------------------------------ in 64 bits

def _bucket_of(d, case):
    """The bucket of whole distances d (key position minus query position), by logarithms in 64 bits: a quotient
    within 1e-9 of a whole number is that number."""
    side = case["buckets"] // 2 if case["two_sided"] else case["buckets"]
    exact = side // 2
    far = d.abs() if case["two_sided"] else torch.relu(-d)
    x = torch.log(far.clamp(min=1).double() / exact) / math.log(case["distance"] / exact) * (side - exact)
    coarse = exact + torch.floor(x + 1e-9).long()
    bucket = torch.where(far < exact, far, coarse.clamp(max=side - 1))
    return bucket + side * (d > 0).long() if case["two_sided"] else bucket


def _exact_relative(s, case):
    h, hd, nb = case["heads"], case["head_dim"], case["buckets"]
    q, k, v, table = (s[x].detach().double() for x in ("q", "k", "v", "bias"))
    g = s["g"].double() if case["train"] else None
    out, dq, dk, dv = (torch.zeros_like(x) for x in (q, q, k, v))
    db = torch.zeros_like(table)
    qs = ks = 0
    starts = s["q_start"].tolist() if s["q_start"] is not None else [0] * len(s["len_q"])
    for lq, lk, start in zip(s["len_q"], s["len_k"], starts):
        d = torch.arange(lq + lk - 1, device=DEV) - (lq - 1) - start   # of the pair (i, j): d[j - i + lq - 1]
        by_d = _bucket_of(d, case)
        for x in range(h):
            qx, kx, vx = q[qs:qs + lq, x], k[ks:ks + lk, x], v[ks:ks + lk, x]
            line = table[by_d, x]
            # row i of the bias is line[lq - 1 - i :][:lk]
            bias = line.unfold(0, lk, 1).flip(0)
            p = torch.softmax(qx @ kx.T / math.sqrt(hd) + bias, 1)
            out[qs:qs + lq, x] = p @ vx
            if g is None:
                continue
            gx = g[qs:qs + lq, x]
            ds = gx @ vx.T
            ds = p * (ds - (p * ds).sum(1, keepdim=True))
            dq[qs:qs + lq, x] = ds @ kx / math.sqrt(hd)
            dk[ks:ks + lk, x] = ds.T @ qx / math.sqrt(hd)
            dv[ks:ks + lk, x] = p.T @ gx
            # one diagonal a column: rows from the last, each one longer by lq and read one short
            skew = torch.nn.functional.pad(ds.flip(0), (0, lq)).reshape(-1)[:lq * (lk + lq - 1)].reshape(lq, -1)
            db[:, x].index_add_(0, by_d, skew.sum(0))
        qs, ks = qs + lq, ks + lk
    return {"out": out, "dq": dq, "dk": dk, "dv": dv, "dbias": db} if case["train"] else {"out": out}


def _exact_qk_norm(s, case):
    res, half = {}, case["rotary"] // 2
    if half:
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV),
                           s["positions"].double()[:, None] * s["frequencies"])[:, None]

    def rotated(x, turn):   # the first dims as complex numbers
        if not half:
            return x
        y = x.clone()
        z = x[..., :2 * half].unflatten(-1, (half, 2) if case["interleaved"] else (2, half))
        z = (z if case["interleaved"] else z.transpose(-1, -2)).contiguous()
        z = torch.view_as_real(torch.view_as_complex(z) * turn)
        y[..., :2 * half] = (z if case["interleaved"] else z.transpose(-1, -2)).flatten(-2)
        return y

    for name in ("q", "k"):
        x, w = s[name].detach().double(), s["w" + name].detach().double()
        rms = torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
        unit = x / rms
        res[name] = rotated(unit * w, turn if half else None)
        if case["train"]:
            g = rotated(s["g" + name].double(), turn.conj() if half else None)
            res["dw" + name] = (g * unit).sum((0, 1))
            res["d" + name] = (g * w - unit * (g * w * unit).mean(-1, keepdim=True)) / rms
    return res


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "relative":
            # a product and some passes for each graph and head: over 4,000 of them take too long
            return _exact_relative(s, case) if len(s["len_q"]) * case["heads"] <= 4000 else None
        if case["kind"] == "qk_norm":
            return _exact_qk_norm(s, case)
        every = [g.double() for g in s["grads"]]
        norm = math.sqrt(math.fsum(float((g * g).sum()) for g in every))
        factor = min(1.0, s["max_norm"] / (norm + 1e-6))
        return {"norm": torch.tensor(norm, dtype=torch.float64), "clipped": torch.cat([g.flatten() * factor for g in every])}

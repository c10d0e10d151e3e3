"""Refusals of the query and key norms and of the gradient norm (no GPU needed)."""
import ctypes
import math

import numpy as np
import pytest
import torch

from mind_amd import _lib
from mind_amd.esa.gradients import clip_gradients, grad_norm
from mind_amd.esa.qk_norm import qk_norm_rotary, rotary_frequencies


def test_frequencies():
    f = rotary_frequencies(8, 10000.0)
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-15)
    for bad in (0, 7, -2):
        with pytest.raises(ValueError):
            rotary_frequencies(bad)


def _x(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


POS, FREQ = torch.arange(6), rotary_frequencies(16)


@pytest.mark.parametrize("args,error", [
    (dict(q=_x(6, 2, 20)), ValueError), (dict(q=_x(6, 32)), ValueError), (dict(q=_x(6, 2, 16, dtype=torch.float16)), TypeError),
    (dict(q=_x(6, 0, 16)), ValueError), (dict(q=_x(1, 2049, 16)), ValueError),
    (dict(k=_x(5, 2, 16)), ValueError), (dict(k=_x(6, 2, 32)), ValueError), (dict(k=_x(6, 2, 16, dtype=torch.bfloat16)), ValueError),
    (dict(q_weight=_x(8)), ValueError), (dict(q_weight=_x(16, dtype=torch.float64)), ValueError),
    (dict(k=None, k_weight=_x(16)), ValueError), (dict(positions=POS), ValueError), (dict(frequencies=FREQ), ValueError),
    (dict(positions=POS.float(), frequencies=FREQ), TypeError), (dict(positions=torch.arange(12)[::2], frequencies=FREQ), TypeError),
    (dict(positions=POS[:5], frequencies=FREQ), ValueError), (dict(positions=POS, frequencies=FREQ.float()), TypeError),
    (dict(positions=POS, frequencies=FREQ[:3]), ValueError), (dict(positions=POS, frequencies=rotary_frequencies(24)), ValueError),
    (dict(positions=POS, frequencies=FREQ[:0]), ValueError), (dict(eps=-1e-6), ValueError), (dict(eps=math.inf), ValueError),
    (dict(), _lib.EsaError)])   # host tensors
def test_qk_norm_refused(args, error):
    with pytest.raises(error):
        qk_norm_rotary(**{"q": _x(6, 2, 16), "k": _x(6, 3, 16), **args})


def test_qk_norm_entry_points_refuse_before_launch():
    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    lib = _lib.load()

    def fwd(q=16, k=16, strides=(32, 16, 32, 16), total=5, hq=2, hk=2, hd=16, dt=0, pos=16, pb=4, f=16, r=16, eps=1e-6, out=16):
        return lib.esa_qk_norm_fwd(q, k, (ctypes.c_longlong * 4)(*strides), total, hq, hk, hd, dt, None, None, pos, pb, f, r, 0,
                                   eps, out, 16, None)
    assert fwd(hd=20) == -3 and fwd(dt=4) == -5 and fwd(total=-1) == -2 and fwd(hq=0) == -2 and fwd(hk=-1) == -2
    assert fwd(hq=3000) == -2 and fwd(eps=-1.0) == -2 and fwd(r=12) == -2 and fwd(r=24) == -2 and fwd(pb=2) == -5
    assert fwd(q=None) == -1 and fwd(k=None) == -1 and fwd(pos=None) == -1 and fwd(f=None) == -1 and fwd(out=None) == -1
    assert fwd(q=8) == -6 and fwd(strides=(33, 16, 32, 16)) == -6 and fwd(out=20) == -6
    assert fwd(total=0, q=None, out=None) == 0
    assert lib.esa_qk_norm_fwd(16, 16, None, 5, 2, 2, 16, 0, None, None, None, 0, None, 0, 0, 0.0, 16, 16, None) == -1
    n = ctypes.c_size_t(0)
    assert lib.esa_qk_norm_bwd_workspace_size(1000, 16, ctypes.byref(n)) == 0 and n.value > 0
    assert lib.esa_qk_norm_bwd_workspace_size(1000, 17, ctypes.byref(n)) == -3
    s = (ctypes.c_longlong * 4)(32, 16, 32, 16)

    def bwd(gq=16, dq=16, dwq=16, ws=16, nbytes=1 << 20):
        return lib.esa_qk_norm_bwd(gq, 16, 16, 16, s, 5, 2, 2, 16, 0, None, None, None, 0, None, 0, 0, 0.0, dq, 16, dwq, None, ws,
                                   nbytes, None)
    assert bwd(gq=None) == -1 and bwd(dq=None) == -1 and bwd(ws=None) == -1 and bwd(nbytes=4) == -4 and bwd(gq=4) == -6
    assert bwd(ws=18) == -6


def test_gradient_norm_refuses_host_tensors():
    with pytest.raises(_lib.EsaError):
        grad_norm([torch.zeros(4)])
    with pytest.raises(TypeError):
        clip_gradients([torch.zeros(4, dtype=torch.float64)], 1.0)
    assert float(grad_norm([])) == 0.0


def _spans(spans):
    """(pointers, counts, codes) of float32 tensors over byte spans."""
    spans = np.array(spans, dtype=np.int64).reshape(-1, 2)
    return spans[:, 0].tobytes(), ((spans[:, 1] - spans[:, 0]) // 4).tobytes(), np.zeros(len(spans), dtype=np.int32).tobytes()


def test_separate_against_every_pair():
    separate, rng = _lib.tensors().separate, np.random.default_rng(0)
    for trial in range(2000):
        n = int(rng.integers(1, 5))
        first = rng.integers(0, 24, size=(2, n)) * 4
        size = rng.integers(0, 5, size=(2, n)) * 4
        if trial % 3 == 0:
            first[1], size[1] = first[0], size[0]
        d, s = ([(int(f), int(f + z)) for f, z in zip(first[i], size[i])] for i in (0, 1))

        def shares(a, b):
            return max(a[0], b[0]) < min(a[1], b[1])
        apart = not any(shares(d[i], d[j]) for i in range(n) for j in range(i))
        assert separate(_spans(d), None) == apart
        want = apart and not any(shares(d[i], s[j]) and not (i == j and d[i] == s[j]) for i in range(n) for j in range(n))
        assert separate(_spans(d), _spans(s)) == want


def test_describe():
    describe = _lib.tensors().describe
    a, b = torch.zeros(3, 5), torch.zeros(8, dtype=torch.bfloat16)
    ptrs, counts, codes, device, contiguous = describe([a, b])
    assert np.frombuffer(ptrs, np.int64).tolist() == [a.data_ptr(), b.data_ptr()] and device == -1 and contiguous
    assert np.frombuffer(counts, np.int64).tolist() == [15, 8] and np.frombuffer(codes, np.int32).tolist() == [0, 1]
    assert describe([a.t()])[4] is False and describe([])[0] == b""
    for bad in ([a, 3], (a,), [a.double()], [a.to_sparse()], [None]):
        with pytest.raises(TypeError):
            describe(bad)
    misfit = _lib.tensors().misfit
    assert misfit([a, b], [a + 1, b.clone()]) is None and misfit([b], [b.float()]) is None
    assert misfit([a], [a.t()]) == misfit([a], [a, b]) == misfit([a], [a.view(-1)]) == "shapes"
    assert misfit([a], [a.bfloat16()]) == misfit([b], [b.half()]) == "dtypes"
    with pytest.raises(TypeError):
        misfit([a], [3])
    version = a._version
    _lib.tensors().changed([a, torch.nn.Parameter(b)])
    assert a._version == version + 1
    with torch.inference_mode():
        inside = torch.zeros(2)
    _lib.tensors().changed([inside])


def test_gradient_entry_points_refuse_before_launch():
    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    lib, n = _lib.load(), ctypes.c_size_t(0)

    def lists(ptrs=(16,), counts=(10,), codes=(0,)):
        k = len(ptrs)
        return (ctypes.c_void_p * k)(*ptrs), (ctypes.c_longlong * k)(*counts), (ctypes.c_int * k)(*codes)

    def norm(n_=1, out=16, ws=16, nbytes=1 << 20, **kw):
        p, c, d = lists(**kw)
        return lib.esa_grad_norm(n_, p, c, d, 0, out, ws, nbytes, None)
    assert norm(n_=-1) == -2 and norm(counts=(-1,)) == -2 and norm(codes=(3,)) == -5 and norm(ptrs=(None,)) == -1
    assert norm(ptrs=(18,)) == -6 and norm(ptrs=(17,), codes=(1,)) == -6 and norm(out=None) == -1 and norm(ws=None) == -1
    assert norm(nbytes=4) == -4
    p, c, d = lists()
    assert lib.esa_grad_workspace_size(1, c, 0, ctypes.byref(n)) == 0 and n.value >= 8
    assert lib.esa_grad_workspace_size(1, None, 0, ctypes.byref(n)) == -1
    assert lib.esa_grad_workspace_size(1, (ctypes.c_longlong * 1)(-3), 1, ctypes.byref(n)) == -2

    def clip(out=(16,), out_codes=(0,), max_norm=1.0, norm_at=16, ws=16, nbytes=1 << 20, **kw):
        p, c, d = lists(**kw)
        return lib.esa_grad_clip(1, p, (ctypes.c_void_p * 1)(*out), c, d, (ctypes.c_int * 1)(*out_codes), 0, max_norm, norm_at,
                                 ws, nbytes, None)
    assert clip(ws=None) == -1 and clip(ws=12) == -6 and clip(nbytes=16) == -4
    assert clip(out=(None,)) == -1 and clip(out=(18,)) == -6 and clip(out_codes=(1,)) == -5 and clip(norm_at=None) == -1
    assert clip(max_norm=-1.0) == -2 and clip(max_norm=float("nan")) == -2


def test_token_order_is_the_packed_encoders():
    from mind_amd.esa.masked_layers import ESA, SABComplete
    from mind_amd.esa.token_order import TokenOrder
    args = (2, 8, [32, 32], [2, 2], ["S", "P"])
    order = TokenOrder(num_buckets=4, max_distance=10)
    for backend in ("xformers", "torch", "flash_varlen"):
        with pytest.raises(ValueError):
            ESA(*args, xformers_or_torch_attn=backend, token_order=order)
    with pytest.raises(ValueError):
        SABComplete(32, 32, 2, 0.0, 2, "LN", xformers_or_torch_attn="hip", token_order=order)   # a decoder layer
    with pytest.raises(ValueError):
        SABComplete(32, 32, 3, 0.0, 0, "LN", xformers_or_torch_attn="hip", token_order=order)   # 32 dims in 3 heads
    with pytest.raises(ValueError):
        SABComplete(32, 32, 4, 0.0, 0, "LN", xformers_or_torch_attn="hip", token_order=order)   # head dim 8
    for bad in (TokenOrder(rotary_dim=12), TokenOrder(rotary_dim=24), TokenOrder(num_buckets=5)):
        with pytest.raises(ValueError):
            ESA(*args, xformers_or_torch_attn="hip", token_order=bad)
    m = ESA(*args, xformers_or_torch_attn="hip", token_order=order)
    x = torch.zeros(1, 4, 32)
    with pytest.raises(TypeError):
        m.encoder[0]((x, None, None, 4, None))
    with pytest.raises(RuntimeError):
        m.encoder[0].sab(x)

"""Tensors whose element offsets pass 2^31 and byte offsets 2^32: the last segment's results are those of the segment
alone.  bf16 rows may take another reference point of the softmax there (their key norms are by 32 tokens of the whole
tensor), which moves each rounding of P by at most a step of 2^-8: outputs and gradients to 1e-2 of their norm."""
import pytest
import torch

from mind_amd.esa.qk_norm import qk_norm_rotary, rotary_frequencies
from mind_amd.esa.relative import relative_attention

pytestmark = pytest.mark.gpu

LAST = 70


@pytest.fixture(autouse=True)
def given_back():
    yield
    torch.cuda.empty_cache()


def _room(gib):
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"needs {gib} GiB of GPU memory")


@pytest.mark.parametrize("dtype,hd,heads,tokens", [(torch.bfloat16, 16, 1024, 135000), (torch.bfloat16, 64, 1024, 34000),
                                                   (torch.float32, 32, 512, 135000)], ids=str)
def test_relative_attention(device, dtype, hd, heads, tokens):
    assert tokens * heads * hd > 2 ** 31
    _room(120)
    gen = torch.Generator(device).manual_seed(3)
    lens = [50] * ((tokens - LAST) // 50) + [(tokens - LAST) % 50, LAST]
    cu = torch.tensor([0] + lens).cumsum(0).int().to(device)
    q, k, v, g = (torch.randn(tokens, heads, hd, device=device, dtype=dtype, generator=gen) for _ in range(4))
    b = torch.randn(8, heads, device=device, generator=gen)
    leaves = [x.requires_grad_(True) for x in (q, k, v, b)]
    out = relative_attention(*leaves, cu, cu, max_distance=20)
    grads = torch.autograd.grad(out, leaves, g)
    small = [x.detach()[-LAST:].clone().requires_grad_(True) for x in (q, k, v)]
    one = torch.tensor([0, LAST], dtype=torch.int32, device=device)
    ref = relative_attention(*small, b, one, one, max_distance=20)
    ref_grads = torch.autograd.grad(ref, small, g[-LAST:])
    for got, want in zip((out.detach(), *grads[:3]), (ref.detach(), *ref_grads)):
        assert float((got[-LAST:].float() - want.float()).norm() / want.float().norm()) <= 1e-2
        assert bool(torch.isfinite(got[-LAST:]).all())


def test_norms_with_rotation(device):
    tokens, heads, hd = 135000, 1024, 16
    _room(60)
    gen = torch.Generator(device).manual_seed(4)
    q, g = (torch.randn(tokens, heads, hd, device=device, dtype=torch.bfloat16, generator=gen) for _ in range(2))
    at, w, f = torch.arange(tokens, device=device), torch.rand(hd, device=device, generator=gen), rotary_frequencies(16, device=device)
    q.requires_grad_(True)
    out = qk_norm_rotary(q, q_weight=w, positions=at, frequencies=f)
    grad, = torch.autograd.grad(out, q, g)
    small = q.detach()[-LAST:].clone().requires_grad_(True)
    ref = qk_norm_rotary(small, q_weight=w, positions=at[-LAST:].clone(), frequencies=f)
    ref_grad, = torch.autograd.grad(ref, small, g[-LAST:].clone())
    assert torch.equal(out[-LAST:], ref) and torch.equal(grad[-LAST:], ref_grad)

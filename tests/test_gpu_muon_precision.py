"""How many bits the orthogonalised updates keep: results in bf16 are the fp32 results rounded once, fp32 results hold their stated error."""
import pytest
import torch

from simple3d_former_amd import ops
from tests.test_gpu_muon import grads, oracle, rel

pytestmark = pytest.mark.gpu
CO = ops.NS_COEFFICIENTS

# one or more shapes for every tile: polynomial and product in one launch, 32 x 32, 64 x 64, 128 x 64, 128 x 128; wide, tall, odd
SHAPES = [(1, 1, 1), (2, 9, 1), (1, 192, 192), (1, 63, 130), (3, 150, 190), (1, 387, 1000), (1, 768, 768), (12, 384, 384), (12, 1536, 384), (12, 384, 1536), (9, 700, 640),
          (2, 2048, 2048), (130, 256, 520)]


@pytest.mark.parametrize('L,r,c', SHAPES)
@pytest.mark.parametrize('src', [torch.float32, torch.bfloat16])
def test_bf16_results_are_the_fp32_results_rounded_once(L, r, c, src):
    x = grads(L, r, c, dtype=src)
    assert torch.equal(ops.orthogonalize(x, out_dtype=torch.bfloat16), ops.orthogonalize(x, out_dtype=torch.float32).to(torch.bfloat16))


@pytest.mark.parametrize('steps', [1, 2, 3, 8])
@pytest.mark.parametrize('co', [CO, (1.875, -1.25, 0.375), (4.275, -13.851, 8.9755)])
@pytest.mark.parametrize('shape', [(2, 70, 200), (2, 500, 300)])
def test_bf16_results_with_other_steps_and_coefficients(steps, co, shape):
    """Few steps, and a polynomial that multiplies small singular values (and what is rounded into them) by 4.3 a step (0.95 T5(0.9 s), T5 the Chebyshev polynomial:
    within 0.95 on [0, 1])."""
    x = grads(*shape)
    got = ops.orthogonalize(x, steps=steps, coefficients=co, out_dtype=torch.bfloat16)
    full = ops.orthogonalize(x, steps=steps, coefficients=co)
    assert torch.equal(got, full.to(torch.bfloat16))


@pytest.mark.parametrize('kind', ['rank one', 'geometric'])
def test_bf16_results_of_hard_spectra_are_rounded_once(kind):
    """Rank one and six decades of singular values: half a step of bf16 (2^-8 at most, 2^-9 and less in the 2-norm of many entries)."""
    g = torch.Generator().manual_seed(3)
    L, r, c = 2, 200, 320
    if kind == 'rank one':
        x = torch.randn(L, r, 1, generator=g) @ torch.randn(L, 1, c, generator=g)
    else:
        u, v = (torch.linalg.qr(torch.randn(n, r, generator=g))[0] for n in (r, c))
        x = ((u * torch.logspace(0, -6, r)) @ v.T).expand(L, r, c).contiguous()
    x = x.to('cuda:0')
    assert torch.equal(ops.orthogonalize(x, out_dtype=torch.bfloat16), ops.orthogonalize(x).to(torch.bfloat16))
    assert rel(ops.orthogonalize(x, out_dtype=torch.bfloat16), oracle(x)) <= 2.0 ** -9


# fp32 results of gradient-like spectra, where all directions grow together and an error keeps its size beside the result.
#   Random part: every step rounds four tensors to pairs, at most 2^-22 of an entry, 2^-22 / sqrt(12) rms: sqrt(5 * 4) 2^-22 / sqrt(12) = 3.1e-7.
#   One-sided part: sums that begin at zero every 64 k take six truncated products, at most 2^-24 each, half on average: 1.8e-7 of a product.  It
#   enters through A with |b + 2 c| = 0.7 and through P X with 1, so 3.1e-7 a step, and is multiplied by p'(1) = a + 3 b + 5 c = -0.72 a step later:
#   3.1e-7 / sqrt(1 - 0.72^2) = 4.4e-7.
# In quadrature 5.4e-7; if all of the one-sided part adds to the random one, 7.5e-7: bounded by the next power of two.  A^2 instead of (A - shift)^2 gives
# 0.6e-6 .. 1.3e-6 here, one running sum instead of the restarted ones 0.6e-6 .. 1.5e-6, both 0.7e-6 .. 2.2e-6 (1 / norm in one part adds 2e-8).
FP32 = 2.0 ** -20


@pytest.mark.parametrize('r,c', [(192, 192), (768, 384), (1536, 384), (192, 768), (384, 1536)])
@pytest.mark.parametrize('L', [1, 12, 40])
def test_fp32_results_hold_the_stated_error(L, r, c):
    x = grads(1, r, c)
    got = ops.orthogonalize(x.expand(L, r, c).contiguous())
    want = oracle(x)
    e = [rel(got[i:i + 1], want) for i in (0, L - 1)]
    print(f'{L} x {r} x {c}: {max(e):.2e}')
    assert max(e) <= FP32

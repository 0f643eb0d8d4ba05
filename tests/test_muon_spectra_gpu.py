"""hold_amd.muon on wide matrices whose singular values are spread: one arithmetic for updates, float32 and 16-bit results, in any batch.
The tolerances are those of test_muon_gpu: at most four times float32's error in norm, half a step of the result's type on top."""
import pytest
import torch

from parity_common import ROOT  # noqa: F401
from test_muon_gpu import iterate, off, step64

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def spread(kind, rows, cols, seed=0):
    """singular values over two decades; or a few strong directions over noise a hundredth as large"""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    m = min(rows, cols)
    if kind == "rank":
        low = torch.randn(rows, 64, generator=gen, device=DEV) @ torch.randn(64, cols, generator=gen, device=DEV)
        return (low + 0.1 * torch.randn(rows, cols, generator=gen, device=DEV)) * 1e-3
    u, _ = torch.linalg.qr(torch.randn(rows, m, generator=gen, device=DEV, dtype=torch.float64))
    v, _ = torch.linalg.qr(torch.randn(cols, m, generator=gen, device=DEV, dtype=torch.float64))
    return ((u * torch.logspace(0, -2, m, device=DEV, dtype=torch.float64)) @ v.T.contiguous()).float()


@pytest.mark.parametrize("kind", ["decades", "rank"])
@pytest.mark.parametrize("shape", [(1024, 2048), (2600, 640)])
def test_wide_updates_are_orthogonalizes(kind, shape):
    """a step from zero without momentum is the iteration itself: bit for bit what orthogonalize gives, and as exact as float32"""
    from hold_amd.muon import muon_step, orthogonalize
    g = spread(kind, *shape)
    p, m = torch.zeros(shape, device=DEV), torch.zeros(shape, device=DEV)
    muon_step([p], [g], [m], lr=1.0, momentum=0.0, scale=1.0)
    assert torch.equal(p, -orthogonalize(g))
    p64, _, u = step64(torch.zeros(shape), g, torch.zeros(shape), 1.0, 0.0, True, 0.0, 1.0)
    assert off(p, p64) <= 4 * off(iterate(u.float()), iterate(u))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["decades", "rank"])
def test_wide_matrices_in_16_bits_are_float32s_rounded(kind, dtype):
    """alone and in a batch the iteration is float32's, rounded once at the end (but for the order of the norm's sum, which moves a rounding
    of the start by 2^-24 in one of some 10^9 elements)"""
    from hold_amd.muon import orthogonalize
    x = torch.stack([spread(kind, 600, 1600, seed=k) for k in range(3)]).to(dtype)
    for v in (x, x[:1]):
        assert float((orthogonalize(v) != orthogonalize(v.float()).to(dtype)).float().mean()) <= 1e-4
    w = iterate(x[0].cpu().double())
    assert off(orthogonalize(x)[0], w) <= 4 * off(iterate(x[0].cpu().float()), w) + torch.finfo(dtype).eps / 2

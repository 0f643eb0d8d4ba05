"""Calls of hold_amd.muon beside the optimiser: what a step tells autograd and the models, degenerate matrices, spread spectra."""
import pytest
import torch

from parity_common import ROOT  # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_a_step_is_seen_by_the_models_weight_packs():
    """muon_step on a model's own matrices between two queries of its SDF: the second answers with the new weights, as a model does that
    was given them by copy_"""
    from parity_common import hip_net, setup
    from hold_amd.muon import muon_step
    from hold_amd.optim import hidden_matrices
    sc, sd_np, _, _ = setup()
    net, twin = hip_net(sc, sd_np), hip_net(sc, sd_np)
    f, g = (n.nodes["object"].implicit_network for n in (net, twin))
    x = torch.rand(500, 3, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1)) - 0.5
    with torch.no_grad():
        before = f.sdf(x)
        ws = hidden_matrices(f)
        gen = torch.Generator(device=DEV).manual_seed(2)
        muon_step(ws, [torch.randn(w.shape, device=DEV, generator=gen) for w in ws], [torch.zeros_like(w) for w in ws], lr=0.02)
        for a, b in zip(hidden_matrices(g), ws):
            a.copy_(b)
        after = f.sdf(x)
        assert not torch.equal(after, before) and torch.equal(after, g.sdf(x))


def test_a_step_is_seen_by_autograd():
    """a parameter that a step moved between forward and backward: the backward pass refuses, as after any in-place operation"""
    from hold_amd.muon import muon_step
    p = torch.randn(40, 40, device=DEV).requires_grad_(True)
    m = torch.zeros(40, 40, device=DEV)
    y = (p @ p).sum()
    at = p._version, m._version
    muon_step([p], [torch.ones(40, 40, device=DEV)], [m], lr=0.1)
    assert p._version > at[0] and m._version > at[1]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("shape", [(20, 30), (300, 200), (700, 1200)])
def test_zeros_without_eps(shape):
    """eps = 0: a matrix of zeros stays zero beside others, an unused parameter beside a moving one; NaN stays NaN"""
    from hold_amd.muon import muon_step, orthogonalize
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.randn(3, *shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(3)).to(dtype)
        want = orthogonalize(x, eps=0.0)
        x[1] = 0
        got = orthogonalize(x, eps=0.0)
        assert not got[1].any() and torch.equal(got[::2], want[::2])
        x[1, 4, 5] = float("nan")
        assert torch.isnan(orthogonalize(x, eps=0.0)[1]).all()
    p, z = torch.ones(shape, device=DEV), torch.zeros(shape, device=DEV)
    m = z.clone()
    muon_step([p], [z], [m], lr=0.5, weight_decay=0.5, eps=0.0)
    assert torch.equal(p, torch.full_like(p, 0.75)) and not m.any()

"""Calls of hold_amd.gated.gated_linear that its documentation allows or names: views, and ways of differentiation."""
import pytest
import torch

from parity_common import ROOT  # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_forward_mode_is_refused():
    """a tangent is never dropped: a dual tensor in any place is refused, with gradients recorded or not; plain ones inside the level go on"""
    import torch.autograd.forward_ad as fa
    from hold_amd.gated import gated_linear
    for T in (5, 100):
        t = [torch.randn(s, device=DEV) for s in ((T, 24), (16, 24), (16, 24), (16,), (16,))]
        want = gated_linear(*t)
        with fa.dual_level():
            assert torch.equal(gated_linear(*t), want)
            for k in range(5):
                a = list(t)
                a[k] = fa.make_dual(t[k], torch.ones_like(t[k]))
                with pytest.raises(NotImplementedError):
                    gated_linear(*a)
                with torch.no_grad(), pytest.raises(NotImplementedError):
                    gated_linear(*a)
                a[0 if k else 1] = a[0 if k else 1].clone().requires_grad_(True)
                with pytest.raises(NotImplementedError):
                    gated_linear(*a)
            leaf = t[0].clone().requires_grad_(True)
            y = gated_linear(leaf, *t[1:])
            with pytest.raises(NotImplementedError):
                torch.autograd.grad(y, leaf, fa.make_dual(torch.ones_like(y), torch.ones_like(y)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T, D", [(3, 40), (20, 40), (70, 40), (70, 300)])
def test_row_strides_beyond_2_to_the_21(T, D, dtype):
    """a slice of wide rows: more than 2^21 elements from one row to the next, for the input, either weight and the result's gradient"""
    from hold_amd.gated import gated_linear
    gen = torch.Generator().manual_seed(4)
    t = [torch.randn(s, generator=gen).to(dtype).to(DEV) for s in ((T, D), (9, D), (9, D))]
    dh = torch.randn(T, 9, generator=gen).to(dtype).to(DEV)

    def far(v):
        w = torch.empty_strided(v.shape, ((1 << 21) + 8, 1), dtype=dtype, device=DEV)
        return w.copy_(v)

    plain = [v.clone().requires_grad_(True) for v in t]
    h = gated_linear(*plain)
    want = torch.autograd.grad(h, plain, dh)
    for k in range(4):
        views = [(far(v) if i == k else v.clone()).requires_grad_(True) for i, v in enumerate(t)]
        y = gated_linear(*views)
        assert torch.equal(y, h)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, views, far(dh) if k == 3 else dh), want))

"""hold_amd.gated.gated_linear refuses a dual tensor before anything is computed: its tangent would be lost (no GPU)."""
import pytest
import torch

from parity_common import ROOT  # noqa: F401


@pytest.mark.parametrize("k", range(5))
@pytest.mark.parametrize("grad", [True, False])
def test_a_tangent_is_refused(k, grad):
    import torch.autograd.forward_ad as fa
    from hold_amd.gated import gated_linear
    t = [torch.zeros(s) for s in ((3, 4), (8, 4), (8, 4), (8,), (8,))]
    with torch.set_grad_enabled(grad), fa.dual_level():
        with pytest.raises(ValueError):  # none has a tangent: on the CPU
            gated_linear(*t)
        t[k] = fa.make_dual(t[k], torch.ones_like(t[k]))
        with pytest.raises(NotImplementedError):
            gated_linear(*t)

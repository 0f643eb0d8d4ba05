"""What hold_amd.muon refuses, and the host side of its entry points (no GPU)."""
import ctypes as C

import pytest
import torch

from parity_common import ROOT  # noqa: F401


@pytest.mark.parametrize("x, kw, error", [
    (torch.zeros(4), {}, ValueError),
    (torch.zeros(4, 4, dtype=torch.float64), {}, TypeError),
    (torch.zeros(4, 4, dtype=torch.int32), {}, TypeError),
    (torch.zeros(4, 4), dict(steps=0), ValueError),
    (torch.zeros(4, 4), dict(steps=33), ValueError),
    (torch.zeros(4, 4), dict(steps=2.0), ValueError),
    (torch.zeros(4, 4), dict(coefficients=(1.0, 2.0)), ValueError),
    (torch.zeros(4, 4), dict(steps=2, coefficients=[(1.0, 2.0, 3.0)]), ValueError),
    (torch.zeros(4, 4), dict(steps=2, coefficients=[(1.0, 2.0, 3.0), (1.0, 2.0)]), ValueError),
    (torch.zeros(4, 4), dict(eps=-1.0), ValueError),
    (torch.zeros(4, 4), dict(eps=float("nan")), ValueError),
    (torch.zeros(1, 1).expand(2, (1 << 20) + 1), {}, ValueError),
    (torch.zeros(1, 1, 1).expand((1 << 24) + 1, 1, 1), {}, ValueError),
    (torch.zeros(4, 4), {}, ValueError),  # on the CPU: there is no fallback
])
def test_orthogonalize_refuses(x, kw, error):
    from hold_amd.muon import orthogonalize
    with pytest.raises(error):
        orthogonalize(x, **kw)


@pytest.mark.parametrize("kw, error", [
    (dict(grads=[]), ValueError),
    (dict(params=[torch.zeros(3)], grads=[torch.zeros(3)], momenta=[torch.zeros(3)]), ValueError),
    (dict(grads=[torch.zeros(3, 5)]), ValueError),
    (dict(momenta=[torch.zeros(4, 3)]), ValueError),
    (dict(grads=[torch.zeros(3, 4, dtype=torch.bfloat16)]), TypeError),
    (dict(lr=-1.0), ValueError),
    (dict(lr=float("inf")), ValueError),
    (dict(momentum=1.0), ValueError),
    (dict(momentum=-0.1), ValueError),
    (dict(weight_decay=-1.0), ValueError),
    (dict(clip_norm=float("nan")), ValueError),
    (dict(grad_mul=float("nan")), ValueError),
    (dict(scale="other"), ValueError),
    (dict(scale=True), ValueError),
    (dict(steps=0), ValueError),
    (dict(), ValueError),  # on the CPU
])
def test_muon_step_refuses(kw, error):
    from hold_amd.muon import muon_step
    a = dict(params=[torch.zeros(3, 4)], grads=[torch.zeros(3, 4)], momenta=[torch.zeros(3, 4)], lr=0.1)
    a.update(kw)
    with pytest.raises(error):
        muon_step(**a)


def test_update_scale():
    from hold_amd.muon import update_scale
    assert update_scale(512, 128, "spectral") == 2.0 and update_scale(128, 512, "spectral") == 1.0
    assert update_scale(400, 100, "rms") == 4.0 and update_scale(3, 4, 0.5) == 0.5


def test_shared_memory_is_found():
    """the check of a step's tensors: whole matrices, overlapping ones, interleaved columns of one wider matrix"""
    from hold_amd.muon import shares_memory
    base = torch.zeros(8, 40)
    a, b, c = base[:, :16], base[:, 16:40], base[:, 10:20]
    assert not shares_memory([a, b], [torch.zeros(8, 16)])
    assert shares_memory([a, c], []) and shares_memory([a, a], []) and shares_memory([base, b], [])
    assert shares_memory([a], [c]) and shares_memory([a], [base]) and not shares_memory([a], [b, b])
    assert not shares_memory([base[:4], base[4:]], [])
    assert shares_memory([base[:5], base[4:]], [])
    assert not shares_memory([torch.zeros(1, 5), torch.zeros(1, 5)], [])


def _ortho(**kw):
    from hold_amd._lib import OrthoDesc
    coef = (C.c_float * 96)(*([3.4445, -4.7750, 2.0315] * 32))
    d = OrthoDesc()
    d.x, d.out, d.coef, d.workspace, d.workspace_bytes = 4096, 8192, C.cast(coef, C.POINTER(C.c_float)), 0, 0  # never a launch: no workspace
    d.batch, d.rows, d.cols, d.dtype, d.steps, d.eps = 2, 200, 300, 0, 5, 1e-7
    for k, v in kw.items():
        setattr(d, k, v)
    d._keep = coef
    return d


def test_entry_points_refuse_bad_descriptors():
    from hold_amd import _lib, build
    build.build()
    L, n = _lib.lib(), C.c_int64()
    assert L.hold_orthogonalize_workspace(C.byref(_ortho()), C.byref(n)) == 0 and n.value > 2 * 200 * 300 * 8
    need = n.value
    for bad in (dict(batch=0), dict(rows=0), dict(cols=0), dict(rows=(1 << 20) + 1), dict(batch=(1 << 24) + 1)):
        assert L.hold_orthogonalize_workspace(C.byref(_ortho(**bad)), C.byref(n)) == -1
    assert L.hold_orthogonalize_workspace(C.byref(_ortho()), None) == -1
    for bad in (dict(), dict(workspace=4096, workspace_bytes=need - 1)):  # no workspace, too small a one
        assert L.hold_orthogonalize(C.byref(_ortho(**bad)), None) == -1
    room = dict(workspace=4096, workspace_bytes=need)
    for bad in (dict(x=0), dict(out=0), dict(steps=0), dict(steps=33), dict(dtype=3), dict(dtype=-1), dict(eps=-1.0), dict(eps=float("nan"))):
        assert L.hold_orthogonalize(C.byref(_ortho(**room, **bad)), None) == -1, bad
    for triple in ((1e12, 0.0, 0.0), (float("nan"), 0.0, 0.0), (0.0, 0.0, 0.0), (1e-12, 0.0, 0.0), (400.0, 0.0, 0.0)):  # the last: 400^5
        coef = (C.c_float * 15)(*(triple * 5))
        assert L.hold_orthogonalize(C.byref(_ortho(**room, coef=C.cast(coef, C.POINTER(C.c_float)))), None) == -1, triple
    items = (_lib.MuonItem * 1)()
    i = items[0]
    i.p, i.g, i.m, i.rows, i.cols, i.ldp, i.ldg, i.ldm, i.scale = 4096, 8192, 16384, 10, 20, 20, 20, 20, 1.0
    coef = (C.c_float * 15)(*([3.4445, -4.7750, 2.0315] * 5))
    d = _lib.MuonDesc()
    d.items, d.n_items, d.coef, d.steps, d.lr = C.cast(items, C.POINTER(_lib.MuonItem)), 1, C.cast(coef, C.POINTER(C.c_float)), 5, 0.1
    assert L.hold_muon_workspace(C.byref(d), C.byref(n)) == 0 and n.value > 0
    assert L.hold_muon_step(C.byref(d), None) == -1  # no workspace
    d.workspace, d.workspace_bytes = 4096, n.value
    for name, bad in (("p", 0), ("g", 0), ("m", 0), ("rows", 0), ("ldp", 19), ("ldg", 19), ("ldm", 19)):
        keep = getattr(i, name)
        setattr(i, name, bad)
        assert L.hold_muon_step(C.byref(d), None) == -1, name
        setattr(i, name, keep)
    d.n_items = 0
    assert L.hold_muon_step(C.byref(d), None) == -1


class _Net(torch.nn.Module):
    """what the flat optimisers need of a model: .nodes[*].params (pose tables) and layers"""

    def __init__(self):
        super().__init__()
        torch.manual_seed(3)
        self.nodes = torch.nn.ModuleDict({"right": torch.nn.Module()})
        self.nodes["right"].params = torch.nn.Embedding(5, 3)
        self.first = torch.nn.Linear(3, 96)
        self.hidden = torch.nn.utils.weight_norm(torch.nn.Linear(96, 64))
        self.wide = torch.nn.Linear(64, 200, bias=False)
        self.last = torch.nn.Linear(200, 3)


def test_flat_muon_bucket_and_state():
    from hold_amd.optim import FlatAdam, FlatMuon, hidden_matrices
    net = _Net()
    assert [tuple(p.shape) for p in hidden_matrices(net)] == [(64, 96), (200, 64)]
    assert len(hidden_matrices(net, smallest=65)) == 0
    values = {n: p.detach().clone() for n, p in net.named_parameters()}
    a = FlatMuon(net, lr=1e-3, matrix_lr=0.02)
    assert all(torch.equal(p, values[n]) for n, p in net.named_parameters())  # re-homed, unchanged
    assert a.n_adam == a.offsets[-2] and [tuple(v.shape) for v in a._views(a.m)] == [(64, 96), (200, 64)]
    assert all(v.data_ptr() == p.data_ptr() for v, p in zip(a._views(a.flat), a.matrices))
    g = torch.Generator().manual_seed(1)
    a.m.copy_(torch.randn(a.m.shape, generator=g))
    a.step_count, a.momentum = 7, 0.9
    b = FlatMuon(_Net(), lr=5e-4)
    b.load_state_dict(a.state_dict())
    assert torch.equal(b.m, a.m) and (b.step_count, b.momentum, b.matrix_lr, b.lr, b.scale) == (7, 0.9, 0.02, 1e-3, "rms")
    assert set(a.named_state()) == {n for n, _ in net.named_parameters()} - {"hidden.weight_v", "wide.weight"}
    assert not any(p in a.torch_optimizer().state for p in a.matrices)
    for other in (FlatAdam(_Net(), lr=5e-4).state_dict(), FlatMuon(_Net(), lr=5e-4, matrices=[]).state_dict()):
        with pytest.raises(ValueError):
            b.load_state_dict(other)
    net = _Net()
    for bad in ([net.first.bias], [net.nodes["right"].params.weight], [torch.nn.Parameter(torch.zeros(4, 4))]):
        with pytest.raises(ValueError):
            FlatMuon(net, matrices=bad)


def test_flat_muon_finds_the_models_matrices():
    import hold_amd
    from parity_common import syn
    from hold_amd.optim import hidden_matrices
    sc = syn.make_scene(n_frames=4)
    net = hold_amd.build_from_scene(sc, syn.make_state_dict(sc), device="cpu")
    names = {id(p): n for n, p in net.named_parameters()}
    got = [names[id(p)] for p in hidden_matrices(net)]
    assert len(got) >= 30 and all(n.endswith(("weight", "weight_v")) for n in got) and not any(".params." in n for n in got)

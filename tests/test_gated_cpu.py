"""What hold_amd.gated.gated_linear refuses, and the host side of its entry points (no GPU)."""
import ctypes as C

import pytest
import torch

from parity_common import ROOT  # noqa: F401


def _t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("kw, error", [
    (dict(activation="tanh"), ValueError),
    (dict(w_up=_t(7, 4)), ValueError),                      # two widths
    (dict(x=_t(3, 5)), ValueError),                         # another number of features
    (dict(x=torch.zeros(())), ValueError),
    (dict(w_gate=_t(8, 4, 1), w_up=_t(8, 4, 1)), ValueError),
    (dict(b_gate=_t(7)), ValueError),
    (dict(b_up=_t(1, 8)), ValueError),
    (dict(x=_t(3, 0), w_gate=_t(8, 0), w_up=_t(8, 0)), ValueError),
    (dict(x=_t(3, 4, dtype=torch.bfloat16)), TypeError),    # mixed types
    (dict(b_gate=_t(8, dtype=torch.bfloat16)), TypeError),
    (dict(x=_t(3, 4, dtype=torch.float64), w_gate=_t(8, 4, dtype=torch.float64), w_up=_t(8, 4, dtype=torch.float64)), TypeError),
    (dict(x=_t(3, 4, dtype=torch.float16), w_gate=_t(8, 4, dtype=torch.float16), w_up=_t(8, 4, dtype=torch.float16)), TypeError),
    (dict(w_gate=_t(1, 4).expand((1 << 21) + 1, 4), w_up=_t(1, 4).expand((1 << 21) + 1, 4)), ValueError),
    (dict(), ValueError),                                   # on the CPU: there is no fallback
])
def test_gated_linear_refuses(kw, error):
    from hold_amd.gated import gated_linear
    a = dict(x=_t(3, 4), w_gate=_t(8, 4), w_up=_t(8, 4))
    a.update(kw)
    with pytest.raises(error):
        gated_linear(**a)


def _desc(T=100, D=64, H=48, dtype=0, act=0, **kw):
    from hold_amd._lib import GatedDesc
    d = GatedDesc()
    d.x, d.w_gate, d.w_up = 4096, 8192, 16384  # never read: every call here ends before a launch
    d.ldx = d.ldwg = d.ldwu = D
    d.T, d.D, d.H, d.dtype, d.act = T, D, H, dtype, act
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_entry_points_refuse_bad_descriptors():
    from hold_amd import _lib, build
    build.build()
    L = _lib.lib()
    n = C.c_int64(-1)
    assert L.hold_gated_workspace(C.byref(_desc()), 1, C.byref(n)) == 0 and n.value > 0
    need = n.value
    for bad in (dict(T=0), dict(T=-1), dict(D=0), dict(H=0), dict(dtype=2), dict(act=4), dict(act=-1), dict(x=0), dict(w_gate=0), dict(w_up=0),
                dict(ldx=63), dict(ldwg=63), dict(ldwu=63), dict(ldx=(1 << 21) + 1), dict(H=(1 << 21) + 1), dict(T=(1 << 31) + 1),
                dict(T=1 << 30), dict(H=1 << 20, D=1 << 20, ldx=1 << 20, ldwg=1 << 20, ldwu=1 << 20)):
        assert L.hold_gated_workspace(C.byref(_desc(**bad)), 1, C.byref(n)) == -1, bad
        assert L.hold_gated_fwd(C.byref(_desc(**{"h": 4096, "ldh": 1 << 22, **bad})), None) == -1, bad
    assert L.hold_gated_workspace(C.byref(_desc()), 1, None) == -1
    assert L.hold_gated_fwd(C.byref(_desc(workspace=4096, workspace_bytes=1 << 40)), None) == -1                  # no result
    assert L.hold_gated_fwd(C.byref(_desc(h=4096, ldh=47, workspace=4096, workspace_bytes=1 << 40)), None) == -1  # rows overlap
    assert L.hold_gated_fwd(C.byref(_desc(h=4096, ldh=48, D=300)), None) == -1                                    # no workspace
    full = dict(dh=4096, lddh=48, dx=4096, dw_gate=4096, dw_up=4096)
    assert L.hold_gated_bwd(C.byref(_desc(**{**full, "dh": 0}, workspace=4096, workspace_bytes=1 << 40)), None) == -1
    assert L.hold_gated_bwd(C.byref(_desc(**{**full, "dw_up": 0}, workspace=4096, workspace_bytes=1 << 40)), None) == -1
    assert L.hold_gated_bwd(C.byref(_desc(**full, workspace=4096, workspace_bytes=need - 1)), None) == -1
    for out in ("dx", "dw_gate", "dw_up"):  # not on a 16-byte boundary
        assert L.hold_gated_bwd(C.byref(_desc(**{**full, out: 4100}, workspace=4096, workspace_bytes=1 << 40)), None) == -1
    # what is kept for a backward call: nothing for few rows, short ones or little work; a buffer that is not wanted, or not aligned
    for want, kw in ((0, dict(T=64, H=1 << 17, D=300)), (0, dict(T=70000, D=256)), (0, dict(T=4000, D=300)), (0, dict(T=70000, D=512, dtype=1)),
                     (70000 * 48 * 8, dict(T=70000, D=257)), (70000 * 48 * 6, dict(T=70000, H=41, D=513, dtype=1))):
        kw = dict(ldx=1 << 10, ldwg=1 << 10, ldwu=1 << 10, **kw)
        assert L.hold_gated_kept(C.byref(_desc(**kw)), C.byref(n)) == 0 and n.value == want, kw
        if not want:
            assert L.hold_gated_workspace(C.byref(_desc(**kw, kept=4096)), 1, C.byref(n)) == -1
    assert L.hold_gated_fwd(C.byref(_desc(T=70000, D=300, kept=4104, h=4096, ldh=48, workspace=4096, workspace_bytes=1 << 40)), None) == -1
    assert L.hold_gated_kept(C.byref(_desc(D=0)), C.byref(n)) == -1 and L.hold_gated_kept(C.byref(_desc()), None) == -1
    # few rows and short ones need no scratch forward; the sizes grow with the rows
    assert L.hold_gated_workspace(C.byref(_desc()), 0, C.byref(n)) == 0 and n.value == 0
    assert L.hold_gated_workspace(C.byref(_desc(T=64, D=300)), 0, C.byref(n)) == 0 and n.value == 0
    assert L.hold_gated_workspace(C.byref(_desc(T=65, D=300)), 0, C.byref(n)) == 0 and n.value >= 65 * 300 * 4

"""The gated layer ``h = act(x Wg^T + bg) * (x Wu^T + bu)`` as one kernel with its backward pass (csrc/gated.hip).

It stands beside the framework's other single-layer products (hold_amd.gemm: linear + activation), for hidden layers whose activation
is a second projection's gate.  ``gated_linear`` takes weights in ``nn.Linear``'s layout [H, D]; the four activations of the gate are
``silu``, ``gelu`` (the exact one, by erf), ``relu`` and ``sigmoid``.

Arithmetic: float32 tensors through two-limb fp16 products with float32 accumulation (errors of float32's own size), bfloat16 tensors
through bf16 products with float32 accumulation, rounded once at the end; in the backward pass of bfloat16, dL/dg and dL/du are rounded
to bfloat16 once as operands of the next products.  Results do not depend on the other rows of a batch, except that above 64 rows
another kernel (of the same accuracy) computes them.  The backward pass computes the projections again instead of keeping them: a call
keeps its inputs only.  All sums have a fixed order.
"""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import GatedDesc, check, ptr, stream_ptr

ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2, "sigmoid": 3}
_DTYPES = {torch.float32: 0, torch.bfloat16: 1}


def _rows(t):
    """[..., n] as [rows, n] with a unit inner stride and a positive row stride of at least n (copied where it is not so already)"""
    t = t.reshape(-1, t.shape[-1])
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        t = t.contiguous()
    return t


def _ld(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _descriptor(x, w_gate, w_up, b_gate, b_up, act):
    d = GatedDesc()
    d.x, d.ldx = ptr(x), _ld(x)
    d.w_gate, d.ldwg, d.w_up, d.ldwu = ptr(w_gate), _ld(w_gate), ptr(w_up), _ld(w_up)
    d.b_gate, d.b_up = ptr(b_gate), ptr(b_up)
    d.T, d.D, d.H, d.dtype, d.act = x.shape[0], x.shape[1], w_gate.shape[0], _DTYPES[x.dtype], act
    return d


def _launch(d, backward, device, what):
    L = _lib.lib()
    n = C.c_int64()
    if L.hold_gated_workspace(C.byref(d), 1 if backward else 0, C.byref(n)) != 0:
        raise ValueError(f"{what}: a size is out of range (T = {d.T}, D = {d.D}, H = {d.H}, strides {d.ldx}, {d.ldwg}, {d.ldwu})")
    # of the allocator's own pool for the current stream (and of a capture's pool while one is recorded): calls share no scratch
    ws = torch.empty(max(n.value, 1), dtype=torch.uint8, device=device)
    d.workspace, d.workspace_bytes = ptr(ws), n.value
    fn = L.hold_gated_bwd if backward else L.hold_gated_fwd
    check(fn(C.byref(d), stream_ptr()), what)


class _GatedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, act):
        ctx.save_for_backward(x, w_gate, w_up, b_gate, b_up)
        ctx.act = act
        H = w_gate.shape[0]
        h = torch.empty(*x.shape[:-1], H, dtype=x.dtype, device=x.device)
        if h.numel():
            x2, wg, wu = _rows(x), _rows(w_gate), _rows(w_up)
            bg, bu = (None if b is None else b.contiguous() for b in (b_gate, b_up))
            with torch.cuda.device(x.device):
                d = _descriptor(x2, wg, wu, bg, bu, act)
                d.h, d.ldh = ptr(h), H
                _launch(d, False, x.device, "gated_linear")
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        x, w_gate, w_up, b_gate, b_up = ctx.saved_tensors
        need = ctx.needs_input_grad
        dw = need[1] or need[2]
        new = lambda t, wanted: torch.empty(t.shape, dtype=t.dtype, device=t.device) if t is not None and wanted else None  # noqa: E731
        out = [new(x, need[0]), new(w_gate, dw), new(w_up, dw), new(b_gate, need[3]), new(b_up, need[4])]
        if dh.numel():
            x2, wg, wu, dh2 = _rows(x), _rows(w_gate), _rows(w_up), _rows(dh)
            bg, bu = (None if b is None else b.contiguous() for b in (b_gate, b_up))
            with torch.cuda.device(x.device):
                d = _descriptor(x2, wg, wu, bg, bu, ctx.act)
                d.dh, d.lddh = ptr(dh2), _ld(dh2)
                d.dx, d.dw_gate, d.dw_up, d.db_gate, d.db_up = (ptr(t) for t in out)
                _launch(d, True, x.device, "gated_linear (backward)")
        else:
            for t in out:
                if t is not None:
                    t.zero_()
        return out[0], out[1] if need[1] else None, out[2] if need[2] else None, out[3], out[4], None


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, activation="silu"):
    """``act(x @ w_gate.T + b_gate) * (x @ w_up.T + b_up)``: x [..., D], w_gate and w_up [H, D], biases [H] or None -> [..., H].

    All tensors on one GPU and of one type, float32 or bfloat16.  Differentiable once in every tensor.  Up to 64 rows go through a
    kernel for few rows that reads the weights as they are, once; more through the matrix cores."""
    if activation not in ACTIVATIONS:
        raise ValueError(f"gated_linear: activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
    if x.dim() < 1 or w_gate.dim() != 2 or w_up.shape != w_gate.shape or x.shape[-1] != w_gate.shape[1]:
        raise ValueError(f"gated_linear: x [..., D] and two weights [H, D] are wanted, got {tuple(x.shape)}, {tuple(w_gate.shape)}, {tuple(w_up.shape)}")
    if w_gate.shape[1] == 0:
        raise ValueError("gated_linear: at least one input feature is wanted")
    given = {"x": x, "w_gate": w_gate, "w_up": w_up, "b_gate": b_gate, "b_up": b_up}
    for name, t in given.items():
        if t is None:
            continue
        if name.startswith("b_") and tuple(t.shape) != (w_gate.shape[0],):
            raise ValueError(f"gated_linear: {name} must have shape ({w_gate.shape[0]},), got {tuple(t.shape)}")
        if t.dtype != x.dtype or t.dtype not in _DTYPES:
            raise TypeError(f"gated_linear: float32 or bfloat16 throughout is wanted, got {name} of {t.dtype} beside x of {x.dtype}")
    for name, t in given.items():
        if t is not None and (t.device != x.device or not t.is_cuda):
            raise ValueError(f"gated_linear: all tensors have to be on one GPU, got {name} on {t.device}, x on {x.device}")
    return _GatedFn.apply(x, w_gate, w_up, b_gate, b_up, ACTIVATIONS[activation])

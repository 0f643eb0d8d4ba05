"""The gated layer ``h = act(x Wg^T + bg) * (x Wu^T + bu)`` as one kernel with its backward pass (csrc/gated.hip).

It stands beside the framework's other single-layer products (hold_amd.gemm: linear + activation), for hidden layers whose activation
is a second projection's gate.  ``gated_linear`` takes weights in ``nn.Linear``'s layout [H, D]; the four activations of the gate are
``silu``, ``gelu`` (the exact one, by erf), ``relu`` and ``sigmoid``.

Arithmetic: float32 tensors through float32 products and sums on the matrix cores, whatever the values' range; bfloat16 tensors through
bf16 products with float32 accumulation, rounded once at the end; in the backward pass of bfloat16, dL/dg and dL/du are rounded to
bfloat16 once as operands of the next products.  Infinities and NaN come out where the formula has them.  Results do not depend on the
other rows of a batch, except that up to 4 and up to 64 rows other kernels (of the same accuracy) compute them.  All sums have a fixed
order.

For a backward pass a call keeps its inputs, and u act'(g) and act(g) where reading them is less time than computing them again
(float32: more than 256 features and 2^21 results, or more than 128 and 2^23; bfloat16: more than 512 and 2^21): 8 bytes a result in
float32, 6 in bfloat16.
"""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import GatedDesc, check, stream_ptr

ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2, "sigmoid": 3}
_DTYPES = {torch.float32: 0, torch.bfloat16: 1}
MAX_WIDTH = 1 << 21
_SHORT = 128  # up to so many features nothing is kept for the backward pass


def _rows(t, most=MAX_WIDTH):
    """[..., n] as [rows, n] with a unit inner stride and a row stride of n to ``most`` (copied where it is not so already)"""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if not t.is_contiguous():
        rows, n = t.shape
        ld, inner = t.stride()
        if n > 1 and inner != 1 or rows > 1 and not n <= ld <= most:
            t = t.contiguous()
    return t


def _call(act, x, w_gate, w_up, b_gate, b_up, h, dh, out, kept):
    """one launch sequence on the current stream: the forward pass into ``h`` (``kept``: True where a backward pass may follow; returns
    what that one needs), or the backward pass from ``dh`` and ``kept`` into ``out``"""
    x, w_gate, w_up = _rows(x), _rows(w_gate), _rows(w_up)
    T, D = x.shape
    H = w_gate.shape[0]
    d = GatedDesc()
    d.x, d.w_gate, d.w_up = x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr()
    d.ldx, d.ldwg, d.ldwu = x.stride(0) if T > 1 else D, w_gate.stride(0) if H > 1 else D, w_up.stride(0) if H > 1 else D
    if b_gate is not None:
        b_gate = b_gate.contiguous()
        d.b_gate = b_gate.data_ptr()
    if b_up is not None:
        b_up = b_up.contiguous()
        d.b_up = b_up.data_ptr()
    d.T, d.D, d.H, d.dtype, d.act = T, D, H, _DTYPES[x.dtype], act
    if dh is None:
        d.h, d.ldh = h.data_ptr(), H
    else:
        dh = _rows(dh, 1 << 62)
        d.dh, d.lddh = dh.data_ptr(), dh.stride(0) if T > 1 else H
        d.dx, d.dw_gate, d.dw_up, d.db_gate, d.db_up = (None if t is None else t.data_ptr() for t in out)
    L, n, what = _lib.lib(), C.c_int64(0), "gated_linear" if dh is None else "gated_linear (backward)"
    if kept is True:
        kept = None
        if D > _SHORT and L.hold_gated_kept(C.byref(d), C.byref(n)) == 0 and n.value:
            kept = torch.empty(n.value, dtype=torch.uint8, device=x.device)
    if kept is not None:
        d.kept = kept.data_ptr()
    if L.hold_gated_workspace(C.byref(d), 0 if dh is None else 1, C.byref(n)) != 0:
        raise ValueError(f"{what}: a size is out of range (T = {T}, D = {D}, H = {H}, strides {d.ldx}, {d.ldwg}, {d.ldwu})")
    if n.value:
        # from the allocator's pool of the current stream (of a capture's while one is recorded): calls share no scratch
        ws = torch.empty(n.value, dtype=torch.uint8, device=x.device)
        d.workspace, d.workspace_bytes = ws.data_ptr(), n.value
    check((L.hold_gated_fwd if dh is None else L.hold_gated_bwd)(C.byref(d), stream_ptr()), what)
    return kept


def _on(device, *args):
    """_call with the tensors' device as the current one"""
    if device.index == torch.cuda.current_device():
        return _call(*args)
    with torch.cuda.device(device):
        return _call(*args)


def _forward(x, w_gate, w_up, b_gate, b_up, act, keep=None):
    h = torch.empty(*x.shape[:-1], w_gate.shape[0], dtype=x.dtype, device=x.device)
    return h, _on(x.device, act, x, w_gate, w_up, b_gate, b_up, h, None, None, keep) if h.numel() else None


def _no_tangents(*tensors):
    """a dual tensor has no requires_grad to be seen by: it is refused, its tangent would be lost"""
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("gated_linear: forward-mode differentiation is not offered")


class _GatedFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, act):
        h, kept = _forward(x, w_gate, w_up, b_gate, b_up, act, True)
        ctx.save_for_backward(x, w_gate, w_up, b_gate, b_up, kept)
        ctx.act = act
        return h

    @staticmethod
    @once_differentiable
    def backward(ctx, dh):
        _no_tangents(dh)
        *given, kept = ctx.saved_tensors
        need = list(ctx.needs_input_grad[:5])
        need[1] = need[2] = need[1] or need[2]  # the weights' gradients come together
        out = [torch.empty(t.shape, dtype=t.dtype, device=t.device) if n else None for t, n in zip(given, need)]
        if dh.numel():
            _on(dh.device, ctx.act, *given, None, dh, out, kept)
        else:
            for t in out:
                if t is not None:
                    t.zero_()
        return (*(t if n else None for t, n in zip(out, ctx.needs_input_grad)), None)


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, activation="silu"):
    """``act(x @ w_gate.T + b_gate) * (x @ w_up.T + b_up)``: x [..., D], w_gate and w_up [H, D], biases [H] or None -> [..., H].

    All tensors on one GPU and of one type, float32 or bfloat16.  Differentiable once in every tensor, in reverse mode (a tensor
    with a forward-mode tangent is refused).  Up to 64 rows go through a kernel for few rows that reads the weights as they are,
    once; more through the tiled ones.  A captured training step takes its gradients by ``torch.autograd.grad``, or by ``backward``
    while no eager graph of the same leaves lives (autograd would otherwise make the capture wait for the eager graph's stream)."""
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"gated_linear: activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
    shape, dtype, device = w_gate.shape, x.dtype, x.device
    if x.dim() < 1 or len(shape) != 2 or w_up.shape != shape or x.shape[-1] != shape[1]:
        raise ValueError(f"gated_linear: x [..., D] and two weights [H, D] are wanted, got {tuple(x.shape)}, {tuple(shape)}, {tuple(w_up.shape)}")
    if shape[1] == 0 or max(shape) > MAX_WIDTH:
        raise ValueError(f"gated_linear: 1 to {MAX_WIDTH} input features and at most as many results are taken, got weights of {tuple(shape)}")
    tensors = [x, w_gate, w_up]
    for name, b in (("b_gate", b_gate), ("b_up", b_up)):
        if b is not None:
            if b.shape != shape[:1]:
                raise ValueError(f"gated_linear: {name} must have shape ({shape[0]},), got {tuple(b.shape)}")
            tensors.append(b)
    if dtype not in _DTYPES or any(t.dtype is not dtype for t in tensors):
        raise TypeError(f"gated_linear: float32 or bfloat16 throughout is wanted, got {[str(t.dtype) for t in tensors]}")
    _no_tangents(*tensors)
    if device.type != "cuda" or any(t.device != device for t in tensors):
        raise ValueError(f"gated_linear: all tensors have to be on one GPU, got {[str(t.device) for t in tensors]}")
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        return _GatedFn.apply(x, w_gate, w_up, b_gate, b_up, act)
    return _forward(x, w_gate, w_up, b_gate, b_up, act)[0]

"""Orthogonalised updates for weight matrices (csrc/muon.hip).

``orthogonalize`` brings all singular values of a matrix near one by a polynomial iteration (K. Jordan et al., "Muon: an optimizer for
hidden layers in neural networks", 2024, whose coefficients are the default), ``muon_step`` is the momentum step that moves weight
matrices by such a matrix; ``hold_amd.optim.FlatMuon`` runs it over a model's hidden matrices beside Adam for everything else.

Inside, matrices are kept in two fp16 limbs (2^-22 of the largest value) and multiplied with float32 accumulation whatever the
input's type: the iteration multiplies the smallest singular values by up to a^steps (485 by default), and the rounding errors
with them.  The iteration is one for updates and results of every type; its error is of float32's own size in the matrix's norm, and a
16-bit result is rounded once, at the end.
"""
from __future__ import annotations

import ctypes as C
import struct

import torch

from . import _lib, config
from ._lib import MuonDesc, MuonItem, OrthoDesc, check, ptr, stream_ptr

#: (a, b, c) of  s -> a s + b s^3 + c s^5
QUINTIC = (3.4445, -4.7750, 2.0315)
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_STEPS, MAX_DIM, MAX_BATCH = 32, 1 << 20, 1 << 24


def _coefficients(coefficients, steps, what):
    """(a, b, c) for every step -> a ctypes array of 3 steps floats"""
    if not isinstance(steps, int) or isinstance(steps, bool) or not 1 <= steps <= MAX_STEPS:
        raise ValueError(f"{what}: steps must be a whole number from 1 to {MAX_STEPS}, got {steps!r}")
    c = [tuple(v) if hasattr(v, "__len__") else v for v in coefficients]
    if len(c) == 3 and not any(isinstance(v, tuple) for v in c):
        c = [tuple(c)] * steps
    if len(c) != steps or not all(isinstance(v, tuple) and len(v) == 3 for v in c):
        raise ValueError(f"{what}: coefficients are (a, b, c), or one such triple for each of the {steps} steps")
    return (C.c_float * (3 * steps))(*[float(x) for v in c for x in v])


def _eps(eps, what):
    if not 0.0 <= float(eps) < float("inf"):
        raise ValueError(f"{what}: eps must be finite and not negative, got {eps!r}")
    return float(eps)


def _diverges(what):
    return ValueError(f"{what}: the coefficients are out of range (the bound on the largest singular value has to stay between 1e-9 and "
                      "1e9 through the steps)")


@torch.no_grad()
def orthogonalize(x, steps=5, coefficients=QUINTIC, eps=1e-7):
    """The iteration X <- a X + (b A + c A A) X, A = X X^T, from x / (|x|_F + eps), for every matrix of x [..., rows, cols].

    x: float32, bfloat16 or float16 on the GPU; returns a new contiguous tensor of its shape and type.  ``coefficients``: (a, b, c), or a
    list with one such triple for each step.  A matrix of zeros stays zero; one with an infinity or NaN in it becomes NaN.  Not
    differentiable."""
    what = "orthogonalize"
    coef = _coefficients(coefficients, steps, what)
    if x.dim() < 2:
        raise ValueError(f"{what}: a matrix or a batch of matrices is wanted, got shape {tuple(x.shape)}")
    if x.dtype not in _DTYPES:
        raise TypeError(f"{what}: float32, bfloat16 or float16 is wanted, got {x.dtype}")
    eps = _eps(eps, what)
    rows, cols = x.shape[-2:]
    batch = x.numel() // max(rows * cols, 1)
    if rows > MAX_DIM or cols > MAX_DIM or batch > MAX_BATCH:
        raise ValueError(f"{what}: at most {MAX_BATCH} matrices of at most {MAX_DIM} on a side are taken, got shape {tuple(x.shape)}")
    if not x.is_cuda:
        raise ValueError(f"{what}: the tensor has to be on a GPU, got {x.device}")
    x = x.detach().contiguous()
    out = torch.empty_like(x)
    if not x.numel():
        return out
    d = OrthoDesc()
    d.x, d.out, d.coef = ptr(x), ptr(out), C.cast(coef, C.POINTER(C.c_float))
    d.rows, d.cols, d.batch = rows, cols, batch
    d.dtype, d.steps, d.eps = _DTYPES[x.dtype], steps, eps
    L, n = _lib.lib(), C.c_int64()
    with torch.cuda.device(x.device):
        if L.hold_orthogonalize_workspace(C.byref(d), C.byref(n)) != 0:
            raise _diverges(what)
        ws = torch.empty(n.value, dtype=torch.uint8, device=x.device)
        d.workspace, d.workspace_bytes = ptr(ws), n.value
        code = L.hold_orthogonalize(C.byref(d), stream_ptr())
        if code == -1:
            raise _diverges(what)
        check(code, "hold_orthogonalize")
    return out


def update_scale(rows, cols, scale):
    """the factor of a matrix's update: "spectral" = sqrt(max(1, rows / cols)), "rms" = 0.2 sqrt(max(rows, cols)) (the root mean square of
    an Adam step), or a number"""
    if scale == "spectral":
        return max(1.0, rows / cols) ** 0.5
    if scale == "rms":
        return 0.2 * max(rows, cols) ** 0.5
    if isinstance(scale, (int, float)) and not isinstance(scale, bool):
        return float(scale)
    raise ValueError(f'muon_step: scale must be "spectral", "rms" or a number, got {scale!r}')


def _row_stride(t, rows, cols):
    if t.is_contiguous():
        return cols
    step, inner = t.stride()
    if rows == 1:
        step = cols
    if cols > 1 and inner != 1 or not cols <= step < 1 << 31:
        raise ValueError(f"muon_step: contiguous rows are wanted, got strides {t.stride()} of shape {tuple(t.shape)}")
    return step


def _spans_overlap(spans):
    """spans: (first byte, end, only read, rows, columns, row stride) of float32 matrices.  Column slices of one wider matrix interleave
    without sharing memory: they are told apart where their row strides agree."""
    spans.sort()
    if all(a[1] <= b[0] for a, b in zip(spans, spans[1:])):
        return False
    for i, (lo, hi, read, rows, cols, ld) in enumerate(spans):
        for j in range(i + 1, len(spans)):
            lo2, _, read2, rows2, cols2, ld2 = spans[j]
            if lo2 >= hi:
                break
            if read and read2:
                continue
            if rows > 1 and rows2 > 1 and ld == ld2:
                c = (lo2 - lo) // 4 % ld
                if c >= cols and c + cols2 <= ld:
                    continue
            return True
    return False


def shares_memory(written, read):
    """whether one of the ``written`` float32 matrices (contiguous rows) shares memory with another one of them or of ``read``"""
    return _spans_overlap([(t.data_ptr(), t.data_ptr() + 4 * ((t.shape[0] - 1) * t.stride(0) + t.shape[1]), k == 1, *t.shape, t.stride(0))
                           for k, ts in enumerate((written, read)) for t in ts])


@torch.no_grad()
def muon_step(params, grads, momenta, lr, momentum=0.95, nesterov=True, weight_decay=0.0, scale="spectral", steps=5, coefficients=QUINTIC,
              eps=1e-7, grad_mul=1.0, clip_norm=0.0, sumsq=None):
    """One step for a list of float32 matrices, in place in ``params`` and ``momenta``:

        m = momentum m + (1 - momentum) f g        u = (1 - momentum) f g + momentum m  (nesterov)  or  m
        p = (1 - lr weight_decay) p - lr scale(rows, cols) orthogonalize(u)

    with f = grad_mul, clipped to a global norm where ``clip_norm`` > 0 and ``sumsq`` (a one-element device tensor with the sum of all
    gradients' squares before grad_mul) are given.  Every tensor is 2-D with contiguous rows; no two of the params and momenta may
    share memory.  All matrices of all shapes go through together, 36 a group: few launches, no host synchronisation.

    The version counters of params and momenta move as under any in-place operation, and cached weight packs of the framework's
    models become stale (hold_amd.config.bump_weights_epoch).  Neither happens where a captured graph is replayed: a program that
    replays a step calls bump_weights_epoch() itself before it uses such a model."""
    what = "muon_step"
    coef = _coefficients(coefficients, steps, what)
    params, grads, momenta = list(params), list(grads), list(momenta)
    if not len(params) == len(grads) == len(momenta):
        raise ValueError(f"{what}: as many gradients and momenta as parameters are wanted, got {len(params)}, {len(grads)}, {len(momenta)}")
    for name, v, high in (("lr", lr, float("inf")), ("momentum", momentum, 1.0), ("weight_decay", weight_decay, float("inf")), ("clip_norm", clip_norm, float("inf"))):
        if not 0.0 <= float(v) < high:
            raise ValueError(f"{what}: {name} is out of range: {v!r}")
    if not abs(float(grad_mul)) < float("inf"):
        raise ValueError(f"{what}: grad_mul has to be finite, got {grad_mul!r}")
    eps = _eps(eps, what)
    if not params:
        return
    device, every = params[0].device, params + grads + momenta
    if {t.dtype for t in every} != {torch.float32}:
        raise TypeError(f"{what}: float32 matrices are wanted, got {sorted({str(t.dtype) for t in every})}")
    flat, spans, gains = [], [], {}
    for p, g, m in zip(params, grads, momenta):
        shape = p.shape
        if len(shape) != 2 or g.shape != shape or m.shape != shape:
            raise ValueError(f"{what}: a parameter, its gradient and its momentum are 2-D and of one shape, got {[tuple(t.shape) for t in (p, g, m)]}")
        rows, cols = shape
        if not (rows and cols):
            continue
        gain = gains.get(shape)
        if gain is None:
            if rows > MAX_DIM or cols > MAX_DIM:
                raise ValueError(f"{what}: a matrix of {tuple(shape)} is larger than {MAX_DIM} on a side")
            gain = gains[shape] = update_scale(rows, cols, scale)
        ldp, ldg, ldm = _row_stride(p, rows, cols), _row_stride(g, rows, cols), _row_stride(m, rows, cols)
        ap, ag, am = p.data_ptr(), g.data_ptr(), m.data_ptr()
        flat += (ap, ag, am, rows, cols, ldp, ldg, ldm, gain)
        rows -= 1
        spans += ((ap, ap + 4 * (rows * ldp + cols), False, rows + 1, cols, ldp), (ag, ag + 4 * (rows * ldg + cols), True, rows + 1, cols, ldg),
                  (am, am + 4 * (rows * ldm + cols), False, rows + 1, cols, ldm))
    if not params[0].is_cuda or len({t.get_device() for t in every}) > 1:
        raise ValueError(f"{what}: all tensors have to be on one GPU, got {sorted({str(t.device) for t in every})}")
    if _spans_overlap(spans):
        raise ValueError(f"{what}: a parameter or momentum shares memory with another tensor of the call")
    if sumsq is not None and (sumsq.numel() != 1 or sumsq.dtype != torch.float32 or sumsq.device != device):
        raise ValueError(f"{what}: sumsq is one float32 value on {device}")
    if not flat:
        return
    d = MuonDesc()
    d.n_items = len(flat) // 9
    array = bytearray(struct.pack("<" + "QQQiiiiif" * d.n_items, *flat))  # MuonItem, laid out in one call
    d.items = C.cast((C.c_char * len(array)).from_buffer(array), C.POINTER(MuonItem))
    d.coef, d.steps, d.nesterov = C.cast(coef, C.POINTER(C.c_float)), steps, 1 if nesterov else 0
    d.lr, d.momentum, d.weight_decay, d.grad_mul, d.clip_norm, d.eps = float(lr), float(momentum), float(weight_decay), float(grad_mul), float(clip_norm), eps
    d.sumsq = ptr(sumsq)
    L, n = _lib.lib(), C.c_int64()
    with torch.cuda.device(device):
        if L.hold_muon_workspace(C.byref(d), C.byref(n)) != 0:
            raise _diverges(what)
        ws = torch.empty(n.value, dtype=torch.uint8, device=device)
        d.workspace, d.workspace_bytes = ws.data_ptr(), n.value
        code = L.hold_muon_step(C.byref(d), stream_ptr())
        if code == -1:
            raise _diverges(what)
        # written through raw pointers: autograd and the models' weight packs have to be told
        torch.autograd.graph.increment_version(params + momenta)
        config.bump_weights_epoch()
        check(code, "hold_muon_step")


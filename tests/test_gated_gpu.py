"""hold_amd.gated.gated_linear against the formula in 64 bits.

Tolerances, element by element (``bounds``).  A sum of products has an error of at most d times the sum of its terms' magnitudes:
float32 operands carry 2^-22 (two limbs) each and a product drops 2^-22, 3 * 2^-22 in all; the accumulation adds a rounding of 2^-24 per
matrix instruction of a partial sum that the magnitudes bound, up to 3 * 33000 / 32 of them here, of random sign: sqrt(3100) 2^-24 <
2^-18 -- d = 2^-18 covers both (2^-18 - 3 * 2^-22 is more than 3 standard deviations above that for the longest sum, and partial sums
stay far below the magnitudes' sum).  r is half a step of the result's type (bfloat16 2^-8, float32 2^-24), q half a step of dL/dg and
dL/du where they become operands (bfloat16 2^-8, float32 2^-22).  They propagate to first order through the formula:
  dg = dh u a'(g): |dh| (|a'| err(u) + |u| |a''| err(g)) with |a''| <= 1 (gelu 0.80, silu 0.50, sigmoid 0.10; relu 0, but a' jumps by 1
  where |g| <= err(g)), then q |dg|; du = dh a(g): |dh| |a'| err(g), then q |du|; bfloat16 keeps u a' and a in 24 bits, cut off: 2^-15;
  dx, dW: the operands' errors through the sum, d times its magnitudes, r of the result."""
import math

import pytest
import torch

from parity_common import ROOT  # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ACTS = ("silu", "gelu", "relu", "sigmoid")


def act64(g, act):
    if act == "relu":
        return torch.relu(g)
    if act == "gelu":
        return g * 0.5 * torch.erfc(-g / math.sqrt(2))
    s = torch.sigmoid(g)
    return s if act == "sigmoid" else g * s


def reference(x, wg, wu, bg, bu, act, dh=None, at="cpu"):
    """(h, its bound), [(gradient, its bound) or None]"""
    t = [None if v is None else v.detach().to(at).double() for v in (x, wg, wu, bg, bu)]
    low = x.dtype == torch.bfloat16
    d, r, q = 2.0 ** -18, 2.0 ** -8 if low else 2.0 ** -24, 2.0 ** -8 if low else 2.0 ** -22
    x_, wg_, wu_ = t[:3]
    g, u, G, U = x_ @ wg_.T, x_ @ wu_.T, x_.abs() @ wg_.abs().T, x_.abs() @ wu_.abs().T
    if t[3] is not None:
        g, G = g + t[3], G + t[3].abs()
    if t[4] is not None:
        u, U = u + t[4], U + t[4].abs()
    g.requires_grad_(True)
    a = act64(g, act)
    da, = torch.autograd.grad(a.sum(), g)
    g, a = g.detach(), a.detach()
    eg, eu, ada = d * G, d * U, da.abs() + d * G
    kink = (g.abs() <= eg).double() if act == "relu" else torch.zeros_like(g)
    h = a * u
    eh = (ada + kink) * eg * u.abs() + a.abs() * eu + (1 + ada + kink) * eg * eu + (d + r) * h.abs()
    if dh is None:
        return (h, eh), None
    dh = dh.detach().to(at).double()
    dg, du = dh * u * da, dh * a
    cut = 2.0 ** -15 if low else 0.0
    fg = dh.abs() * (ada * eu + u.abs() * ((0 if act == "relu" else 1) * eg + kink) + kink * eu) + (d + cut) * dg.abs()
    fu = dh.abs() * (ada + kink) * eg + (d + cut) * du.abs()
    qg, qu = fg * (1 + q) + q * dg.abs(), fu * (1 + q) + q * du.abs()
    out = [(dg @ wg_ + du @ wu_, qg @ wg_.abs() + qu @ wu_.abs() + d * (dg.abs() @ wg_.abs() + du.abs() @ wu_.abs())),
           (dg.T @ x_, qg.T @ x_.abs() + d * (dg.abs().T @ x_.abs())), (du.T @ x_, qu.T @ x_.abs() + d * (du.abs().T @ x_.abs()))]
    out += [None if t[3] is None else (dg.sum(0), fg.sum(0) + d * dg.abs().sum(0)), None if t[4] is None else (du.sum(0), fu.sum(0) + d * du.abs().sum(0))]
    return (h, eh), [None if v is None else (v[0], v[1] * (1 + r) + r * v[0].abs()) for v in out]


def make(T, D, H, dtype, bias, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    t = [r(T, D), r(H, D) * D ** -0.5, r(H, D) * D ** -0.5, 0.3 * r(H) if bias else None, 0.3 * r(H) if bias else None]
    return [None if v is None else v.to(dtype).to(DEV) for v in t], r(T, H).to(dtype).to(DEV)


def close(got, want, what=""):
    b, bound = want
    a = got.detach().to(b.device).double()
    assert a.shape == b.shape and bool(torch.isfinite(a).all()), what
    over = (a - b).abs() - bound * (1 + 1e-6)
    assert not bool((over > 0).any()), (what, float(over.max()), float(((a - b).abs() / bound.clamp(min=1e-300)).max()))


SIZES = [(1, 1, 1), (1, 256, 256), (3, 7, 5), (4, 129, 66), (16, 64, 200), (17, 33, 9), (64, 260, 31), (9, 1100, 20), (20, 1025, 40), (60, 2050, 17), (65, 8, 8), (65, 40, 72), (127, 64, 64),
         (129, 65, 63), (130, 256, 256), (300, 136, 520), (257, 31, 1), (200, 1, 130), (1000, 72, 24), (100, 300, 24), (128, 264, 40),
         (700, 257, 1500)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T, D, H", SIZES)
def test_matches_the_formula(T, D, H, dtype):
    from hold_amd.gated import gated_linear
    for k, act in enumerate(ACTS):
        args, dh = make(T, D, H, dtype, bias=(k + T) % 2 == 0, seed=k)
        leaves = [None if v is None else v.requires_grad_(True) for v in args]
        h = gated_linear(*leaves, activation=act)
        want, grads = reference(*args, act, dh)
        close(h, want, (act, "h"))
        live = [v for v in leaves if v is not None]
        got = iter(torch.autograd.grad(h, live, dh))
        for name, w in zip(("x", "w_gate", "w_up", "b_gate", "b_up"), grads):
            if w is not None:
                close(next(got), w, (act, name))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_short_rows_and_split_sums(dtype):
    """rows of up to 256 elements through many blocks, sums over tokens split between blocks, a ragged end in every direction"""
    from hold_amd.gated import gated_linear
    for T, D, H, act in ((33000, 72, 257, "silu"), (8321, 200, 1032, "gelu")):
        args, dh = make(T, D, H, dtype, bias=True)
        leaves = [v.requires_grad_(True) for v in args]
        h = gated_linear(*leaves, activation=act)
        want, grads = reference(*args, act, dh)
        close(h, want, "h")
        for name, a, w in zip("x w_gate w_up b_gate b_up".split(), torch.autograd.grad(h, leaves, dh), grads):
            close(a, w, name)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_large_tiles(dtype):
    """the tiles of 256 rows of every product with ragged ends: h (short and long sums), dx, and the weights' gradients; dg and du
    from what is kept, and (263 in bfloat16) computed again; a narrow layer in tiles of 128 rows"""
    from hold_amd.gated import gated_linear
    for T, D, H, act in ((32700, 263, 380, "relu"), (16300, 1020, 1019, "silu"), (2000, 2563, 2570, "gelu"), (70000, 520, 33, "sigmoid")):
        args, dh = make(T, D, H, dtype, bias=D in (1020, 520))
        leaves = [v.requires_grad_(True) for v in args if v is not None]
        h = gated_linear(*leaves, activation=act)
        want, grads = reference(*args, act, dh, at=DEV)
        close(h, want, "h")
        assert torch.equal(h, gated_linear(*[v.detach() for v in leaves], activation=act))  # where no backward pass follows
        got = torch.autograd.grad(h, leaves, dh, retain_graph=True)
        for name, a, w in zip("x w_gate w_up b_gate b_up".split(), got, grads):
            close(a, w, name)
        assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(h, leaves, dh)))


def test_gradient_agrees_with_differences():
    """central differences of the formula in 64 bits along random directions: a truncation of 1e-8 of the third derivative, and the
    kernel's own error, under 8e-6 of the gradient's norm by the bounds above times the direction's norm"""
    from hold_amd.gated import gated_linear
    for act in ("silu", "gelu", "sigmoid"):
        args, dh = make(70, 24, 40, torch.float32, bias=True, seed=3)
        leaves = [v.requires_grad_(True) for v in args]
        grads = torch.autograd.grad(gated_linear(*leaves, activation=act), leaves, dh)
        base = [v.detach().cpu().double() for v in args]
        gen = torch.Generator().manual_seed(5)
        for i, g in enumerate(grads):
            v = torch.randn(base[i].shape, generator=gen, dtype=torch.float64)
            f = lambda s: float((reference(*[b + s * v if k == i else b for k, b in enumerate(base)], act)[0][0] * dh.cpu().double()).sum())  # noqa: E731
            want = (f(1e-4) - f(-1e-4)) / 2e-4
            got = float((g.cpu().double() * v).sum())
            assert abs(got - want) <= 1e-6 * abs(want) + 8e-6 * float(g.cpu().double().norm() * v.norm()), (act, i)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_unaligned_views(dtype):
    """column slices, rows that start off a 16-byte boundary, transposed and broadcast tensors give what contiguous copies give"""
    from hold_amd.gated import gated_linear
    for T in (5, 150):
        (x, wg, wu, bg, bu), dh = make(T, 48, 40, dtype, True)
        wide = torch.full((T, 100), float("nan"), dtype=dtype, device=DEV)
        wide[:, 3:51] = x
        wgt = wg.t().contiguous().t()                       # columns contiguous
        wuw = torch.full((40, 57), float("nan"), dtype=dtype, device=DEV)
        wuw[:, 1:49] = wu
        dhw = torch.full((T, 61), float("nan"), dtype=dtype, device=DEV)
        dhw[:, 5:45] = dh
        bgw = torch.zeros(41, dtype=dtype, device=DEV)
        bgw[1:] = bg
        plain = [v.clone().requires_grad_(True) for v in (x, wg, wu, bg, bu)]
        views = [v.detach().requires_grad_(True) for v in (wide[:, 3:51], wgt, wuw[:, 1:49], bgw[1:], bu)]
        a, b = gated_linear(*plain), gated_linear(*views)
        assert torch.equal(a, b)
        for p, q in zip(torch.autograd.grad(a, plain, dh), torch.autograd.grad(b, views, dhw[:, 5:45])):
            assert torch.equal(p, q)
        # a gradient that is one broadcast value (what .sum().backward() sends)
        one = torch.ones((), dtype=dtype, device=DEV).expand(T, 40)
        for p, q in zip(torch.autograd.grad(gated_linear(*plain), plain, one), torch.autograd.grad(gated_linear(*plain), plain, one.contiguous())):
            assert torch.equal(p, q)
    # one row of input for all rows; batch axes
    x1 = torch.randn(1, 48, dtype=dtype, device=DEV).expand(70, 48)
    h = gated_linear(x1, wg, wu)
    assert torch.equal(h[0], h[69]) and gated_linear(x1.reshape(2, 5, 7, 48), wg, wu).shape == (2, 5, 7, 40)
    assert gated_linear(x[0], wg, wu).shape == (40,)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_empty(dtype):
    from hold_amd.gated import gated_linear
    for T, H in ((0, 8), (5, 0), (0, 0)):
        x, wg, wu = (torch.randn(*s, dtype=dtype, device=DEV).requires_grad_(True) for s in ((T, 16), (H, 16), (H, 16)))
        b = torch.randn(H, dtype=dtype, device=DEV).requires_grad_(True)
        h = gated_linear(x, wg, wu, b, None)
        assert h.shape == (T, H)
        for v, g in zip((x, wg, wu, b), torch.autograd.grad(h, (x, wg, wu, b), torch.zeros_like(h))):
            assert g.shape == v.shape and not g.any()


def test_magnitudes():
    """float32 rows, weights and gradients far from one, and rows of zeros: every row keeps its own relative accuracy"""
    from hold_amd.gated import gated_linear
    for T in (40, 200):
        (x, wg, wu, bg, bu), dh = make(T, 64, 72, torch.float32, False)
        scale = torch.logspace(-12, 8, T, device=DEV)[:, None]
        x, dh = x * scale, dh / scale
        x[3] = 0
        dh[5] = 0
        wg, wu = wg * 1e-9, wu * 1e12
        leaves = [v.requires_grad_(True) for v in (x, wg, wu)]
        h = gated_linear(*leaves, None, None, "silu")
        want, grads = reference(x, wg, wu, None, None, "silu", dh)
        got = torch.autograd.grad(h, leaves, dh)
        close(h, want, "h")
        for name, a, b in zip(("x", "w_gate", "w_up"), got, grads):
            close(a, b, name)
        assert not h[3].any() and not got[0][5].any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_values_that_are_not_finite_stay_in_their_rows(dtype):
    from hold_amd.gated import gated_linear
    for T in (30, 300):
        (x, wg, wu, bg, bu), dh = make(T, 40, 48, dtype, True)
        clean = gated_linear(x, wg, wu, bg, bu)
        x[7, 3], x[11, 0] = float("nan"), float("inf")
        leaves = [v.requires_grad_(True) for v in (x, wg, wu, bg, bu)]
        h = gated_linear(*leaves)
        bad = torch.zeros(T, dtype=torch.bool, device=DEV)
        bad[7] = bad[11] = True
        assert torch.equal(h[~bad], clean[~bad]) and not torch.isfinite(h[7]).any() and not torch.isfinite(h[11]).all()
        dx, dwg, dwu, dbg, dbu = torch.autograd.grad(h, leaves, dh)
        assert torch.isfinite(dx[~bad]).all() and torch.isnan(dx[7]).all()
        assert not torch.isfinite(dwg).any() and not torch.isfinite(dbu).any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_do_not_depend_on_each_other_and_runs_repeat(dtype):
    from hold_amd.gated import gated_linear
    args, dh = make(1500, 96, 160, dtype, True)
    leaves = [v.requires_grad_(True) for v in args]
    h = gated_linear(*leaves)
    g = torch.autograd.grad(h, leaves, dh)
    h2 = gated_linear(*leaves)
    assert torch.equal(h, h2) and all(torch.equal(a, b) for a, b in zip(g, torch.autograd.grad(h2, leaves, dh)))
    part = gated_linear(args[0][100:400], *args[1:])
    assert torch.equal(part, h[100:400])


def test_only_wanted_gradients():
    from hold_amd.gated import gated_linear
    args, dh = make(80, 24, 16, torch.float32, True)
    full = [v.clone().requires_grad_(True) for v in args]
    want = torch.autograd.grad(gated_linear(*full), full, dh)
    for k in range(5):
        one = [v.clone().requires_grad_(i == k) for i, v in enumerate(args)]
        gated_linear(*one).backward(dh)
        assert torch.equal(one[k].grad, want[k]) and all(v.grad is None for i, v in enumerate(one) if i != k)
    # the same tensor twice: both weights one leaf
    w = args[1].clone().requires_grad_(True)
    gated_linear(args[0], w, w).backward(dh)
    a, b = (args[1].clone().requires_grad_(True) for _ in range(2))
    gated_linear(args[0], a, b).backward(dh)
    assert torch.equal(w.grad, a.grad + b.grad)


def test_other_stream_and_captured_graph():
    """a call on another stream than the default, and a captured training step replayed with new inputs beside eager calls"""
    from hold_amd.gated import gated_linear
    for dtype, size in ((torch.float32, (520, 48, 64)), (torch.bfloat16, (520, 48, 64)), (torch.float32, (4200, 520, 510)), (torch.bfloat16, (4200, 520, 510))):
        args, dh = make(*size, dtype, True)
        leaves = [v.requires_grad_(True) for v in args]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(2):
                h = gated_linear(*leaves)
                g = torch.autograd.grad(h, leaves, dh)
        s.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            hc = gated_linear(*leaves)
            gc = torch.autograd.grad(hc, leaves, dh)
        for seed in (1, 2, 3):
            new, ndh = make(*size, dtype, True, seed=seed)
            with torch.no_grad():
                for a, b in zip(args, new):
                    a.copy_(b)
                dh.copy_(ndh)
            graph.replay()
            torch.cuda.synchronize()
            eager = [v.detach().clone().requires_grad_(True) for v in args]
            he = gated_linear(*eager)
            assert torch.equal(hc, he)
            for a, b in zip(gc, torch.autograd.grad(he, eager, dh)):
                assert torch.equal(a, b)

"""hold_amd.gated.gated_linear in float32 where features, weights and gradients of one row span many decades, and where they are not finite.

Tolerances, element by element (``bounds``): float32 products and sums round to 2^-24 of a partial sum that the terms' magnitudes M bound, n of
them for n terms, of random sign: sqrt(n / 3) 2^-24 M is one standard deviation at most, d(n) = 2^-23 sqrt(n) M is 3.4 of them.  relu is
exact, so a' is 0 or 1 and only its jump where |g| <= err(g) counts; dg = dh u a' and du = dh a round twice at most (2^-23), and the
errors go through the next sums:
  err(g) = d(D + 1) (|x| |Wg|^T + |bg|), err(u) alike;   err(h) = |u| err(g) + a err(u) + err(g) err(u) + 2^-24 |h|
  err(dg) = |dh| (a' err(u) + jump (|u| + err(u))) + 2^-23 |dg|;   err(du) = |dh| err(g) + 2^-24 |du|
  dx = dg Wg + du Wu: 2 H terms;  dW, db: T terms;  each with its operands' errors and half a step of the result."""
import pytest
import torch

from parity_common import ROOT  # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NAMES = "x w_gate w_up b_gate b_up".split()


def d(n):
    return 2.0 ** -23 * n ** 0.5


def bounds(x, wg, wu, bg, bu, dh):
    """[(h, its bound), (dx, ..), (dWg, ..), (dWu, ..), (dbg, ..), (dbu, ..)] of the relu layer, in 64 bits on the CPU"""
    x, wg, wu, bg, bu, dh = (v.detach().cpu().double() for v in (x, wg, wu, bg, bu, dh))
    (T, D), H = x.shape, wg.shape[0]
    g, u = x @ wg.T + bg, x @ wu.T + bu
    eg, eu = d(D + 1) * (x.abs() @ wg.abs().T + bg.abs()), d(D + 1) * (x.abs() @ wu.abs().T + bu.abs())
    a, da, jump = g.clamp(min=0), (g > 0).double(), (g.abs() <= eg).double()
    h, dg, du = a * u, dh * u * da, dh * a
    fg = dh.abs() * (da * eu + jump * (u.abs() + eu)) + 2.0 ** -23 * dg.abs()
    fu = dh.abs() * eg + 2.0 ** -24 * du.abs()
    out = [(h, u.abs() * eg + a * eu + eg * eu)]
    G, U = dg.abs() + fg, du.abs() + fu
    out.append((dg @ wg + du @ wu, fg @ wg.abs() + fu @ wu.abs() + d(2 * H) * (G @ wg.abs() + U @ wu.abs())))
    out += [(v.T @ x, e.T @ x.abs() + d(T) * (m.T @ x.abs())) for v, e, m in ((dg, fg, G), (du, fu, U))]
    out += [(v.sum(0), e.sum(0) + d(T) * m.sum(0)) for v, e, m in ((dg, fg, G), (du, fu, U))]
    return [(v, e + 2.0 ** -24 * v.abs()) for v, e in out]


def check(x, wg, wu, bg, bu, dh):
    from hold_amd.gated import gated_linear
    leaves = [v.detach().clone().requires_grad_(True) for v in (x, wg, wu, bg, bu)]
    h = gated_linear(*leaves, activation="relu")
    for name, a, (b, e) in zip(["h"] + NAMES, (h, *torch.autograd.grad(h, leaves, dh)), bounds(x, wg, wu, bg, bu, dh)):
        a = a.detach().cpu().double()
        assert bool(torch.isfinite(a).all()), name
        over = ((a - b).abs() - e * (1 + 1e-9)).amax()
        assert float(over) <= 0, (name, float(over), float(((a - b).abs() / e.clamp(min=1e-300)).max()))


def make(T, D, H, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    return [v.to(DEV) for v in (r(T, D), r(H, D) * D ** -0.5, r(H, D) * D ** -0.5, 0.3 * r(H), 0.3 * r(H), r(T, H))]


def decades(n, p, seed):
    """factors from 10^-p to 10^p in random order"""
    order = torch.randperm(n, generator=torch.Generator().manual_seed(seed))
    return (10.0 ** (torch.linspace(-p, p, n)))[order].to(DEV)


# the kernels for few rows, short and long sums, small tiles and others, kept and recomputed values, split sums; sizes that divide nothing
SIZES = [(1, 8, 8), (40, 300, 20), (65, 5, 9), (70, 32, 16), (130, 256, 256), (257, 31, 1), (700, 96, 60), (300, 513, 130), (200, 1024, 33),
         (1237, 517, 101), (9000, 40, 70), (4200, 520, 510)]


@pytest.mark.parametrize("T, D, H", SIZES)
def test_sums_are_float32s(T, D, H):
    check(*make(T, D, H))


@pytest.mark.parametrize("T", [40, 200])
@pytest.mark.parametrize("D, p", [(96, 5), (256, 4), (512, 5), (1024, 6)])
def test_features_over_decades(T, D, p):
    """features of 10^-p to 10^p and weights that compensate: every feature counts alike in every result"""
    x, wg, wu, bg, bu, dh = make(T, D, 48)
    s = decades(D, p, 1)
    check(x * s, wg / s, wu / s, bg, bu, dh)


@pytest.mark.parametrize("T, D, H", [(200, 1024, 96), (300, 200, 130), (4200, 520, 510)])
def test_gradients_over_decades(T, D, H):
    """units whose gradient is up to 10^8 times smaller than another's, by their dL/dh, by a row of either weight matrix, and by their token: each
    row of the weights' gradients keeps its own digits"""
    x, wg, wu, bg, bu, dh = make(T, D, H)
    s = decades(H, 4, 2)
    check(x, wg, wu, bg, bu, dh * s)
    check(x, wg, wu * s[:, None], bg, bu * s, dh)
    check(x, wg * s[:, None], wu, bg * s, bu, dh)
    t = decades(T, 4, 3)[:, None]
    check(x * t, wg, wu, bg, bu, dh / t)
    dh[:, 3] = 0
    dh[5, 7] = 1e6  # one outlier
    check(x, wg, wu, bg, bu, dh)


def kind(v):
    """0 finite, 1 inf, 2 -inf, 3 NaN"""
    v = v.detach().cpu()
    return torch.isnan(v) * 3 + torch.isposinf(v) * 1 + torch.isneginf(v) * 2


@pytest.mark.parametrize("T", [3, 30, 300])
@pytest.mark.parametrize("D", [40, 512])
def test_infinities_are_the_formulas(T, D):
    """an infinity among a row's features, or among a unit's weights, gives the infinities and NaN that the formula has, for any number of rows"""
    from hold_amd.gated import gated_linear
    from test_gated_gpu import ACTS, act64
    x, wg, wu, bg, bu, _ = make(T, D, 48)
    x[1, 0], x[2, 7] = float("inf"), float("-inf")
    wg[4, 3], wu[6, 1], wu[9, 0] = float("inf"), float("-inf"), float("nan")
    bg[11] = float("inf")
    for act in ACTS:
        t = [v.cpu().double() for v in (x, wg, wu, bg, bu)]
        want = act64(t[0] @ t[1].T + t[3], act) * (t[0] @ t[2].T + t[4])
        assert torch.equal(kind(gated_linear(x, wg, wu, bg, bu, act)), kind(want)), act

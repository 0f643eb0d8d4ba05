"""hold_amd.muon against its formulas in 64 bits.

Tolerances.  The iteration multiplies the smallest singular values, and every rounding with them, by up to a^steps, so its error in
any arithmetic depends on the matrix; what is derived is its ratio to float32's on the same matrix: every stored number carries 2^-22
(two limbs) where float32 carries 2^-24, every product 2^-22 more where float32 rounds once, and the accumulation is float32 in both:
at most 4 times float32's error in norm for matrices large enough (32 and more rows and columns) that errors average; for smaller ones
a worst case instead: a step's roundings, 25 * 2^-22 (|a| + 3 |b| + 5 |c| of the operands' 2^-22), grow by at most |p'| < 4 a step:
25 * 2^-22 * (1 + 4 + 16 + 64 + 256) < 2^-9 of the norm.  Half a step of the result's type comes on top."""
import pytest
import torch

from parity_common import ROOT  # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
QUINTIC = (3.4445, -4.7750, 2.0315)


def iterate(x, steps=5, coefficients=QUINTIC, eps=1e-7):
    """the formula in x's own type and on its device"""
    x = x.detach()
    tall = x.shape[-2] > x.shape[-1]
    x = x.transpose(-1, -2).contiguous() if tall else x
    x = x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True) + eps)
    for k in range(steps):
        a, b, c = coefficients[k] if hasattr(coefficients[0], "__len__") else coefficients
        gram = x @ x.transpose(-1, -2).contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(-1, -2) if tall else x


def make(*shape, seed=0, dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    k = max(1, min(shape[-2:]) // 8)
    low = torch.randn(*shape[:-1], k, generator=gen) @ torch.randn(*shape[:-2], k, shape[-1], generator=gen)
    return ((low + torch.randn(*shape, generator=gen)) * 1e-3).to(dtype).to(DEV)


def off(a, b):
    """2-norm of the difference over that of the value, matrix by matrix: the largest"""
    a, b = a.detach().cpu().double(), b.cpu().double()
    assert a.shape == b.shape and bool(torch.isfinite(a).all())
    d, n = torch.linalg.vector_norm(a - b, dim=(-2, -1)), torch.linalg.vector_norm(b, dim=(-2, -1))
    return float((d / n).max())


def allowed(x, **kw):
    if min(x.shape[-2:]) < 32:
        tol = 2.0 ** -9
    else:
        tol = 4 * off(iterate(x.float(), **kw), iterate(x.double(), **kw))
    return tol * (4 if joins(x) else 1) + torch.finfo(x.dtype).eps / 2


def joins(x):
    """whether a batch's steps are joined on the small side (16-bit results and updates of many wide matrices): A's errors then grow by up to
    a^2 = 12 a step where X's grow by a = 3.4, over at most two steps of a group: 12 / 3.4 < 4 times"""
    m, n = sorted(x.shape[-2:])
    return n >= 1.5 * m and m * m * n * (x.numel() // (m * n)) >= 1e9 and x.dtype != torch.float32


# the borders of the kernel for small matrices among them: (128, 160) and (32, 1024) are its largest, (128, 161), (129, 129) and (31, 1025) are not its
SHAPES = [(1, 1), (1, 7), (9, 1), (2, 3), (8, 8), (5, 64), (33, 47), (64, 64), (65, 64), (72, 130), (257, 63), (256, 256), (256, 84), (256, 304),
          (3, 31, 40), (2, 2, 100, 36), (5, 1, 1), (24, 130, 129), (128, 128), (160, 128), (128, 161), (129, 129), (32, 1024), (31, 1025), (2, 96, 250),
          (64, 512), (513, 64), (300, 17, 50)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize_matches_the_formula(shape, dtype):
    from hold_amd.muon import orthogonalize
    x = make(*shape, dtype=dtype)
    keep = x.clone()
    y = orthogonalize(x)
    assert y.dtype == dtype and y.shape == x.shape and y.is_contiguous() and torch.equal(x, keep)
    assert off(y, iterate(x.double())) <= allowed(x)
    assert torch.equal(y, orthogonalize(x))


@pytest.mark.parametrize("shape", [(1030, 1100), (2100, 520), (700, 2304), (40, 256, 256)])
def test_large_tiles(shape):
    from hold_amd.muon import orthogonalize
    for dtype in (torch.float32, torch.bfloat16):
        x = make(*shape, dtype=dtype)
        assert off(orthogonalize(x), iterate(x.double())) <= allowed(x)


def test_joined_steps():
    """wide and tall matrices large enough that steps are joined on the small side: other step counts, and a step's list in which they
    stand beside others"""
    from hold_amd.muon import muon_step, orthogonalize, update_scale
    for dtype in (torch.bfloat16, torch.float16):
        for shape in ((640, 2600), (2600, 640)):
            x = make(*shape, dtype=dtype)
            assert joins(x)
            for steps in (1, 2, 3, 5, 7):
                assert off(orthogonalize(x, steps=steps), iterate(x.double(), steps=steps)) <= allowed(x, steps=steps)
    big = (30.0, 0.0, 0.0)
    assert off(orthogonalize(x, steps=3, coefficients=big), iterate(x.double(), 3, big)) <= allowed(x, steps=3, coefficients=big)
    shapes = [(256, 256), (2600, 640), (64, 300), (640, 2600), (256, 256)]
    p, g, m = ([make(*s, seed=k + 7 * i) * (100 if i == 0 else 1) for i, s in enumerate(shapes)] for k in range(3))
    p0, m0 = [t.clone() for t in p], [t.clone() for t in m]
    muon_step(p, g, m, lr=0.05)
    for a, b, c, d, e, s in zip(p, m, p0, m0, g, shapes):
        f = update_scale(*s, "spectral")
        check_step(a, b, c, d, step64(c, e, d, 0.05, 0.95, True, 0.0, f), 0.05, f, joined=s in ((2600, 640), (640, 2600)))


# one batch for each tile size of each product (256, 192, 128 and 64 rows), most with a ragged last tile
@pytest.mark.parametrize("shape", [(36, 736, 1408), (36, 736, 800), (20, 1000, 1100), (3, 1500, 1500), (9, 736, 1408), (60, 500, 500), (2, 1900, 2900), (1, 3000, 900)])
def test_tile_sizes(shape):
    from hold_amd.muon import orthogonalize
    x = make(*shape)
    for y in (x, x.to(torch.bfloat16)):
        assert off(orthogonalize(y), iterate(y.double())) <= allowed(y)


def test_singular_values_come_near_one():
    """the polynomial in the singular values themselves: U p(..p(S)..) V^T, for full-rank and rank-deficient matrices"""
    from hold_amd.muon import orthogonalize
    for shape, rank in (((96, 200), 96), ((200, 96), 20), ((64, 64), 1)):
        gen = torch.Generator().manual_seed(2)
        x = torch.randn(shape[0], rank, generator=gen, dtype=torch.float64) @ torch.randn(rank, shape[1], generator=gen, dtype=torch.float64)
        u, s, vt = torch.linalg.svd(x, full_matrices=False)
        s = s / (s.norm() + 1e-7)
        s[rank:] = 0
        for _ in range(5):
            s = QUINTIC[0] * s + QUINTIC[1] * s ** 3 + QUINTIC[2] * s ** 5
        y = orthogonalize(x.float().to(DEV)).cpu().double()
        # x rounded to float32: 2^-24 of the norm, grown by at most a^5 = 485 in the directions behind the rank, like the roundings inside
        # (2^-22 each, 25 of them a step at most): (485 * 2^-24 + 2^-9) in the worst case
        assert float((y - (u * s) @ vt).norm() / ((u * s) @ vt).norm()) <= 485 * 2.0 ** -24 + 2.0 ** -9
        got = torch.linalg.svdvals(y)[:rank]
        assert float((got - s[:rank].sort(descending=True).values).abs().max()) <= 2.0 ** -8


def test_steps_and_coefficients():
    from hold_amd.muon import orthogonalize
    x = make(70, 90)
    for steps in (1, 2, 7, 8, 9):  # nine are too many for the kernel for small matrices
        assert off(orthogonalize(x, steps=steps), iterate(x.double(), steps=steps)) <= allowed(x, steps=steps)
    cubic = (1.5, -0.5, 0.0)
    assert off(orthogonalize(x, steps=12, coefficients=cubic), iterate(x.double(), 12, cubic)) <= allowed(x, steps=12, coefficients=cubic)
    each = [(4.0, -6.0, 3.0), (3.0, -4.0, 2.0), (1.875, -1.25, 0.375)]
    assert off(orthogonalize(x, steps=3, coefficients=each), iterate(x.double(), 3, each)) <= allowed(x, steps=3, coefficients=each)
    big = (30.0, 0.0, 0.0)  # grows: entries up to 30^3, scales follow
    assert off(orthogonalize(x, steps=3, coefficients=big), iterate(x.double(), 3, big)) <= allowed(x, steps=3, coefficients=big) + 2.0 ** -20
    for bad in ((1e4, 0.0, 0.0), (0.0, 0.0, 0.0), (float("nan"), 1.0, 1.0)):
        with pytest.raises(ValueError):
            orthogonalize(x, coefficients=bad)


def test_magnitudes_zeros_and_values_that_are_not_finite():
    from hold_amd.muon import orthogonalize
    x = make(6, 48, 40)
    want = iterate(x.double(), eps=0.0)
    for k in (-100, -60, 40, 100):  # powers of two leave the bits of the quotient: sums of squares in fp64 reach them all
        assert off(orthogonalize(x * 2.0 ** k, eps=0.0), want) <= allowed(x, eps=0.0)
    y = x.clone()
    y[1] = 0
    y[2, 3, 4] = float("nan")
    y[4, 0, 0] = float("inf")
    got = orthogonalize(y)
    assert not got[1].any() and torch.isnan(got[2]).all() and torch.isnan(got[4]).all()
    clean = orthogonalize(x)
    for k in (0, 3, 5):
        assert torch.equal(got[k], clean[k])


def test_views_empty_and_batches():
    from hold_amd.muon import orthogonalize
    x = make(5, 40, 56)
    one = torch.stack([orthogonalize(v) for v in x])
    assert torch.equal(orthogonalize(x), one)                              # a matrix does not depend on its batch
    assert torch.equal(orthogonalize(x.transpose(1, 2)).transpose(1, 2), orthogonalize(x.transpose(1, 2).contiguous()).transpose(1, 2))
    assert torch.equal(orthogonalize(x[1::2]), one[1::2])
    assert torch.equal(orthogonalize(x[:1].expand(3, 40, 56)), one[:1].expand(3, 40, 56))
    for shape in ((0, 4, 4), (4, 0), (0, 3)):
        assert orthogonalize(torch.zeros(shape, device=DEV)).shape == shape


def test_batches_in_parts():
    """more matrices than one launch takes: every one as alone, in the kernel for small ones and (nine steps) in the other"""
    from hold_amd.muon import orthogonalize
    for n, steps in (((1 << 21) + 3, 5), (9001, 9)):
        x = make(n, 3, 2)
        y = orthogonalize(x, steps=steps)
        for at in (slice(0, 5), slice(4085, 4095), slice(8170, 8180), slice(n - 5, n)):
            assert torch.equal(y[at], orthogonalize(x[at], steps=steps))


def step64(p, g, m, lr, momentum, nesterov, wd, scale, f=1.0):
    p, g, m = (t.detach().cpu().double() for t in (p, g, m))
    m = momentum * m + (1 - momentum) * f * g
    u = (1 - momentum) * f * g + momentum * m if nesterov else m
    return (1 - lr * wd) * p - lr * scale * iterate(u), m, u


def check_step(got_p, got_m, p, m, want, lr, scale, f=1.0, joined=False):
    """m: three roundings of float32 and the factor's own; p: lr scale times the iteration's error, and three roundings"""
    p64, m64, u = want
    small = 2.0 ** -9 if min(p.shape) < 32 else 4 * (4 if joined else 1) * off(iterate(u.float()), iterate(u))
    assert float((got_m.cpu().double() - m64).norm()) <= 2.0 ** -22 * float(m64.norm() + m.double().norm().cpu())
    # an error of 2^-22 in u, relative to its norm, passes the iteration like its own first rounding: inside `small`'s margin twice over
    assert float((got_p.cpu().double() - p64).norm()) <= lr * scale * 2 * small * float(iterate(u).norm()) + 2.0 ** -22 * float(p64.norm() + p.double().norm().cpu())


@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_step_matches_the_formula(nesterov):
    from hold_amd.muon import muon_step, update_scale
    shapes = [(256, 256), (256, 84), (40, 300), (1, 9), (13, 1), (64, 64), (129, 257)]
    for scale in ("spectral", "rms", 0.3):
        p, g, m = ([make(*s, seed=k + 7 * i) * (100 if i == 0 else 1) for i, s in enumerate(shapes)] for k in range(3))
        p0, m0 = [t.clone() for t in p], [t.clone() for t in m]
        muon_step(p, g, m, lr=0.05, momentum=0.9, nesterov=nesterov, weight_decay=0.1, scale=scale)
        for a, b, c, d, e, s in zip(p, m, p0, m0, g, shapes):
            f = update_scale(*s, scale)
            check_step(a, b, c, d, step64(c, e, d, 0.05, 0.9, nesterov, 0.1, f), 0.05, f)


def test_many_matrices_views_and_clipping():
    """more matrices than a group holds, of mixed shapes, as column slices of wider rows; the clip to a global norm from the device"""
    from hold_amd.muon import muon_step
    shapes = [(32 + k % 5, 33 + k % 7) for k in range(80)]
    wide = [make(r, 3 * c + 5, seed=k) for k, (r, c) in enumerate(shapes)]
    p, m = [w[:, :s[1]] for w, s in zip(wide, shapes)], [w[:, s[1]:2 * s[1]] for w, s in zip(wide, shapes)]
    g = [w[:, 2 * s[1]:3 * s[1]] for w, s in zip(wide, shapes)]
    keep = [w.clone() for w in wide]
    sumsq = sum(t.double().square().sum() for t in g).float().reshape(1)
    clip = 0.5 * float(sumsq.sqrt())
    muon_step(p, g, m, lr=0.02, clip_norm=clip, sumsq=sumsq, grad_mul=2.0)
    f = 2.0 * min(1.0, clip / (2.0 * float(sumsq.double().sqrt()) + 1e-6))
    for w, k, s in zip(wide, keep, shapes):
        c = s[1]
        assert torch.equal(w[:, 2 * c:], k[:, 2 * c:])  # the gradient and what is behind it stay
        check_step(w[:, :c], w[:, c:2 * c], k[:, :c], k[:, c:2 * c], step64(k[:, :c], k[:, 2 * c:3 * c], k[:, c:2 * c], 0.02, 0.95, True, 0.0, 1.0 if s[0] <= c else (s[0] / c) ** 0.5, f), 0.02,
                   max(1.0, s[0] / c) ** 0.5)
    before = [w.clone() for w in wide]
    for bad in (([p[0], p[0]], [g[0], g[0]], [m[0], m[0].clone()]), ([p[0]], [p[0]], [m[0]]), ([p[0]], [g[0]], [p[0]]), ([p[0]], [g[0]], [g[0]])):
        with pytest.raises(ValueError):
            muon_step(*bad, lr=0.1)
    assert all(torch.equal(a, b) for a, b in zip(wide, before))
    muon_step([], [], [], lr=0.1)
    e = torch.zeros(0, 4, device=DEV)
    muon_step([e], [e.clone()], [e.clone()], lr=0.1)


def test_other_stream_and_captured_graphs():
    """two graphs, each with its own workspace, replayed in turn with eager calls between: every replay against the eager result"""
    from hold_amd.muon import muon_step, orthogonalize
    x, p, g, m = make(3, 96, 70), make(80, 64, seed=1), make(80, 64, seed=2), make(80, 64, seed=3)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        orthogonalize(x)
        muon_step([p.clone()], [g], [m.clone()], lr=0.1)
    s.synchronize()
    a, b = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(a, stream=s):
        y = orthogonalize(x)
    with torch.cuda.graph(b, stream=s):
        muon_step([p], [g], [m], lr=0.1)
    for k in range(4):
        x.copy_(make(3, 96, 70, seed=20 + k))
        g.copy_(make(80, 64, seed=30 + k))
        p2, m2 = p.clone(), m.clone()
        a.replay()
        b.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, orthogonalize(x))
        muon_step([p2], [g], [m2], lr=0.1)
        assert torch.equal(p, p2) and torch.equal(m, m2)


class _GatedNet(torch.nn.Module):
    """two gated layers between a first and a last linear one, as a coordinate network has them; .nodes as the optimiser wants it"""

    def __init__(self):
        super().__init__()
        torch.manual_seed(4)
        self.nodes = torch.nn.ModuleDict()
        self.first = torch.nn.Linear(3, 96)
        self.gates = torch.nn.ModuleList([torch.nn.Linear(96, 128), torch.nn.Linear(128, 96)])
        self.ups = torch.nn.ModuleList([torch.nn.Linear(96, 128), torch.nn.Linear(128, 96)])
        self.last = torch.nn.Linear(96, 3)

    def forward(self, x, layer):
        h = torch.sin(self.first(x))
        for g, u in zip(self.gates, self.ups):
            h = layer(h, g.weight, u.weight, g.bias, u.bias)
        return self.last(h)


def _layer64(x, wg, wu, bg, bu):
    return torch.nn.functional.silu(x @ wg.T + bg) * (x @ wu.T + bu)


def test_gated_layers_trained_by_orthogonalised_momentum():
    """three steps of a network of gated layers under FlatMuon: every gradient against the formula's in 64 bits, every update against the
    optimiser's formulas applied to the gradients that it was given.  Gradients: float32 layers in a row, each adding some 2^-18 of
    its terms (the layer's own bound), six of them with cancellation: 2^-12 of a gradient's norm"""
    from hold_amd.gated import gated_linear
    from hold_amd.optim import FlatMuon
    net, twin = _GatedNet().to(DEV), _GatedNet().double()
    opt = FlatMuon(net, lr=1e-3, matrix_lr=0.02, momentum=0.9, weight_decay=0.01, clip_norm=0.5)
    assert len(opt.matrices) == 4
    gen = torch.Generator().manual_seed(8)
    for k in range(3):
        x, y = torch.randn(700, 3, generator=gen), torch.randn(700, 3, generator=gen)
        with torch.no_grad():
            for p, q in zip(net.parameters(), twin.parameters()):
                q.copy_(p)
        opt.zero_grad()
        ((net(x.to(DEV), gated_linear) - y.to(DEV)) ** 2).mean().backward()
        opt.gather_stray_grads()
        grads = torch.autograd.grad(((twin(x.double(), _layer64) - y.double()) ** 2).mean(), list(twin.parameters()))
        for (n, p), g in zip(net.named_parameters(), grads):
            assert float((p.grad.cpu().double() - g).norm()) <= 2.0 ** -12 * float(g.norm()), n
        before, m0, g0 = opt.flat.clone(), opt.m.clone(), opt.grad.clone()
        f = min(1.0, 0.5 / (opt.grad_norm() + 1e-6))
        opt.step()
        for p, c, d, e, m in zip(opt.matrices, opt._views(before), opt._views(m0), opt._views(g0), opt._views(opt.m)):
            s = 0.2 * max(p.shape) ** 0.5
            check_step(p.detach(), m, c, d, step64(c, e, d, 0.02, 0.9, True, 0.01, s, f), 0.02, s, f)
        n = opt.n_adam
        b1, b2 = opt.betas
        m, v = (1 - b1) * g0[:n].double() * f + b1 * m0[:n].double(), opt.v[:n].double()  # v: as the step left it
        want = before[:n].double() - 1e-3 * (m / (1 - b1 ** (k + 1))) / ((v / (1 - b2 ** (k + 1))).sqrt() + opt.eps)
        assert float((opt.flat[:n].double() - want).abs().max()) <= 1e-6 and float(opt.v[n:].abs().max()) == 0.0


def test_flat_muon_on_the_model():
    """a step of the scene's model: Adam's part has the bits of FlatAdam, the matrices those of muon_step"""
    from parity_common import hip_net, setup
    from hold_amd.muon import muon_step
    from hold_amd.optim import FlatAdam, FlatMuon
    sc, sd_np, _, _ = setup()
    a, b = hip_net(sc, sd_np, train=True), hip_net(sc, sd_np, train=True)
    muon, adam = FlatMuon(a, lr=5e-4, matrix_lr=1e-3, clip_norm=0.0), FlatAdam(b, lr=5e-4, clip_norm=0.0)
    other, names = dict(b.named_parameters()), {id(p): n for n, p in a.named_parameters()}
    assert len(muon.matrices) >= 30
    gen = torch.Generator(device=DEV).manual_seed(3)
    p, m = [t.clone() for t in muon._views(muon.flat)], [t.clone() for t in muon._views(muon.m)]
    for _ in range(2):
        muon.zero_grad()
        adam.zero_grad()
        for q in muon.params:
            q.grad.copy_(torch.randn(q.shape, device=DEV, generator=gen))
            other[names[id(q)]].grad.copy_(q.grad)
        g = [t.clone() for t in muon._views(muon.grad)]
        muon.step()
        adam.step()
        muon_step(p, g, m, lr=1e-3, scale="rms")
        for q in muon.params:
            if not any(q is o for o in muon.matrices):
                assert torch.equal(q, other[names[id(q)]]), names[id(q)]
        assert all(torch.equal(x, y) for x, y in zip(p, muon._views(muon.flat))) and all(torch.equal(x, y) for x, y in zip(m, muon._views(muon.m)))

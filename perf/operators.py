"""The cases by which the gated layer (hold_amd.gated) and the orthogonalised update (hold_amd.muon) are timed and compared.

``run`` computes an operator either in its plain form -- elementary torch operations in 32 bits -- or, with ``own`` set, through
the calls that a user makes.  ``exact`` computes the same outputs from the definitions in 64 bits."""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
QUINTIC = (3.4445, -4.7750, 2.0315)
STEPS, EPS = 5, 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01


def listed():
    return [
        # one query point through a layer of the model's width: the latency of a call
        {"name": "gated_point_fp32", "op": "gated", "T": 1, "D": 256, "H": 256, "type": "fp32", "act": "silu", "bias": True, "train": False},
        # a few rows through a wide layer while answering: bound by the weights' bytes
        {"name": "gated_rows_bf16", "op": "gated", "T": 4, "D": 4096, "H": 8192, "type": "bf16", "act": "silu", "bias": False, "train": False},
        # a chunk of sample points through a layer of the rendering net's width, while rendering
        {"name": "gated_chunk_fp32", "op": "gated", "T": 131072, "D": 256, "H": 256, "type": "fp32", "act": "relu", "bias": True, "train": False},
        # the same kind of layer in a training step: the result and every gradient
        {"name": "gated_train_fp32", "op": "gated", "T": 65536, "D": 256, "H": 512, "type": "fp32", "act": "silu", "bias": True, "train": True},
        # a wide layer in a training step, the largest work
        {"name": "gated_train_bf16", "op": "gated", "T": 16384, "D": 2048, "H": 8192, "type": "bf16", "act": "gelu", "bias": False, "train": True},
        # nothing divides anything: a ragged last batch and odd widths
        {"name": "gated_ragged_bf16", "op": "gated", "T": 1237, "D": 517, "H": 1021, "type": "bf16", "act": "sigmoid", "bias": True, "train": True},
        # one layer's update on its own
        {"name": "ortho_one_fp32", "op": "ortho", "B": 1, "R": 256, "C": 256, "type": "fp32"},
        # the updates of a stack of equal layers, kept in 16 bits
        {"name": "ortho_stack_bf16", "op": "ortho", "B": 24, "R": 256, "C": 304, "type": "bf16"},
        # one large square matrix
        {"name": "ortho_large_fp32", "op": "ortho", "B": 1, "R": 4096, "C": 4096, "type": "fp32"},
        # tall and odd
        {"name": "ortho_tall_fp16", "op": "ortho", "B": 3, "R": 1531, "C": 517, "type": "fp16"},
        # an optimiser step over the hidden matrices of a scene's networks
        {"name": "muon_scene_fp32", "op": "muon", "B": 36, "R": 256, "C": 256, "type": "fp32", "nesterov": True},
        # an optimiser step over wide matrices
        {"name": "muon_wide_fp32", "op": "muon", "B": 6, "R": 1024, "C": 4096, "type": "fp32", "nesterov": False},
    ]


def _size(rng, low, high):
    """a size between low and high, spread over the logarithm"""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["gated", "gated", "gated", "ortho", "muon"])
    if op == "gated":
        kind = rng.choice(["rows", "forward", "train"])
        D, H = _size(rng, 32, 4096), _size(rng, 32, 8192)
        if rng.random() < 0.5:  # widths are multiples of 32 about as often as not
            D, H = max(32, D // 32 * 32), max(32, H // 32 * 32)
        most = int(2.7e11 / (D * H))  # the largest listed case's work
        T = _size(rng, 1, 64) if kind == "rows" else _size(rng, 65, max(66, min(262144, most, int(2.5e8 / max(D, H)))))
        return {"op": op, "T": T, "D": D, "H": H, "type": rng.choice(["fp32", "bf16"]), "act": rng.choice(["silu", "gelu", "relu", "sigmoid"]),
                "bias": rng.random() < 0.5, "train": kind == "train"}
    R, C = _size(rng, 16, 4096), _size(rng, 16, 4096)
    if rng.random() < 0.5:
        R, C = max(16, R // 32 * 32), max(16, C // 32 * 32)
    most = max(1, int(4096.0 ** 3 / (min(R, C) ** 2 * max(R, C))))
    B = _size(rng, 1, min(48, most))
    if op == "ortho":
        return {"op": op, "B": B, "R": R, "C": C, "type": rng.choice(["fp32", "bf16", "fp16"])}
    return {"op": op, "B": B, "R": R, "C": C, "type": "fp32", "nesterov": rng.random() < 0.5}


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda")


def _gradients(gen, B, R, C):
    """matrices as gradients are: a few strong directions over a floor of noise"""
    k = max(1, min(R, C) // 8)
    strong = _normal(gen, B, R, k) / torch.arange(1, k + 1, device="cuda").sqrt() @ _normal(gen, B, k, C)
    return (strong + _normal(gen, B, R, C)) * 1e-3


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = TYPES[case["type"]]
    s = {"case": dict(case)}
    if case["op"] == "gated":
        T, D, H = case["T"], case["D"], case["H"]
        s["x"] = _normal(gen, T, D).to(dt)
        s["w_gate"] = (_normal(gen, H, D) * D ** -0.5).to(dt)
        s["w_up"] = (_normal(gen, H, D) * D ** -0.5).to(dt)
        s["b_gate"] = (0.1 * _normal(gen, H)).to(dt) if case["bias"] else None
        s["b_up"] = (0.1 * _normal(gen, H)).to(dt) if case["bias"] else None
        if case["train"]:
            s["dh"] = (_normal(gen, T, H) / T).to(dt)
            for k in ("x", "w_gate", "w_up", "b_gate", "b_up"):
                if s[k] is not None:
                    s[k].requires_grad_(True)
    elif case["op"] == "ortho":
        s["x"] = _gradients(gen, case["B"], case["R"], case["C"]).to(dt)
    else:
        B, R, C = case["B"], case["R"], case["C"]
        s["p"] = _normal(gen, B, R, C) * C ** -0.5
        s["g"] = _gradients(gen, B, R, C)
        s["m"] = _gradients(gen, B, R, C)
        s["lists"] = [list(s[k].unbind(0)) for k in "pgm"]
    return s


# ---- the gated layer: h = act(x Wg^T + bg) * (x Wu^T + bu) -----------------------------------------------------------------------


def _act(g, act):
    """(act(g), act'(g))"""
    if act == "relu":
        return g.clamp(min=0), (g > 0).to(g.dtype)
    if act == "gelu":
        phi = 0.5 * (1 + torch.erf(g * 0.5 ** 0.5))
        return g * phi, phi + g * torch.exp(-0.5 * g * g) * (2 * math.pi) ** -0.5
    sig = 1 / (1 + torch.exp(-g))
    if act == "sigmoid":
        return sig, sig * (1 - sig)
    return g * sig, sig * (1 + g * (1 - sig))


def _plain_gated(s):
    case, dt = s["case"], s["x"].dtype
    x, wg, wu = s["x"].detach().float(), s["w_gate"].detach().float(), s["w_up"].detach().float()
    g, u = x @ wg.t(), x @ wu.t()
    if case["bias"]:
        g, u = g + s["b_gate"].detach().float(), u + s["b_up"].detach().float()
    a, da = _act(g, case["act"])
    out = {"h": (a * u).to(dt)}
    if case["train"]:
        dh = s["dh"].float()
        dg, du = dh * u * da, dh * a
        out["x"] = (dg @ wg + du @ wu).to(dt)
        out["w_gate"], out["w_up"] = (dg.t() @ x).to(dt), (du.t() @ x).to(dt)
        if case["bias"]:
            out["b_gate"], out["b_up"] = dg.sum(0).to(dt), du.sum(0).to(dt)
    return out


def _own_gated(s):
    from hold_amd.gated import gated_linear
    h = gated_linear(s["x"], s["w_gate"], s["w_up"], s["b_gate"], s["b_up"], activation=s["case"]["act"])
    out = {"h": h}
    if s["case"]["train"]:
        names = ["x", "w_gate", "w_up"] + (["b_gate", "b_up"] if s["case"]["bias"] else [])
        out.update(zip(names, torch.autograd.grad(h, [s[n] for n in names], s["dh"])))
        out["h"] = h.detach()
    return out


def _exact_gated(case, s):
    D = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    zero = torch.zeros(case["H"], dtype=torch.float64, device="cuda")
    g = torch.addmm(D.get("b_gate", zero), D["x"], D["w_gate"].t())
    u = torch.addmm(D.get("b_up", zero), D["x"], D["w_up"].t())
    g.requires_grad_(True)
    if case["act"] == "relu":
        a = torch.relu(g)
    elif case["act"] == "gelu":
        a = torch.special.ndtr(g) * g
    else:
        a = torch.sigmoid(g) if case["act"] == "sigmoid" else g * torch.sigmoid(g)
    out = {"h": a.detach() * u}
    if case["train"]:
        du = D["dh"] * a.detach()
        dg, = torch.autograd.grad(a, g, D["dh"] * u)
        out["x"] = torch.cat([dg, du], 1) @ torch.cat([D["w_gate"], D["w_up"]], 0)
        out["w_gate"], out["w_up"] = dg.t() @ D["x"], du.t() @ D["x"]
        if case["bias"]:
            out["b_gate"], out["b_up"] = dg.sum(0), du.sum(0)
    return out


# ---- the orthogonalised update: X <- a X + (b A + c A^2) X with A = X X^T ----------------------------------------------------


def _newton_schulz(x, dtype):
    x = x.to(dtype)
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-1, -2)
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + EPS)
    a, b, c = QUINTIC
    for _ in range(STEPS):
        gram = x @ x.transpose(-1, -2)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(-1, -2) if tall else x


def _muon_scale(R, C):
    return max(1.0, R / C) ** 0.5


def _plain_muon(s):
    case, p, g, m = s["case"], s["p"], s["g"], s["m"]
    m.mul_(MOMENTUM).add_(g, alpha=1 - MOMENTUM)
    u = (1 - MOMENTUM) * g + MOMENTUM * m if case["nesterov"] else m
    p.mul_(1 - LR * DECAY).add_(_newton_schulz(u, torch.float32), alpha=-LR * _muon_scale(case["R"], case["C"]))
    return {"p": p, "m": m}


def _own_muon(s):
    from hold_amd.muon import muon_step
    muon_step(*s["lists"], lr=LR, momentum=MOMENTUM, nesterov=s["case"]["nesterov"], weight_decay=DECAY, steps=STEPS, coefficients=QUINTIC, eps=EPS)
    return {"p": s["p"], "m": s["m"]}


def _exact_ortho(x):
    """the polynomial a s + b s^3 + c s^5, five times over the singular values of x / (|x| + eps)"""
    x = x.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.transpose(-1, -2).contiguous() if tall else x
    x = x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True) + EPS)
    a, b, c = QUINTIC
    eye = torch.eye(x.shape[-2], dtype=torch.float64, device=x.device)
    for _ in range(STEPS):
        gram = torch.matmul(x, x.transpose(-1, -2).contiguous())
        x = torch.matmul(a * eye + torch.matmul(gram, c * gram + b * eye), x)
    return x.transpose(-1, -2) if tall else x


def run(state):
    op = state["case"]["op"]
    if op == "gated":
        return _own_gated(state) if own else _plain_gated(state)
    if op == "muon":
        return _own_muon(state) if own else _plain_muon(state)
    if own:
        from hold_amd.muon import orthogonalize
        return orthogonalize(state["x"], steps=STEPS, coefficients=QUINTIC, eps=EPS)
    return _newton_schulz(state["x"], torch.float32).to(state["x"].dtype)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "gated":
        return _exact_gated(case, s)
    if case["op"] == "ortho":
        return _exact_ortho(s["x"])
    p, g, m = s["p"].double(), s["g"].double(), s["m"].double()
    m = MOMENTUM * m + (1 - MOMENTUM) * g
    u = (1 - MOMENTUM) * g + MOMENTUM * m if case["nesterov"] else m
    return {"p": (1 - LR * DECAY) * p - LR * _muon_scale(case["R"], case["C"]) * _exact_ortho(u), "m": m}


def work(case):
    size = 4 if case["type"] == "fp32" else 2
    if case["op"] == "gated":
        T, D, H = case["T"], case["D"], case["H"]
        weights = 2 * H * (D + (1 if case["bias"] else 0))
        if not case["train"]:
            return {"bytes": size * (T * D + weights + T * H), "flops": 4 * T * D * H}
        # two products forward, two for the input's gradient, two for the weights' gradients
        return {"bytes": size * (T * D + weights + T * H + T * H + T * D + weights), "flops": 12 * T * D * H}
    B, m, n = case["B"], min(case["R"], case["C"]), max(case["R"], case["C"])
    # a step's two symmetric products count half: m^2 n for X X^T, m^3 for A A, 2 m^2 n for the product with X
    flops = B * STEPS * (3 * m * m * n + m * m * m)
    return {"bytes": size * B * m * n * (2 if case["op"] == "ortho" else 5), "flops": flops}

"""The measured operators of training a dense network: the linear layer with its epilogue, the Newton-Schulz orthogonalisation of a weight's
update, and the optimiser step that is built on it.

    linear   y = act(x W^T + b) + residual, and with "train" the gradients of x, W, b and the residual for a given dy
    orth     X0 = G / max(||G||_F, eps);  `steps` times  X <- a X + (b A + c A A) X,  A = X X^T  (the shorter side's Gram matrix)
    muon     m <- lerp(m, g, 1 - mu);  u = lerp(g, m, mu);  p <- (1 - lr wd) p - lr sqrt(max(1, rows / cols)) orth(u)

Where `own` is false, `run` computes them in elementary torch operations in 32 bits, rounded once at the end (the Frobenius norm, a sum over up to
millions of squares that every later step scales with, in 64).  Where it is true, it calls this package's entry points."""
import math

import torch

own = False

STEPS, COEFFICIENTS, EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7
LR, WEIGHT_DECAY, MOMENTUM = 0.02, 0.01, 0.95
SLOPE = 0.02      # the slope of leaky_relu below zero: the audio encoder's
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
ACTIVATIONS = ("none", "relu", "leaky_relu", "gelu", "silu")
# every trained matrix of the lip model (convolution weights as out x (in * taps)): the eight 256-wide layers, the input projections, the audio encoder
LIP_MODEL = "256x256*7,256x512,256x42*2,256x64*2,256x20*2,32x87,32x96,64x96,64x192,64x64*2"
# a residual block of width 1024: four square projections, one widening and one narrowing layer
WIDE_BLOCK = "1024x1024*4,4096x1024,1024x4096"


def _linear(rows, inner, outer, dtype, act, residual, train, **name):
    return {**name, "op": "linear", "rows": rows, "inner": inner, "outer": outer, "dtype": dtype, "act": act, "residual": residual, "train": train}


def _orth(batch, rows, cols, dtype, **name):
    return {**name, "op": "orth", "batch": batch, "rows": rows, "cols": cols, "dtype": dtype}


def _muon(shapes, **name):
    return {**name, "op": "muon", "shapes": shapes}


def listed():
    return [
        # one sample through one layer of the lip model: what a call costs
        _linear(1, 256, 256, "float32", "relu", False, False, name="linear-one-row"),
        # the pixels of one 96 x 96 frame through one layer, inference
        _linear(9216, 256, 256, "bfloat16", "relu", False, False, name="linear-frame"),
        # one 64 x 64 frame through the skip layer (512 in), exact-parity type, a training step
        _linear(4096, 512, 256, "float32", "silu", False, True, name="linear-skip-train"),
        # the four-tap ensemble of one 96 x 96 frame through one residual layer, a training step
        _linear(36864, 256, 256, "bfloat16", "relu", True, True, name="linear-ensemble-train"),
        # nothing a multiple of anything: ragged rows, odd widths, unaligned rows in memory
        _linear(4099, 333, 201, "float16", "leaky_relu", True, True, name="linear-odd-train"),
        # a wide layer over many samples: the matrix cores' rate
        _linear(16384, 1024, 4096, "bfloat16", "gelu", False, True, name="linear-wide-train"),
        # the seven square layers of the lip model at once
        _orth(7, 256, 256, "float32", name="orth-layers"),
        # one 3x3 convolution of the post-fusion U-Net (64 x 64*9): the smallest call
        _orth(1, 64, 576, "bfloat16", name="orth-conv"),
        # a tall matrix of odd size, worked on from its shorter side
        _orth(1, 1000, 333, "float32", name="orth-odd"),
        # large squares: the matrix cores' rate
        _orth(4, 2048, 2048, "bfloat16", name="orth-large"),
        # the optimiser step of the whole lip model: 20 matrices of ten shapes
        _muon(LIP_MODEL, name="muon-lip-model"),
        # the optimiser step of a wide residual block
        _muon(WIDE_BLOCK, name="muon-wide-block"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _shapes(text):
    out = []
    for item in text.split(","):
        size, _, count = item.partition("*")
        rows, _, cols = size.partition("x")
        out += [(int(rows), int(cols))] * int(count or 1)
    return out


def _orth_flops(rows, cols):
    m, n = min(rows, cols), max(rows, cols)
    return STEPS * (m * m * n + m * m * m + 2 * m * m * n)      # X X^T and A A are symmetric: half of each


def draw(rng):
    op = rng.choice(("linear", "linear", "orth", "muon"))
    if op == "linear":
        while True:
            rows, inner, outer = _spread(rng, 1, 36864), _spread(rng, 16, 4096), _spread(rng, 16, 4096)
            if rows * inner * outer <= 16384 * 1024 * 4096 and rows * max(inner, outer) <= 16384 * 4096:
                break
        dtype, train = rng.choice(("float32", "bfloat16", "float16")), rng.random() < 0.6
        # a kinked activation's gradient in 32 bits jumps where z is within a rounding of 0: there two right answers differ, so smooth ones are drawn
        act = rng.choice(("none", "gelu", "silu") if train and dtype == "float32" else ACTIVATIONS)
        return _linear(rows, inner, outer, dtype, act, rng.random() < 0.5, train)
    if op == "orth":
        while True:
            batch, rows, cols = _spread(rng, 1, 8), _spread(rng, 16, 4096), _spread(rng, 16, 4096)
            if batch * _orth_flops(rows, cols) <= 4 * _orth_flops(2048, 2048):
                break
        return _orth(batch, rows, cols, rng.choice(("float32", "bfloat16", "float16")))
    while True:
        shapes = ["%dx%d*%d" % (_spread(rng, 16, 4096), _spread(rng, 16, 4096), rng.choice((1, 1, 2, 4))) for _ in range(rng.randint(1, 6))]
        if sum(_orth_flops(*s) for s in _shapes(",".join(shapes))) <= sum(_orth_flops(*s) for s in _shapes(WIDE_BLOCK)):
            return _muon(",".join(shapes))


def _gradient(shape, gen):
    """A weight's gradient as training makes it: a few shared directions over a floor of noise, rows and columns of unlike size."""
    rows, cols = shape[-2:]
    lead = shape[:-2]
    normal = lambda *s: torch.randn(*lead, *s, generator=gen, device="cuda")  # noqa: E731
    size = lambda n: torch.exp(0.5 * torch.randn(*lead, n, generator=gen, device="cuda"))  # noqa: E731
    shared = normal(rows, 8) @ normal(8, cols) * 0.2
    return 1e-3 * size(rows)[..., :, None] * (normal(rows, cols) + shared) * size(cols)[..., None, :]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "linear":
        rows, inner, outer, dtype = case["rows"], case["inner"], case["outer"], DTYPES[case["dtype"]]
        normal = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
        s = {"case": case,
             "x": normal(rows, inner).to(dtype),
             "weight": (normal(outer, inner) / math.sqrt(inner)).to(dtype),
             "bias": (0.1 * normal(outer)).to(dtype),
             "residual": normal(rows, outer).to(dtype) if case["residual"] else None,
             "dy": normal(rows, outer).to(dtype) if case["train"] else None}
        if case["train"]:
            for k in ("x", "weight", "bias", "residual"):
                if s[k] is not None:
                    s[k].requires_grad_()
        return s
    if case["op"] == "orth":
        return {"case": case, "update": _gradient((case["batch"], case["rows"], case["cols"]), gen).to(DTYPES[case["dtype"]])}
    shapes = _shapes(case["shapes"])
    params = [torch.nn.Parameter(torch.randn(*s, generator=gen, device="cuda") / math.sqrt(s[1])) for s in shapes]
    buffers = [0.3 * _gradient(s, gen) for s in shapes]      # the running mean of earlier gradients
    for p in params:
        p.grad = _gradient(p.shape, gen)
    s = {"case": case, "params": params, "buffers": buffers}
    if own:      # the optimiser that a training program keeps
        from speech2lip_amd import FusedMuon
        s["optimizer"] = FusedMuon(params, lr=LR, weight_decay=WEIGHT_DECAY, momentum=MOMENTUM, nesterov=True, ns_coefficients=COEFFICIENTS,
                                   eps=EPS, ns_steps=STEPS)
        for p, b in zip(params, buffers):
            s["optimizer"].state[p]["momentum_buffer"] = b
    return s


def _act(z, act):
    if act == "relu":
        return torch.clamp(z, min=0)
    if act == "leaky_relu":
        return torch.where(z > 0, z, SLOPE * z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "leaky_relu":
        return torch.where(z > 0, 1.0, SLOPE)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


@torch.no_grad()
def _linear_plain(s):
    act, dtype = s["case"]["act"], s["x"].dtype
    x, w, b = s["x"].float(), s["weight"].float(), s["bias"].float()
    z = x @ w.t() + b
    y = _act(z, act)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    if s["dy"] is None:
        return {"y": y.to(dtype)}
    dz = s["dy"].float()
    if act != "none":
        dz = dz * _act_slope(z, act)
    out = {"y": y.to(dtype), "dx": (dz @ w).to(dtype), "dweight": (dz.t() @ x).to(dtype), "dbias": dz.sum(0).to(dtype)}
    if s["residual"] is not None:
        out["dresidual"] = s["dy"]
    return out


def _orth_plain(u):
    """u [..., rows, cols] in 32 bits."""
    tall = u.shape[-2] > u.shape[-1]
    x = u.mT if tall else u
    norm = x.double().square().sum((-2, -1), keepdim=True).sqrt().clamp(min=EPS)
    x = (x / norm.float())
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.mT if tall else x


@torch.no_grad()
def _muon_plain(s):
    groups = {}
    for p, m in zip(s["params"], s["buffers"]):
        groups.setdefault(tuple(p.shape), []).append((p, m))
    for (rows, cols), members in groups.items():      # the matrices of one shape together
        g = torch.stack([p.grad for p, _ in members])
        m = torch.stack([m for _, m in members])
        m = m + (1 - MOMENTUM) * (g - m)
        o = _orth_plain(g + MOMENTUM * (m - g))
        p = torch.stack([p for p, _ in members]) * (1 - LR * WEIGHT_DECAY) - LR * math.sqrt(max(1.0, rows / cols)) * o
        for k, (param, buffer) in enumerate(members):
            param.copy_(p[k])
            buffer.copy_(m[k])


def run(state):
    op = state["case"]["op"]
    if op == "linear":
        if not own:
            return _linear_plain(state)
        from speech2lip_amd import autograd
        y = autograd.linear(state["x"], state["weight"], state["bias"], residual=state["residual"], activation=state["case"]["act"])
        if state["dy"] is None:
            return {"y": y}
        names = [k for k in ("x", "weight", "bias", "residual") if state[k] is not None]
        grads = torch.autograd.grad(y, [state[k] for k in names], state["dy"])
        return {"y": y, **{"d" + k: g for k, g in zip(names, grads)}}
    if op == "orth":
        if not own:
            u = state["update"]
            return _orth_plain(u.float()).to(u.dtype)
        from speech2lip_amd import optim
        return optim.orthogonalize(state["update"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
    if own:
        state["optimizer"].step()
    else:
        _muon_plain(state)
    return {"params": state["params"], "buffers": state["buffers"]}


def work(case):
    if case["op"] == "linear":
        size = 4 if case["dtype"] == "float32" else 2
        x, w, y = case["rows"] * case["inner"], case["inner"] * case["outer"], case["rows"] * case["outer"]
        values, flops = x + w + case["outer"] + y * (1 + case["residual"]), 2 * case["rows"] * w
        if case["train"]:
            values, flops = values + y + x + w + case["outer"], 3 * flops      # dy in; dx, dW, db out
        return {"bytes": size * values, "flops": flops}
    if case["op"] == "orth":
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": 2 * size * case["batch"] * case["rows"] * case["cols"], "flops": case["batch"] * _orth_flops(case["rows"], case["cols"])}
    shapes = _shapes(case["shapes"])
    return {"bytes": sum(5 * 4 * r * c for r, c in shapes), "flops": sum(_orth_flops(r, c) for r, c in shapes)}      # p, m in and out, g in


def _orth_exact(u):
    """The iteration from the other side, X <- X (a I + b S + c S S) with S = X^T X of the shorter side, in 64 bits."""
    a, b, c = COEFFICIENTS
    wide = u.shape[-1] > u.shape[-2]
    x = u.double()
    x = x.transpose(-1, -2) if wide else x
    x = x / torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True).clamp_min(EPS)
    eye = torch.eye(x.shape[-1], dtype=torch.float64, device=u.device)
    for _ in range(STEPS):
        s = torch.matmul(x.transpose(-1, -2), x)
        x = torch.matmul(x, a * eye + torch.matmul(s, b * eye + c * s))
    return x.transpose(-1, -2) if wide else x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        f = torch.nn.functional
        names = [k for k in ("x", "weight", "bias", "residual") if s[k] is not None]
        v = {k: s[k].detach().double().requires_grad_(case["train"]) for k in names}
        z = f.linear(v["x"], v["weight"], v["bias"])
        y = {"none": lambda t: t, "relu": f.relu, "leaky_relu": lambda t: f.leaky_relu(t, SLOPE), "gelu": f.gelu, "silu": f.silu}[case["act"]](z)
        y = y + v["residual"] if "residual" in v else y
        if not case["train"]:
            return {"y": y}
        grads = torch.autograd.grad(y, [v[k] for k in names], s["dy"].double())
        return {"y": y.detach(), **{"d" + k: g for k, g in zip(names, grads)}}
    if case["op"] == "orth":
        return _orth_exact(s["update"])
    params, buffers = [], []
    for p, m in zip(s["params"], s["buffers"]):
        g, m = p.grad.double(), MOMENTUM * m.double() + (1 - MOMENTUM) * p.grad.double()
        step = _orth_exact((1 - MOMENTUM) * g + MOMENTUM * m) * max(1.0, p.shape[0] / p.shape[1]) ** 0.5
        params.append((p.detach().double() - LR * (WEIGHT_DECAY * p.detach().double() + step)))
        buffers.append(m)
    return {"params": params, "buffers": buffers}

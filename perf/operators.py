"""Cases, plain forms and calls of the layer operators: a linear layer with its epilogue, its
training step, batch normalisation with activation and dropout, and 8-bit activation checkpoints.

The conditional VAE's stacks are [Linear, BatchNorm1d, activation, Dropout] blocks; these operators
are that block's pieces, forward and backward, for batches from one row to a whole data set and for
networks wider than the shipped one.

  linear         y = act(x W^T + b) + r                       inference: one row up to a large batch
  linear_train   the same, and dx, dW, db for a given dy; with "eight" the input and the activation's
                 derivative are held in 8 bits between the two passes
  norm_train     y = keep/(1-p) * act(batch_norm(x)), and dx, dgamma, dbeta; with "eight" the input
                 is held in 8 bits between the two passes
  checkpoint     a tensor packed to 8 bits and restored

8-bit input: blocks of 32 along a row share the power of two 2^E with E = floor(log2(max |x|)); an
element is the nearest multiple q 2^(E-6), |q| <= 127 (ties to even).  8-bit derivative: the nearest
multiple of 1/200 (tanh, gelu, silu); relu and leaky_relu keep the sign of the pre-activation.
"""
import math

import torch

own = False

SLOPE = 0.2          # the framework's leaky_relu
EPS, MOMENTUM = 1e-5, 0.1
DROP = 0.15          # the conditional VAE's dropout
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one sample through a wide layer: what a request waits for
        {"name": "serve one row", "op": "linear", "type": "bf16", "m": 1, "k": 4096, "n": 4096, "act": "silu", "residual": True},
        # 100 samples of one date (the generator's ensemble) through the VAE's 128 -> 64 layer
        {"name": "serve ensemble", "op": "linear", "type": "f32", "m": 100, "k": 128, "n": 64, "act": "tanh", "residual": False},
        # ragged in every direction
        {"name": "serve odd", "op": "linear", "type": "f16", "m": 777, "k": 1003, "n": 2055, "act": "gelu", "residual": False},
        # a large batch through a wide layer
        {"name": "serve large", "op": "linear", "type": "bf16", "m": 16384, "k": 4096, "n": 8192, "act": "gelu", "residual": True},
        # the VAE's first encoder layer at its batch of 64
        {"name": "train vae layer", "op": "linear_train", "type": "f32", "m": 64, "k": 13, "n": 128, "act": "none", "residual": False, "eight": True},
        # single precision, a middling layer
        {"name": "train f32", "op": "linear_train", "type": "f32", "m": 8192, "k": 1024, "n": 512, "act": "tanh", "residual": False, "eight": False},
        # ragged in every direction, with the skip connection
        {"name": "train odd", "op": "linear_train", "type": "f16", "m": 3001, "k": 777, "n": 1025, "act": "leaky_relu", "residual": True, "eight": True},
        # a large batch through a wide layer, checkpoints in 8 bits
        {"name": "train large", "op": "linear_train", "type": "bf16", "m": 16384, "k": 4096, "n": 4096, "act": "gelu", "residual": False, "eight": True},
        # the VAE's first encoder layer at its batch of 64
        {"name": "norm vae layer", "op": "norm_train", "type": "f32", "m": 64, "n": 128, "act": "tanh", "drop": True, "eight": True},
        # a whole data set as one batch
        {"name": "norm large", "op": "norm_train", "type": "bf16", "m": 131072, "n": 1024, "act": "relu", "drop": True, "eight": True},
        # ragged rows
        {"name": "checkpoint odd", "op": "checkpoint", "type": "f16", "m": 1001, "k": 333},
        # the input of a wide layer at a large batch
        {"name": "checkpoint large", "op": "checkpoint", "type": "bf16", "m": 32768, "k": 4096},
    ]


def _size(rng, lo, hi):
    """Spread over the logarithm; a third are odd numbers, a third multiples of 8."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    how = rng.randrange(3)
    if how == 0:
        v |= 1
    elif how == 1:
        v = max(8, v // 8 * 8)
    return min(max(v, lo), hi)


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_train", "linear_train", "norm_train", "checkpoint"])
    typ = rng.choice(["f32", "bf16", "bf16", "f16"])
    if op == "checkpoint":
        return {"op": op, "type": typ, "m": _size(rng, 1, 32768), "k": _size(rng, 4, 4096)}
    if op == "norm_train":
        return {"op": op, "type": typ, "m": _size(rng, 2, 131072), "n": _size(rng, 4, 1024),
                "act": rng.choice(["none", "relu", "leaky_relu", "tanh", "gelu", "silu"]), "drop": rng.random() < 0.7, "eight": rng.random() < 0.6}
    m, k, n = _size(rng, 1, 16384), _size(rng, 8, 4096), _size(rng, 4, 8192)
    if op == "linear":
        return {"op": op, "type": typ, "m": m, "k": k, "n": n, "act": rng.choice(["none", "relu", "leaky_relu", "tanh", "gelu", "silu"]), "residual": rng.random() < 0.5}
    n = min(n, 4096)
    eight = rng.random() < 0.6
    # a derivative that jumps (relu's at zero, an 8-bit derivative's at half steps) follows the last bits of the
    # pre-activation, which no two orders of a sum share: single precision takes the smooth ones, wide rows the others
    smooth = ["none", "tanh", "gelu", "silu"]
    acts = (["none"] if eight else smooth) if typ == "f32" else smooth + (["relu", "leaky_relu"] if n >= 64 else [])
    return {"op": op, "type": typ, "m": m, "k": k, "n": n, "act": rng.choice(acts), "residual": rng.random() < 0.3, "eight": eight}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = _TYPES[case["type"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(t)

    m, n = case["m"], case.get("n")
    s = {"case": case}
    if case["op"] == "checkpoint":
        # a hidden activation after dropout: exact zeros among the values
        x = normal(m, case["k"])
        s["x"] = x * (torch.rand(m, case["k"], generator=g, device="cuda") >= DROP)
        return s
    if case["op"] == "norm_train":
        # columns of different size and offset, as pre-activations are
        x = torch.randn(m, n, generator=g, device="cuda") * (0.25 + torch.rand(n, generator=g, device="cuda")) + torch.randn(n, generator=g, device="cuda")
        s["x"] = x.to(t)
        s["gamma"] = 0.5 + torch.rand(n, generator=g, device="cuda")
        s["beta"] = 0.3 * torch.randn(n, generator=g, device="cuda")
        s["mean"] = torch.zeros(n, device="cuda")
        s["var"] = torch.ones(n, device="cuda")
        s["keep"] = torch.rand(m, n, generator=g, device="cuda") >= DROP if case["drop"] else None
        s["dy"] = normal(m, n)
        return s
    k = case["k"]
    s["x"] = normal(m, k)
    lim = 1.0 / math.sqrt(k)
    s["w"] = ((2 * torch.rand(n, k, generator=g, device="cuda") - 1) * lim).to(t)
    s["b"] = ((2 * torch.rand(n, generator=g, device="cuda") - 1) * lim).to(t)
    s["r"] = normal(m, n) if case["residual"] else None
    if case["op"] == "linear_train":
        s["dy"] = normal(m, n)
    return s


# ---- plain forms -----------------------------------------------------------------------------
def _act(z, act):
    if act == "none":
        return z
    if act == "relu":
        return z.clamp(min=0)
    if act == "leaky_relu":
        return torch.where(z > 0, z, SLOPE * z)
    if act == "tanh":
        return torch.tanh(z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z * torch.sigmoid(z)


def _derivative(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "leaky_relu":
        return torch.where(z > 0, 1.0, SLOPE)
    if act == "tanh":
        return 1 - torch.tanh(z).square()
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * math.sqrt(0.5 / math.pi)
    p = torch.sigmoid(z)
    return p * (1 + z * (1 - p))


def _in_eight_bits(x):
    """x (float32) after its 8-bit checkpoint."""
    m, k = x.shape
    b = torch.nn.functional.pad(x, (0, -k % 32)).view(m, -1, 32)
    e = torch.frexp(b.abs().amax(-1, keepdim=True))[1] - 1
    q = torch.ldexp(b, 6 - e).round().clamp(-127, 127)
    return torch.ldexp(q, e - 6).view(m, -1)[:, :k]


def _plain_linear(s):
    c = s["case"]
    z = torch.addmm(s["b"].float(), s["x"].float(), s["w"].float().t())
    y = _act(z, c["act"])
    return z, (y if s["r"] is None else y + s["r"].float())


def _plain_linear_train(s):
    c, t = s["case"], s["x"].dtype
    z, y = _plain_linear(s)
    x, dz = s["x"].float(), s["dy"].float()
    if c["eight"]:
        x = _in_eight_bits(x)
    if c["act"] != "none":
        d = _derivative(z, c["act"])
        if c["eight"] and c["act"] not in ("relu", "leaky_relu"):
            d = (d * 200).round() / 200
        dz = dz * d
    return {"y": y.to(t), "dx": (dz @ s["w"].float()).to(t), "dw": (dz.t() @ x).to(t), "db": dz.sum(0).to(t)}


def _plain_norm_train(s):
    c, t, m = s["case"], s["x"].dtype, s["x"].shape[0]
    # relu's derivative jumps at zero: the side of the border is taken in 64 bits, and the statistics with it
    x = s["x"].double() if c["act"] in ("relu", "leaky_relu") else s["x"].float()
    gamma, beta = s["gamma"].to(x.dtype), s["beta"].to(x.dtype)
    mean = x.mean(0)
    var = (x - mean).square().mean(0)
    rstd = torch.rsqrt(var + EPS)
    scale = 1.0 / (1.0 - DROP)
    y = _act((x - mean) * rstd * gamma + beta, c["act"])
    if s["keep"] is not None:
        y = y * s["keep"] * scale
    s["mean"].mul_(1 - MOMENTUM).add_(MOMENTUM * mean.float())
    s["var"].mul_(1 - MOMENTUM).add_(MOMENTUM * (var * (m / (m - 1))).float())
    if c["eight"]:
        x = _in_eight_bits(s["x"].float()).to(x.dtype)
    h = (x - mean) * rstd
    g = s["dy"].float()
    if c["act"] != "none":
        g = g * _derivative(h * gamma + beta, c["act"]).float()
    if s["keep"] is not None:
        g = g * s["keep"] * scale
    h, rstd, gamma = h.float(), rstd.float(), gamma.float()
    dbeta, dgamma = g.sum(0), (g * h).sum(0)
    dx = gamma * rstd * (g - dbeta / m - h * (dgamma / m))
    return {"y": y.to(t), "dx": dx.to(t), "dgamma": dgamma, "dbeta": dbeta, "mean": s["mean"], "var": s["var"]}


# ---- the framework's calls ---------------------------------------------------------------------
def _afiv():
    import afiv_bootstrap
    return afiv_bootstrap.load()


def _own(s):
    afiv, c = _afiv(), s["case"]
    if c["op"] == "checkpoint":
        return afiv.checkpoint8(s["x"]).restore()
    if c["op"] == "linear":
        return afiv.linear_act(s["x"], s["w"], s["b"], residual=s["r"], act=c["act"])
    if c["op"] == "linear_train":
        y, saved = afiv.linear_act_forward(s["x"], s["w"], s["b"], residual=s["r"], act=c["act"], checkpoint8=c["eight"])
        dx, dw, db = afiv.linear_act_backward(s["dy"], s["w"], saved)
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    y, saved = afiv.batch_norm_act_forward(s["x"], s["gamma"], s["beta"], s["mean"], s["var"], act=c["act"], keep=s["keep"],
                                           drop_p=DROP if c["drop"] else 0.0, momentum=MOMENTUM, eps=EPS, checkpoint8=c["eight"])
    dx, dgamma, dbeta = afiv.batch_norm_act_backward(s["dy"], s["gamma"], s["beta"], saved)
    return {"y": y, "dx": dx, "dgamma": dgamma, "dbeta": dbeta, "mean": s["mean"], "var": s["var"]}


def run(state):
    if own:
        return _own(state)
    c = state["case"]
    if c["op"] == "checkpoint":
        return _in_eight_bits(state["x"].float()).to(state["x"].dtype)
    if c["op"] == "linear":
        return _plain_linear(state)[1].to(state["x"].dtype)
    if c["op"] == "linear_train":
        return _plain_linear_train(state)
    return _plain_norm_train(state)


def work(case):
    size = 4 if case["type"] == "f32" else 2
    m, k, n = case["m"], case.get("k", 0), case.get("n", 0)
    if case["op"] == "checkpoint":
        return {"bytes": 2 * m * k * size, "flops": 3 * m * k}
    if case["op"] == "linear":
        return {"bytes": (m * k + n * k + n + m * n * (2 if case["residual"] else 1)) * size, "flops": 2 * m * n * k}
    if case["op"] == "linear_train":
        # x, W, b, r, dy in; y, dx, dW, db out; three products
        return {"bytes": (2 * m * k + 2 * n * k + 2 * n + m * n * (3 if case["residual"] else 2)) * size, "flops": 6 * m * n * k}
    # x, dy, keep in; y, dx out; per column: gamma, beta, two running statistics in and out, two gradients
    return {"bytes": m * n * (4 * size + (1 if case["drop"] else 0)) + 8 * n * 4, "flops": 30 * m * n}


# ---- the definition in 64 bits -----------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    f8 = torch.float64

    def eight(v):
        rows, cols = v.shape
        out = torch.empty_like(v)
        for lo in range(0, cols, 32):
            part = v[:, lo:lo + 32]
            top = part.abs().max(dim=1, keepdim=True).values
            unit = torch.exp2(torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top)))) - 6)
            out[:, lo:lo + 32] = torch.clamp(torch.round(part / unit), -127, 127) * unit
        return out

    def f(z):
        return {"none": lambda: z, "relu": lambda: torch.relu(z), "leaky_relu": lambda: torch.nn.functional.leaky_relu(z, SLOPE), "tanh": lambda: torch.tanh(z),
                "gelu": lambda: z * torch.special.ndtr(z), "silu": lambda: z / (1 + torch.exp(-z))}[case["act"]]()

    def df(z):
        one = torch.ones_like(z)
        return {"none": lambda: one, "relu": lambda: torch.where(z > 0, one, 0 * one), "leaky_relu": lambda: torch.where(z > 0, one, SLOPE * one),
                "tanh": lambda: 1 / torch.cosh(z) ** 2, "gelu": lambda: torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi),
                "silu": lambda: 1 / (1 + torch.exp(-z)) + z * torch.exp(-z) / (1 + torch.exp(-z)) ** 2}[case["act"]]()

    x = s["x"].to(f8)
    if case["op"] == "checkpoint":
        return eight(x)
    if case["op"] in ("linear", "linear_train"):
        w = s["w"].to(f8)
        z = torch.matmul(x, w.T) + s["b"].to(f8)
        y = f(z)
        if s["r"] is not None:
            y = y + s["r"].to(f8)
        if case["op"] == "linear":
            return y
        d = df(z)
        if case["eight"]:
            x = eight(x)
            if case["act"] in ("tanh", "gelu", "silu"):
                d = torch.round(200 * d) / 200
        d = d * s["dy"].to(f8)
        return {"y": y, "dx": torch.matmul(d, w), "dw": torch.matmul(d.T, x), "db": d.sum(dim=0)}
    m = case["m"]
    gamma, beta = s["gamma"].to(f8), s["beta"].to(f8)
    var, mean = torch.var_mean(x, dim=0, correction=0)
    sd = torch.sqrt(var + EPS)
    up = s["keep"].to(f8) / (1 - DROP) if s["keep"] is not None else 1.0
    y = f((x - mean) / sd * gamma + beta) * up
    if case["eight"]:
        x = eight(x)
    h = (x - mean) / sd
    g = s["dy"].to(f8) * up * df(h * gamma + beta)
    dbeta, dgamma = g.sum(dim=0), (g * h).sum(dim=0)
    return {"y": y, "dx": gamma / sd * (g - (dbeta + h * dgamma) / m), "dgamma": dgamma, "dbeta": dbeta,
            "mean": (1 - MOMENTUM) * s["mean"].to(f8) + MOMENTUM * mean, "var": (1 - MOMENTUM) * s["var"].to(f8) + MOMENTUM * var * m / (m - 1)}

"""GPU tests of the layer operators (linear + activation + residual, batch norm + activation + dropout,
8-bit checkpoints) against their formulas in 64 bits.

Tolerances come from the arithmetic.  u = 2^-24 is FP32's half step, h = finfo(T).eps / 2 the half step
of the element type.  A sum of L products, added in FP32 in any order, is off by at most 2 L u times the sum
of the magnitudes (one step, not half, per addition: the matrix unit's adder is not documented to
round to nearest), the FP32 split adds 4 u of each product; an activation or derivative evaluated in
FP32 is off by a few u of its terms (16 u taken); every output is rounded to T once.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ACTS = ["none", "relu", "leaky_relu", "tanh", "gelu", "silu"]
SECOND = {"none": 0.0, "relu": 0.0, "leaky_relu": 0.0, "tanh": 0.77, "gelu": 0.8, "silu": 0.5}     # sup |f''|


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).smallest_normal * half(t)          # half the smallest step


def act64(z, act):
    return {"none": lambda: z, "relu": lambda: z.clamp(min=0), "leaky_relu": lambda: torch.where(z > 0, z, 0.2 * z), "tanh": lambda: z.tanh(),
            "gelu": lambda: z * torch.special.ndtr(z), "silu": lambda: z * torch.sigmoid(z)}[act]()


def der64(z, act):
    one = torch.ones_like(z)
    p = torch.sigmoid(z)
    return {"none": lambda: one, "relu": lambda: (z > 0).double(), "leaky_relu": lambda: torch.where(z > 0, one, 0.2 * one),
            "tanh": lambda: 1 / torch.cosh(z) ** 2, "gelu": lambda: torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi),
            "silu": lambda: p + z * p * (1 - p)}[act]()


def within(got, want, tol, what):
    got = got.double()
    assert torch.isfinite(got).all(), what
    off = (got - want).abs() - tol
    assert float(off.max()) <= 0, "%s: off by %.3g where %.3g is allowed" % (
        what, float((got - want).abs().flatten()[off.argmax()]), float(tol.expand_as(off).flatten()[off.argmax()]))


def inputs(t, m, k, n, seed, residual=False):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=g, device="cuda")
    x, w, b = r(m, k).to(t), (r(n, k) / math.sqrt(k)).to(t), r(n).to(t)
    return x, w, b, (r(m, n).to(t) if residual else None), r(m, n).to(t)


def check_forward(x, w, b, r, act, y, saved=None):
    t, k = x.dtype, x.shape[1]
    xd, wd = x.double(), w.double()
    z, mag = xd @ wd.T, xd.abs() @ wd.abs().T
    if b is not None:
        z, mag = z + b.double(), mag + b.double().abs()
    zerr = (2 * k + 8) * U * mag
    f = act64(z, act)
    want = f if r is None else f + r.double()
    within(y, want, 1.13 * zerr + 16 * U * (1 + z.abs()) + (want.abs() + zerr) * (half(t) + 2 * U) + tiny(t), "y")
    if saved is not None and saved.pre is not None:
        within(saved.pre, z, zerr + (z.abs() + zerr) * half(t) + tiny(t), "pre")
    if saved is not None and saved.dcodes is not None:
        c = saved.dcodes.double()
        if act in ("relu", "leaky_relu"):
            assert ((c == (z > 0)) | (z.abs() <= zerr)).all()
        else:
            within(c, 200 * der64(z, act) + 27, 0.5 + 200 * (SECOND[act] * zerr + 16 * U * (1 + z.abs())), "derivative codes")


def check_backward(dy, w, saved, act, dx, dw, db):
    t, (m, n), k = dy.dtype, dy.shape, w.shape[1]
    x = (saved.x if saved.eight is None else saved.eight.restore()).double().reshape(-1, k)
    if act == "none":
        d = torch.ones(m, n, dtype=torch.float64, device=dy.device)
    elif saved.pre is not None:
        d = der64(saved.pre.double(), act)
    elif act in ("relu", "leaky_relu"):
        d = torch.where(saved.dcodes > 0, 1.0, 0.2 if act == "leaky_relu" else 0.0).double()
    else:
        d = (saved.dcodes.double() - 27) / 200
    dz = dy.double() * d
    zero = torch.zeros((), dtype=torch.float64, device=dy.device)
    e = (0.0 if act == "none" else 16 * U) * dy.double().abs() * 1.2      # dz before it is rounded to T
    eh = e + (half(t) * (dz.abs() + e) + tiny(t) if act != "none" and t != torch.float32 else zero)
    for got, a, b, err, length, what in ((dx, dz, w.double(), eh @ w.double().abs(), n, "dx"), (dw, dz.T, x, eh.T @ x.abs(), m, "dw")):
        want = a @ b
        tol = err + (2 * length + 8) * U * (a.abs() @ b.abs())
        within(got, want, tol + (want.abs() + tol) * half(t) + tiny(t), what)
    want, tol = dz.sum(0), e.sum(0) + 2 * m * U * dz.abs().sum(0)
    within(db, want, tol + (want.abs() + tol) * half(t) + tiny(t), "db")


# one row to thousands; every residue of the tiles; lengths below, at and beyond a step of 32
SHAPES = [(1, 1, 1), (1, 4096, 64), (2, 7, 3), (16, 33, 17), (17, 32, 16), (5, 1000, 1001), (31, 13, 128), (64, 13, 128), (100, 128, 64),
          (33, 31, 65), (65, 64, 63), (129, 100, 127), (257, 8, 4), (1000, 77, 5), (3, 5000, 20), (130, 2048, 130), (2049, 257, 513), (32, 1056, 40), (24, 530, 9000)]


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear_forward_and_backward(afiv, typ, m, k, n):
    t = TYPES[typ]
    for i, act in enumerate(ACTS):
        x, w, b, r, dy = inputs(t, m, k, n, 100 * m + i, residual=i % 2 == 0)
        for eight in (False, True):
            y, saved = afiv.linear_act_forward(x, w, b if i != 3 else None, residual=r, act=act, checkpoint8=eight)
            check_forward(x, w, b if i != 3 else None, r, act, y, saved)
            dx, dw, db = afiv.linear_act_backward(dy, w, saved)
            check_backward(dy, w, saved, act, dx, dw, db)
        assert torch.equal(y, afiv.linear_act(x, w, b if i != 3 else None, residual=r, act=act))


@pytest.mark.parametrize("typ,m,k,n", [("bf16", 2048, 1024, 2048), ("f16", 4096, 512, 1024), ("f32", 2048, 512, 2304), ("bf16", 2300, 1096, 2056),
                                       ("bf16", 40000, 64, 72), ("f32", 40000, 24, 40), ("bf16", 4104, 200, 4112), ("f16", 4104, 4120, 136),
                                       ("bf16", 1000, 4096, 4200), ("f16", 136, 1288, 6008),
                                       ("bf16", 1501, 777, 1029), ("f32", 1501, 777, 1029), ("f32", 4104, 200, 4112), ("f32", 300, 4096, 2100)])
def test_linear_large_tiles(afiv, typ, m, k, n):
    x, w, b, r, dy = inputs(TYPES[typ], m, k, n, 5, residual=True)
    for act, eight in (("gelu", True), ("tanh", False)):
        y, saved = afiv.linear_act_forward(x, w, b, residual=r, act=act, checkpoint8=eight)
        check_forward(x, w, b, r, act, y, saved)
        check_backward(dy, w, saved, act, *afiv.linear_act_backward(dy, w, saved))


@pytest.mark.parametrize("typ", TYPES)
def test_linear_strides_alignment_and_leading_dimensions(afiv, typ):
    t = TYPES[typ]
    x, w, b, _, dy = inputs(t, 40, 30, 24, 3)
    y = afiv.linear_act(x, w, b, act="silu")
    buf = torch.empty(40 * 30 + 1, dtype=t, device="cuda")[1:].view(40, 30)      # one element off any alignment
    buf.copy_(x)
    assert torch.equal(afiv.linear_act(buf, w, b, act="silu"), y)
    assert torch.equal(afiv.linear_act(x.T.contiguous().T, w.T.contiguous().T, b, act="silu"), y)
    assert torch.equal(afiv.linear_act(x.view(2, 20, 30), w, b, act="silu"), y.view(2, 20, 24))
    y3, s3 = afiv.linear_act_forward(x.view(2, 20, 30), w, b, act="silu", checkpoint8=True)
    y2, s2 = afiv.linear_act_forward(x, w, b, act="silu", checkpoint8=True)
    for a, c in zip(afiv.linear_act_backward(dy.view(2, 20, 24), w, s3), afiv.linear_act_backward(dy.T.contiguous().T, w, s2)):
        assert torch.equal(a.reshape(-1), c.reshape(-1))


@pytest.mark.parametrize("typ", TYPES)
def test_linear_without_rows(afiv, typ):
    x, w, b, r, dy = inputs(TYPES[typ], 0, 12, 5, 1, residual=True)
    for eight in (False, True):
        y, saved = afiv.linear_act_forward(x, w, b, residual=r, act="tanh", checkpoint8=eight)
        dx, dw, db = afiv.linear_act_backward(dy, w, saved)
        assert y.shape == (0, 5) and dx.shape == (0, 12)
        assert not dw.any() and not db.any() and dw.shape == (5, 12)


def test_linear_needed_gradients_only(afiv):
    x, w, b, _, dy = inputs(torch.float32, 300, 40, 50, 2)
    y, saved = afiv.linear_act_forward(x, w, b, act="gelu")
    every = afiv.linear_act_backward(dy, w, saved)
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, True, True), (True, False, True)):
        got = afiv.linear_act_backward(dy, w, saved, need)
        for g, e, n in zip(got, every, need):
            assert (g is None) if not n else torch.equal(g, e)


# at these sizes dz is made by a pass of its own, which sums db as it goes, with or without dW
@pytest.mark.parametrize("typ,m,k,n", [("bf16", 2048, 512, 300), ("f16", 1999, 1001, 515), ("f32", 1024, 1000, 515)])
def test_linear_needed_gradients_only_large(afiv, typ, m, k, n):
    for act in ("none", "gelu", "relu"):
        x, w, b, _, dy = inputs(TYPES[typ], m, k, n, 3)
        y, saved = afiv.linear_act_forward(x, w, b, act=act, checkpoint8=act == "relu")
        every = afiv.linear_act_backward(dy, w, saved)
        check_backward(dy, w, saved, act, *every)
        for need in ((True, False, False), (False, True, False), (False, False, True), (False, True, True), (True, False, True)):
            got = afiv.linear_act_backward(dy, w, saved, need)
            for g, e, wanted in zip(got, every, need):
                assert (g is None) if not wanted else torch.equal(g, e)


@pytest.mark.parametrize("typ", TYPES)
def test_linear_values_that_are_not_finite(afiv, typ):
    """An infinity or NaN of one row reaches that row of y and no other; in FP32 so do magnitudes that do
    not split into three parts."""
    t = TYPES[typ]
    for m, k, n in ((8, 70, 30), (200, 70, 30), (1500, 136, 520)):      # the kernels for few rows, small and large products
        x, w, b, _, dy = inputs(t, m, k, n, 9)
        w = w.abs() + 0.01
        clean = afiv.linear_act(x, w, b)
        for bad in (float("inf"), float("-inf"), float("nan"), torch.finfo(t).max / 16):
            xb = x.clone()
            xb[3, 5] = bad
            y = afiv.linear_act(xb, w, b)
            want = (xb.double() @ w.double().T + b.double()).to(t)
            assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(torch.isinf(y), torch.isinf(want))
            assert torch.equal(y[3][torch.isinf(want[3])], want[3][torch.isinf(want[3])])
            rows = torch.arange(m, device="cuda") != 3
            tol = 300 * U * (1 + clean.double().abs()) * k + half(t) * clean.double().abs()
            within(y[rows], clean.double()[rows], 2 * tol[rows], "other rows")
            fin = torch.isfinite(want[3])
            assert torch.allclose(y[3][fin].double(), want[3][fin].double(), rtol=4 * half(t) + 1e-5)
    # a gradient: row 3 of dy, and a column of it
    for m, k, n in ((200, 70, 30), (1500, 520, 1030)):
        for eight in (False, True):
            x, w, b, _, dy = inputs(t, m, k, n, 9)
            y, saved = afiv.linear_act_forward(x, w, b, act="tanh", checkpoint8=eight)
            row = dy.clone()
            row[3] = float("inf")
            dx, dw, db = afiv.linear_act_backward(row, w, saved)
            assert not torch.isfinite(dx[3]).any() and torch.isfinite(dx[torch.arange(m, device="cuda") != 3]).all()
            if not eight:                                   # a derivative of 0 in 8 bits makes NaN, which is not finite either
                assert not torch.isfinite(dw).all(1).any() and not torch.isfinite(db).any()
            clean = afiv.linear_act_backward(dy, w, saved)
            dy[5, 7] = float("nan")
            dx, dw, db = afiv.linear_act_backward(dy, w, saved)
            rows, cols = torch.arange(m, device="cuda") != 5, torch.arange(n, device="cuda") != 7
            assert torch.isnan(dx[5]).all() and torch.equal(dx[rows], clean[0][rows])
            assert torch.isnan(dw[7]).all() and torch.equal(dw[cols], clean[1][cols]) and torch.isnan(db[7]) and torch.equal(db[cols], clean[2][cols])


def test_linear_small_magnitudes(afiv):
    """FP16 and BF16 subnormals count at full value."""
    for t, v in ((torch.float16, 2.0 ** -20), (torch.bfloat16, 2.0 ** -130)):
        big = 2.0 ** 15 if t == torch.float16 else 2.0 ** 120
        for m in (4, 100):
            x = torch.full((m, 64), v, dtype=t, device="cuda")
            w = torch.full((8, 64), big, dtype=t, device="cuda")
            assert torch.equal(afiv.linear_act(x, w), torch.full((m, 8), v * big * 64, dtype=t, device="cuda"))


def test_linear_is_deterministic(afiv):
    for typ, m, k, n in (("f32", 5000, 24, 40), ("bf16", 5000, 130, 70), ("bf16", 100, 3000, 100)):
        x, w, b, r, dy = inputs(TYPES[typ], m, k, n, 4)
        runs = []
        for _ in range(3):
            y, saved = afiv.linear_act_forward(x, w, b, act="gelu", checkpoint8=True)
            runs.append((y, *afiv.linear_act_backward(dy, w, saved)))
        for other in runs[1:]:
            assert all(torch.equal(a, c) for a, c in zip(runs[0], other))


def test_linear_offsets_beyond_32_bits(afiv):
    """More than 2^31 elements in x and dx: the last rows are those of a small call."""
    m, k, n = (1 << 21) + 5, 1030, 9
    w = torch.randn(n, k, device="cuda").bfloat16()
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    x[-300:] = torch.randn(300, k, device="cuda").bfloat16()
    y, saved = afiv.linear_act_forward(x, w, act="relu", checkpoint8=True)
    check_forward(x[-300:], w, None, None, "relu", y[-300:])
    assert not y[:-300].any()
    dy = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    dy[-300:] = torch.randn(300, n, device="cuda").bfloat16()
    dx, dw, db = afiv.linear_act_backward(dy, w, saved)
    y2, saved2 = afiv.linear_act_forward(x[-300:], w, act="relu", checkpoint8=True)
    dx2, dw2, db2 = afiv.linear_act_backward(dy[-300:], w, saved2)
    assert torch.equal(dx[-300:], dx2) and not dx[:-300].any()
    assert torch.equal(saved.eight.codes[-300:], saved2.eight.codes)
    within(dw, dw2.double(), dw2.double().abs() * 2 * half(torch.bfloat16) + 1e-3, "dw")
    within(db, db2.double(), db2.double().abs() * 2 * half(torch.bfloat16) + 1e-3, "db")


@pytest.mark.parametrize("eight", [False, True])
def test_linear_autograd(afiv, eight):
    x, w, b, r, dy = inputs(torch.float32, 50, 20, 30, 8, residual=True)
    y0, saved = afiv.linear_act_forward(x, w, b, residual=r, act="tanh", checkpoint8=eight)
    want = afiv.linear_act_backward(dy, w, saved)
    leaves = [v.clone().requires_grad_() for v in (x, w, b, r)]
    y = afiv.linear_act(leaves[0], leaves[1], leaves[2], residual=leaves[3], act="tanh", checkpoint8=eight)
    assert torch.equal(y, y0)
    y.backward(dy)
    for v, g in zip(leaves, (*want, dy)):
        assert torch.equal(v.grad, g)
    # an expanded output gradient, a leaf that needs none
    x1 = x.clone().requires_grad_()
    afiv.linear_act(x1, w, b, act="tanh", checkpoint8=eight).sum().backward()
    one = afiv.linear_act_backward(torch.ones_like(dy), w, afiv.linear_act_forward(x, w, b, act="tanh", checkpoint8=eight)[1])
    assert torch.equal(x1.grad, one[0])
    # the same tensor as input and residual: its gradients add up
    sq = torch.randn(20, 20, device="cuda")
    x2 = x.clone().requires_grad_()
    afiv.linear_act(x2, sq, residual=x2, act="silu").backward(x)
    s = afiv.linear_act_forward(x, sq, residual=x, act="silu")[1]
    assert torch.equal(x2.grad, afiv.linear_act_backward(x, sq, s)[0] + x)
    with pytest.raises(RuntimeError):                       # an input changed between the passes
        w1 = w.clone().requires_grad_()
        out = afiv.linear_act(x, w1, b)
        with torch.no_grad():
            w1.mul_(2)
        out.sum().backward()


@pytest.mark.parametrize("act", ACTS)
def test_linear_gradient_against_differences(afiv, act):
    """Central differences of the FP32 operator itself.  Their truncation error is that of the 64-bit formula's
    differences at the same points; FP32 adds the error of two sums of outputs over 2 h."""
    x, w, b, _, dy = inputs(torch.float32, 24, 18, 20, 11)
    g = torch.Generator(device="cuda").manual_seed(12)
    dirs = [torch.randn(v.shape, generator=g, device="cuda") for v in (x, w, b)]
    step = 2.0 ** -7

    def value64(s):
        z = (x.double() + s * dirs[0].double()) @ (w.double() + s * dirs[1].double()).T + b.double() + s * dirs[2].double()
        return (act64(z, act) * dy.double()).sum()

    def value(s):
        xs, ws, bs = (v + s * d for v, d in zip((x, w, b), dirs))
        return (afiv.linear_act(xs, ws, bs, act=act).double() * dy.double()).sum(), xs, ws, bs
    _, saved = afiv.linear_act_forward(x, w, b, act=act)
    grads = afiv.linear_act_backward(dy, w, saved)
    got = sum((gr.double() * d.double()).sum() for gr, d in zip(grads, dirs))
    up, down = value(step), value(-step)
    z = x.double() @ w.double().T + b.double()
    d = der64(z, act) * dy.double()
    exact = (d @ w.double() * dirs[0].double()).sum() + (d.T @ x.double() * dirs[1].double()).sum() + (d.sum(0) * dirs[2].double()).sum()
    truncation = ((value64(step) - value64(-step)) / (2 * step) - exact).abs()
    mag = (x.double().abs() + step * dirs[0].double().abs()) @ (w.double().abs() + step * dirs[1].double().abs()).T + b.double().abs() + 1
    rounding = ((2 * 18 + 40) * U * mag * dy.double().abs()).sum() / step
    assert abs(got - (up[0] - down[0]) / (2 * step)) <= truncation + rounding + 1e-4 * abs(exact)


def test_linear_refusals(afiv):
    x, w, b, r, dy = inputs(torch.float32, 6, 5, 4, 1, residual=True)
    bad = [lambda: afiv.linear_act(x, w.half(), b), lambda: afiv.linear_act(x, w[:, :4], b), lambda: afiv.linear_act(x, w, b[:3]),
           lambda: afiv.linear_act(x, w, b, residual=r[:5]), lambda: afiv.linear_act(x.double(), w.double()), lambda: afiv.linear_act(x, w.cpu()),
           lambda: afiv.linear_act(x[:, :0], w[:, :0]), lambda: afiv.linear_act(x, w[:0]), lambda: afiv.linear_act(x, w, b, residual=r[0]),
           lambda: afiv.linear_act(x, w, b, act="elu"), lambda: afiv.linear_act(x.int(), w.int()), lambda: afiv.linear_act(x, w.view(-1))]
    _, saved = afiv.linear_act_forward(x, w, b, act="tanh")
    bad += [lambda: afiv.linear_act_backward(dy[:5], w, saved), lambda: afiv.linear_act_backward(dy.half(), w.half(), saved),
            lambda: afiv.linear_act_backward(dy, w[:, :4], saved), lambda: afiv.linear_act_backward(dy.cpu(), w, saved)]
    # saved tensors of another call: another width, another batch, a derivative that is missing
    import dataclasses
    other = afiv.linear_act_forward(x, w[:3], b[:3], act="tanh", checkpoint8=True)[1]
    bad += [lambda: afiv.linear_act_backward(dy, w, other), lambda: afiv.linear_act_backward(dy, w, dataclasses.replace(saved, pre=saved.pre[:5])),
            lambda: afiv.linear_act_backward(dy, w, dataclasses.replace(saved, pre=None)),
            lambda: afiv.linear_act_backward(dy, w, dataclasses.replace(saved, pre=saved.pre.half())),
            lambda: afiv.Checkpoint8(other.eight.codes, other.eight.scales[:5], torch.float32),
            lambda: afiv.Checkpoint8(other.eight.codes.T, other.eight.scales, torch.float32),
            lambda: afiv.Checkpoint8(other.eight.codes, other.eight.scales, torch.float64)]
    for call in bad:
        with pytest.raises((ValueError, TypeError)):
            call()


# ---- 8-bit checkpoints -----------------------------------------------------------------------
def oracle_eight(x):
    """(values, E) of the 8-bit format, block by block, in 64 bits."""
    m, k = x.shape
    v = x.double().cpu().numpy()
    out, es = np.empty((m, k)), np.empty((m, (k + 31) // 32), dtype=np.uint8)
    for lo in range(0, k, 32):
        blk = v[:, lo:lo + 32]
        fin = np.isfinite(blk)
        top = np.where(fin, np.abs(blk), 0).max(axis=1)
        e = np.maximum(np.frexp(np.maximum(top, 2.0 ** -140))[1] - 1, -126)
        q = np.clip(np.rint(np.ldexp(np.where(fin, blk, 0), (6 - e)[:, None])), -127, 127)
        out[:, lo:lo + 32] = np.where(fin, np.ldexp(q, (e - 6)[:, None]), np.nan)
        es[:, lo // 32] = e + 127
    return out, es


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 31), (4, 32), (7, 33), (2, 64), (9, 100), (1001, 333), (3, 4096)])
def test_checkpoint_is_the_format(afiv, typ, rows, cols):
    t = TYPES[typ]
    g = torch.Generator(device="cuda").manual_seed(rows * cols)
    x = (torch.randn(rows, cols, generator=g, device="cuda") * torch.exp(3 * torch.randn(rows, 1, generator=g, device="cuda"))).to(t)
    x = x * (torch.rand(rows, cols, generator=g, device="cuda") > 0.15)
    c = afiv.checkpoint8(x)
    want, es = oracle_eight(x)
    assert np.array_equal(c.scales.cpu().numpy(), es)
    back = c.restore()
    assert back.dtype == t and back.shape == x.shape and np.array_equal(back.double().cpu().numpy(), want)
    assert c.nbytes == rows * cols + rows * ((cols + 31) // 32)
    # at most half a step, 2^(E - 6) / 2; less than a step above 127.5 steps
    step = torch.exp2(c.scales.double() - 133).repeat_interleave(32, 1)[:, :cols]
    off = (back.double() - x.double()).abs()
    assert (off <= torch.where(x.double().abs() > 127.5 * step, step, step / 2)).all()
    assert torch.equal(afiv.checkpoint8(x.view(1, rows, cols)).restore()[0], back)
    again = afiv.checkpoint8(back)                          # what is on the grid stays there
    assert torch.equal(again.restore(), back)


@pytest.mark.parametrize("typ", TYPES)
def test_checkpoint_of_unusual_values(afiv, typ):
    t = TYPES[typ]
    f = torch.finfo(t)
    x = torch.zeros(12, 40, dtype=t, device="cuda")
    x[1, 3] = f.max
    x[1, 4] = -f.max
    x[2, 0], x[2, 1], x[2, 2] = float("inf"), float("nan"), 1.5
    x[3] = float("nan")
    x[4, 7] = f.smallest_normal
    x[5, 7], x[5, 8] = f.smallest_normal * f.eps, -f.smallest_normal * f.eps * 3      # subnormal
    x[6, :3] = torch.tensor([1.0, 1.5 / 64, 2.5 / 64])                               # ties go to even
    x[7, :2] = torch.tensor([1.9999, 1.99])                                          # the top of a binade saturates
    x[8, 33] = float("-inf")
    x[9, 39] = -1.0
    c = afiv.checkpoint8(x)
    want, es = oracle_eight(x)
    assert np.array_equal(c.scales.cpu().numpy(), es)
    back = c.restore()
    assert np.array_equal(back.double().cpu().numpy(), want, equal_nan=True)
    assert torch.isfinite(back[1]).all() and not back[0].any()
    assert back[6, 1].item() == 2 / 64 and back[6, 2].item() == 2 / 64
    # 1.9999 is the number 2 in the 16-bit types, whose steps below 2 are 2^-10 and 2^-7: there it stays what it is
    assert back[7, 0].item() == (127 / 64 if t == torch.float32 else 2.0)


def test_checkpoint_edges(afiv):
    e = afiv.checkpoint8(torch.empty(0, 5, device="cuda"))
    assert e.restore().shape == (0, 5)
    x = torch.randn(11, 50, device="cuda")
    assert torch.equal(afiv.checkpoint8(x.T).restore(), afiv.checkpoint8(x.T.contiguous()).restore())
    assert torch.equal(afiv.checkpoint8(x[0]).restore(), afiv.checkpoint8(x).restore()[0])
    for bad in (torch.zeros(3, 4, dtype=torch.float64, device="cuda"), torch.zeros(3, 0, device="cuda"), torch.zeros((), device="cuda")):
        with pytest.raises((TypeError, ValueError)):
            afiv.checkpoint8(bad)


def test_checkpoint_offsets_beyond_32_bits(afiv):
    rows, cols = (1 << 20) + 3, 2056
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[-5:] = torch.randn(5, cols, device="cuda").bfloat16()
    back = afiv.checkpoint8(x).restore()
    assert torch.equal(back[-5:], afiv.checkpoint8(x[-5:]).restore()) and not back[:-5].any()


# ---- batch norm, activation, dropout -----------------------------------------------------------
def norm_inputs(t, m, n, seed, drop=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(m, n, generator=g, device="cuda") * (0.2 + torch.rand(n, generator=g, device="cuda")) + 2 * torch.randn(n, generator=g, device="cuda")
    gamma, beta = 0.5 + torch.rand(n, generator=g, device="cuda"), torch.randn(n, generator=g, device="cuda") * 0.3
    keep = torch.rand(m, n, generator=g, device="cuda") >= 0.3 if drop else None
    return x.to(t), gamma, beta, keep, torch.randn(m, n, generator=g, device="cuda").to(t)


def check_norm(x, gamma, beta, keep, p, act, dy, y, saved, dx, dgamma, dbeta, eps=1e-5):
    t, (m, n) = x.dtype, x.shape
    xd, ga, be = x.double(), gamma.double(), beta.double()
    mu = xd.mean(0)
    rstd = 1 / torch.sqrt((xd - mu).square().mean(0) + eps)
    s = 1.0 / (1.0 - p)
    k = torch.ones_like(xd) if keep is None else keep.double()
    z = (xd - mu) * rstd * ga + be
    want = act64(z, act) * k * s
    # FP64 inside (its cancellation, 1e-16 mu^2 / var, is far below u); z, f and the scale round in FP32
    tol = s * 20 * U * (1 + z.abs())
    within(y, want, tol + (want.abs() + tol) * half(t) + tiny(t), "y")
    within(saved.stats[0], mu, 1e-13 * (1 + mu.abs()), "mean")
    within(saved.stats[1], rstd, 1e-10 * rstd * (1 + (mu * rstd).square()), "rstd")
    xs = xd if saved.eight is None else saved.eight.restore().double()
    h = (xs - mu) * rstd
    z = h * ga + be
    g = dy.double() * k * s * der64(z, act)
    eg = 24 * U * dy.double().abs() * k * s * (1 + SECOND[act] * z.abs())
    sb, sg = g.sum(0), (g * h).sum(0)
    eb, egg = eg.sum(0), (eg * h.abs() + 4 * U * (g * h).abs()).sum(0)
    within(dbeta, sb, eb + 2 * U * sb.abs() + 1e-30, "dbeta")
    within(dgamma, sg, egg + 2 * U * sg.abs() + 1e-30, "dgamma")
    want = ga * rstd * (g - sb / m - h * sg / m)
    tol = ga * rstd * (eg + eb / m + h.abs() * egg / m + 8 * U * (g.abs() + sb.abs() / m + (h * sg).abs() / m))
    within(dx, want, tol + (want.abs() + tol) * half(t) + tiny(t), "dx")


@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("m,n", [(2, 1), (2, 128), (3, 33), (64, 13), (64, 128), (100, 31), (1024, 40), (1025, 40), (1500, 7), (3000, 65), (2500, 333), (20000, 5)])
def test_norm_forward_and_backward(afiv, typ, m, n):
    t = TYPES[typ]
    for i, act in enumerate(ACTS):
        x, gamma, beta, keep, dy = norm_inputs(t, m, n, m + n + i, drop=i % 3 != 0)
        p = 0.3 if keep is not None else 0.0
        for eight in (False, True):
            rm, rv = torch.randn(n, device="cuda"), torch.rand(n, device="cuda")
            rm0, rv0 = rm.double(), rv.double()
            y, saved = afiv.batch_norm_act_forward(x, gamma, beta, rm, rv, act=act, keep=keep, drop_p=p, momentum=0.2, checkpoint8=eight)
            dx, dgamma, dbeta = afiv.batch_norm_act_backward(dy, gamma, beta, saved)
            check_norm(x, gamma, beta, keep, p, act, dy, y, saved, dx, dgamma, dbeta)
            if eight:
                assert torch.equal(saved.eight.codes, afiv.checkpoint8(x).codes) and torch.equal(saved.eight.scales, afiv.checkpoint8(x).scales)
            var, mean = torch.var_mean(x.double(), dim=0, correction=1)
            within(rm, 0.8 * rm0 + 0.2 * mean, 4 * U * (rm0.abs() + mean.abs()), "running mean")
            within(rv, 0.8 * rv0 + 0.2 * var, 4 * U * (rv0 + var) + 1e-13 * mean.square(), "running var")


# workgroups whose last lanes have no columns, or some of theirs, beside full ones
@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("m,n", [(700, 300), (700, 299), (1100, 300), (1100, 299), (1100, 3), (4100, 76)])
def test_norm_ragged_workgroups(afiv, typ, m, n):
    test_norm_forward_and_backward(afiv, typ, m, n)


def test_norm_matches_torch_modules(afiv):
    x, gamma, beta, _, dy = norm_inputs(torch.float32, 300, 50, 4, drop=False)
    bn = torch.nn.BatchNorm1d(50).cuda()
    with torch.no_grad():
        bn.weight.copy_(gamma), bn.bias.copy_(beta)
    x1, x2 = x.clone().requires_grad_(), x.clone().requires_grad_()
    ga, be = gamma.clone().requires_grad_(), beta.clone().requires_grad_()
    rm, rv = torch.zeros(50, device="cuda"), torch.ones(50, device="cuda")
    version = rm._version
    torch.tanh(bn(x1)).backward(dy)
    afiv.batch_norm_act(x2, ga, be, rm, rv, act="tanh").backward(dy)
    assert rm._version > version and rv._version > version
    for a, b in ((x1.grad, x2.grad), (bn.weight.grad, ga.grad), (bn.bias.grad, be.grad), (bn.running_mean, rm), (bn.running_var, rv)):
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("m", [50, 2000])
def test_norm_extremes(afiv, m):
    x, gamma, beta, keep, dy = norm_inputs(torch.float32, m, 40, 6)
    # a mask that leaves nothing: zeros, and no gradient but beta's share of none
    none = torch.zeros_like(keep)
    y, saved = afiv.batch_norm_act_forward(x, gamma, beta, act="gelu", keep=none, drop_p=0.3)
    dx, dgamma, dbeta = afiv.batch_norm_act_backward(dy, gamma, beta, saved)
    assert not y.any() and not dx.any() and not dgamma.any() and not dbeta.any()
    # a constant column: variance 0, rstd = 1 / sqrt(eps)
    x[:, 7] = 3.25
    y, saved = afiv.batch_norm_act_forward(x, gamma, beta)
    assert torch.equal(y[:, 7], beta[7].expand(m)) and abs(float(saved.stats[1, 7]) - 1e-5 ** -0.5) < 1e-6
    # a far-off column: FP64 sums keep its variance
    x[:, 8] = 1e5 + torch.randn(m, device="cuda")
    y, saved = afiv.batch_norm_act_forward(x, gamma, beta)
    check_norm(x, gamma, beta, None, 0.0, "none", dy, y, saved, *afiv.batch_norm_act_backward(dy, gamma, beta, saved))
    # NaN stays in its column, also through the 8-bit checkpoint
    x[1, 9] = float("nan")
    for eight in (False, True):
        y, saved = afiv.batch_norm_act_forward(x, gamma, beta, act="tanh", checkpoint8=eight)
        dx, dgamma, dbeta = afiv.batch_norm_act_backward(dy, gamma, beta, saved)
        cols = torch.arange(40, device="cuda") != 9
        assert torch.isnan(y[:, 9]).all() and torch.isfinite(y[:, cols]).all() and torch.isfinite(dx[:, cols]).all()
        assert torch.isnan(dx[:, 9]).all() and torch.isnan(dgamma[9]) and torch.isfinite(dgamma[cols]).all()
    # a dropped element is 0 whatever its activation
    big = torch.full((m, 4), 3e38, device="cuda")
    big[::2] = -3e38
    y, _ = afiv.batch_norm_act_forward(big, gamma[:4], beta[:4], keep=torch.zeros(m, 4, dtype=torch.uint8, device="cuda"), drop_p=0.5)
    assert not y.any()


def test_norm_strides_and_determinism(afiv):
    for m, n in ((60, 37), (5000, 37)):
        x, gamma, beta, keep, dy = norm_inputs(torch.bfloat16, m, n, 3)
        first = None
        for xx, kk, dd in ((x, keep, dy), (x, keep.to(torch.uint8), dy), (x.T.contiguous().T, keep.T.contiguous().T, dy.T.contiguous().T),
                           (torch.empty(m * n + 1, dtype=x.dtype, device="cuda")[1:].view(m, n).copy_(x), keep, dy)):
            y, saved = afiv.batch_norm_act_forward(xx, gamma, beta, act="silu", keep=kk, drop_p=0.3, checkpoint8=True)
            got = (y, *afiv.batch_norm_act_backward(dd, gamma, beta, saved))
            first = first or got
            assert all(torch.equal(a, b) for a, b in zip(first, got))
        only = afiv.batch_norm_act_backward(dy, gamma, beta, saved, need_dx=False)
        assert only[0] is None and torch.equal(only[1], first[2]) and torch.equal(only[2], first[3])


def test_norm_refusals(afiv):
    x, gamma, beta, keep, dy = norm_inputs(torch.float32, 8, 6, 1)
    rm = torch.zeros(6, device="cuda")
    bad = [lambda: afiv.batch_norm_act(x[:1], gamma, beta), lambda: afiv.batch_norm_act(x, gamma[:5], beta), lambda: afiv.batch_norm_act(x, gamma.half(), beta),
           lambda: afiv.batch_norm_act(x, gamma, beta, rm), lambda: afiv.batch_norm_act(x, gamma, beta, drop_p=0.2),
           lambda: afiv.batch_norm_act(x, gamma, beta, keep=keep, drop_p=1.0), lambda: afiv.batch_norm_act(x, gamma, beta, keep=keep[:5], drop_p=0.1),
           lambda: afiv.batch_norm_act(x, gamma, beta, keep=keep.float(), drop_p=0.1), lambda: afiv.batch_norm_act(x.view(-1), gamma, beta),
           lambda: afiv.batch_norm_act(x, gamma, beta, torch.zeros(12, device="cuda")[::2], torch.ones(12, device="cuda")[::2]),
           lambda: afiv.batch_norm_act(x, gamma.cpu(), beta), lambda: afiv.batch_norm_act(x.double(), gamma, beta)]
    saved = afiv.batch_norm_act_forward(x, gamma, beta)[1]
    bad += [lambda: afiv.batch_norm_act_backward(dy[:4], gamma, beta, saved), lambda: afiv.batch_norm_act_backward(dy.half(), gamma, beta, saved)]
    import dataclasses
    bad += [lambda: afiv.batch_norm_act_backward(dy, gamma, beta, dataclasses.replace(saved, stats=saved.stats[:, :5])),
            lambda: afiv.batch_norm_act_backward(dy, gamma, beta, dataclasses.replace(saved, keep=keep[:4]))]
    for call in bad:
        with pytest.raises((ValueError, TypeError)):
            call()


# ---- together ------------------------------------------------------------------------------------
def layer_step(afiv, x, w, b, gamma, beta, keep, dy, eight):
    z, s1 = afiv.linear_act_forward(x, w, b, checkpoint8=eight)
    y, s2 = afiv.batch_norm_act_forward(z, gamma, beta, act="tanh", keep=keep, drop_p=0.3, checkpoint8=eight)
    dz, dgamma, dbeta = afiv.batch_norm_act_backward(dy, gamma, beta, s2)
    dx, dw, db = afiv.linear_act_backward(dz, w, s1)
    return y, dx, dw, db, dgamma, dbeta


@pytest.mark.parametrize("m,k,n", [(64, 13, 128), (3000, 24, 40), (8, 700, 48)])
def test_layer_step_in_graphs_and_streams(afiv, m, k, n):
    """A layer's training step captured twice (two graphs, one pool each) and replayed on new inputs, and run
    eagerly on a stream of its own, equals the eager step bit for bit."""
    x, w, b, _, _ = inputs(torch.float32, m, k, n, 21)
    _, gamma, beta, keep, dy = norm_inputs(torch.float32, m, n, 22)
    static = [[v.clone() for v in (x, w, b, gamma, beta, keep, dy)] for _ in range(2)]
    layer_step(afiv, *static[0], True)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(layer_step(afiv, *static[i], True))
        graphs.append(graph)
    for seed in (31, 32, 33):
        news = []
        for i in range(2):
            new = [torch.randn_like(v) if v.dtype != torch.bool else v for v in static[i]]
            for a, c in zip(static[i], new):
                a.copy_(c)
            news.append(new)
        graphs[0].replay()
        graphs[1].replay()
        eager = [layer_step(afiv, *new, True) for new in news]
        torch.cuda.synchronize()
        for got, want in zip(outs, eager):
            assert all(torch.equal(a, c) for a, c in zip(got, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer_step(afiv, *news[0], True)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(got, eager[0]))


def test_calls_at_once_on_two_streams(afiv):
    x, w, b, _, dy = inputs(torch.bfloat16, 3000, 200, 100, 41)
    want = [afiv.linear_act_backward(dy, w, afiv.linear_act_forward(x, w, b, act=a, checkpoint8=True)[1]) for a in ("gelu", "silu")]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for s, a in zip(streams, ("gelu", "silu")):
            with torch.cuda.stream(s):
                got.append(afiv.linear_act_backward(dy, w, afiv.linear_act_forward(x, w, b, act=a, checkpoint8=True)[1]))
        torch.cuda.synchronize()
        for g, e in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(g, e))

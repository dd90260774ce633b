"""GPU tests of calls of the layer operators that the header and the docstrings allow beside the usual ones: gradients
without the operands they do not need, through the C ABI."""
import ctypes
import dataclasses
import types

import pytest
import torch

from test_gpu_layers import ACTS, SECOND, TYPES, U, check_backward, check_forward, check_norm, der64, half, inputs, tiny, within

pytestmark = pytest.mark.gpu


def abi_backward(afiv, dy, w, saved, k, dx=False, codes=None):
    """(dx, db) through the C ABI with no dW and no input (codes: a pointer without scales)."""
    lib, (m, n), t = afiv._lib.lib(), dy.shape, dy.dtype

    def p(v):
        return None if v is None else ctypes.c_void_p(v.data_ptr())
    out = torch.full((m, k), float("nan"), dtype=t, device="cuda") if dx else None
    db = torch.full((n,), float("nan"), dtype=t, device="cuda")
    dtype, act = afiv.layers.DTYPES[t], afiv.layers.ACTIVATIONS[saved.act]
    need = lib.afiv_linear_act_backward_scratch(m, n, k, dtype, act, 0)
    scratch = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    rc = lib.afiv_linear_act_backward(p(dy), None, p(codes), None, p(w) if dx else None, p(saved.pre), p(saved.dcodes), dtype, act, m, n, k,
                                      p(out), None, p(db), p(scratch) if need else None, need, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    return out, db


# products of every kind: one tile, a sum cut into runs (up to 16 of them, and more), many tiles, a pass over dz that sums it
@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (2, 5, 3), (64, 13, 128), (300, 40, 50), (33, 64, 129), (2500, 24, 130), (40000, 64, 5), (40000, 24, 72),
                                   (700, 1030, 1100), (1999, 1001, 515), (0, 4, 5)])
def test_db_without_the_layers_input(afiv, typ, m, k, n):
    for act, eight in (("none", False), ("gelu", False), ("silu", True), ("relu", False)):
        x, w, b, _, dy = inputs(TYPES[typ], m, k, n, 7)
        _, saved = afiv.linear_act_forward(x, w, b, act=act, checkpoint8=eight)
        every = afiv.linear_act_backward(dy, w, saved)
        if m:
            check_backward(dy, w, saved, act, *every)
        codes = torch.zeros(max(m * k, 1), dtype=torch.int8, device="cuda")
        for want_dx, c in ((False, None), (True, None), (False, codes)):
            dx, db = abi_backward(afiv, dy, w, saved, k, want_dx, c)
            assert torch.equal(db, every[2]), (act, want_dx)
            assert not want_dx or torch.equal(dx, every[0])


@pytest.mark.parametrize("typ", TYPES)
def test_db_without_the_layers_input_of_a_misaligned_gradient(afiv, typ):
    """A size whose dz is read in place, from an address that is no multiple of 16."""
    t = TYPES[typ]
    m, k, n = 1500, 520, 1032
    x, w, b, _, dy = inputs(t, m, k, n, 8)
    off = torch.empty(m * n + 1, dtype=t, device="cuda")[1:].view(m, n).copy_(dy)
    _, saved = afiv.linear_act_forward(x, w, b)
    _, db = abi_backward(afiv, off, w, saved, k)
    want, tol = dy.double().sum(0), 2 * m * U * dy.double().abs().sum(0)
    within(db, want, tol + (want.abs() + tol) * half(t) + tiny(t), "db")
    assert torch.equal(db, afiv.linear_act_backward(off, w, saved)[2])


def test_transforms_that_the_operators_do_not_know(afiv):
    """Forward-mode tangents, and torch.func's wrapped tensors, are refused on every operand; nothing is computed from them."""
    from torch.autograd import forward_ad
    x, w, b, r, dy = inputs(torch.float32, 6, 5, 4, 1, residual=True)
    gamma, beta = torch.ones(5, device="cuda"), torch.zeros(5, device="cuda")
    mean, var = torch.zeros(5, device="cuda"), torch.ones(5, device="cuda")
    _, saved = afiv.linear_act_forward(x, w, b, act="tanh")
    _, norm = afiv.batch_norm_act_forward(x, gamma, beta, act="tanh")
    linear = lambda *a: afiv.linear_act(a[0], a[1], a[2], residual=a[3], act="tanh")      # noqa: E731
    bn = lambda *a: afiv.batch_norm_act(*a, mean, var, act="tanh")                        # noqa: E731
    for call, args in ((linear, (x, w, b, r)), (bn, (x, gamma, beta)), (lambda *a: afiv.linear_act_backward(*a, saved)[0], (dy, w)),
                       (lambda *a: afiv.batch_norm_act_backward(*a, norm)[0], (x, gamma, beta))):
        for i in range(len(args)):
            for grad in (False, True):
                with forward_ad.dual_level():
                    a = [v.clone().requires_grad_(grad) for v in args]
                    a[i] = forward_ad.make_dual(a[i], torch.ones_like(a[i]))
                    with pytest.raises(NotImplementedError, match="tangent"):
                        call(*a)
            rest = list(args)

            def one(v):
                return call(*rest[:i], v, *rest[i + 1:])
            with pytest.raises(NotImplementedError, match="tangent"):
                torch.func.jvp(one, (args[i],), (torch.ones_like(args[i]),))
    for call, args in ((linear, (x, w, b, r)), (bn, (x, gamma, beta))):
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda v: call(v, *args[1:]).sum())(x)
        with pytest.raises(RuntimeError):
            torch.vmap(lambda v: call(v, *args[1:]))(torch.stack([x, x]))
    assert not mean.any() and bool((var == 1).all())


# Relative errors in FP32 half steps: f = (constant of 2^x, the reciprocal, the polynomial and a handful of roundings)
# + (two or three roundings of the exponent's argument, multiplied up by the argument: z^2 / 2 of exp(-z^2 / 2), |z| of
# exp(-|z|), 2 |z| of exp(-2 |z|))
@pytest.mark.parametrize("m", [30, 4000])
def test_activations_keep_their_relative_accuracy_in_the_tails(afiv, m):
    one = torch.ones(1, 1, device="cuda")
    for act, lo, hi in (("gelu", -12.0, 6.0), ("silu", -80.0, 20.0), ("tanh", -30.0, 30.0)):
        x = torch.linspace(lo, hi, m, device="cuda").view(m, 1) + 1e-3          # with one weight of 1 the pre-activation is x itself
        y, saved = afiv.linear_act_forward(x, one, act=act)
        assert torch.equal(saved.pre, x)
        d = afiv.linear_act_backward(torch.ones_like(x), one, saved, (True, False, False))[0].double()
        z, y = x.double(), y.double()
        a = z.abs()
        if act == "gelu":
            tail = 0.5 * torch.special.erfcx(a / 2 ** 0.5) * torch.exp(-z * z / 2)
            phi, pdf = torch.where(z > 0, 1 - tail, tail), torch.exp(-z * z / 2) / (2 * torch.pi) ** 0.5
            value, slope, terms, steps, dsteps = z * phi, phi + z * pdf, phi + a * pdf, 16 + 1.5 * z * z, 16 + 1.5 * z * z
        elif act == "silu":
            p, q = 1 / (1 + torch.exp(-z)), 1 / (1 + torch.exp(z))
            value, slope, terms, steps, dsteps = z * p, p + z * p * q, p + a * p * q, 8 + 2 * a, 8 + 2 * a
        else:
            e = torch.exp(-2 * a)
            value, slope = torch.tanh(z), 4 * e / (1 + e) ** 2
            terms, steps, dsteps = slope, 16.0, 12 + 4 * a
        for got, want, tol, what in ((y, value, steps * U * value.abs(), "value"), (d, slope, dsteps * U * terms, "derivative")):
            off = (got - want).abs() / tol
            assert float(off.max()) <= 1, (act, what, float(off.max()), float(z.flatten()[off.argmax()]))


# The whole gradient, from the layer's inputs and not from what the forward pass saved: the saved pre-activation is rounded
# to T (half(T) |z|, times f''), its side is FP32's (relu, leaky_relu), 8-bit derivatives are off by 1/400 and 8-bit inputs
# by less than a step of their block
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("typ", TYPES)
@pytest.mark.parametrize("m,k,n", [(64, 40, 30), (1500, 264, 520), (1501, 261, 515)])
def test_gradients_against_the_formula_from_the_inputs(afiv, typ, m, k, n, eight):
    t = TYPES[typ]
    for act in ACTS:
        x, w, b, _, dy = inputs(t, m, k, n, 17)
        _, saved = afiv.linear_act_forward(x, w, b, act=act, checkpoint8=eight)
        dx, dw, db = afiv.linear_act_backward(dy, w, saved)
        xd, wd, g = x.double(), w.double(), dy.double()
        z, mag = xd @ wd.T + b.double(), xd.abs() @ wd.abs().T + b.double().abs()
        zerr = (2 * k + 8) * U * mag
        if act in ("relu", "leaky_relu"):
            derr = torch.where(z.abs() <= zerr, 1.0, 0.0).double() + 2 * U
        elif eight and act != "none":
            derr = SECOND[act] * zerr + 16 * U * (1 + z.abs()) + 0.5 / 200 + 4 * U
        else:
            derr = SECOND[act] * (zerr + (z.abs() + zerr) * half(t) + tiny(t)) + 16 * U * (1 + z.abs())
        if act == "none":
            derr = torch.zeros_like(z)
        dz = g * der64(z, act)
        e = g.abs() * derr + 2 * U * dz.abs()
        eh = e + (half(t) * (dz.abs() + e) + tiny(t) if act != "none" and t != torch.float32 else 0.0)
        xerr = torch.zeros_like(xd)
        if eight:
            xerr = torch.exp2(saved.eight.scales.double() - 133).repeat_interleave(32, 1)[:, :k]
        for got, a, c, err, length, what in ((dx, dz, wd, eh @ wd.abs(), n, "dx"),
                                             (dw, dz.T, xd, eh.T @ (xd.abs() + xerr) + dz.abs().T @ xerr, m, "dw")):
            want = a @ c
            tol = err + (2 * length + 8) * U * (a.abs() @ c.abs() + err)
            within(got, want, tol + (want.abs() + tol) * half(t) + tiny(t), what)
        want = dz.sum(0)
        tol = e.sum(0) + 2 * m * U * (dz.abs() + e).sum(0)
        within(db, want, tol + (want.abs() + tol) * half(t) + tiny(t), "db")


@pytest.mark.parametrize("typ", TYPES)
def test_large_products_of_misaligned_operands(afiv, typ):
    """Sizes whose operands are read in place where they are aligned; here each in turn, and all, stand one element off."""
    t = TYPES[typ]
    m, k, n = 1500, 520, 1032
    x, w, b, r, dy = inputs(t, m, k, n, 9, residual=True)

    def off(v):
        return torch.empty(v.numel() + 1, dtype=t, device="cuda")[1:].view(v.shape).copy_(v)
    for which in ("x", "w", "dy", "all"):
        xs, ws, ds = (off(v) if which in (name, "all") else v for name, v in (("x", x), ("w", w), ("dy", dy)))
        bs, rs = (off(b), off(r)) if which == "all" else (b, r)
        for act, eight in (("none", False), ("gelu", False), ("leaky_relu", True)):
            y, saved = afiv.linear_act_forward(xs, ws, bs, residual=rs, act=act, checkpoint8=eight)
            check_forward(x, w, b, r, act, y, saved)
            check_backward(dy, w, saved, act, *afiv.linear_act_backward(ds, ws, saved))


@pytest.mark.parametrize("typ,m,k,n", [("f16", 1501, 777, 1029), ("bf16", 2048, 512, 1024), ("f32", 2048, 260, 515)])
def test_large_steps_in_graphs_and_on_streams(afiv, typ, m, k, n):
    """Steps whose operands are prepared in scratch memory: two captured graphs replayed on new inputs, and two streams at
    once, give the eager step's bits."""
    def step(x, w, b, dy, act):
        y, saved = afiv.linear_act_forward(x, w, b, act=act, checkpoint8=True)
        return (y, *afiv.linear_act_backward(dy, w, saved))
    acts = ("gelu", "tanh")
    static = [[v for v in inputs(TYPES[typ], m, k, n, 50 + i) if v is not None] for i in range(2)]
    step(*static[0], "gelu")
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s, act in zip(static, acts):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(*s, act))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for seed in (60, 70, 80):
        news = [[v for v in inputs(TYPES[typ], m, k, n, seed + i) if v is not None] for i in range(2)]
        for s, new in zip(static, news):
            for a, c in zip(s, new):
                a.copy_(c)
        for g in graphs:
            g.replay()
        eager = [step(*new, act) for new, act in zip(news, acts)]
        torch.cuda.synchronize()
        at_once = []
        for new, act, stream in zip(news, acts, streams):
            with torch.cuda.stream(stream):
                at_once.append(step(*new, act))
        torch.cuda.synchronize()
        for got in (outs, at_once):
            assert all(torch.equal(a, c) for g, e in zip(got, eager) for a, c in zip(g, e))


@pytest.mark.parametrize("k,n", [(264, 136), (261, 131)])
def test_large_products_beyond_32_bits(afiv, k, n):
    """More than 2^31 elements in x and dx, through the kernels for large products: rows at the start, about the 2^31st
    element, about the 2^32nd byte and at the end; the others are zeros."""
    m = (1 << 23) + 77
    torch.manual_seed(13)
    w = torch.randn(n, k, device="cuda").half()
    x, dy = torch.zeros(m, k, dtype=torch.float16, device="cuda"), torch.zeros(m, n, dtype=torch.float16, device="cuda")
    cross = (1 << 31) // k
    rows = torch.cat([torch.arange(a, b, device="cuda") for a, b in ((0, 60), (cross // 2 - 40, cross // 2 + 40), (cross - 40, cross + 40), (m - 150, m))])
    x[rows], dy[rows] = torch.randn(len(rows), k, device="cuda").half(), torch.randn(len(rows), n, device="cuda").half()
    for eight in (False, True):
        y, saved = afiv.linear_act_forward(x, w, act="relu", checkpoint8=eight)
        assert int(y.any(1).sum()) == int(y[rows].any(1).sum())
        dx, dw, db = afiv.linear_act_backward(dy, w, saved)
        few = dataclasses.replace(afiv.linear_act_forward(x[rows], w, act="relu", checkpoint8=eight)[1], dcodes=saved.dcodes[rows])
        check_forward(x[rows], w, None, None, "relu", y[rows], few)
        assert not eight or torch.equal(saved.eight.codes[rows], few.eight.codes)
        check_backward(dy[rows], w, few, "relu", dx[rows], dw, db)          # rows of zeros add nothing to dW and db
        assert int(dx.any(1).sum()) == int(dx[rows].any(1).sum())
        del y, dx, saved


def test_norm_beyond_32_bits(afiv):
    """More than 2^31 elements: columns at both ends against the formula (a column's result depends on it alone)."""
    m, n = (1 << 22) + 5, 520
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(m, n, generator=g, device="cuda", dtype=torch.float16)
    dy = torch.randn(m, n, generator=g, device="cuda", dtype=torch.float16)
    keep = torch.rand(m, n, generator=g, device="cuda", dtype=torch.float16) >= 0.25
    gamma, beta = 0.5 + torch.rand(n, generator=g, device="cuda"), torch.randn(n, generator=g, device="cuda")
    for eight in (False, True):
        y, saved = afiv.batch_norm_act_forward(x, gamma, beta, act="silu", keep=keep, drop_p=0.25, checkpoint8=eight)
        dx, dgamma, dbeta = afiv.batch_norm_act_backward(dy, gamma, beta, saved)
        back = saved.eight.restore() if eight else None
        for c in (slice(0, 3), slice(n - 3, n)):
            part = types.SimpleNamespace(stats=saved.stats[:, c], eight=types.SimpleNamespace(restore=lambda: back[:, c]) if eight else None)
            check_norm(x[:, c], gamma[c], beta[c], keep[:, c], 0.25, "silu", dy[:, c], y[:, c], part, dx[:, c], dgamma[c], dbeta[c])
        del y, dx, saved, back

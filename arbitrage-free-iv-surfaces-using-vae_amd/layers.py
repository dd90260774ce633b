"""Layer operators over the C ABI: a linear layer with bias, activation and residual; training-mode
batch normalisation with activation and dropout; 8-bit activation checkpoints.

These are the pieces of the conditional VAE's [Linear, BatchNorm1d, activation, Dropout] stacks
(cvae_model.py:64-105), forward and backward, for layers of any width.  ``linear_act`` and
``batch_norm_act`` are differentiable in reverse mode; their ``_forward`` / ``_backward`` halves are for training
loops that hold the backward pass themselves (graph capture, pipelines).  Forward-mode tangents are refused.  Every function takes CUDA tensors
in float32, bfloat16 or float16, enqueues on torch's current stream of the tensors' device and does not
synchronise.  Inputs that are not contiguous are copied first.
"""
from __future__ import annotations

from dataclasses import dataclass
from functools import lru_cache

import torch
from torch.autograd import forward_ad

from . import _lib

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
ACTIVATIONS = {"none": 0, "relu": 1, "leaky_relu": 2, "tanh": 3, "gelu": 4, "silu": 5}
NORM_SCRATCH_DOUBLES = 2 * 256 + 2      # afiv.h: AFIV_NORM_SCRATCH_DOUBLES, per column
NORM_SMALL_ROWS = 1024                  # afiv.h: AFIV_NORM_SMALL_ROWS, up to which none is needed


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _run(name: str, device: torch.device, *args) -> None:
    """One call of the library on the current stream of ``device``."""
    fn, index = getattr(_lib.lib(), name), device.index
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc, name)


def _act(name: str) -> int:
    try:
        return ACTIVATIONS[name]
    except (KeyError, TypeError):
        raise ValueError(f"unknown activation {name!r}: one of {', '.join(ACTIVATIONS)}") from None


def _refuse_tangent(t: torch.Tensor, what: str) -> None:
    """Inside a forward-mode level: the kernels would drop a tangent, which reads as a derivative of zero."""
    if forward_ad.unpack_dual(t).tangent is not None:
        raise NotImplementedError(f"{what} has a forward-mode tangent: the layer operators differentiate in reverse mode only")


def _first(x, what: str) -> torch.Tensor:
    """The operand that sets the device and the element type."""
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{what} must be a torch.Tensor")
    if forward_ad._current_level >= 0:
        _refuse_tangent(x, what)
    if not x.is_cuda:
        raise ValueError(f"{what} is on {x.device}: the layer kernels need a GPU (no CPU fallback)")
    if x.dtype not in DTYPES:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, got {x.dtype}")
    return _plain(x)


def _plain(t: torch.Tensor) -> torch.Tensor:
    if t.requires_grad:
        t = t.detach()
    return t if t.is_contiguous() else t.contiguous()


def _like(t, x: torch.Tensor, shape, what: str, dtypes=None, output: bool = False) -> torch.Tensor:
    """Another operand: on x's device, of x's type (or one of ``dtypes``), of the given shape."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a torch.Tensor")
    if forward_ad._current_level >= 0:
        _refuse_tangent(t, what)
    if t.get_device() != x.get_device():
        raise ValueError(f"{what} is on {t.device}, expected {x.device}")
    if (t.dtype != x.dtype) if dtypes is None else (t.dtype not in dtypes):
        raise TypeError(f"{what} must be {' or '.join(map(str, dtypes or (x.dtype,)))}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{what} must be {list(shape)}, got {list(t.shape)}")
    if output and not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous: the kernels write into it in place")
    return _plain(t)


def _held(t, x: torch.Tensor, shape, what: str, dtype=None) -> None:
    """A saved tensor, if there is one, is what the forward pass made for such an output gradient x."""
    if t is not None and (t.get_device() != x.get_device() or t.shape != shape or not t.is_contiguous() or (dtype is not None and t.dtype != dtype)):
        raise ValueError(f"{what} ({t.dtype} {list(t.shape)} on {t.device}) does not belong to dy {list(x.shape)} on {x.device}")


def _made(cls, **fields):
    """A frozen record of tensors that were made here: its checks, and a setattr a field, are for callers'."""
    record = object.__new__(cls)
    record.__dict__.update(fields)
    return record


def _rows(x: torch.Tensor, what: str) -> int:
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{what} must be [..., features] with at least one feature, got {list(x.shape)}")
    return x.numel() // x.shape[-1]


# ---- 8-bit checkpoints -----------------------------------------------------------------------
@dataclass(frozen=True)
class Checkpoint8:
    """A tensor in 8 bits (see afiv_checkpoint8_pack): ``codes`` int8 of its shape and one ``scales``
    byte per 32 elements of a row."""
    codes: torch.Tensor
    scales: torch.Tensor
    dtype: torch.dtype

    def __post_init__(self):
        c, s = self.codes, self.scales
        if c.dtype != torch.int8 or s.dtype != torch.uint8 or self.dtype not in DTYPES:
            raise TypeError("a checkpoint is int8 codes, uint8 scales and a float32, bfloat16 or float16 dtype")
        if c.dim() < 1 or c.shape[-1] < 1 or s.shape != c.shape[:-1] + ((c.shape[-1] + 31) // 32,) or c.device != s.device \
                or not (c.is_contiguous() and s.is_contiguous()):
            raise ValueError(f"codes {list(c.shape)} and scales {list(s.shape)} are not one contiguous checkpoint")

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    @property
    def nbytes(self) -> int:
        return self.codes.numel() + self.scales.numel()

    def restore(self) -> torch.Tensor:
        """The tensor the codes stand for, in the type it was packed from."""
        out = self.codes.new_empty(self.codes.shape, dtype=self.dtype)
        cols = out.shape[-1]
        _run("afiv_checkpoint8_restore", out.device, self.codes.data_ptr(), self.scales.data_ptr(), DTYPES[self.dtype],
             out.numel() // cols, cols, out.data_ptr())
        return out


def _empty_checkpoint(x: torch.Tensor) -> Checkpoint8:
    shape = x.shape
    return _made(Checkpoint8, codes=x.new_empty(shape, dtype=torch.int8),
                 scales=x.new_empty((*shape[:-1], (shape[-1] + 31) // 32), dtype=torch.uint8), dtype=x.dtype)


def checkpoint8(x: torch.Tensor) -> Checkpoint8:
    """x [..., cols] in 8 bits: blocks of 32 elements of a row share a power-of-two step, 1/64 of the
    binade of their largest magnitude.  Elements that are not finite come back as NaN."""
    return _pack(_first(x, "x"))


def _pack(v: torch.Tensor) -> Checkpoint8:
    rows, cols = _rows(v, "x"), v.shape[-1]
    out = _empty_checkpoint(v)
    _run("afiv_checkpoint8_pack", v.device, v.data_ptr(), DTYPES[v.dtype], rows, cols, out.codes.data_ptr(), out.scales.data_ptr())
    return out


# ---- linear layer ----------------------------------------------------------------------------
@dataclass(frozen=True)
class LinearSaved:
    """What ``linear_act_backward`` needs besides the weight: the input (``x``, or ``eight``), and the
    pre-activation (``pre``) or the derivative's codes (``dcodes``); neither for act "none"."""
    x: torch.Tensor | None
    eight: Checkpoint8 | None
    pre: torch.Tensor | None
    dcodes: torch.Tensor | None
    act: str

    @property
    def shape(self) -> torch.Size:
        return self.x.shape if self.eight is None else self.eight.shape

    @property
    def dtype(self) -> torch.dtype:
        return self.x.dtype if self.eight is None else self.eight.dtype


@lru_cache(maxsize=4096)
def _scratch_bytes(query: str, m: int, n: int, k: int, *how: int) -> int:
    nbytes = getattr(_lib.lib(), query)(m, n, k, *how)
    if nbytes < 0:
        _lib.check(int(nbytes), query)
    return nbytes


def _scratch(nbytes: int, device) -> torch.Tensor | None:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _linear(x, weight, bias, residual, act, want_pre: bool, want_codes: bool):
    code = _act(act)
    v = _first(x, "x")
    m, k = _rows(v, "x"), v.shape[-1]
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or weight.shape[0] < 1:
        raise ValueError("weight must be [out features, in features] with at least one of each")
    n = weight.shape[0]
    w = _like(weight, v, (n, k), "weight")
    shape = (*v.shape[:-1], n)
    b = None if bias is None else _like(bias, v, (n,), "bias")
    r = None if residual is None else _like(residual, v, shape, "residual")
    y = v.new_empty(shape)
    pre = v.new_empty(shape) if want_pre else None
    dcodes = v.new_empty(shape, dtype=torch.uint8) if want_codes else None
    nbytes = _scratch_bytes("afiv_linear_act_scratch", m, n, k, DTYPES[v.dtype])
    scratch = _scratch(nbytes, v.device)
    _run("afiv_linear_act", v.device, v.data_ptr(), w.data_ptr(), _ptr(b), _ptr(r), DTYPES[v.dtype], code, m, n, k, y.data_ptr(), _ptr(pre),
         _ptr(dcodes), _ptr(scratch), nbytes)
    return v, y, pre, dcodes


def linear_act_forward(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                       residual: torch.Tensor | None = None, act: str = "none", checkpoint8: bool = False):
    """``act(x @ weight.T + bias) + residual`` and what its backward pass needs: (y, LinearSaved).
    x [..., in], weight [out, in], bias [out], residual [..., out], all of one type.  With ``checkpoint8``
    the input and the activation's derivative are kept in 8 bits (33/32 and 1 byte an element);
    otherwise they are the input itself and the pre-activation rounded to x's type (relu, leaky_relu: its sign,
    one byte)."""
    signs = act in ("relu", "leaky_relu")
    want_codes = signs or (checkpoint8 and act != "none")
    v, y, pre, dcodes = _linear(x, weight, bias, residual, act, act != "none" and not want_codes, want_codes)
    eight = _pack(v) if checkpoint8 else None
    return y, _made(LinearSaved, x=None if checkpoint8 else v, eight=eight, pre=pre, dcodes=dcodes, act=act)


def linear_act_backward(dy: torch.Tensor, weight: torch.Tensor, saved: LinearSaved, need=(True, True, True)):
    """(dx, dweight, dbias) of ``linear_act_forward`` for the output gradient dy, each None where ``need`` is
    false.  The residual's gradient is dy."""
    g = _first(dy, "dy")
    k, n = saved.shape[-1], weight.shape[0]
    if g.dtype != saved.dtype:
        raise TypeError(f"dy must be {saved.dtype}, got {g.dtype}")
    g = _like(g, g, (*saved.shape[:-1], n), "dy")
    w = _like(weight, g, (n, k), "weight")
    m = g.numel() // n
    dx = g.new_empty(saved.shape) if need[0] else None
    dw = g.new_empty((n, k)) if need[1] else None
    db = g.new_empty((n,)) if need[2] else None
    _held(saved.x if saved.eight is None else saved.eight.codes, g, saved.shape, "the saved input")
    if saved.act != "none" and saved.pre is None and saved.dcodes is None:
        raise ValueError(f"nothing is saved of the derivative of {saved.act}")
    _held(saved.pre, g, g.shape, "the saved pre-activation", g.dtype)
    _held(saved.dcodes, g, g.shape, "the saved derivative", torch.uint8)
    act, eight = _act(saved.act), saved.eight
    nbytes = _scratch_bytes("afiv_linear_act_backward_scratch", m, n, k, DTYPES[g.dtype], act, int(eight is not None))
    scratch = _scratch(nbytes, g.device)
    _run("afiv_linear_act_backward", g.device, g.data_ptr(), _ptr(saved.x), eight and eight.codes.data_ptr(), eight and eight.scales.data_ptr(),
         w.data_ptr(), _ptr(saved.pre), _ptr(saved.dcodes), DTYPES[g.dtype], act, m, n, k, _ptr(dx), _ptr(dw), _ptr(db),
         _ptr(scratch), nbytes)
    return dx, dw, db


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, eight):
        y, s = linear_act_forward(x, weight, bias, residual, act, eight)
        ctx.save_for_backward(weight, s.x, s.pre, s.dcodes, *((s.eight.codes, s.eight.scales) if eight else (None, None)))
        ctx.act, ctx.dtype = act, y.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        weight, x, pre, dcodes, codes, scales = ctx.saved_tensors
        eight = None if codes is None else _made(Checkpoint8, codes=codes, scales=scales, dtype=ctx.dtype)
        saved = _made(LinearSaved, x=x, eight=eight, pre=pre, dcodes=dcodes, act=ctx.act)
        need = ctx.needs_input_grad
        grads = linear_act_backward(dy, weight, saved, need[:3]) if any(need[:3]) else (None, None, None)
        return (*grads, dy if need[3] else None, None, None)


def _graph(*tensors) -> bool:
    """Whether autograd records the call."""
    if forward_ad._current_level >= 0:                   # inside Function.apply tangents can no longer be seen
        for t in tensors:
            if isinstance(t, torch.Tensor):
                _refuse_tangent(t, "an operand")
    if torch.is_grad_enabled():
        for t in tensors:
            if isinstance(t, torch.Tensor) and t.requires_grad:
                return True
    return False


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, residual: torch.Tensor | None = None,
               act: str = "none", checkpoint8: bool = False) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``, differentiable once; arguments as ``linear_act_forward``."""
    if _graph(x, weight, bias, residual):
        return _LinearAct.apply(x, weight, bias, residual, act, bool(checkpoint8))
    return _linear(x, weight, bias, residual, act, False, False)[1]


# ---- batch normalisation, activation, dropout ---------------------------------------------------
@dataclass(frozen=True)
class NormSaved:
    """What ``batch_norm_act_backward`` needs besides gamma and beta."""
    x: torch.Tensor | None
    eight: Checkpoint8 | None
    stats: torch.Tensor                  # [2, features] float64: mean, 1 / sqrt(var + eps)
    keep: torch.Tensor | None
    act: str
    drop_p: float


def _norm_scratch(m: int, n: int, device) -> torch.Tensor | None:
    if m <= NORM_SMALL_ROWS:
        return None
    return torch.empty(NORM_SCRATCH_DOUBLES * n, dtype=torch.float64, device=device)


def batch_norm_act_forward(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, running_mean: torch.Tensor | None = None,
                           running_var: torch.Tensor | None = None, act: str = "none", keep: torch.Tensor | None = None,
                           drop_p: float = 0.0, momentum: float = 0.1, eps: float = 1e-5, checkpoint8: bool = False):
    """``keep / (1 - drop_p) * act(batch_norm(x))`` with the batch's own statistics, and what its backward pass
    needs: (y, NormSaved).  x [rows, features]; weight (gamma) and bias (beta) float32 [features]; running_mean and
    running_var (both or none) float32 [features], updated in place as nn.BatchNorm1d does; keep: bool or
    uint8 mask of x's shape, needed where drop_p > 0.  With ``checkpoint8`` x is kept in 8 bits, and the backward
    pass takes the activation's derivative from those (relu's side too)."""
    code = _act(act)
    v = _first(x, "x")
    if v.dim() != 2 or v.shape[1] < 1:
        raise ValueError(f"x must be [rows, features], got {list(v.shape)}")
    m, n = v.shape
    if m < 2:
        raise ValueError(f"batch statistics need more than one row, got {m}")
    f32 = (torch.float32,)
    gamma, beta = _like(weight, v, (n,), "weight", f32), _like(bias, v, (n,), "bias", f32)
    if (running_mean is None) != (running_var is None):
        raise ValueError("running_mean and running_var come together")
    if running_mean is not None:
        _like(running_mean, v, (n,), "running_mean", f32, output=True)
        _like(running_var, v, (n,), "running_var", f32, output=True)
    drop_p = float(drop_p)
    if not 0.0 <= drop_p < 1.0:
        raise ValueError(f"drop_p must lie in [0, 1), got {drop_p}")
    if keep is None and drop_p > 0.0:
        raise ValueError("drop_p > 0 needs a keep mask")
    if keep is not None:
        keep = _like(keep, v, (m, n), "keep", (torch.bool, torch.uint8))
    y = torch.empty_like(v)
    stats = v.new_empty((2, n), dtype=torch.float64)
    eight = _empty_checkpoint(v) if checkpoint8 else None
    scratch = _norm_scratch(m, n, v.device)
    _run("afiv_norm_act", v.device, v.data_ptr(), gamma.data_ptr(), beta.data_ptr(), _ptr(keep), DTYPES[v.dtype], code, m, n, float(eps),
         float(momentum), drop_p, _ptr(running_mean), _ptr(running_var), y.data_ptr(), stats.data_ptr(), eight and eight.codes.data_ptr(),
         eight and eight.scales.data_ptr(), _ptr(scratch))
    # written behind torch's back: caches keyed on versions must see it (inference tensors have none)
    if running_mean is not None and not running_mean.is_inference() and not running_var.is_inference():
        torch.autograd.graph.increment_version((running_mean, running_var))
    return y, _made(NormSaved, x=None if checkpoint8 else v, eight=eight, stats=stats, keep=keep, act=act, drop_p=drop_p)


def batch_norm_act_backward(dy: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, saved: NormSaved, need_dx: bool = True):
    """(dx, dweight, dbias) of ``batch_norm_act_forward`` for the output gradient dy; dx is None without ``need_dx``."""
    g = _first(dy, "dy")
    held = saved.x if saved.eight is None else saved.eight
    if g.dtype != held.dtype:
        raise TypeError(f"dy must be {held.dtype}, got {g.dtype}")
    g = _like(g, g, held.shape, "dy")
    m, n = g.shape
    _held(saved.x if saved.eight is None else saved.eight.codes, g, g.shape, "the saved input")
    _held(saved.stats, g, (2, n), "the saved statistics", torch.float64)
    _held(saved.keep, g, g.shape, "the saved mask")
    f32 = (torch.float32,)
    gamma, beta = _like(weight, g, (n,), "weight", f32), _like(bias, g, (n,), "bias", f32)
    dx = torch.empty_like(g) if need_dx else None
    dgamma, dbeta = torch.empty_like(gamma), torch.empty_like(beta)
    scratch, eight = _norm_scratch(m, n, g.device), saved.eight
    _run("afiv_norm_act_backward", g.device, g.data_ptr(), _ptr(saved.x), eight and eight.codes.data_ptr(), eight and eight.scales.data_ptr(),
         gamma.data_ptr(), beta.data_ptr(), _ptr(saved.keep), saved.stats.data_ptr(), DTYPES[g.dtype], _act(saved.act), m, n, saved.drop_p,
         _ptr(dx), dgamma.data_ptr(), dbeta.data_ptr(), _ptr(scratch))
    return dx, dgamma, dbeta


class _BatchNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, running_mean, running_var, act, keep, drop_p, momentum, eps, eight):
        y, s = batch_norm_act_forward(x, weight, bias, running_mean, running_var, act, keep, drop_p, momentum, eps, eight)
        ctx.save_for_backward(weight, bias, s.x, s.stats, s.keep, *((s.eight.codes, s.eight.scales) if eight else (None, None)))
        ctx.act, ctx.drop_p, ctx.dtype = act, s.drop_p, y.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        weight, bias, x, stats, keep, codes, scales = ctx.saved_tensors
        eight = None if codes is None else _made(Checkpoint8, codes=codes, scales=scales, dtype=ctx.dtype)
        saved = _made(NormSaved, x=x, eight=eight, stats=stats, keep=keep, act=ctx.act, drop_p=ctx.drop_p)
        need = ctx.needs_input_grad
        dx, dgamma, dbeta = batch_norm_act_backward(dy, weight, bias, saved, need[0])
        return (dx, dgamma if need[1] else None, dbeta if need[2] else None) + (None,) * 8


def batch_norm_act(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, running_mean: torch.Tensor | None = None,
                   running_var: torch.Tensor | None = None, act: str = "none", keep: torch.Tensor | None = None, drop_p: float = 0.0,
                   momentum: float = 0.1, eps: float = 1e-5, checkpoint8: bool = False) -> torch.Tensor:
    """``keep / (1 - drop_p) * act(batch_norm(x))`` with the batch's own statistics, differentiable once;
    arguments as ``batch_norm_act_forward``."""
    if _graph(x, weight, bias):
        return _BatchNormAct.apply(x, weight, bias, running_mean, running_var, act, keep, drop_p, momentum, eps, bool(checkpoint8))
    return batch_norm_act_forward(x, weight, bias, running_mean, running_var, act, keep, drop_p, momentum, eps)[0]

"""CPU tests of the layer operators' boundary: refusals of the C ABI (before any device call) and of
the Python wrappers.  No compute call is made here."""
import ctypes

import pytest
import torch

from test_abi_and_host import declared_symbols

E_NULL, E_SHAPE, E_ARG, E_WORKSPACE = -1, -2, -4, -5


@pytest.fixture()
def lib(afiv):
    return afiv._lib.lib()


def _ptr():
    """A pointer that no refused call may follow."""
    return ctypes.c_void_p(64)


def test_entry_points_are_declared():
    for s in ("afiv_checkpoint8_pack", "afiv_checkpoint8_restore", "afiv_linear_act", "afiv_linear_act_scratch",
              "afiv_linear_act_backward", "afiv_linear_act_backward_scratch", "afiv_norm_act", "afiv_norm_act_backward"):
        assert s in declared_symbols()


def test_checkpoint_refusals(lib):
    p = _ptr()
    assert lib.afiv_checkpoint8_pack(p, 3, 4, 4, p, p, None) == E_ARG
    assert lib.afiv_checkpoint8_pack(p, -1, 4, 4, p, p, None) == E_ARG
    assert lib.afiv_checkpoint8_pack(p, 0, -1, 4, p, p, None) == E_SHAPE
    assert lib.afiv_checkpoint8_pack(p, 0, 4, 0, p, p, None) == E_SHAPE
    assert lib.afiv_checkpoint8_pack(p, 0, 4, (1 << 24) + 1, p, p, None) == E_SHAPE
    assert lib.afiv_checkpoint8_pack(p, 0, (1 << 36) + 1, 1, p, p, None) == E_SHAPE
    for i in range(3):
        a = [p, p, p]
        a[i] = None
        assert lib.afiv_checkpoint8_pack(a[0], 0, 4, 4, a[1], a[2], None) == E_NULL
        assert lib.afiv_checkpoint8_restore(a[0], a[1], 0, 4, 4, a[2], None) == E_NULL
    assert lib.afiv_checkpoint8_pack(None, 0, 0, 4, None, None, None) == 0       # no rows: nothing to do
    assert lib.afiv_checkpoint8_restore(None, None, 0, 0, 4, None, None) == 0


def test_linear_refusals(lib):
    p = _ptr()

    def fwd(x=p, w=p, dtype=0, act=0, m=4, n=4, k=4, y=p, scratch=p, nbytes=1 << 40):
        return lib.afiv_linear_act(x, w, None, None, dtype, act, m, n, k, y, None, None, scratch, nbytes, None)

    assert fwd(dtype=3) == E_ARG and fwd(act=6) == E_ARG and fwd(act=-1) == E_ARG
    assert fwd(m=-1) == E_SHAPE and fwd(n=0) == E_SHAPE and fwd(k=0) == E_SHAPE
    assert fwd(m=1 << 35, n=1 << 20) == E_SHAPE                                  # more tiles than a launch has
    assert fwd(x=None) == E_NULL and fwd(w=None) == E_NULL and fwd(y=None) == E_NULL
    assert fwd(m=0, x=None, y=None) == 0
    need = lib.afiv_linear_act_scratch(64, 64, 4096, 0)
    assert need > 0
    assert fwd(m=64, n=64, k=4096, scratch=None) == E_WORKSPACE
    assert fwd(m=64, n=64, k=4096, nbytes=need - 1) == E_WORKSPACE
    assert lib.afiv_linear_act_scratch(-1, 4, 4, 0) == E_SHAPE and lib.afiv_linear_act_backward_scratch(4, 4, 0, 0, 0, 0) == E_SHAPE
    assert lib.afiv_linear_act_backward_scratch(4, 4, 4, 3, 0, 0) == E_ARG
    assert lib.afiv_linear_act_backward_scratch(4, 4, 4, 0, 6, 0) == E_ARG
    assert lib.afiv_linear_act_scratch(1 << 20, 1024, 1024, 1) == 0                 # enough tiles: the sum is not cut

    def bwd(dy=p, x=p, codes=None, scales=None, w=p, pre=None, dcodes=None, act=0, m=4, n=4, k=4, dx=p, dw=p, db=p, nbytes=1 << 40):
        return lib.afiv_linear_act_backward(dy, x, codes, scales, w, pre, dcodes, 0, act, m, n, k, dx, dw, db, p, nbytes, None)

    assert bwd(dy=None) == E_NULL and bwd(w=None) == E_NULL and bwd(x=None) == E_NULL and bwd(x=None, codes=p) == E_NULL
    assert bwd(act=3) == E_NULL                                                  # no derivative
    assert bwd(act=7) == E_ARG and bwd(k=0) == E_SHAPE
    need = lib.afiv_linear_act_backward_scratch(1 << 16, 64, 64, 0, 0, 0)
    assert need > 0 and bwd(m=1 << 16, n=64, k=64, nbytes=need - 1) == E_WORKSPACE
    # room for dz and a restored x only where they are made
    size = [lib.afiv_linear_act_backward_scratch(1 << 14, 4096, 4096, 1, act, eight) for act, eight in ((0, 0), (4, 0), (0, 1), (4, 1))]
    assert size[0] < 1 << 23 and size[1] - size[0] >= 1 << 27 and size[2] - size[0] >= 1 << 27 and size[3] - size[0] >= 1 << 28
    assert fwd(m=1 << 30, n=64) == E_SHAPE                                       # a launch's limit of work items


def test_norm_refusals(lib):
    p = _ptr()

    def fwd(x=p, keep=None, dtype=0, act=0, m=4, n=4, eps=1e-5, momentum=0.1, drop=0.0, rm=None, rv=None, y=p, stats=p, codes=None,
            scales=None, scratch=p):
        return lib.afiv_norm_act(x, p, p, keep, dtype, act, m, n, eps, momentum, drop, rm, rv, y, stats, codes, scales, scratch, None)

    assert fwd(dtype=5) == E_ARG and fwd(act=6) == E_ARG
    assert fwd(drop=0.5) == E_ARG                                                # dropout without a mask
    assert fwd(keep=p, drop=1.0) == E_ARG and fwd(keep=p, drop=-0.1) == E_ARG and fwd(keep=p, drop=float("nan")) == E_ARG
    assert fwd(eps=-1.0) == E_ARG and fwd(momentum=float("inf")) == E_ARG
    assert fwd(m=1) == E_SHAPE and fwd(m=0) == E_SHAPE and fwd(n=0) == E_SHAPE
    assert fwd(rm=p) == E_NULL and fwd(codes=p) == E_NULL and fwd(x=None) == E_NULL and fwd(stats=None) == E_NULL and fwd(m=2000, scratch=None) == E_NULL

    def bwd(dy=p, x=p, codes=None, scales=None, drop=0.0, m=4, dgamma=p):
        return lib.afiv_norm_act_backward(dy, x, codes, scales, p, p, None, p, 0, 0, m, 4, drop, p, dgamma, p, p, None)

    assert bwd(dy=None) == E_NULL and bwd(x=None) == E_NULL and bwd(x=None, codes=p) == E_NULL and bwd(dgamma=None) == E_NULL
    assert bwd(m=1) == E_SHAPE and bwd(drop=0.1) == E_ARG


def test_wrappers_refuse_what_is_not_on_a_gpu(afiv):
    x, w = torch.zeros(4, 8), torch.zeros(3, 8)
    for call in (lambda: afiv.checkpoint8(x), lambda: afiv.linear_act(x, w), lambda: afiv.linear_act_forward(x, w),
                 lambda: afiv.batch_norm_act(x, torch.ones(8), torch.zeros(8))):
        with pytest.raises(ValueError, match="no CPU fallback"):
            call()
    with pytest.raises(TypeError):
        afiv.checkpoint8([1.0])
    with pytest.raises(ValueError, match="unknown activation"):
        afiv.linear_act(x, w, act="swish")
    with pytest.raises(ValueError, match="unknown activation"):
        afiv.batch_norm_act(x, torch.ones(8), torch.zeros(8), act=None)


def test_abi_limits_match_the_wrappers(afiv):
    import os
    import re
    text = open(os.path.join(os.path.dirname(__file__), "..", "include", "afiv.h")).read()
    chunks = int(re.search(r"#define AFIV_NORM_CHUNKS (\d+)", text).group(1))
    assert afiv.layers.NORM_SCRATCH_DOUBLES == 2 * chunks + 2
    assert afiv.layers.NORM_SMALL_ROWS == int(re.search(r"#define AFIV_NORM_SMALL_ROWS (\d+)", text).group(1))
    for name, value in afiv.layers.ACTIVATIONS.items():
        assert re.search(r"AFIV_ACT_%s = %d\b" % (name.upper(), value), text)
    for name, value in (("F32", 0), ("BF16", 1), ("F16", 2)):
        assert re.search(r"AFIV_%s = %d\b" % (name, value), text)


def test_forward_mode_tangents_are_refused(afiv):
    """A tangent that an operator cannot carry on must not vanish.  (Operands beside the first need a GPU: test_gpu_layers_calls.py.)"""
    from torch.autograd import forward_ad
    x, w = torch.randn(4, 8), torch.randn(3, 8)
    calls = (afiv.checkpoint8, lambda v: afiv.linear_act(v, w), lambda v: afiv.linear_act_forward(v, w),
             lambda v: afiv.batch_norm_act(v, torch.ones(8), torch.zeros(8)))
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in calls:
            with pytest.raises(NotImplementedError, match="tangent"):
                call(dual)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="tangent"):
                call(dual)
            with pytest.raises(ValueError, match="no CPU fallback"):          # a tensor without one goes on to the next check
                call(x)
    for call in calls:
        with pytest.raises(NotImplementedError, match="tangent"):
            torch.func.jvp(call, (x,), (torch.ones_like(x),))


PLAN_PROGRAM = r"""
#include "afiv_linear_plan.h"
#include <cstdio>
int main()
{
    long long m, n, k;
    while (std::scanf("%lld %lld %lld", &m, &n, &k) == 3) {
        const Plan dx = plan_for(m, k, n), dw = plan_for(n, k, m);
        std::printf("%d %lld %lld\n", (int)one_launch(m, n, k), (long long)(dx.tiles * dx.splits), (long long)(dw.tiles * dw.splits));
    }
}
"""


def test_joint_launches_stay_within_a_launch(tmp_path):
    """dx and dW share a launch only while their workgroups of 256 number fewer than 2^24; either alone does at any size that
    the entry points accept."""
    import os
    import subprocess
    root = os.path.join(os.path.dirname(__file__), "..")
    (tmp_path / "plan.cpp").write_text(PLAN_PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-w", "-I", os.path.join(root, "include"), "-I",
                    os.path.join(root, "arbitrage-free-iv-surfaces-using-vae_amd", "csrc"), "-o", str(tmp_path / "plan"), str(tmp_path / "plan.cpp")], check=True)
    sizes = [(64, 128, 13), (131072, 64, 128), ((1 << 30) - 64, 1, 64), ((1 << 30) - 64, 64, 64), ((1 << 30) - 64 * 600, 1, 64), ((1 << 24) - 64, 1, 4096)]
    out = subprocess.run([str(tmp_path / "plan")], input="\n".join("%d %d %d" % s for s in sizes), capture_output=True, text=True, check=True).stdout
    joint = []
    for (m, n, k), line in zip(sizes, out.splitlines()):
        one, dx, dw = map(int, line.split())
        assert dx < 1 << 24 and dw < 1 << 24 and bool(one) == (dx + dw < 1 << 24), (m, n, k)
        joint.append(bool(one))
    assert joint == [True, True, False, False, True, False]

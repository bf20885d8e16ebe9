"""The paged cache's entry points without a GPU, at the edges: sizes of the workspace and what Python passes on. The
handles are test_paged_host.py's stand-ins."""
import ctypes

import numpy as np
import pytest

from test_paged_host import CACHE


class _Ctx(ctypes.Structure):  # the fields that the workspace's size is worked out from
    _fields_ = [("device", ctypes.c_int), ("stream", ctypes.c_void_p), ("sms", ctypes.c_int)]


def _workspace(T, heads, S=1, G=0, sms=148, cache=CACHE):
    from decision_js_b200._lib import lib
    ctx, n = _Ctx(0, None, sms), ctypes.c_size_t()
    assert lib().dc_attention_paged_workspace(ctypes.addressof(ctx), ctypes.addressof(cache), T, heads, S, G, ctypes.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("T,heads", [(1, 2), (7, 4), (64, 16), (5000, 24)])
def test_the_workspace_may_start_at_any_multiple_of_16(pkg, T, heads):
    """The header asks for 16 bytes, parts are stored 32 at a time: the layout (whole multiples of 256 bytes) starts at the
    next multiple of 256, up to 240 bytes behind the address given."""
    assert _workspace(T, heads) % 256 == 240


def _no_context(pkg):
    ctx = pkg.Context.__new__(pkg.Context)  # no device: a call's arguments are converted and checked, and it ends there
    ctx.h = None
    return ctx


@pytest.mark.parametrize("eps", [1e-6, np.float64(1e-6)])
def test_a_call_takes_any_float(pkg, eps):
    """numpy's 64-bit scalar is a float, as it comes out of 1 / np.sqrt(D); with a host array next to it, too."""
    import enum
    ctx, x = _no_context(pkg), np.zeros(64, np.float32)
    one = enum.IntEnum("One", dict(one=1)).one
    for X in (0x10000, x):
        with pytest.raises(pkg.DecisionError, match="null context"):
            ctx.call("add_rmsnorm", X, None, 0x10000, 0x10000, one, 64, 0, eps)
    with pytest.raises(TypeError):
        ctx.call("add_rmsnorm", "x", None, 0x10000, 0x10000, 1, 64, 0, eps)


@pytest.mark.parametrize("dtype", ["bfloat16", "int16", "float32", "uint8"])
@pytest.mark.parametrize("which", [0, 1])
def test_a_cache_is_f16(pkg, dtype, which):
    """Two-byte elements of another type would be read as f16."""
    import torch
    kv = [torch.zeros(2, 1, 16, 64, dtype=torch.float16) for _ in range(2)]
    with pytest.raises(pkg.DecisionError, match="null context"):
        _no_context(pkg).kv_cache(*kv)
    kv[which] = kv[which].to(getattr(torch, dtype))
    with pytest.raises(pkg.DecisionError, match="contiguous f16"):
        _no_context(pkg).kv_cache(*kv)


def test_a_plan_refuses_a_factor_without_what_it_belongs_to(pkg):
    """`factor` is the context's beside a scaling, that of cos and sin beside frequencies; alone it was left out."""
    plan = _no_context(pkg).rope_plan
    with pytest.raises(pkg.DecisionError, match="a factor without") as e:
        plan(64, factor=8.0)
    assert e.value.code == 1
    with pytest.raises(pkg.DecisionError, match="a factor without"):
        plan(64, theta=1e6, factor=8.0)
    for good in (dict(), dict(theta=1e6), dict(scaling="linear", factor=8.0), dict(frequencies=[0.5] * 32, factor=8.0),
                 dict(scaling="none", factor=8.0)):
        with pytest.raises(pkg.DecisionError, match="null context"):
            plan(64, **good)

"""The paged cache's entry points without a GPU: frequencies, slots and refusals. The handles here are stand-ins with
the fields the checks read; the pointers are never dereferenced, each call returns before any device work."""
import ctypes
import math

import numpy as np
import pytest

import paged_ref as R


class _Plan(ctypes.Structure):
    _fields_ = [("device", ctypes.c_int), ("rot", ctypes.c_int), ("layout", ctypes.c_int), ("factor", ctypes.c_float),
                ("freq", ctypes.c_void_p)]


class _Cache(ctypes.Structure):
    _fields_ = [("device", ctypes.c_int), ("pages", ctypes.c_int), ("page", ctypes.c_int), ("kv", ctypes.c_int),
                ("D", ctypes.c_int), ("K", ctypes.c_void_p), ("V", ctypes.c_void_p)]


A, B = 0x10000, 0x10002          # 16-byte aligned; 2 bytes past a boundary
FAR = 0x40000000
CACHE = _Cache(0, 4, 16, 2, 128, 0x20000000, 0x30000000)
PLAN = _Plan(0, 128, 0, 1.0, 0x50000000)


def _says(rc, *words):
    from decision_js_b200._lib import DC_EINVAL, lib
    assert rc == DC_EINVAL
    text = lib().dc_last_error().decode()
    assert text.startswith("decision.js:") and all(w in text for w in words), text


def _rope(plan=PLAN, X=A, xs=512, pos=A, Y=FAR, ys=512, T=4, heads=4, D=128):
    from decision_js_b200._lib import lib
    return lib().dc_rope(None, ctypes.addressof(plan) if plan else None, X, xs, pos, Y, ys, T, heads, D)


def _append(cache=CACHE, plan=PLAN, Z=A, zs=1024, qn=A, kn=A, pos=A, slots=A, Q=FAR, qs=512, T=4, heads=4):
    from decision_js_b200._lib import lib
    return lib().dc_kv_append(None, ctypes.addressof(cache) if cache else None, ctypes.addressof(plan) if plan else None, Z,
                              zs, qn, kn, 1e-6, 0, pos, slots, Q, qs, T, heads)


def _attend(cache=CACHE, Q=A, qs=512, table=A, ts=4, lens=A, qoff=A, S=2, ptable=A, ps=4, plens=A, goff=A, G=1, Y=FAR,
            ys=512, T=4, heads=4, ws=A, n=1 << 40):
    from decision_js_b200._lib import lib
    return lib().dc_attention_paged(None, ctypes.addressof(cache) if cache else None, Q, qs, table, ts, lens, qoff, S, ptable, ps,
                                    plens, goff, G, Y, ys, T, heads, 0.1, ws, n)


def test_good_arguments_stop_at_the_context(pkg):
    for call in (_rope, _append, _attend):
        _says(call(), "null context")
    _says(_rope(Y=A), "null context")                        # in place
    _says(_rope(Y=A + 2 * 512, xs=1024, ys=1024), "null context")  # other columns of the same rows
    _says(_append(Q=A, qs=1024), "null context")             # q in place
    _says(_append(plan=None, pos=None, qn=None, kn=None), "null context")
    _says(_attend(G=0, ptable=None, plens=None, goff=None), "null context")
    _says(_attend(Y=A), "null context")                      # Y is Q


@pytest.mark.parametrize("change,words", [
    (dict(plan=None), ["null pointer"]), (dict(X=None), ["null pointer"]), (dict(pos=None), ["null pointer"]),
    (dict(D=72), ["multiple of 16"]), (dict(D=528, xs=4096, ys=4096), ["at most 512"]), (dict(D=64), ["128 dims"]),
    (dict(xs=508), ["multiples of 8"]), (dict(ys=504), ["hold 4 heads"]), (dict(T=-1), ["rope"]),
    (dict(heads=0), ["rope"]), (dict(X=B), ["aligned"]), (dict(Y=FAR + 2), ["aligned"]), (dict(pos=A + 2), ["aligned"]),
    (dict(Y=A + 16), ["overlaps"]), (dict(Y=A, ys=520), ["overlaps"]),
    (dict(Y=A + 2 * 520, xs=1024, ys=1024), ["overlaps"])])
def test_rope_refusals(pkg, change, words):
    _says(_rope(**change), *words)


@pytest.mark.parametrize("change,words", [
    (dict(cache=None), ["null pointer"]), (dict(pos=None), ["null pointer"]), (dict(slots=None), ["null pointer"]),
    (dict(heads=3), ["multiple of kv"]), (dict(heads=0), ["multiple of kv"]), (dict(T=-2), ["kv_append"]),
    (dict(plan=_Plan(0, 256, 0, 1.0, 0)), ["256 dims"]), (dict(zs=1016), ["hold"]), (dict(zs=1028), ["multiples of 8"]),
    (dict(qs=504), ["hold"]), (dict(Z=B), ["aligned"]), (dict(qn=B), ["aligned"]), (dict(slots=A + 2), ["aligned"]),
    (dict(Q=A, qs=512), ["overlap"]), (dict(Q=A + 64, qs=1024), ["overlap"]), (dict(Q=0x20000000), ["overlap"]),
    (dict(Z=0x30000000 - 4096), ["overlap"])])
def test_append_refusals(pkg, change, words):
    _says(_append(**change), *words)


@pytest.mark.parametrize("change,words", [
    (dict(cache=None), ["null cache"]), (dict(Q=None), ["null pointer"]), (dict(goff=None), ["null pointer"]),
    (dict(lens=None), ["null pointer"]), (dict(ws=None), ["null pointer"]), (dict(heads=5), ["multiple of kv"]),
    (dict(heads=130, qs=65536, ys=65536), ["64 times"]), (dict(T=-1), ["bad sizes"]), (dict(S=-1), ["bad sizes"]),
    (dict(G=-1), ["bad sizes"]), (dict(qs=510), ["multiples of 8"]), (dict(ys=504), ["hold"]), (dict(ts=-1), ["negative"]),
    (dict(Q=B), ["aligned"]), (dict(ws=A + 8), ["aligned"]), (dict(plens=A + 1), ["aligned"]),
    (dict(Y=A + 256), ["overlaps"]), (dict(Y=0x20000000 + 64), ["cache"])])
def test_attention_refusals(pkg, change, words):
    _says(_attend(**change), *words)


@pytest.mark.parametrize("K,V,pages,page,kv,D,word", [
    (None, A, 4, 16, 2, 128, "null pointer"), (A, FAR, 4, 24, 2, 128, "page"), (A, FAR, 4, 256, 2, 128, "page"),
    (A, FAR, 4, 16, 2, 96, "head dim"), (A, FAR, 0, 16, 2, 128, "pages"), (A, FAR, 1 << 24, 128, 1, 64, "2^31"),
    (B, FAR, 4, 16, 2, 128, "aligned"), (A, A + 16384, 4, 16, 2, 128, "overlap"), (A, FAR, 4, 16, 2, 128, "null context")])
def test_cache_refusals(pkg, K, V, pages, page, kv, D, word):
    from decision_js_b200._lib import lib
    h = ctypes.c_void_p(1)
    _says(lib().dc_kv_cache_create(None, K, V, pages, page, kv, D, ctypes.byref(h)), word)
    assert not h.value or word == "null pointer"


def test_plan_refusals(pkg):
    from decision_js_b200._lib import lib
    h = ctypes.c_void_p()
    f = (ctypes.c_double * 256)(*([0.5] * 256))
    make = lambda rot, layout, freq, factor: lib().dc_rope_plan_create(None, rot, layout, freq, factor, ctypes.byref(h))  # noqa: E731
    _says(make(24, 0, f, 1.0), "multiple of 16")
    _says(make(0, 0, f, 1.0), "multiple of 16")
    _says(make(528, 0, f, 1.0), "at most 512")
    _says(make(64, 2, f, 1.0), "layout")
    _says(make(64, 0, f, math.inf), "factor")
    _says(make(64, 0, None, 1.0), "null pointer")
    f[31] = math.nan
    _says(make(64, 0, f, 1.0), "frequency 31")
    f[31] = 0.5
    _says(make(64, 0, f, 1.0), "null context")


@pytest.mark.parametrize("rot,theta", [(128, 10000.0), (64, 1e7), (16, 500.0)])
@pytest.mark.parametrize("scaling,factor", [("none", 1.0), ("linear", 4.0), ("ntk", 8.0), ("yarn", 16.0), ("bands", 8.0)])
def test_frequencies(pkg, rot, theta, scaling, factor):
    trained = 4096.0
    got, mul = pkg.rope_frequencies(rot, theta=theta, scaling=scaling, factor=factor, trained=trained)
    i = np.arange(rot // 2)
    plain = theta ** (-2.0 * i / rot)
    want, want_mul = plain, 1.0
    if scaling == "linear":
        want = plain / factor
    elif scaling == "ntk":
        want = (theta * factor ** (rot / (rot - 2))) ** (-2.0 * i / rot)
        # the slowest pair is slowed by the factor, the fastest not at all
        assert want[0] == 1 and abs(want[-1] * factor / plain[-1] - 1) < 1e-12
    elif scaling == "yarn":
        at = lambda turns: rot * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        lo, hi = max(math.floor(at(32)), 0), min(math.ceil(at(1)), rot - 1)
        ramp = np.clip((i - lo) / max(hi - lo, 1e-3), 0, 1)
        want, want_mul = plain * (1 - ramp) + plain / factor * ramp, 0.1 * math.log(factor) + 1
    elif scaling == "bands":
        keep = np.clip((trained * plain / (2 * math.pi) - 1) / 3, 0, 1)
        want = plain * keep + plain / factor * (1 - keep)
    # pow and a handful of products in 64 bits on both sides
    assert np.allclose(got, want, rtol=2.0 ** -46, atol=0) and abs(mul - want_mul) < 2.0 ** -50


def test_frequency_refusals(pkg):
    for kw in (dict(rot=7), dict(rot=0), dict(rot=514), dict(rot=64, theta=1.0), dict(rot=64, theta=math.nan),
               dict(rot=64, scaling="linear", factor=0.5), dict(rot=64, scaling="yarn", factor=2.0),
               dict(rot=64, scaling="bands", factor=2.0, trained=4096, a=1.0, b=4.0), dict(rot=2, scaling="ntk", factor=2.0),
               dict(rot=64, scaling="other")):
        with pytest.raises(pkg.DecisionError) as e:
            pkg.rope_frequencies(**kw)
        assert str(e.value).startswith("decision.js:")


def test_slots(pkg):
    assert pkg.kv_slots([5, 2, 9], 16, 14, 20) == [5 * 16 + 14, 5 * 16 + 15] + [2 * 16 + i for i in range(16)] + [144, 145]
    assert pkg.kv_slots([5], 16, 16, 0) == []
    for first, count in ((-1, 2), (0, 17), (3, -1)):
        with pytest.raises(pkg.DecisionError):
            pkg.kv_slots([5], 16, first, count)


def test_reference_rotation_is_exact_at_far_positions():
    """The 64-bit reference itself: turning by p and then by -p is the identity, and by p = 2^20 it agrees with cos and
    sin of the product where the product in 64 bits is still good (2^20 * 2^-53 radians)."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((3, 2, 32))
    freq = 10000.0 ** (-np.arange(16) / 16)
    y, _ = R.rotate(x, [1 << 20, 7, -(1 << 30)], freq, 1.0, 32, "half")
    z, _ = R.rotate(y, [-(1 << 20), -7, 1 << 30], freq, 1.0, 32, "half")
    assert np.abs(z - x).max() < 1e-12
    c = np.cos((1 << 20) * freq)
    s = np.sin((1 << 20) * freq)
    assert np.abs(y[0, :, :16] - (x[0, :, :16] * c - x[0, :, 16:] * s)).max() < 1e-8

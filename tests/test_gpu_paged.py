"""The paged cache on the GPU: rotation, append and attention against plain 64-bit implementations (paged_ref.py).

Tolerances, from the formats: one rounding to f16 is at most 2^-11 of the value (2^-25 below the normal range).
Rotation: that, and a dozen f32 operations and a sine of 2 ulp, 2^-16 of |a| + |b| (with a norm, whose sum of at most 256
squares is good to 2^-16 and its root to half that, within the same). Attention: the weights are rounded to f16 and
summed as rounded, so the row moves by at most 2 * 2^-11 of sum p |v| / sum p; scores in f32 and the exponential add less
than 2^-11 of it for the values here; then the output's own rounding.
"""
import math

import numpy as np
import pytest

import paged_ref as R
from conftest import to_dev

pytestmark = pytest.mark.gpu

SMALL = 2.0 ** -25


def _f16(rng, *shape, scale=1.0):
    return (rng.standard_normal(shape) * scale).astype(np.float16)


def _i32(v, dev):
    import torch
    return torch.tensor(np.asarray(v, dtype=np.int32), device=dev)


def _half(a, dev):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a)).to(dev)


def _f64(t):
    return t.detach().cpu().numpy().astype(np.float64)


def _within(got, want, tol):
    bad = ~(np.abs(got - want) <= tol)  # NaN fails too
    assert not bad.any(), f"{bad.sum()} of {bad.size} off; worst {np.max(np.abs(got - want) / tol)} of the tolerance"


FREQ = {"plain": dict(scaling="none"), "linear": dict(scaling="linear", factor=4.0),
        "ntk": dict(scaling="ntk", factor=8.0), "yarn": dict(scaling="yarn", factor=16.0, trained=4096.0),
        "bands": dict(scaling="bands", factor=8.0, trained=4096.0)}


# ---------------------------------------------------------------- rotation

@pytest.mark.parametrize("T,heads,D,rot,layout,scaling,pad", [
    (1, 1, 16, 16, "half", "plain", 0), (1, 24, 128, 128, "half", "plain", 0), (3, 5, 80, 32, "interleaved", "linear", 8),
    (7, 3, 256, 64, "half", "yarn", 24), (33, 9, 96, 96, "interleaved", "bands", 0), (130, 7, 64, 48, "half", "ntk", 16),
    (257, 2, 512, 512, "half", "plain", 0), (64, 4, 512, 496, "interleaved", "yarn", 0), (1000, 40, 128, 64, "interleaved", "yarn", 40),
    (5000, 3, 192, 80, "half", "linear", 0)])
def test_rope(ctx, dev, pkg, T, heads, D, rot, layout, scaling, pad):
    import torch
    rng = np.random.default_rng(T + D)
    x = _f16(rng, T, heads * D + pad)
    pos = rng.integers(0, 1 << 20, T)
    pos[0] = 0
    if T > 2:
        pos[1], pos[2] = 2 ** 31 - 1, -5
    freq, factor = pkg.rope_frequencies(rot, **FREQ[scaling])
    plan = ctx.rope_plan(rot, layout, **FREQ[scaling])
    y = torch.full((T, heads * D + 8), 77.0, dtype=torch.float16, device=dev)
    dx, dp = _half(x, dev), _i32(pos, dev)
    torch.cuda.synchronize()
    ctx.call("rope", plan, dx, dx.shape[1], dp, y, y.shape[1], T, heads, D)
    ctx.sync(60000)
    xs = x[:, :heads * D].astype(np.float64).reshape(T, heads, D)
    want, size = R.rotate(xs, pos, freq, factor, rot, layout)
    got = _f64(y)
    assert (got[:, heads * D:] == 77.0).all()
    got = got[:, :heads * D].reshape(T, heads, D)
    assert (got[..., rot:] == xs[..., rot:]).all()
    _within(got, want, R.HALF_STEP * np.abs(want) + 2.0 ** -16 * size + SMALL)
    # in place, and from one column of the same rows to another: the same bits
    ctx.call("rope", plan, dx, dx.shape[1], dp, dx, dx.shape[1], T, heads, D)
    w = heads * D
    both = torch.cat([_half(x[:, :w], dev), torch.zeros(T, w, dtype=torch.float16, device=dev)], 1).contiguous()
    torch.cuda.synchronize()
    ctx.call("rope", plan, both, 2 * w, dp, both.data_ptr() + 2 * w, 2 * w, T, heads, D)
    ctx.sync(60000)
    assert torch.equal(dx[:, :w], y[:, :w]) and torch.equal(both[:, w:], y[:, :w])
    assert (dx[:, w:].cpu().numpy() == x[:, w:]).all() and (both[:, :w].cpu().numpy() == x[:, :w]).all()
    plan.close()


def test_rope_beside_the_packed_rows_rotation(ctx, dev, pkg):
    """On the packed rows' own case (half layout, plain frequencies, near positions) both give the same rows: each rounds
    once, from f32 angles that differ by 2^-22 or so at these positions."""
    import torch
    rng = np.random.default_rng(3)
    T, heads, kv, D, rot = 200, 8, 2, 256, 64
    z = _half(_f16(rng, T, (heads + kv) * D), dev)
    pos = _i32(np.arange(T), dev)
    y = torch.empty_like(z)
    plan = ctx.rope_plan(rot, theta=1e7)
    torch.cuda.synchronize()
    ctx.call("rope", plan, z, z.shape[1], pos, y, y.shape[1], T, heads + kv, D)
    ctx.call("qk_rope", z, None, None, pos, T, heads, kv, D, z.shape[1], rot, 0, 1e-6, 1e7)
    ctx.sync(60000)
    a, b = _f64(z), _f64(y)
    _within(b, a, 2 * R.HALF_STEP * np.abs(a) + 2.0 ** -12)


def test_nothing_to_do(ctx, dev):
    import torch
    plan = ctx.rope_plan(64)
    k = torch.zeros(2, 1, 16, 64, dtype=torch.float16, device=dev)
    cache = ctx.kv_cache(k, torch.zeros_like(k))
    buf = torch.full((64, 256), 3.0, dtype=torch.float16, device=dev)
    one = _i32([0, 0], dev)
    ws = torch.empty(ctx.attention_paged_workspace(cache, 4, 1, 1, 0), dtype=torch.uint8, device=dev)
    torch.cuda.synchronize()
    ctx.call("rope", plan, buf, 256, one, buf.data_ptr() + 16384, 256, 0, 1, 64)
    ctx.call("kv_append", cache, plan, buf, 256, None, None, 1e-6, 0, one, one, buf.data_ptr() + 16384, 64, 0, 1)
    ctx.call("attention_paged", cache, buf, 256, one, 1, one, one, 0, None, 0, None, None, 0, buf.data_ptr() + 16384, 64, 4,
             1, 0.1, ws, ws.numel())
    ctx.call("attention_paged", cache, buf, 256, one, 1, one, one, 1, None, 0, None, None, 0, buf.data_ptr() + 16384, 64, 4,
             1, 0.1, ws, ws.numel())  # one sequence without rows
    ctx.sync(60000)
    assert (buf == 3.0).all() and (k == 0).all()


# ---------------------------------------------------------------- append

@pytest.mark.parametrize("T,heads,kv,D,page,rot,layout,scaling,norm,vnorm,place", [
    (1, 16, 8, 128, 16, 128, "half", "plain", True, False, "apart"), (64, 24, 8, 128, 64, 128, "half", "yarn", True, True, "place"),
    (37, 32, 8, 64, 32, 32, "interleaved", "bands", False, False, "apart"), (5, 8, 2, 256, 128, 64, "half", "linear", True, False, "place"),
    (300, 5, 1, 128, 16, 16, "interleaved", "ntk", False, True, "apart"), (5000, 7, 7, 64, 64, 64, "half", "plain", True, True, "apart"),
    (9, 3, 3, 256, 16, 0, "half", "plain", True, False, "place")])
def test_kv_append(ctx, dev, pkg, T, heads, kv, D, page, rot, layout, scaling, norm, vnorm, place):
    import torch
    rng = np.random.default_rng(T * 3 + D)
    w = (heads + 2 * kv) * D
    z = _f16(rng, T, w + 16)
    qn, kn = (1 + 0.2 * rng.standard_normal((2, D))).astype(np.float16) if norm else (None, None)
    pages = -(-T // page) + 3
    slots = rng.permutation(pages * page)[:T].astype(np.int32)
    if T > 4:
        slots[T // 2], slots[-1] = -1, -7
    pos = rng.integers(0, 200000, T)
    old = _f16(rng, 2, pages, kv, page, D)
    k, v = _half(old[0], dev), _half(old[1], dev)
    cache = ctx.kv_cache(k, v)
    plan = ctx.rope_plan(rot, layout, **FREQ[scaling]) if rot else None
    dz = _half(z, dev)
    q = dz if place == "place" else torch.full((T, heads * D + 8), 9.0, dtype=torch.float16, device=dev)
    dqn, dkn = (_half(x, dev) if norm else None for x in (qn, kn))
    dp, ds = _i32(pos, dev), _i32(slots, dev)
    torch.cuda.synchronize()
    ctx.call("kv_append", cache, plan, dz, dz.shape[1], dqn, dkn, 1e-6, int(vnorm), dp if rot else None, ds, q, q.shape[1], T,
             heads)
    ctx.sync(60000)
    x = z[:, :w].astype(np.float64).reshape(T, heads + 2 * kv, D)
    xq, xk, xv = x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]
    if norm:
        xq, xk = R.rms(xq, qn.astype(np.float64), 1e-6), R.rms(xk, kn.astype(np.float64), 1e-6)
    if vnorm:
        xv = R.rms(xv, None, 1e-6)
    sq, sk = np.abs(xq), np.abs(xk)
    if rot:
        freq, factor = pkg.rope_frequencies(rot, **FREQ[scaling])
        xq, sq = R.rotate(xq, pos, freq, factor, rot, layout)
        xk, sk = R.rotate(xk, pos, freq, factor, rot, layout)
    tol = lambda y, s: R.HALF_STEP * np.abs(y) + 2.0 ** -16 * s + SMALL  # noqa: E731
    got = _f64(q)[:, :heads * D].reshape(T, heads, D)
    _within(got, xq, tol(xq, sq))
    rest = q[:, heads * D:].cpu().numpy()
    assert (rest == (z[:, heads * D:] if place == "place" else 9.0)).all()
    live = slots >= 0
    kept = np.ones(pages * page, bool)
    kept[slots[live]] = False
    for buf, was, y, s in ((k, old[0], xk, sk), (v, old[1], xv, np.abs(xv))):
        rows = lambda c: np.ascontiguousarray(c.swapaxes(1, 2)).reshape(pages * page, kv, D)  # noqa: E731
        now = rows(buf.cpu().numpy())
        assert (now[kept] == rows(was)[kept]).all()  # every other slot as it was
        _within(now[slots[live]].astype(np.float64), y[live], tol(y[live], s[live]))


def test_kv_append_flags_a_slot_past_the_cache(ctx, dev, pkg):
    import torch
    k = torch.zeros(2, 1, 16, 64, dtype=torch.float16, device=dev)
    v = torch.zeros_like(k)
    cache = ctx.kv_cache(k, v)
    z = torch.ones(3, 3 * 64, dtype=torch.float16, device=dev)
    q = torch.zeros(3, 64, dtype=torch.float16, device=dev)
    slots = _i32([5, 32, -1], dev)
    torch.cuda.synchronize()
    ctx.call("kv_append", cache, None, z, 192, None, None, 1e-6, 0, None, slots, q, 64, 3, 1)
    with pytest.raises(pkg.DecisionError) as e:
        ctx.sync(60000)
    assert e.value.code == 1
    assert (q == 1).all() and k.sum().item() == 64 and (k[0, 0, 5] == 1).all() and v.sum().item() == 64
    ctx.sync(60000)


def test_handles_check_their_memory(ctx, dev, pkg):
    import torch
    k = torch.zeros(2, 1, 16, 64, dtype=torch.float16, device=dev)
    with pytest.raises(pkg.DecisionError, match="not memory of device"):
        ctx.kv_cache(k.cpu(), k)
    with pytest.raises(pkg.DecisionError, match="contiguous"):
        ctx.kv_cache(k.transpose(2, 3), k.transpose(2, 3))
    cache = ctx.kv_cache(k, torch.zeros_like(k))
    ws = torch.empty(64, dtype=torch.uint8, device=dev)
    one = _i32([0, 1], dev)
    with pytest.raises(pkg.DecisionError, match="workspace"):
        ctx.call("attention_paged", cache, k, 64, one, 1, one, one, 1, None, 0, None, None, 0, ws.data_ptr(), 64, 1, 1, 0.1, ws, 64)
    cache.close()
    with pytest.raises(pkg.DecisionError, match="closed"):
        ctx.attention_paged_workspace(cache, 1, 1, 1, 0)


# ---------------------------------------------------------------- attention

class Case:
    """groups = [(prefix tokens, [(rows, own tokens), ...]), ...] in a cache whose other slots hold NaN, page tables
    whose other entries hold rubbish, and rows before and after the sequences'."""

    def __init__(self, ctx, dev, groups, heads, kv, D, page, first=0, after=0, seed=0, prefixes=True, qscale=1.5, pad=0,
                 rubbish=(-9, 1 << 30)):
        import torch
        rng = np.random.default_rng(seed)
        self.ctx, self.groups, self.heads, self.kv, self.D, self.first = ctx, groups, heads, kv, D, first
        seqs = [s for _, g in groups for s in g]
        need = lambda n: -(-n // page)  # noqa: E731
        total = sum(need(n) for _, n in seqs) + sum(need(p) for p, _ in groups) + 2
        ids = iter(rng.permutation(total))
        self.k = np.full((total, kv, page, D), np.nan, np.float16)
        self.v = self.k.copy()

        def take(lengths):
            t = np.full((len(lengths), max([need(n) for n in lengths] + [0]) + 1), rubbish[0], np.int32)
            t[:, -1] = rubbish[1]
            for i, n in enumerate(lengths):
                for j in range(need(n)):
                    p = t[i, j] = next(ids)
                    m = min(page, n - j * page)
                    self.k[p, :, :m], self.v[p, :, :m] = _f16(rng, kv, m, D), _f16(rng, kv, m, D)
            return t

        self.table, self.ptable = take([n for _, n in seqs]), take([p for p, _ in groups])
        self.lens, self.plens = [n for _, n in seqs], [p for p, _ in groups]
        self.qoff = first + np.concatenate([[0], np.cumsum([n for n, _ in seqs])])
        self.goff = np.concatenate([[0], np.cumsum([len(g) for _, g in groups])])
        self.T = int(self.qoff[-1]) + after
        self.q = _f16(rng, self.T, heads * D + pad, scale=qscale)
        self.pad, self.G = pad, len(groups) if prefixes else 0
        self.scale = D ** -0.5
        self.dev = dev
        self.dk, self.dv, self.dq = _half(self.k, dev), _half(self.v, dev), _half(self.q, dev)
        self.cache = ctx.kv_cache(self.dk, self.dv)
        self.meta = {n: _i32(getattr(self, n), dev) for n in ("table", "ptable", "lens", "plens", "qoff", "goff")}
        self.y = torch.full((self.T, heads * D + pad), 55.0, dtype=torch.float16, device=dev)
        self.ws = torch.full((ctx.attention_paged_workspace(self.cache, self.T, heads, len(seqs), self.G),), 255, dtype=torch.uint8,
                             device=dev)  # NaN in every f32
        torch.cuda.synchronize()

    def call(self, y=None, ctx=None):
        m, y = self.meta, self.y if y is None else y
        pre = (m["ptable"], self.ptable.shape[1], m["plens"], m["goff"], self.G) if self.G else (None, 0, None, None, 0)
        (ctx or self.ctx).call("attention_paged", self.cache, self.dq, self.dq.shape[1], m["table"], self.table.shape[1], m["lens"],
                               m["qoff"], len(self.lens), *pre, y, y.shape[1], self.T, self.heads, self.scale, self.ws,
                               self.ws.numel())

    def want(self):
        q = self.q[:, :self.heads * self.D].astype(np.float64).reshape(self.T, self.heads, self.D)
        return R.attention(q, self.k.astype(np.float64), self.v.astype(np.float64), self.table, self.ptable, self.groups,
                           self.first, self.heads, self.kv, self.scale)

    def check(self, y=None, rows=None):
        got = _f64(self.y if y is None else y)
        want = self.want()
        w = self.heads * self.D
        keep = np.ones(self.T, bool)
        for t, (a, size) in want.items():
            keep[t] = False
            if rows is None or t in rows:
                _within(got[t, :w].reshape(self.heads, self.D), a, R.HALF_STEP * np.abs(a) + 3 * R.HALF_STEP * size + SMALL)
        if y is None:
            assert (got[keep] == 55.0).all() and (got[:, w:] == 55.0).all()  # rows and columns that are nobody's


HEADS = [(16, 8, 128, 16), (24, 8, 128, 64), (32, 8, 64, 32), (8, 2, 256, 32), (5, 1, 128, 128), (7, 7, 64, 16),
         (64, 1, 64, 16), (2, 1, 256, 128)]

SHAPES = {
    "one_key": [(0, [(1, 1)])],
    "one_prefix_key": [(1, [(1, 0)])],
    "no_keys": [(0, [(1, 0), (3, 0)]), (0, [(2, 0)])],
    "edges": [(0, [(1, n) for n in (63, 64, 65, 127, 128, 129, 1, 2)])],
    "prefix_edges": [(p, [(1, 5), (2, 3)]) for p in (1, 15, 16, 17, 63, 64, 65, 127, 129)],
    "decode": [(700, [(1, n) for n in (5, 0, 64, 200, 1, 33, 130, 90)])],
    "causal": [(0, [(200, 200)]), (70, [(131, 140), (1, 7)])],
    "fewer_keys_than_rows": [(0, [(90, 70)]), (33, [(40, 3), (5, 5)])],
    "empty_sequences": [(40, [(0, 12), (3, 3), (0, 0), (0, 5)]), (9, []), (64, [(0, 3)]), (128, [(70, 71), (0, 0)])],
    "questions": [(300, [(17, 17), (40, 55), (1, 1)]), (129, [(64, 64), (23, 90)])],
}


@pytest.mark.parametrize("heads,kv,D,page", HEADS)
@pytest.mark.parametrize("shape", SHAPES)
def test_attention_paged(ctx, dev, heads, kv, D, page, shape):
    c = Case(ctx, dev, SHAPES[shape], heads, kv, D, page, first=2, after=3, seed=len(shape) + D, pad=8 if D == 64 else 0)
    c.call()
    ctx.sync(60000)
    c.check()


@pytest.mark.parametrize("heads,kv,D,page", [h for h in HEADS if h[2] <= 128])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention_paged_with_rows_behind(ctx, dev, heads, kv, D, page, shape):
    """The same sequences in front of rows that are nobody's, so many that the kernel for many rows takes the call."""
    groups = SHAPES[shape]
    c = Case(ctx, dev, groups, heads, kv, D, page, first=1, after=512 * len(groups) * kv // heads, seed=len(shape) + D)
    c.call()
    ctx.sync(60000)
    c.check()


@pytest.mark.parametrize("heads,kv,D,page", [(16, 8, 128, 16), (3, 1, 64, 64), (8, 2, 256, 128), (1, 1, 128, 32)])
@pytest.mark.parametrize("n,plen,own", [(1, 9000, 2000), (64, 5003, 77), (3, 0, 7001)])
def test_attention_paged_cut_over_many_ctas(ctx, dev, heads, kv, D, page, n, plen, own):
    """Long rows in parts, joined: one sequence, 64 of them at one token each, no prefix."""
    c = Case(ctx, dev, [(plen, [(1, max(own - 31 * i, 0)) for i in range(n)])], heads, kv, D, page, seed=n)
    c.call()
    ctx.sync(60000)
    c.check()


@pytest.mark.parametrize("heads,kv,D,many,after", [(16, 8, 128, 70, 0), (2, 1, 64, 120, 0), (2, 1, 64, 120, 31000), (2, 1, 128, 120, 31000),
                                                   (8, 4, 256, 60, 0)])
def test_attention_paged_one_long_group_among_short_ones(ctx, dev, heads, kv, D, many, after):
    """One tile in a hundred parts and more among many that are whole."""
    c = Case(ctx, dev, [(20, [(1, 5)]), (30000, [(3, 5), (1, 70)])] + [(i % 3, [(1, 5 + i)]) for i in range(many)], heads, kv, D, 64,
             after=after, seed=many)
    c.call()
    ctx.sync(60000)
    c.check()


@pytest.mark.parametrize("heads,kv,D", [(16, 8, 128), (32, 8, 64), (8, 2, 256)])
def test_attention_paged_without_groups(ctx, dev, heads, kv, D):
    c = Case(ctx, dev, [(0, [(1, 40 + i) for i in range(50)] + [(70, 100), (2, 2), (0, 0), (9, 300)])], heads, kv, D, 16, prefixes=False,
             first=1, after=1)
    c.call()
    ctx.sync(60000)
    c.check()


def test_attention_paged_many_sequences_and_groups(ctx, dev):
    """More sequences than a CTA has threads and more groups than its table holds."""
    rng = np.random.default_rng(5)
    groups = [(int(rng.integers(0, 40)), [(int(rng.integers(0, 3)), int(rng.integers(0, 20))) for _ in range(2)]) for _ in range(700)]
    c = Case(ctx, dev, groups, 4, 2, 64, 16, seed=2)
    c.call()
    ctx.sync(60000)
    c.check()


def test_attention_paged_sharp_and_flat_rows(ctx, dev):
    """Weights from one key alone to all alike, growing and falling along the keys, a scale below zero."""
    for i, (qscale, after) in enumerate(zip((0.0, 0.01, 8.0, 60.0) * 2, (0,) * 4 + (260,) * 4)):
        c = Case(ctx, dev, [(900, [(3, 200), (1, 70)])], 8, 4, 128, 32, seed=i % 4, qscale=qscale, after=after)
        ramp = np.linspace(-3, 3, c.k.shape[0], dtype=np.float16)[:, None, None, None]
        for flip in (1, -1):
            c.k = (c.k * 0 + ramp * flip + c.k * np.float16(0.1)).astype(np.float16)
            c.dk.copy_(_half(c.k, dev))
            c.scale = flip * 0.02
            c.call()
            ctx.sync(60000)
            if qscale < 60:
                c.check()
            else:  # scores in the hundreds: their f32 error, 128 products' 2^-20 of the size, is no longer small
                got, want = _f64(c.y), c.want()
                for t, (a, size) in want.items():
                    assert np.abs(got[t].reshape(8, 128) - a).max() <= 2.0 ** -8 * size.max()


def test_attention_paged_weights_far_below_the_largest(ctx, dev):
    """One key 2^13 above 32,768 equal others that carry most of the row together: their weights stay off f16's
    subnormals."""
    c = Case(ctx, dev, [(32768, [(1, 1)])], 2, 1, 64, 64, qscale=0)
    c.q[:] = 0
    c.q[:, 0::64] = 1
    c.k[:, :, :, 0] = np.where(np.isnan(c.k[:, :, :, 0]), np.nan, 0)
    c.k[c.table[0, 0], 0, 0, 0] = 13 * math.log(2)
    c.scale = 1.0
    c.dq.copy_(_half(c.q, dev)), c.dk.copy_(_half(c.k, dev))
    c.call()
    ctx.sync(60000)
    c.check()


@pytest.mark.parametrize("D,heads,kv,after", [(128, 16, 8, 0), (64, 4, 1, 0), (256, 2, 1, 0), (128, 16, 8, 300), (64, 4, 1, 200)])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_attention_paged_keeps_broken_rows_apart(ctx, dev, D, heads, kv, after, value):
    """A sequence whose last token has a key and a value that are not finite: its own earlier rows do not see them, nor
    do the other sequences of the tile; the row that sees them is not finite."""
    c = Case(ctx, dev, [(100, [(5, 70), (9, 9), (1, 130), (3, 3)])], heads, kv, D, 16, seed=3, after=after)
    s, n = 1, 9
    p, off = c.table[s, (n - 1) // 16], (n - 1) % 16
    c.v[p, :, off, 3] = value
    c.k[p, :, off, 5] = value
    c.dv.copy_(_half(c.v, dev)), c.dk.copy_(_half(c.k, dev))
    c.call()
    ctx.sync(60000)
    row = int(c.qoff[s + 1]) - 1
    c.v[p, :, off, 3] = c.k[p, :, off, 5] = 0  # for the rows that do not see it
    c.check(rows=set(range(c.T)) - {row})
    assert not np.isfinite(_f64(c.y)[row].reshape(heads, D)[:, 3]).any()


def test_attention_paged_broken_prefix_reaches_every_row(ctx, dev):
    c = Case(ctx, dev, [(100, [(1, 3), (2, 2)]), (50, [(4, 4)])], 4, 2, 64, 16)
    c.v[c.ptable[0, 2], :, 3, 7] = np.nan
    c.q[3, 0] = np.nan  # and a query of its own: a row that is not finite, not zeros
    c.dv.copy_(_half(c.v, dev)), c.dq.copy_(_half(c.q, dev))
    c.call()
    ctx.sync(60000)
    y = _f64(c.y).reshape(c.T, 4, 64)
    assert np.isnan(y[:3, :, 7]).all() and np.isnan(y[3, 0]).all()
    c.check(rows={4, 5, 6})


def test_attention_paged_in_place_and_repeatable(ctx, dev):
    import torch
    c = Case(ctx, dev, [(3000, [(1, 50 * i) for i in range(20)]), (10, [(150, 150)])], 16, 8, 128, 16)
    c.call()
    again = torch.empty_like(c.y)
    c.call(again)
    ctx.sync(60000)
    c.check()
    assert torch.equal(again, c.y)
    c.call(c.dq)  # Y is Q
    ctx.sync(60000)
    assert torch.equal(c.dq, c.y)


@pytest.mark.parametrize("heads,kv,D,groups", [
    (16, 8, 128, [(5000 - 300 * g, [(1, 40 * i + 1) for i in range(12)]) for g in range(6)]),
    (32, 8, 64, [(3000, [(1, 70 * i) for i in range(9)]), (4111, [(1, 5)])]),
    (24, 8, 128, [(2100, [(37, 37 + i) for i in range(20)])]), (8, 2, 256, [(1500, [(20, 90)] * 9)]),
    (32, 8, 64, [(700, [(80, 80 + i) for i in range(9)])] * 3)])
def test_attention_paged_many_calls_in_a_row(ctx, dev, heads, kv, D, groups):
    """Two hundred calls without a wait between them, all the same bits: the roles within a CTA, which run at their own
    pace, never lose step (a wait that ran out would flag the next sync)."""
    import torch
    c = Case(ctx, dev, groups, heads, kv, D, 32, seed=8)
    c.call()
    ctx.sync(60000)
    first = c.y.clone()
    for i in range(200):
        c.call()
        if i % 40 == 39:
            ctx.sync(60000)
            assert torch.equal(c.y, first)
    c.check(rows={0, c.T - 1})


def test_attention_paged_from_two_contexts_at_once(ctx, dev, pkg):
    """Calls of two contexts side by side on the device, of both kernels, each with its own workspace and cache."""
    import torch
    cases = [Case(ctx, dev, [(2000, [(1, 40 * i + 1) for i in range(12)])], 16, 8, 128, 32, seed=1),
             Case(ctx, dev, [(900, [(60, 60 + i) for i in range(8)])], 32, 8, 64, 32, seed=2)]
    firsts = []
    for c in cases:
        c.call()
        ctx.sync(60000)
        c.check(rows={0, c.T - 1})
        firsts.append(c.y.clone())
    torch.cuda.synchronize()
    other = pkg.Context(0)
    for i in range(60):
        cases[0].call()
        cases[1].call(ctx=other)
        if i % 20 == 19:
            ctx.sync(60000), other.sync(60000)
            assert all(torch.equal(c.y, f) for c, f in zip(cases, firsts))
    other.close()


def test_attention_paged_refuses_bad_arrays(ctx, dev, pkg):
    """Offsets that fall, reach past their table or rows: nothing is written, the next sync says so, and the context
    works on."""
    import torch
    c = Case(ctx, dev, [(100, [(2, 30), (3, 3)]), (20, [(1, 9)])], 4, 2, 64, 16)
    page = 16
    changes = [("qoff", 1, 0), ("qoff", 0, -1), ("qoff", 3, c.T + 1), ("lens", 1, -1), ("lens", 0, c.table.shape[1] * page + 1),
               ("plens", 0, c.ptable.shape[1] * page + 1), ("plens", 1, -3), ("goff", 0, 1), ("goff", 2, 2), ("goff", 1, 4)]
    changes[0] = ("qoff", 1, int(c.qoff[2]) + 1)
    for name, i, value in changes:
        good = c.meta[name][i].item()
        c.meta[name][i] = value
        torch.cuda.synchronize()
        c.call()
        with pytest.raises(pkg.DecisionError) as e:
            ctx.sync(60000)
        assert e.value.code == 1, name
        assert (c.y == 55.0).all(), (name, i)
        c.meta[name][i] = good
    for name, value in (("table", -1), ("ptable", len(c.k)), ("table", 1 << 30)):  # a page outside the cache
        good = c.meta[name][0, 0].item()
        c.meta[name][0, 0] = value
        torch.cuda.synchronize()
        c.call()
        with pytest.raises(pkg.DecisionError):
            ctx.sync(60000)
        c.meta[name][0, 0] = good
    torch.cuda.synchronize()
    c.call()
    ctx.sync(60000)
    c.check()


def test_attention_paged_refuses_a_workspace_in_its_tensors(ctx, dev, pkg):
    import torch
    c = Case(ctx, dev, [(20, [(2, 30)])], 4, 2, 64, 16)
    c.call()
    ctx.sync(60000)
    n = c.ws.numel() + (1 << 16)
    big = torch.zeros(2 * n, dtype=torch.uint8, device=dev)
    inside = big[n - 256:]
    for name in ("dq", "y"):
        mine = big[n - 2 * c.T * 256:].view(torch.float16)[:c.T * 256].view(c.T, 256)
        was, ws = getattr(c, name), c.ws
        setattr(c, name, mine), setattr(c, "ws", inside[:ws.numel()])
        with pytest.raises(pkg.DecisionError) as e:
            c.call()
        assert e.value.code == 1 and "workspace overlaps" in str(e.value)
        setattr(c, name, was), setattr(c, "ws", ws)
    k, v = torch.zeros(2, n // 512 + 1, 2, 16, 64, dtype=torch.float16, device=dev)
    c.cache, c.ws = ctx.kv_cache(k, v), v.view(-1).view(torch.uint8)[:c.ws.numel()]
    with pytest.raises(pkg.DecisionError) as e:
        c.call()
    assert e.value.code == 1 and "workspace overlaps" in str(e.value)


def test_attention_paged_in_a_graph(ctx, dev):
    """A captured call follows new lengths, offsets, tables and contents of the same arrays."""
    import torch
    a = Case(ctx, dev, [(900, [(1, 100), (1, 33), (2, 64)]), (64, [(4, 40)])], 16, 8, 128, 16, seed=1)
    # the same shapes and buffers, filled from another case
    b = Case(ctx, dev, [(300, [(2, 20), (0, 5), (1, 90)]), (800, [(5, 41)])], 16, 8, 128, 16, seed=2)
    pages = max(len(a.k), len(b.k))
    big = torch.full((2, pages, 8, 16, 128), float("nan"), dtype=torch.float16, device=dev)
    cache = ctx.kv_cache(big[0], big[1])
    rows = {n: max(getattr(a, n).shape[1], getattr(b, n).shape[1]) for n in ("table", "ptable")}
    meta = {n: torch.zeros((x.shape[0], rows[n]) if n in rows else x.shape, dtype=torch.int32, device=dev) for n, x in a.meta.items()}
    q = torch.zeros(8, 2048, dtype=torch.float16, device=dev)
    ws = torch.empty(ctx.attention_paged_workspace(cache, 8, 16, 4, 2), dtype=torch.uint8, device=dev)
    y = torch.zeros_like(q)

    def call():
        ctx.call("attention_paged", cache, q, 2048, meta["table"], rows["table"], meta["lens"], meta["qoff"], 4, meta["ptable"],
                 rows["ptable"], meta["plens"], meta["goff"], 2, y, 2048, 8, 16, 128 ** -0.5, ws, ws.numel())

    def fill(c):
        big[0, :len(c.k)].copy_(c.dk), big[1, :len(c.k)].copy_(c.dv)
        for n, x in c.meta.items():
            (meta[n][:, :x.shape[1]] if n in rows else meta[n]).copy_(x)
        q[:c.T].copy_(c.dq)
        y.fill_(55.0)
        torch.cuda.synchronize()

    fill(a)
    stream = torch.cuda.ExternalStream(ctx.stream, device=dev)
    call()
    ctx.sync(60000)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call()
    for c in (a, b, a):
        fill(c)
        graph.replay()
        torch.cuda.synchronize()
        c.check(y[:c.T])
    ctx.sync(60000)
    del graph


def test_append_then_attend_as_a_decoder_does(ctx, dev, pkg):
    """A state's keys appended once as a shared prefix, three questions appended to their own pages, then two more
    tokens each, one at a time: every row equals attention over the whole text in 64 bits, from the cache's own
    contents. The pages of a text are not in order and sequences end inside pages."""
    import torch
    rng = np.random.default_rng(11)
    heads, kv, D, page, rot = 16, 8, 128, 16, 128
    state, quests, extra = 203, [19, 1, 40], 2
    pages = 40
    k = torch.full((pages, kv, page, D), float("nan"), dtype=torch.float16, device=dev)
    v = torch.full_like(k, float("nan"))
    cache = ctx.kv_cache(k, v)
    plan = ctx.rope_plan(rot, scaling="yarn", factor=4.0, trained=4096.0)
    qn, kn = (_half((1 + 0.1 * rng.standard_normal(D)).astype(np.float16), dev) for _ in range(2))
    ids = list(rng.permutation(pages))
    take = lambda n: [ids.pop() for _ in range(-(-n // page))]  # noqa: E731
    trunk, own = take(state), [take(n + extra) for n in quests]
    width = max(len(o) for o in own)
    table = np.full((3, width), 0, np.int32)
    for i, o in enumerate(own):
        table[i, :len(o)] = o
    dtable, dptable = _i32(table, dev), _i32([trunk], dev)
    w = (heads + 2 * kv) * D

    def append(pos, slots):
        n = len(pos)
        z = _half(_f16(rng, n, w), dev)
        dp, ds = _i32(pos, dev), _i32(slots, dev)
        torch.cuda.synchronize()
        ctx.call("kv_append", cache, plan, z, w, qn, kn, 1e-6, 0, dp, ds, z, w, n, heads)  # q in place
        return z, dp, ds

    held = [append(range(state), pkg.kv_slots(trunk, page, 0, state))]
    have = [0, 0, 0]
    for step in range(1 + extra):
        new = quests if step == 0 else [1, 1, 1]
        pos = [state + have[i] + j for i in range(3) for j in range(new[i])]
        slots = sum((pkg.kv_slots(own[i], page, have[i], new[i]) for i in range(3)), [])
        z, *rest = append(pos, slots)
        have = [h + n for h, n in zip(have, new)]
        T = sum(new)
        lens, qoff = _i32(have, dev), _i32(np.concatenate([[0], np.cumsum(new)]), dev)
        plens, goff = _i32([state], dev), _i32([0, 3], dev)
        ws = torch.empty(ctx.attention_paged_workspace(cache, T, heads, 3, 1), dtype=torch.uint8, device=dev)
        y = torch.empty(T, heads * D, dtype=torch.float16, device=dev)
        torch.cuda.synchronize()
        ctx.call("attention_paged", cache, z, w, dtable, width, lens, qoff, 3, dptable, len(trunk), plens, goff, 1, y, heads * D, T,
                 heads, D ** -0.5, ws, ws.numel())
        ctx.sync(60000)
        q = _f64(z)[:, :heads * D].reshape(T, heads, D)
        want = R.attention(q, _f64(k), _f64(v), table, [trunk], [(state, list(zip(new, have)))], 0, heads, kv, D ** -0.5)
        got = _f64(y).reshape(T, heads, D)
        for t, (a, size) in want.items():
            _within(got[t], a, R.HALF_STEP * np.abs(a) + 3 * R.HALF_STEP * size + SMALL)


def test_far_pages_of_a_long_cache(ctx, dev, pkg):
    """Pages past 2^32 elements of K and of V: the same answers, to the bit, as from a cache of a few pages."""
    import torch
    heads, kv, D, page, far = 16, 8, 128, 64, 66_000  # 65,536 elements a page
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("two caches of 8.7 GB")
    c = Case(ctx, dev, [(150, [(1, 70), (3, 64), (2, 1)])], heads, kv, D, page, seed=6)
    n = len(c.k)
    k, v = (torch.empty((far, kv, page, D), dtype=torch.float16, device=dev) for _ in range(2))
    k[-n:].copy_(c.dk), v[-n:].copy_(c.dv)
    cache = ctx.kv_cache(k, v)
    z = torch.randn((6, (heads + 2 * kv) * D), device=dev).half()
    q = [torch.empty((6, heads * D), dtype=torch.float16, device=dev) for _ in range(2)]
    own = [(s, lo - m + i) for s, (m, lo) in enumerate([(1, 70), (3, 64), (2, 1)]) for i in range(m)]
    slots = [-1 if at < 0 else int(c.table[s, at // page]) * page + at % page for s, at in own]
    far_slots = [x if x < 0 else x + (far - n) * page for x in slots]
    torch.cuda.synchronize()
    y = [c.y, torch.full_like(c.y, 55.0)]
    tables = [torch.where((c.meta[t] >= 0) & (c.meta[t] < n), c.meta[t] + far - n, c.meta[t]) for t in ("table", "ptable")]
    for i, (kc, sl, (table, ptable)) in enumerate([(c.cache, slots, (c.meta["table"], c.meta["ptable"])), (cache, far_slots, tables)]):
        sl = _i32(sl, dev)
        torch.cuda.synchronize()
        ctx.call("kv_append", kc, None, z, z.shape[1], None, None, 0.0, 0, None, sl, q[i], heads * D, 6, heads)
        m = c.meta
        ctx.call("attention_paged", kc, q[i], heads * D, table, table.shape[1], m["lens"], m["qoff"], 3, ptable, ptable.shape[1],
                 m["plens"], m["goff"], 1, y[i], heads * D, 6, heads, c.scale, c.ws, c.ws.numel())
        ctx.sync(60000)
    assert torch.equal(q[0], q[1]) and torch.equal(y[0], y[1]) and torch.isfinite(y[0]).all() and (y[0] != 55.0).any()
    assert torch.equal(k[-n:].nan_to_num(7), c.dk.nan_to_num(7)) and torch.equal(v[-n:].nan_to_num(7), c.dv.nan_to_num(7))


@pytest.mark.parametrize("D,heads,kv", [(128, 16, 8), (64, 32, 8), (256, 8, 2)])
def test_paged_beside_packed_attention(ctx, dev, pkg, D, heads, kv):
    """A trunk and two branches: the packed pass over key ranges and the cached one give the same rows (each within its
    own f16 weights' roundings of the exact ones: 2 * 4 half steps of the largest value)."""
    import torch
    rng = np.random.default_rng(9)
    trunk, br = 150, [33, 21]
    T = trunk + sum(br)
    w = (heads + 2 * kv) * D
    z = _f16(rng, T, w)
    rngs, starts = [[0, t + 1, 0, 0] for t in range(trunk)], [trunk, trunk + br[0]]
    for s, n in zip(starts, br):
        rngs += [[0, trunk, s, s + i + 1] for i in range(n)]
    dz, dr = _half(z, dev), _i32(rngs, dev)
    packed = torch.empty(T, heads * D, dtype=torch.float16, device=dev)
    page = 16
    pages = 30
    k = torch.zeros(pages, kv, page, D, dtype=torch.float16, device=dev)
    v = torch.zeros_like(k)
    cache = ctx.kv_cache(k, v)
    ids = rng.permutation(pages)
    tp, own = ids[:10], [ids[10:13], ids[13:15]]
    slots = sum((pkg.kv_slots(p, page, 0, n) for p, n in zip([tp, *own], [trunk, *br])), [])
    ds = _i32(slots, dev)
    q = torch.empty(T, heads * D, dtype=torch.float16, device=dev)
    table = np.zeros((2, 3), np.int32)
    table[0], table[1, :2] = own[0], own[1]
    n = sum(br)
    args = [_i32(x, dev) for x in (table, br, [0, br[0], n], [tp], [trunk], [0, 2])]
    ws = torch.empty(ctx.attention_paged_workspace(cache, n, heads, 2, 1), dtype=torch.uint8, device=dev)
    y = torch.empty(n, heads * D, dtype=torch.float16, device=dev)
    torch.cuda.synchronize()
    ctx.call("attention", dz, dr, packed, T, heads, kv, D, D ** -0.5)
    ctx.call("kv_append", cache, None, dz, w, None, None, 1e-6, 0, None, ds, q, heads * D, T, heads)
    ctx.call("attention_paged", cache, q.data_ptr() + 2 * trunk * heads * D, heads * D, args[0], 3, args[1], args[2], 2, args[3], 10,
             args[4], args[5], 1, y, heads * D, n, heads, D ** -0.5, ws, ws.numel())
    ctx.sync(60000)
    assert len(slots) == T and torch.equal(q, dz[:, :heads * D])
    a, b = _f64(packed)[trunk:], _f64(y)
    assert np.abs(a - b).max() <= 8 * R.HALF_STEP * np.abs(z[:, (heads + kv) * D:].astype(np.float64)).max()

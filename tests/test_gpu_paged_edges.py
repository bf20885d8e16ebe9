"""The paged cache's calls at the edges of what the header allows: addresses, tables and contents that the shapes in
test_gpu_paged.py do not meet. Cases and tolerances are those of its Case."""
import ctypes

import numpy as np
import pytest

import paged_ref as R
from test_gpu_paged import SMALL, Case, _f16, _f64, _half, _i32, _within

pytestmark = pytest.mark.gpu


# One sequence over 9,000 tokens and many over a long prefix (tiles in parts, joined by row and by tile; both kernels).
CUT = [(16, 8, 128, [(9000, [(1, 2000)])], 0), (16, 8, 128, [(9000, [(1, 2000)])], 700), (32, 8, 64, [(5000, [(3, 9)] * 12)], 0),
       (32, 8, 64, [(3000, [(40, 90)] * 4), (300, [(70, 70)])], 0), (8, 2, 256, [(4000, [(1, 5), (30, 40)])], 0),
       (24, 8, 128, [(3000, [(33, 40)] * 3)], 1500), (24, 8, 256, [(1500, [(33, 40)] * 3), (0, [(1, 3000)])], 700)]


@pytest.mark.parametrize("heads,kv,D,groups,after", CUT)
@pytest.mark.parametrize("at", [16, 32, 48, 240])
def test_workspace_at_any_multiple_of_16(ctx, dev, heads, kv, D, groups, after, at):
    """Parts are stored 32 bytes at a time; a workspace at 16 past a multiple of 32 serves as any other, and nothing is
    written before or behind it."""
    import torch
    c = Case(ctx, dev, groups, heads, kv, D, 32, after=after, seed=at)
    n = c.ws.numel()
    whole = torch.full((n + 512,), 0xA5, dtype=torch.uint8, device=dev)
    lead = -whole.data_ptr() % 256 + at
    c.ws = whole[lead:lead + n]
    torch.cuda.synchronize()
    c.call()
    ctx.sync(60000)
    c.check()
    assert (whole[:lead] == 0xA5).all() and (whole[lead + n:] == 0xA5).all()


@pytest.mark.parametrize("heads,kv,D,after", [(16, 8, 128, 0), (8, 2, 128, 54000), (32, 8, 64, 0), (32, 8, 64, 54000), (8, 4, 256, 0)])
def test_marks_of_one_tile_reach_no_other(ctx, dev, heads, kv, D, after):
    """Tiles in a row in which a row sees a value that is not finite (and is marked) among tiles of one block that nothing
    is looked over in (one token, own keys a multiple of 16), whose end does not wait for that: only rows that see such a
    value are not finite, in call after call."""
    import torch
    n = 420
    groups = [(0, [(3, 19)]) if i % 5 == 0 else (0, [(1, 16 * (1 + i % 4))]) for i in range(n)]
    c = Case(ctx, dev, groups, heads, kv, D, 16, after=after, seed=4)
    broken = []
    for s in range(0, n, 5):
        p, off = c.table[s, 1], 18 - 16  # its last token: its last row alone sees it
        c.v[p, :, off, 3] = np.nan
        broken.append(int(c.qoff[s + 1]) - 1)
    c.dv.copy_(_half(c.v, dev))
    for i in range(60):
        c.call()
        if i % 20 == 0:
            ctx.sync(60000)
            finite = torch.isfinite(c.y).all(1)
            assert finite.sum().item() == c.T - len(broken) and not finite[broken].any()
    ctx.sync(60000)
    for s in range(0, n, 5):
        c.v[c.table[s, 1], :, 2, 3] = 0
    c.check(rows=set(range(c.T)) - set(broken))


@pytest.mark.parametrize("heads,kv,D,n", [(2, 1, 128, 1), (16, 8, 128, 40), (32, 8, 64, 1), (4, 2, 64, 120)])
def test_maxima_that_move_from_half_to_half(ctx, dev, heads, kv, D, n):
    """In the kernel for few rows two warps share a row, half of a block's 64 keys each, and exchange maxima. Here the
    largest score of each block is 2^12 above the one before and lies in the halves in turn: with a maximum of an earlier
    turn the weights would leave f16's range."""
    import torch
    c = Case(ctx, dev, [(2500, [(1, 70 + i % 3) for i in range(n)])], heads, kv, D, 64, qscale=0)
    c.q[:] = 0
    c.q[:, 0::D] = 1
    step = 12 * np.log(2)
    for pages, length, start in [(c.ptable[0], 2500, 0)] + [(c.table[s], c.lens[s], 2560) for s in range(n)]:
        for j in range(-(-length // 64)):
            block = start // 64 + j
            score = np.full(64, step * block - 30)
            score[32 * (block & 1) + 5] = step * block
            m = min(64, length - 64 * j)
            if m <= 32 * (block & 1) + 5:
                score[m - 1] = step * block
            c.k[pages[j], :, :m] = 0
            c.k[pages[j], :, :m, 0] = score[:m]
    c.scale = 1.0
    c.dq.copy_(_half(c.q, dev)), c.dk.copy_(_half(c.k, dev))
    torch.cuda.synchronize()
    c.call()
    first = c.y.clone()
    for _ in range(50):
        c.call()
    ctx.sync(60000)
    c.check()
    assert torch.equal(first, c.y)


@pytest.mark.parametrize("heads,kv,D,after", [(16, 8, 128, 0), (16, 8, 128, 4000), (32, 8, 64, 0), (8, 2, 256, 0)])
@pytest.mark.parametrize("S", [5, 600])
def test_tables_that_end_with_their_memory(ctx, dev, pkg, heads, kv, D, after, S):
    """Tables that are the last columns of wider arrays (rows far apart): of a row the pages of its length are read and
    nothing behind them, which for the last row is the end of the allocation."""
    from decision_js_b200._lib import lib
    c = Case(ctx, dev, [(40, [(1, 1 + i % 20) for i in range(S)])], heads, kv, D, 16, after=after, seed=S)
    stride, size = 48, 2 << 20
    held = []
    for name, rows in (("table", c.table), ("ptable", c.ptable)):
        at = ctypes.c_void_p()
        assert lib().dc_alloc(ctx.h, size, ctypes.byref(at)) == 0
        held.append(at)
        need = [-(-n // 16) for n in (c.lens if name == "table" else c.plens)]
        host = np.full(size // 4, 1 << 30, np.int32)
        start = size // 4 - stride * (len(rows) - 1) - need[-1]  # row r at start + r * stride, the last one's pages at the end
        for r, n in enumerate(need):
            host[start + r * stride:start + r * stride + n] = rows[r, :n]
        assert lib().dc_upload(ctx.h, at, host.ctypes.data, size) == 0
        c.meta[name] = at.value + 4 * start
    m = c.meta
    ctx.call("attention_paged", c.cache, c.dq, c.dq.shape[1], m["table"], stride, m["lens"], m["qoff"], S, m["ptable"], stride,
             m["plens"], m["goff"], 1, c.y, c.y.shape[1], c.T, heads, c.scale, c.ws, c.ws.numel())
    ctx.sync(60000)
    c.check()
    for at in held:
        assert lib().dc_free(ctx.h, at) == 0


# Rotation, each term by itself: a cos and b sin are the product of a value, of cos or sin and of the factor. In steps of
# u = 2^-24: cos and sin are off by 3.2 of themselves (an angle of at most pi/4 from 64-bit fixed point by 2.4, its series by
# the rest), the factor and the two products by one each: 7 u < 2^-21 of the term, however small it is beside the pair; the
# sum rounds once to f32, which the f16 rounding's half step covers with the rest of the 2^-21. The plan's frequency, 53
# bits, adds 2^-40 rad at the positions here.
def _rotate_terms(x, pos, freq, factor, rot, layout):
    i = np.arange(rot // 2)
    a = i if layout == "half" else 2 * i
    only = np.zeros(x.shape[-1])
    only[a] = 1
    only[rot:] = 1
    ya, _ = R.rotate(x * only, pos, freq, factor, rot, layout)
    yb, _ = R.rotate(x * (1 - only), pos, freq, factor, rot, layout)
    size = R.rotate(np.abs(x), pos, freq, factor, rot, layout)[1]
    y = ya + yb
    return y, R.HALF_STEP * np.abs(y) + 2.0 ** -21 * (np.abs(ya) + np.abs(yb)) + 2.0 ** -40 * size + SMALL


def _unequal(rng, T, heads, D, rot, layout):
    """Pairs with a zero, with one value 2^12 times the other, and like ones; angles small, and next to quarter turns."""
    x = _f16(rng, T, heads, D)
    i = np.arange(rot // 2)
    a, b = (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)
    x[:, 0, a], x[:, 1, b] = 0, 0
    x[:, 2, a] *= np.float16(2.0 ** 12)
    x[:, 3, b] *= np.float16(2.0 ** 12)
    freq = np.empty(rot // 2)
    n = rot // 4
    freq[:n] = 10000.0 ** (-np.arange(n) / n)
    freq[n:] = np.pi / 2 * (1 + 2.0 ** -rng.uniform(8, 24, rot // 2 - n))
    return x, freq


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("D,rot", [(128, 128), (256, 64)])
@pytest.mark.parametrize("op", ["rope", "append"])
def test_rotation_of_unequal_pairs(ctx, dev, layout, D, rot, op):
    """A result that is small beside its pair is as good as any: an angle's sine that is off by 2^-21, not of itself but
    of 1, would show in it."""
    import torch
    rng = np.random.default_rng(D + rot)
    T, heads, factor = 1500, 5, 1.25
    x, freq = _unequal(rng, T, heads, D, rot, layout)
    pos = rng.integers(0, 4096, T)
    plan = ctx.rope_plan(rot, layout, frequencies=list(freq), factor=factor)
    dp = _i32(pos, dev)
    if op == "rope":
        dx = _half(x.reshape(T, -1), dev)
        y = torch.empty_like(dx)
        torch.cuda.synchronize()
        ctx.call("rope", plan, dx, heads * D, dp, y, heads * D, T, heads, D)
    else:
        k = torch.zeros(2, 1, 16, D, dtype=torch.float16, device=dev)
        cache = ctx.kv_cache(k, torch.zeros_like(k))
        z = _half(np.concatenate([x.reshape(T, -1), np.zeros((T, 2 * D), np.float16)], 1), dev)
        y, slots = torch.empty(T, heads * D, dtype=torch.float16, device=dev), _i32([-1] * T, dev)
        torch.cuda.synchronize()
        ctx.call("kv_append", cache, plan, z, z.shape[1], None, None, 0.0, 0, dp, slots, y, heads * D, T, heads)
    ctx.sync(60000)
    want, tol = _rotate_terms(x.astype(np.float64), pos, freq, factor, rot, layout)
    _within(_f64(y).reshape(T, heads, D), want, tol)


# few rows and many, whole tiles, tiles in parts joined by row, and by tile
LOW = [(16, 8, 128, [(0, [(1, 40), (2, 70), (3, 20)]), (0, [(1, 33)])], 0), (16, 8, 128, [(0, [(1, 40), (2, 70), (3, 20)])], 600),
       (16, 8, 128, [(0, [(1, 9000), (1, 30)])], 0), (2, 1, 64, [(0, [(1, 9000), (1, 30)])], 600), (4, 2, 256, [(0, [(1, 5000), (1, 90)])], 0),
       (16, 8, 128, [(0, [(8, 1500 + i), (1, 7)]) for i in range(14)], 0), (32, 8, 64, [(0, [(8, 1500 + i), (1, 7)]) for i in range(14)], 4000),
       (8, 2, 256, [(0, [(8, 1500 + i), (1, 7)]) for i in range(14)], 300)]


@pytest.mark.filterwarnings("ignore:invalid value")  # the reference's own NaN
@pytest.mark.parametrize("heads,kv,D,groups,after", LOW)
def test_rows_whose_scores_are_all_minus_infinity(ctx, dev, heads, kv, D, groups, after):
    """A row that sees keys and scores minus infinity with each is NaN, as softmax is; one more key, which scores anything
    else, has all the weight; rows without a key stay zeros."""
    import torch
    c = Case(ctx, dev, groups, heads, kv, D, 16, after=after, seed=len(groups))
    c.q[:, 0::D] = 1
    c.dq.copy_(_half(c.q, dev))
    for s, n in enumerate(c.lens):
        if s % 2 == 0:  # every key of the even sequences
            for j in range(n):
                c.k[c.table[s, j // 16], :, j % 16, 0] = -np.inf
    c.dk.copy_(_half(c.k, dev))
    c.call()
    ctx.sync(60000)
    rows = lambda s: range(int(c.qoff[s]), int(c.qoff[s + 1]))  # noqa: E731
    low = [t for s in range(0, len(c.lens), 2) for t in rows(s)]
    assert torch.isnan(c.y[low]).all()
    c.check(rows=set(range(c.T)) - set(low))
    for s in range(0, len(c.lens), 2):  # its first key
        c.k[c.table[s, 0], :, 0, 0] = 1
    c.dk.copy_(_half(c.k, dev))
    c.call()
    ctx.sync(60000)
    c.check()
    c.meta["lens"].zero_()
    torch.cuda.synchronize()
    c.call()
    ctx.sync(60000)
    assert (c.y[int(c.qoff[0]):int(c.qoff[-1])] == 0).all()


@pytest.mark.parametrize("heads,kv,D,groups,after", CUT + [(16, 8, 128, [(300, [(17, 17), (40, 55), (1, 1)]), (129, [(64, 64), (23, 90)])], 0)])
def test_error_of_the_attention(ctx, dev, heads, kv, D, groups, after):
    """The weights of the product with v are rounded to f16, off by 2^-11 of themselves; their sum is of the f32 ones. Scores
    (D products summed in f32) and the exponential add less than 2^-11 again for the values here, the output rounds once: two
    half steps of sum p |v| and one of the result."""
    c = Case(ctx, dev, groups, heads, kv, D, 64, after=after, seed=21)
    c.call()
    ctx.sync(60000)
    got = _f64(c.y)[:, :heads * D]
    for t, (a, size) in c.want().items():
        _within(got[t].reshape(heads, D), a, R.HALF_STEP * np.abs(a) + 2 * R.HALF_STEP * size + SMALL)


@pytest.mark.parametrize("heads,kv,D,S", [(16, 8, 128, 5), (32, 8, 64, 3), (8, 2, 256, 4)])
def test_a_captured_decode_step(ctx, dev, pkg, heads, kv, D, S):
    """Append and attention of one token a sequence in one graph, replayed step after step with positions, slots and lengths
    in the same arrays: each row is attention over all that was appended, from the cache's own contents."""
    import torch
    rng = np.random.default_rng(D)
    page, state, steps = 16, 75, 6
    width = 3
    ids = list(rng.permutation(S * width + -(-state // page)))
    trunk, own = [ids.pop() for _ in range(-(-state // page))], [[ids.pop() for _ in range(width)] for _ in range(S)]
    n = S * width + len(trunk)
    k, v = (torch.full((n, kv, page, D), float("nan"), dtype=torch.float16, device=dev) for _ in range(2))
    for c in (k, v):
        for i, p in enumerate(trunk):
            m = min(page, state - i * page)
            c[p, :, :m] = _half(_f16(rng, kv, m, D), dev)
    cache, plan = ctx.kv_cache(k, v), ctx.rope_plan(D, scaling="linear", factor=2.0)
    table, ptable, plens, goff, qoff = (_i32(x, dev) for x in (own, [trunk], [state], [0, S], range(S + 1)))
    pos, slots, lens = (torch.zeros(S, dtype=torch.int32, device=dev) for _ in range(3))
    w = (heads + 2 * kv) * D
    z, y = torch.zeros(S, w, dtype=torch.float16, device=dev), torch.zeros(S, heads * D, dtype=torch.float16, device=dev)
    ws = torch.empty(ctx.attention_paged_workspace(cache, S, heads, S, 1), dtype=torch.uint8, device=dev)

    def step():
        ctx.call("kv_append", cache, plan, z, w, None, None, 1e-6, 1, pos, slots, z, w, S, heads)
        ctx.call("attention_paged", cache, z, w, table, width, lens, qoff, S, ptable, len(trunk), plens, goff, 1, y, heads * D, S, heads,
                 D ** -0.5, ws, ws.numel())

    def fill(have):
        pos.copy_(_i32([state + h for h in have], dev)), lens.copy_(_i32([h + 1 for h in have], dev))
        slots.copy_(_i32([pkg.kv_slots(own[s], page, h, 1)[0] for s, h in enumerate(have)], dev))
        z.copy_(_half(_f16(rng, S, w), dev))
        torch.cuda.synchronize()

    have = [0] * S
    fill(have)
    step()  # (a kernel's first call sets its attributes)
    ctx.sync(60000)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.ExternalStream(ctx.stream, device=dev)):
        step()
    for i in range(steps):
        have = [h + 1 + (s * 7 if i == 2 else 0) % 11 for s, h in enumerate(have)] if i else [page - 2] * S
        for s in range(S):  # what lies between is filled as an append would
            for h in range(have[s]):
                for c in (k, v):
                    row = c[own[s][h // page], :, h % page]
                    if torch.isnan(row).any():
                        row.copy_(_half(_f16(rng, kv, D), dev))
        fill(have)
        graph.replay()
        torch.cuda.synchronize()
        want = R.attention(_f64(z)[:, :heads * D].reshape(S, heads, D), _f64(k), _f64(v), own, [trunk],
                           [(state, [(1, h + 1) for h in have])], 0, heads, kv, D ** -0.5)
        got = _f64(y).reshape(S, heads, D)
        for t, (a, size) in want.items():
            _within(got[t], a, R.HALF_STEP * np.abs(a) + 2 * R.HALF_STEP * size + SMALL)
    ctx.sync(60000)
    del graph

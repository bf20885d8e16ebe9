"""Plain 64-bit implementations of the paged cache's operators (numpy, from the formulas) and their cases."""
import numpy as np

HALF_STEP = 2.0 ** -11  # f16 rounding, relative


def rotate(x, pos, freq, factor, rot, layout):
    """x [T, heads, D] float64, pos [T] ints, freq [rot/2] radians per position. Returns (y, |a| + |b| of the pair)."""
    i = np.arange(rot // 2)
    a, b = (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)
    # the whole turns go before the product is rounded: integers times a 64-bit fraction of a turn
    turn = np.array([[(int(p) * int(np.ldexp(np.longdouble(f) / (2 * np.pi) % 1.0, 62))) % (1 << 62) for f in freq]
                     for p in pos], dtype=np.float64) * 2.0 ** -62
    ang = turn[:, None, :] * (2 * np.pi)
    y, size = x.copy(), np.abs(x)
    c, s = np.cos(ang) * factor, np.sin(ang) * factor
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    size[..., a] = size[..., b] = (np.abs(x[..., a]) + np.abs(x[..., b])) * abs(factor)
    return y, size


def rms(x, w, eps):
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return y if w is None else y * w


def visible(groups, qoff):
    """For each query row: (group, sequence, own keys it sees). groups = [(plen, [(n, len), ...]), ...]."""
    out, s, t = {}, 0, qoff
    for g, (_, seqs) in enumerate(groups):
        for n, ln in seqs:
            for i in range(n):
                out[t] = (g, s, max(ln - n + 1 + i, 0))
                t += 1
            s += 1
    return out


def attention(q, kc, vc, table, ptable, groups, first, heads, kv, scale):
    """q [T, heads, D]; kc, vc [pages, kv, page, D] float64 (whatever lies past a length is not read). Returns
    {row: (y [heads, D], sum p |v| / sum p)}."""
    page, r = kc.shape[2], heads // kv
    out = {}
    for t, (g, s, lim) in visible(groups, first).items():
        plen = groups[g][0]
        rows = [(ptable[g][j // page], j % page) for j in range(plen)] + [(table[s][j // page], j % page) for j in range(lim)]
        y, size = np.zeros((heads, q.shape[-1])), np.zeros((heads, q.shape[-1]))
        if rows:
            pg, off = np.array(rows).T
            k, v = kc[pg, :, off], vc[pg, :, off]  # [keys, kv, D]
            for h in range(heads):
                a = (k[:, h // r] @ q[t, h]) * scale
                p = np.exp(a - a.max())
                p /= p.sum()
                y[h], size[h] = p @ v[:, h // r], p @ np.abs(v[:, h // r])
        out[t] = (y, size)
    return out

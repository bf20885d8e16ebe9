"""Cases for three operators of a decoder that answers many short sequences against a long shared one: rotary
positions, appending keys and values to a paged cache with the rotation on the way, and the attention that reads that
cache, the shared part once for all sequences that share it.

`run` computes the plain form in torch, or (with `own`) makes the framework's calls on the same state.
"""
import math
import random

import torch

own = False

DEV = "cuda"
F16 = torch.float16

# ---------------------------------------------------------------- cases


def listed():
    return [
        # one token of a 16-head decoder: the latency of a call
        dict(name="rope_token", op="rope", T=1, heads=24, D=128, rot=128, layout="half", scaling="none", far=2048, pad=0),
        # q and k heads of 16,384 packed tokens, interleaved pairs in half of each head, positions of a long context
        dict(name="rope_prompt", op="rope", T=16384, heads=32, D=128, rot=64, layout="interleaved", scaling="yarn",
             far=131072, pad=1024),
        # 256-wide heads rotated in their first 64 dims, an odd token count, rows that hold more than the heads
        dict(name="rope_partial", op="rope", T=4099, heads=10, D=256, rot=64, layout="half", scaling="linear",
             far=32768, pad=2560),
        # one new token for each of 64 sequences, q and k norms: a decode step's append
        dict(name="append_step", op="append", seqs=64, tokens=1, past=700, heads=16, kv=8, D=128, page=16, rot=128,
             layout="half", scaling="none", norm=True, vnorm=False, pads=0),
        # 16 prompts of 1,024 tokens into an empty cache
        dict(name="append_prompts", op="append", seqs=16, tokens=1024, past=0, heads=24, kv=8, D=128, page=64, rot=128,
             layout="half", scaling="bands", norm=True, vnorm=False, pads=0),
        # ragged continuations with padding rows, 64-wide heads without norms, interleaved pairs
        dict(name="append_ragged", op="append", seqs=37, tokens=61, past=333, heads=32, kv=8, D=64, page=32, rot=64,
             layout="interleaved", scaling="ntk", norm=False, vnorm=False, pads=75),
        # four sequences at one token each over a short shared text: the latency of a call
        dict(name="shared_small", op="attention", groups=1, seqs=4, tokens=1, own=24, prefix=512, heads=16, kv=8, D=128,
             page=16, ragged=True, layout=1),
        # a decode step of 64 sequences over one long shared text
        dict(name="shared_step", op="attention", groups=1, seqs=64, tokens=1, own=512, prefix=32768, heads=16, kv=8,
             D=128, page=64, ragged=True, layout=2),
        # a decode step of 24 requests with up to 12 branches each, 64-wide heads
        dict(name="shared_groups", op="attention", groups=24, seqs=12, tokens=1, own=300, prefix=6000, heads=32, kv=8,
             D=64, page=32, ragged=True, layout=3),
        # 32 requests of 3 questions of about 40 tokens over texts of 512 tokens
        dict(name="questions", op="attention", groups=32, seqs=3, tokens=40, own=0, prefix=512, heads=16, kv=8, D=128,
             page=16, ragged=False, layout=4),
        # 60 questions of up to 50 tokens over one text of 16,000 tokens: bound by the products
        dict(name="questions_long", op="attention", groups=1, seqs=60, tokens=50, own=0, prefix=16000, heads=24, kv=8,
             D=128, page=64, ragged=True, layout=5),
        # 256-wide heads, 4 requests, answers of some length behind each question
        dict(name="questions_wide", op="attention", groups=4, seqs=10, tokens=33, own=200, prefix=4000, heads=8, kv=2,
             D=256, page=32, ragged=True, layout=6),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "attention", "attention"])
    layout = rng.choice(["half", "interleaved"])
    scaling = rng.choice(["none", "linear", "ntk", "yarn", "bands"])
    if op == "rope":
        D = rng.choice([64, 80, 96, 128, 192, 256])
        return dict(op=op, T=_log(rng, 1, 12000), heads=rng.randint(1, 32), D=D, rot=16 * rng.randint(1, D // 16),
                    layout=layout, scaling=scaling, far=_log(rng, 256, 1 << 20), pad=8 * rng.randint(0, 64))
    heads, kv, D = rng.choice([(16, 8, 128), (24, 8, 128), (32, 8, 64), (8, 2, 256), (8, 2, 64), (12, 4, 128),
                               (5, 1, 128), (7, 7, 64)])
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        tokens = _log(rng, 1, 500)
        return dict(op=op, seqs=_log(rng, 1, max(1, min(200, 16000 // tokens))), tokens=tokens, past=_log(rng, 1, 900),
                    heads=heads, kv=kv, D=D, page=page, rot=16 * rng.randint(1, D // 16), layout=layout,
                    scaling=scaling, norm=rng.random() < 0.5, vnorm=rng.random() < 0.3, pads=rng.randint(0, 50))
    tokens = rng.choice([1, 1, _log(rng, 1, 64)])
    groups = _log(rng, 1, 16)
    seqs = _log(rng, 1, max(1, 2400 // (groups * tokens) if tokens > 1 else 256 // groups))
    most = 16000 if tokens > 1 else 40000
    prefix = _log(rng, 64, max(64, min(most, 60000000 // (groups * seqs * tokens * heads), 200000 // groups)))
    return dict(op=op, groups=groups, seqs=seqs, tokens=tokens, own=_log(rng, 1, 600) - 1, prefix=prefix, heads=heads,
                kv=kv, D=D, page=page, ragged=rng.random() < 0.7, layout=rng.randint(10, 1 << 20))


# ---------------------------------------------------------------- inputs


def _frequencies(rot, scaling, far, theta=10000.0):
    """Radians per position of each pair, and the factor on cos and sin, for a context `far` long trained at 4,096."""
    trained = 4096.0
    s = max(1.0, far / trained)
    if scaling == "ntk" and rot > 2:
        theta *= s ** (rot / (rot - 2.0))
    w = [theta ** (-2.0 * i / rot) for i in range(rot // 2)]
    if scaling == "linear":
        w = [x / s for x in w]
    elif scaling == "yarn":
        at = [rot * math.log(trained / (b * 2 * math.pi)) / (2 * math.log(theta)) for b in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
        ramp = [min(max((i - lo) / max(hi - lo, 1e-3), 0.0), 1.0) for i in range(rot // 2)]
        w = [x / s * k + x * (1 - k) for x, k in zip(w, ramp)]
        return w, 0.1 * math.log(s) + 1.0
    elif scaling == "bands":
        turns = [trained * x / (2 * math.pi) for x in w]
        keep = [min(max((t - 1.0) / 3.0, 0.0), 1.0) for t in turns]
        w = [x / s * (1 - k) + x * k for x, k in zip(w, keep)]
    return w, 1.0


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 7919 + 13)
    return g


def _randn(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(F16)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _lengths(c):
    """Sequences per group, new tokens and own keys per sequence, prefix keys per group: by the case alone."""
    r = random.Random(c["layout"])
    some = (lambda hi, lo: r.randint(min(lo, hi), hi)) if c["ragged"] else (lambda hi, lo: hi)
    per = [some(c["seqs"], max(1, c["seqs"] // 2)) for _ in range(c["groups"])]
    new = [some(c["tokens"], 1) for _ in range(sum(per))]
    keys = [n + some(c["own"], 0) for n in new]
    pre = [some(c["prefix"], c["prefix"] // 2) for _ in range(c["groups"])]
    return per, new, keys, pre


def _tables(lengths, page, ids):
    """Page tables [len(lengths), most pages]; `ids` gives the pages out. Unused entries are 0."""
    need = [-(-n // page) for n in lengths]
    rows = torch.zeros(len(lengths), max(max(need), 1), dtype=torch.int32)
    for i, n in enumerate(need):
        rows[i, :n] = torch.tensor([next(ids) for _ in range(n)], dtype=torch.int32)
    return rows


def _starts(v):
    out = [0]
    for x in v:
        out.append(out[-1] + x)
    return out


def prepare(case, seed):
    c, g = case, _gen(seed)
    r = random.Random(seed)
    s = {"case": c}
    if c["op"] == "rope":
        w, s["factor"] = _frequencies(c["rot"], c["scaling"], c["far"])
        s["freq"] = torch.tensor(w, dtype=torch.float64, device=DEV)
        s["x"] = _randn(g, c["T"], c["heads"] * c["D"] + c["pad"])
        s["pos"] = torch.randint(0, c["far"], (c["T"],), generator=g, device=DEV, dtype=torch.int32)
        s["y"] = torch.empty(c["T"], c["heads"] * c["D"], dtype=F16, device=DEV)
        return s
    heads, kv, D, page = c["heads"], c["kv"], c["D"], c["page"]
    if c["op"] == "append":
        w, s["factor"] = _frequencies(c["rot"], c["scaling"], 16384)
        s["freq"] = torch.tensor(w, dtype=torch.float64, device=DEV)
        per = -(-(c["past"] + c["tokens"]) // page)
        ids = list(range(c["seqs"] * per + 3))
        r.shuffle(ids)
        table = torch.tensor(ids[:c["seqs"] * per]).view(c["seqs"], per)
        at = c["past"] + torch.arange(c["tokens"])
        slots = (table[:, at // page] * page + at % page).reshape(-1)
        T = slots.numel() + c["pads"]
        s["slots"] = torch.cat([slots, torch.full((c["pads"],), -1)]).to(torch.int32).to(DEV)
        s["pos"] = torch.cat([at.repeat(c["seqs"]), torch.zeros(c["pads"], dtype=torch.int64)]).to(torch.int32).to(DEV)
        s["z"] = _randn(g, T, (heads + 2 * kv) * D)
        s["qn"], s["kn"] = (1 + _randn(g, D, scale=0.1), 1 + _randn(g, D, scale=0.1)) if c["norm"] else (None, None)
        s["k"], s["v"] = _randn(g, len(ids), kv, page, D), _randn(g, len(ids), kv, page, D)
        s["q"] = torch.empty(T, heads * D, dtype=F16, device=DEV)
        return s
    per, new, keys, pre = _lengths(c)
    pages = sum(-(-n // page) for n in keys) + sum(-(-n // page) for n in pre) + 2
    ids = list(range(pages))
    r.shuffle(ids)
    ids = iter(ids)
    s["table"], s["ptable"] = _tables(keys, page, ids).to(DEV), _tables(pre, page, ids).to(DEV)
    s["lens"], s["plens"] = _ints(keys), _ints(pre)
    s["qoff"], s["goff"] = _ints(_starts(new)), _ints(_starts(per))
    s["T"], s["most_new"], s["most_group"] = sum(new), max(new), max(
        sum(new[a:b]) for a, b in zip(_starts(per), _starts(per)[1:]))
    s["k"], s["v"] = _randn(g, pages, kv, page, D), _randn(g, pages, kv, page, D)
    s["q"] = _randn(g, s["T"], heads * D, scale=1.5)
    s["y"] = torch.empty(s["T"], heads * D, dtype=F16, device=DEV)
    return s


# ---------------------------------------------------------------- the plain form


def _rotate(x, pos, freq, factor, rot, layout):
    """x [T, heads, D] f32 at positions pos [T]; the angles in 64 bits."""
    a = pos.double()[:, None] * freq[None, :]
    cs, sn = (torch.cos(a) * factor).float()[:, None, :], (torch.sin(a) * factor).float()[:, None, :]
    h = rot // 2
    p, q = (x[..., :h], x[..., h:rot]) if layout == "half" else (x[..., 0:rot:2], x[..., 1:rot:2])
    u, v = p * cs - q * sn, q * cs + p * sn
    turned = torch.cat([u, v], -1) if layout == "half" else torch.stack([u, v], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def _rms(x, w):
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    return x if w is None else x * w.float()


def _partial(q, k, v, seen):
    """Maxima, sums and weighted values of softmax parts: q [B, n, kv, r, D], k and v [B, kv, L, D], seen [B, n, L]."""
    s = torch.einsum("bnkrd,bkld->bkrnl", q, k)
    s = torch.where(seen[:, None, None], s, -math.inf)
    m = s.max(-1, keepdim=True).values.clamp(min=-1e30)
    p = torch.exp(s - m)
    o = torch.einsum("bkrnl,bkld->bnkrd", p, v)
    return m[..., 0].permute(0, 3, 1, 2), p.sum(-1).permute(0, 3, 1, 2), o


def _paged(cache, table):
    """[B, kv, L, D] f32 of the pages of each row of a table."""
    x = cache[table.long()]
    return x.transpose(1, 2).flatten(2, 3).float()


def _attention(s):
    c = s["case"]
    kv, D, T = c["kv"], c["D"], s["T"]
    r = c["heads"] // kv
    q = s["q"].float().view(T, kv, r, D) / math.sqrt(D)
    dev = q.device
    qoff, goff, lens, plens = (s[n].long() for n in ("qoff", "goff", "lens", "plens"))
    t = torch.arange(T, device=dev)
    seq = torch.searchsorted(qoff, t, right=True) - 1
    grp = torch.searchsorted(goff, seq, right=True) - 1
    parts = []
    first = qoff[goff]
    for start, most, table, cache_len, own_part in ((first, s["most_group"], s["ptable"], plens, False),
                                                    (qoff, s["most_new"], s["table"], lens, True)):
        at = start[:-1, None] + torch.arange(most, device=dev)[None]
        rows = q[at.clamp(max=T - 1)]
        k, v = _paged(s["k"], table), _paged(s["v"], table)
        key = torch.arange(k.shape[2], device=dev)[None, None]
        limit = cache_len[:, None].expand(at.shape)
        if own_part:
            limit = limit - (start[1:, None] - 1 - at)
        m, l, o = _partial(rows, k, v, key < limit[:, :, None])
        b = seq if own_part else grp
        i = t - start[b]
        parts.append((m[b, i], l[b, i], o[b, i]))
    (m0, l0, o0), (m1, l1, o1) = parts
    m = torch.maximum(m0, m1)
    e0, e1 = torch.exp(m0 - m), torch.exp(m1 - m)
    y = (o0 * e0[..., None] + o1 * e1[..., None]) / (l0 * e0 + l1 * e1)[..., None]
    return y.reshape(T, -1).to(F16)


def _plain(s):
    c = s["case"]
    if c["op"] == "rope":
        T, heads, D = c["T"], c["heads"], c["D"]
        x = s["x"][:, :heads * D].float().view(T, heads, D)
        return _rotate(x, s["pos"], s["freq"], s["factor"], c["rot"], c["layout"]).reshape(T, -1).to(F16)
    if c["op"] == "append":
        heads, kv, D, page = c["heads"], c["kv"], c["D"], c["page"]
        q, k, v = s["z"].float().view(-1, heads + 2 * kv, D).split([heads, kv, kv], 1)
        if c["norm"]:
            q, k = _rms(q, s["qn"]), _rms(k, s["kn"])
        if c["vnorm"]:
            v = _rms(v, None)
        q, k = (_rotate(x, s["pos"], s["freq"], s["factor"], c["rot"], c["layout"]) for x in (q, k))
        live = s["slots"] >= 0
        at = s["slots"][live].long()
        s["k"][at // page, :, at % page] = k[live].to(F16)
        s["v"][at // page, :, at % page] = v[live].to(F16)
        return {"q": q.reshape(q.shape[0], -1).to(F16), "k": s["k"], "v": s["v"]}
    return _attention(s)


# ---------------------------------------------------------------- the framework's calls

_program = {}  # the program's one context


def _handles(s):
    """What a program makes once: the context, and for this state the rotation plan, the cache and the workspace."""
    from __graft_entry__ import load_package
    dj = load_package()
    if "ctx" not in _program:
        _program["ctx"] = dj.Context(0)
    ctx, c = _program["ctx"], s["case"]
    if "freq" in s:
        s["plan"] = ctx.rope_plan(c["rot"], c["layout"], frequencies=s["freq"].tolist(), factor=s["factor"])
    if "k" in s:
        s["cache"] = ctx.kv_cache(s["k"], s["v"])
    if c["op"] == "attention":
        size = ctx.attention_paged_workspace(s["cache"], s["T"], c["heads"], len(s["lens"]), len(s["plens"]))
        s["work"] = torch.empty(size, dtype=torch.uint8, device=DEV)
    s["ctx"] = ctx
    torch.cuda.synchronize()


def _calls(s):
    if "ctx" not in s:
        _handles(s)
    ctx, c = s["ctx"], s["case"]
    if c["op"] == "rope":
        x, y = s["x"], s["y"]
        ctx.call("rope", s["plan"], x, x.shape[1], s["pos"], y, y.shape[1], c["T"], c["heads"], c["D"])
        return y
    if c["op"] == "append":
        z, q = s["z"], s["q"]
        ctx.call("kv_append", s["cache"], s["plan"], z, z.shape[1], s["qn"], s["kn"], 1e-6, int(c["vnorm"]), s["pos"],
                 s["slots"], q, q.shape[1], len(z), c["heads"])
        return {"q": q, "k": s["k"], "v": s["v"]}
    q, y, table, ptable, work = s["q"], s["y"], s["table"], s["ptable"], s["work"]
    ctx.call("attention_paged", s["cache"], q, q.shape[1], table, table.shape[1], s["lens"], s["qoff"], len(table),
             ptable, ptable.shape[1], s["plens"], s["goff"], len(ptable), y, y.shape[1], s["T"], c["heads"],
             1.0 / math.sqrt(c["D"]), work, work.numel())
    return y


def run(state):
    return _calls(state) if own else _plain(state)


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    c = case
    if c["op"] == "rope":
        n = c["T"] * c["heads"]
        return {"bytes": 4.0 * n * c["D"] + 4.0 * c["T"] + 4.0 * c["rot"], "flops": 3.0 * n * c["rot"]}
    heads, kv, D = c["heads"], c["kv"], c["D"]
    if c["op"] == "append":
        T = c["seqs"] * c["tokens"] + c["pads"]
        live = c["seqs"] * c["tokens"]
        read = 2.0 * (T * heads + live * 2 * kv) * D + 8.0 * T
        normed = (heads + kv if c["norm"] else 0) + (kv if c["vnorm"] else 0)
        return {"bytes": read + 2.0 * (T * heads + live * 2 * kv) * D,
                "flops": T * (3.0 * (heads + kv) * c["rot"] + 4.0 * normed * D)}
    per, new, keys, pre = _lengths(c)
    pairs, at = 0, 0
    for g, n in enumerate(per):
        for i in range(at, at + n):
            pairs += new[i] * pre[g] + new[i] * keys[i] - new[i] * (new[i] - 1) // 2
        at += n
    held = sum(keys) + sum(pre)
    return {"bytes": 4.0 * sum(new) * heads * D + 4.0 * held * kv * D + 4.0 * held / c["page"],
            "flops": 4.0 * D * heads * pairs}


# ---------------------------------------------------------------- from the definitions, in 64 bits


def _exact_rotation(x, pos, freq, factor, rot, layout):
    """Pairs as complex numbers, turned by exp(i pos w)."""
    turn = torch.polar(torch.full((), float(factor), dtype=torch.float64, device=x.device),
                       pos.double()[:, None, None] * freq)
    y = x.clone()
    i = torch.arange(rot // 2, device=x.device)
    a, b = (i, i + rot // 2) if layout == "half" else (2 * i, 2 * i + 1)
    z = torch.complex(x[..., a], x[..., b]) * turn
    y[..., a], y[..., b] = z.real, z.imag
    return y


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "rope":
        x = s["x"][:, :c["heads"] * c["D"]].double().reshape(c["T"], c["heads"], c["D"])
        return _exact_rotation(x, s["pos"], s["freq"], s["factor"], c["rot"], c["layout"]).reshape(c["T"], -1)
    heads, kv, D, page = c["heads"], c["kv"], c["D"], c["page"]
    if c["op"] == "append":
        z = s["z"].double().reshape(-1, heads + 2 * kv, D)
        size = z.pow(2).mean(-1, keepdim=True).add(1e-6).sqrt()
        n = z / size
        q, k, v = z[:, :heads], z[:, heads:heads + kv], z[:, heads + kv:]
        if c["norm"]:
            q, k = n[:, :heads] * s["qn"].double(), n[:, heads:heads + kv] * s["kn"].double()
        if c["vnorm"]:
            v = n[:, heads + kv:]
        q = _exact_rotation(q, s["pos"], s["freq"], s["factor"], c["rot"], c["layout"])
        k = _exact_rotation(k, s["pos"], s["freq"], s["factor"], c["rot"], c["layout"])
        kc, vc = s["k"].double().transpose(1, 2).flatten(0, 1), s["v"].double().transpose(1, 2).flatten(0, 1)
        live = (s["slots"] >= 0).nonzero()[:, 0]
        kc[s["slots"][live].long()], vc[s["slots"][live].long()] = k[live], v[live]
        back = lambda x: x.view(-1, page, kv, D).transpose(1, 2).contiguous()  # noqa: E731
        return {"q": q.reshape(len(z), -1), "k": back(kc), "v": back(vc)}
    per, new, keys, pre = _lengths(c)
    if work(case)["flops"] > 2e12:
        return None
    r = heads // kv
    y = torch.empty(s["T"], heads, D, dtype=torch.float64, device=DEV)
    take = lambda cache, row, n: cache[row[:-(-n // page)].long()].double().transpose(0, 1).reshape(kv, -1, D)[:, :n]  # noqa: E731
    t, i = 0, 0
    for g, count in enumerate(per):
        pk, pv = (take(s[x], s["ptable"][g], pre[g]) for x in "kv")
        for i in range(i, i + count):
            n = new[i]
            k = torch.cat([pk, take(s["k"], s["table"][i], keys[i])], 1).repeat_interleave(r, 0)
            v = torch.cat([pv, take(s["v"], s["table"][i], keys[i])], 1).repeat_interleave(r, 0)
            q = s["q"][t:t + n].double().view(n, heads, D).transpose(0, 1)
            a = q @ k.transpose(1, 2) * D ** -0.5
            hidden = torch.ones(n, k.shape[1], dtype=torch.bool, device=DEV).triu(k.shape[1] - n + 1)
            y[t:t + n] = (torch.softmax(a.masked_fill(hidden, -math.inf), -1) @ v).transpose(0, 1)
            t += n
        i += 1
    return y.reshape(s["T"], -1)

"""An 8-bit paged KV cache that is planned on the GPU, and the operators around it.

  map     block tables, positions and slot maps of a step from request lengths
          that live on the GPU: rows take pages from a stack and give them back
  rope    rotary positions of q and k heads, with their norms: half and
          interleaved layouts, part of the head, scaled for long contexts
  append  new keys and values into the cache, e4m3 under a power-of-two scale for
          each block of 64 tokens and head, and the blocks read back
  attn    attention over that cache: one new token a sequence or many, scores
          capped, windows, prefixes, a bias by distance, an output gate

Sizes are those of the attention layers that the tests and the benchmark use (16
query and 2 key/value heads of 256) and generic ones. With `own` false, run()
computes the operators with elementary torch operations; with `own` true it calls
the library.
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda:0"
BF = torch.bfloat16
F8 = torch.float8_e4m3fn
F32 = torch.float32
F64 = torch.float64
I32 = torch.int32
PAGE = 64
E_MIN, E_MAX = -40, 56  # exponents of a block's scale


def _gdn():
    path = os.path.join(os.getcwd(), "qwen-mlx_amd")
    if path not in sys.path:
        sys.path.insert(1, path)
    import gdn_amd
    return gdn_amd


# ------------------------------------------------------------------- cases --

def _map(**kw):
    # rows: sequences of the step; new: their most new tokens; done, padding: shares of
    # rows that leave and of rows that stand for none; short: the pages do not suffice
    c = dict(op="map", rows=64, ctx=4096, new=1, done=0.0, padding=0.0, short=False, mix=1)
    c.update(kw)
    return c


def _rope(**kw):
    c = dict(op="rope", tokens=64, hq=16, hk=2, dim=256, rot=64, interleaved=False,
             scaling="none", factor=1.0, base=1.0e7, norm=True, f32=False, far=8192)
    c.update(kw)
    return c


def _append(**kw):
    c = dict(op="append", rows=64, ctx=4096, new=1, hq=16, hk=2, dim=256, mix=1)
    c.update(kw)
    return c


def _attn(**kw):
    c = dict(op="attn", rows=64, ctx=4096, new=1, hq=16, hk=2, dim=256, cap=0.0, window=0,
             slopes=False, prefix=False, gate=False, mix=1)
    c.update(kw)
    return c


def listed():
    return [
        # a full decode batch that grows by a token each: one launch, latency
        _map(name="map_b64"),
        # many requests: prompts admitted, tokens decoded, some done, some rows
        # only padding, and not enough pages for all of them
        _map(name="map_700_mixed", rows=700, ctx=3000, new=900, done=0.1, padding=0.05, short=True),
        # a decode batch's heads, norm and a quarter of the head turned
        _rope(name="rope_b64"),
        # a long prompt's heads
        _rope(name="rope_16384", tokens=16384, far=16384),
        # an odd prompt in f32 at far positions of a stretched context, the whole
        # head turned in neighbouring pairs
        _rope(name="rope_far_5003", tokens=5003, hq=32, hk=8, dim=128, rot=128, interleaved=True,
              scaling="yarn", factor=32.0, base=1.0e4, norm=False, f32=True, far=1000000),
        # a decode batch's keys and values
        _append(name="append_b64"),
        # ragged prompts behind cached tokens, other heads
        _append(name="append_ragged", rows=11, ctx=500, new=3000, hq=32, hk=8, dim=128),
        # one user far into a conversation
        _attn(name="attn_b1_ctx32k", rows=1, ctx=32767, gate=True),
        # a full decode batch at ragged lengths
        _attn(name="attn_b64_ctx4k", gate=True),
        # a small batch of another model: a window, capped scores
        _attn(name="attn_b23_window", rows=23, ctx=9000, hq=32, hk=8, dim=128, cap=30.0,
              window=1024),
        # a long prompt into an empty cache
        _attn(name="attn_prompt_8192", rows=1, ctx=0, new=8192, gate=True),
        # ragged prompts, follow-ups and single tokens with a bias by distance
        # and a prefix that every token sees
        _attn(name="attn_ragged", rows=19, ctx=4000, new=700, hq=16, hk=4, dim=64, slopes=True,
              prefix=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["map", "rope", "append", "attn", "attn"])
    mix = rng.randrange(1 << 30)
    dim = rng.choice([64, 128, 256])
    hk = rng.choice([1, 2, 4, 8])
    hq = hk * rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 16])
    if op == "map":
        rows = _log(rng, 1, 1000)
        return _map(rows=rows, ctx=_log(rng, 1, 8000), new=_log(rng, 1, max(1, 200000 // rows)),
                    done=rng.choice([0.0, 0.2]), padding=rng.choice([0.0, 0.1]),
                    short=rng.random() < 0.4, mix=mix)
    if op == "rope":
        dim = rng.choice([64, 96, 128, 192, 256, 512])
        rot = rng.choice([dim, dim, dim // 2, dim // 4, 2 * rng.randint(1, dim // 2)])
        hq, hk = rng.randint(1, 40), rng.randint(0, 8)
        f32 = rng.random() < 0.4
        most = 16384 * 18 * 256 // (hq + hk) // dim // (2 if f32 else 1)
        scaling = rng.choice(["none", "linear", "yarn", "bands"])
        return _rope(tokens=_log(rng, 1, min(most, 16384)), hq=hq, hk=hk, dim=dim, rot=rot,
                     interleaved=rng.random() < 0.5, scaling=scaling,
                     factor=1.0 if scaling == "none" else rng.choice([2.0, 8.0, 32.0]),
                     base=rng.choice([1.0e4, 5.0e5, 1.0e7]), norm=rng.random() < 0.5, f32=f32,
                     far=_log(rng, 100, 1000000))
    # keys of all rows, in heads of this size
    keys = min(262144, 262144 * 512 // (hk * dim))
    if op == "append":
        rows = _log(rng, 1, 256)
        most = min(keys, 33000 * 1024 // (hk * dim)) // rows
        return _append(rows=rows, ctx=_log(rng, 1, max(1, min(keys // rows - 1, 8000))),
                       new=_log(rng, 1, max(1, min(most, 16384))), hq=hq, hk=hk, dim=dim, mix=mix)
    rows = _log(rng, 1, 256)
    ctx = _log(rng, 1, max(1, min(32768, keys // rows)))
    new = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 16, 8192)])
    if new > 1:
        # the products of the listed prompt, and no more keys than above
        pairs = 4096 * 8192 * 8192 // (2 * hq * dim)
        new = min(new, max(2, int(pairs / rows / (ctx + 64))), max(2, int(math.sqrt(pairs / rows))),
                  max(2, keys // rows))
    return _attn(rows=rows, ctx=rng.choice([0, ctx]) if new > 1 else ctx, new=new, hq=hq, hk=hk,
                 dim=dim, cap=rng.choice([0.0, 0.0, 20.0, 50.0]),
                 window=rng.choice([0, 0, _log(rng, 1, 4096)]), slopes=rng.random() < 0.3,
                 prefix=rng.random() < 0.3, gate=rng.random() < 0.5, mix=mix)


# -------------------------------------------------------------------- rows --

def _lengths(case):
    """Per row the cached and the new tokens, from the case alone."""
    rng = random.Random(case["mix"])
    n, ctx, new = case["rows"], case["ctx"], case["new"]
    if n == 1:
        return [ctx], [new]
    old = [rng.randint(ctx // 2, ctx + ctx // 2) for _ in range(n)]
    fresh = [new if new == 1 else _log(rng, 1, new) for _ in range(n)]
    return old, fresh


def _pages(tokens):
    return -(-tokens // PAGE)


def _plan(case):
    """A step's rows: slots, cached and new tokens, what is cached before the step, and
    the sizes of the cache."""
    rng = random.Random(case["mix"] + 1)
    old, new = _lengths(case)
    n = case["rows"]
    num_slots = n + n // 4 + 1
    slots = rng.sample(range(num_slots), n)
    before = list(old)
    if case["op"] == "map":
        for i in range(n):
            kind = rng.random()
            if kind < case["done"]:  # done: its pages go back
                old[i] = new[i] = 0
            elif kind < case["done"] + case["padding"]:
                slots[i], old[i], new[i], before[i] = -1, 0, 0, 0
            elif kind < case["done"] + case["padding"] + 0.3 and case["new"] > 1:
                new[i] = 1  # decodes while others are admitted
            elif kind > 0.9 and old[i] > 8:
                old[i] -= 8  # the last tokens were rejected
    last = [a + b for a, b in zip(old, new)]
    owned = sum(_pages(t) for t in before)
    need = sum(max(0, _pages(t) - _pages(b)) for t, b in zip(last, before))
    num_pages = owned + (need // 2 if case.get("short") else need + 7) + 1
    return dict(slots=slots, old=old, new=new, before=before, num_slots=num_slots,
                num_pages=num_pages, max_pages=_pages(max(last + before)) + 1,
                tokens=max(1, sum(new)))


def _growth(plan):
    """Steps without tokens that reserve the pages of what is cached: in four rounds, so
    that the rows' pages lie between each other's."""
    slots = [s for s in plan["slots"] if s >= 0]
    before = [b for s, b in zip(plan["slots"], plan["before"]) if s >= 0]
    return slots, [[(b * r) // 4 for b in before] for r in range(1, 5)]


def _ordered(case, seed):
    """The map cases' rows in the order that the seed gives them."""
    p = _plan(case)
    order = list(range(len(p["slots"])))
    random.Random(seed).shuffle(order)
    for x in ("slots", "old", "new", "before"):
        p[x] = [p[x][i] for i in order]
    return p


# ------------------------------------------------------------------ inputs --

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _n(g, *shape, std=1.0, dtype=BF):
    return torch.empty(shape, device=DEV, dtype=F32).normal_(0, std, generator=g).to(dtype)


def _i(values):
    return torch.tensor(values, device=DEV, dtype=I32)


def _kv(g, tokens, case):
    """Keys and values: channels of different sizes, stretches of different loudness."""
    hk, d = case["hk"], case["dim"]
    out = []
    for _ in range(2):
        chan = torch.exp2(_n(g, hk, d, std=0.7, dtype=F32))
        loud = torch.exp2(_n(g, -(-tokens // 96), hk, 1, std=0.5, dtype=F32))
        x = torch.empty(tokens, hk, d, device=DEV, dtype=BF)
        for a in range(0, tokens, 96 * 512):
            b = min(a + 96 * 512, tokens)
            s = loud[a // 96:-(-b // 96)].repeat_interleave(96, 0)[:b - a]
            x[a:b] = (_n(g, b - a, hk, d, dtype=F32) * chan * s).to(BF)
        out.append(x)
    return out


def _rope_inputs(case, seed):
    g = _gen(seed)
    t, d = case["tokens"], case["dim"]
    dt = F32 if case["f32"] else BF
    first = int(torch.randint(0, max(1, case["far"] - t), (1,), device=DEV, generator=g))
    pos = torch.arange(first, first + t, device=DEV, dtype=I32)
    if t > 8:  # packed sequences: the second half starts elsewhere
        pos[t // 2:] -= int(pos[t // 2]) // 3
    wt = lambda: (1.0 + 0.1 * _n(g, d, dtype=F32)).to(BF)  # noqa: E731
    return dict(q=_n(g, t, case["hq"], d, dtype=dt), pos=pos,
                k=_n(g, t, case["hk"], d, dtype=dt) if case["hk"] else None,
                qw=wt() if case["norm"] else None,
                kw=wt() if case["norm"] and case["hk"] else None)


def _step_inputs(case, seed):
    """What the append and attention cases have in hand: the rows, the cached tokens' keys
    and values, the new ones'."""
    g = _gen(seed)
    p = _plan(case)
    s = dict(plan=p, slots=_i(p["slots"]), lens=_i(p["old"]), ntok=_i(p["new"]))
    s["ck"], s["cv"] = _kv(g, max(1, sum(p["old"])), case)
    s["k"], s["v"] = _kv(g, p["tokens"], case)
    if case["op"] == "attn":
        t, hq, d = p["tokens"], case["hq"], case["dim"]
        s["q"] = _n(g, t, hq, d, std=1.5)
        s["gate"] = _n(g, t, hq, d) if case["gate"] else None
        s["slopes"] = torch.exp2(torch.empty(hq, device=DEV).uniform_(-9, -1, generator=g)) \
            if case["slopes"] else None
        s["prefix"] = None
        if case["prefix"]:
            r = torch.rand(len(p["old"]), device=DEV, generator=g, dtype=F64)
            s["prefix"] = (r * 0.5 * (s["lens"] + s["ntok"])).to(I32)
    return s


# ----------------------------------------------------- plain form: the map --

def _empty_map(plan):
    n, m = plan["num_slots"], plan["num_pages"]
    return dict(table=torch.full((n, plan["max_pages"]), -1, device=DEV, dtype=I32),
                owned=torch.zeros(n, device=DEV, dtype=I32),
                free=torch.arange(m - 1, -1, -1, device=DEV, dtype=I32),
                count=torch.full((1,), m, device=DEV, dtype=I32))


def _plain_map(m, slots, lens, ntok, tokens):
    """One step on the tables m; new ones, with cu, pos, map and the new lengths."""
    table, owned, free, count = (m[x].clone() for x in ("table", "owned", "free", "count"))
    n, top = slots.numel(), table.shape[1] * PAGE
    there = slots >= 0
    take = torch.where(there, ntok, 0)
    cu = torch.zeros(n + 1, device=DEV, dtype=I32)
    cu[1:] = torch.cumsum(take, 0)
    last = lens + ntok
    ok = there & (last <= top) & (cu[1:] <= tokens)
    sl = torch.where(ok, slots, 0).long()
    have = torch.where(ok, owned[sl], 0)
    need = torch.where(ok, (last + PAGE - 1) // PAGE, 0)
    give = torch.clamp(have - need, min=0)
    grow = torch.clamp(need - have, min=0)
    # pages given back: row after row, a row's last page first
    rows = torch.repeat_interleave(torch.arange(n, device=DEV), give.long())
    j = torch.arange(rows.numel(), device=DEV) - (torch.cumsum(give, 0) - give)[rows]
    at = have[rows] - 1 - j
    free[count.long() + torch.arange(rows.numel(), device=DEV)] = table[sl[rows], at.long()]
    table[sl[rows], at.long()] = -1
    count = count + rows.numel()
    # pages taken: from the top of the stack, row after row, in order of position
    ok = ok & ((grow == 0) | (torch.cumsum(grow, 0) <= count))
    grow = torch.where(ok, grow, 0)
    rows = torch.repeat_interleave(torch.arange(n, device=DEV), grow.long())
    j = torch.arange(rows.numel(), device=DEV) - (torch.cumsum(grow, 0) - grow)[rows]
    src = count.long() - 1 - torch.arange(rows.numel(), device=DEV)
    table[sl[rows], (have[rows] + j).long()] = free[src]
    free[src] = -1
    count = (count - rows.numel()).to(I32)
    owned[sl[ok]] = need[ok].to(I32)
    # tokens
    t = torch.arange(tokens, device=DEV, dtype=I32)
    row = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=n - 1)
    live = (t < cu[n]) & ok[row]
    pos = torch.where(live, lens[row] + t - cu[row], -1).to(I32)
    page = table[sl[row], torch.clamp(pos, min=0).long() // PAGE]
    where = torch.where(live, page * PAGE + pos % PAGE, -1).to(I32)
    new_lens = torch.where(ok, last, lens).to(I32)
    return dict(table=table, owned=owned, free=free, count=count, cu=cu, pos=pos, map=where,
                lens=new_lens)


def _grown(plan):
    m = _empty_map(plan)
    slots, rounds = _growth(plan)
    if slots:
        for lens in rounds:
            m = _plain_map(m, _i(slots), _i(lens), torch.zeros(len(slots), device=DEV, dtype=I32), 1)
    return m


# --------------------------------------------------- plain form: the cache --

def _exponent(amax):
    """The least e with amax <= 448 * 2^e, inside [E_MIN, E_MAX]."""
    mant, ex = torch.frexp(amax)
    e = torch.where(mant <= 0.875, ex - 9, ex - 8)
    return torch.where(amax > 0, e, E_MIN).clamp(E_MIN, E_MAX).to(I32)


def _e4m3(y):
    """y rounded to the nearest e4m3 number, ties to even, saturating."""
    _, ex = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), torch.clamp(ex - 1, min=-6) - 3)
    return torch.clamp(torch.round(y / step) * step, -448.0, 448.0)


def _hold(x):
    """Blocks [b, 64, heads, dim] in f32 -> what is held: e4m3 numbers, exponents [b, heads]."""
    e = _exponent(x.abs().amax(dim=(1, 3)))
    q = _e4m3(torch.ldexp(x, -e[:, None, :, None]))
    return q.to(F8), e


def _values(q, e):
    return torch.ldexp(q.to(F32), e[:, None, :, None])


def _plain_append(c, table, slots, lens, ntok, cu, k, v):
    """The rows' new tokens into the cache c; blocks of rows in order. Returns the values
    that the touched blocks stand for, [tokens, heads, dim] of each."""
    outs = ([], [])
    for i, (s, a, b) in enumerate(zip(slots, lens, ntok)):
        if b == 0 or s < 0:
            continue
        b0, b1 = a // PAGE, _pages(a + b)
        pages = table[s, b0:b1].long()
        for z, x in enumerate((k, v)):
            for h in range(0, b1 - b0, 256):
                pg = pages[h:h + 256]
                first = (b0 + h) * PAGE
                blk = torch.zeros(pg.numel() * PAGE, *x.shape[1:], device=DEV, dtype=F32)
                if a > first:  # tokens of the first block that were there
                    blk[:a - first] = _values(c["q"][pg[:1], z], c["e"][pg[:1], z])[0, :a - first]
                lo, hi = max(a, first), min(a + b, first + blk.shape[0])
                blk[lo - first:hi - first] = x[cu[i] + lo - a:cu[i] + hi - a].to(F32)
                q, e = _hold(blk.view(pg.numel(), PAGE, *x.shape[1:]))
                c["q"][pg, z], c["e"][pg, z] = q, e
                outs[z].append(_values(q, e).view(-1, *x.shape[1:])[:hi - first].to(BF))
    return torch.cat(outs[0]), torch.cat(outs[1])


def _blank(case, plan):
    return dict(q=torch.zeros(plan["num_pages"], 2, PAGE, case["hk"], case["dim"], device=DEV,
                              dtype=F8),
                e=torch.zeros(plan["num_pages"], 2, case["hk"], device=DEV, dtype=I32))


def _starts(counts):
    out = [0]
    for x in counts:
        out.append(out[-1] + x)
    return out


def _plain_cache(case, s):
    """Tables and cache with the cached tokens in place, and the step's map."""
    p = s["plan"]
    m = _grown(p)
    c = _blank(case, p)
    if sum(p["old"]):
        zero = [0] * len(p["old"])
        _plain_append(c, m["table"], p["slots"], zero, p["old"], _starts(p["old"]), s["ck"], s["cv"])
    return _plain_map(m, s["slots"], s["lens"], s["ntok"], p["tokens"]), c


# ----------------------------------------------------- plain form: the rest --

def _frequencies(c):
    """Turns of a pair per position (in 64 bits) and the factor on cos and sin."""
    half, base, f = c["rot"] // 2, c["base"], c["factor"]
    i = torch.arange(half, device=DEV, dtype=F64)
    w = base ** (-2.0 * i / c["rot"])
    if c["scaling"] == "linear":
        w = w / f
    if c["scaling"] == "yarn":  # between pairs that turn 32 times and once in 4096 positions
        at = [c["rot"] * math.log(4096 / (b * 2 * math.pi)) / (2 * math.log(base)) for b in (32, 1)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), c["rot"] - 1)
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        w = w / f * ramp + w * (1 - ramp)
    if c["scaling"] == "bands":  # by turns in 8192 positions: below 1 slowed, above 4 kept
        turns = 8192 * w / (2 * math.pi)
        keep = ((turns - 1) / 3).clamp(0, 1)
        w = w / f * (1 - keep) + w * keep
    return w, 0.1 * math.log(f) + 1.0 if c["scaling"] == "yarn" else 1.0


def _plain_rope(s):
    c = s["case"]
    rot, half = c["rot"], c["rot"] // 2
    w, mag = _frequencies(c)
    ang = s["pos"].to(F64)[:, None] * w
    cos, sin = ((mag * f(ang)).to(F32)[:, None, :] for f in (torch.cos, torch.sin))

    def one(x, wt):
        y = x.to(F32)
        if wt is not None:
            y = y / torch.sqrt(y.square().mean(2, keepdim=True) + 1e-6) * wt.to(F32)
        z = y.clone()
        if c["interleaved"]:
            a, b = y[..., 0:rot:2], y[..., 1:rot:2]
            z[..., 0:rot:2], z[..., 1:rot:2] = a * cos - b * sin, a * sin + b * cos
        else:
            a, b = y[..., :half], y[..., half:rot]
            z[..., :half], z[..., half:rot] = a * cos - b * sin, a * sin + b * cos
        return z.to(x.dtype)

    out = [one(s["q"], s["qw"])]
    if s["k"] is not None:
        out.append(one(s["k"], s["kw"]))
    return tuple(out)


def _attend(s, dtype):
    """Rows in order, queries in pieces whose scores fit."""
    c, p, m = s["case"], s["plan"], s["map"]
    hq, hk, d = c["hq"], c["hk"], c["dim"]
    g = hq // hk
    out = torch.zeros(p["tokens"], hq, d, device=DEV, dtype=dtype)
    cu = _starts(p["new"])
    for i, slot in enumerate(p["slots"]):
        n, total = p["new"][i], p["old"][i] + p["new"][i]
        pages = m["table"][slot, :_pages(total)].long()
        kv = []
        for z in range(2):
            x = _values(s["cache"]["q"][pages, z], s["cache"]["e"][pages, z])
            kv.append(x.reshape(-1, hk, d)[:total].to(dtype).permute(1, 0, 2).contiguous())
        kt = kv[0].transpose(1, 2).contiguous()
        key = torch.arange(total, device=DEV)
        piece = max(1, 2 ** 28 // (hq * total))
        for a in range(0, n, piece):
            b = min(a + piece, n)
            q = s["q"][cu[i] + a:cu[i] + b].to(dtype).view(b - a, hk, g, d).permute(1, 2, 0, 3)
            sc = torch.matmul(q.reshape(hk, g * (b - a), d), kt) / math.sqrt(d)
            if c["cap"]:
                sc = c["cap"] * torch.tanh(sc / c["cap"])
            sc = sc.view(hk, g, b - a, total)
            pos = p["old"][i] + torch.arange(a, b, device=DEV)[:, None]
            if s["slopes"] is not None:
                sc = sc - s["slopes"].to(dtype).view(hk, g, 1, 1) * (pos - key).to(dtype)
            see = key <= pos
            if c["window"]:
                see = see & (key > pos - c["window"])
            if s["prefix"] is not None:
                see = see | (key < s["prefix"][i])
            sc = torch.where(see, sc, float("-inf"))
            pr = torch.exp(sc - sc.amax(3, keepdim=True))
            pr = (pr / pr.sum(3, keepdim=True)).view(hk, g * (b - a), total)
            o = torch.matmul(pr, kv[1]).view(hk, g, b - a, d).permute(2, 0, 1, 3)
            out[cu[i] + a:cu[i] + b] = o.reshape(b - a, hq, d)
    if s["gate"] is not None:
        out = out / (1 + torch.exp(-s["gate"].to(dtype)))
    return out


# ----------------------------------------------------------------- prepare --

def _handle(case, plan, tokens):
    return _gdn().KV8Cache(1, plan["num_slots"], plan["num_pages"], plan["max_pages"],
                           case.get("hq", 16), case.get("hk", 2), case.get("dim", 256),
                           max_step_tokens=tokens)


def _reserve(kv, plan):
    slots, rounds = _growth(plan)
    if slots:
        s, zero = _i(slots), torch.zeros(len(slots), device=DEV, dtype=I32)
        for lens in rounds:
            kv.step(s, _i(lens), zero, 1)


def _own_cache(case, s):
    p = s["plan"]
    most = 32768
    kv = _handle(case, p, max(most, p["tokens"], max(p["old"])))
    _reserve(kv, p)
    cu, i = _starts(p["old"]), 0
    while i < len(p["old"]):  # whole rows, as many as a step takes
        j = i + 1
        while j < len(p["old"]) and cu[j + 1] - cu[i] <= most:
            j += 1
        n = cu[j] - cu[i]
        if n:
            kv.step(s["slots"][i:j].clone(), torch.zeros(j - i, device=DEV, dtype=I32),
                    s["lens"][i:j].clone(), n)
            kv.append(0, s["ck"][cu[i]:cu[j]], s["cv"][cu[i]:cu[j]])
        i = j
    kv.step(s["slots"], s["lens"], s["ntok"], p["tokens"], max(p["new"]))
    return kv


def _touched(case, plan, table):
    """Where the blocks that the step's tokens fall into lie in the cache, token by token."""
    at = []
    for s, a, b in zip(plan["slots"], plan["old"], plan["new"]):
        t = torch.arange(a // PAGE * PAGE, a + b, device=DEV)
        at.append(table[s, t // PAGE] * PAGE + t % PAGE)
    return torch.cat(at).to(I32)


def prepare(case, seed):
    if case["op"] == "map":
        p = _ordered(case, seed)
        s = dict(plan=p, slots=_i(p["slots"]), lens=_i(p["old"]), ntok=_i(p["new"]))
        if own:
            s["kv"] = _handle(case, p, p["tokens"])
            _reserve(s["kv"], p)
            s["views"] = s["kv"].views()
            s["lens_out"] = torch.empty_like(s["lens"])
        else:
            s["tables"] = _grown(p)
    elif case["op"] == "rope":
        s = _rope_inputs(case, seed)
        if own:
            kw = {"linear": {}, "none": {}, "yarn": dict(original=4096, fast=32.0, slow=1.0),
                  "bands": dict(original=8192, fast=4.0, slow=1.0)}[case["scaling"]]
            s["rope"] = _gdn().Rope(case["dim"], case["rot"], case["base"],
                                    interleaved=case["interleaved"], scaling=case["scaling"],
                                    factor=case["factor"], **kw)
            s["qo"] = torch.empty_like(s["q"])
            s["ko"] = None if s["k"] is None else torch.empty_like(s["k"])
    else:
        s = _step_inputs(case, seed)
        p = s["plan"]
        if own:
            s["kv"] = _own_cache(case, s)
            if case["op"] == "append":
                s["at"] = _touched(case, p, s["kv"].views()["table"])
                s["ko"] = torch.empty(s["at"].numel(), case["hk"], case["dim"], device=DEV, dtype=BF)
                s["vo"] = torch.empty_like(s["ko"])
            else:
                s["kv"].append(0, s["k"], s["v"])
                s["out"] = torch.empty_like(s["q"])
        else:
            s["map"], s["cache"] = _plain_cache(case, s)
            if case["op"] == "attn":
                _plain_append(s["cache"], s["map"]["table"], p["slots"], p["old"], p["new"],
                              _starts(p["new"]), s["k"], s["v"])
        del s["ck"], s["cv"]
    s["case"] = case
    return s


# --------------------------------------------------------------------- run --

def run(state):
    s = state
    c = s["case"]
    if c["op"] == "map":
        p = s["plan"]
        n, t = len(p["slots"]), p["tokens"]
        if own:
            s["kv"].step(s["slots"], s["lens"], s["ntok"], t, lens_out=s["lens_out"])
            o = s["views"]
            return (o["table"], o["owned"], o["free"], o["count"], o["cu"][:n + 1], o["pos"][:t],
                    o["map"][:t], s["lens_out"])
        o = _plain_map(s["tables"], s["slots"], s["lens"], s["ntok"], t)
        return tuple(o[x] for x in ("table", "owned", "free", "count", "cu", "pos", "map", "lens"))
    if c["op"] == "rope":
        if not own:
            return _plain_rope(s)
        s["rope"].forward(s["pos"], s["q"], s["k"], q_out=s["qo"], k_out=s["ko"], q_norm_w=s["qw"],
                          k_norm_w=s["kw"], eps=1e-6)
        return (s["qo"],) if s["ko"] is None else (s["qo"], s["ko"])
    if c["op"] == "append":
        if own:
            s["kv"].append(0, s["k"], s["v"])
            s["kv"].gather(0, s["at"], s["ko"], s["vo"])
            return s["ko"], s["vo"]
        p = s["plan"]
        return _plain_append(s["cache"], s["map"]["table"], p["slots"], p["old"], p["new"],
                             _starts(p["new"]), s["k"], s["v"])
    if own:
        s["kv"].attention(0, s["q"], s["out"], softcap=c["cap"], window=c["window"],
                          slopes=s["slopes"], prefix=s["prefix"], gate=s["gate"])
        return s["out"]
    return _attend(s, F32).to(BF)


# ------------------------------------------------------------ work, exact --

def work(case):
    c = case
    if c["op"] == "rope":
        t, h = c["tokens"], c["hq"] + c["hk"]
        return {"bytes": 2 * t * h * c["dim"] * (4 if c["f32"] else 2) + 4 * t,
                "flops": t * h * (3 * c["rot"] + (4 * c["dim"] if c["norm"] else 0))}
    p = _plan(c)
    if c["op"] == "map":
        # the rows' numbers, the tables' changes, a position and a place for each token
        moved = sum(abs(_pages(a + b) - _pages(x)) for a, b, x in zip(p["old"], p["new"], p["before"]))
        return {"bytes": 20 * c["rows"] + 8 * p["tokens"] + 12 * moved,
                "flops": 10 * c["rows"] + 8 * p["tokens"]}
    row = 2 * c["hk"] * c["dim"]  # keys and values of a token
    if c["op"] == "append":
        old = sum(a % PAGE for a in p["old"])
        tok = old + p["tokens"]
        # new rows in, the blocks' old bytes in, bytes out, and read back as bf16
        return {"bytes": row * (2 * p["tokens"] + old + tok + tok + 2 * tok), "flops": 8 * row * tok}
    keys = pairs = 0
    for a, b in zip(p["old"], p["new"]):
        if c["prefix"]:  # a quarter of the row on average
            pre = (a + b) // 4
        else:
            pre = 0
        w = c["window"] or a + b
        lo = max(0, a + 1 - w)
        keys += a + b - max(0, lo - min(lo, pre))
        for t in range(a, a + b):
            pairs += min(t + 1, w) + min(pre, max(0, t + 1 - w)) + max(0, pre - t - 1)
    io = 2 * p["tokens"] * c["hq"] * c["dim"] * (3 if c["gate"] else 2)
    return {"bytes": keys * row + io, "flops": 4 * pairs * c["hq"] * c["dim"]}


def _exact_map(case, seed):
    """Row by row, on lists."""
    p = _ordered(case, seed)
    n, top = len(p["slots"]), p["max_pages"]
    table = [[] for _ in range(p["num_slots"])]
    free = list(range(p["num_pages"] - 1, -1, -1))

    def step(slots, lens, ntok, tokens):
        cu, ok, at = [0], [], 0
        for s, a, b in zip(slots, lens, ntok):
            at += b if s >= 0 else 0
            cu.append(at)
            ok.append(s >= 0 and a + b <= top * PAGE and at <= tokens)
        need = [-(-(a + b) // PAGE) for a, b in zip(lens, ntok)]
        for i, s in enumerate(slots):
            while ok[i] and len(table[s]) > need[i]:
                free.append(table[s].pop())
        budget = len(free)
        for i, s in enumerate(slots):
            grow = need[i] - len(table[s]) if ok[i] else 0
            if grow > 0:
                budget -= grow
                if budget < 0:
                    ok[i] = False
                    continue
                table[s] += [free.pop() for _ in range(grow)]
        pos, where = [-1] * tokens, [-1] * tokens
        for i, s in enumerate(slots):
            for t in range(cu[i], cu[i + 1]):
                if ok[i]:
                    pos[t] = lens[i] + t - cu[i]
                    where[t] = table[s][pos[t] // PAGE] * PAGE + pos[t] % PAGE
        return cu, pos, where, [a + b if o else a for a, b, o in zip(lens, ntok, ok)]

    slots, rounds = _growth(p)
    for lens in rounds if slots else []:
        step(slots, lens, [0] * len(slots), 1)
    cu, pos, where, last = step(p["slots"], p["old"], p["new"], p["tokens"])
    wide = [r + [-1] * (top - len(r)) for r in table]
    return (_i(wide), _i([len(r) for r in table]), _i(free + [-1] * (p["num_pages"] - len(free))),
            _i([len(free)]), _i(cu), _i(pos), _i(where), _i(last))


def _exact_rope(case, i):
    """Each pair as a complex number, turned by exp(i angle)."""
    half, rot = case["rot"] // 2, case["rot"]
    w = []
    for j in range(half):
        f = case["base"] ** (-(2.0 * j) / rot)
        if case["scaling"] == "linear":
            f /= case["factor"]
        elif case["scaling"] == "yarn":
            near, far = (rot / 2 * math.log(4096 / (2 * math.pi * b), case["base"]) for b in (32, 1))
            near, far = max(math.floor(near), 0), min(math.ceil(far), rot - 1)
            slow = min(1.0, max(0.0, (j - near) / max(far - near, 0.001)))
            f = f * (slow / case["factor"] + 1 - slow)
        elif case["scaling"] == "bands":
            keep = min(1.0, max(0.0, (8192 * f / (2 * math.pi) - 1) / 3))
            f = f * ((1 - keep) / case["factor"] + keep)
        w.append(f)
    mag = 1 + math.log(case["factor"]) / 10 if case["scaling"] == "yarn" else 1.0
    turn = torch.polar(torch.full((1, half), mag, device=DEV, dtype=F64).expand(len(i["pos"]), half),
                       i["pos"].double()[:, None] * torch.tensor(w, device=DEV, dtype=F64))

    def one(x, wt):
        y = x.double()
        if wt is not None:
            y = y * torch.rsqrt(torch.linalg.vector_norm(y, dim=2, keepdim=True) ** 2 / y.shape[2]
                                + 1e-6) * wt.double()
        head = y[..., :rot]
        pair = head.unflatten(2, (half, 2)) if case["interleaved"] else \
            head.unflatten(2, (2, half)).transpose(2, 3)
        z = torch.view_as_real(torch.complex(pair[..., 0], pair[..., 1]) * turn[:, None, :])
        z = z if case["interleaved"] else z.transpose(2, 3)
        return torch.cat([z.flatten(2), y[..., rot:]], 2)

    out = [one(i["q"], i["qw"])]
    if i["k"] is not None:
        out.append(one(i["k"], i["kw"]))
    return tuple(out)


def _exact_hold(x):
    """One block [tokens, heads, dim] in 64 bits -> the values that are held, by a search
    among all of e4m3's numbers."""
    grid = torch.tensor([m * 2.0 ** -9 for m in range(8)] +
                        [(8 + m) * 2.0 ** (e - 3) for e in range(-6, 9) for m in range(8)][:-1],
                        device=DEV, dtype=F64)
    out = torch.empty_like(x)
    for h in range(x.shape[1]):
        e, most = E_MIN, float(x[:, h].abs().max())
        while most > 448 * 2.0 ** e and e < E_MAX:
            e += 1
        y = x[:, h].abs() / 2.0 ** e
        hi = torch.searchsorted(grid, y).clamp(max=grid.numel() - 1)
        lo = (hi - 1).clamp(min=0)
        up, down = grid[hi] - y, y - grid[lo]
        hi = torch.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
        out[:, h] = torch.copysign(grid[hi] * 2.0 ** e, x[:, h])
    return out


def _exact_append(case, seed):
    s = _step_inputs(case, seed)
    p = s["plan"]
    if sum(_pages(a + b) - a // PAGE for a, b in zip(p["old"], p["new"])) * case["hk"] > 6000:
        return None
    outs = ([], [])
    old, new = _starts(p["old"]), _starts(p["new"])
    for i in range(len(p["slots"])):
        a, b = p["old"][i], p["new"][i]
        for z, (c, x) in enumerate(((s["ck"], s["k"]), (s["cv"], s["v"]))):
            for t in range(a // PAGE * PAGE, a + b, PAGE):
                lo, hi = max(t, a), min(t + PAGE, a + b)
                part = x[new[i] + lo - a:new[i] + hi - a].double()
                if t < a:
                    was = _exact_hold(c[old[i] + t:old[i] + a].double())
                    part = torch.cat([was, part])
                outs[z].append(_exact_hold(part))
    return torch.cat(outs[0]), torch.cat(outs[1])


def _exact_attn(case, seed):
    """Query by query where there are few, head by head where there are many."""
    s = _step_inputs(case, seed)
    p, d = s["plan"], case["dim"]
    m, cache = _plain_cache(case, s)
    _plain_append(cache, m["table"], p["slots"], p["old"], p["new"], _starts(p["new"]), s["k"], s["v"])
    group = case["hq"] // case["hk"]
    out = torch.zeros(p["tokens"], case["hq"], d, device=DEV, dtype=F64)
    start = 0
    for i, slot in enumerate(p["slots"]):
        total = p["old"][i] + p["new"][i]
        t = torch.arange(total, device=DEV)
        where = m["table"][slot, t // PAGE].long()
        for j in range(case["hk"]):
            k, v = (cache["q"][where, z, t % PAGE, j].double() *
                    torch.exp2(cache["e"][where, z, j].double())[:, None] for z in range(2))
            size = max(1, 2 ** 26 // (group * total))
            for a in range(p["old"][i], total, size):
                at = torch.arange(a, min(a + size, total), device=DEV)
                rows = slice(start + a - p["old"][i], start + a - p["old"][i] + len(at))
                far = at[:, None] - t[None, :]
                hidden = far < 0
                if case["window"]:
                    hidden |= far >= case["window"]
                if s["prefix"] is not None:
                    hidden &= t[None, :] >= s["prefix"][i]
                for h in range(j * group, (j + 1) * group):
                    x = torch.mm(s["q"][rows, h].double(), k.t()) * d ** -0.5
                    if case["cap"]:
                        x = torch.tanh(x / case["cap"]) * case["cap"]
                    if s["slopes"] is not None:
                        x = x - float(s["slopes"][h]) * far.double()
                    x = x.masked_fill(hidden, float("-inf"))
                    out[rows, h] = torch.mm(torch.softmax(x, 1), v)
        start += p["new"][i]
    return out if s["gate"] is None else out * torch.sigmoid(s["gate"].double())


def exact(case, seed):
    if case["op"] == "map":
        return _exact_map(case, seed)
    if case["op"] == "rope":
        return _exact_rope(case, _rope_inputs(case, seed))
    if case["op"] == "append":
        return _exact_append(case, seed)
    return _exact_attn(case, seed)

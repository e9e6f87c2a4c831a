"""The operators of the decoder layer's sparse MLP half and their plain forms.

  route    scores of E experts -> the chosen experts' ids and weights per token
           (softmax or sigmoid, a bias for balance, groups, top-k, renormalised
           weights, shared experts appended)
  experts  the chosen experts' 4-bit gate / up / down products, weighted and
           summed per token
  norm     the norms after and before a block, with the block's gate, residual
           scale and residual add

Sizes are those of the Qwen3.5-35B-A3B decoder (hidden 2048, 256 experts of
inner size 512, 8 of them and one shared expert per token) and generic ones.
With `own` false, run() computes the operators with elementary torch
operations; with `own` true it calls the library.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
BF = torch.bfloat16
F32 = torch.float32
F64 = torch.float64


def _gdn():
    path = os.path.join(os.getcwd(), "qwen-mlx_amd")
    if path not in sys.path:
        sys.path.insert(1, path)
    import gdn_amd
    return gdn_amd


# ------------------------------------------------------------------- cases --

def _route(**kw):
    c = dict(op="route", tokens=64, experts=256, top_k=8, score="softmax", f32=False, bias=False,
             groups=1, top_groups=1, group_top=1, renorm=True, scale=1.0, shared=0,
             shared_gate=False, masked=0.0)
    c.update(kw)
    return c


def _experts(**kw):
    # entries of a token: top_k of `experts`, then the `shared` ones behind them
    c = dict(op="experts", tokens=64, hidden=2048, inner=512, experts=256, top_k=8, shared=1,
             pad=0.0)
    c.update(kw)
    return c


def _norm(**kw):
    c = dict(op="norm", rows=64, hidden=2048, f32=False, post=True, pre=True, gate="row",
             sigmoid=True, scale=1.0, offset=False)
    c.update(kw)
    return c


def listed():
    return [
        # a full decode batch of the model: one launch, latency
        _route(name="route_b64", shared=1, shared_gate=True),
        # a long prompt of the model
        _route(name="route_16384", tokens=16384, shared=1, shared_gate=True),
        # an odd prompt through a router of the sigmoid kind: f32 logits, a bias
        # for balance, half of the groups, some experts masked out
        _route(name="route_groups_4099", tokens=4099, score="sigmoid", f32=True, bias=True,
               groups=8, top_groups=4, group_top=2, scale=2.5, masked=0.05),
        # one user's token: nine experts' weights, launches and latency
        _experts(name="experts_b1", tokens=1),
        # a full decode batch: nearly every expert's weights once
        _experts(name="experts_b64", tokens=64),
        # a short prompt, a few rows an expert, ragged, with padded rows
        _experts(name="experts_317", tokens=317, pad=0.05),
        # a prompt over fewer, wider experts of an odd inner size, none shared
        _experts(name="experts_1500_e32", tokens=1500, hidden=1024, inner=1408, experts=32, top_k=4,
                 shared=0),
        # a long prompt of the model
        _experts(name="experts_16384", tokens=16384),
        # the seam behind a gated block of a decode batch
        _norm(name="norm_b64"),
        # the same seam of a long prompt
        _norm(name="norm_16384", rows=16384),
        # an odd prompt on an f32 residual stream, a learned scale per channel
        # instead of a gate, norm weights stored as offsets from one
        _norm(name="norm_f32_5003", rows=5003, hidden=4096, f32=True, gate="channel",
              sigmoid=False, scale=0.22, offset=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "experts", "experts", "norm"])
    if op == "route":
        e = rng.choice([8, 16, 60, 64, 128, 160, 256, 384, 512])
        k = rng.randint(1, min(e // 2, 12))
        groups = rng.choice([g for g in (1, 1, 2, 4, 8) if e % g == 0])
        # the groups that stay hold at least k experts
        top = rng.randint(-(-k * groups // e), groups)
        score = rng.choice(["softmax", "sigmoid"])
        shared = rng.choice([0, 1, 2])
        return _route(tokens=_log(rng, 1, 16384), experts=e, top_k=k, score=score,
                      f32=rng.random() < 0.5, bias=rng.random() < 0.5, groups=groups,
                      top_groups=top, group_top=rng.choice([1, 2]), renorm=rng.random() < 0.7,
                      scale=rng.choice([1.0, 2.5]), shared=shared,
                      shared_gate=shared > 0 and rng.random() < 0.5,
                      masked=rng.choice([0.0, 0.1]))
    if op == "experts":
        hidden = rng.choice([512, 1024, 2048, 2048, 2560, 4096])
        inner = rng.choice([128, 256, 384, 512, 512, 640, 768, 1024, 1408])
        most = 256 * 2048 * 512 // (hidden * inner)
        e = min(rng.choice([4, 8, 32, 60, 64, 128, 256]), most)
        k = rng.randint(1, min(e, 10))
        shared = rng.choice([0, 1])
        rows = 16384 * 9 * 2048 * 512 // (hidden * inner * (k + shared))
        return _experts(tokens=_log(rng, 1, min(16384, rows)), hidden=hidden, inner=inner,
                        experts=e, top_k=k, shared=shared, pad=rng.choice([0.0, 0.1]))
    hidden = rng.choice([64, 512, 1000, 1024, 2048, 2560, 4096, 5120, 8192])
    return _norm(rows=_log(rng, 1, min(16384, 16384 * 4096 // hidden)), hidden=hidden,
                 f32=rng.random() < 0.4, post=rng.random() < 0.6, pre=rng.random() < 0.8,
                 gate=rng.choice(["none", "row", "channel", "element"]),
                 sigmoid=rng.random() < 0.5, scale=rng.choice([1.0, 0.22]),
                 offset=rng.random() < 0.3)


# ------------------------------------------------------------------ inputs --

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _n(g, *shape, std=1.0, dtype=BF):
    return torch.empty(shape, device=DEV, dtype=F32).normal_(0, std, generator=g).to(dtype)


def _u(g, lo, hi, *shape):
    return torch.empty(shape, device=DEV, dtype=F32).uniform_(lo, hi, generator=g)


def _w4(g, experts, n, k, std):
    """4-bit weights of `experts` matrices [n, k]: words, scales, biases."""
    w = torch.randint(-2 ** 31, 2 ** 31, (experts, n, k // 8), device=DEV, dtype=torch.int32,
                      generator=g)
    s = (_u(g, 0.5, 1.5, experts, n, k // 64) * (std / 4.8)).to(BF)
    b = (-7.5 * s.float() * _u(g, 0.9, 1.1, experts, n, k // 64)).to(BF)
    return w, s, b


def _inputs(case, seed):
    g = _gen(seed)
    if case["op"] == "route":
        t, e = case["tokens"], case["experts"]
        cols = e + (1 if case["shared_gate"] else 0)
        # popular and rare experts, as a trained router has
        logits = _n(g, t, cols, std=1.5, dtype=F32) + _n(g, cols, std=0.5, dtype=F32)
        if case["masked"]:
            gone = torch.rand(t, e, device=DEV, generator=g) < case["masked"]
            logits[:, :e] = torch.where(gone, float("-inf"), logits[:, :e])
        return dict(logits=logits if case["f32"] else logits.to(BF),
                    bias=_n(g, e, std=0.1, dtype=F32) if case["bias"] else None)
    if case["op"] == "experts":
        t, h, i, e, k = (case[x] for x in ("tokens", "hidden", "inner", "experts", "top_k"))
        like = _n(g, t, e, dtype=F32) + _n(g, e, std=0.3, dtype=F32)
        top = torch.topk(like, k, dim=1)
        ids, w = top.indices.to(torch.int32), torch.softmax(top.values, dim=1)
        if case["shared"]:
            ids = torch.cat([ids, torch.full((t, 1), e, device=DEV, dtype=torch.int32)], 1)
            w = torch.cat([w, torch.sigmoid(_n(g, t, 1, dtype=F32))], 1)
        if case["pad"]:  # padded rows take no expert
            ids[torch.rand(t, device=DEV, generator=g) < case["pad"]] = -1
        parts = []
        for n in [e] + ([1] if case["shared"] else []):
            parts.append((_w4(g, n, i, h, h ** -0.5), _w4(g, n, i, h, h ** -0.5),
                          _w4(g, n, h, i, i ** -0.5)))
        return dict(x=_n(g, t, h), ids=ids.contiguous(), weights=w.contiguous(), parts=parts)
    n, h = case["rows"], case["hidden"]
    wt = lambda: ((0.0 if case["offset"] else 1.0) + 0.1 * _n(g, h, dtype=F32)).to(BF)  # noqa: E731
    i = dict(h=_n(g, n, h, std=2.0, dtype=F32 if case["f32"] else BF), d=_n(g, n, h),
             post=wt() if case["post"] else None, pre=wt() if case["pre"] else None, gate=None)
    if case["gate"] != "none":
        shape = {"row": (n, 1), "channel": (h,), "element": (n, h)}[case["gate"]]
        i["gate"] = _n(g, *shape)
    return i


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] == "route":
        shape = (case["tokens"], case["top_k"] + case["shared"])
        if own:
            s["ids"] = torch.empty(shape, device=DEV, dtype=torch.int32)
            s["weights"] = torch.empty(shape, device=DEV, dtype=F32)
    elif case["op"] == "experts":
        if own:
            s["moe"] = _gdn().MoE(case["hidden"], case["inner"], s.pop("parts"))
            s["workspace"] = s["moe"].workspace(*s["ids"].shape)
            s["out"] = torch.empty_like(s["x"])
    elif own:
        s["hn"] = torch.empty_like(s["d"]) if case["pre"] else None
        s["stream"] = torch.empty_like(s["h"])
    return s


# ------------------------------------------------------------- plain forms --

def _topk_low(score, k):
    """Indices of the k largest per row, ties to the lowest index."""
    return torch.sort(score, dim=1, descending=True, stable=True).indices[:, :k]


def _plain_route(s):
    c = s["case"]
    t, e, k = c["tokens"], c["experts"], c["top_k"]
    neg = float("-inf")
    top = torch.finfo(F32).max
    # 64 bits: the order of scores next to each other decides
    l = torch.nan_to_num(s["logits"].to(F64), nan=neg, posinf=top, neginf=neg)
    lr = l[:, :e]
    there = lr > neg
    sig = c["score"] == "sigmoid"
    if s["bias"] is None and c["group_top"] == 1:
        score = lr  # softmax and sigmoid keep the logits' order
    else:
        p = torch.sigmoid(lr) if sig else torch.nan_to_num(torch.softmax(lr, 1), nan=0.0)
        score = torch.where(there, p if s["bias"] is None else p + s["bias"].to(F64), neg)
    if c["groups"] > 1:
        grp = score.view(t, c["groups"], -1)
        best = torch.sort(grp, dim=2, descending=True).values[:, :, :c["group_top"]]
        some = best[:, :, 0] > neg
        gscore = torch.where(some, torch.where(best > neg, best, 0.0).sum(2), neg)
        stay = torch.zeros_like(some).scatter_(1, _topk_low(gscore, c["top_groups"]), True)
        score = torch.where((stay & some)[:, :, None], grp, neg).view(t, e)
    pick = _topk_low(score, k)
    ok = torch.gather(score, 1, pick) > neg
    lp = torch.gather(lr, 1, pick)
    if sig:
        # log sigmoid: small scores keep their ratio when renormalised
        ls = torch.clamp(lp, max=0.0) - torch.log1p(torch.exp(-lp.abs()))
        base = ls
    else:
        base = lp - torch.amax(lr, 1, keepdim=True)
        if not c["renorm"]:
            ex = torch.where(there, torch.exp(lr - torch.amax(lr, 1, keepdim=True)), 0.0)
            base = base - torch.log(ex.sum(1, keepdim=True))
    base = torch.where(ok, base, neg)
    if c["renorm"]:
        m = torch.amax(base, 1, keepdim=True)
        ex = torch.where(ok, torch.exp(base - m), 0.0)
        w = ex / ex.sum(1, keepdim=True)
    else:
        w = torch.exp(base)
    w = torch.where(ok, w * c["scale"], 0.0)
    ids = torch.where(ok, pick, -1)
    if c["shared"]:
        gate = torch.sigmoid(l[:, e:e + 1]) if c["shared_gate"] else torch.ones(t, 1, device=DEV,
                                                                               dtype=F64)
        w = torch.cat([w, gate.expand(t, c["shared"])], 1)
        more = e + torch.arange(c["shared"], device=DEV)
        ids = torch.cat([ids, more.expand(t, c["shared"])], 1)
    return ids.to(torch.int32), w.to(F32)


def _dequant(w, s, b, dtype):
    """[n, k/8] words, [n, k/64] scales and biases -> [n, k]: s * q + b."""
    shift = torch.arange(0, 32, 4, device=DEV, dtype=torch.int32)
    q = (w[:, :, None] >> shift) & 15
    q = q.view(w.shape[0], -1, 64).to(dtype)
    return (q * s.to(dtype)[:, :, None] + b.to(dtype)[:, :, None]).view(w.shape[0], -1)


def _moe(s, dtype):
    x, ids, weights = s["x"].to(dtype), s["ids"], s["weights"].to(dtype)
    out = torch.zeros(x.shape, device=DEV, dtype=dtype)
    flat = ids.view(-1)
    order = torch.argsort(flat, stable=True)
    total = sum(p[0][0].shape[0] for p in s["parts"])
    inside = (flat >= 0) & (flat < total)
    count = torch.bincount(flat[inside], minlength=total).tolist()
    order = order[int((flat < 0).sum()):]
    tok = order // ids.shape[1]
    wt = weights.view(-1)[order]
    at, e = 0, 0
    for gate, up, down in s["parts"]:
        for i in range(gate[0].shape[0]):
            n = count[e]
            e += 1
            if n == 0:
                continue
            rows = tok[at:at + n]
            xr = x[rows]
            a = xr @ _dequant(*(v[i] for v in gate), dtype).t()
            u = xr @ _dequant(*(v[i] for v in up), dtype).t()
            y = (a / (1 + torch.exp(-a)) * u) @ _dequant(*(v[i] for v in down), dtype).t()
            out.index_add_(0, rows, y * wt[at:at + n, None])
            at += n
    return out


def _block_norm(s, dtype):
    c = s["case"]
    one = 1.0 if c["offset"] else 0.0

    def rms(v, w):
        return v / torch.sqrt(v.square().mean(1, keepdim=True) + 1e-6) * (w.to(dtype) + one)

    d = s["d"].to(dtype)
    if s["post"] is not None:
        d = rms(d, s["post"])
    if s["gate"] is not None:
        gate = s["gate"].to(dtype)
        d = d * (1 / (1 + torch.exp(-gate)) if c["sigmoid"] else gate)
    h = s["h"].to(dtype) + c["scale"] * d
    return h, None if s["pre"] is None else rms(h, s["pre"])


# --------------------------------------------------------------------- run --

def run(state):
    s = state
    c = s["case"]
    if c["op"] == "route":
        if not own:
            return _plain_route(s)
        _gdn().moe_route(s["logits"], s["ids"], s["weights"], c["experts"], c["top_k"],
                         score=c["score"], bias=s["bias"], num_groups=c["groups"],
                         top_groups=c["top_groups"], group_top=c["group_top"], renorm=c["renorm"],
                         scale=c["scale"], num_shared=c["shared"], shared_gate=c["shared_gate"])
        return s["ids"], s["weights"]
    if c["op"] == "experts":
        if not own:
            return _moe(s, F32).to(BF)
        s["moe"].forward(s["x"], s["ids"], s["weights"], s["out"], s["workspace"])
        return s["out"]
    if not own:
        h, hn = _block_norm(s, F32)
        h = h.to(s["h"].dtype)
        return (h,) if hn is None else (h, hn.to(BF))
    _gdn().block_norm(s["h"], s["d"], h_out=s["stream"], hn=s["hn"], pre_w=s["pre"],
                      post_w=s["post"], gate=s["gate"], gate_sigmoid=c["sigmoid"], scale=c["scale"],
                      unit_offset=c["offset"])
    return (s["stream"],) if s["hn"] is None else (s["stream"], s["hn"])


# ------------------------------------------------------------ work, exact --

def work(case):
    c = case
    if c["op"] == "route":
        t = c["tokens"]
        cols = c["experts"] + (1 if c["shared_gate"] else 0)
        return {"bytes": t * cols * (4 if c["f32"] else 2) + t * (c["top_k"] + c["shared"]) * 8
                + (4 * c["experts"] if c["bias"] else 0),
                # an exponential and the comparisons of the choice per score
                "flops": t * c["experts"] * 4}
    if c["op"] == "experts":
        t, h, i = c["tokens"], c["hidden"], c["inner"]
        live = t * (1 - c["pad"])
        # experts that some token takes, each taken with the same likelihood
        used = c["experts"] * (1 - (1 - c["top_k"] / c["experts"]) ** live) + c["shared"]
        k = c["top_k"] + c["shared"]
        return {"bytes": int(used * 3 * h * i * (0.5 + 4 / 64)) + 2 * 2 * t * h + 8 * t * k,
                "flops": int(live * k * 6 * h * i)}
    n, h = c["rows"], c["hidden"]
    gate = {"none": 0, "row": 2 * n, "channel": 2 * h, "element": 2 * n * h}[c["gate"]]
    b = 2 * n * h * (4 if c["f32"] else 2) + 2 * n * h + gate
    b += (2 * n * h + 2 * h if c["pre"] else 0) + (2 * h if c["post"] else 0)
    return {"bytes": b, "flops": n * h * 8}


def _exact_route(case, i):
    """The definition, one token after the other, on the host."""
    if case["tokens"] * case["experts"] > 2 ** 21:
        return None
    logits = i["logits"].double().cpu().tolist()
    bias = i["bias"].double().cpu().tolist() if i["bias"] is not None else None
    e, k = case["experts"], case["top_k"]
    size = e // case["groups"]
    by_logit = bias is None and case["group_top"] == 1
    all_ids, all_w = [], []
    for row in logits:
        row = [min(v, torch.finfo(F32).max) if v == v else -math.inf for v in row]
        sig = [1 / (1 + math.exp(-v)) if v >= 0 else math.exp(v) / (1 + math.exp(v)) for v in row]
        live = [x for x in range(e) if row[x] > -math.inf]
        prob = [0.0] * e
        if live:
            m = max(row[x] for x in live)
            tot = math.fsum(math.exp(row[x] - m) for x in live)
            for x in live:
                prob[x] = math.exp(row[x] - m) / tot
        base = sig if case["score"] == "sigmoid" else prob
        key = {x: row[x] if by_logit else base[x] + (bias[x] if bias else 0.0) for x in live}
        if case["groups"] > 1:
            ranks = []
            for gi in range(case["groups"]):
                best = sorted((key[x] for x in range(gi * size, gi * size + size) if x in key),
                              reverse=True)[:case["group_top"]]
                if best:
                    ranks.append((-math.fsum(best), gi))
            stay = {gi for _, gi in sorted(ranks)[:case["top_groups"]]}
            key = {x: v for x, v in key.items() if x // size in stay}
        pick = sorted(key, key=lambda x: (-key[x], x))[:k]
        if case["renorm"] and pick:
            if case["score"] == "sigmoid":
                logs = [min(row[x], 0.0) - math.log1p(math.exp(-abs(row[x]))) for x in pick]
            else:
                logs = [row[x] for x in pick]
            m = max(logs)
            ex = [math.exp(v - m) for v in logs]
            w = [case["scale"] * v / math.fsum(ex) for v in ex]
        else:
            w = [case["scale"] * base[x] for x in pick]
        ids = pick + [-1] * (k - len(pick))
        w = w + [0.0] * (k - len(w))
        gate = sig[e] if case["shared_gate"] else 1.0
        all_ids.append(ids + [e + x for x in range(case["shared"])])
        all_w.append(w + [gate] * case["shared"])
    return (torch.tensor(all_ids, dtype=torch.int32, device=DEV),
            torch.tensor(all_w, dtype=F64, device=DEV))


def _exact_experts(i):
    """Per entry column j the tokens' products, expert by expert, in 64 bits."""
    x = i["x"].double()
    out = torch.zeros_like(x)

    def full(w, s, b):
        cols = torch.arange(w.shape[-1] * 8, device=DEV)
        q = (w[:, cols // 8].long() >> (4 * (cols % 8))) % 16
        return q.double() * s.double()[:, cols // 64] + b.double()[:, cols // 64]

    first = 0
    for gate, up, down in i["parts"]:
        for n in range(gate[0].shape[0]):
            share = torch.where(i["ids"] == first + n, i["weights"].double(), 0.0).sum(1)
            rows = (i["ids"] == first + n).any(1).nonzero()[:, 0]
            if rows.numel():
                xr = x[rows]
                a = torch.matmul(full(*(v[n] for v in gate)), xr.t())
                a = a * torch.sigmoid(a) * torch.matmul(full(*(v[n] for v in up)), xr.t())
                y = torch.matmul(full(*(v[n] for v in down)), a).t()
                out[rows] += share[rows, None] * y
        first += gate[0].shape[0]
    return out


def _exact_norm(case, i):
    def norm(v, w):
        r = torch.rsqrt((v * v).sum(-1) / v.shape[-1] + 1e-6)
        w = w.double() + 1 if case["offset"] else w.double()
        return torch.einsum("nh,n,h->nh", v, r, w)

    d = i["d"].double()
    if i["post"] is not None:
        d = norm(d, i["post"])
    gate = 1.0
    if i["gate"] is not None:
        gate = torch.sigmoid(i["gate"].double()) if case["sigmoid"] else i["gate"].double()
    h = torch.add(i["h"].double(), d * gate, alpha=case["scale"])
    return (h,) if i["pre"] is None else (h, norm(h, i["pre"]))


def exact(case, seed):
    i = _inputs(case, seed)
    if case["op"] == "route":
        return _exact_route(case, i)
    if case["op"] == "experts":
        return _exact_experts(i)
    return _exact_norm(case, i)

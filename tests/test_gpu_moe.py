"""Expert routing, the experts' 4-bit products and the block norm against plain
64-bit forms, at the sizes, masks and strides where they can go wrong.

Tolerances. A rounding is off by at most half a step, 2^-8 of the value in bf16
and 2^-24 in f32; each bound below counts the roundings on the way to a value,
with the magnitudes that enter them taken from the 64-bit form.
"""
import math

import pytest
import torch

import gdn_amd

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
HALF_BF, HALF_F32 = 2.0 ** -8, 2.0 ** -24
INF = math.inf


# ------------------------------------------------------------------ router --

def ref_route(logits, E, k, score="softmax", bias=None, groups=1, top_groups=1, group_top=1,
              renorm=True, scale=1.0, shared=0, shared_gate=False):
    """One token after the other, 64 bits."""
    ids, weights = [], []
    for row in logits.double().tolist():
        row = [-INF if v != v else min(v, torch.finfo(F32).max) for v in row]
        live = [e for e in range(E) if row[e] > -INF]

        def sig(v):
            return 1 / (1 + math.exp(-v)) if v >= 0 else math.exp(v) / (1 + math.exp(v))

        p = {}
        if score == "softmax" and live:
            m = max(row[e] for e in live)
            tot = math.fsum(math.exp(row[e] - m) for e in live)
            p = {e: math.exp(row[e] - m) / tot for e in live}
        elif live:
            p = {e: sig(row[e]) for e in live}
        if bias is None and (group_top == 1 or groups == 1):
            key = {e: row[e] for e in live}
        else:
            b = [0.0] * E if bias is None else bias.double().tolist()
            key = {e: p[e] + b[e] for e in live}
        key = {e: v for e, v in key.items() if v > -INF}  # a NaN or -inf bias takes one out
        if groups > 1:
            size = E // groups
            best = []
            for g in range(groups):
                s = sorted((v for e, v in key.items() if e // size == g), reverse=True)
                if s:
                    best.append((-sum(s[:group_top]), g))
            stay = {g for _, g in sorted(best)[:top_groups]}
            key = {e: v for e, v in key.items() if e // size in stay}
        pick = sorted(key, key=lambda e: (-key[e], e))[:k]
        if renorm and pick:
            ls = [row[e] if score == "softmax" else min(row[e], 0.0) - math.log1p(math.exp(-abs(row[e])))
                  for e in pick]
            ex = [math.exp(v - max(ls)) for v in ls]
            w = [scale * v / math.fsum(ex) for v in ex]
        else:
            w = [scale * p[e] for e in pick]
        gate = sig(row[E]) if shared_gate else 1.0
        ids.append(pick + [-1] * (k - len(pick)) + [E + s for s in range(shared)])
        weights.append(w + [0.0] * (k - len(w)) + [gate] * shared)
    return torch.tensor(ids, dtype=torch.int32), torch.tensor(weights, dtype=F64)


def run_route(logits, E, k, **kw):
    kw = dict(kw)
    for a, b in (("groups", "num_groups"), ("shared", "num_shared")):
        if a in kw:
            kw[b] = kw.pop(a)
    n = k + kw.get("num_shared", 0)
    ids = torch.full((logits.shape[0], n), -7, device=DEV, dtype=torch.int32)
    w = torch.full((logits.shape[0], n), -7.0, device=DEV)
    if kw.get("bias") is not None:
        kw["bias"] = kw["bias"].to(DEV)
    gdn_amd.moe_route(logits, ids, w, E, k, **kw)
    torch.cuda.synchronize()
    return ids.cpu(), w.double().cpu()


def check_route(logits, E, k, dev=None, **kw):
    ids, w = run_route(logits.to(DEV) if dev is None else dev, E, k, **kw)
    rids, rw = ref_route(logits, E, k, **kw)
    assert torch.equal(ids, rids)
    # A weight is an exponential (its f32 argument off by a half step of at most
    # 2^5 = 2^-19 for logits to 30 apart, 2 ulp = 4 half steps of its own) over a
    # sum of at most 1024 of them (each as far off, plus 16 steps of a tree and
    # 16 in a lane), a division and the scale: below 2^-17.
    assert ((w - rw).abs() <= 2.0 ** -17 * rw.abs() + 1e-38).all()


def _logits(seed, T, cols, dtype=BF, std=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, cols, generator=g) * std).to(dtype)


@pytest.mark.parametrize("T,E,k,kw", [
    (1, 1, 1, {}),
    (1, 256, 8, dict(shared=1, shared_gate=True)),
    (67, 256, 8, dict(renorm=False)),
    (5, 8, 2, dict(score="sigmoid")),
    (130, 60, 4, dict(score="sigmoid", renorm=False, shared=2)),
    (33, 160, 6, dict(groups=8, top_groups=3, scale=16.0, renorm=False)),
    (33, 256, 8, dict(groups=8, top_groups=4, group_top=2, score="sigmoid", scale=2.5)),
    (9, 384, 32, dict(groups=64, top_groups=33)),
    (7, 1024, 32, dict(groups=2, top_groups=1, group_top=2, shared=8, shared_gate=True)),
    (3, 65, 5, dict(groups=13, top_groups=2, group_top=2)),
    (4, 128, 1, dict(groups=64, top_groups=1, group_top=1)),
])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("biased", [False, True])
def test_route(gpu, T, E, k, kw, dtype, biased):
    kw = dict(kw)
    if biased:
        kw["bias"] = torch.randn(E, generator=torch.Generator().manual_seed(E)) * 0.1
    check_route(_logits(T + E, T, E + 1, dtype), E, k, **kw)


def test_route_ties_go_to_the_lowest_index(gpu):
    for E, kw in ((256, {}), (60, dict(score="sigmoid")),
                  (256, dict(groups=8, top_groups=2, group_top=2)),
                  (256, dict(score="sigmoid", bias=torch.zeros(256)))):
        same = torch.zeros(3, E, dtype=BF)
        ids, w = run_route(same.to(DEV), E, 6, **kw)
        assert ids.tolist() == [list(range(6))] * 3
        coarse = torch.randint(0, 3, (17, E), generator=torch.Generator().manual_seed(1)).to(BF)
        check_route(coarse, E, 6, **kw)


def test_route_tells_scores_apart_that_f32_does_not(gpu):
    """Sigmoids plus a bias that differ by 1e-12: the order is that of the scores."""
    E = 64
    logits = torch.full((1, E), 20.0)
    logits[0, 5], logits[0, 40], logits[0, 9] = 21.0, 21.5, 20.5
    check_route(logits, E, 4, score="sigmoid", bias=torch.ones(E))
    ids, _ = run_route(logits.to(DEV), E, 3, score="sigmoid", bias=torch.ones(E))
    assert ids.tolist() == [[40, 5, 9]]


@pytest.mark.parametrize("kw", [dict(), dict(renorm=False), dict(score="sigmoid"),
                                dict(score="sigmoid", renorm=False),
                                dict(bias=torch.linspace(-1, 1, 32)),
                                dict(groups=4, top_groups=2, group_top=2),
                                dict(score="sigmoid", groups=4, top_groups=2, shared=1,
                                     shared_gate=True)])
def test_route_masks_infinities_and_nan(gpu, kw):
    E, k = 32, 6
    low = torch.finfo(F32).min
    l = _logits(3, 12, E + 1, F32)
    l[0] = -INF                       # nothing left
    l[1] = math.nan
    l[2, :E] = -INF
    l[2, 7] = 0.5                     # fewer than k
    l[3, :E - 3] = -INF
    l[4, :] = low                     # the type's lowest value is a value
    l[5, 3] = INF
    l[6, 3] = l[6, 20] = INF
    l[7, 1::2] = math.nan
    l[8, :E] = low
    l[8, 9] = 1.0
    l[9, 16:] = -INF                  # whole groups gone
    l[10, :24] = -INF
    l[11, ::8] = INF
    l[:, E] = l[:, E].clamp(-5, 5)
    l[0, E] = -INF
    l[1, E] = math.nan
    check_route(l, E, k, **kw)


@pytest.mark.parametrize("E,k", [(1, 1), (3, 3), (16, 7), (63, 4), (64, 15), (65, 15), (100, 15),
                                 (128, 8), (200, 3), (255, 8), (256, 15), (257, 8), (400, 11),
                                 (512, 15), (512, 16), (513, 4), (60, 17)])
@pytest.mark.parametrize("kw", [dict(), dict(renorm=False, scale=2.5), dict(score="sigmoid"),
                                dict(score="sigmoid", renorm=False)])
def test_route_bf16_rows(gpu, E, k, kw):
    """bf16 logits in their own order: every size of a lane's share, rows with few or no
    numbers, both zeros, subnormals, the type's lowest value, infinities and NaN."""
    T = 37
    g = torch.Generator().manual_seed(E + k)
    l = torch.randn(T, E + 1, generator=g).mul(2).to(BF)
    fin = torch.finfo(BF)
    l[1, :E] = -INF
    l[2, :E] = math.nan
    l[3, :E] = torch.where(torch.rand(E, generator=g) < 0.5, 0.0, -0.0).to(BF)
    l[4, :E] = torch.randint(-3, 4, (E,), generator=g).to(torch.int16).abs().view(BF)  # subnormals
    l[5, :E] = fin.min
    l[6, :E] = torch.where(torch.rand(E, generator=g) < 0.3, -INF, fin.min).to(BF)
    l[7, :E:2] = math.nan
    l[8, :E:3] = -INF
    l[9, E - 1] = INF
    l[10, :E] = INF
    l[11, : E - 1] = -INF
    l[12, 1:E] = math.nan
    l[13, :E] = torch.randint(-2, 3, (E,), generator=g).to(BF)
    shared = dict(shared=1, shared_gate=True) if k < 16 else {}
    check_route(l, E, k, **kw, **shared)


def test_route_bias_takes_experts_out(gpu):
    b = torch.zeros(16)
    b[3], b[5] = -INF, math.nan
    check_route(_logits(8, 9, 16), 16, 15, bias=b)


def test_route_column_slices_and_no_rows(gpu):
    wide = _logits(4, 21, 300, BF)
    dev = wide.to(DEV)
    for lo in (0, 1, 17):
        check_route(wide[:, lo:lo + 257], 256, 8, dev=dev[:, lo:lo + 257], shared=1,
                    shared_gate=True)
    run_route(dev[:0, :256], 256, 8)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_route_of_more_rows_than_a_launch(gpu, dtype):
    """2^22 rows go in a launch; the rows on both sides of the cut and the last ones."""
    T, E, k = (1 << 22) + 5, 8, 2
    g = torch.Generator(DEV).manual_seed(6)
    l = torch.randn(T, E + 1, generator=g, device=DEV).to(dtype)
    ids = torch.full((T, k + 1), -7, device=DEV, dtype=torch.int32)
    w = torch.full((T, k + 1), -7.0, device=DEV)
    gdn_amd.moe_route(l, ids, w, E, k, num_shared=1, shared_gate=True)
    torch.cuda.synchronize()
    for lo, hi in ((0, 4), ((1 << 22) - 4, T)):
        rids, rw = ref_route(l[lo:hi].cpu(), E, k, shared=1, shared_gate=True)
        assert torch.equal(ids[lo:hi].cpu(), rids)
        assert ((w[lo:hi].cpu().double() - rw).abs() <= 2.0 ** -17 * rw).all()
    assert int(ids.min()) == 0 and int(ids.max()) == E


# ----------------------------------------------------------------- experts --

def w4(g, e, n, k):
    w = torch.randint(-2 ** 31, 2 ** 31, (e, n, k // 8), dtype=torch.int32, generator=g)
    s = ((torch.rand(e, n, k // 64, generator=g) + 0.5) * k ** -0.5 / 4.8).to(BF)
    b = (-7.5 * s.float() * (0.9 + 0.2 * torch.rand(e, n, k // 64, generator=g))).to(BF)
    return w, s, b


def full(w, s, b):
    q = (w[..., None] >> torch.arange(0, 32, 4, dtype=torch.int32)) & 15
    q = q.reshape(*w.shape[:-1], -1, 64).double()
    return (q * s.double()[..., None] + b.double()[..., None]).flatten(-2)


class Experts:
    def __init__(self, hidden, inner, parts, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.hidden, self.inner = hidden, inner
        self.parts = [(w4(g, n, inner, hidden), w4(g, n, inner, hidden), w4(g, n, hidden, inner))
                      for n in parts]
        dev = [tuple(tuple(t.to(DEV) for t in m) for m in p) for p in self.parts]
        self.moe = gdn_amd.MoE(hidden, inner, dev)
        self.E = sum(parts)

    def ref(self, x, ids, weights):
        """(out, bound) in 64 bits: the result and how far f32 sums, the bf16
        rounding of h, the rows' of long prompts to 11 bits and the last rounding may
        move it. A row's f16 has its power of two within 2^3 of 2^15 times the bound
        max |h| * max sum |w|: half a step of its smallest numbers is 2^-37 of that."""
        x = x.double()
        out, tol = torch.zeros_like(x), torch.zeros_like(x)
        e = 0

        def err(m, i, v):
            # s (128 X + sum x q) + (b - 128 s) X in f32: every term of a group
            # enters 64 / 16 + 2 adds in the group and one for each group
            s, b = m[1][i].double().abs(), m[2][i].double().abs()
            mag = (271 * s + b).repeat_interleave(64, 1)
            return (v.shape[1] // 64 + 8) * HALF_F32 * (v.abs() @ mag.t())

        for part in self.parts:
            mats = [[full(*(t[i] for t in m)) for m in part] for i in range(part[0][0].shape[0])]
            for i, (wg, wu, wd) in enumerate(mats):
                w = torch.where(ids == e, weights.double(), 0.0)
                rows = (ids == e).any(1)
                e += 1
                if not rows.any():
                    continue
                xr = x[rows]
                a, u = xr @ wg.t(), xr @ wu.t()
                h = a * torch.sigmoid(a) * u
                ea, eu = err(part[0], i, xr), err(part[1], i, xr)
                # |silu'| <= 1.1, |silu(a)| <= |a|; 8 half steps for the exponential
                eh = 1.1 * ea * u.abs() + a.abs() * eu + ea * eu + (HALF_BF + 8 * HALF_F32) * h.abs()
                y = h @ wd.t()
                ey = eh @ wd.abs().t() + err(part[2], i, h) + 2.0 ** -11 * y.abs()
                ey += 2.0 ** -37 * (h.abs() + eh).amax(1, True) * wd.abs().sum(1).max()
                out[rows] += w[rows].sum(1, keepdim=True) * y
                tol[rows] += w[rows].abs().sum(1, keepdim=True) * ey
        return out, tol + HALF_BF * (out.abs() + tol)

    def run(self, x, ids, weights, stream=None):
        T, k = ids.shape
        wide = torch.full((T, self.hidden + 12), 3.0, device=DEV, dtype=BF)
        ws = self.moe.workspace(T, k)
        ws.fill_(255)
        self.moe.forward(x.to(DEV), ids.to(DEV), weights.to(DEV), wide[:, :self.hidden], ws,
                         stream=stream)
        torch.cuda.synchronize()
        assert (wide[:, self.hidden:] == 3.0).all()
        return wide[:, :self.hidden].cpu()

    def check(self, x, ids, weights):
        out = self.run(x, ids, weights)
        ref, tol = self.ref(x, ids, weights)
        d = (out.double() - ref).abs()
        assert (d <= tol).all(), float((d / tol.clamp_min(1e-30)).max())
        return out


def draw_ids(seed, T, E, k, distinct=True):
    g = torch.Generator().manual_seed(seed)
    x_ids = (torch.rand(T, E, generator=g).argsort(1)[:, :k] if distinct
             else torch.randint(0, E, (T, k), generator=g))
    return x_ids.to(torch.int32), torch.rand(T, k, generator=g) + 0.05


def draw_x(seed, T, hidden):
    return torch.randn(T, hidden, generator=torch.Generator().manual_seed(seed)).to(BF)


@pytest.mark.parametrize("hidden,inner,parts,T,k", [
    (128, 128, [1], 1, 1),
    (2048, 512, [8, 1], 1, 3),
    (512, 128, [5], 3, 2),
    (256, 384, [7, 1], 17, 3),
    (640, 256, [3], 40, 2),
    (1024, 640, [4], 64, 2),
    (128, 1408, [3], 33, 3),
    (384, 128, [16, 2], 100, 5),
    (256, 128, [40], 257, 4),
    (512, 256, [2], 700, 2),
    (256, 128, [64], 1000, 8),
    (128, 128, [4], 3001, 3),
    (4096, 128, [2], 5, 1),
    (128, 2048, [2], 5, 2),
    (2176, 256, [3], 130, 2),
    (128, 128, [300], 3000, 4),   # more than 8192 entries
    (128, 128, [1030], 2100, 4),  # and more experts than threads that place them
    (2048, 128, [2], 1700, 2),    # tiles of 64 rows, down's input in LDS
    (1792, 384, [3, 1], 2100, 3),
    (1152, 640, [2, 1], 1700, 3), # and in stages, half a block of columns over
    (128, 128, [24], 3, 20),      # more columns than waves of a work-group
    (256, 128, [50], 10, 40),
    (1408, 1152, [40], 20, 3),    # stages in two parts of unequal length
    (128, 128, [1500], 6, 64),
])
def test_experts(gpu, hidden, inner, parts, T, k):
    ex = Experts(hidden, inner, parts, seed=hidden + inner)
    ids, w = draw_ids(T, T, ex.E, k)
    ex.check(draw_x(T, T, hidden), ids, w)


@pytest.mark.parametrize("T,hidden,inner", [(1, 256, 256), (4, 256, 256), (12, 256, 256),
                                            (19, 256, 256), (300, 256, 256), (1100, 256, 256),
                                            (2500, 256, 256), (900, 2048, 128), (800, 1536, 640)])
def test_experts_uneven_absent_and_repeated_ids(gpu, T, hidden, inner):
    """All rows on one expert, experts without rows, ids outside the layer, tokens
    without any, an expert twice in a token, weights that are zero or negative."""
    ex = Experts(hidden, inner, [6, 1], seed=5)
    x = draw_x(1, T, hidden)
    _, w = draw_ids(2, T, 7, 4)
    one = torch.full((T, 4), 3, dtype=torch.int32)
    one[:, 1:] = -1
    ex.check(x, one, w)
    g = torch.Generator().manual_seed(T)
    ids = torch.randint(-2, 9, (T, 4), generator=g, dtype=torch.int32)
    ids[0] = torch.tensor([-1, 7, 1 << 30, -(1 << 31)], dtype=torch.int32)
    w[:, 1] *= -1
    w[::2, 2] = 0
    out = ex.check(x, ids, w)
    assert (out[0] == 0).all()
    same = torch.full((T, 4), 6, dtype=torch.int32)
    ex.check(x, same, w)
    assert (ex.run(x, torch.full((T, 4), -1, dtype=torch.int32), w) == 0).all()


@pytest.mark.parametrize("T,hidden,inner", [(2, 256, 256), (20, 256, 256), (300, 256, 256),
                                            (1700, 2048, 128), (1750, 2048, 384)])
def test_experts_of_all_magnitudes(gpu, T, hidden, inner):
    """Tokens from 2^-30 to 2^30 (h to 2^60 either way), weights of 2^-40 to 2^40 in one
    token, zeros among both, an expert whose down has no finite columns but one."""
    ex = Experts(hidden, inner, [2], seed=11)
    g = torch.Generator().manual_seed(T)
    ids, w = draw_ids(T, T, 2, 2)
    x = draw_x(T, T, hidden).double() * 2.0 ** torch.randint(-30, 31, (T, 1), generator=g)
    x[:: 7] = 0
    w = (w * 2.0 ** torch.randint(-40, 41, (T, 2), generator=g)).float()
    w[::5, 0] = 0
    ex.check(x.to(BF), ids, w)
    wide = Experts(hidden, inner, [2], seed=12)
    (_, _, (dw, ds, db)), = wide.parts
    db[1, 1:] = INF
    dev = [tuple(tuple(t.to(DEV) for t in m) for m in p) for p in wide.parts]
    wide.moe = gdn_amd.MoE(hidden, inner, dev)
    x = draw_x(T + 1, T, hidden)
    only = torch.stack([torch.full((T,), 1), torch.full((T,), -1)], 1).to(torch.int32)
    only[:, 1] = torch.where(torch.arange(T) % 2 == 0, 0, -1)
    w = torch.ones(T, 2)
    out = wide.run(x, only, w)
    db[1, 1:] = 0
    ref, tol = wide.ref(x, only, w)
    assert ((out.double() - ref).abs() <= tol)[:, 0].all()
    assert not out[:, 1:].isfinite().any()


def test_experts_rows_keep_to_themselves(gpu):
    """NaN and infinities in one token reach no other; a token's result does not
    depend on where it stands in the batch."""
    ex = Experts(256, 128, [4], seed=2)
    x, (ids, w) = draw_x(3, 50, 256), draw_ids(4, 50, 4, 2)
    clean = ex.run(x, ids, w)
    bad = x.clone()
    bad[7, 3], bad[20, 100], bad[33] = math.nan, INF, -INF
    out = ex.run(bad, ids, w)
    keep = torch.ones(50, dtype=torch.bool)
    keep[[7, 20, 33]] = False
    assert torch.equal(out[keep].view(torch.int16), clean[keep].view(torch.int16))
    assert out[7].isnan().all() and not out[33].isfinite().any()
    back = ex.run(x.flip(0), ids.flip(0), w.flip(0)).flip(0)
    assert torch.equal(back.view(torch.int16), clean.view(torch.int16))


@pytest.mark.parametrize("T,hidden,inner,E", [
    (5, 256, 256, 4),         # very few entries
    (60, 1024, 1152, 40),     # tiles of 16 rows by the weights' stream
    (100, 256, 256, 12),      # tiles of 16
    (200, 256, 128, 12),      # and of 32
    (1700, 2048, 384, 4),     # of 64, down's input in LDS
    (1700, 1792, 640, 4),     # and in stages
    (4500, 256, 128, 40),     # sorted in two launches
    (7000, 1024, 256, 4),
])
def test_experts_rows_keep_to_themselves_in_every_kernel(gpu, T, hidden, inner, E):
    ex = Experts(hidden, inner, [E], seed=T)
    x, (ids, w) = draw_x(3, T, hidden), draw_ids(4, T, E, 2)
    clean = ex.run(x, ids, w)
    assert clean.isfinite().all()
    g = torch.Generator().manual_seed(T)
    at = torch.randperm(T, generator=g)[:max(1, T // 20)]
    bad = x.clone()
    bad[at, torch.randint(0, hidden, (len(at),), generator=g)] = math.nan
    bad[at[::2]] = INF
    out = ex.run(bad, ids, w)
    keep = torch.ones(T, dtype=torch.bool)
    keep[at] = False
    assert torch.equal(out[keep].view(torch.int16), clean[keep].view(torch.int16))
    assert not out[at].isfinite().any()
    for order in (torch.arange(T).flip(0), torch.randperm(T, generator=g)):
        there = ex.run(x[order], ids[order], w[order])
        assert torch.equal(there.view(torch.int16), clean[order].view(torch.int16))


@pytest.mark.parametrize("T", [2, 60, 900])
def test_experts_strided_rows_other_stream_and_repeat(gpu, T):
    ex = Experts(256, 128, [6], seed=9)
    x, (ids, w) = draw_x(5, T, 256), draw_ids(6, T, 6, 3)
    want = ex.check(x, ids, w)
    wide = torch.zeros(T, 400, dtype=BF)
    wide[:, 64:320] = x
    dev = wide.to(DEV)
    out = torch.empty(T, 256, device=DEV, dtype=BF)
    ws = ex.moe.workspace(T, 3)
    di, dw = ids.to(DEV), w.to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for s in (None, side, side):
        out.fill_(9.0)
        side.wait_stream(torch.cuda.current_stream())
        ex.moe.forward(dev[:, 64:320], di, dw, out, ws, stream=s)
        torch.cuda.synchronize()
        assert torch.equal(out.cpu().view(torch.int16), want.view(torch.int16))


def test_experts_no_rows_and_workspace_of_a_larger_call(gpu):
    ex = Experts(128, 128, [3])
    big = ex.moe.workspace(500, 4)
    e = torch.empty(0, 128, device=DEV, dtype=BF)
    ex.moe.forward(e, torch.empty(0, 2, device=DEV, dtype=torch.int32),
                   torch.empty(0, 2, device=DEV), e, big)
    x, (ids, w) = draw_x(5, 9, 128), draw_ids(6, 9, 3, 2)
    out = torch.empty(9, 128, device=DEV, dtype=BF)
    ex.moe.forward(x.to(DEV), ids.to(DEV), w.to(DEV), out, big)
    assert torch.equal(out.cpu().view(torch.int16), ex.run(x, ids, w).view(torch.int16))
    last = 0
    for T in (1, 2, 7, 64, 65, 100, 255, 1000, 1001, 5000, 40000, 400000):
        n = [ex.moe.workspace_bytes(T, k) for k in (1, 2, 3, 8, 64)]
        assert n == sorted(n) and n[0] >= last
        last = n[0]


def test_experts_rows_far_apart(gpu):
    """Rows of x whose byte offsets pass 32 bits: the call goes in pieces."""
    ex = Experts(128, 128, [3], seed=11)
    T, stride = 2500, 1 << 20
    x, (ids, w) = draw_x(1, T, 128), draw_ids(2, T, 3, 2)
    far = torch.empty(T * stride, device=DEV, dtype=BF).view(T, stride)[:, :128]
    far.copy_(x)
    out = torch.empty(T, 128, device=DEV, dtype=BF)
    ex.moe.forward(far, ids.to(DEV), w.to(DEV), out, ex.moe.workspace(T, 2))
    ref, tol = ex.ref(x, ids, w)
    assert ((out.cpu().double() - ref).abs() <= tol).all()


def test_experts_two_streams_at_once(gpu):
    """Calls with work-spaces of their own may overlap."""
    ex = Experts(512, 256, [9], seed=6)
    calls = []
    for T in (700, 40, 5):
        x, (ids, w) = draw_x(T, T, 512), draw_ids(T + 1, T, 9, 2)
        calls.append((x.to(DEV), ids.to(DEV), w.to(DEV), torch.empty(T, 512, device=DEV, dtype=BF),
                      ex.moe.workspace(T, 2), torch.cuda.Stream(), ex.run(x, ids, w)))
    torch.cuda.synchronize()
    for _ in range(10):
        for x, ids, w, out, ws, s, _ in calls:
            ex.moe.forward(x, ids, w, out, ws, stream=s)
    torch.cuda.synchronize()
    for *_, out, ws, s, want in calls:
        assert torch.equal(out.cpu().view(torch.int16), want.view(torch.int16))


def test_experts_call_of_more_than_one_pass(gpu):
    """262,144 / 64 tokens go at once: 5000 tokens of 64 columns take two passes."""
    ex = Experts(128, 128, [2], seed=4)
    T = 5000
    ids = torch.full((T, 64), -1, dtype=torch.int32)
    few, w2 = draw_ids(3, T, 2, 2)
    ids[:, 5], ids[:, 63] = few[:, 0], few[:, 1]
    w = torch.zeros(T, 64)
    w[:, 5], w[:, 63] = w2[:, 0], w2[:, 1]
    ex.check(draw_x(9, T, 128), ids, w)


# -------------------------------------------------------------- block norm --

def ref_norm(h, x, pre_w, post_w, gate, sig, scale, offset, pre_eps, post_eps):
    one = 1.0 if offset else 0.0
    b = x.double()
    if post_w is not None:
        b = b / (b.square().mean(1, keepdim=True) + post_eps).sqrt() * (post_w.double() + one)
    if gate is not None:
        gt = gate.double()
        b = b * (torch.sigmoid(gt) if sig else gt)
    y = h.double() + scale * b
    hn = None
    if pre_w is not None:
        hn = y / (y.square().mean(1, keepdim=True) + pre_eps).sqrt() * (pre_w.double() + one)
    return y, hn, (scale * b).abs()


@pytest.mark.parametrize("n,hidden", [(1, 8), (3, 64), (5, 512), (2, 520), (7, 1000), (64, 2048),
                                      (3, 2056), (2, 4096), (3, 5120), (2, 8192), (2, 8200),
                                      (1, 16384), (1037, 2048), (2049, 256)])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("gate,sig,post,pre,offset", [
    ("none", False, False, True, False), ("row", True, True, True, False),
    ("element", True, True, True, True), ("channel", False, True, False, True),
    ("element", False, False, False, False), ("row", False, False, True, True)])
def test_block_norm(gpu, n, hidden, f32, gate, sig, post, pre, offset):
    g = torch.Generator().manual_seed(n * hidden)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    h = (2 * rnd(n, hidden)).to(F32 if f32 else BF)
    x = rnd(n, hidden).to(BF)
    wt = lambda: ((0 if offset else 1) + 0.1 * rnd(hidden)).to(BF)  # noqa: E731
    post_w, pre_w = (wt() if post else None), (wt() if pre else None)
    gt = {"none": None, "row": (n, 1), "element": (n, hidden), "channel": (hidden,)}[gate]
    gt = None if gt is None else rnd(*gt).to(BF)
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    out = torch.empty_like(h, device=DEV)
    hn = torch.empty(n, hidden, device=DEV, dtype=BF) if pre else None
    gdn_amd.block_norm(dev(h), dev(x), h_out=out, hn=hn, pre_w=dev(pre_w), pre_eps=1e-5,
                       post_w=dev(post_w), post_eps=1e-6, gate=dev(gt), gate_sigmoid=sig,
                       scale=0.75, unit_offset=offset)
    torch.cuda.synchronize()
    y, yn, b = ref_norm(h, x, pre_w, post_w, gt, sig, 0.75, offset, 1e-5, 1e-6)
    # b: a mean of up to 16384 squares (64 in a lane, 6 steps across it, 8 waves),
    # root, division, exponential and products: below 128 half steps; h one more
    tb = 128 * HALF_F32 * b
    half = HALF_F32 if f32 else HALF_BF
    assert ((out.double().cpu() - y).abs() <= tb + half * (y.abs() + tb)).all()
    if pre:
        # tb moves the row's mean square by no more than it moves the row
        r = yn.abs() / y.abs().clamp_min(1e-30)
        rel = (tb.square().sum(1) / y.square().sum(1)).sqrt()[:, None] + 128 * HALF_F32
        t = tb * r + rel * yn.abs()
        assert ((hn.double().cpu() - yn).abs() <= t + HALF_BF * (yn.abs() + t)).all()


def test_block_norm_in_place_strided_and_no_rows(gpu):
    g = torch.Generator().manual_seed(3)
    n, hidden = 19, 264
    wide = torch.randn(n, 3 * hidden + 16, generator=g).to(BF).to(DEV)
    keep = wide.clone()
    h, x = wide[:, :hidden], wide[:, hidden + 8:2 * hidden + 8]
    gate, w = wide[:, -1:].clone(), torch.ones(hidden, device=DEV, dtype=BF)
    h1, hn1 = torch.empty(n, hidden, device=DEV, dtype=BF), torch.empty(n, hidden, device=DEV, dtype=BF)
    kw = dict(pre_w=w, post_w=w, gate=wide[:, -1:], gate_sigmoid=True)
    gdn_amd.block_norm(h, x, h_out=h1, hn=hn1, **kw)
    assert torch.equal(wide, keep)
    gdn_amd.block_norm(h, x, hn=x, **kw)  # h in place, hn over x
    assert torch.equal(h, h1) and torch.equal(x, hn1)
    assert torch.equal(wide[:, 2 * hidden + 8:], keep[:, 2 * hidden + 8:])
    assert torch.equal(wide[:, hidden:hidden + 8], keep[:, hidden:hidden + 8])
    assert torch.equal(gate, wide[:, -1:])
    gdn_amd.block_norm(h[:0], x[:0], hn=x[:0], pre_w=w)
    assert torch.equal(h, h1)


def test_block_norm_of_more_rows_than_a_launch(gpu):
    """2^22 rows go in a launch: the rows around the cut as a small call gives them."""
    n, hidden = (1 << 22) + 3, 8
    g = torch.Generator(DEV).manual_seed(8)
    h = torch.randn(n, hidden, generator=g, device=DEV)
    x = torch.randn(n, 2 * hidden, generator=g, device=DEV).to(BF)[:, hidden:]
    gate = torch.rand(n, 1, generator=g, device=DEV).to(BF)
    w = torch.rand(hidden, generator=g, device=DEV).to(BF)
    out, hn = torch.empty_like(h), torch.empty(n, hidden, device=DEV, dtype=BF)
    kw = dict(pre_w=w, post_w=w, gate_sigmoid=True)
    gdn_amd.block_norm(h, x, h_out=out, hn=hn, gate=gate, **kw)
    for lo, hi in ((0, 3), ((1 << 22) - 3, n)):
        o1, hn1 = torch.empty_like(out[lo:hi]), torch.empty_like(hn[lo:hi])
        gdn_amd.block_norm(h[lo:hi], x[lo:hi], h_out=o1, hn=hn1, gate=gate[lo:hi], **kw)
        assert torch.equal(out[lo:hi], o1) and torch.equal(hn[lo:hi], hn1)


def test_block_norm_agrees_with_add_rms_norm(gpu):
    """Without gate, scale and post norm it is the decoder's seam, whose hn is of the
    rounded h and has a rounding more before its weight."""
    g = torch.Generator().manual_seed(4)
    h, d = (torch.randn(33, 2048, generator=g).to(BF).to(DEV) for _ in range(2))
    w = (1 + 0.1 * torch.randn(2048, generator=g)).to(BF).to(DEV)
    h1, a, b = h.clone(), torch.empty_like(h), torch.empty_like(h)
    gdn_amd.add_rms_norm(h1, d, w, 1e-6, a)
    gdn_amd.block_norm(h, d, hn=b, pre_w=w)
    assert torch.equal(h, h1)
    assert ((a.double() - b.double()).abs() <= 4.2 * HALF_BF * b.double().abs()).all()


# ----------------------------------------------------------------- together --

class Half:
    """The sparse MLP half of a decoder layer, as a program would hold it."""

    def __init__(self, T, hidden=512, inner=128, E=24, k=4, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.k, self.E, self.T = k, E, T
        self.ex = Experts(hidden, inner, [E, 1], seed=seed + 1)
        gw = w4(g, 1, 32, hidden)  # E logits, the shared expert's gate, padding
        self.gate_parts = tuple(t[0] for t in gw)
        self.gate = gdn_amd.QLinear(hidden, [tuple(t.to(DEV) for t in self.gate_parts)])
        self.w = (1 + 0.1 * torch.randn(hidden, generator=g)).to(BF)
        self.dw = self.w.to(DEV)
        new = lambda *s, dtype=BF: torch.empty(*s, device=DEV, dtype=dtype)  # noqa: E731
        self.x, self.hn, self.y = new(T, hidden), new(T, hidden), new(T, hidden)
        self.logits = new(T, 32)
        self.ids, self.weights = new(T, k + 1, dtype=torch.int32), new(T, k + 1, dtype=F32)
        self.ws = self.ex.moe.workspace(T, k + 1)

    def run(self, h, mix):
        """h += mix; h += experts(norm(h)); hn = norm(h)"""
        gdn_amd.block_norm(h, mix, hn=self.x, pre_w=self.dw)
        self.gate.forward(self.x, self.logits)
        gdn_amd.moe_route(self.logits, self.ids, self.weights, self.E, self.k, num_shared=1,
                          shared_gate=True)
        self.ex.moe.forward(self.x, self.ids, self.weights, self.y, self.ws)
        gdn_amd.block_norm(h, self.y, hn=self.hn, pre_w=self.dw)


@pytest.mark.parametrize("T", [1, 7, 64, 400])
def test_the_half_as_a_program_runs_it(gpu, T):
    m = Half(T)
    g = torch.Generator().manual_seed(T)
    h, mix = (torch.randn(T, 512, generator=g).to(BF) for _ in range(2))
    dh = h.to(DEV)
    m.run(dh, mix.to(DEV))
    torch.cuda.synchronize()
    # the same values step by step in 64 bits, from what each step was given
    x, logits, ids, weights, y = (t.cpu() for t in (m.x, m.logits, m.ids, m.weights, m.y))
    h1 = (h.double() + mix.double()).to(BF)
    ri, rw = ref_route(logits[:, :25], 24, 4, shared=1, shared_gate=True)
    assert torch.equal(ids, ri) and ((weights.double() - rw).abs() <= 2.0 ** -17 * rw).all()
    d = h.double() + mix.double()
    hn0 = d / (d.square().mean(1, keepdim=True) + 1e-6).sqrt() * m.w.double()
    # f32 sums of 512 squares and the products: below 2^-17
    assert ((x.double() - hn0).abs() <= (HALF_BF + 2.0 ** -17) * hn0.abs()).all()
    gw = full(*m.gate_parts)
    lo, mag = x.double() @ gw.t(), x.double().abs() @ gw.abs().t()
    assert ((logits.double() - lo).abs() <= HALF_BF * lo.abs() + 2.0 ** -13 * mag).all()
    ref, tol = m.ex.ref(x, ids, weights)
    assert ((y.double() - ref).abs() <= tol).all()
    out = h1.double() + y.double()
    assert ((dh.double().cpu() - out).abs() <= HALF_BF * out.abs() * 1.001).all()


@pytest.mark.parametrize("T", [1, 33, 500])
def test_the_half_captured_and_replayed(gpu, T):
    """A captured step replays with other inputs, eager calls and another graph on
    the same workspace in between."""
    m = Half(T, seed=3)
    g = torch.Generator().manual_seed(T)
    ins = [tuple(torch.randn(T, 512, generator=g).to(BF).to(DEV) for _ in range(2))
           for _ in range(4)]
    want = []
    for h, mix in ins:
        hh = h.clone()
        m.run(hh, mix)
        want.append((hh, m.hn.clone()))
    sh, smix = torch.empty_like(ins[0][0]), torch.empty_like(ins[0][0])
    graphs = []
    for _ in range(2):
        sh.copy_(ins[0][0])
        smix.copy_(ins[0][1])
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            m.run(sh, smix)
        graphs.append(gr)
    for rep in range(6):
        i = rep % 4
        sh.copy_(ins[i][0])
        smix.copy_(ins[i][1])
        graphs[rep % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(sh, want[i][0]) and torch.equal(m.hn, want[i][1]), rep
        eager = ins[3 - i][0].clone()
        m.run(eager, ins[3 - i][1])
        assert torch.equal(eager, want[3 - i][0])


def test_binding_refuses_what_the_kernels_cannot_take(gpu):
    """Tensors of another device, type, size or layout are refused before a launch."""
    def z(*shape, dtype=BF, device=DEV):
        return torch.zeros(shape, dtype=dtype, device=device)

    ids, w = z(4, 2, dtype=torch.int32), z(4, 2, dtype=F32)
    gdn_amd.moe_route(z(4, 8), ids, w, 8, 2)
    for l, i, v, kw in ((z(4, 8, device="cpu"), ids, w, {}), (z(4, 8, dtype=F64), ids, w, {}),
                        (z(8, 4).t(), ids, w, {}), (z(4, 7), ids, w, {}),
                        (z(4, 8), ids.long(), w, {}), (z(4, 8), ids[:3], w, {}),
                        (z(4, 8), ids, w.to(BF), {}), (z(4, 8), z(2, 4, dtype=torch.int32).t(), w, {}),
                        (z(4, 8), ids, w.cpu(), {}), (z(4, 8), ids, w, dict(bias=z(7, dtype=F32))),
                        (z(4, 8), ids, w, dict(bias=z(8)))):
        with pytest.raises(ValueError):
            gdn_amd.moe_route(l, i, v, 8, 2, **kw)

    h, x, n = z(4, 64), z(4, 64), z(64)
    gdn_amd.block_norm(h, x, hn=z(4, 64), pre_w=n)
    for a, b, kw in ((h.cpu(), x, {}), (h, x.cpu(), {}), (h, x.float(), {}), (h, z(3, 64), {}),
                     (h.to(F64), x, {}), (z(64, 4).t(), x, {}), (h, x, dict(h_out=h.float())),
                     (h, x, dict(hn=z(4, 32), pre_w=n)), (h, x, dict(hn=z(4, 64), pre_w=n.float())),
                     (h, x, dict(post_w=z(32))), (h, x, dict(post_w=z(128)[::2])),
                     (h, x, dict(gate=z(4, 2))), (h, x, dict(gate=z(4, 1, dtype=F32)))):
        with pytest.raises(ValueError):
            gdn_amd.block_norm(a, b, **kw)

    ex = Experts(128, 128, [2])
    ws, x = ex.moe.workspace(4, 2), z(4, 128)
    ex.moe.forward(x, ids, w, z(4, 128), ws)
    for a, i, v, o, s in ((x.cpu(), ids, w, z(4, 128), ws), (z(4, 64), ids, w, z(4, 128), ws),
                          (x.float(), ids, w, z(4, 128), ws), (x, ids.long(), w, z(4, 128), ws),
                          (x, ids, w.double(), z(4, 128), ws), (x, ids, w[:2], z(4, 128), ws),
                          (x, ids, w, z(3, 128), ws), (x, ids, w, z(4, 128, dtype=F32), ws),
                          (x, ids, w, z(4, 128), ws.cpu()), (x, ids, w, z(4, 128), ws.float())):
        with pytest.raises(ValueError):
            ex.moe.forward(a, i, v, o, s)
    with pytest.raises(gdn_amd.GdnError):
        ex.moe.forward(x, ids, w, z(4, 128), ws[:256])
    torch.cuda.synchronize()

"""The 8-bit paged cache where its kernels' own limits lie, against its definition in 64 bits
(tests/kv8_testlib.py)."""
import numpy as np
import pytest

from gdn_testlib import say
from test_gpu_kv8 import Pair, bf, i32, num

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,dim,cached,new,window", [
    (1, 128, 1000, 1537, 1900), (1, 256, 258, 769, 856), (1, 64, 1, 1025, 896),
    (3, 64, 266, 806, 933), (5, 128, 214, 868, 948), (6, 256, 225, 861, 948)])
def test_windows_on_prompts_in_pieces(gpu, hq, dim, cached, new, window):
    """A tile between the first, which starts below its window, and the last, which has few
    tokens, sees more pages than both: every one of its keys counts. (hq query heads on one.)"""
    rng = np.random.default_rng(cached)
    p = Pair(2, 50, 48, hq=hq, hk=1, dim=dim, tokens=1600)
    say("kv8 window on pieces", hq, dim, cached, new, window)
    p.step([1], [0], [cached])
    p.append(rng)
    p.step([1], [cached], [new])
    p.append(rng)
    p.attention(rng, label=f"window {window}", window=window)
    p.kv.close()


def captured_step(kv, slots, lens, ntok, tokens, most):
    """A graph of a step on a cache, planned once before."""
    import torch
    args = i32(slots), i32(lens), i32(ntok)
    kv.step(*args, tokens, most)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv.step(*args, tokens, most)
    return graph, args


def held(kv, places):
    import torch
    out = torch.full((2, len(places), kv.Hkv, kv.D), 9.0, dtype=torch.bfloat16, device="cuda:0")
    kv.gather(0, places, out[0], out[1])
    return out


@pytest.mark.parametrize("rows,ntok", [
    (12, [200, 3, 130, 64, 77]),  # more rows in the call than in the plan
    (70, [1, 65, 0, 400, 2, 190] * 11),
    (2, [70, 130, 200, 64, 9]),   # fewer
    (5, [70, 130, 200, 64, 9]),
    (65, [100] * 70)])
def test_append_behind_another_steps_replay(gpu, rows, ntok):
    """Rows of many pages planned by a graph, appended under bounds of `rows` rows, of which
    an earlier step of single tokens was: the first `rows` hold what a cache that planned
    them itself does, and the others' pages are as they were."""
    import gdn_amd
    import torch
    rng = np.random.default_rng(rows)
    hk, d, n, T = 2, 64, len(ntok), sum(ntok)
    lens = rng.integers(0, 150, n).tolist()
    slots = rng.permutation(200)[:n].tolist()
    others = [s for s in range(200) if s not in slots][:rows]
    fill = [bf(rng, sum(lens), hk, d)[0] for _ in range(2)]
    kv, twin = (gdn_amd.KV8Cache(1, 200, 1200, 10, 4, hk, d, 8000) for _ in range(2))
    for c in (kv, twin):
        c.step(i32(slots), i32([0] * n), i32(lens), sum(lens))
        c.append(0, *fill)
    say("kv8 append behind a replay", rows, n)
    graph, args = captured_step(kv, slots, lens, ntok, T, max(ntok))
    twin.step(*args, T, max(ntok))
    single = i32(others), i32([0] * rows), i32([1] * rows)
    for c in (kv, twin):
        c.step(*single, T, max(ntok))
    graph.replay()
    twin.step(*args, T, max(ntok))
    places = twin.views()["map"][:T].clone()
    assert torch.equal(places, kv.views()["map"][:T])
    before = held(kv, places)
    k, v = (bf(rng, T, hk, d)[0] for _ in range(2))
    kv.append(0, k, v)
    twin.append(0, k, v)
    inside = sum(ntok[:rows])
    assert torch.equal(held(kv, places)[:, :inside], held(twin, places)[:, :inside])
    assert torch.equal(held(kv, places)[:, inside:], before[:, inside:])
    for c in (kv, twin):
        assert c.check() == 0
        c.close()


@pytest.mark.parametrize("rows", [4, 2, 64, 100])
@pytest.mark.parametrize("longest", [1, 20])
def test_attention_behind_another_steps_replay(gpu, rows, longest):
    """64 rows planned by a graph, long ones first, under bounds of another number of rows, by
    which keys are split otherwise: the rows inside them by the definition, the others'
    tokens left as they were."""
    rng = np.random.default_rng(rows)
    n = 64
    p = Pair(170, 560, 66, hq=4, hk=2, dim=64, tokens=17000)
    slots = rng.permutation(170).tolist()
    slots, others = slots[:n], slots[n:n + rows]
    lens, ntok = [4096, 4000, 4096, 3000] + [5] * (n - 4), [longest] + [1] * (n - 1)
    T = sum(ntok)
    p.step(slots, [0] * n, lens)
    p.append(rng)
    say("kv8 attention behind a replay", rows, longest)
    graph, _ = captured_step(p.kv, slots, lens, ntok, T, longest)
    p.ref.step(slots, lens, ntok, T, longest)
    p.step(others, [0] * rows, [1] * rows, max(T, rows), longest)
    graph.replay()
    p.ref.step(slots, lens, ntok, T, longest)
    p.check_tables()
    p.ref.plan = p.ref.plan[:rows]
    p.ref.end = sum(ntok[:rows])
    p.append(rng)
    p.attention(rng, label=f"{rows} of {n} rows", gate=True)
    p.kv.close()


@pytest.mark.parametrize("new", [2, 20])
def test_tokens_behind_a_replayed_plan_are_left_alone(gpu, new):
    """A step whose later rows are refused, then the replay of a shorter one: the tokens that
    were refused are none of the plan's any more, and their outputs stay."""
    rng = np.random.default_rng(new)
    p = Pair(4, 12, 6, hq=4, hk=2, dim=64, tokens=200)
    p.step([1, 2], [0, 0], [70, 40])
    p.append(rng)
    graph, _ = captured_step(p.kv, [2, 1], [40, 70], [new, 1], new + 1, new)
    p.ref.step([2, 1], [40, 70], [new, 1], new + 1, new)
    p.step([0, 9, 9], [0, 0, 0], [1, new, new], 2 * new + 90, new)
    graph.replay()
    p.ref.step([2, 1], [40, 70], [new, 1], new + 1, new)
    assert p.kv.check() == 1
    p.append(rng)
    p.attention(rng, label="a shorter plan")  # rows behind the plan's tokens stay as they were
    p.kv.close()


def capped_reference(ref, q, cap, scale):
    """(out, tolerance) as Ref.attention's, but for a capped score, whose error is within 2^-19 of
    itself: f32 roundings of its factors, and of the function, whose worst is at -1/2 where
    2 / (1 + e^2y) is 1.46 with a relative error of 2 2^-23 (a reciprocal's and an exponential's
    last places, two roundings), 6.5 2^-23 of the result."""
    out, tol = np.zeros((2, ref.end) + q.shape[1:])
    G = q.shape[1] // ref.heads
    for s, a, b, c in ref.plan:
        for t in range(b):
            for h in range(q.shape[1]):
                k, v = (x[:a + t + 1, h // G] for x in ref.held[s])
                qk = q[c + t, h] * k
                y = qk.sum(1) * scale / cap
                sc = cap * np.tanh(y)
                err = np.abs(qk).sum(1) * abs(scale) * ref.dim * 2.0 ** -24 / np.cosh(np.minimum(
                    np.abs(y) * 0.99, 300)) ** 2
                err += 2.0 ** -19 * np.abs(sc)
                w = np.exp(sc - sc.max())
                w /= w.sum()
                o, av = w @ v, w @ np.abs(v)
                out[c + t, h] = o
                tol[c + t, h] = ((2.0 ** -11 + 2 * err.max() + (len(k) + 16) * 2.0 ** -24 + 2.0 ** -20) * av +
                                 2.0 ** -25 * np.abs(v).sum(0) + 2.0 ** -8 * np.abs(o)) * (1 + 2.0 ** -7)
    return out, tol


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("cap,loud", [(1e-30, 1e10), (1e-30, 1.0), (1e-3, 1.0), (0.5, 1.0), (6.0, 1.0),
                                      (1e3, 1.0), (1e4, 1.0), (1e6, 1.0), (1e8, 1.0), (1e30, 1.0)])
def test_caps_of_every_size(gpu, dim, cap, loud):
    """Scores far above their cap and far below it, where it changes nothing, and a key of zeros,
    in a step of tiles and in one of chunks."""
    import torch
    rng = np.random.default_rng(dim)
    p = Pair(2, 12, 6, hq=4, hk=2, dim=dim)
    scale = 3 * loud / dim ** 0.5
    cap = float(np.float32(cap))
    for step in ([1, 0], [0, 0], [130, 33]), ([0, 1], [33, 130], [1, 3]):
        p.step(*step)
        p.append(rng, change=lambda x: x[0].zero_())
        q, qn = bf(rng, p.kv.tokens, 4, dim)
        out = torch.zeros_like(q)
        p.kv.attention(0, q, out, scale=scale, softcap=cap)
        want, tol = capped_reference(p.ref, qn, cap, float(np.float32(scale)))
        err = np.abs(num(out) - want)
        say("kv8 cap", cap, "worst error / tolerance", float((err / np.maximum(tol, 1e-30)).max()))
        assert np.all(err <= tol)
    p.kv.close()


def test_caps_that_are_refused(gpu):
    import gdn_amd
    import torch
    kv = gdn_amd.KV8Cache(1, 2, 4, 4, 4, 2, 64, 8)
    kv.step(i32([0]), i32([0]), i32([4]), 4)
    q = torch.zeros(4, 4, 64, device="cuda:0", dtype=torch.bfloat16)
    for cap in (1e-31, 1e-40, 1.1e30, 3e38, float("inf"), -1.0):
        with pytest.raises(gdn_amd.GdnError, match="softcap"):
            kv.attention(0, q, q.clone(), softcap=cap)
    kv.close()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("scale", [1e-6, 1e-13, 1e-38, 1e-42, -1e-13])
def test_scales_that_leave_nothing_of_the_scores(gpu, dim, scale):
    """Queries of zeros and others, a page of zeros, in a step of tiles and in one of chunks."""
    rng = np.random.default_rng(dim)
    p = Pair(2, 12, 6, hq=4, hk=2, dim=dim)
    p.step([1], [0], [64])
    p.append(rng, change=lambda x: x.zero_())
    for step in ([1, 0], [64, 0], [70, 33]), ([0, 1], [33, 134], [1, 3]):
        p.step(*step)
        p.append(rng)
        p.attention(rng, label=f"scale {scale}", std=0.0, scale=scale)
        p.attention(rng, label=f"scale {scale}", scale=scale)
        p.attention(rng, label=f"scale {scale}, window", scale=scale, window=50)
    p.kv.close()


def test_rows_that_run_into_each_other_are_refused(gpu):
    """A stride of one head where a row has several: append and gather take whole rows. A single
    row's stride does not matter."""
    import gdn_amd
    import torch
    kv = gdn_amd.KV8Cache(1, 2, 4, 4, 4, 2, 64, 8)
    kv.step(i32([0]), i32([0]), i32([4]), 4)
    flat = torch.zeros(4 * 128, device="cuda:0", dtype=torch.bfloat16)
    good = flat.view(4, 2, 64)
    for stride in (64, 72, 120):
        bad = flat.as_strided((4, 2, 64), (stride, 64, 1))
        for call in (lambda: kv.append(0, bad, good), lambda: kv.append(0, good, bad),
                     lambda: kv.gather(0, i32(range(4)), bad, None),
                     lambda: kv.gather(0, i32(range(4)), None, bad)):
            with pytest.raises(gdn_amd.GdnError, match="row strides"):
                call()
    kv.append(0, good, good)
    for stride in (64, 8, 0, 1000):
        one = flat.as_strided((1, 2, 64), (stride, 64, 1))
        kv.gather(0, i32([0]), one, one.clone())
        kv.step(i32([0]), i32([4]), i32([1]), 1)
        kv.append(0, one, one)
    kv.close()


@pytest.mark.parametrize("most", [1, 20])
def test_a_million_faint_keys(gpu, most):
    """One key by 2^25.2 stronger than 2^20 others, which together weigh 2.6%, in one piece (the
    bounds leave no more): where all values are the same, so is the output; where the strong
    key's is zero, it is the others' weight."""
    import gdn_amd
    import torch
    say("kv8 a million keys", most)
    step, n = 262144, 1024
    kv = gdn_amd.KV8Cache(1, 1024, 16400, 16400, 1, 1, 64, step)
    k = torch.zeros(step, 1, 64, device="cuda:0", dtype=torch.bfloat16)
    v = torch.full_like(k, 4.0)
    slots = i32([0] + [-1] * (n - 1))
    out = torch.zeros_like(k)
    strong = 7.0 * 2.5
    for first, want in ((4.0, 4.0), (0.0, 4.0 * 2 ** 20 / (2 ** 20 + np.exp(strong)))):
        for i in range(4):
            kk, vv = k.clone(), v.clone()
            if i == 0:
                kk[0, 0, 0] = 7.0
                vv[0] = first
            kv.step(i32([0]), i32([i * step]), i32([step]), step)
            kv.append(0, kk, vv)
        q = torch.zeros_like(k)
        q[:most, 0, 0] = 2.5
        kv.step(slots, i32([4 * step] + [0] * (n - 1)), i32([most] + [0] * (n - 1)),
                n if most == 1 else step, most)
        t = kv.tokens
        kv.append(0, k[:t], v[:t])
        kv.attention(0, q[:t], out[:t], scale=1.0)
        assert kv.check() == 0
        # each weight within 2^-11 of itself, or 2^-29 of the largest; f32 sums, of 2^20 / 32 additions
        # to the weights' and 2^20 / 16 to the outputs', 2^-24 of a sum each; the result's rounding
        got = num(out[:most])
        tol = want * (2.0 ** -8 + 2.0 ** -10 + (2.0 ** 15 + 2.0 ** 16) * 2.0 ** -24)
        tol += 2.0 ** 20 * 2.0 ** -29 * 4.0 if first == 0 else 0
        say("kv8 a million keys", float(got.min()), float(got.max()), want, tol)
        assert np.all(np.abs(got - want) <= tol)
    kv.close()

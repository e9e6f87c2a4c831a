"""The 8-bit paged cache where its kernels' own limits lie, against its definition in 64 bits
(tests/kv8_testlib.py)."""
import numpy as np
import pytest

from gdn_testlib import say
from test_gpu_kv8 import Pair, bf, i32

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

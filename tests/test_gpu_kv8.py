"""The 8-bit paged cache on the GPU (gdn_kv8_*) against its definition in 64 bits
(tests/kv8_testlib.py): tables, maps and held values exactly, attention inside the sum
of the roundings that its contract names."""
import numpy as np
import pytest

from gdn_testlib import say
from kv8_testlib import PAGE, Ref

pytestmark = pytest.mark.gpu


def i32(x):
    import torch
    return torch.tensor(list(x), dtype=torch.int32, device="cuda:0")


def bf(rng, *shape, std=1.0):
    """(device bf16, the same numbers in 64 bits)"""
    import torch
    t = torch.from_numpy((rng.standard_normal(shape) * std).astype(np.float32)).to(torch.bfloat16)
    return t.to("cuda:0"), t.double().numpy()


def num(t):
    return t.detach().double().cpu().numpy()


class Pair:
    """The cache and its reference, driven together."""

    def __init__(self, slots, pages, max_pages, hq=8, hk=2, dim=64, tokens=512, layers=1):
        import gdn_amd
        self.kv = gdn_amd.KV8Cache(layers, slots, pages, max_pages, hq, hk, dim, tokens)
        self.ref = Ref(slots, pages, max_pages, hk, dim)
        self.views = self.kv.views()
        self.hq, self.hk, self.dim = hq, hk, dim

    def step(self, slots, lens, ntok, tokens=None, max_row=0, stream=None):
        import torch
        tokens = sum(max(b, 0) for s, b in zip(slots, ntok) if s >= 0) if tokens is None else tokens
        out = torch.full((len(slots),), -7, dtype=torch.int32, device="cuda:0")
        self.kv.step(i32(slots), i32(lens), i32(ntok), tokens, max_row, lens_out=out, stream=stream)
        cu, pos, where, new = self.ref.step(slots, lens, ntok, tokens, max_row)
        v = self.views
        assert v["cu"][:len(cu)].tolist() == cu
        assert v["pos"][:tokens].tolist() == pos.tolist()
        assert v["map"][:tokens].tolist() == where.tolist()
        assert out.tolist() == new
        self.check_tables()
        return new

    def check_tables(self):
        v, r = self.views, self.ref
        assert v["owned"].tolist() == [len(t) for t in r.table]
        assert v["table"].tolist() == [t + [-1] * (r.max_pages - len(t)) for t in r.table]
        assert v["count"].tolist() == [len(r.free)]
        assert v["free"].tolist() == r.free + [-1] * (r.num_pages - len(r.free))

    def append(self, rng, std=1.0, layer=0, change=None):
        t = self.kv.tokens
        out = []
        for _ in range(2):
            x, _ = bf(rng, t, self.hk, self.dim, std=std)
            if change is not None:
                change(x)
            out.append(x)
        self.kv.append(layer, *out)
        self.ref.append(num(out[0]), num(out[1]))
        return out

    def check_held(self, layer=0):
        import torch
        for s, (k, v) in self.ref.held.items():
            n = min(len(k), len(self.ref.table[s]) * PAGE)
            if n == 0 or s in self.ref.unknown:
                continue
            at = i32(self.ref.table[s][t // PAGE] * PAGE + t % PAGE for t in range(n))
            ko = torch.full((n, self.hk, self.dim), 9.0, dtype=torch.bfloat16, device="cuda:0")
            vo = torch.full_like(ko, 9.0)
            self.kv.gather(layer, at, ko, vo)
            np.testing.assert_array_equal(num(ko), k[:n])
            np.testing.assert_array_equal(num(vo), v[:n])

    def attention(self, rng, gate=False, layer=0, label="", std=1.5, **kw):
        import torch
        t = self.kv.tokens
        q, qn = bf(rng, t, self.hq, self.dim, std=std)
        out = torch.full_like(q, 7.0)
        g, gn = bf(rng, t, self.hq, self.dim) if gate else (None, None)
        dev = dict(kw)
        if kw.get("slopes") is not None:
            dev["slopes"] = torch.tensor(kw["slopes"], dtype=torch.float32, device="cuda:0")
        if kw.get("prefix") is not None:
            dev["prefix"] = i32(kw["prefix"])
        self.kv.attention(layer, q, out, gate=g, **dev)
        want, tol = self.ref.attention(qn, gate=gn, **kw)
        got = num(out)
        end = min(self.ref.end, t)
        err = np.abs(got[:end] - want[:end])
        say("kv8 attention", label, f"worst error / tolerance "
            f"{float(np.nanmax(err / np.maximum(tol[:end], 1e-30), initial=0)):.3f}")
        assert np.all(err <= tol[:end])
        assert np.all(got[end:] == 7.0)  # rows behind the last token
        return q, out


def test_tables_follow_the_lengths(gpu):
    """Rows admitted, grown, cut back, released and admitted again, padding among them."""
    p = Pair(6, 20, 8)
    say("kv8 step")
    p.step([3, 0, -1, 5], [0, 0, 9, 0], [1, 64, 4, 130])
    p.step([3, 0, 5], [1, 64, 130], [63, 1, 1])
    p.step([5, 3], [100, 64], [0, 200])       # cut back while another grows
    p.step([0, 1, 2], [0, 0, 0], [0, 65, 0])  # released; its pages go on
    p.step([3], [264], [0])
    p.step([5, 1, 3, 2, 4, 0], [0, 0, 0, 0, 0, 0], [0, 0, 0, 0, 0, 0])
    assert p.views["count"].item() == 20
    assert p.kv.check() == 0
    p.kv.close()


def test_the_same_step_twice_changes_nothing(gpu):
    p = Pair(4, 12, 8)
    for _ in range(2):
        p.step([0, 2, 1], [100, 0, 5], [30, 128, 0])
    p.kv.close()


@pytest.mark.parametrize("slots,lens,ntok,tokens,max_row,flags", [
    ([0, 9], [0, 0], [3, 4], 7, 0, 1),                 # no such slot
    ([1, 1, 0], [0, 5, 0], [3, 4, 2], 9, 0, 2),        # twice
    ([0, 1], [500, 0], [13, 2], 15, 0, 4),             # past max_pages
    ([0, 1], [-1, 0], [3, 2], 5, 0, 4),
    ([0, 1], [0, 0], [-3, 2], 2, 0, 4),
    ([0, 1], [0, 0], [3, 2], 5, 2, 4),                 # past max_row_tokens
    ([0, 1, 2], [0, 0, 0], [3, 4, 2], 5, 0, 4),        # past max_tokens: the second, then the third
    ([0, 1], [2 ** 31 - 1, 0], [1, 2], 3, 0, 4),
    ([0, 1, 2, 0], [0, 0, 0, 0], [200, 400, 64, 0], 664, 0, 2 | 8),
    ([0, 1, 2], [200, 500, 64], [1, 1, 0], 2, 0, 8)])
def test_refused_rows(gpu, slots, lens, ntok, tokens, max_row, flags):
    """Refused rows change nothing, their tokens have no place and attention gives zeros."""
    p = Pair(3, 8, 8, tokens=700)
    say("kv8 refused rows", slots, lens, ntok)
    p.step([2], [0], [70])
    rng = np.random.default_rng(1)
    p.append(rng)
    p.step(slots, lens, ntok, tokens, max_row)
    assert p.kv.check() == flags == p.ref.flags
    assert p.kv.check() == 0
    p.append(rng)
    p.check_held()
    import torch
    q = torch.randn(tokens, p.hq, p.dim, device="cuda:0").to(torch.bfloat16)
    out = torch.full_like(q, 7.0)
    p.kv.attention(0, q, out)
    want, tol = p.ref.attention(num(q)) if tokens < 20 and not p.ref.unknown else (None, None)
    pos = p.views["pos"][:tokens].cpu().numpy()
    end = min(p.ref.end, tokens)
    got = num(out)
    assert np.all(got[:end][pos[:end] < 0] == 0.0)
    assert np.all(got[end:] == 7.0)
    if want is not None:
        assert np.all(np.abs(got[:end] - want[:end]) <= tol[:end])
    p.kv.close()


@pytest.mark.parametrize("n", [1, 63, 65, 257, 1025, 4096])
def test_many_rows(gpu, n):
    """Every size of the plan's kernel; slots in a mixed order, lengths that grow and fall."""
    rng = np.random.default_rng(n)
    p = Pair(n, 3 * n + 5, 8, hq=1, hk=1, tokens=9000)
    for lo, hi in ((0, 3), (0, 2)):
        slots = rng.permutation(n).tolist()
        lens = rng.integers(0, 200, n).tolist()
        ntok = rng.integers(lo, hi, n).tolist()
        if n > 3:
            slots[n // 2] = -1
            ntok[n // 3] = 150
        say("kv8 step of", n)
        p.step(slots, lens, ntok)
    p.kv.close()


def test_many_tokens_are_mapped_by_their_own_kernel(gpu):
    p = Pair(5, 400, 300, hq=1, hk=1, tokens=20000)
    p.step([4, 0, 2], [5, 0, 77], [9001, 0, 6999])
    p.kv.close()


@pytest.mark.parametrize("dim,hk", [(64, 1), (128, 3), (256, 2)])
def test_held_values(gpu, dim, hk):
    """Prompts, single tokens that raise a page's exponent and ones that do not, cuts back
    inside a page, numbers of every size: what is held is the definition's, bit for bit."""
    import torch
    rng = np.random.default_rng(dim + hk)
    p = Pair(4, 24, 8, hq=hk, hk=hk, dim=dim)
    say("kv8 append", dim, hk)
    p.step([1, 3], [0, 0], [70, 130])
    p.append(rng)
    p.check_held()
    for i, std in enumerate([1.0, 30.0, 0.01, 1e4, 1.0]):
        p.step([3, 1, 0], [130 + i, 70 + i, i], [1, 1, 1])
        p.append(rng, std=std)
        p.check_held()
    p.step([3, 1], [131, 64], [3, 5])
    p.append(rng, std=1e-3)
    p.check_held()
    p.step([2], [0], [64])
    # every exponent of bf16 in a page, and zeros
    p.append(rng, change=lambda x: x.copy_(
        x * (2.0 ** torch.arange(-40, 24, device="cuda:0"))[:, None, None]))
    p.check_held()
    p.kv.close()


def test_pages_of_zeros_infinities_and_nan(gpu):
    rng = np.random.default_rng(5)
    p = Pair(3, 9, 3, hq=2, hk=2, dim=64)
    p.step([0], [0], [64])
    p.append(rng, change=lambda x: x.zero_())
    p.check_held()

    def odd(x):
        x[1, 0, 3], x[2, 1, 5], x[3, 0, 0] = float("inf"), float("nan"), float("-inf")

    p.step([1], [0], [10])
    p.append(rng, change=odd)
    p.check_held()
    p.step([1], [10], [2])  # they stay, and do not enter the exponent
    p.append(rng, std=20.0)
    p.check_held()
    p.step([2], [0], [4])   # the largest and the smallest numbers
    p.append(rng, change=lambda x: (x.fill_(3e38), x[0].fill_(1e-38)))
    p.check_held()
    p.step([2], [0], [4])
    p.append(rng, change=lambda x: x.fill_(1e-14))
    p.check_held()
    p.kv.close()


def test_append_twice_leaves_the_same_bits(gpu):
    rng = np.random.default_rng(6)
    p = Pair(2, 9, 4, hq=2, hk=2, dim=128)
    p.step([0], [0], [40])
    p.append(rng)
    p.step([0], [40], [50])
    k, v = p.append(rng, std=100.0)
    p.kv.append(0, k, v)
    p.check_held()
    p.kv.close()


@pytest.mark.parametrize("hq,hk,dim", [(8, 1, 256), (16, 2, 256), (4, 4, 64), (12, 4, 128),
                                       (16, 1, 64), (5, 1, 128), (7, 7, 256)])
def test_attention_of_single_tokens_and_prompts(gpu, hq, hk, dim):
    """Page edges, one cached token, prompts beside single tokens, none in a row."""
    rng = np.random.default_rng(hq * hk + dim)
    p = Pair(6, 40, 12, hq=hq, hk=hk, dim=dim)
    say("kv8 attention", hq, hk, dim)
    p.step([0, 4, 2], [0, 0, 0], [1, 63, 130])
    p.append(rng)
    p.attention(rng, label="prompts")
    p.step([2, 0, 4, 5], [130, 1, 63, 0], [1, 1, 1, 0])
    p.append(rng)
    p.attention(rng, gate=True, label="single tokens")
    p.step([1, 4, 0, 2], [0, 64, 2, 131], [20, 1, 0, 5], tokens=31)
    p.append(rng)
    p.attention(rng, label="mixed, rows to spare")
    p.kv.close()


@pytest.mark.parametrize("kw", [
    dict(window=1), dict(window=64), dict(window=70, softcap=5.0), dict(softcap=30.0),
    dict(slopes=0.05), dict(prefix=1), dict(window=20, prefix=90), dict(window=3, prefix=1000),
    dict(scale=0.5, slopes=-0.01), dict(scale=-0.2, softcap=2.0, window=200)])
def test_attention_options(gpu, kw):
    rng = np.random.default_rng(11)
    kw = dict(kw)
    hq, hk = 6, 2
    if "slopes" in kw:
        kw["slopes"] = [kw["slopes"] * 2.0 ** -h for h in range(hq)]
    far = kw.pop("prefix", None)
    p = Pair(4, 40, 12, hq=hq, hk=hk, dim=64, tokens=600)
    p.step([0, 3], [0, 0], [300, 95])
    p.append(rng)
    if far:
        kw["prefix"] = [far, 0]
    p.attention(rng, label=f"prompts {kw}", **kw)
    p.step([3, 1, 0], [95, 0, 300], [1, 7, 1])
    p.append(rng)
    if far:
        kw["prefix"] = [far, -3, far + 5]
    p.attention(rng, gate=True, label=f"tokens {kw}", **kw)
    p.kv.close()


def test_long_rows_and_loud_pages(gpu):
    """Many pages for a token; pages whose exponents differ by far, either way."""
    rng = np.random.default_rng(12)
    p = Pair(2, 80, 70, hq=8, hk=1, dim=128, tokens=4400)
    sizes = 2.0 ** np.repeat(rng.integers(-12, 13, 70), 64)[:4300]

    def loud(x):
        import torch
        x.mul_(torch.tensor(sizes, device="cuda:0", dtype=torch.bfloat16)[:, None, None])

    p.step([1], [0], [4300])
    ks = [None]

    def values_only(x):
        if ks[0] is None:
            ks[0] = x
        else:
            loud(x)

    p.append(rng, change=values_only)
    p.step([1, 0], [4300, 0], [1, 1])
    p.append(rng)
    p.attention(rng, label="loud values")
    p.attention(rng, label="sharp", std=30.0)
    p.step([1], [4300], [9])
    p.append(rng)
    p.attention(rng, label="nine tokens", gate=True)
    p.kv.close()


@pytest.mark.parametrize("hq,hk,dim", [(8, 1, 256), (12, 4, 128), (3, 3, 64)])
def test_prompts_behind_long_contexts(gpu, hq, hk, dim):
    """Few tiles whose keys are split: pieces that a tile does not reach, windows that leave
    some out, tokens of tiles and of groups in one step, enough tokens for every kernel that
    joins pieces."""
    rng = np.random.default_rng(17)
    p = Pair(5, 120, 60, hq=hq, hk=hk, dim=dim, tokens=4200)
    p.step([0, 1], [0, 0], [2900, 1200])
    p.append(rng)
    p.step([0, 4, 1], [2900, 0, 1200], [35, 17, 3])
    p.append(rng)
    p.attention(rng, label="split tiles", gate=True)
    p.attention(rng, label="split tiles, window", window=300, softcap=20.0)
    p.step([1, 3, 0], [1203, 0, 2935], [16, 700, 1], tokens=900)
    p.append(rng)
    p.attention(rng, label="long step", slopes=[0.01] * hq)
    p.kv.close()


def test_nan_reaches_those_that_see_it(gpu):
    """A NaN key or value of a later token, of one outside the window, behind a cut."""
    import torch
    rng = np.random.default_rng(13)
    p = Pair(2, 12, 5, hq=4, hk=2, dim=64)
    p.step([0], [0], [100])
    nan = float("nan")
    k, v = (bf(rng, 100, 2, 64)[0] for _ in range(2))
    v[70, 1, 7] = nan
    k[90, 0, 0] = float("inf")
    p.kv.append(0, k, v)
    q, _ = bf(rng, 100, 4, 64)
    out = torch.zeros_like(q)
    p.kv.attention(0, q, out)
    bad = torch.isnan(out)
    want = torch.zeros_like(bad)
    want[70:, 2:] = True      # head 1's queries that see the value
    want[90:, :2] = True      # head 0's queries that see the key
    assert torch.equal(bad, want)
    clean_k, clean_v = k.clone(), v.clone()
    clean_v[70, 1, 7] = 0.25
    clean_k[90, 0, 0] = 0.25
    p.kv.append(0, clean_k, clean_v)
    ref = torch.zeros_like(q)
    p.kv.attention(0, q, ref)
    p.kv.append(0, k, v)
    assert torch.equal(out[:70], ref[:70])
    # outside the window
    p.kv.attention(0, q, out, window=5)
    bad = torch.isnan(out)
    want.zero_()
    want[70:75, 2:] = True
    want[90:95, :2] = True
    assert torch.equal(bad, want)
    # the row is cut back before them: single tokens do not see what is left in the page
    p.kv.step(i32([0]), i32([66]), i32([1]), 1, 1)
    one_k, one_v = (bf(rng, 1, 2, 64)[0] for _ in range(2))
    p.kv.append(0, one_k, one_v)
    o = torch.zeros(1, 4, 64, device="cuda:0", dtype=torch.bfloat16)
    p.kv.attention(0, q[:1].contiguous(), o)
    assert not torch.isnan(o).any()
    p.kv.close()


def test_rows_do_not_depend_on_each_other(gpu):
    """A row's bits beside rows of other lengths, contents and sizes, under the same bounds of
    the step; and the same step twice."""
    import torch
    import gdn_amd
    rng = np.random.default_rng(14)
    hq, hk, d = 16, 2, 256
    kv = gdn_amd.KV8Cache(1, 40, 300, 40, hq, hk, d, 4096)
    mine, len0 = 7, 1500
    first = [bf(rng, len0, hk, d)[0] for _ in range(2)]
    for n in (2, 30):  # few segments and many
        for new in (1, 5, 90):
            q, k, v = (bf(rng, new, h, d)[0] for h in (hq, hk, hk))
            outs = []
            for other in range(3):
                slots = [s for s in rng.permutation(40).tolist() if s != mine][:n]
                slots[rng.integers(n)] = mine
                lens = rng.integers(0, 300, n).tolist()
                ntok = rng.integers(1, 3, n).tolist()
                at = slots.index(mine)
                lens[at], ntok[at] = len0, new
                T, cu = 300, [0]
                for x in ntok:
                    cu.append(cu[-1] + x)
                kv.step(i32([mine]), i32([0]), i32([len0]), len0)
                kv.append(0, *first)
                kv.step(i32(range(40)), i32([len0 if s == mine else 0 for s in range(40)]),
                        i32([0] * 40), 0)
                kv.step(i32(slots), i32(lens), i32(ntok), T, 90)
                wide = [bf(rng, T, h, d)[0] for h in (hq, hk, hk)]
                for w, x in zip(wide, (q, k, v)):
                    w[cu[at]:cu[at] + new] = x
                kv.append(0, *wide[1:])
                for _ in range(2):
                    out = torch.empty_like(wide[0])
                    kv.attention(0, wide[0], out)
                    outs.append(out[cu[at]:cu[at] + new])
            assert kv.check() == 0
            for o in outs[1:]:
                assert torch.equal(outs[0], o), (n, new)
    kv.close()


def test_strides_streams_and_layers(gpu):
    """Columns of wider tensors, heads first, another stream than the current one, a second
    layer on the same plan."""
    import torch
    import gdn_amd
    rng = np.random.default_rng(15)
    hq, hk, d, T = 8, 2, 128, 37
    kv = gdn_amd.KV8Cache(2, 3, 9, 4, hq, hk, d, 64)
    wide = bf(rng, T, hq * 2 * d + 2 * hk * d)[0]
    q = wide[:, :hq * 2 * d].view(T, hq, 2 * d)
    gate, q = q[:, :, d:], q[:, :, :d]
    k, v = wide[:, hq * 2 * d:hq * 2 * d + hk * d], wide[:, hq * 2 * d + hk * d:]
    plain = torch.empty(T, hq, d, device="cuda:0", dtype=torch.bfloat16)
    kv.step(i32([2]), i32([0]), i32([T]), T)
    kv.append(0, k, v)
    kv.attention(0, q, plain, gate=gate)
    kv.append(1, k.contiguous().view(T, hk, d), v.contiguous().view(T, hk, d))
    out = torch.zeros(hq, T + 1, d + 4, device="cuda:0", dtype=torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    kv.attention(1, q.contiguous(), out[:, 1:, 4:].transpose(0, 1), gate=gate.contiguous(),
                 stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out[:, 1:, 4:].transpose(0, 1), plain)
    assert not out[:, 0].any() and not out[:, :, :4].any()
    kv.close()


def test_a_step_in_a_graph_follows_the_lengths(gpu):
    """Map, rotation, append and attention of two layers captured once and replayed while the
    lengths advance on the GPU, eager work between the replays; every replay against a
    twin cache's eager calls."""
    import torch
    import gdn_amd
    rng = np.random.default_rng(16)
    hq, hk, d, n = 8, 2, 128, 5
    twin = [gdn_amd.KV8Cache(2, n, 40, 8, hq, hk, d, 512) for _ in range(2)]
    rope = gdn_amd.Rope(d, 64)
    lens0 = [62, 0, 130, 5, 190]
    slots = i32([3, 1, 4, -1, 0])
    fill = [bf(rng, sum(lens0), hk, d)[0] for _ in range(2)]
    for kv in twin:
        for layer in range(2):
            kv.step(slots, i32([0] * n), i32(lens0), sum(lens0))
            kv.append(layer, *fill)
    ones = i32([1] * n)
    bufs = [dict(lens=i32(lens0), q=torch.zeros(n, hq, d, device="cuda:0", dtype=torch.bfloat16),
                 k=torch.zeros(n, hk, d, device="cuda:0", dtype=torch.bfloat16),
                 v=torch.zeros(n, hk, d, device="cuda:0", dtype=torch.bfloat16)) for _ in twin]
    for b in bufs:
        b["qr"], b["kr"] = torch.zeros_like(b["q"]), torch.zeros_like(b["k"])
        b["out"] = [torch.zeros_like(b["q"]) for _ in range(2)]

    def step(kv, b):
        kv.step(slots, b["lens"], ones, n, 1, lens_out=b["lens"])
        pos = kv.views()["pos"][:n]
        rope.forward(pos, b["q"], b["k"], q_out=b["qr"], k_out=b["kr"])
        for layer in range(2):
            kv.append(layer, b["kr"], b["v"])
            kv.attention(layer, b["qr"], b["out"][layer], window=100 * layer)

    pos_view = twin[0].views()["pos"][:n]

    def step_captured(kv, b):
        kv.step(slots, b["lens"], ones, n, 1, lens_out=b["lens"])
        rope.forward(pos_view, b["q"], b["k"], q_out=b["qr"], k_out=b["kr"])
        for layer in range(2):
            kv.append(layer, b["kr"], b["v"])
            kv.attention(layer, b["qr"], b["out"][layer], window=100 * layer)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step_captured(twin[0], bufs[0])
    for i in range(6):
        x = {w: bf(rng, n, h, d)[0] for w, h in (("q", hq), ("k", hk), ("v", hk))}
        for b in bufs:
            for w in x:
                b[w].copy_(x[w])
        graph.replay()
        step(twin[1], bufs[1])
        torch.cuda.synchronize()
        assert bufs[0]["lens"].tolist() == bufs[1]["lens"].tolist()
        for layer in range(2):
            assert torch.equal(bufs[0]["out"][layer], bufs[1]["out"][layer]), (i, layer)
    assert bufs[0]["lens"].tolist() == [68, 6, 136, 5, 196]
    for kv in twin:
        assert kv.check() == 0
        kv.close()


def test_refused_calls(gpu):
    """Arguments that break the contract raise before anything runs."""
    import torch
    import gdn_amd
    kv = gdn_amd.KV8Cache(1, 3, 9, 4, 8, 2, 128, 64)
    E = gdn_amd.GdnError
    z = torch.zeros
    bf16 = dict(device="cuda:0", dtype=torch.bfloat16)
    q, k = z(4, 8, 128, **bf16), z(4, 2, 128, **bf16)
    with pytest.raises(ValueError):
        kv.append(0, k, k)  # no step: no rows
    kv.tokens = 4
    for call in (lambda: kv.append(0, k, k), lambda: kv.attention(0, q, q)):
        with pytest.raises(E, match="no step planned"):
            call()
    one = i32([0])
    for bad in (lambda: kv.step(one, one, one, 65), lambda: kv.step(one, one, one, -1),
                lambda: kv.step(one, one, one, 4, 5),
                lambda: kv.step(i32([]), i32([]), i32([]), 0),
                lambda: kv.step(i32([0] * 4097), i32([0] * 4097), i32([0] * 4097), 0)):
        with pytest.raises(E):
            bad()
    for bad in (lambda: kv.step(one, one.long(), one, 4), lambda: kv.step(one, i32([0, 0]), one, 4),
                lambda: kv.step(one.cpu(), one, one, 4)):
        with pytest.raises(ValueError):
            bad()
    kv.step(one, one, i32([4]), 4)
    for bad in (lambda: kv.append(1, k, k), lambda: kv.append(-1, k, k),
                lambda: kv.attention(1, q, q), lambda: kv.attention(0, q, q, softcap=-1.0),
                lambda: kv.attention(0, q, q, softcap=float("nan")),
                lambda: kv.attention(0, q, q, window=-1),
                lambda: kv.attention(0, q, q, scale=float("inf")),
                lambda: kv.attention(0, z(4, 8, 132, **bf16)[:, :, 4:], q),
                lambda: kv.attention(0, z(4, 8, 130, **bf16)[:, :, :128], q),
                lambda: kv.append(0, z(4, 260, **bf16)[:, 4:], k),
                lambda: kv.attention(0, q, z(4, 8, 129, **bf16)[:, :, 1:]),
                # heads' planes that run into each other
                lambda: kv.attention(0, q, z(4 * 8 * 128, **bf16).as_strided((4, 8, 128), (128, 256, 1)))):
        with pytest.raises(E):
            bad()
    for bad in (lambda: kv.append(0, k[:3], k), lambda: kv.append(0, k.float(), k),
                lambda: kv.attention(0, q[:3], q), lambda: kv.attention(0, q, q.float()),
                lambda: kv.attention(0, q, q, slopes=z(7, device="cuda:0")),
                lambda: kv.attention(0, q, q, prefix=i32([0, 0])),
                lambda: kv.attention(0, q, q, gate=z(4, 8, 64, **bf16)),
                lambda: kv.gather(0, i32([0, 1]), k, k)):
        with pytest.raises(ValueError):
            bad()
    out = z(3, 2, 128, **bf16) + 1
    kv.gather(0, i32([-1, 9 * 64, 2 ** 31 - 1]), out, None)  # places outside the cache
    assert not out.any()
    kv.close()


def test_steps_without_tokens(gpu):
    import torch
    import gdn_amd
    kv = gdn_amd.KV8Cache(1, 2, 4, 4, 4, 1, 64, 8)
    kv.step(i32([0, 1]), i32([100, 0]), i32([0, 0]), 0)
    e = torch.zeros(0, 4, 64, device="cuda:0", dtype=torch.bfloat16)
    kv.append(0, e[:, :1], e[:, :1])
    kv.attention(0, e, e)
    kv.gather(0, i32([]), e[:, :1], e[:, :1])
    assert kv.views()["owned"].tolist() == [2, 0]
    # tokens at positions that were never appended read as zeros
    kv.step(i32([0]), i32([100]), i32([1]), 3)
    out = torch.ones(64, 1, 64, device="cuda:0", dtype=torch.bfloat16)
    kv.gather(0, i32(range(64)), out, None)
    assert not out.any()
    kv.close()


@pytest.mark.parametrize("hq,hk,dim", [(16, 1, 64), (6, 2, 128), (16, 2, 256)])
def test_few_tokens_beside_prompts(gpu, hq, hk, dim):
    """Rows of 1 to 15 tokens in steps with longer ones, in two tiles where 16 query heads share
    keys, their pages in many pieces; options; a refused row among them."""
    rng = np.random.default_rng(18)
    p = Pair(7, 110, 40, hq=hq, hk=hk, dim=dim, tokens=2700)
    p.step([0, 1, 5], [0, 0, 0], [2300, 300, 64])
    p.append(rng)
    p.step([5, 0, 2, 1, 9, 3], [64, 2300, 0, 300, 0, 0], [1, 15, 20, 9, 3, 2], tokens=52)
    assert p.kv.check() == 1
    p.append(rng)
    p.ref.flags = 0
    p.attention(rng, label="few beside many", gate=True)
    p.attention(rng, label="few beside many, window", window=200, softcap=10.0)
    p.attention(rng, label="few beside many, prefix", prefix=[3, 500, 0, 9, 7, 40], window=30,
                slopes=[0.02 * (h - 2) for h in range(hq)])
    p.step([0, 2], [2315, 20], [1, 18], tokens=30)
    p.append(rng)
    p.attention(rng, label="one beside many")
    p.kv.close()


@pytest.mark.parametrize("n,longest", [(4096, 1), (700, 30)])
def test_attention_of_many_rows(gpu, n, longest):
    rng = np.random.default_rng(19)
    p = Pair(n, 3 * n, 3, hq=2, hk=1, dim=64, tokens=60 * n)
    slots = rng.permutation(n).tolist()
    lens = rng.integers(0, 80, n).tolist()
    p.step(slots, [0] * n, lens)
    p.append(rng)
    ntok = [1] * n
    ntok[n // 2] = longest
    p.step(slots, lens, ntok)
    p.append(rng)
    p.attention(rng, label=f"{n} rows")
    p.kv.close()


@pytest.mark.parametrize("dim", [64, 256])
def test_queries_of_every_size(gpu, dim):
    """A head's dimensions from its largest down to 2^-30 of it, where the largest meet keys of
    zero, so that the small ones make the scores."""
    import torch
    rng = np.random.default_rng(20)
    p = Pair(2, 12, 6, hq=4, hk=2, dim=dim)
    small = torch.arange(dim, device="cuda:0") % 31
    done = []

    def keys(x):
        if not done:
            x[:, :, small < 12] = 0
            x[:, :, small >= 12] *= 64
        done.append(x)

    for step in ([0, 1], [0, 0], [20, 130]), ([0, 1], [20, 130], [20, 1]), ([1, 0], [131, 40], [2, 1]):
        p.step(*step)
        done.clear()
        p.append(rng, change=keys)
        t = p.kv.tokens
        q, _ = bf(rng, t, 4, dim)
        q = (q.float() * 2.0 ** (14 - small)).to(torch.bfloat16)
        out = torch.zeros_like(q)
        p.kv.attention(0, q, out, scale=0.05)
        want, tol = p.ref.attention(num(q), scale=0.05)
        assert np.all(np.abs(num(out) - want) <= tol)
    p.kv.close()


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_infinities_and_nan_in_queries_stay_in_their_heads(gpu, dim):
    import torch
    rng = np.random.default_rng(21)
    p = Pair(2, 12, 6, hq=8, hk=2, dim=dim)
    for step in ([1, 0], [0, 0], [70, 33]), ([0, 1], [33, 70], [1, 3]):  # tiles, chunks
        p.step(*step)
        p.append(rng)
        t = p.kv.tokens
        q, _ = bf(rng, t, 8, dim)
        clean = torch.zeros_like(q)
        p.kv.attention(0, q, clean)
        odd = q.clone()
        want = torch.zeros(t, 8, dtype=torch.bool, device="cuda:0")
        for at, h, value in ((0, 0, "inf"), (1, 3, "nan"), (t - 1, 7, "-inf"), (2, 4, "nan")):
            odd[at, h, (5 * h) % dim] = float(value)
            want[at, h] = True
        out = torch.zeros_like(q)
        p.kv.attention(0, odd, out)
        assert torch.equal(torch.isnan(out).all(2), want)
        assert torch.equal(out[~want], clean[~want])
    p.kv.close()


def test_offsets_past_32_bits(gpu):
    """More than 4 GiB of pages in a layer, the last of them in use."""
    rng = np.random.default_rng(22)
    pages = 17000
    p = Pair(3, pages, pages, hq=16, hk=8, dim=256, tokens=200)
    assert pages * 2 * 8 * 64 * 256 > 2 ** 32 + 2 ** 27
    p.step([0], [(pages - 6) * 64], [0])
    p.step([1, 2], [0, 0], [100, 20])
    p.append(rng)
    p.check_held()
    p.attention(rng, label="far pages")
    p.step([2, 1], [20, 100], [1, 5])
    p.append(rng)
    p.check_held()
    p.attention(rng, label="far pages, tokens")
    p.kv.close()


def test_graphs_that_share_a_cache(gpu):
    """Two captured steps of one cache, of tokens and of prompts, replayed in turn with eager
    steps between them; every replay against a twin cache's eager calls."""
    import torch
    import gdn_amd
    rng = np.random.default_rng(23)
    hq, hk, d = 8, 2, 64
    twin = [gdn_amd.KV8Cache(1, 6, 60, 20, hq, hk, d, 256) for _ in range(2)]
    plans = [dict(slots=i32([4, 0]), tok=i32([1, 2]), T=4, most=2),
             dict(slots=i32([1, 5, 3]), tok=i32([40, 7, 0]), T=60, most=40)]
    bufs = []
    for kv in twin:
        mine = []
        for pl in plans:
            b = {w: torch.zeros(pl["T"], h, d, device="cuda:0", dtype=torch.bfloat16)
                 for w, h in (("q", hq), ("k", hk), ("v", hk), ("out", hq))}
            b["lens"] = torch.zeros_like(pl["slots"])
            mine.append(b)
        bufs.append(mine)

    def step(kv, pl, b):
        kv.step(pl["slots"], b["lens"], pl["tok"], pl["T"], pl["most"], lens_out=b["lens"])
        kv.append(0, b["k"], b["v"])
        kv.attention(0, b["q"], b["out"])

    for kv, mine in zip(twin, bufs):  # both once before the capture
        for pl, b in zip(plans, mine):
            step(kv, pl, b)
    torch.cuda.synchronize()
    graphs = []
    for pl, b in zip(plans, bufs[0]):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(twin[0], pl, b)
        graphs.append(g)
    for i in range(8):
        which = (0, 1, 1, 0, 0, 1, 0, 1)[i]
        for w, h in (("q", hq), ("k", hk), ("v", hk)):
            x = bf(rng, plans[which]["T"], h, d)[0]
            for mine in bufs:
                mine[which][w].copy_(x)
        if i == 4:  # an eager step between the replays
            step(twin[0], plans[which], bufs[0][which])
        else:
            graphs[which].replay()
        step(twin[1], plans[which], bufs[1][which])
        torch.cuda.synchronize()
        a, b = bufs[0][which], bufs[1][which]
        assert a["lens"].tolist() == b["lens"].tolist()
        used = int(plans[which]["tok"].sum())
        assert torch.equal(a["out"][:used], b["out"][:used]), i
    for kv in twin:
        assert kv.check() == 0
        kv.close()


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 30, 1000])
def test_windows_longer_than_any_row(gpu, window):
    import torch
    rng = np.random.default_rng(24)
    p = Pair(2, 12, 6, hq=4, hk=2, dim=64)
    for step in ([1, 0], [0, 0], [70, 33]), ([0, 1], [33, 70], [1, 3]):  # tiles, chunks
        p.step(*step)
        p.append(rng)
        q, _ = bf(rng, p.kv.tokens, 4, 64)
        whole, out = torch.zeros_like(q), torch.zeros_like(q)
        p.kv.attention(0, q, whole)
        p.kv.attention(0, q, out, window=window)
        assert torch.equal(whole, out)
    p.kv.close()


def test_eager_calls_behind_another_steps_replay(gpu):
    """Append and attention under one step's bounds where a replayed graph has planned another:
    its rows that fit are worked on, nothing outside the tensors or the pages is touched."""
    import torch
    import gdn_amd
    rng = np.random.default_rng(25)
    hq, hk, d = 4, 2, 64
    kv = gdn_amd.KV8Cache(1, 8, 40, 10, hq, hk, d, 256)
    wide = dict(slots=i32([0, 1, 2]), lens=i32([0, 0, 0]), tok=i32([9, 30, 80]))
    kv.step(wide["slots"], wide["lens"], wide["tok"], 120, 80)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv.step(wide["slots"], wide["lens"], wide["tok"], 120, 80)
    # rows of a step that releases the slots, so that nothing behind its n may be followed
    kv.step(i32([5, 4, 3, 2, 1, 0]), i32([70, 0, 0, 0, 0, 0]), i32([2, 1, 1, 0, 0, 0]), 20, 20)
    graph.replay()  # three rows, of which the first fits 20 tokens, and none 8 rows
    q, k, v = (bf(rng, 24, h, d)[0] for h in (hq, hk, hk))
    out = torch.full_like(q, 7.0)
    kv.append(0, k[:20], v[:20])
    kv.attention(0, q[:20], out[:20])
    ko = torch.zeros(9, hk, d, device="cuda:0", dtype=torch.bfloat16)
    kv.gather(0, kv.views()["map"][:9].contiguous(), ko, None)
    torch.cuda.synchronize()
    assert (ko - k[:9]).abs().max() <= k.abs().max() * 2.0 ** -4
    assert torch.all(out[9:] == 7.0) and not torch.any(out[:9] == 7.0)
    # fewer rows on the GPU than the bounds say
    alone = i32([6]), i32([0]), i32([1])
    kv.step(*alone, 1, 1)
    torch.cuda.synchronize()
    one = torch.cuda.CUDAGraph()
    with torch.cuda.graph(one):
        kv.step(*alone, 1, 1)
    kv.step(i32(range(8)), i32([0] * 8), i32([3] * 8), 24, 3)
    one.replay()
    out.fill_(7.0)
    kv.append(0, k, v)
    kv.attention(0, q, out)
    torch.cuda.synchronize()
    assert torch.all(out[1:] == 7.0) and not torch.any(out[:1] == 7.0)
    kv.close()


@pytest.mark.parametrize("slope,scale", [(1.0, 0.125), (3e6, 0.125), (0.5, 1e-13), (0.25, -0.1),
                                         (1e-9, 4.0)])
def test_distance_terms_of_every_size(gpu, slope, scale):
    """Slopes and scales either side of where the term starts the accumulators; a page of zeros
    and queries of zeros, whose scores have no size of their own."""
    rng = np.random.default_rng(26)
    p = Pair(3, 12, 6, hq=4, hk=2, dim=64)
    p.step([1], [0], [64])
    p.append(rng, change=lambda x: x.zero_())
    p.step([1, 0], [64, 0], [70, 33])
    p.append(rng)
    p.attention(rng, label="slopes", scale=scale, slopes=[slope, -slope, 0.0, slope / 3])
    p.attention(rng, label="zero queries", std=0.0, scale=scale, slopes=[slope, 0.1, 0.0, slope / 3])
    p.kv.close()

"""Rotary positions (gdn_rope_forward) against the formula in 64 bits.

Tolerance: the result's own rounding (bf16 2^-8, f32 2^-24 of it) and, of its pair's size,
2^-19: the angle's fraction in f32 (2^-25 turns, 2^-22 rad), sine and cosine (2^-22), three
roundings of the turn, and with a norm a sum of up to 512 squares in a tree of 14 steps under
a root, and three roundings."""
import numpy as np
import pytest

from gdn_testlib import say
from kv8_testlib import frequencies, rope

pytestmark = pytest.mark.gpu

SCALED = dict(yarn=dict(factor=16.0, original=4096.0, fast=32.0, slow=1.0),
              bands=dict(factor=8.0, original=8192.0, fast=4.0, slow=1.0),
              linear=dict(factor=4.0), none={})


def _check(got, want, size, f32):
    err = np.abs(got.double().cpu().numpy() - want)
    tol = (2.0 ** -24 if f32 else 2.0 ** -8) * np.abs(want) + 2.0 ** -19 * size
    say("rope", f"worst error / tolerance {float((err / np.maximum(tol, 1e-300)).max()):.3f}")
    assert np.all(err <= tol)


@pytest.mark.parametrize("hq,hk,dim,rot", [(16, 2, 256, 64), (4, 4, 64, 64), (3, 0, 96, 46),
                                           (5, 1, 128, 2), (1, 1, 8, 8), (9, 2, 512, 512),
                                           (2, 3, 192, 0), (33, 8, 80, 80)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("f32", [False, True])
def test_rotation(gpu, hq, hk, dim, rot, interleaved, f32):
    import torch
    import gdn_amd
    rng = np.random.default_rng(hq + dim + rot)
    dt = torch.float32 if f32 else torch.bfloat16
    T = 37
    pos = rng.integers(0, 300000, T)
    pos[:3] = 0, 1, -1
    q, k = (torch.from_numpy(rng.standard_normal((T, h, dim)).astype(np.float32)).to(dt).cuda()
            for h in (hq, hk))
    w = [torch.from_numpy((1 + 0.2 * rng.standard_normal(dim)).astype(np.float32)).bfloat16().cuda()
         for _ in range(2)]
    pd = torch.tensor(pos, dtype=torch.int32, device="cuda:0")
    for scaling, kw in SCALED.items():
        say("rope", hq, hk, dim, rot, interleaved, f32, scaling)
        r = gdn_amd.Rope(dim, rot, 1.0e4, interleaved, scaling, **kw)
        freq = frequencies(rot, 1.0e4, scaling, **kw)
        mag = 0.1 * np.log(kw["factor"]) + 1 if scaling == "yarn" else 1.0
        for norm in (False, True):
            qo, ko = torch.full_like(q, 5.0), torch.full_like(k, 5.0)
            r.forward(pd, q, k if hk else None, q_out=qo, k_out=ko if hk else None,
                      q_norm_w=w[0] if norm else None, k_norm_w=w[1] if norm and hk else None,
                      eps=1e-5)
            for x, o, ww in ((q, qo, w[0]), (k, ko, w[1]))[:2 if hk else 1]:
                want, size = rope(x.double().cpu().numpy(), pos, freq, interleaved, mag,
                                  ww.double().cpu().numpy() if norm else None, 1e-5)
                _check(o, want, size, f32)
        r.close()


def test_far_positions(gpu):
    """Positions up to 2^31 - 1: the angle is formed in 64 bits."""
    import torch
    import gdn_amd
    rng = np.random.default_rng(3)
    pos = np.array([2 ** 31 - 1, 2 ** 30 + 1, 999_999, 123_456_789])
    q = torch.from_numpy(rng.standard_normal((4, 2, 128)).astype(np.float32)).cuda()
    out = torch.empty_like(q)
    r = gdn_amd.Rope(128, base=1.0e7)
    r.forward(torch.tensor(pos, dtype=torch.int32, device="cuda:0"), q, q_out=out)
    # 2^-53 of 2^31 radians is 2^-22: twice, for the two ways of forming the product
    want, size = rope(q.double().cpu().numpy(), pos, frequencies(128, 1.0e7))
    err = np.abs(out.double().cpu().numpy() - want)
    assert np.all(err <= 2.0 ** -24 * np.abs(want) + (2.0 ** -19 + 2.0 ** -21) * size)
    r.close()


def test_in_place_views_and_the_way_back(gpu):
    """Columns of a wider tensor in place, heads first, many tokens; the inverse is the
    transpose: <turn(x), y> = <x, inverse(y)>, and differences of the turn are its own."""
    import torch
    import gdn_amd
    rng = np.random.default_rng(4)
    T, h, d = 700, 3, 64
    r = gdn_amd.Rope(d, 48, 1.0e4)
    pos = torch.arange(5, 5 + T, dtype=torch.int32, device="cuda:0")
    wide = torch.from_numpy(rng.standard_normal((T, h, 2 * d)).astype(np.float32)).bfloat16().cuda()
    x = wide[:, :, :d]
    keep = wide.clone()
    want = torch.empty(T, h, d, device="cuda:0", dtype=torch.bfloat16)
    r.forward(pos, x, q_out=want)
    planes = torch.zeros(h, T, d, device="cuda:0", dtype=torch.bfloat16)
    r.forward(pos, x, q_out=planes.transpose(0, 1))
    r.forward(pos, x)
    assert torch.equal(x, want) and torch.equal(planes.transpose(0, 1), want)
    assert torch.equal(wide[:, :, d:], keep[:, :, d:])
    a, b = (torch.from_numpy(rng.standard_normal((T, h, d)).astype(np.float32)).cuda()
            for _ in range(2))
    ta, ib, diff = torch.empty_like(a), torch.empty_like(a), torch.empty_like(a)
    r.forward(pos, a, q_out=ta)
    r.forward(pos, b, q_out=ib, inverse=True)
    # both products sum T h d terms that are each off by some 2^-20
    left, right = (ta.double() * b.double()).sum(), (a.double() * ib.double()).sum()
    assert abs(float(left - right)) <= 2.0 ** -18 * float((a.double().abs() * ib.double().abs()).sum())
    r.forward(pos, a + b, q_out=diff)
    bound = 2.0 ** -18 * (a.abs() + b.abs()).amax()
    tb = torch.empty_like(b)
    r.forward(pos, b, q_out=tb)
    assert float((diff - ta - tb).abs().max()) <= 2 * float(bound)
    r.close()


@pytest.mark.parametrize("dim,rot,interleaved", [(64, 32, False), (64, 32, True), (96, 46, False)])
@pytest.mark.parametrize("T", [3, 600, 2100])
def test_what_does_not_turn_keeps_its_bits(gpu, dim, rot, interleaved, T):
    """Infinities and NaN among the dimensions behind rotary_dim and in tokens at negative
    positions stay where they are; a turned pair takes only its own."""
    import torch
    import gdn_amd
    inf, nan = float("inf"), float("nan")
    x = torch.randn(T, 3, dim, device="cuda:0").bfloat16()
    x[0, 1, rot], x[0, 2, rot + 3], x[1, 0, 0], x[1, 1, dim - 1] = inf, nan, nan, -inf
    x[2, 0, 1] = nan
    pos = torch.arange(T, dtype=torch.int32, device="cuda:0")
    pos[1] = -1
    out = torch.empty_like(x)
    r = gdn_amd.Rope(dim, rot, 1.0e4, interleaved)
    r.forward(pos, x, q_out=out)
    bits = lambda t: t.view(torch.int16)  # noqa: E731
    assert torch.equal(bits(out[:, :, rot:]), bits(x[:, :, rot:]))
    assert torch.equal(bits(out[1]), bits(x[1]))
    bad = torch.isnan(out[:, :, :rot])
    bad[1] = False
    want = torch.zeros_like(bad)
    want[2, 0, [0, 1] if interleaved else [1, 1 + rot // 2]] = True
    assert torch.equal(bad, want)
    r.close()


def test_refused_calls(gpu):
    import torch
    import gdn_amd
    E = gdn_amd.GdnError
    r = gdn_amd.Rope(64, 32)
    pos = torch.zeros(4, dtype=torch.int32, device="cuda:0")
    q = torch.zeros(4, 2, 64, device="cuda:0", dtype=torch.bfloat16)
    w = torch.ones(64, device="cuda:0", dtype=torch.bfloat16)
    wide = torch.zeros(4, 2, 72, device="cuda:0", dtype=torch.bfloat16)
    for bad in (lambda: r.forward(pos, wide[:, :, 4:68]), lambda: r.forward(pos, q, eps=-1.0),
                lambda: r.forward(pos, q, q_norm_w=w, inverse=True),
                lambda: r.forward(pos, torch.zeros(4, 2, 68, device="cuda:0",
                                                   dtype=torch.bfloat16)[:, :, :64]),
                lambda: r.forward(pos, q[:, :0]),
                lambda: r.forward(pos, q, q_out=torch.zeros(
                    512, device="cuda:0", dtype=torch.bfloat16).as_strided((4, 2, 64), (64, 128, 1)))):
        with pytest.raises(E):
            bad()
    for bad in (lambda: r.forward(pos[:3], q), lambda: r.forward(pos, q, q.float()),
                lambda: r.forward(pos.long(), q), lambda: r.forward(pos, q.half()),
                lambda: r.forward(pos, q, k_out=q), lambda: r.forward(pos, q, q_norm_w=w[:32]),
                lambda: r.forward(pos.cpu(), q)):
        with pytest.raises(ValueError):
            bad()
    r.forward(pos[:0], q[:0])
    r.close()


@pytest.mark.parametrize("hq,hk,dim,rot", [(16, 2, 256, 64), (3, 0, 96, 46), (9, 2, 512, 512),
                                           (33, 8, 80, 80), (1, 1, 8, 8)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("f32", [False, True])
def test_long_steps_are_their_tokens(gpu, hq, hk, dim, rot, interleaved, f32):
    """2,051 tokens in one call, in place and not, against calls of 64 tokens and less."""
    import torch
    import gdn_amd
    T, dt = 2051, torch.float32 if f32 else torch.bfloat16
    g = torch.Generator(device="cuda:0").manual_seed(dim + rot)
    q, k = (torch.randn(T, h, dim, device="cuda:0", generator=g).to(dt) for h in (hq, hk))
    w = torch.randn(dim, device="cuda:0", generator=g).bfloat16()
    pos = torch.randint(-1, 100000, (T,), device="cuda:0", generator=g, dtype=torch.int32)
    r = gdn_amd.Rope(dim, rot, 1.0e4, interleaved)

    def turn(a, b, qo, ko):
        r.forward(pos[a:b], q[a:b], k[a:b] if hk else None, q_out=qo[a:b],
                  k_out=ko[a:b] if hk else None, q_norm_w=w, k_norm_w=w if hk else None, eps=1e-5)

    whole, parts = ([torch.full_like(x, 3.0) for x in (q, k)] for _ in range(2))
    turn(0, T, *whole)
    for a in range(0, T, 64):
        turn(a, min(a + 64, T), *parts)
    turn(0, T, q, k)
    for a, b, c in zip(whole, parts, (q, k)):
        assert torch.equal(a, b) and torch.equal(a, c)
    r.close()

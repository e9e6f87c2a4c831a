"""How many bits of h = silu(gate) * up the experts' kernels keep.

The last rounding to bf16 hides what h lost, so a token here takes two experts whose
h differ by about one part in a hundred, with weights 1 and -1: the result is their
small difference. Only a few of the inner columns are there (the others have a gate of
zeros, so that their h is zero), and a row of down takes one of them in a group: no
sum is long enough to hide the rounding either.
"""
import pytest
import torch

from test_gpu_moe import BF, DEV, HALF_BF, HALF_F32, full

import gdn_amd

pytestmark = pytest.mark.gpu

HALF_F16 = 2.0 ** -11


def _expert_pair(g, hidden, inner, spread):
    """((gate, up, down) of expert A, of expert B)."""
    live = torch.arange(inner // 64) * 64 + torch.randint(0, 64, (inner // 64,), generator=g)

    def mat(n, k):
        w = torch.randint(-2 ** 31, 2 ** 31, (n, k // 8), dtype=torch.int32, generator=g)
        s = ((torch.rand(n, k // 64, generator=g) + 0.5) * 0.125).to(BF)
        return w, s, (-7.5 * s.float()).to(BF)

    gate, up = mat(inner, hidden), mat(inner, hidden)
    there = torch.zeros(inner, dtype=torch.bool)
    there[live] = True
    for t in gate[1:]:
        t[~there] = 0
    if spread:  # one column with far larger weights: it alone sets the layer's bound
        for t in gate[1:]:
            t[live[0]] *= 2.0 ** spread
    # down: 8 s - 8 s = 0 everywhere but at the live columns, where it is s
    w = torch.full((hidden, inner // 8), -0x77777778, dtype=torch.int32)  # every nibble 8
    for c in live.tolist():
        w[:, c // 8] += 1 << (4 * (c % 8))
    pick = torch.randint(1 if spread else 0, inner // 64, (hidden,), generator=g)
    s = torch.zeros(hidden, inner // 64, dtype=BF)
    s[torch.arange(hidden), pick] = 1.0
    down = (w, s, (-8.0 * s.float()).to(BF))
    near = (gate[0], (gate[1].float() * (1 + 2.0 ** -6)).to(BF), gate[2])
    return (gate, up, down), (near, up, down)


@pytest.mark.parametrize("T,hidden,inner,pairs", [
    (6, 256, 512, 2),        # very few entries
    (40, 1024, 256, 40),     # the weights' stream, stages in two parts
    (40, 256, 128, 40),      # and in one
    (60, 256, 256, 4),       # tiles of 16 rows
    (100, 256, 128, 4),      # and of 32
    (3300, 1024, 384, 2),    # of 64, down's input in LDS
    (3300, 1024, 640, 2),    # and in stages
])
@pytest.mark.parametrize("spread", [0, 12])
def test_h_keeps_eleven_bits(gpu, T, hidden, inner, pairs, spread):
    g = torch.Generator().manual_seed(T + inner + spread)
    made = [_expert_pair(g, hidden, inner, spread) for _ in range(pairs)]
    experts = [e for p in made for e in p]
    part = tuple(tuple(torch.stack([e[m][t] for e in experts]).to(DEV) for t in range(3))
                 for m in range(3))
    moe = gdn_amd.MoE(hidden, inner, [part])
    x = torch.zeros(T, hidden)
    at = torch.randperm(hidden, generator=g)[:8]
    x[:, at] = torch.randn(T, 8, generator=g)
    x = x.to(BF)
    pair = torch.randint(0, pairs, (T,), generator=g)
    ids = torch.stack([2 * pair, 2 * pair + 1], 1).to(torch.int32)
    wt = torch.tensor([1.0, -1.0]).expand(T, 2).contiguous()
    out = torch.empty(T, hidden, device=DEV, dtype=BF)
    ws = moe.workspace(T, 2)
    ws.fill_(255)
    moe.forward(x.to(DEV), ids.to(DEV), wt.to(DEV), out, ws)
    torch.cuda.synchronize()
    out = out.cpu().double()
    ref, tol = torch.zeros(T, hidden, dtype=torch.float64), torch.zeros(T, hidden, dtype=torch.float64)
    for e, (mg, mu, md) in enumerate(experts):
        rows = (ids == e).any(1)
        sign = 1.0 if e % 2 == 0 else -1.0
        xr = x[rows].double()
        wg, wu, wd = full(*mg), full(*mu), full(*md)

        def err(m, v):
            # s (128 X + sum v q) + (b - 128 s) X in f32: every term of a group enters
            # 64 / 16 + 2 adds in the group and one for each group
            s, b = m[1].double().abs(), m[2].double().abs()
            mag = (271 * s + b).repeat_interleave(64, 1)
            return (v.shape[1] // 64 + 8) * HALF_F32 * (v.abs() @ mag.t())

        a, u = xr @ wg.t(), xr @ wu.t()
        h = a * torch.sigmoid(a) * u
        ea, eu = err(mg, xr), err(mu, xr)
        eh = 1.1 * ea * u.abs() + a.abs() * eu + ea * eu + (HALF_F16 + 8 * HALF_F32) * h.abs()
        # the smallest numbers of h's f16: half a step is 2^-25 of a power of two that is
        # within 2^4 of 2^-15 times the product of the gate's and up's largest row sums of
        # |w| (and 2^-8 of |s| more) and the largest |x|, squared
        top = 2.0 ** -35 * xr.abs().amax(1, True) ** 2
        eh += top * wg.abs().sum(1).max() * wu.abs().sum(1).max() * (h != 0)
        ref[rows] += sign * (h @ wd.t())
        # down: a group's sum is one product, of 11 bits each, and X is h: exact. Its scale,
        # the parts of X and the groups' sum are at most 8 roundings of values below
        # 1033 s |h|
        tol[rows] += eh @ wd.abs().t() + 8 * HALF_F32 * 1033 * (h.abs() @ wd.abs().t())
    tol += HALF_F32 * 4 * ref.abs()
    # rows of long prompts pass to the sum in 11 bits of the row's own power of two
    hs = torch.zeros(T, 1, dtype=torch.float64)
    for e, (mg, mu, md) in enumerate(experts):
        rows = (ids == e).any(1)
        a, u = x[rows].double() @ full(*mg).t(), x[rows].double() @ full(*mu).t()
        y = (a * torch.sigmoid(a) * u) @ full(*md).t()
        if T > 3000 and inner <= 512:
            tol[rows] += HALF_F16 * y.abs()
            hs[rows] = torch.maximum(hs[rows], (a * torch.sigmoid(a) * u).abs().amax(1, True))
    tol += 2 * 2.0 ** -37 * hs
    tol += HALF_BF * (ref.abs() + tol)
    d = (out - ref).abs()
    assert (d <= tol).all(), float((d / tol.clamp_min(1e-30)).max())
    assert (ref != 0).any(1).float().mean() > 0.9


@pytest.mark.parametrize("T,hidden,inner,E", [(6, 256, 256, 2), (40, 256, 256, 40), (60, 256, 256, 4),
                                              (1700, 2048, 384, 2), (1700, 2048, 640, 2)])
@pytest.mark.parametrize("which", ["gate", "down"])
def test_weights_that_cancel(gpu, T, hidden, inner, E, which):
    """All weights of a matrix are 8 s - 8 s = 0, but for a group of about 2^-40: what the
    sums leave of the zeros is far above those, and stays within the sums' error."""
    g = torch.Generator().manual_seed(T + inner)

    def mat(n, k, zeros):
        w = torch.randint(-2 ** 31, 2 ** 31, (E, n, k // 8), dtype=torch.int32, generator=g)
        s = ((torch.rand(E, n, k // 64, generator=g) + 0.5) * k ** -0.5 / 4.8).to(BF)
        b = (-7.5 * s.float()).to(BF)
        if zeros:
            w[:, :, 8:] = -0x77777778  # every nibble 8
            s[:, :, 1:], b[:, :, 1:] = 1.0, -8.0
            s[:, :, 0] *= 2.0 ** -40
            b[:, :, 0] *= 2.0 ** -40
        return w, s, b

    part = (mat(inner, hidden, which == "gate"), mat(inner, hidden, False),
            mat(hidden, inner, which == "down"))
    moe = gdn_amd.MoE(hidden, inner, [tuple(tuple(t.to(DEV) for t in m) for m in part)])
    x = torch.randn(T, hidden, generator=g).to(BF)
    ids = torch.rand(T, E, generator=g).argsort(1)[:, :2].to(torch.int32)
    out = torch.empty(T, hidden, device=DEV, dtype=BF)
    moe.forward(x.to(DEV), ids.to(DEV), torch.ones(T, 2, device=DEV), out, moe.workspace(T, 2))
    out = out.cpu().double()
    tol = torch.zeros(T, hidden, dtype=torch.float64)
    for e in range(E):
        rows = (ids == e).any(1)
        xr = x[rows].double()
        (wg, wu, wd) = (full(*(t[e] for t in m)) for m in part)
        # as in test_h_keeps_eleven_bits; the magnitudes of a group add up to 271 s + |b|,
        # of down's f16 numbers 2063 s + |b|
        ea = (hidden // 64 + 8) * HALF_F32 * xr.abs().sum(1, True) * (271 + 8)
        a, u = (xr @ wg.t()).abs() + (ea if which == "gate" else 0), (xr @ wu.t()).abs()
        h = 1.001 * a * (u + ea)
        ey = (inner // 64 + 8) * HALF_F32 * h.sum(1, True) * (2063 + 8) if which == "down" else 0
        tol[rows] += 1.01 * (h @ wd.abs().t() + ey)
    assert (out.abs() <= tol).all()

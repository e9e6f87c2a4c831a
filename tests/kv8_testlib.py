"""The 8-bit paged cache in plain numpy, 64 bits: pages, what is held, attention, rotary
positions. Written from the operators' definitions (include/gdn.h)."""
import math

import numpy as np

PAGE, E_MIN, E_MAX = 64, -40, 56
# e4m3's numbers >= 0 in order: 8 subnormals, then 8 of each exponent but the last pattern
GRID = np.array([m * 2.0 ** -9 for m in range(8)] +
                [(8 + m) * 2.0 ** (e - 3) for e in range(-6, 9) for m in range(8)][:-1])


def hold(x):
    """Values of one page [tokens, heads, dim] -> what is held of them."""
    out = np.empty_like(x)
    for h in range(x.shape[1]):
        a = np.abs(x[:, h])
        fin = np.isfinite(a)
        most = a[fin].max() if fin.any() else 0.0
        e = E_MIN
        while most > 448 * 2.0 ** e and e < E_MAX:
            e += 1
        y = np.where(fin, a, 0.0) / 2.0 ** e
        hi = np.minimum(np.searchsorted(GRID, y), len(GRID) - 1)
        lo = np.maximum(hi - 1, 0)
        up, down = GRID[hi] - y, y - GRID[lo]
        pick = np.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
        out[:, h] = np.copysign(GRID[pick] * 2.0 ** e, x[:, h])
        out[:, h][~fin] = np.nan
    return out


class Ref:
    """Tables, lengths and held values of every slot (one layer)."""

    def __init__(self, num_slots, num_pages, max_pages, heads, dim):
        self.free = list(range(num_pages - 1, -1, -1))
        self.table = [[] for _ in range(num_slots)]
        self.num_pages, self.max_pages = num_pages, max_pages
        self.held = {}  # slot -> (k, v) [tokens, heads, dim]
        self.unknown = set()
        self.heads, self.dim = heads, dim
        self.flags = 0

    def step(self, slots, lens, ntok, tokens, max_row=None):
        """Returns (cu, pos, map, new lengths); the plan stays in self.plan."""
        max_row = tokens if not max_row else max_row
        n, top = len(slots), len(self.table)
        cu, ok, seen = [0], [], set()
        for s, a, b in zip(slots, lens, ntok):
            cu.append(cu[-1] + (min(max(b, 0), tokens + 1) if s >= 0 else 0))
            good = 0 <= s < top
            if s >= top:
                self.flags |= 1
            if good and s in seen:
                self.flags |= 2
                good = False
            seen.add(s)
            if s >= 0 and (a < 0 or b < 0 or b > max_row or a + b > self.max_pages * PAGE or
                           (good and cu[-1] > tokens)):
                self.flags |= 4
                good = False
            ok.append(good)
        need = [-(-(a + b) // PAGE) for a, b in zip(lens, ntok)]
        for i, s in enumerate(slots):
            while ok[i] and len(self.table[s]) > need[i]:
                self.free.append(self.table[s].pop())
        budget = len(self.free)
        for i, s in enumerate(slots):
            grow = need[i] - len(self.table[s]) if ok[i] else 0
            if grow > 0:
                budget -= grow
                if budget < 0:
                    self.flags |= 8
                    ok[i] = False
                else:
                    self.table[s] += [self.free.pop() for _ in range(grow)]
        pos, where = np.full(tokens, -1, np.int32), np.full(tokens, -1, np.int32)
        for i, s in enumerate(slots):
            for t in range(cu[i], min(cu[i + 1], tokens)):
                if ok[i]:
                    pos[t] = lens[i] + t - cu[i]
                    where[t] = self.table[s][pos[t] // PAGE] * PAGE + pos[t] % PAGE
        self.plan = [(s, a, b if o else 0, c) for s, a, b, c, o in zip(slots, lens, ntok, cu, ok)]
        self.end = cu[-1]
        out = [a + b if o else a for a, b, o in zip(lens, ntok, ok)]
        return cu, pos, where, out

    def append(self, k, v):
        for s, a, b, c in self.plan:
            if b == 0:
                continue
            old = self.held.get(s)
            if a > (0 if old is None else len(old[0])):
                # positions that were never appended: their page holds anything
                self.unknown.add(s)
            new = []
            for z, x in enumerate((k, v)):
                full = np.zeros((a + b, self.heads, self.dim))
                if old is not None:
                    m = min(a, len(old[z]))
                    full[:m] = old[z][:m]
                full[a:] = x[c:c + b]
                for t in range(a // PAGE * PAGE, a + b, PAGE):
                    full[t:t + PAGE] = hold(full[t:t + PAGE])
                new.append(full)
            self.held[s] = tuple(new)

    def attention(self, q, scale=0.0, softcap=0.0, window=0, slopes=None, prefix=None, gate=None):
        """(out, tolerance) [end, Hq, dim] of the planned tokens.

        The tolerance adds what the contract allows: bf16's half step 2^-8 of the result; the
        weights' half step 2^-11 of sum p|v| (f16), or 2^-25 of each |v| below f16's normal
        numbers; f32 sums of D products in a score (D 2^-24 of sum |q k|), of f32 scores
        (2^-22 of their size, of the cap where there is one, of the distance term) and q's
        dimensions below 2^-13 of its head's largest to 2^-21 of that, each moving weights by
        twice its size; f32 sums over the keys, n 2^-24 of sum p|v|; some
        roundings of f32 in the norm and gate (2^-20)."""
        Hq = q.shape[1]
        G = Hq // self.heads
        scale = scale or 1.0 / math.sqrt(self.dim)
        out, tol = np.zeros((self.end, Hq, self.dim)), np.zeros((self.end, Hq, self.dim))
        for i, (s, a, b, c) in enumerate(self.plan):
            for t in range(b):
                p = a + t
                keys = np.arange(a + b)
                see = keys <= p
                if window:
                    see &= keys > p - window
                if prefix is not None:
                    see |= keys < prefix[i]
                for h in range(Hq):
                    k, v = (x[:a + b][see, h // G] for x in self.held[s])
                    qk = q[c + t, h] * k
                    sc = qk.sum(1) * scale
                    err = np.abs(qk).sum(1) * abs(scale) * self.dim * 2.0 ** -24
                    err += 2.0 ** -22 * np.abs(sc)
                    most = np.abs(q[c + t, h]).max()
                    low = np.abs(q[c + t, h]) < 2.0 ** -13 * most
                    err += 2.0 ** -21 * most * abs(scale) * np.abs(k[:, low]).sum(1)
                    if softcap:
                        sc = softcap * np.tanh(sc / softcap)
                        err += 2.0 ** -21 * softcap
                    if slopes is not None:
                        far = slopes[h] * (p - keys[see])
                        sc = sc - far
                        err += 2.0 ** -22 * np.abs(far)
                    w = np.exp(sc - sc.max())
                    w /= w.sum()
                    o, av = w @ v, w @ np.abs(v)
                    e = (2.0 ** -11 + 2 * err.max() + (len(k) + 16) * 2.0 ** -24 + 2.0 ** -20) * av
                    e = e + 2.0 ** -25 * np.abs(v).sum(0) + 2.0 ** -8 * np.abs(o)
                    if gate is not None:
                        g = 1 / (1 + np.exp(-gate[c + t, h]))
                        o, e = o * g, e * g
                    out[c + t, h], tol[c + t, h] = o, e * (1 + 2.0 ** -7)
        return out, tol


def frequencies(rot, base, scaling="none", factor=1.0, original=0.0, fast=32.0, slow=1.0):
    i = np.arange(rot // 2, dtype=np.float64)
    f = base ** (-2.0 * i / max(rot, 1))
    if scaling == "linear":
        return f / factor
    if scaling == "yarn":
        lo, hi = (rot * math.log(original / (2 * math.pi * b)) / (2 * math.log(base))
                  for b in (fast, slow))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), rot - 1)
        r = np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
        return f / factor * r + f * (1 - r)
    if scaling == "bands":
        m = np.clip((original * f / (2 * math.pi) - slow) / (fast - slow), 0, 1)
        return f / factor * (1 - m) + f * m
    return f


def rope(x, pos, freq, interleaved=False, magnitude=1.0, w=None, eps=1e-6, inverse=False):
    """(out, size of each element's pair) of x [tokens, heads, dim]."""
    rot = 2 * len(freq)
    y = x.astype(np.float64)
    if w is not None:
        y = np.where((pos >= 0)[:, None, None],
                     y / np.sqrt((y * y).mean(2, keepdims=True) + eps) * w, y)
    ang = (pos[:, None] * freq)[:, None, :] * (-1 if inverse else 1)
    c, s = magnitude * np.cos(ang), magnitude * np.sin(ang)
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else \
        (slice(0, rot // 2), slice(rot // 2, rot))
    out, size = y.copy(), np.abs(y)
    out[..., a], out[..., b] = y[..., a] * c - y[..., b] * s, y[..., a] * s + y[..., b] * c
    size[..., a] = size[..., b] = abs(magnitude) * np.hypot(y[..., a], y[..., b])
    stay = pos < 0
    out[stay], size[stay] = y[stay], np.abs(y[stay])
    return out, size

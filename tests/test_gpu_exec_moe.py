"""The executor with sparse MLP halves (gdn_exec_set_moe) against the same
public calls made one by one, bit for bit: a stack of GatedDeltaNet, attention,
GatedDeltaNet layers, the first two with an MLP half of routed experts and a
gated shared one. Decode steps run launch by launch and as replayed graphs."""
import numpy as np
import pytest
import torch

import gdn_amd
from gdn_testlib import O, DV, conv_dim, dev, quantize_w4
from test_gpu_moe import Experts

pytestmark = pytest.mark.gpu

HK, HV, HIDDEN, VOCAB, INNER, E, TOPK = 8, 16, 512, 2048, 128, 24, 4
HQ, HKV, THETA, ROT, EPS = 8, 2, 1.0e7, 64, 1e-6
NQ, NKV = HQ * 512, HKV * 256
MAX_BATCH, MAX_PROMPT = 4, 160


def _bfw(rng, n):
    return dev(O.f32_to_bf16((1 + 0.1 * rng.standard_normal(n)).astype(np.float32)))


def _ql(rng, k, rows, std=0.05):
    return gdn_amd.QLinear(k, [(dev(w.view(np.int32)), dev(s), dev(b)) for w, s, b in
                               (quantize_w4(rng.standard_normal((n, k)) * std) for n in rows)])


class Model:
    def __init__(self, seed):
        rng = np.random.default_rng(seed)
        d = conv_dim(HK, HV)
        self.gdn = [dict(i=_ql(rng, HIDDEN, (d, HV * DV, HV, HV)), o=_ql(rng, HV * DV, (HIDDEN,), 0.03),
                         A_log=dev(rng.uniform(0.0, np.log(16.0), HV).astype(np.float32)),
                         dt=dev((rng.standard_normal(HV) * 0.1).astype(np.float32)),
                         conv=dev(O.f32_to_bf16((rng.standard_normal((d, 4)) * 0.25).astype(np.float32))),
                         nw=_bfw(rng, DV)) for _ in range(2)]
        self.attn = dict(qkv=_ql(rng, HIDDEN, (NQ + 2 * NKV,)), o=_ql(rng, HQ * 256, (HIDDEN,), 0.03),
                         qn=_bfw(rng, 256), kn=_bfw(rng, 256))
        self.norms = [_bfw(rng, HIDDEN) for _ in range(3)]
        self.final = _bfw(rng, HIDDEN)
        self.embed = dev(O.f32_to_bf16(rng.standard_normal((VOCAB, HIDDEN)).astype(np.float32)))
        self.head = _ql(rng, HIDDEN, (VOCAB,))
        self.moe = []
        for p, kw in ((0, {}), (1, dict(score="sigmoid", num_groups=4, top_groups=2, group_top=2))):
            bias = dev((rng.standard_normal(E) * 0.1).astype(np.float32)) if p else None
            self.moe.append((p, _bfw(rng, HIDDEN), _ql(rng, HIDDEN, (E + 8,)),
                             dict(num_experts=E, top_k=TOPK, num_shared=1, shared_gate=True, **kw),
                             bias, Experts(HIDDEN, INNER, [E, 1], seed=p).moe))

    def parts(self):
        pool = gdn_amd.Pool(2, 6, HK, HV)
        layers = [gdn_amd.Layer(pool, i, L["i"], L["o"], L["A_log"], L["dt"], L["conv"], L["nw"], EPS)
                  for i, L in enumerate(self.gdn)]
        kv = gdn_amd.KVCache(1, 6, 48, 8, HQ, HKV, max_step_tokens=MAX_PROMPT)
        return pool, layers, kv

    def moe_layers(self):
        return [(p, w, g, gdn_amd.route_desc(**kw), b, m) for p, w, g, kw, b, m in self.moe]

    def executor(self, moe=True):
        pool, layers, kv = self.parts()
        a = self.attn
        return gdn_amd.Executor(pool, layers, self.norms, self.final, self.embed, self.head, EPS,
                                MAX_BATCH, MAX_PROMPT, attn_layers=[(1, a["qkv"], a["o"], a["qn"], a["kn"])],
                                kv=kv, rope_theta=THETA, rotary_dim=ROT,
                                moe_layers=self.moe_layers() if moe else ())


def _e(*shape, dtype=torch.int16):
    return torch.empty(shape, device="cuda:0", dtype=dtype)


class Calls:
    """The executor's step as single calls on a pool and cache of its own."""

    def __init__(self, model):
        self.m = model
        self.pool, self.layers, self.kv = model.parts()

    def run(self, slots, ntok, tokens, prefill):
        m, n = self.m, len(tokens)
        ids = torch.tensor(slots, device="cuda:0", dtype=torch.int32)
        if prefill:
            for s in slots:
                self.kv.release(s)
            self.pool.zero(gdn_amd.GDN_ALL_LAYERS, ids)
        self.kv.step(slots, ntok)
        h = m.embed[torch.tensor(tokens, device="cuda:0")].clone()
        cu = torch.tensor(np.cumsum([0] + ntok), device="cuda:0", dtype=torch.int32)
        hn, mix = torch.empty_like(h), None
        half = {p: x for p, *x in m.moe}
        for p in range(3):
            gdn_amd.add_rms_norm(h, mix, m.norms[p], EPS, hn)
            mix = torch.empty_like(h)
            if p == 1:
                a = m.attn
                qkv, att = _e(n, NQ + 2 * NKV), _e(n, HQ * 256)
                a["qkv"].forward(hn, qkv)
                self.kv.forward(0, qkv[:, :NQ], qkv[:, NQ:NQ + NKV], qkv[:, NQ + NKV:], a["qn"], a["kn"],
                                EPS, THETA, ROT, att)
                a["o"].forward(att, mix)
            elif prefill:
                self.layers[p // 2].prefill(ids, cu, n, hn, mix)
            else:
                self.layers[p // 2].decode(ids, hn, mix)
            if p in half:
                w, gate, kw, bias, moe = half[p]
                gdn_amd.add_rms_norm(h, mix, w, EPS, hn)
                logits, k = _e(n, E + 8), TOPK + 1
                gate.forward(hn, logits)
                eid, ew = _e(n, k, dtype=torch.int32), _e(n, k, dtype=torch.float32)
                gdn_amd.moe_route(logits, eid, ew, bias=bias, **kw)
                moe.forward(hn, eid, ew, mix, moe.workspace(n, k))
        gdn_amd.add_rms_norm(h, mix, m.final, EPS, hn)
        last = hn[cu[1:].long() - 1].contiguous()
        out = _e(len(slots), VOCAB)
        m.head.forward(last, out)
        torch.cuda.synchronize()
        return out


@pytest.fixture(scope="module")
def model(gpu):
    return Model(77)


@pytest.mark.parametrize("graphs", ["0", "1"])
def test_executor_equals_the_calls(model, monkeypatch, graphs):
    monkeypatch.setenv("GDN_EXEC_GRAPHS", graphs)
    # the projections form their group sums themselves, as the single calls do
    monkeypatch.setenv("GDN_EXEC_SPLIT_SUMS", "0")
    ex, calls = model.executor(), Calls(model)
    rng = np.random.default_rng(5)
    prompts = [[int(t) for t in rng.integers(0, VOCAB, n)] for n in (70, 3, 41)]
    first = ex.prefill_batch([10, 11, 12], prompts)
    slots = [ex.slot(i) for i in (10, 11, 12)]
    want = calls.run(slots, [len(p) for p in prompts], sum(prompts, []), True)
    assert torch.equal(ex.logits(), want)
    assert first == [int(t) for t in want.view(torch.bfloat16).float().argmax(1).tolist()]
    cur = first
    for step in range(5):
        cur2 = ex.decode_batch([10, 11, 12], cur)
        want = calls.run(slots, [1, 1, 1], cur, False)
        assert torch.equal(ex.logits(), want), step
        cur = cur2
    # another batch size, then a chained step
    ex.release(11)
    two = [cur[0], cur[2]]
    ex.submit_batch([10, 12], two)
    ex.submit_next(2)
    a = ex.collect_batch(2)
    b = ex.collect_batch(2)
    calls.run([slots[0], slots[2]], [1, 1], two, False)
    want = calls.run([slots[0], slots[2]], [1, 1], a, False)
    assert torch.equal(ex.logits(), want)
    assert b == want.view(torch.bfloat16).float().argmax(1).tolist()
    ex.close()


def test_halves_given_and_taken_away(model):
    """Without halves the executor gives what it gave before them; they are refused
    while sequences are held."""
    plain, ex = model.executor(moe=False), model.executor(moe=True)
    prompt = list(range(30))
    t0 = plain.prefill(1, prompt)
    base = plain.logits().clone()
    ex.prefill(1, prompt)
    assert not torch.equal(ex.logits(), base)
    with pytest.raises(gdn_amd.GdnError, match="holds 1 sequences"):
        ex.set_moe([])
    ex.release(1)
    ex.set_moe([])
    assert ex.prefill(1, prompt) == t0 and torch.equal(ex.logits(), base)
    t1 = ex.decode_batch([1], [t0])
    assert t1 == plain.decode_batch([1], [t0]) and torch.equal(ex.logits(), plain.logits())
    ex.release(1)
    ex.set_moe(model.moe_layers())
    ex.prefill(1, prompt)
    assert not torch.equal(ex.logits(), base)
    for x in (plain, ex):
        x.close()


def test_set_moe_refusals(model):
    ex = model.executor(moe=False)
    (p, w, gate, _, bias, moe) = model.moe[0]
    ok = gdn_amd.route_desc(E, TOPK, num_shared=1, shared_gate=True)
    for bad in ([(3, w, gate, ok, None, moe)], [(-1, w, gate, ok, None, moe)],
                [(0, w, gate, ok, None, moe), (0, w, gate, ok, None, moe)],
                [(0, None, gate, ok, None, moe)],
                [(0, w, model.attn["o"], ok, None, moe)],
                [(0, w, gate, gdn_amd.route_desc(E, TOPK), None, moe)],
                [(0, w, gate, gdn_amd.route_desc(E, TOPK, num_shared=1, logits_f32=True), None, moe)],
                [(0, w, gate, gdn_amd.route_desc(E, 0, num_shared=1), None, moe)],
                [(0, w, gate, gdn_amd.route_desc(E + 40, TOPK, num_shared=1), None, moe)]):
        with pytest.raises(gdn_amd.GdnError):
            ex.set_moe(bad)
    # more halves than layers are refused before any of them is read
    one = (gdn_amd.ExecMoe * 1)()
    for n in (4, 2 ** 31 - 1, -1):
        assert ex.lib.gdn_exec_set_moe(ex.handle, n, one) != 0
        assert b"3 layers" in ex.lib.gdn_last_error()
    assert ex.prefill(1, [1, 2, 3]) >= 0  # nothing changed
    ex.close()

"""The executor with sparse MLP halves in its default configuration, bit for bit
against single calls: the seam behind a half writes the group sums of its rows, and
the next layer's in_proj or lm_head takes them. That happens where the projections
run whole rows of 2048 columns (a GatedDeltaNet in_proj of 12,352) or at least
131,072 outputs (lm_head), so the stack has those widths: GatedDeltaNet, attention,
GatedDeltaNet, a half behind each. Decode steps launch by launch and as replayed
graphs."""
import numpy as np
import pytest
import torch

import gdn_amd
from gdn_testlib import DV, conv_dim
from test_gpu_moe import w4

pytestmark = pytest.mark.gpu

HK, HV, HIDDEN, VOCAB, INNER, E, TOPK = 16, 32, 2048, 131088, 128, 12, 3
HQ, HKV, THETA, ROT, EPS = 16, 2, 1.0e7, 64, 1e-6
NQ, NKV = HQ * 512, HKV * 256
MAX_BATCH, MAX_PROMPT = 8, 96
BF = torch.bfloat16


def _bfw(g, n):
    return (1 + 0.1 * torch.randn(n, generator=g)).to(BF).cuda()


def _ql(g, k, rows):
    return gdn_amd.QLinear(k, [tuple(t[0].cuda() for t in w4(g, 1, n, k)) for n in rows])


def _e(*shape, dtype=BF):
    return torch.empty(shape, device="cuda:0", dtype=dtype)


class Stack:
    def __init__(self):
        g = torch.Generator().manual_seed(9)
        d = conv_dim(HK, HV)
        self.gdn = [dict(i=_ql(g, HIDDEN, (d, HV * DV, HV, HV)), o=_ql(g, HV * DV, (HIDDEN,)),
                         A_log=(torch.rand(HV, generator=g) * np.log(16.0)).cuda(),
                         dt=(torch.randn(HV, generator=g) * 0.1).cuda(),
                         conv=(torch.randn(d, 4, generator=g) * 0.25).to(BF).cuda(),
                         nw=_bfw(g, DV)) for _ in range(2)]
        self.attn = dict(qkv=_ql(g, HIDDEN, (NQ + 2 * NKV,)), o=_ql(g, HQ * 256, (HIDDEN,)),
                         qn=_bfw(g, 256), kn=_bfw(g, 256))
        self.norms = [_bfw(g, HIDDEN) for _ in range(3)]
        self.final = _bfw(g, HIDDEN)
        self.embed = torch.randn(VOCAB, HIDDEN, generator=g).to(BF).cuda()
        self.head = _ql(g, HIDDEN, (VOCAB,))
        self.halves = []
        for p in range(3):
            parts = [tuple(tuple(t.cuda() for t in w4(g, n, r, c)) for r, c in
                           ((INNER, HIDDEN), (INNER, HIDDEN), (HIDDEN, INNER))) for n in (E, 1)]
            self.halves.append((p, _bfw(g, HIDDEN), _ql(g, HIDDEN, (16,)),
                                dict(num_experts=E, top_k=TOPK, num_shared=1, shared_gate=True), None,
                                gdn_amd.MoE(HIDDEN, INNER, parts)))

    def parts(self):
        pool = gdn_amd.Pool(2, MAX_BATCH + 2, HK, HV)
        layers = [gdn_amd.Layer(pool, i, L["i"], L["o"], L["A_log"], L["dt"], L["conv"], L["nw"], EPS)
                  for i, L in enumerate(self.gdn)]
        kv = gdn_amd.KVCache(1, MAX_BATCH + 2, 48, 8, HQ, HKV, max_step_tokens=MAX_PROMPT)
        return pool, layers, kv


class Calls:
    def __init__(self, m):
        self.m = m
        self.pool, self.layers, self.kv = m.parts()

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
        sums = None if prefill else _e(3, 64, HIDDEN // 64)
        for p in range(3):
            gdn_amd.add_rms_norm(h, mix, m.norms[p], EPS, hn, group_sums=None if p == 1 else sums)
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
            else:  # the layer's own chain, its in_proj with the seam's sums
                L, D = m.gdn[p // 2], conv_dim(HK, HV)
                proj, gated = _e(n, D + HV * DV + 2 * HV), _e(n, HV, DV)
                L["i"].forward_sums(hn, sums, proj)
                self.pool.decode_gated(p // 2, ids, proj[:, :D + HV * DV], proj[:, D + HV * DV:],
                                       L["A_log"], L["dt"], L["conv"], L["nw"], EPS, gated)
                L["o"].forward(gated.view(n, HV * DV), mix)
            _, w, gate, kw, bias, moe = m.halves[p]
            gdn_amd.add_rms_norm(h, mix, w, EPS, hn)
            logits, k = _e(n, 16), TOPK + 1
            gate.forward(hn, logits)
            eid, ew = _e(n, k, dtype=torch.int32), _e(n, k, dtype=torch.float32)
            gdn_amd.moe_route(logits, eid, ew, bias=bias, **kw)
            moe.forward(hn, eid, ew, mix, moe.workspace(n, k))
        gdn_amd.add_rms_norm(h, mix, m.final, EPS, hn, group_sums=sums)
        out = _e(len(slots), VOCAB)
        if prefill:
            m.head.forward(hn[cu[1:].long() - 1].contiguous(), out)
        else:
            m.head.forward_sums(hn, sums, out)
        torch.cuda.synchronize()
        return out


@pytest.fixture(scope="module")
def stack(gpu):
    return Stack()


@pytest.mark.parametrize("graphs", ["0", "1"])
def test_executor_in_its_default_configuration_equals_the_calls(stack, monkeypatch, graphs):
    monkeypatch.setenv("GDN_EXEC_GRAPHS", graphs)
    monkeypatch.delenv("GDN_EXEC_SPLIT_SUMS", raising=False)
    pool, layers, kv = stack.parts()
    a = stack.attn
    ex = gdn_amd.Executor(pool, layers, stack.norms, stack.final, stack.embed, stack.head, EPS,
                          MAX_BATCH, MAX_PROMPT, attn_layers=[(1, a["qkv"], a["o"], a["qn"], a["kn"])],
                          kv=kv, rope_theta=THETA, rotary_dim=ROT,
                          moe_layers=[(p, w, g, gdn_amd.route_desc(**kw), b, m)
                                      for p, w, g, kw, b, m in stack.halves])
    calls = Calls(stack)
    rng = np.random.default_rng(5)
    seqs = [10, 11, 12, 13, 14]
    prompts = [[int(t) for t in rng.integers(0, VOCAB, n)] for n in (30, 3, 1, 17, 40)]
    cur = ex.prefill_batch(seqs, prompts)
    slots = [ex.slot(i) for i in seqs]
    want = calls.run(slots, [len(p) for p in prompts], sum(prompts, []), True)
    assert torch.equal(ex.logits().view(torch.int16)[:5], want.view(torch.int16))
    for step in range(4):
        nxt = ex.decode_batch(seqs, cur)
        want = calls.run(slots, [1] * 5, cur, False)
        assert torch.equal(ex.logits().view(torch.int16)[:5], want.view(torch.int16)), step
        assert nxt == want.float().argmax(1).tolist()
        cur = nxt
    assert pool.check() == 0
    ex.close()


def test_the_stack_takes_the_seams_sums(stack):
    """in_proj and lm_head of this stack read the sums that they are given: others give
    other outputs."""
    hn = torch.randn(5, HIDDEN, generator=torch.Generator().manual_seed(1)).to(BF).cuda()
    sums = torch.zeros(3, 64, HIDDEN // 64, device="cuda:0", dtype=BF)
    for q in (stack.gdn[0]["i"], stack.head):
        a, b = _e(5, q.N), _e(5, q.N)
        q.forward(hn, a)
        q.forward_sums(hn, sums, b)
        assert not torch.equal(a, b)

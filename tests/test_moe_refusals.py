"""What the entries of the sparse MLP half refuse, on the host, before any
launch (no GPU)."""
import ctypes
import math

import pytest

import gdn_amd

OK, INVALID, UNSUPPORTED = (gdn_amd.GDN_OK, gdn_amd.GDN_ERR_INVALID, gdn_amd.GDN_ERR_UNSUPPORTED)
A = 0x10000  # stands for an aligned device pointer; nothing here reaches a device


def route(T=4, logits=A, stride=256, bias=None, ids=A, weights=A, **kw):
    f = dict(num_experts=256, top_k=8, score=0, num_groups=1, top_groups=1, group_top=1, renorm=1,
             scale=1.0, num_shared=0, shared_gate=0, logits_f32=0)
    f.update(kw)
    return gdn_amd.load().gdn_moe_route(ctypes.byref(gdn_amd.MoeRouteDesc(**f)), logits, stride, T,
                                        bias, ids, weights, None)


@pytest.mark.parametrize("bad,code", [
    (dict(num_experts=0), UNSUPPORTED), (dict(num_experts=1025), UNSUPPORTED),
    (dict(top_k=0), INVALID), (dict(top_k=33), INVALID), (dict(num_experts=4, top_k=5), INVALID),
    (dict(score=2), INVALID), (dict(num_groups=0), INVALID), (dict(num_groups=7), INVALID),
    (dict(num_groups=128), INVALID), (dict(num_groups=8, top_groups=9), INVALID),
    (dict(top_groups=0), INVALID), (dict(group_top=3), INVALID), (dict(num_shared=9), INVALID),
    (dict(num_shared=-1), INVALID), (dict(shared_gate=1), INVALID),
    (dict(scale=math.inf), INVALID), (dict(scale=math.nan), INVALID), (dict(T=-1), INVALID),
    (dict(logits=None), INVALID), (dict(ids=None), INVALID), (dict(weights=None), INVALID),
    (dict(stride=255), INVALID), (dict(num_shared=1, shared_gate=1), INVALID),
    (dict(logits=A + 1), INVALID), (dict(logits=A + 2, logits_f32=1), INVALID),
    (dict(bias=A + 2), INVALID), (dict(ids=A + 2), INVALID)])
def test_route_refuses(bad, code):
    assert route(**bad) == code
    assert gdn_amd.load().gdn_last_error().startswith(b"gdn_moe_route")


def test_route_without_rows_or_descriptor():
    assert route(T=0, logits=None, ids=None, weights=None) == OK
    assert gdn_amd.load().gdn_moe_route(None, A, 256, 1, None, A, A, None) == INVALID


def create(hidden=256, inner=128, n=1, parts=None, gs=64, bits=4, experts=2, hole=None, dev=0):
    lib = gdn_amd.load()
    h = ctypes.c_void_p()
    p = (gdn_amd.MoePart * max(n, 1))()
    for i in range(max(n, 1)):
        p[i] = gdn_amd.MoePart(experts, *[hole[1] if hole and j == hole[0] else A for j in range(9)])
    st = lib.gdn_moe_create(hidden, inner, n, p if parts is None else parts, gs, bits, dev, None,
                            ctypes.byref(h))
    assert h.value is None
    return st


@pytest.mark.parametrize("bad,code", [
    (dict(bits=8), UNSUPPORTED), (dict(gs=32), UNSUPPORTED), (dict(hidden=64), UNSUPPORTED),
    (dict(hidden=200), UNSUPPORTED), (dict(inner=8320), UNSUPPORTED), (dict(inner=0), UNSUPPORTED),
    (dict(n=0), INVALID), (dict(n=65), INVALID), (dict(experts=0), INVALID),
    (dict(experts=4097), UNSUPPORTED), (dict(experts=2049, n=2), UNSUPPORTED),
    (dict(hole=(0, None)), INVALID), (dict(hole=(8, None)), INVALID), (dict(hole=(3, A + 2)), INVALID),
    (dict(hole=(4, A + 1)), INVALID), (dict(dev=-1), INVALID), (dict(dev=99), INVALID)])
def test_moe_create_refuses(bad, code):
    assert create(**bad) == code
    assert gdn_amd.load().gdn_last_error().startswith(b"gdn_moe_create")


def test_moe_entries_refuse_null():
    lib = gdn_amd.load()
    n = ctypes.c_size_t()
    assert lib.gdn_moe_create(256, 128, 1, None, 64, 4, 0, None, None) == INVALID
    assert lib.gdn_moe_destroy(None) == OK
    assert lib.gdn_moe_dims(None, None, None, None) == INVALID
    assert lib.gdn_moe_workspace_bytes(None, 1, 1, ctypes.byref(n)) == INVALID
    assert lib.gdn_moe_forward(None, A, 256, 1, 1, A, A, A, 256, A, 1 << 20, None) == INVALID


def norm(n=3, h=A, hs=256, x=A, xs=256, post=A, gate=A, gs=1, pre=A, o=A, os=256, hn=A, hns=256,
         kind=1, **kw):
    f = dict(hidden=256, h_f32=0, gate=kind, gate_sigmoid=1, unit_offset=0, scale=1.0,
             post_eps=1e-6, pre_eps=1e-6)
    f.update(kw)
    return gdn_amd.load().gdn_block_norm(ctypes.byref(gdn_amd.BlockNormDesc(**f)), n, h, hs, x, xs,
                                         post, gate, gs, pre, o, os, hn, hns, None)


@pytest.mark.parametrize("bad,code", [
    (dict(hidden=0), UNSUPPORTED), (dict(hidden=252), UNSUPPORTED), (dict(hidden=16392), UNSUPPORTED),
    (dict(kind=0), INVALID), (dict(gate=None), INVALID), (dict(kind=3), INVALID),
    (dict(post_eps=-1.0), INVALID), (dict(pre_eps=math.nan), INVALID), (dict(n=-1), INVALID),
    (dict(h=None), INVALID), (dict(x=None), INVALID), (dict(o=None), INVALID),
    (dict(pre=None), INVALID), (dict(hn=None), INVALID), (dict(hs=248, os=248), INVALID),
    (dict(xs=260, hns=260), INVALID), (dict(hns=128), INVALID), (dict(h=A + 8), INVALID),
    (dict(post=A + 4), INVALID), (dict(pre=A + 2), INVALID), (dict(gs=-1), INVALID),
    (dict(kind=2, gs=4), INVALID), (dict(kind=2, gs=128), INVALID), (dict(os=264), INVALID),
    (dict(hns=264), INVALID)])
def test_block_norm_refuses(bad, code):
    assert norm(**bad) == code
    assert gdn_amd.load().gdn_last_error().startswith(b"gdn_block_norm")


def test_block_norm_without_rows_or_descriptor():
    lib = gdn_amd.load()
    d = gdn_amd.BlockNormDesc(256, 0, 0, 0, 0, 1.0, 1e-6, 1e-6)
    assert lib.gdn_block_norm(ctypes.byref(d), 0, None, 0, None, 0, None, None, 0, None, None, 0,
                              None, 0, None) == OK
    assert lib.gdn_block_norm(None, 1, A, 256, A, 256, None, None, 0, None, A, 256, None, 0,
                              None) == INVALID

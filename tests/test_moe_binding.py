"""The binding of the sparse MLP half on the host: what the library is handed for a
call's arguments (no GPU; the library's entries are stood in for)."""
import ctypes

import pytest
import torch

import gdn_amd

BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32


class Recorder:
    """Stands in for the library: keeps the arguments of every call."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return gdn_amd.GDN_OK
        return call


@pytest.fixture
def lib(monkeypatch):
    gdn_amd.load()
    rec = Recorder()
    monkeypatch.setattr(gdn_amd, "load", lambda *a: rec)
    # CPU tensors say that they are on device -1
    monkeypatch.setattr(gdn_amd, "_current_device", lambda: -1)
    monkeypatch.setattr(gdn_amd, "_raw_stream", lambda dev: None)
    return rec


def _desc(rec, kind):
    ref = rec.calls[-1][1][0]
    return ctypes.cast(ref, ctypes.POINTER(kind)).contents


def _route(T=4, E=256, k=8, **kw):
    gdn_amd.moe_route(torch.zeros(T, E, dtype=BF), torch.zeros(T, k, dtype=I32), torch.zeros(T, k),
                      E, k, **kw)


def test_a_descriptor_belongs_to_its_caller(lib):
    mine = gdn_amd.route_desc(256, 8)
    mine.renorm, mine.scale, mine.top_k = 0, 7.0, 3
    other = gdn_amd.route_desc(256, 8)
    assert (other.renorm, other.scale, other.top_k) == (1, 1.0, 8)
    _route()
    d = _desc(lib, gdn_amd.MoeRouteDesc)
    assert (d.renorm, d.scale, d.top_k) == (1, 1.0, 8)


@pytest.mark.parametrize("name", ["scale"])
def test_route_takes_the_value_that_a_tensor_has_at_the_call(lib, name):
    t = torch.tensor(2.5)
    for v in (2.5, 1.0, 0.25):
        t.fill_(v)
        _route(**{name: t})
        assert getattr(_desc(lib, gdn_amd.MoeRouteDesc), name) == v


@pytest.mark.parametrize("name", ["scale", "pre_eps", "post_eps"])
def test_block_norm_takes_the_value_that_a_tensor_has_at_the_call(lib, name):
    h, x, w = torch.zeros(3, 64), torch.zeros(3, 64, dtype=BF), torch.ones(64, dtype=BF)
    t = torch.tensor(2.5)
    for v in (2.5, 1.0, 0.25):
        t.fill_(v)
        gdn_amd.block_norm(h, x, hn=torch.zeros_like(x), pre_w=w, **{name: t})
        assert getattr(_desc(lib, gdn_amd.BlockNormDesc), name) == v


def test_flags_of_any_type(lib):
    t = torch.tensor(True)
    for v in (True, False):
        t.fill_(v)
        _route(renorm=t)
        assert _desc(lib, gdn_amd.MoeRouteDesc).renorm == int(v)

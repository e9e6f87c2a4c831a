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


def _part(n=2, hidden=128, inner=128):
    def mat(r, c):
        return (torch.zeros(n, r, c // 8, dtype=I32), torch.zeros(n, r, c // 64, dtype=BF),
                torch.zeros(n, r, c // 64, dtype=BF))
    return [mat(inner, hidden), mat(inner, hidden), mat(hidden, inner)]


def _swap(part, m, t, tensor):
    part = [list(x) for x in part]
    part[m][t] = tensor
    return part


def test_experts_refuse_parts_of_another_type_size_layout_or_device(lib, monkeypatch):
    """What the kernels would read as something else, or past its end."""
    asked = []
    monkeypatch.setattr(gdn_amd, "_raw_stream", lambda dev: asked.append(dev))
    ok = _part()
    bits = [[w.view(torch.uint32), s.view(torch.int16), b.view(torch.uint16)] for w, s, b in ok]
    for part in (ok, bits):
        assert gdn_amd.MoE(128, 128, [part], device=-1).experts == 2
        assert lib.calls[-1][0] == "gdn_moe_create"
    assert asked == [-1, -1]  # the stream of the layer's device
    made = len(lib.calls)
    for bad in (_swap(ok, 0, 0, torch.zeros(2, 128, 16)),                     # floats as packed weights
                _swap(ok, 1, 0, torch.zeros(2, 128, 16, dtype=torch.int64)),
                _swap(ok, 2, 0, torch.zeros(2, 128, 8, dtype=I32)),           # too short
                _swap(ok, 0, 1, torch.zeros(2, 128, 2)),                      # f32 scales
                _swap(ok, 1, 2, torch.zeros(2, 128, 2, dtype=torch.float16)),
                _swap(ok, 2, 1, torch.zeros(1, 128, 2, dtype=BF)),            # fewer experts
                _swap(ok, 0, 0, torch.zeros(2, 16, 128, dtype=I32).transpose(1, 2))):
        with pytest.raises(ValueError):
            gdn_amd.MoE(128, 128, [bad], device=-1)
    with pytest.raises(ValueError, match="cuda:0"):  # parts of another device than the layer's
        gdn_amd.MoE(128, 128, [ok], device=0)
    assert len([c for c in lib.calls[made:] if c[0] == "gdn_moe_create"]) == 0


class _Handle:
    handle = ctypes.c_void_p(1)
    device = -1


def test_set_moe_refuses_weights_of_another_type_size_layout_or_device(lib):
    """A half's norm weights and bias are read by every later step."""
    ex = gdn_amd.Executor.__new__(gdn_amd.Executor)
    ex.lib, ex.handle, ex.device, ex.hidden = lib, ctypes.c_void_p(1), -1, 128
    norm, bias = torch.ones(128, dtype=BF), torch.zeros(24)
    route = gdn_amd.route_desc(24, 4)
    half = lambda w=norm, b=bias, g=_Handle: (0, w, g, route, b, _Handle)  # noqa: E731
    for b in (bias, None):
        ex.set_moe([half(b=b)])
        assert lib.calls[-1][0] == "gdn_exec_set_moe"
    ex.set_moe([half(w=norm.view(torch.int16))])
    made = len(lib.calls)

    class Elsewhere(_Handle):
        device = 0

    for bad in (half(w=torch.ones(128)), half(w=torch.ones(64, dtype=BF)),
                half(w=torch.ones(256, dtype=BF)[::2]), half(w=torch.ones(1, 128, dtype=BF)),
                half(b=bias.to(BF)), half(b=torch.zeros(23)), half(b=torch.zeros(48)[::2]),
                half(b=torch.zeros(24, dtype=torch.float64)), half(g=Elsewhere)):
        with pytest.raises(ValueError):
            ex.set_moe([bad])
    ex.device = 0
    with pytest.raises(ValueError, match="cuda:0"):
        ex.set_moe([half()])
    assert len(lib.calls) == made


def test_one_row_of_any_stride(lib):
    """The stride of a single row does not matter: torch gives it none in particular."""
    def one(n, dtype):  # [1, n], contiguous, with a row stride of 1
        t = torch.zeros(n, 1, dtype=dtype).t()
        assert t.is_contiguous() and t.stride(0) == 1
        return t

    def odd(n, dtype):  # a row of a matrix whose rows are n + 3 apart
        return torch.zeros(2, n + 3, dtype=dtype)[:1, :n]

    for row in (one, odd):
        gdn_amd.moe_route(row(257, BF), torch.zeros(1, 9, dtype=I32), torch.zeros(1, 9), 256, 8,
                          num_shared=1, shared_gate=True)
        assert lib.calls[-1][1][2] >= 257
        gdn_amd.block_norm(row(64, F32), row(64, BF), h_out=row(64, F32), hn=row(64, BF),
                           pre_w=torch.ones(64, dtype=BF), gate=row(64, BF))
        a = lib.calls[-1][1]
        for stride in (a[3], a[5], a[8], a[11], a[13]):
            assert stride >= 64 and stride % 8 == 0
        moe = gdn_amd.MoE(128, 128, [_part()], device=-1)
        ws = torch.zeros(256, dtype=torch.uint8)
        moe.forward(row(128, BF), torch.zeros(1, 2, dtype=I32), torch.zeros(1, 2), row(128, BF), ws)
        a = lib.calls[-1][1]
        assert a[2] >= 128 and a[2] % 8 == 0 and a[8] >= 128 and a[8] % 4 == 0

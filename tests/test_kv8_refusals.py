"""What the entries of the 8-bit cache and the rotary positions refuse on the host, before
any launch (no GPU)."""
import ctypes
import math

import pytest

import gdn_amd

OK, INVALID, UNSUPPORTED = (gdn_amd.GDN_OK, gdn_amd.GDN_ERR_INVALID, gdn_amd.GDN_ERR_UNSUPPORTED)


@pytest.mark.parametrize("bad,code", [
    (dict(num_layers=0), INVALID), (dict(num_slots=0), INVALID), (dict(num_pages=0), INVALID),
    (dict(max_pages_per_slot=0), INVALID), (dict(num_q_heads=0), INVALID),
    (dict(num_kv_heads=0), INVALID), (dict(max_step_tokens=0), INVALID),
    (dict(head_dim=96), UNSUPPORTED), (dict(num_q_heads=9), UNSUPPORTED),
    (dict(num_q_heads=34), UNSUPPORTED), (dict(num_q_heads=257, num_kv_heads=257), UNSUPPORTED),
    (dict(num_slots=4097), UNSUPPORTED), (dict(max_step_tokens=262145), UNSUPPORTED),
    (dict(num_pages=(1 << 24) + 1), UNSUPPORTED), (dict(max_pages_per_slot=1 << 25), UNSUPPORTED),
    (dict(num_slots=4096, max_pages_per_slot=1 << 20), UNSUPPORTED), (dict(device=-1), INVALID),
    (dict(device=99), INVALID)])
def test_create_refuses(bad, code):
    lib = gdn_amd.load()
    f = dict(num_layers=1, num_slots=2, num_pages=4, max_pages_per_slot=2, num_q_heads=16,
             num_kv_heads=2, head_dim=256, max_step_tokens=8, device=0)
    f.update(bad)
    h = ctypes.c_void_p()
    d = gdn_amd.KV8Desc(**f)
    assert lib.gdn_kv8_create(ctypes.byref(d), ctypes.byref(h)) == code
    assert h.value is None and lib.gdn_last_error().startswith(b"gdn_kv8_create")


def test_entries_refuse_null():
    lib = gdn_amd.load()
    h, n, v = ctypes.c_void_p(), ctypes.c_uint32(), gdn_amd.KV8View()
    assert lib.gdn_kv8_create(None, ctypes.byref(h)) == INVALID
    d = gdn_amd.KV8Desc(1, 2, 4, 2, 16, 2, 256, 8, 0)
    assert lib.gdn_kv8_create(ctypes.byref(d), None) == INVALID
    assert lib.gdn_kv8_destroy(None) == OK
    assert lib.gdn_kv8_describe(None, ctypes.byref(d)) == INVALID
    assert lib.gdn_kv8_views(None, ctypes.byref(v)) == INVALID
    assert lib.gdn_kv8_check(None, None, ctypes.byref(n)) == INVALID
    assert lib.gdn_kv8_step(None, 1, 4096, 4096, 4096, None, 1, 1, None) == INVALID
    assert lib.gdn_kv8_append(None, 0, 4096, 512, 4096, 512, None) == INVALID
    assert lib.gdn_kv8_gather(None, 0, 1, 4096, 4096, 512, None, 0, None) == INVALID
    a = gdn_amd.KV8AttnDesc(0.0, 0.0, 0)
    assert lib.gdn_kv8_attention(None, 0, ctypes.byref(a), 4096, 4096, 256, None, None, None, 0, 0,
                                 4096, 4096, 256, None) == INVALID
    r = gdn_amd.RopeRows()
    assert lib.gdn_rope_forward(None, 1, 4096, ctypes.byref(r), None, 0, 0.0, 0, None) == INVALID
    assert lib.gdn_rope_create(None, 0, ctypes.byref(h)) == INVALID
    assert lib.gdn_rope_destroy(None) == OK


@pytest.mark.parametrize("bad,code", [
    (dict(head_dim=4), UNSUPPORTED), (dict(head_dim=100), UNSUPPORTED),
    (dict(head_dim=520), UNSUPPORTED), (dict(rotary_dim=33), INVALID),
    (dict(rotary_dim=-2), INVALID), (dict(rotary_dim=66), INVALID), (dict(scaling=4), INVALID),
    (dict(scaling=-1), INVALID), (dict(base=1.0), INVALID), (dict(base=math.inf), INVALID),
    (dict(factor=0.0), INVALID), (dict(factor=math.nan), INVALID),
    (dict(magnitude=math.nan), INVALID), (dict(scaling=2, original=0.0), INVALID),
    (dict(scaling=2, slow=0.0), INVALID), (dict(scaling=3, fast=1.0), INVALID),
    (dict(scaling=3, original=math.inf), INVALID)])
def test_rope_create_refuses(bad, code):
    lib = gdn_amd.load()
    f = dict(head_dim=64, rotary_dim=64, interleaved=0, scaling=0, base=1e4, factor=2.0,
             original=4096.0, fast=32.0, slow=1.0, magnitude=0.0)
    f.update(bad)
    h = ctypes.c_void_p()
    d = gdn_amd.RopeDesc(**f)
    assert lib.gdn_rope_create(ctypes.byref(d), 0, ctypes.byref(h)) == code
    assert h.value is None and lib.gdn_last_error().startswith(b"gdn_rope_create")


def test_rope_names_its_scalings():
    with pytest.raises(ValueError, match="scaling"):
        gdn_amd.Rope(64, scaling="ntk")

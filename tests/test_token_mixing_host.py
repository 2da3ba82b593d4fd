"""The token-mixing entry points refuse bad arguments on the host, before they
touch a device, and the rope specification is filled as documented.  Status
codes: 1 null, 2 shape, 3 alignment, 6 workspace, 7 value."""
import ctypes
import math
import struct

import pytest

import mcv_b200

NULL, SHAPE, ALIGN, WORKSPACE, VALUE = 1, 2, 3, 6, 7
F, F2 = 256, 256 + 2     # 16-byte aligned stand-in for a device address, and one that is not
BIG = 1 << 30


@pytest.fixture(scope="module")
def L():
    return mcv_b200.lib()


def rows(data=F, ts=2048, hs=256):
    return ctypes.byref(mcv_b200._Rows(data, ts, hs))


def cache(k=F, v=F, stride=2 * 16 * 256, pages=10, page=16, heads=2, dim=256):
    return ctypes.byref(mcv_b200._KVCache(k, v, stride, pages, page, heads, dim))


def spec(rotary=64, sections=(12, 10, 10), interleaved=True):
    return mcv_b200.MRope(rotary, list(sections), interleaved)


@pytest.mark.parametrize("rotary,sections,interleaved,theta,status", [
    (60, [30], 0, 1e4, SHAPE), (0, [0], 0, 1e4, SHAPE), (272, [136], 0, 1e4, SHAPE), (64, [12, 10], 0, 1e4, SHAPE),
    (64, [40, -8], 0, 1e4, VALUE), (64, [32], 0, 1.0, VALUE), (64, [32], 0, math.nan, VALUE),
    (64, [32], 0, math.inf, VALUE), (64, [6, 6, 6, 6, 8], 0, 1e4, VALUE), (64, [], 0, 1e4, VALUE),
    (64, [10, 11, 11], 1, 1e4, SHAPE), (64, [0, 32], 1, 1e4, SHAPE)])
def test_mrope_init_refuses(L, rotary, sections, interleaved, theta, status):
    arr = (ctypes.c_int32 * max(1, len(sections)))(*sections)
    s = mcv_b200._MRopeSpec()
    assert L.mcv_mrope_init(ctypes.byref(s), rotary, len(sections), arr, interleaved, theta) == status


@pytest.mark.parametrize("sections,interleaved", [([32], False), ([12, 10, 10], False), ([12, 10, 10], True),
                                                  ([0, 20, 12], False), ([16, 16], True), ([8, 8, 8, 8], True),
                                                  ([26, 0, 6], True)])
def test_mrope_init_axes_and_frequencies(sections, interleaved):
    rope = mcv_b200.MRope(64, sections, interleaved, theta=10000.0)
    n = len(sections)
    for i in range(32):
        if interleaved:
            want = i % n if i % n and i < n * sections[i % n] else 0
        else:
            want = next(a for a in range(n) if i < sum(sections[:a + 1]))
        assert rope._c.axis[i] == want
        assert math.isclose(rope._c.turns[i], 10000.0 ** (-i / 32) / (2 * math.pi), rel_tol=1e-14)
    assert [list(rope._c.axis)[:32].count(a) for a in range(n)] == sections


def test_mrope_arguments(L):
    f, s = L.mcv_mrope, ctypes.byref(spec()._c)
    ok = [rows(), F, s, F, 5, 8, 256, None]
    def with_(i, x):
        return [*ok[:i], x, *ok[i + 1:]]
    assert f(*with_(0, None)) == NULL and f(*with_(0, rows(None))) == NULL
    assert f(*with_(1, None)) == NULL and f(*with_(2, None)) == NULL and f(*with_(3, None)) == NULL
    assert f(*with_(0, rows(F2))) == ALIGN and f(*with_(1, F2)) == ALIGN
    assert f(*with_(0, rows(F, 2047))) == ALIGN and f(*with_(0, rows(F, 2048, 252))) == ALIGN
    assert f(*with_(0, rows(F, 2048, 248))) == SHAPE            # heads overlap
    assert f(*with_(0, rows(F, -2048))) == SHAPE
    assert f(*with_(4, 0)) == SHAPE and f(*with_(4, BIG)) == SHAPE
    assert f(*with_(5, 0)) == SHAPE and f(*with_(6, 1032)) == SHAPE and f(*with_(6, 252)) == SHAPE
    assert f(*with_(6, 56)) == SHAPE                             # rotary_dim beyond head_dim
    assert f(rows(F + 16, 0, 256), F + 16, s, F, 5, 8, 256, None) == SHAPE   # in place on one shared token
    bad = spec()
    bad._c.axis[3] = 3
    assert f(*with_(2, ctypes.byref(bad._c))) == VALUE


def test_mrope_append_arguments(L):
    f, s = L.mcv_mrope_append_kv, ctypes.byref(spec()._c)
    ok = [rows(), F, rows(F, 512), rows(F, 512), s, F, cache(), F, 9, 4, None, F, 5, 8, None]
    def with_(i, x):
        return f(*[*ok[:i], x, *ok[i + 1:]])
    for i in (0, 1, 2, 3, 4, 5, 6, 7, 11):
        assert with_(i, None) == NULL, i
    assert with_(8, 4) == SHAPE                    # fewer table rows than tokens without seq
    assert with_(8, 0) == SHAPE and with_(9, 0) == SHAPE and with_(12, 0) == SHAPE and with_(13, 0) == SHAPE
    assert with_(6, cache(k=None)) == NULL and with_(6, cache(k=F2)) == ALIGN
    assert with_(6, cache(stride=8191)) == ALIGN and with_(6, cache(stride=8184)) == SHAPE
    assert with_(6, cache(pages=0)) == SHAPE and with_(6, cache(page=0)) == SHAPE
    assert with_(2, rows(F2)) == ALIGN and with_(3, rows(F, 512, 128)) == SHAPE


def test_attention_arguments(L):
    n = L.mcv_paged_attention_workspace_size(8, 2, 256)
    assert n > 0 and L.mcv_paged_attention_workspace_size(7, 2, 256) == 0
    assert L.mcv_paged_attention_workspace_size(8, 2, 96) == 0 and L.mcv_paged_attention_workspace_size(8, 0, 64) == 0
    f = L.mcv_paged_attention_decode
    ok = [rows(), cache(), F, 4, F, F, None, 3, 8, 0.0625, F, n, None]
    def with_(i, x):
        return f(*[*ok[:i], x, *ok[i + 1:]])
    for i in (0, 1, 2, 4, 5):
        assert with_(i, None) == NULL, i
    assert with_(10, None) == WORKSPACE and with_(11, n - 1) == WORKSPACE and with_(10, F2) == ALIGN
    assert with_(5, F2) == ALIGN and with_(0, rows(F2)) == ALIGN
    assert with_(7, 0) == SHAPE and with_(7, 4097) == SHAPE
    assert with_(8, 7) == SHAPE and with_(8, 0) == SHAPE and with_(3, 0) == SHAPE and with_(3, 1 << 27) == SHAPE
    assert with_(1, cache(dim=96, stride=2 * 16 * 96)) == SHAPE
    for scale in (0.0, -1.0, math.inf, math.nan):
        assert with_(9, scale) == VALUE


def delta(**change):
    a = mcv_b200._GatedDelta()
    a.q = a.k = a.v = mcv_b200._Rows(F, 6144, 128)
    a.g = a.beta = a.out = a.state_in = a.state_out = F
    a.slots, a.k_heads, a.v_heads, a.key_dim, a.value_dim, a.scale, a.l2_eps = 3, 16, 16, 128, 128, 0.1, 1e-6
    for name, x in change.items():
        setattr(a, name, x)
    return ctypes.byref(a)


@pytest.mark.parametrize("change,status", [
    ({"g": None}, NULL), ({"beta": None}, NULL), ({"out": None}, NULL), ({"key_dim": 96}, SHAPE),
    ({"value_dim": 24}, SHAPE), ({"value_dim": 0}, SHAPE), ({"value_dim": 1040}, SHAPE), ({"v_heads": 24}, SHAPE),
    ({"k_heads": 0}, SHAPE), ({"slots": 2}, SHAPE), ({"slots": 0}, SHAPE), ({"out": F2}, ALIGN),
    ({"state_in": F2}, ALIGN), ({"scale": math.nan}, VALUE), ({"l2_eps": math.nan}, VALUE),
    ({"q": mcv_b200._Rows(None, 6144, 128)}, NULL), ({"k": mcv_b200._Rows(F, 6143, 128)}, ALIGN),
    ({"v": mcv_b200._Rows(F, 6144, 120)}, SHAPE)])
def test_delta_arguments(L, change, status):
    n = L.mcv_gated_delta_workspace_size(40, 3, 16, 128, 128)
    assert L.mcv_gated_delta_step(delta(**change), 3, None) == status
    assert L.mcv_gated_delta_prefill(delta(**change), F, 40, 3, F, n, None) == status


def test_delta_call_arguments(L):
    n = L.mcv_gated_delta_workspace_size(40, 3, 16, 128, 128)
    assert n > 0
    assert L.mcv_gated_delta_workspace_size(0, 3, 16, 128, 128) == 0
    assert L.mcv_gated_delta_workspace_size(40, 3, 16, 96, 128) == 0
    assert L.mcv_gated_delta_step(None, 3, None) == NULL
    assert L.mcv_gated_delta_step(delta(state_in=None), 3, None) == NULL
    assert L.mcv_gated_delta_step(delta(state_out=None), 3, None) == NULL
    assert L.mcv_gated_delta_step(delta(), 0, None) == SHAPE
    f = L.mcv_gated_delta_prefill
    assert f(delta(), None, 40, 3, F, n, None) == NULL
    assert f(delta(), F, 40, 3, None, n, None) == WORKSPACE
    assert f(delta(), F, 40, 3, F, n - 1, None) == WORKSPACE
    assert f(delta(), F, 40, 3, F2, n, None) == ALIGN
    assert f(delta(), F, 0, 3, F, n, None) == SHAPE
    assert f(delta(), F, 40, 0, F, n, None) == SHAPE


def test_python_checks():
    """The binding refuses tensors of the wrong place, type or shape."""
    import torch
    with pytest.raises(RuntimeError, match="CUDA"):
        mcv_b200.PagedKVCache(torch.zeros(2, 2, 16, 64).half(), torch.zeros(2, 2, 16, 64).half())
    with pytest.raises(RuntimeError, match="float16"):
        mcv_b200.PagedKVCache(torch.zeros(2, 2, 16, 64), torch.zeros(2, 2, 16, 64))
    x, pos = torch.zeros(3, 2, 64).half(), torch.zeros(1, 3, dtype=torch.int32)
    rope = mcv_b200.MRope(64, [32])
    with pytest.raises(RuntimeError, match="CUDA"):
        mcv_b200.mrope(x, pos, rope, x)
    with pytest.raises(RuntimeError, match="positions"):
        mcv_b200.mrope(x, pos.long(), rope, x)
    with pytest.raises(RuntimeError, match="positions"):
        mcv_b200.mrope(x, pos[:, :2], rope, x)
    with pytest.raises(RuntimeError, match="float16"):
        mcv_b200.mrope(x.float(), pos, rope, x)
    with pytest.raises(RuntimeError, match="out"):
        mcv_b200.mrope(x, pos, rope, torch.zeros(3, 2, 72).half()[:, :, :64])
    with pytest.raises(mcv_b200.McvError):
        mcv_b200.MRope(64, [30])


def test_packed_structures():
    """The bytes that the binding passes are the C structures of the header."""
    assert struct.calcsize("@3q") == ctypes.sizeof(mcv_b200._Rows)
    assert struct.calcsize("@9q6Pq4i2f") == ctypes.sizeof(mcv_b200._GatedDelta)
    assert mcv_b200._pack_rows(F, 24, 8) == bytes(mcv_b200._Rows(F, 24, 8))
    a = mcv_b200._GatedDelta()
    a.q, a.k, a.v = (mcv_b200._Rows(10 * i, 10 * i + 1, 10 * i + 2) for i in (1, 2, 3))
    a.g, a.beta, a.out, a.state_in, a.state_out, a.state_index = 40, 50, 60, 70, 80, 90
    a.slots, a.k_heads, a.v_heads, a.key_dim, a.value_dim, a.scale, a.l2_eps = 5, 6, 7, 8, 9, 0.5, 0.25
    assert mcv_b200._pack_delta(10, 11, 12, 20, 21, 22, 30, 31, 32, 40, 50, 60, 70, 80, 90, 5, 6, 7, 8, 9, 0.5, 0.25) == bytes(a)

"""The 4-bit cache without a GPU: the oracle's own format, and every refusal of the
C entries and of the Python calls before a launch."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import ttcd_amd
from oracle import kv4_ref
from ttcd_amd import _lib

INV, UNSUP = _lib.TTCD_ERR_INVALID_ARGUMENT, _lib.TTCD_ERR_UNSUPPORTED
P = 0x10000  # never dereferenced


def test_the_oracle_rounds_as_the_format_says():
    x = torch.zeros(32, dtype=torch.bfloat16)
    x[:13] = torch.tensor([6, 5, 4.5, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25, -0.25, -0.3, -2.5, 0.5])
    code, e = kv4_ref.quantise(x)
    assert e.tolist() == [0]
    assert kv4_ref.values(code, e)[:13].tolist() == [6, 4, 4, 4, 2, 2, 1, 1, 0, 0, -0.5, -2, 0.5]
    for top, exp in ((6.0, 0), (6.03125, 1), (3.0, -1), (3.1, 0), (math.inf, 125), (0.0, -125),
                     (2.0 ** -133, -125), (3.3e38, 125)):
        x[:] = 0
        x[3] = top
        assert kv4_ref.quantise(x)[1].item() == exp, top
    h = torch.full((32,), 65504.0, dtype=torch.float16)
    assert kv4_ref.quantise(h)[1].item() == 13 and kv4_ref.held(h)[0] == 6 * 2 ** 13
    # every held value is a number of the type
    for dt, (lo, hi) in kv4_ref.E_RANGE.items():
        for exp in (lo, hi):
            v = kv4_ref.GRID * 2.0 ** exp
            assert torch.equal(v.to(dt).double(), v)


def _struct(**over):
    f = dict(k_codes=P, k_scales=P, v_codes=P, v_scales=P, lengths=P, batch=2, kv_heads=2,
             head_dim=64, capacity=64)
    f.update(over)
    return ctypes.byref(_lib.KV4CacheStruct(**f))


BAD_CACHES = [({"k_codes": 0}, INV), ({"lengths": 0}, INV), ({"batch": 0}, INV),
              ({"kv_heads": 0}, INV), ({"head_dim": 96}, UNSUP), ({"capacity": 0}, INV),
              ({"capacity": 48}, INV), ({"capacity": -32}, INV), ({"k_codes": P + 8}, UNSUP),
              ({"v_codes": P + 4}, UNSUP), ({"v_scales": P + 2}, UNSUP),
              ({"lengths": P + 1}, UNSUP), ({"capacity": (1 << 30) + 32}, INV),
              ({"batch": 40000}, UNSUP)]

ST = (64 * 4 * 8, 64 * 4, 64, 1)


def _append(c=None, k=P, v=P, T=4, ks=ST, vs=ST, dt=0):
    return _lib.lib().ttcd_kv4_append(c or _struct(), k, v, T, _lib.strides4(ks),
                                      _lib.strides4(vs), None, None, dt, None)


def _attn(c=None, q=P, o=P, Tq=4, Hq=4, qs=ST, os=ST, scale=0.125, dt=0):
    return _lib.lib().ttcd_kv4_attn_fwd(c or _struct(), q, o, None, Tq, Hq, _lib.strides4(qs),
                                        _lib.strides4(os), None, 0, scale, dt, None, 0, None)


def _weights(c=None, q=P, lse=P, w=P, Tq=4, Hq=4, qs=ST, scale=0.125, dt=0):
    return _lib.lib().ttcd_kv4_key_weights_fwd(c or _struct(), q, lse, w, Tq, Hq,
                                               _lib.strides4(qs), None, 0, scale, 0, dt, None)


def _read(c=None, k=P, v=P, count=4, dt=0):
    return _lib.lib().ttcd_kv4_read(c or _struct(), k, v, count, dt, None)


Q = P + 0x1000


def _evict(c=None, out=None, w=P, keep=8, recent=2, nw=Q, index=P):
    o = out or _struct(k_codes=Q, k_scales=Q, v_codes=Q, v_scales=Q, lengths=Q)
    return _lib.lib().ttcd_kv4_evict(c or _struct(), w, keep, recent, o, nw, index, None)


@pytest.mark.parametrize("call", [_append, _attn, _weights, _read, _evict])
@pytest.mark.parametrize("fields,status", BAD_CACHES)
def test_bad_caches(call, fields, status):
    assert call(c=_struct(**fields)) == status
    assert _lib.lib().ttcd_last_error()


def test_bad_arguments():
    odd, wide = (ST[0], ST[1], 60, 1), (ST[0], ST[1], 64, 2)
    assert _append(k=None) == _append(v=None) == _append(T=0) == _append(T=65) == INV
    assert _append(ks=wide) == INV
    assert _append(vs=odd) == _append(k=P + 2) == _append(dt=2) == _append(ks=(-8, 8, 8, 1)) == UNSUP
    assert _attn(q=None) == _attn(o=None) == _attn(Tq=0) == _attn(Hq=3) == _attn(Hq=0) == INV
    assert _attn(scale=0.0) == _attn(scale=math.nan) == _attn(scale=math.inf) == INV
    assert _attn(qs=odd) == _attn(os=odd) == _attn(o=P + 8) == _attn(dt=2) == UNSUP
    assert _attn(Tq=1 << 29) == UNSUP
    assert _weights(lse=None) == _weights(w=None) == _weights(Tq=0) == _weights(Hq=5) == INV
    assert _weights(qs=odd) == _weights(dt=7) == _weights(w=P + 4) == UNSUP
    assert _read(k=None) == _read(count=0) == INV
    assert _read(v=P + 8) == _read(dt=2) == UNSUP
    assert _evict(w=None) == _evict(index=None) == _evict(keep=0) == _evict(keep=65) == INV
    assert _evict(recent=-1) == _evict(nw=P) == INV
    other = dict(k_codes=Q, k_scales=Q, v_codes=Q, v_scales=Q, lengths=Q)
    for over in ({"k_codes": P}, {"v_scales": P}, {"lengths": P}, {"batch": 1}, {"kv_heads": 4},
                 {"head_dim": 128}, {"capacity": 0}):
        assert _evict(out=_struct(**dict(other, **over))) == INV
    assert _lib.lib().ttcd_kv4_append(None, P, P, 1, _lib.strides4(ST), _lib.strides4(ST), None,
                                      None, 0, None) == INV


def test_workspace_of_bad_arguments_is_none():
    f = _lib.lib().ttcd_kv4_attn_workspace_bytes
    assert f(None, 1, 4, 0) == f(_struct(head_dim=32), 1, 4, 0) == f(_struct(), 0, 4, 0) == 0
    assert f(_struct(), 1, 3, 0) == f(_struct(batch=0), 1, 4, 0) == f(_struct(capacity=0), 1, 4, 0) == 0
    assert f(_struct(), 1, 4, 0) == 0  # a short cache is not split
    big = _struct(batch=1, capacity=1 << 16)
    assert f(big, 1, 4, 0) > f(big, 1, 4, 4096) > 0


def test_python_refusals_on_the_cpu():
    with pytest.raises(ValueError, match="head_dim"):
        ttcd_amd.KV4Cache(1, 1, 96, 64, device="cpu")
    with pytest.raises(ValueError, match="multiple of 32"):
        ttcd_amd.KV4Cache(1, 1, 64, 40, device="cpu")
    with pytest.raises(ValueError, match="batch"):
        ttcd_amd.KV4Cache(0, 1, 64, 64, device="cpu")
    with pytest.raises(ValueError, match="dtype"):
        ttcd_amd.KV4Cache(1, 1, 64, 64, torch.float32, device="cpu")
    with pytest.raises(ValueError, match="GPU"):
        ttcd_amd.KV4Cache(1, 1, 64, 64, device="cpu")
    x = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16)
    for call in (lambda: ttcd_amd.kv4_append(None, x, x), lambda: ttcd_amd.kv4_attn(x, None),
                 lambda: ttcd_amd.kv4_read(None, 1), lambda: ttcd_amd.kv4_evict(None, x, 1),
                 lambda: ttcd_amd.kv4_key_weights(x, None, x)):
        with pytest.raises(ValueError, match="KV4Cache"):
            call()


def test_model_cache_arguments():
    from ttcd_amd import IPTTCDv9Cache
    for bad in (dict(bits=8), dict(bits=4), dict(bits=4, capacity=0), dict(capacity=64),
                dict(keep=4), dict(bits=4, capacity=64, keep=65),
                dict(bits=4, capacity=64, keep=0), dict(bits=4, capacity=64, recent=-1)):
        with pytest.raises(ValueError):
            IPTTCDv9Cache(**bad)
    c = IPTTCDv9Cache(bits=4, capacity=70)
    assert c.capacity == 96
    c.reserve(96, None)
    with pytest.raises(ValueError, match="positions"):
        c.reserve(97, None)
    c.held = 500  # a window's ring has wrapped
    c.reserve(33, 64)
    with pytest.raises(ValueError, match="positions"):
        c.reserve(34, 64)
    with pytest.raises(NotImplementedError):
        IPTTCDv9Cache(bits=4, capacity=64, keep=8).reserve(1, 32)


def test_no_stage_is_rewritten_while_it_may_be_read():
    """The many-row attention's order of loads, conversions, products and barriers, by the
    code that the kernel runs (kv4_sweep.h)."""
    f = _lib.lib().ttcd_kv4_block_stages
    for t0 in range(4):
        for n in range(1, 40):
            assert f(t0, t0 + n) == 0, (t0, n, _lib.lib().ttcd_last_error())
    assert f((1 << 30) - 9, 1 << 30) == 0
    assert f(3, 3) == f(-1, 4) == f(2, 1) == f(0, (1 << 31) - 1) == INV


def test_a_student_window_over_dropped_keys_is_refused():
    """The newest `recent` of the kept keys, and what came after them, are in a row."""
    from ttcd_amd import IPTTCDv9Cache
    c = IPTTCDv9Cache(bits=4, capacity=512, keep=100, recent=20)
    c._spare = object()  # no layers: nothing is evicted but in the counts
    c.reserve(256, None, 256)
    c.advance(90)
    c.reserve(256, None, 256)  # nothing dropped yet: the student sees all there is
    c.advance(170)
    assert (c.seen, c.held, c.run) == (260, 100, 20)
    c.reserve(256, None, 21)
    c.reserve(1, None)
    with pytest.raises(NotImplementedError, match="student"):
        c.reserve(256, None, 22)
    c.advance(1)
    with pytest.raises(NotImplementedError, match="student"):
        c.reserve(256, None, 22)
    assert (c.seen, c.held, c.run) == (261, 100, 20)
    c = IPTTCDv9Cache(bits=4, capacity=64)
    c.advance(500)  # a ring has dropped no key between others
    c.reserve(9, 32, 32)


def test_room_for_a_student_window_wider_than_the_teachers():
    """The student's rows would see as much of their window as the ring happens to hold."""
    from ttcd_amd import IPTTCDv9Cache
    c = IPTTCDv9Cache(bits=4, capacity=320)
    c.reserve(256, 64, 256)  # the prompt's first tokens: all of them are there
    c.advance(256)
    c.reserve(256, 64)       # no student runs: the teacher's window and the call
    with pytest.raises(ValueError, match="positions"):
        c.reserve(256, 64, 256)
    big = IPTTCDv9Cache(bits=4, capacity=511)
    big.advance(5000)
    big.reserve(256, 64, 256)
    with pytest.raises(ValueError, match="positions"):
        big.reserve(256, 64, 258)


def test_a_cache_whose_last_call_did_not_end_is_refused(monkeypatch):
    """Its first layers hold the call's positions and the others do not."""
    from ttcd_amd import IPTTCDv9Cache, kv4
    monkeypatch.setattr(kv4, "KV4Cache", lambda *a, **kw: object())
    monkeypatch.setattr(kv4, "kv4_append", lambda held, k, v: None)
    c = IPTTCDv9Cache(bits=4, capacity=64)
    c.check(1, 2, 64, torch.bfloat16, "cpu")
    for layers in (2, 1):  # a call of both layers, and one that ends behind the first
        c.reserve(5, None)
        for i in range(layers):
            c.append(i, None, None)
        if layers == 2:
            c.advance(5)
    with pytest.raises(RuntimeError, match="did not end"):
        c.reserve(5, None)
    assert (c.seen, c.held) == (5, 5)


def test_eviction_refuses_any_shared_memory():
    """Not only the same pointers: ranges that overlap."""
    kc, ks, vc, vs = 2 * 2 * 64 * 32, 2 * 2 * 64 * 2, 2 * 2 * 64 * 32, 2 * 2 * 64 * 2
    w, index, lens = 2 * 2 * 64 * 4, 2 * 2 * 8 * 4, 8

    def spread(base):
        at, out = base, {}
        for name, n in (("k_codes", kc), ("k_scales", ks), ("v_codes", vc), ("v_scales", vs),
                        ("lengths", lens)):
            out[name], at = at, at + -(-n // 16) * 16
        return out, at

    old, end = spread(P)
    new, last = spread(end + w)
    parts = [(old[n], size) for n, size in zip(old, (kc, ks, vc, vs, lens))] + [(end, w)]
    nw, idx = last, last + w
    f = _lib.lib().ttcd_kv4_evict

    def call(**over):
        a = dict(new, nw=nw, idx=idx, **{})
        a.update(over)
        return f(_struct(**old), end, 8, 2, _struct(**{n: a[n] for n in new}), a["nw"], a["idx"],
                 None)

    for name, size in (("k_codes", kc), ("k_scales", ks), ("v_codes", vc), ("v_scales", vs),
                       ("lengths", lens), ("nw", w), ("idx", index)):
        for at, n in parts:
            # the last and the first 16 bytes (or all) of what is read
            for over in (at + n - min(n, 16), at - size + min(size, 16)):
                if over % 16 == 0 and over > 0:
                    assert call(**{name: over}) == INV, (name, hex(over))
                    assert b"share" in _lib.lib().ttcd_last_error()
    for name, size in (("k_codes", kc), ("v_scales", vs), ("lengths", lens), ("idx", index)):
        assert call(**{name: nw + 16}) == INV  # written twice
    assert call(idx=nw - 16) == INV


def test_rows_past_64_bits_are_refused():
    """Rows whose number, or whose blocks', wraps around to 0: each ended the process with a
    division by it."""
    one, many = _struct(batch=1, kv_heads=1), _struct(batch=16, kv_heads=1)
    f = _lib.lib().ttcd_kv4_attn_workspace_bytes
    assert f(one, 1 << 30, 512, 0) == f(many, 1 << 30, 1 << 30, 0) == 0
    assert f(one, (1 << 31) - 1, (1 << 31) - 1, 0) == 0
    assert _attn(c=many, Tq=1 << 30, Hq=1 << 30) == UNSUP
    assert _weights(c=many, Tq=1 << 30, Hq=1 << 30) == UNSUP
    assert _attn(c=one, Tq=1 << 30, Hq=512) == UNSUP

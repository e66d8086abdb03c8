"""Sampling and the walk over a tree without a GPU: the oracle on cases that are plain by
hand, and the refusals of the C entries and of the Python calls."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import ttcd_amd
from oracle import drafted_ref as ref
from ttcd_amd import _lib

INV, UNSUP = _lib.TTCD_ERR_INVALID_ARGUMENT, _lib.TTCD_ERR_UNSUPPORTED
P = 0x10000  # never dereferenced


def test_the_oracle_samples():
    x = [0.0, math.log(4), -math.inf, math.log(2), math.log(2), math.nan]
    # in order: 1 (4), 3 (2), 4 (2), 0 (1), of 9
    for u, want in ((0.0, 1), (0.44, 1), (0.45, 3), (0.66, 3), (0.67, 4), (0.88, 4), (0.89, 0),
                    (0.999, 0)):
        assert ref.sample(x, u)[0] == want
    assert math.isclose(ref.sample(x, 0.5)[1], math.log(2 / 9))
    assert ref.sample(x, 0.999, top_k=2)[0] == 3 and ref.sample(x, 0.999, top_k=1)[0] == 1
    assert ref.sample(x, 0.999, top_p=0.6)[0] == 3 and ref.sample(x, 0.999, top_p=0.7)[0] == 4
    assert ref.sample(x, 0.999, top_p=0.1)[0] == 1
    assert ref.sample(x, 0.999, top_k=2, top_p=0.6)[0] == 1  # 0.6 of the first two's sum
    assert ref.sample(x, 0.999, min_p=0.4)[0] == 4 and ref.sample(x, 0.999, min_p=0.6)[0] == 1
    assert ref.sample(x, 0.999, temperature=0)[:2] == (1, 0.0)
    assert ref.sample([-math.inf, math.nan], 0.5) == (-1, -math.inf)
    assert ref.sample([1.0, math.inf, math.inf], 0.6)[0] == 2


def test_the_oracle_walks():
    parents, tokens = [-1, 0, 0, 1, 2, 4], [9, 5, 6, 7, 8, 3]
    assert ref.accept(parents, tokens, [6, 0, 8, 0, 3, 1], 6) == ([0, 2, 4, 5], 1)
    assert ref.accept(parents, tokens, [6, 0, 8, 0, 3, 1], 4) == ([0, 2], 8)
    assert ref.accept(parents, tokens, [4, 0, 8, 0, 3, 1], 6) == ([0], 4)
    assert ref.accept(parents, tokens, [4, 0, 8, 0, 3, 1], 0) == ([], -1)
    assert ref.lineage([-1, 0, 1, 0, 9, -7]) == [[0], [0, 1], [0, 1, 2], [0, 3], [4], [5]]


def _sample(x=P, st=100, R=2, V=100, u=P, ts=None, t=1.0, ks=None, k=0, ps=None, p=1.0, ms=None,
            m=0.0, tok=P, lp=None, dt=0):
    return _lib.lib().ttcd_sample_fwd(x, st, R, V, u, ts, t, ks, k, ps, p, ms, m, tok, lp, dt, None)


def test_bad_arguments():
    assert _sample(x=None) == _sample(u=None) == _sample(tok=None) == INV
    assert _sample(R=0) == _sample(V=0) == _sample(st=-1) == _sample(x=P + 1) == INV
    assert _sample(t=-0.5) == _sample(t=math.nan) == _sample(k=-1) == INV
    assert _sample(p=0.0) == _sample(p=math.nan) == _sample(m=-0.1) == _sample(m=1.5) == INV
    assert _sample(m=math.nan) == INV
    assert _sample(V=(1 << 20) + 1) == _sample(dt=2) == _sample(dt=9) == UNSUP

    def walk(a=P, b=P, c=P, d=P, e=P, f=P, B=1, N=4):
        return _lib.lib().ttcd_tree_accept(a, b, c, None, d, e, f, B, N, None)
    assert walk(a=None) == walk(b=None) == walk(c=None) == walk(d=None) == walk(e=None) == INV
    assert walk(f=None) == walk(B=0) == walk(N=0) == INV
    assert walk(N=257) == UNSUP
    # more threads than a launch has
    assert _sample(R=1 << 22) == _sample(R=2 ** 31 - 1) == UNSUP
    assert walk(B=1 << 26) == walk(B=2 ** 31 - 1) == UNSUP


def test_python_refuses_the_cpu():
    with pytest.raises(ValueError, match="GPU"):
        ttcd_amd.sample(torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(2))
    with pytest.raises(ValueError, match="GPU"):
        ttcd_amd.tree_accept(torch.zeros(1, 2, dtype=torch.int32), None, None)


C = dict(k_codes=P, k_scales=P, v_codes=P, v_scales=P, lengths=P, batch=2, kv_heads=2, head_dim=64,
         capacity=64)
Q = 0x100000
D = dict(C, k_codes=Q, k_scales=Q, v_codes=Q, v_scales=Q, lengths=Q)
ST = (64 * 4 * 8, 64 * 4, 64, 1)


def _struct(fields):
    return ctypes.byref(_lib.KV4CacheStruct(**fields))


def _attn(c=C, d=D, q=P, o=P, N=4, Hq=4, qs=ST, os=ST, parents=P, scale=0.125, dt=0):
    return _lib.lib().ttcd_kv4_tree_attn_fwd(
        _struct(c), _struct(d), q, o, None, N, Hq, _lib.strides4(qs), _lib.strides4(os), parents,
        None, 0, scale, dt, None, 0, None)


def _commit(c=C, d=D, path=P, n=4):
    return _lib.lib().ttcd_kv4_commit(_struct(c), _struct(d), path, None, n, None, 0, None)


@pytest.mark.parametrize("call", [_attn, _commit])
@pytest.mark.parametrize("over,status", [
    ({"k_codes": 0}, INV), ({"lengths": 0}, INV), ({"head_dim": 96}, UNSUP), ({"capacity": 48}, INV),
    ({"k_codes": P + 8}, UNSUP), ({"lengths": P + 1}, UNSUP), ({"batch": 1}, INV),
    ({"kv_heads": 1}, INV), ({"head_dim": 128}, INV)])
def test_caches_that_do_not_fit(call, over, status):
    assert call(c=dict(C, **over)) == status
    assert call(d=dict(D, **over)) == status


@pytest.mark.parametrize("call", [_attn, _commit])
def test_caches_that_share_memory(call):
    assert call(d=C) == INV
    for part in ("k_codes", "k_scales", "v_codes", "v_scales", "lengths"):
        assert call(d=dict(D, **{part: P})) == INV


def test_bad_trees():
    assert _attn(q=None) == _attn(o=None) == _attn(parents=None) == _attn(N=0) == _attn(Hq=3) == INV
    assert _attn(scale=0.0) == _attn(scale=math.nan) == _attn(N=65) == INV  # the draft holds 64
    assert _attn(d=dict(D, capacity=512), N=257) == UNSUP
    assert _attn(qs=(ST[0], ST[1], 60, 1)) == _attn(o=P + 8) == _attn(dt=2) == UNSUP
    assert _commit(path=None) == _commit(n=0) == _commit(n=65) == INV
    assert _commit(d=dict(D, capacity=32), n=33) == INV
    f = _lib.lib().ttcd_kv4_tree_attn_workspace_bytes
    assert f(_struct(C), 4, 4, 0) == f(None, 4, 4, 0) == f(_struct(C), 0, 4, 0) == 0
    long = dict(C, capacity=1 << 16)
    assert f(_struct(long), 4, 4, 0) > 0 and f(_struct(long), 257, 4, 0) == 0


def test_python_refuses_other_caches():
    x = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16)
    i = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="KV4Cache"):
        ttcd_amd.kv4_tree_attn(x, None, None, i)
    with pytest.raises(ValueError, match="KV4Cache"):
        ttcd_amd.kv4_commit(None, None, i)

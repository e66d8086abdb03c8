"""The C entries of trees of drafted tokens over the 4-bit cache without a GPU: what they refuse,
and how much workspace a split takes."""
from __future__ import annotations

import ctypes
import math

import pytest

from ttcd_amd import _lib

INV, UNSUP = _lib.TTCD_ERR_INVALID_ARGUMENT, _lib.TTCD_ERR_UNSUPPORTED
P = 0x10000  # never dereferenced


def _cache(at=1, B=2, H=2, D=64, C=64):
    """A cache whose parts lie from at * 2^40 on, each far from the others."""
    p = [(at << 40) + (i << 36) for i in range(5)]
    return _lib.KV4CacheStruct(*p, B, H, D, C)


def _tree(c=None, d=None, q=P, o=P, N=8, Hq=4, qs=(2048, 256, 64, 1), os=(2048, 256, 64, 1),
          parents=P, window=0, sm=0.125, dt=0):
    c, d = c or _cache(), d or _cache(2)
    return _lib.lib().ttcd_kv4_tree_attn_fwd(
        ctypes.byref(c), ctypes.byref(d), q, o, None, N, Hq, _lib.strides4(qs), _lib.strides4(os),
        parents, None, window, sm, dt, None, 0, None)


def test_tree_refusals():
    assert _tree(q=None) == _tree(o=None) == _tree(parents=None) == INV
    assert _tree(N=0) == _tree(Hq=0) == _tree(Hq=3) == INV
    assert _tree(N=257, d=_cache(2, C=512)) == _tree(q=P + 2) == _tree(qs=(2048, 256, 63, 1)) == UNSUP
    assert _tree(N=65) == INV  # more than the draft has slots
    assert _tree(sm=0.0) == _tree(sm=math.inf) == _tree(sm=math.nan) == INV
    assert _tree(dt=2) == UNSUP
    for other in (_cache(2, B=3), _cache(2, H=1), _cache(2, D=128), _cache(1)):
        assert _tree(d=other) == INV
    shifted = _cache(2)
    shifted.v_codes = _cache().k_codes + 64  # within the cache's
    assert _tree(d=shifted) == INV


def _commit(c=None, d=None, path=P, n=4):
    c, d = c or _cache(), d or _cache(2)
    return _lib.lib().ttcd_kv4_commit(ctypes.byref(c), ctypes.byref(d), path, None, n, None, 0, None)


def test_commit_refusals():
    assert _commit(path=None) == _commit(n=0) == _commit(n=65) == INV
    assert _commit(n=40, c=_cache(C=32)) == _commit(n=40, d=_cache(2, C=32)) == INV
    assert _commit(d=_cache()) == _commit(d=_cache(2, B=1)) == INV


def _bytes(B, H, D, C, N, Hq, window=0):
    c = _cache(B=B, H=H, D=D, C=C)
    return _lib.lib().ttcd_kv4_tree_attn_workspace_bytes(ctypes.byref(c), N, Hq, window)


@pytest.mark.parametrize("B,H,D,C,N,Hq,window,units", [
    (8, 8, 128, 16384, 16, 16, 0, 64), (1, 8, 128, 16384, 16, 16, 8192, 64),
    (4, 8, 128, 12288, 64, 16, 8192, 64), (64, 2, 64, 2048, 8, 4, 0, 256),
    (65, 2, 64, 2048, 8, 4, 0, 0), (8, 8, 128, 1024, 16, 16, 0, 0)])
def test_workspace(B, H, D, C, N, Hq, window, units):
    """units parts of every row: sums, the maximum and the sum, and each sequence's share."""
    assert _bytes(B, H, D, C, N, Hq, window) == (
        units * Hq * N * (D + 2) * 4 + B * 8 if units else 0)


def test_no_split_of_more_rows_than_a_launch_sums():
    """The sum over the parts gives a row 64 threads, and a launch has fewer than 2^32."""
    assert _bytes(64, 1, 64, 65536, 256, 4095) > 0
    assert _bytes(64, 1, 64, 65536, 256, 4096) == 0
    assert _bytes(1, 1, 64, 65536, 256, 1 << 18) == 0

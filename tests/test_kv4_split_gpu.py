"""Attention over the 4-bit cache where its keys are split over workgroups, and
selections of every register count, against the float64 oracle with the bounds of
test_kv4_gpu.py. Each case first asks the library how it would split it, so that a
change of the plan cannot leave a path untested unnoticed."""
from __future__ import annotations

import math

import pytest
import torch

from test_kv4_gpu import (BF, E, HF, U, _check_attn, _evict_case, _pair, _rand,
                          _score_error)
from ttcd_amd import KV4Cache, _lib, kv4_append, kv4_attn, kv4_key_weights, kv4_read

pytestmark = pytest.mark.gpu


def _parts(c, T, Hq, window):
    """Parts of the keys in which the call is swept: 0 for a call that is not split."""
    n = _lib.lib().ttcd_kv4_attn_workspace_bytes(c._ref, T, Hq, window or 0)
    return n // (c.batch * T * Hq * (c.head_dim + 2) * 4)


def _case(c, r, T, Hq, window, counts, seed):
    q = _rand(seed, r.B, T, Hq, r.D, dtype=r.dtype, scale=1.5)
    n = None if counts is None else torch.tensor(counts, dtype=torch.int32)
    if n is not None:
        for b in range(r.B):
            q[b, n[b]:] = math.nan
    nc, qc = None if n is None else n.cuda(), q.cuda()
    got = kv4_attn(qc, c, window, counts=nc, return_lse=True)
    _check_attn(r, q, *got, window, n)
    whole = kv4_attn(qc, c, window, counts=nc, return_lse=True, split_keys=False)
    _check_attn(r, q, *whole, window, n)
    for _ in range(8):  # no sum depends on who comes first
        for split, want in ((True, got), (False, whole)):
            for x, y in zip(kv4_attn(qc, c, window, counts=nc, return_lse=True,
                                     split_keys=split), want):
                assert torch.equal(x, y)


MANY = [  # over 32 rows a kv head, 2 to 16 parts and 1024 rows or more: summed a row a wavefront
    # B, T, Hq, H, D, C, lengths, window, counts, dtype
    (2, 100, 8, 4, 128, 4096, (4096, 70), None, None, BF),         # the second's parts empty
    (2, 100, 8, 4, 64, 4096, (9000, 150), None, (100, 41), HF),
    (3, 90, 6, 2, 64, 4096, (4000, 90, 2500), 1500, (90, 0, 7), BF),
    (3, 90, 6, 2, 128, 4096, (1, 4096, 13000), 1500, (1, 90, 66), HF),
    (4, 70, 8, 2, 64, 2048, (2048, 0, 2047, 33), None, None, BF),
    (1, 150, 15, 5, 64, 4096, (4000,), None, None, HF),            # an odd group
    (3, 130, 4, 4, 128, 2048, (2048, 130, 5000), 1000, None, BF),
]


@pytest.mark.parametrize("B,T,Hq,H,D,C,lengths,window,counts,dtype", MANY)
def test_many_rows_in_a_few_parts(gpu, B, T, Hq, H, D, C, lengths, window, counts, dtype):
    c, r = _pair(B, H, D, C, dtype, lengths, seed=T)
    assert T * Hq // H > 32 and B * T * Hq >= 1024 and 2 <= _parts(c, T, Hq, window) <= 16
    _case(c, r, T, Hq, window, counts, seed=T + 1)


@pytest.mark.parametrize("B,T,Hq,H,D,C,lengths,window,counts,dtype", [
    (1, 40, 2, 1, 64, 16384, (16000,), None, None, HF),
    (1, 35, 1, 1, 128, 16384, (20000,), None, None, BF),
    (2, 40, 2, 1, 64, 16384, (100, 16384), 8000, (40, 3), BF),
])
def test_many_rows_in_many_parts(gpu, B, T, Hq, H, D, C, lengths, window, counts, dtype):
    c, r = _pair(B, H, D, C, dtype, lengths, seed=T)
    assert T * Hq // H > 32 and _parts(c, T, Hq, window) > 16
    _case(c, r, T, Hq, window, counts, seed=T + 1)


@pytest.mark.parametrize("B,T,Hq,H,D,C,lengths,window,counts,dtype", [
    (1, 5, 16, 4, 128, 8192, (8000,), None, None, BF),             # two row tiles, 20 rows
    (2, 3, 16, 2, 64, 8192, (11000, 40), None, None, HF),
    (1, 20, 1, 1, 64, 16384, (16384,), None, None, BF),
    (1, 1, 32, 1, 128, 32768, (32768,), None, None, HF),           # 64 parts
    (2, 12, 4, 2, 128, 4096, (4096, 700), 3000, (5, 12), BF),
])
def test_two_row_tiles_over_many_keys(gpu, B, T, Hq, H, D, C, lengths, window, counts, dtype):
    """17 to 32 rows a kv head: several tiles a wavefront, whose running maxima move, in
    parts and in one."""
    c, r = _pair(B, H, D, C, dtype, lengths, seed=T)
    assert 16 < T * Hq // H <= 32 and _parts(c, T, Hq, window) > 1
    _case(c, r, T, Hq, window, counts, seed=T + 1)


@pytest.mark.parametrize("D,dtype", [(64, BF), (128, HF)])
def test_one_row_in_64_parts(gpu, D, dtype):
    c, r = _pair(1, 1, D, 65536, dtype, (65000,), seed=5)
    assert _parts(c, 1, 2, None) == 64
    _case(c, r, 1, 2, None, None, seed=6)


@pytest.mark.parametrize("T", [3, 40])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_scores_that_grow_along_the_keys_of_several_row_tiles(gpu, T, dtype):
    """Maxima that move at every tile of a wavefront, by more and less than the lazy limit.

    One key is 88 and more (in the exponent of e) above all others for some rows, and where
    its value is 0 the result is a sum of n probabilities under 2^-126, the least normal
    number of fp32 and bf16, which the exponential and the product take as 0. The sum of
    a row's probabilities is 1 and more (its reference is some key's own score), so that is
    at most n 2^-126 max |v|, beside the bounds of _check_attn, which know no underflow."""
    c, r = _pair(1, 1, 64, 4096, dtype)
    k = _rand(1, 1, 4096, 1, 64, dtype=dtype) * torch.linspace(0.1, 6, 4096)[:, None, None]
    k[0, 3003] *= 4
    k, v = k.to(dtype), _rand(2, 1, 4096, 1, 64, dtype=dtype)
    kv4_append(c, k.cuda(), v.cuda())
    r.append(k, v)
    q = _rand(3, 1, T, 8, 64, dtype=dtype, scale=3.0)
    for split in (False, True):
        o, lse = kv4_attn(q.cuda(), c, return_lse=True, split_keys=split)
        want, wl, mag = r.attn(q)
        d, chain, top = _score_error(r, q)[0], (4096 / 8 + 64) * E, r.rows[0][1].abs().max()
        limit = U[dtype] * want.abs() + (U[dtype] + 4 * d + chain) * mag + 4096 * 2.0 ** -126 * top
        if dtype == HF:
            limit += 4096 * 2.0 ** -32 * top
        assert ((o.double().cpu() - want).abs() <= limit).all()
        assert ((lse.double().cpu() - wl).abs() <= 2 * d + chain + 8 * E * (1 + wl.abs())).all()
        w = kv4_key_weights(q.cuda(), c, lse).double().cpu().sum(-1)
        assert (w - T * 8).abs().max() <= 1e-3 * T * 8


@pytest.mark.parametrize("D,dtype", [(64, HF), (128, BF)])
@pytest.mark.parametrize("T", [1, 12])
def test_many_keys_of_a_cache_past_the_last_level_cache(gpu, D, dtype, T):
    """Read past the caches and through them: the bits of a small cache with the same
    window of positions, in as many parts, and the oracle's numbers."""
    H, Hq, W, start = 8, 16, 3000, 262144 * 2 - 1000
    big, small = KV4Cache(1, H, D, 262144, dtype), KV4Cache(1, H, D, 4096, dtype)
    r = _pair(1, H, D, 4096, dtype)[1]
    k, v = (_rand(i, 1, 3100, H, D, dtype=dtype) for i in (1, 2))
    r.append(k, v)
    q = _rand(3, 1, T, Hq, D, dtype=dtype)
    out = []
    for c in (big, small):
        c.lengths.fill_(start)
        kv4_append(c, k.cuda(), v.cuda())
        out.append(kv4_attn(q.cuda(), c, W, return_lse=True) + kv4_read(c, 3100))
    assert _parts(big, T, Hq, W) == _parts(small, T, Hq, W) > 1
    for x, y in zip(*out):
        assert torch.equal(x, y)
    _check_attn(r, q, out[0][0], out[0][1], W, None)


@pytest.mark.parametrize("C,lengths,keep,recent", [
    (8224, (8224, 30000), 4000, 100), (12288, (12288, 9000), 6000, 0),
    (32768, (40000, 1001), 16384, 1024), (32768, (32768, 8193), 100, 50)])
def test_evict_of_caches_of_8193_to_32768_slots(gpu, C, lengths, keep, recent):
    c, r = _pair(2, 1, 64, C, BF, lengths)
    g = torch.Generator().manual_seed(C + keep)
    w = torch.rand(2, 1, C, generator=g)
    ties = (w * 7).floor()
    odd = (w - 0.5) * 1e-3
    odd[..., ::7], odd[..., 5::11], odd[..., 6::11] = -0.0, math.nan, -math.inf
    for x in (w.log().square(), ties, odd, torch.zeros(2, 1, C)):
        _evict_case(c, r, x.cuda(), keep, recent)


def test_graphs_of_split_calls_replay_at_once(gpu):
    """One call of each kernel and sum captured, each graph with its workspace, replayed on
    streams of their own over one cache, several times, with eager calls between."""
    c, r = _pair(2, 2, 128, 8192, BF, (8192, 6000))
    qs = [_rand(i, 2, T, 8, 128) for i, T in ((1, 1), (2, 7), (3, 10), (4, 130))]
    want = [kv4_attn(q.cuda(), c, return_lse=True) for q in qs]
    graphs, inputs = [], [q.cuda() for q in qs]
    for q, x, w in zip(qs, inputs, want):
        assert _parts(c, q.shape[1], 8, None) > 1
        _check_attn(r, q, *w, None, None)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = kv4_attn(x, c, return_lse=True)
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        torch.cuda.synchronize()
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                for _ in range(4):
                    g.replay()
        torch.cuda.synchronize()
        for (_, out), w in zip(graphs, want):
            for x, y in zip(out, w):
                assert torch.equal(x, y)
                x.zero_()
        assert torch.equal(kv4_attn(inputs[3], c), want[3][0])


def test_a_captured_follow_up_goes_by_the_lengths_it_finds(gpu):
    """Append of a chunk (lengths by a second launch), split attention of many rows, key
    weights: each replay is the next chunk, over the ring's end and past empty parts."""
    B, T, Hq, H, D, C = 2, 130, 8, 4, 64, 2048
    c, r = _pair(B, H, D, C, HF, (1900, 3), weights=True)
    assert 1 < _parts(c, T, Hq, None) <= 16
    k, v, q = (torch.zeros(B, T, h, D, dtype=HF, device=gpu) for h in (H, H, Hq))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kv4_append(c, k, v)
        o, lse = kv4_attn(q, c, return_lse=True)
        w = kv4_key_weights(q, c, lse)
    for i in range(4):
        new = [_rand(7 * i + j, B, T, h, D, dtype=HF) for j, h in enumerate((H, H, Hq))]
        for x, y in zip((k, v, q), new):
            x.copy_(y)
        g.replay()
        torch.cuda.synchronize()
        r.append(new[0], new[1])
        _check_attn(r, new[2], o, lse, None, None)
        seen = torch.full((B, H), T * Hq / H, dtype=torch.float64)
        assert ((w.double().sum(-1).cpu() - seen).abs() <= 1e-3 * seen).all()
        for x, y in zip(kv4_attn(q, c, return_lse=True), (o, lse)):
            assert torch.equal(x, y)

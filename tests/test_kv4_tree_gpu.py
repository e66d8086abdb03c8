"""Attention of a tree of drafted tokens over the 4-bit cache and the commit of its accepted
nodes on the GPU against the float64 oracle, with test_kv4_gpu's bounds (a node's sum runs
over the cache and its ancestors, one key after the other as there)."""
from __future__ import annotations

import math

import pytest
import torch

import ttcd_amd
from oracle import drafted_ref, kv4_ref
from test_kv4_gpu import BF, E, HF, U, _pair, _rand
from ttcd_amd import (KV4Cache, kv4_append, kv4_attn, kv4_commit, kv4_read, kv4_tree_attn,
                      sample, tree_accept)

pytestmark = pytest.mark.gpu


def _trees(seed, B, N, back=6):
    """(B, N): every node's parent is one of the `back` before it; some are roots."""
    g = torch.Generator().manual_seed(seed)
    p = torch.full((B, N), -1, dtype=torch.int32)
    for b in range(B):
        for i in range(1, N):
            if torch.rand((), generator=g) < 0.95:
                p[b, i] = i - 1 - int(torch.randint(0, min(i, back), (), generator=g))
    return p


def _drafted(c, N, seed, counts=None, cap=None):
    """A draft of N nodes for the cache c, the slots behind them garbage, and its oracle."""
    cap = cap or 32 * ((N + 31) // 32)
    d, r = _pair(c.batch, c.kv_heads, c.head_dim, cap, c.dtype)
    k, v = (_rand(seed + j, c.batch, N, c.kv_heads, c.head_dim, dtype=c.dtype, scale=1 + 2 * j)
            for j in (0, 1))
    n = None if counts is None else torch.tensor(counts, dtype=torch.int32)
    kv4_append(d, k.cuda(), v.cuda(), counts=None if n is None else n.cuda())
    r.append(k, v, n)
    return d, r


def _check(r, rd, q, parents, o, lse, window, counts):
    want, wl, mag = drafted_ref.tree_attn(r, rd, q, parents, window, counts)
    keys = max(r.length(b) + rd.length(b) for b in range(r.B))
    chain = (keys / 8 + 64) * E
    u, G = U[r.dtype], q.shape[2] // r.H
    d = []
    for b in range(r.B):
        k = torch.cat((r.rows[b][0], rd.rows[b][0])).abs().repeat_interleave(G, 1)
        s = torch.einsum("thd,lhd->htl", q[b].double().cpu().abs().nan_to_num(0), k)
        d.append((r.D + 4) * E * (s.max().item() if s.numel() else 0.0) * r.D ** -0.5)
    d = torch.tensor(d)[:, None, None]
    limit = u * want.abs() + (u + 4 * d[..., None] + chain) * mag
    if r.dtype == HF:
        limit += torch.tensor([keys * 2.0 ** -32 * max((x[1].abs().max().item() for x in
                                                        (r.rows[b], rd.rows[b]) if len(x[1])),
                                                       default=0.0)
                               for b in range(r.B)])[:, None, None, None]
    assert o.shape == q.shape and o.dtype == r.dtype
    bad = ((o.double().cpu() - want).abs() - limit).max().item()
    assert bad <= 0, bad
    empty = wl == -math.inf
    assert torch.equal(lse.cpu() == -math.inf, empty)
    ll = 2 * d + chain + 8 * E * (1 + wl.masked_fill(empty, 0).abs())
    assert ((lse.double().cpu() - wl).masked_fill(empty, 0).abs() <= ll).all()


CASES = [
    # B, N, Hq, H, D, capacity, lengths, window, counts
    (1, 1, 2, 2, 64, 32, (0,), None, None),
    (1, 1, 4, 2, 128, 64, (33,), None, None),
    (3, 8, 4, 2, 64, 64, (0, 31, 200), None, None),
    (3, 8, 4, 2, 128, 64, (0, 31, 200), 5, (8, 3, 0)),
    (2, 16, 2, 2, 128, 96, (96, 97), 40, None),
    (2, 7, 6, 2, 64, 64, (64, 5), 1, None),         # a window of the node itself
    (2, 17, 4, 2, 128, 128, (100, 400), 3, (17, 16)),
    (2, 16, 4, 2, 128, 2048, (2000, 1), None, None),  # split
    (1, 31, 2, 2, 64, 4096, (9000,), 1500, None),
    (2, 11, 6, 2, 128, 96, (50, 0), None, None),    # 33 rows: the other kernel
    (2, 33, 4, 2, 64, 160, (159, 3), 20, (33, 32)),
    (2, 64, 4, 2, 128, 96, (96, 500), None, None),
    (1, 65, 2, 1, 64, 2048, (2048,), 700, None),
    (2, 100, 6, 2, 128, 128, (0, 128), 7, (100, 64)),
    (1, 256, 4, 2, 64, 96, (40,), None, None),
    (2, 256, 4, 2, 128, 1536, (1500, 4000), 300, (256, 129)),
    (1, 64, 4, 2, 128, 4096, (4096,), None, None),
    (1, 64, 4, 2, 128, 4096, (70,), 10, None),      # most parts find nothing
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("B,N,Hq,H,D,C,lengths,window,counts", CASES)
def test_trees_match_64_bits(gpu, B, N, Hq, H, D, C, lengths, window, counts, dtype):
    c, r = _pair(B, H, D, C, dtype, lengths, seed=N)
    d, rd = _drafted(c, N, N + 1, counts)
    q = _rand(N + 9, B, N, Hq, D, dtype=dtype, scale=1.5)
    n = None if counts is None else torch.tensor(counts, dtype=torch.int32).cuda()
    for back in (1, 6, 300):  # a chain, a bush, anything
        parents = _trees(N + back, B, N, back)
        for split in (True, False):
            o, lse = kv4_tree_attn(q.cuda(), c, d, parents.cuda(), window, counts=n,
                                   return_lse=True, split_keys=split)
            _check(r, rd, q, parents, o, lse, window, counts)
        assert torch.equal(o, kv4_tree_attn(q.cuda(), c, d, parents.cuda(), window, counts=n,
                                            split_keys=False))


@pytest.mark.parametrize("D,Hq,H,N", [(64, 3, 1, 4), (128, 4, 2, 16), (128, 4, 2, 40)])
@pytest.mark.parametrize("window", [None, 6, 50])
def test_a_chain_is_the_tokens_appended(gpu, D, Hq, H, N, window):
    """A chain's nodes see what the same tokens see that are appended to the cache; and a
    commit of all is that append, bit by bit."""
    c, r = _pair(2, H, D, 96, BF, (70, 200))
    one, _ = _pair(2, H, D, 96, BF, (70, 200))
    k, v = _rand(3, 2, N, H, D).cuda(), _rand(4, 2, N, H, D).cuda()
    q = _rand(5, 2, N, Hq, D)
    d, rd = _pair(2, H, D, 64, BF)
    kv4_append(d, k, v)
    rd.append(k, v)
    parents = (torch.arange(N, dtype=torch.int32) - 1).expand(2, N)
    o, lse = kv4_tree_attn(q.cuda(), c, d, parents.cuda(), window, return_lse=True)
    _check(r, rd, q, parents, o, lse, window, None)
    kv4_append(one, k, v)
    if window is not None:  # without one, the ring drops what the first tokens would see
        w, wl = kv4_attn(q.cuda(), one, window, return_lse=True)
        if window + N <= 96:
            assert (o.double() - w.double()).abs().max() <= 4 * U[BF] * w.abs().max().double()
            assert (lse - wl).abs().max() < 1e-4
    kv4_commit(c, d, torch.arange(N, dtype=torch.int32).expand(2, N).contiguous().cuda())
    assert torch.equal(c.lengths, one.lengths) and d.lengths.tolist() == [N, N]
    for a, b in zip((c.k_codes, c.k_scales, c.v_codes, c.v_scales),
                    (one.k_codes, one.k_scales, one.v_codes, one.v_scales)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("N,Hq", [(8, 2), (20, 4), (64, 4)])
def test_malformed_trees_and_lengths_read_nothing_wrong(gpu, N, Hq):
    """A parent that does not come before its node is none; nodes that the draft does not hold
    are none; lengths out of range are the nearest."""
    c, r = _pair(2, 2, 128, 64, BF, (10, 64))
    d, rd = _drafted(c, N, 1)
    q = _rand(2, 2, N, Hq, 128)
    parents = _trees(1, 2, N)
    for i, x in ((0, 5), (1, 1), (2, 2 ** 31 - 1), (3, -2 ** 31), (4, 4), (5, N), (6, 0)):
        parents[:, i] = x
    o, lse = kv4_tree_attn(q.cuda(), c, d, parents.cuda(), return_lse=True)
    _check(r, rd, q, parents, o, lse, None, None)
    d.lengths.copy_(torch.tensor([3, -9], dtype=torch.int32))
    few = kv4_ref.Ref(2, 2, 128, d.capacity, BF)
    few.rows = [tuple(x[:3] for x in rd.rows[0]), tuple(x[:0] for x in rd.rows[1])]
    o, lse = kv4_tree_attn(q.cuda(), c, d, parents.cuda(), return_lse=True)
    _check(r, few, q, parents, o, lse, None, (3, 0))
    d.lengths.fill_(2 ** 31 - 1)
    counts = torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32).cuda()
    o, lse = kv4_tree_attn(q.cuda(), c, d, parents.cuda(), counts=counts, return_lse=True)
    _check(r, rd, q, parents, o, lse, None, (N, 0))


@pytest.mark.parametrize("N,Hq", [(5, 2), (12, 4), (40, 4)])
def test_nan_queries_stay_in_their_row(gpu, N, Hq):
    c, r = _pair(1, 2, 64, 64, BF, (50,))
    d, rd = _drafted(c, N, 1)
    q = _rand(2, 1, N, Hq, 64)
    parents = _trees(3, 1, N)
    o = kv4_tree_attn(q.cuda(), c, d, parents.cuda())
    q[0, 2, 1] = math.nan
    p = kv4_tree_attn(q.cuda(), c, d, parents.cuda())
    assert torch.isnan(p[0, 2, 1]).all()
    p[0, 2, 1] = o[0, 2, 1]
    assert torch.equal(o, p)


def test_views_and_odd_addresses(gpu):
    c, r = _pair(2, 2, 64, 64, BF, (20, 64))
    d, rd = _drafted(c, 9, 1)
    parents = _trees(2, 2, 9)
    wide = _rand(3, 2, 9, 12, 64).cuda()
    odd = torch.empty(2 * 9 * 4 * 64 + 1, dtype=BF, device="cuda")[1:].view(2, 9, 4, 64)
    odd.copy_(wide[:, :, 4:8])
    for q in (wide[:, :, 4:8], odd, wide[:, :, 4:8].transpose(1, 2).contiguous().transpose(1, 2)):
        o, lse = kv4_tree_attn(q, c, d, parents.cuda(), 30, return_lse=True)
        _check(r, rd, q.cpu(), parents, o, lse, 30, None)
    skewed = torch.zeros(2, 18, dtype=torch.int32, device="cuda")
    skewed[:, ::2] = parents.cuda()
    assert torch.equal(kv4_tree_attn(q, c, d, skewed[:, ::2], 30), o)


@pytest.mark.parametrize("dtype,D,H", [(BF, 128, 2), (HF, 64, 3)])
@pytest.mark.parametrize("P,N,counts", [(1, 1, None), (3, 8, (3, 0, 1)), (5, 33, (5, 2, 9)),
                                        (64, 64, (64, 63, -2)), (250, 256, None)])
def test_commit_moves_the_bits(gpu, dtype, D, H, P, N, counts):
    """Accepted nodes become the next positions; no other slot changes, the draft neither."""
    c, r = _pair(3, H, D, 256, dtype, (0, 255, 700), weights=True)
    c.weights.fill_(7.0)
    d, rd = _drafted(c, N, 2)
    path = torch.stack([torch.randperm(N, generator=torch.Generator().manual_seed(b))[:P]
                        for b in range(3)]).int()
    taken = [P if counts is None else min(max(counts[b], 0), P) for b in range(3)]
    before = [t.clone() for t in (c.k_codes, c.k_scales, c.v_codes, c.v_scales)]
    held = [t.clone() for t in (d.k_codes, d.k_scales, d.v_codes, d.v_scales, d.lengths)]
    junk = path.clone()
    for b in range(3):
        junk[b, taken[b]:] = torch.tensor(2 ** 31 - 1)
    kv4_commit(c, d, junk.cuda(),
               None if counts is None else torch.tensor(counts, dtype=torch.int32).cuda())
    old = [r.length(b) for b in range(3)]
    for b in range(3):
        r.rows[b] = tuple(torch.cat((x, y[path[b, :taken[b]].long()]))
                          for x, y in zip(r.rows[b], rd.rows[b]))
    assert c.lengths.tolist() == [n + t for n, t in zip(old, taken)]
    for x, y in zip(kv4_read(c, 256), r.read(256)):
        assert torch.equal(x.cpu(), y)
    for b in range(3):
        other = torch.ones(256, dtype=torch.bool)
        other[(old[b] + torch.arange(taken[b])) % 256] = False
        for now, was, is_v in zip((c.k_codes, c.k_scales, c.v_codes, c.v_scales), before,
                                  (0, 0, 1, 1)):
            s = other.nonzero().flatten().cuda()
            if is_v:
                assert torch.equal(now[b][:, s // 4, :, s % 4], was[b][:, s // 4, :, s % 4])
            else:
                assert torch.equal(now[b][:, s], was[b][:, s])
        assert (c.weights[b].cpu() == torch.where(other, 7.0, 0.0)).all()
    for t, was in zip((d.k_codes, d.k_scales, d.v_codes, d.v_scales, d.lengths), held):
        assert torch.equal(t, was)


@pytest.mark.parametrize("P", [4, 256])
def test_commit_of_malformed_paths_and_resets(gpu, P):
    c, _ = _pair(2, 8, 64, 256, BF, (9, 300))
    d, rd = _drafted(c, 256, 1)
    path = torch.arange(P, dtype=torch.int32).expand(2, P).clone()
    path[0, 0], path[0, 1], path[1, 2] = -1, 2 ** 31 - 1, -2 ** 31
    kv4_commit(c, d, path.cuda(), reset=True)
    assert c.lengths.tolist() == [9 + P, 300 + P] and d.lengths.tolist() == [0, 0]
    k, v = (x.cpu() for x in kv4_read(c, P))
    for i, want in ((0, k), (1, v)):
        for b in range(2):
            assert torch.equal(rd.rows[b][i][path[b].clamp(0, 255).long()].to(BF), want[b])


def test_a_ring_goes_on_past_the_largest_length(gpu):
    c, _ = _pair(1, 2, 64, 96, BF, (96,))
    d, rd = _drafted(c, 8, 1)
    top = 2 ** 30
    c.lengths.fill_(top - 3)
    kv4_commit(c, d, torch.arange(8, dtype=torch.int32)[None].cuda())
    n = c.lengths.item()
    assert 96 <= n < top and (n - (top + 5)) % 96 == 0
    assert torch.equal(kv4_read(c, 8)[0].cpu()[0], rd.rows[0][0].to(BF))


def test_offsets_past_32_bits(gpu):
    """A cache whose codes pass 4 GB: the last head's rows."""
    B, H, D, C = 1, 8, 128, 9 << 20
    c = KV4Cache(B, H, D, C)
    assert c.k_codes.numel() > 1 << 32
    c.lengths.fill_(C - 20)
    k, v = _rand(1, 1, 20, H, D), _rand(2, 1, 20, H, D)
    kv4_append(c, k.cuda(), v.cuda())  # the last 20 slots
    r = kv4_ref.Ref(B, H, D, C)
    r.append(k, v)
    for N, Hq in ((6, 16), (24, 16)):
        d, rd = _drafted(c, N, 5)
        q, parents = _rand(3, 1, N, Hq, D), (torch.arange(N, dtype=torch.int32) - 1)[None]
        o, lse = kv4_tree_attn(q.cuda(), c, d, parents.cuda(), 20, return_lse=True)
        _check(r, rd, q, parents, o, lse, 20, None)
        assert torch.isfinite(o).all()
    kv4_commit(c, d, torch.arange(5, dtype=torch.int32)[None].cuda())  # into the first slots
    assert torch.equal(kv4_read(c, 5)[0].cpu()[0], rd.rows[0][0][:5].to(BF))
    del c
    torch.cuda.empty_cache()


def test_a_captured_step_verifies_on(gpu):
    """append to the draft, attention, sampling, the walk and the commit in one graph, replayed
    over other tokens and trees, against the same calls eagerly; eager work between replays."""
    B, N, Hq, H, D, V = 2, 12, 4, 2, 64, 500
    caches = [_pair(B, H, D, 2048, BF, (1990, 40))[0] for _ in range(2)]
    drafts = [KV4Cache(B, H, D, 32) for _ in range(2)]
    k, v = torch.zeros(B, N, H, D, dtype=BF, device="cuda"), torch.zeros(B, N, H, D, dtype=BF,
                                                                        device="cuda")
    q = torch.zeros(B, N, Hq, D, dtype=BF, device="cuda")
    head = _rand(1, Hq * D, V).cuda()
    parents = torch.full((B, N), -1, dtype=torch.int32, device="cuda")
    tokens = torch.zeros(B, N, dtype=torch.int64, device="cuda")
    u = torch.zeros(B, N, device="cuda")

    def step(c, d):
        kv4_append(d, k, v)
        o = kv4_tree_attn(q, c, d, parents, 1500)
        picked = sample((o.flatten(2).reshape(B * N, -1) @ head), u.flatten(), top_k=3)
        path, n, following = tree_accept(parents, tokens, picked.view(B, N))
        kv4_commit(c, d, path, n, reset=True)
        return o, picked, path, n, following

    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):  # what a first call sets up is not captured
            step(caches[0], drafts[0])
        torch.cuda.current_stream().wait_stream(side)
        step(caches[1], drafts[1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step(caches[0], drafts[0])
        took = set()
        for i in range(6):
            for t, seed in ((k, 1), (v, 2), (q, 3)):
                t.copy_(_rand(10 * i + seed, *t.shape))
            parents.copy_(_trees(i, B, N, 1 + i))
            u.copy_(torch.rand(B, N, generator=torch.Generator().manual_seed(i)))
            if i:  # half of the tokens are what the last step picked
                tokens.copy_(torch.where(torch.rand(B, N, device="cuda") < 0.5, 0, held[1].view(B, N)))
            graph.replay()
            torch.cuda.synchronize()
            want = step(caches[1], drafts[1])
            for a, b in zip(held, want):
                assert torch.equal(a, b)
            assert torch.equal(caches[0].lengths, caches[1].lengths)
            assert drafts[0].lengths.tolist() == [0, 0]
            took |= set(held[3].tolist())
        for a, b in zip(kv4_read(caches[0], 2048), kv4_read(caches[1], 2048)):
            assert torch.equal(a, b)


def test_two_calls_at_once(gpu):
    """Two streams, trees over the same cache: each has a workspace of its own."""
    c, r = _pair(2, 2, 128, 4096, BF, (4000, 4096))
    d, rd = _drafted(c, 16, 1)
    q = [_rand(i, 2, 16, 4, 128).cuda() for i in range(2)]
    parents = [_trees(i, 2, 16).cuda() for i in range(2)]
    want = [kv4_tree_attn(x, c, d, p) for x, p in zip(q, parents)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        got = []
        for s, x, p in zip(streams, q, parents):
            with torch.cuda.stream(s):
                got.append(kv4_tree_attn(x, c, d, p))
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals(gpu):
    c, _ = _pair(2, 2, 64, 64, BF, (9, 9))
    d, _ = _drafted(c, 8, 1)
    q = _rand(1, 2, 8, 4, 64).cuda()
    p = torch.zeros(2, 8, dtype=torch.int32, device="cuda")
    one = torch.ones(2, dtype=torch.int32, device="cuda")
    many, wide = _rand(1, 2, 33, 4, 64).cuda(), torch.zeros(2, 33, dtype=torch.int32, device="cuda")
    bad = [lambda: kv4_tree_attn(q, c, c, p), lambda: kv4_tree_attn(q, c, q, p),
           lambda: kv4_tree_attn(q, c, KV4Cache(2, 2, 128, 32), p),
           lambda: kv4_tree_attn(q, c, KV4Cache(1, 2, 64, 32), p),
           lambda: kv4_tree_attn(q, c, KV4Cache(2, 2, 64, 32, HF), p),
           lambda: kv4_tree_attn(q, c, d, p[:, :7]), lambda: kv4_tree_attn(q, c, d, p.long()),
           lambda: kv4_tree_attn(q, c, d, p.cpu()), lambda: kv4_tree_attn(q, c, d, p, 0),
           lambda: kv4_tree_attn(q.half(), c, d, p), lambda: kv4_tree_attn(q[:, :, :3], c, d, p),
           lambda: kv4_tree_attn(q, c, d, p, counts=one[:1]),
           lambda: kv4_tree_attn(many, c, d, wide),
           lambda: kv4_commit(c, c, p), lambda: kv4_commit(c, d, p[:1]),
           lambda: kv4_commit(c, d, p.long()), lambda: kv4_commit(c, d, p[:, :0]),
           lambda: kv4_commit(c, d, wide), lambda: kv4_commit(c, d, p, one.long())]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError, match="forward-only"):
        kv4_tree_attn(q.requires_grad_(), c, d, p)
    empty = kv4_tree_attn(q.detach()[:, :0], c, d, p[:, :0], return_lse=True)
    assert [x.shape for x in empty] == [(2, 0, 4, 64), (2, 4, 0)]
    assert c.lengths.tolist() == [9, 9]


def test_inference_mode(gpu):
    with torch.inference_mode():
        c, d = KV4Cache(1, 2, 64, 64), KV4Cache(1, 2, 64, 32)
        x = torch.ones(1, 4, 2, 64, dtype=BF, device="cuda")
        kv4_append(d, x, x)
    p = torch.arange(4, device="cuda", dtype=torch.int32)[None] - 1
    o = kv4_tree_attn(x, c, d, p)
    assert (o == 1).all()
    kv4_commit(c, d, p + 1, reset=True)
    assert c.lengths.item() == 4 and d.lengths.item() == 0
    assert (kv4_attn(x, c) == 1).all()


def test_the_package_offers_them():
    for name in ("kv4_tree_attn", "kv4_commit", "rope", "rope_frequencies", "sample",
                 "tree_accept"):
        assert name in ttcd_amd.__all__ and hasattr(ttcd_amd, name)


def _mixed(B, lengths, counts):
    return ([lengths[b] if b < len(lengths) else (b * 37) % 300 for b in range(B)],
            None if counts is None else [counts[b] if b < len(counts) else counts[-1]
                                         for b in range(B)])


@pytest.mark.parametrize("B,N,Hq,H,D,C,lengths,window,counts", [
    # 64 parts for a head: some 56 of one sequence, more than 16 in the sum over the parts of
    # many rows; others of one part (written at once), of none (counts 0), and of nothing held
    (8, 16, 16, 8, 128, 16384, (16000, 0, 33, 200, 0, 5000, 64, 1), None,
     (16, 16, 3, 0, 0, 16, 16, 1)),
    (8, 16, 16, 8, 128, 16384, (16000, 0, 33, 200, 0, 5000, 64, 1), 9000, None),
    # the same in blocks of 128 rows, and 64 parts of one sequence
    (4, 64, 4, 2, 64, 8192, (20, 8000, 0, 300), None, (64, 40, 0, 33)),
    (1, 20, 4, 2, 64, 65536, (65000,), None, None),
    # as many sequences as lanes deal, and one more
    (64, 8, 4, 2, 64, 2048, (2048, 0, 2000, 1), None, (8, 8, 0, 5)),
    (65, 8, 4, 2, 64, 2048, (2048, 0, 2000, 1), None, (8, 8, 0, 5)),
    (64, 40, 2, 2, 64, 2048, (2048, 0, 3000, 1), 1500, (40, 8, 0, 33)),
])
def test_parts_dealt_by_the_lengths(gpu, B, N, Hq, H, D, C, lengths, window, counts):
    lengths, counts = _mixed(B, lengths, counts)
    c, r = _pair(B, H, D, C, BF, lengths, seed=B)
    d, rd = _drafted(c, N, N + 1, counts)
    q, parents = _rand(N + 9, B, N, Hq, D, scale=1.5), _trees(N, B, N)
    n = None if counts is None else torch.tensor(counts, dtype=torch.int32).cuda()
    o, lse = kv4_tree_attn(q.cuda(), c, d, parents.cuda(), window, counts=n, return_lse=True)
    _check(r, rd, q, parents, o, lse, window, counts)
    for b in range(B):  # rows behind the last node
        k = N if counts is None else counts[b]
        assert (o[b, k:] == 0).all() and (lse[b, :, k:] == -math.inf).all()

"""The 4-bit key / value cache on the GPU against the float64 oracle.

Bounds, with u half a step of the type (bf16 2^-8, f16 2^-11) and e = 2^-24:
* what the cache holds is determined: codes, scales and read values are equal;
* lse: a score is a sum of D exact products and one scaling, off by at most
  d = (D + 4) e scale max_j sum |q k_j|; the exponential's argument and the
  logarithm are rounded at the lse's own size; the sum over n keys is in chains of
  at most n / 8 + 64 additions;
* o: probabilities are rounded once, u, beside what their scores are off by, and
  the result once: u |o| + (u + 4 d + chain e) sum p |v|. f16 rounds those under
  2^-14 to multiples of 2^-24, off by 2^-25; they are held times 2^7 against a
  maximum that is some key's own, so sum p >= 1 and n keys add n 2^-32 max |v|;
* key weights: sums of exp(score - lse), off by the scores' and the lse's share.
"""
from __future__ import annotations

import math

import pytest
import torch

import ttcd_amd
from oracle import kv4_ref
from ttcd_amd import KV4Cache, kv4_append, kv4_attn, kv4_evict, kv4_key_weights, kv4_read

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
U = {BF: 2.0 ** -8, HF: 2.0 ** -11}
E = 2.0 ** -24


def _rand(seed, *shape, dtype=BF, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def _pair(B, H, D, C, dtype, lengths=(), seed=0, weights=False):
    """A cache whose slots all start as garbage (NaN scales), and its oracle, with
    lengths[b] positions appended."""
    c = KV4Cache(B, H, D, C, dtype, weights=weights)
    for t in (c.k_codes, c.k_scales, c.v_codes, c.v_scales):
        t.fill_(255)
    r = kv4_ref.Ref(B, H, D, C, dtype)
    left = list(lengths)
    i = 0
    while any(left):
        step = [min(n, C) for n in left]
        T = max(step)
        k, v = (_rand(seed + 7 * i + j, B, T, H, D, dtype=dtype, scale=1 + 2 * j) for j in (0, 1))
        n = torch.tensor(step, dtype=torch.int32)
        kv4_append(c, k.cuda(), v.cuda(), counts=n.cuda())
        r.append(k, v, n)
        left = [a - b for a, b in zip(left, step)]
        i += 1
    return c, r


def _score_error(r, q):
    """d of the bounds: over all queries and positions of the call, per sequence."""
    out = []
    for b in range(r.B):
        k = r.rows[b][0].abs()
        if not len(k):
            out.append(0.0)
            continue
        k = k.repeat_interleave(q.shape[2] // r.H, 1)
        s = torch.einsum("thd,lhd->htl", q[b].double().cpu().abs().nan_to_num(0), k).max().item()
        out.append((r.D + 4) * E * s * r.D ** -0.5)
    return torch.tensor(out)


def _check_attn(r, q, o, lse, window, counts):
    want, wl, mag = r.attn(q, window, counts)
    chain = (max(r.length(b) for b in range(r.B)) / 8 + 64) * E
    d = _score_error(r, q)[:, None, None]
    u = U[r.dtype]
    assert o.shape == q.shape and o.dtype == r.dtype
    limit = u * want.abs() + (u + 4 * d[..., None] + chain) * mag
    if r.dtype == HF:
        limit += torch.tensor([len(v) * 2.0 ** -32 * v.abs().max() if len(v) else 0.0
                               for _, v in r.rows])[:, None, None, None]
    bad = ((o.double().cpu() - want).abs() - limit).max().item()
    assert bad <= 0, bad
    empty = wl == -math.inf
    assert torch.equal(lse.cpu() == -math.inf, empty)
    ll = 2 * d + chain + 8 * E * (1 + wl.masked_fill(empty, 0).abs())
    assert ((lse.double().cpu() - wl).masked_fill(empty, 0).abs() <= ll).all()


# ------------------------------------------------------------ append and read

@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [1, 2, 4, 5, 33, 64])
def test_append_holds_what_the_format_says(gpu, dtype, D, T):
    B, H, C = 3, 2, 64
    c, r = _pair(B, H, D, C, dtype, (0, 63, 129), seed=T)
    before = [t.cpu().clone() for t in (c.k_codes, c.k_scales, c.v_codes, c.v_scales)]
    k, v = _rand(1, B, T, H, D, dtype=dtype), _rand(2, B, T, H, D, dtype=dtype, scale=40.0)
    kv4_append(c, k.cuda(), v.cuda())
    r.append(k, v)
    assert c.lengths.tolist() == [T, 63 + T, 129 + T]
    for x, y in zip(kv4_read(c, C), r.read(C)):
        assert torch.equal(x.cpu(), y)
    # the new slots' bytes as the layout says, every other slot as it was
    for b, old in enumerate((0, 63, 129)):
        slots = (old + torch.arange(T)) % C
        kk, vv = (torch.zeros(1, H, C, D, dtype=dtype) for _ in range(2))
        kk[0, :, slots] = k[b].transpose(0, 1)
        vv[0, :, slots] = v[b].transpose(0, 1)
        want = kv4_ref.codes_of(kk, vv)
        for got, w, was, is_v in zip((c.k_codes, c.k_scales, c.v_codes, c.v_scales), want, before,
                                     (0, 0, 1, 1)):
            exp = was[b].clone()
            if is_v:
                exp[:, slots // 4, :, slots % 4] = w[0][:, slots // 4, :, slots % 4]
            else:
                exp[:, slots] = w[0][:, slots]
            assert torch.equal(got[b].cpu(), exp)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_append_of_any_value(gpu, dtype):
    """Ties, zeros of both signs, subnormals, the largest values, infinities, NaN."""
    g = torch.Generator().manual_seed(3)
    bits = torch.randint(-2 ** 15, 2 ** 15, (1, 64, 4, 128), generator=g, dtype=torch.int16)
    k = bits.view(dtype)
    v = (torch.randint(-26, 27, (1, 64, 4, 128), generator=g) / 4).to(dtype)
    for i, x in enumerate((0.0, -0.0, math.inf, -math.inf, math.nan, torch.finfo(dtype).max,
                           torch.finfo(dtype).tiny, torch.finfo(dtype).smallest_normal / 4)):
        v[0, 2 * i, :, :] = 0
        v[0, 2 * i, :, 5::9] = x
        v[0, 2 * i + 1, :, 7] = x
    c, r = _pair(1, 4, 128, 64, dtype)
    kv4_append(c, k.cuda(), v.cuda())
    r.append(k, v)
    for x, y in zip(kv4_read(c, 64), r.read(64)):
        assert torch.isfinite(x).all() and torch.equal(x.cpu(), y)


@pytest.mark.parametrize("counts", [(0, 9, 30), (30, 1, 0), (0, 0, 0), (-5, 2, 99)])
def test_padded_batch(gpu, counts):
    c, r = _pair(3, 2, 64, 64, BF, (50, 3, 64), weights=True)
    c.weights.fill_(2.0)
    k, v = _rand(4, 3, 30, 2, 64), _rand(5, 3, 30, 2, 64)
    n = torch.tensor(counts, dtype=torch.int32)
    m = n.clamp(0, 30)
    for b in range(3):  # what is not appended is not looked at
        k[b, m[b]:] = math.nan
    kv4_append(c, k.cuda(), v.cuda(), counts=n.cuda())
    r.append(k, v, m)
    assert c.lengths.tolist() == [r.length(b) for b in range(3)]
    for x, y in zip(kv4_read(c, 100), r.read(100)):
        assert torch.equal(x.cpu(), y)
    new = torch.zeros(3, 64, dtype=torch.bool)
    for b, old in enumerate((50, 3, 64)):
        new[b, (old + torch.arange(int(m[b]))) % 64] = True
    assert torch.equal(c.weights.cpu(), torch.where(new, 0.0, 2.0)[:, None].expand(3, 2, 64))


def test_views_of_a_fused_projection(gpu):
    """k and v as slices of one (B, T, Hq + 2 Hkv, D) output, a transposed layout, a
    broadcast row, and rows off 16-byte alignment (copied)."""
    B, T, H, D = 2, 37, 2, 128
    qkv = _rand(6, B, T, 8, D).cuda()
    _, k, v = qkv.split((4, H, H), 2)
    kt = _rand(7, B, H, T, D).cuda().transpose(1, 2)
    odd = _rand(8, B * T * H * D + 3).cuda()[3:].view(B, T, H, D)
    row = _rand(9, B, 1, H, D).cuda().expand(B, T, H, D)
    for a, b in ((k, v), (kt, v), (odd, kt), (row, odd)):
        c, r = _pair(B, H, D, 64, BF, (5, 0))
        kv4_append(c, a, b)
        r.append(a, b)
        for x, y in zip(kv4_read(c, 64), r.read(64)):
            assert torch.equal(x.cpu(), y)


@pytest.mark.parametrize("T", [300, 2048])
def test_large_append(gpu, T):
    """More rows than one workgroup writes, over the ring's end."""
    c, r = _pair(2, 3, 128, 2048, HF, (2040, 1111))
    k, v = _rand(1, 2, T, 3, 128, dtype=HF), _rand(2, 2, T, 3, 128, dtype=HF)
    n = torch.tensor([T, T - 3], dtype=torch.int32)
    kv4_append(c, k.cuda(), v.cuda(), counts=n.cuda())
    r.append(k, v, n)
    assert c.lengths.tolist() == [r.length(0), r.length(1)]
    for x, y in zip(kv4_read(c, 2048), r.read(2048)):
        assert torch.equal(x.cpu(), y)


@pytest.mark.parametrize("count", [0, 1, 3, 64, 65, 200])
def test_read_counts(gpu, count):
    c, r = _pair(3, 1, 64, 64, HF, (0, 2, 99))
    for x, y in zip(kv4_read(c, count), r.read(count)):
        assert torch.equal(x.cpu(), y)


# ------------------------------------------------------------------ attention

ATTN = [
    # B, T, Hq, H, D, C, lengths, window, counts, dtype
    (1, 1, 4, 2, 64, 64, (1,), None, None, BF),
    (1, 1, 4, 2, 64, 64, (0,), None, None, BF),                  # nothing held
    (2, 1, 16, 8, 128, 96, (33, 96), None, None, BF),
    (1, 1, 15, 5, 64, 512, (2000,), None, None, HF),             # wrapped ring, odd group
    (3, 1, 8, 1, 128, 256, (31, 32, 700), 32, None, HF),
    (1, 1, 20, 1, 64, 128, (128,), 1, None, BF),                 # two row tiles, window 1
    (2, 5, 6, 2, 64, 64, (64, 150), 20, None, BF),
    (2, 7, 16, 8, 128, 160, (7, 200), None, (7, 3), HF),
    (3, 9, 4, 4, 128, 64, (40, 9, 500), 8, (0, 9, 4), BF),
    (1, 33, 8, 2, 64, 192, (33,), None, None, BF),               # a prompt of its own
    (1, 64, 4, 4, 128, 96, (97,), 64, None, HF),                 # queries lose their oldest keys
    (2, 130, 6, 2, 128, 320, (130, 1000), 100, (130, 77), BF),
    (1, 200, 12, 2, 64, 256, (256,), None, None, HF),
    (1, 100, 2, 2, 64, 64, (50,), None, None, BF),               # more queries than positions
    (1, 3, 48, 1, 128, 4096, (4000,), None, None, BF),           # split over keys
    (4, 1, 9, 3, 64, 8192, (8192, 100, 5000, 20000), 3000, None, HF),
    (1, 2, 4, 2, 128, 32768, (40000,), None, None, BF),
]


@pytest.mark.parametrize("B,T,Hq,H,D,C,lengths,window,counts,dtype", ATTN)
def test_attention_matches_64_bits(gpu, B, T, Hq, H, D, C, lengths, window, counts, dtype):
    c, r = _pair(B, H, D, C, dtype, lengths, seed=T + D)
    q = _rand(11, B, T, Hq, D, dtype=dtype, scale=1.5)
    n = None if counts is None else torch.tensor(counts, dtype=torch.int32)
    if n is not None:
        for b in range(B):
            q[b, n[b]:] = math.nan  # padding does not matter
    o, lse = kv4_attn(q.cuda(), c, window, counts=None if n is None else n.cuda(),
                      return_lse=True)
    _check_attn(r, q, o, lse, window, n)
    whole, wl = kv4_attn(q.cuda(), c, window, counts=None if n is None else n.cuda(),
                         return_lse=True, split_keys=False)
    _check_attn(r, q, whole, wl, window, n)
    assert torch.equal(kv4_attn(q.cuda(), c, window, counts=None if n is None else n.cuda()), o)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_scores_that_grow_along_the_keys(gpu, dtype):
    """Running maxima that move at every tile, by more and less than the lazy limit,
    and one key far above all."""
    B, H, D, C = 1, 2, 64, 1024
    c, r = _pair(B, H, D, C, dtype)
    k = _rand(1, B, C, H, D, dtype=dtype) * torch.linspace(0.1, 6, C)[:, None, None]
    k[0, 777] *= 4
    k, v = k.to(dtype), _rand(2, B, C, H, D, dtype=dtype)
    kv4_append(c, k.cuda(), v.cuda())
    r.append(k, v)
    q = _rand(3, B, 3, 4, D, dtype=dtype, scale=3.0)
    for split in (False, True):
        o, lse = kv4_attn(q.cuda(), c, return_lse=True, split_keys=split)
        _check_attn(r, q, o, lse, None, None)


def test_nan_queries_stay_in_their_row(gpu):
    c, r = _pair(1, 2, 64, 4096, BF, (4096,))
    q = _rand(3, 1, 4, 4, 64)
    good = kv4_attn(q.cuda(), c)
    q[0, 1, 2, 5] = math.nan
    for split in (True, False):
        o, lse = kv4_attn(q.cuda(), c, return_lse=True, split_keys=split)
        assert torch.isnan(o[0, 1, 2]).all() and torch.isnan(lse[0, 2, 1])
        o[0, 1, 2] = good[0, 1, 2]
        assert torch.isfinite(o).all()
        assert (o - good).abs().max() < 0.02


def test_strided_queries(gpu):
    c, r = _pair(2, 2, 128, 64, BF, (64, 20))
    wide = _rand(3, 2, 5, 12, 128).cuda()
    for q in (wide[:, :, 2:6], wide.transpose(1, 2)[:, :5].transpose(1, 2)[:, :, :4],
              wide[:, :, ::3], wide[:, 1:2].expand(2, 5, 12, 128)):
        o, lse = kv4_attn(q, c, return_lse=True)
        _check_attn(r, q, o, lse, None, None)
        w = kv4_key_weights(q, c, lse)
        assert torch.equal(w, kv4_key_weights(q.contiguous(), c, lse))


def test_contiguous_with_odd_strides_of_one(gpu):
    """Dimensions of 1 may have any stride, and rows may start off 16 bytes."""
    c, r = _pair(1, 1, 64, 64, BF, (33,))
    flat = _rand(5, 4 * 64 + 9).cuda()
    for off in (0, 3):
        x = flat[off:].as_strided((1, 1, 1, 64), (77, 5, 3, 1))
        q = flat[off:].as_strided((1, 1, 4, 64), (13, 7, 64, 1))
        assert x.is_contiguous() and q.is_contiguous()
        kv4_append(c, x, x)
        r.append(x, x)
        o, lse = kv4_attn(q, c, return_lse=True)
        _check_attn(r, q, o, lse, None, None)
        kv4_key_weights(q, c, lse)


def test_lengths_out_of_range_read_nothing_wrong(gpu):
    """Entries that no append leaves: every slot is still in range and rows without a
    position are empty."""
    c, _ = _pair(3, 1, 64, 64, BF, (64, 64, 64))
    c.lengths.copy_(torch.tensor([-7, 2 ** 31 - 1, 3], dtype=torch.int32))
    q = _rand(1, 3, 8, 2, 64).cuda()
    o, lse = kv4_attn(q, c, return_lse=True)
    assert (o[0] == 0).all() and (lse[0] == -math.inf).all()
    assert torch.isfinite(o).all()
    assert (lse[2, :, :5] == -math.inf).all() and torch.isfinite(lse[2, :, 5:]).all()
    kv4_key_weights(q, c, lse)
    kv4_evict(c, torch.rand(3, 1, 64, device=gpu), 32)
    for x in kv4_read(c, 10):
        assert (x[0] == 0).all()


# ---------------------------------------------------------------- key weights

@pytest.mark.parametrize("B,T,Hq,H,D,C,lengths,window,counts,dtype", ATTN)
def test_key_weights_match_64_bits(gpu, B, T, Hq, H, D, C, lengths, window, counts, dtype):
    c, r = _pair(B, H, D, C, dtype, lengths, seed=T + D)
    q = _rand(11, B, T, Hq, D, dtype=dtype, scale=1.5)
    n = None if counts is None else torch.tensor(counts, dtype=torch.int32)
    nc = None if n is None else n.cuda()
    if n is not None:
        for b in range(B):
            q[b, n[b]:] = math.nan
    _, lse = kv4_attn(q.cuda(), c, window, counts=nc, return_lse=True)
    w = kv4_key_weights(q.cuda(), c, lse, window, counts=nc)
    want = r.key_weights(q, lse, window, n)
    rows = T * (Hq // H)
    top = 0 if not torch.isfinite(lse).any() else lse[torch.isfinite(lse)].abs().max().item()
    d = _score_error(r, q)[:, None, None] + 8 * E * (1 + 2 * top) + (rows / 16 + 16) * E
    assert w.shape == (B, H, C)
    assert ((w.double().cpu() - want).abs() <= 2 * d * want + 1e-30).all()
    # accumulated, and every weight is some row's: their sum is the number of rows
    twice = kv4_key_weights(q.cuda(), c, lse, window, counts=nc, out=w.clone(), accumulate=True)
    assert torch.equal(twice, 2 * w)
    seen = torch.isfinite(lse).view(B, H, -1).sum(-1).double().cpu()
    assert ((w.double().sum(-1).cpu() - seen).abs() <= 1e-3 * seen).all()


@pytest.mark.parametrize("T,Hq,window", [(1, 2, 40), (1, 2, None), (9, 2, 33), (30, 2, 20), (90, 4, 64)])
@pytest.mark.parametrize("dtype,D", [(BF, 128), (HF, 64)])
def test_values_that_no_query_sees_may_be_nan(gpu, T, Hq, window, dtype, D):
    """NaN scales, as no append leaves, in positions before every query's window and in
    slots past the end."""
    c, r = _pair(1, 2, D, 256, dtype, (200,))
    seen = 256 if window is None else window + T - 1
    for t, shape in ((c.k_scales, None), (c.v_scales, True)):
        x = t if shape is None else t.transpose(3, 4).flatten(2, 3)
        hidden = torch.ones(256, dtype=torch.bool)
        hidden[max(0, 200 - seen):200] = False
        x = x.clone()
        x[:, :, hidden.cuda()] = 255
        t.copy_(x if shape is None else x.unflatten(2, (64, 4)).transpose(3, 4))
    q = _rand(4, 1, T, Hq, D, dtype=dtype)
    o, lse = kv4_attn(q.cuda(), c, window, return_lse=True)
    _check_attn(r, q, o, lse, window, None)
    w = kv4_key_weights(q.cuda(), c, lse, window)
    assert torch.isfinite(w).all() and (w[..., 200:] == 0).all()


@pytest.mark.parametrize("T,Hq,D,dtype", [(70, 1, 64, BF), (100, 2, 128, HF), (7, 2, 64, BF)])
def test_a_nan_query_weighs_only_what_it_sees(gpu, T, Hq, D, dtype):
    c, r = _pair(1, 1, D, 192, dtype, (130,))
    q = _rand(2, 1, T, Hq, D, dtype=dtype)
    _, lse = kv4_attn(q.cuda(), c, return_lse=True)
    good = kv4_key_weights(q.cuda(), c, lse)
    q[0, 3, 0, 1] = math.nan
    _, lse = kv4_attn(q.cuda(), c, return_lse=True)
    w = kv4_key_weights(q.cuda(), c, lse)
    pos = 130 - T + 3
    assert torch.isnan(w[0, 0, :pos + 1]).all()
    assert torch.equal(w[0, 0, pos + 1:], good[0, 0, pos + 1:])


# ------------------------------------------------------------------- eviction

def _evict_case(c, r, w, keep, recent, out=None):
    new, index, nw = kv4_evict(c, w, keep, recent, out=out)
    wi, ww = r.evict(w.cpu(), keep, recent)
    assert torch.equal(index.cpu(), wi)
    assert torch.equal(torch.nan_to_num(nw[..., :keep].cpu(), nan=9.0),
                       torch.nan_to_num(ww, nan=9.0))
    assert (nw[..., keep:] == 0).all()
    rn = r.take(wi, new.capacity)
    assert new.lengths.tolist() == [rn.length(b) for b in range(r.B)]
    for x, y in zip(kv4_read(new, keep), rn.read(keep)):
        assert torch.equal(x.cpu(), y)
    return new, rn


@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 5), (20, 0), (20, 7), (20, 20), (64, 3),
                                         (63, 0), (50, 100)])
@pytest.mark.parametrize("kind", ["random", "ties", "signs"])
def test_evict_keeps_the_heaviest(gpu, keep, recent, kind):
    c, r = _pair(4, 2, 64, 64, BF, (0, 13, 64, 150))
    g = torch.Generator().manual_seed(keep + recent)
    w = torch.rand(4, 2, 64, generator=g)
    if kind == "ties":
        w = (w * 4).floor()
    elif kind == "signs":
        w = (w - 0.5) * 1e-3
        w[..., ::7] = -0.0
        w[..., 3::7] = 0.0
        w[..., 5::11] = math.nan
        w[..., 6::11] = math.inf
        w[..., 8::11] = -math.inf
    _evict_case(c, r, w.cuda(), keep, recent)


@pytest.mark.parametrize("C,lengths,keep,recent,dtype", [
    (4096, (4096, 9001), 1500, 100, HF), (8192, (8000, 5), 4095, 0, BF),
    (2048, (1025, 2048), 1024, 1024, BF), (40960, (40960, 123), 9999, 77, BF),
    (65568, (70000, 65000), 32768, 1, BF)])
def test_evict_of_long_caches(gpu, C, lengths, keep, recent, dtype):
    c, r = _pair(2, 2, 128, C, dtype, lengths)
    g = torch.Generator().manual_seed(C)
    for w in (torch.rand(2, 2, C, generator=g).log().square(),
              torch.randint(0, 3, (2, 2, C), generator=g).float(), torch.ones(2, 2, C)):
        _evict_case(c, r, w.cuda(), keep, recent)


def test_evict_into_another_cache(gpu):
    c, r = _pair(2, 2, 64, 64, BF, (64, 10))
    out = KV4Cache(2, 2, 64, 32, weights=True)
    w = torch.rand(2, 2, 64, device=gpu)
    new, _ = _evict_case(c, r, w, 32, 4, out)
    assert new is out
    with pytest.raises(ValueError):
        kv4_evict(c, w, 33, out=out)
    with pytest.raises(ValueError):
        kv4_evict(c, w, 8, out=c)
    with pytest.raises(ValueError):
        kv4_evict(c, None, 8)
    with pytest.raises(ValueError):
        kv4_evict(c, w, 8, out=KV4Cache(2, 2, 64, 32, HF))


def test_a_refused_eviction_changes_neither_cache(gpu):
    c, _ = _pair(2, 2, 64, 64, BF, (64, 10), weights=True)
    held = c.weights
    held.fill_(3.0)
    for keep, out in ((8, c), (8, KV4Cache(1, 2, 64, 64)), (8, KV4Cache(2, 2, 128, 64)),
                      (33, KV4Cache(2, 2, 64, 32))):
        had = out.weights
        with pytest.raises(ValueError):
            kv4_evict(c, None, keep, out=out)
        assert out.weights is had and c.weights is held
    assert (held == 3.0).all() and c.lengths.tolist() == [64, 10]


def test_evict_by_the_weights_of_the_cache_written(gpu):
    """The written cache keeps the new weights, also where its own were gone by."""
    c, r = _pair(2, 2, 64, 64, BF, (64, 10))
    out = KV4Cache(2, 2, 64, 64, weights=True)
    w = torch.rand(2, 2, 64, device=gpu)
    out.weights.copy_(w)
    _, index, new = kv4_evict(c, out.weights, 20, 4, out=out)
    want, ww = r.evict(w.cpu(), 20, 4)
    assert torch.equal(index.cpu(), want) and torch.equal(new[..., :20].cpu(), ww)
    assert out.weights is new


def test_weights_that_do_not_fit_are_refused(gpu):
    c = KV4Cache(2, 2, 64, 64, weights=True)
    held = c.weights
    for w in (torch.zeros(2, 2, 32, device=gpu), torch.zeros(2, 2, 64),
              torch.zeros(2, 2, 64, device=gpu, dtype=HF),
              torch.zeros(2, 2, 128, device=gpu)[..., ::2], [0.0]):
        with pytest.raises(ValueError):
            c.weights = w
    assert c.weights is held
    c.weights = None
    kv4_append(c, *[_rand(1, 2, 4, 2, 64).cuda()] * 2)
    assert c.lengths.tolist() == [4, 4]


# ------------------------------------------------------------------- together

@pytest.mark.parametrize("dtype,D,Hq,H", [(BF, 128, 4, 2), (HF, 64, 9, 3)])
def test_prefill_decode_evict_and_on(gpu, dtype, D, Hq, H):
    """A prompt in chunks, tokens one by one, a cut by accumulated weight, more tokens:
    every output against the oracle's own cache."""
    B, C = 2, 160
    c, r = _pair(B, H, D, C, dtype, weights=True)
    acc = torch.zeros(B, H, C, dtype=torch.float64)

    def step(T, seed):
        k, v = _rand(seed, B, T, H, D, dtype=dtype), _rand(seed + 1, B, T, H, D, dtype=dtype)
        q = _rand(seed + 2, B, T, Hq, D, dtype=dtype, scale=2.0)
        kv4_append(c, k.cuda(), v.cuda())
        r.append(k, v)
        o, lse = kv4_attn(q.cuda(), c, return_lse=True)
        _check_attn(r, q, o, lse, None, None)
        kv4_key_weights(q.cuda(), c, lse, out=c.weights, accumulate=True)
        acc.add_(r.key_weights(q, lse))

    for i, T in enumerate((60, 37, 1, 1, 1, 20, 1)):
        step(T, 10 * i)
    assert torch.allclose(c.weights.double().cpu(), acc, rtol=1e-3, atol=1e-6)
    index, _ = r.evict(c.weights.cpu(), 48, 16)
    new, got, w = kv4_evict(c, None, 48, 16)
    assert torch.equal(got.cpu(), index) and new.weights is w
    r, c = r.take(index, C), new
    acc = w.double().cpu()
    for i, T in enumerate((1, 1, 30, 1)):
        step(T, 1000 + 10 * i)
    assert torch.allclose(c.weights.double().cpu(), acc, rtol=1e-3, atol=1e-6)


def test_two_calls_at_once_on_one_cache(gpu):
    """Reads of one cache on two streams, each with its own workspace: the results of
    the calls one after the other, every time."""
    c, _ = _pair(2, 2, 128, 8192, BF, (8192, 6000))
    qs = [_rand(i, 2, t, 8, 128).cuda() for i, t in ((1, 1), (2, 100))]
    want = [kv4_attn(q, c, return_lse=True) for q in qs]
    ww = [kv4_key_weights(q, c, l) for q, (_, l) in zip(qs, want)]
    streams = [torch.cuda.Stream() for _ in qs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(20):
        for s, q, (_, l) in zip(streams, qs, want):
            with torch.cuda.stream(s):
                got.append((*kv4_attn(q, c, return_lse=True), kv4_key_weights(q, c, l)))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        for x, y in zip(g, (*want[i % 2], ww[i % 2])):
            assert torch.equal(x, y)


def test_caches_made_in_inference_mode(gpu):
    with torch.inference_mode():
        c = KV4Cache(1, 1, 64, 64, weights=True)
        kv4_append(c, *[_rand(1, 1, 5, 1, 64).cuda()] * 2)
    c.reset()
    assert c.lengths.tolist() == [0]
    kv4_append(c, *[_rand(1, 1, 5, 1, 64).cuda()] * 2)
    assert c.lengths.tolist() == [5]


def test_another_stream(gpu):
    c, r = _pair(1, 2, 64, 256, BF, (200,))
    k, v, q = (_rand(i, 1, 9, h, 64).cuda() for i, h in ((1, 2), (2, 2), (3, 4)))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        kv4_append(c, k, v)
        o, lse = kv4_attn(q, c, return_lse=True)
        w = kv4_key_weights(q, c, lse)
        new, index, _ = kv4_evict(c, w, 100)
        got = kv4_read(new, 100)
    torch.cuda.current_stream().wait_stream(s)
    r.append(k, v)
    _check_attn(r, q, o, lse, None, None)
    wi, _ = r.evict(w.cpu(), 100, 0)
    assert torch.equal(index.cpu(), wi)
    for x, y in zip(got, r.take(wi, 256).read(100)):
        assert torch.equal(x.cpu(), y)


def test_a_captured_step_decodes_on(gpu):
    """One decode step in a graph (append, attention split over keys, key weights):
    each replay is the next position, over the ring's end, with eager work between."""
    B, H, Hq, D, C = 2, 2, 8, 64, 2048
    c, r = _pair(B, H, D, C, BF, (2040, 300), weights=True)
    k, v, q = (torch.zeros(B, 1, h, D, dtype=BF, device=gpu) for h in (H, H, Hq))

    def step():
        kv4_append(c, k, v)
        o, lse = kv4_attn(q, c, return_lse=True)
        kv4_key_weights(q, c, lse, out=c.weights, accumulate=True)
        return o, lse

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        kept = [t.clone() for t in (c.k_codes, c.k_scales, c.v_codes, c.v_scales, c.lengths)]
        step()
        for t, x in zip((c.k_codes, c.k_scales, c.v_codes, c.v_scales, c.lengths), kept):
            t.copy_(x)
        c.weights.zero_()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o, lse = step()
    acc = torch.zeros(B, H, C, dtype=torch.float64)
    for i in range(12):
        kn, vn = _rand(40 + i, B, 1, H, D), _rand(80 + i, B, 1, H, D)
        qn = _rand(120 + i, B, 1, Hq, D, scale=2.0)
        k.copy_(kn)
        v.copy_(vn)
        q.copy_(qn)
        g.replay()
        r.append(kn, vn)
        _check_attn(r, qn, o, lse, None, None)
        new = torch.stack([torch.arange(C) == (r.length(b) - 1) % C for b in range(B)])[:, None]
        acc = acc.masked_fill(new, 0) + r.key_weights(qn, lse)
        eager = kv4_attn(q, c)
        assert torch.equal(eager, o)
        torch.cuda.synchronize()
    assert torch.allclose(c.weights.double().cpu(), acc, rtol=1e-3, atol=1e-6)


def test_a_captured_eviction_goes_by_the_lengths_it_finds(gpu):
    """Replays over other lengths, weights and rows, with eager calls between them."""
    C, keep = 2080, 600
    c = KV4Cache(2, 2, 64, C)
    out = KV4Cache(2, 2, 64, C)
    w = torch.zeros(2, 2, C, device=gpu)
    kv4_evict(c, w, keep, 9, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        _, index, nw = kv4_evict(c, w, keep, 9, out=out)
        k, v = kv4_read(out, keep)
    for i, lengths in enumerate(((2000, 3), (600, 601), (0, 2080), (5000, 1100))):
        held, r = _pair(2, 2, 64, C, BF, lengths, seed=50 + i)
        for name in ("k_codes", "k_scales", "v_codes", "v_scales", "lengths"):
            getattr(c, name).copy_(getattr(held, name))
        w.copy_(torch.rand(2, 2, C, generator=torch.Generator().manual_seed(i)))
        g.replay()
        torch.cuda.synchronize()
        wi, ww = r.evict(w.cpu(), keep, 9)
        assert torch.equal(index.cpu(), wi) and torch.equal(nw[..., :keep].cpu(), ww)
        for x, y in zip((k, v), r.take(wi, C).read(keep)):
            assert torch.equal(x.cpu(), y)


def test_offsets_past_32_bits(gpu):
    """Codes of more than 4 GiB: the last sequence's rows lie behind them."""
    B, H, D, C = 66, 8, 128, 131072
    c = KV4Cache(B, H, D, C)
    assert c.k_codes.numel() > 2 ** 32
    r = kv4_ref.Ref(1, H, D, C)
    n = torch.zeros(B, dtype=torch.int32, device=gpu)
    n[-1] = 40
    k, v = _rand(1, 1, 40, H, D), _rand(2, 1, 40, H, D)
    wide = [x.cuda().expand(B, 40, H, D) for x in (k, v)]
    c.lengths[-1] = C - 17  # over the ring's end
    kv4_append(c, *wide, counts=n)
    r.append(k, v)
    for x, y in zip(kv4_read(c, 40), r.read(40)):
        assert torch.equal(x[-1:].cpu(), y)
    q = _rand(3, 1, 2, 16, D)
    o, lse = kv4_attn(q.cuda().expand(B, 2, 16, D).contiguous(), c, 30, return_lse=True)
    _check_attn(r, q, o[-1:], lse[-1:], 30, None)
    w = kv4_key_weights(q.cuda().expand(B, 2, 16, D).contiguous(), c, lse, 30)
    want = r.key_weights(q, lse[-1:], 30)[0]
    at = (C - 17 + torch.arange(40)) % C
    assert torch.allclose(w[-1][:, at.cuda()].double().cpu(), want[:, :40], rtol=1e-4, atol=1e-9)
    new, index, _ = kv4_evict(c, w, 20, 4, out=KV4Cache(B, H, D, 32))
    assert new.lengths.tolist()[-1] == 20 and int(index[-1].max()) == C + 22


@pytest.mark.parametrize("D,dtype", [(64, BF), (64, HF), (128, BF), (128, HF)])
@pytest.mark.parametrize("T", [1, 12])
def test_caches_past_the_last_level_cache(gpu, D, dtype, T):
    """A cache of more than 128 MiB is read past the caches: the bits of a small one with
    the same window of positions."""
    H, Hq, start = 8, 16, 262144 * 3 - 20
    big, small = KV4Cache(1, H, D, 262144, dtype), KV4Cache(1, H, D, 128, dtype)
    k, v = _rand(1, 1, 90, H, D, dtype=dtype).cuda(), _rand(2, 1, 90, H, D, dtype=dtype).cuda()
    q = _rand(3, 1, T, Hq, D, dtype=dtype).cuda()
    out = []
    for c in (big, small):
        c.lengths.fill_(start)
        kv4_append(c, k, v)
        out.append(kv4_attn(q, c, 60, return_lse=True) + kv4_read(c, 90))
    for x, y in zip(*out):
        assert torch.equal(x, y)
    r = kv4_ref.Ref(1, H, D, 128, dtype)
    r.append(k, v)
    _check_attn(r, q, out[0][0], out[0][1], 60, None)


@pytest.mark.parametrize("weights", [False, True])
def test_a_cache_of_given_parts_shares_them(gpu, weights):
    c, _ = _pair(2, 2, 64, 64, BF, (64, 10), weights=weights)
    d = KV4Cache.from_parts(c.k_codes, c.k_scales, c.v_codes, c.v_scales, c.lengths, BF,
                            c.weights)
    assert d.weights is c.weights and d.lengths is c.lengths
    kv4_append(d, *[_rand(1, 2, 4, 2, 64).cuda()] * 2)
    assert c.lengths.tolist() == [68, 14]
    for x, y in zip(kv4_read(c, 64), kv4_read(d, 64)):
        assert torch.equal(x, y)


def test_refusals(gpu):
    c = KV4Cache(2, 2, 64, 64)
    x = _rand(1, 2, 4, 2, 64).cuda()
    q = _rand(1, 2, 4, 4, 64).cuda()
    lse = torch.zeros(2, 4, 4, device=gpu)
    n = torch.zeros(2, dtype=torch.int32, device=gpu)
    bad = [lambda: kv4_append(c, x[:1], x[:1]), lambda: kv4_append(c, x, x[:, :3]),
           lambda: kv4_append(c, x.half(), x.half()), lambda: kv4_append(c, q, q),
           lambda: kv4_append(c, x.cpu(), x.cpu()), lambda: kv4_append(c, x[0], x[0]),
           lambda: kv4_append(c, x, x, counts=n.long()), lambda: kv4_append(c, x, x, counts=n[:1]),
           lambda: kv4_append(c, *[x[:, :1].expand(2, 65, 2, 64)] * 2),
           lambda: kv4_attn(q[..., :32], c), lambda: kv4_attn(q[:, :, :3], c),
           lambda: kv4_attn(q, c, 0), lambda: kv4_attn(q, c, counts=n.cpu()),
           lambda: kv4_key_weights(q, c, lse[:, :, :3]), lambda: kv4_key_weights(q, c, lse.double()),
           lambda: kv4_key_weights(q, c, lse, accumulate=True),
           lambda: kv4_key_weights(q, c, lse, out=torch.zeros(2, 2, 32, device=gpu)),
           lambda: kv4_read(c, -1), lambda: kv4_evict(c, torch.zeros(2, 2, 32, device=gpu), 4),
           lambda: kv4_evict(c, torch.zeros(2, 2, 64, device=gpu), 0),
           lambda: kv4_evict(c, torch.zeros(2, 2, 64, device=gpu), 4, -1),
           lambda: KV4Cache.from_parts(c.k_codes, c.k_scales, c.v_codes, c.v_codes, c.lengths),
           lambda: KV4Cache.from_parts(c.k_codes[:, :, ::2], c.k_scales, c.v_codes, c.v_scales,
                                       c.lengths)]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    with pytest.raises(RuntimeError, match="forward-only"):
        kv4_attn(q.clone().requires_grad_(), c)
    assert kv4_attn(q[:, :0], c).shape == (2, 0, 4, 64)
    kv4_append(c, x[:, :0], x[:, :0])
    assert (kv4_key_weights(q[:, :0], c, lse[:, :, :0]) == 0).all()
    assert c.lengths.tolist() == [0, 0]
    c.lengths.fill_(5)
    c.reset()
    assert c.lengths.tolist() == [0, 0]


def test_evict_into_a_cache_that_shares_its_weights(gpu):
    """The old cache stays as it is: the written one, whose weights are the old one's (or a
    part of the memory that is read), gets new ones."""
    both = torch.rand(2, 3, 2, 64, device=gpu)
    own = both.flatten()[:2 * 2 * 64].view(2, 2, 64)       # the old cache's
    other = both.flatten()[3 * 64:7 * 64].view(2, 2, 64)   # overlaps it
    for held, given, target in ((own, torch.rand(2, 2, 64, device=gpu), own), (own, None, other),
                                (None, own, other)):
        c, r = _pair(2, 2, 64, 64, BF, (64, 10))
        c.weights = held
        out = KV4Cache(2, 2, 64, 64)
        out.weights = target
        was, go_by = both.clone(), (held if given is None else given).clone()
        _, index, new = kv4_evict(c, given, 20, 4, out=out)
        want, ww = r.evict(go_by.cpu(), 20, 4)
        assert torch.equal(both, was)
        assert torch.equal(index.cpu(), want) and torch.equal(new[..., :20].cpu(), ww)
        assert out.weights is new and c.weights is held


def test_gradients_are_refused_and_not_dropped(gpu):
    c = KV4Cache(2, 2, 64, 64, weights=True)
    x, q = _rand(1, 2, 4, 2, 64).cuda(), _rand(1, 2, 4, 4, 64).cuda()
    kv4_append(c, x, x)
    _, lse = kv4_attn(q, c, return_lse=True)
    w = torch.rand(2, 2, 64, device=gpu, requires_grad=True)

    def given():
        c.weights = w

    calls = (lambda: kv4_key_weights(q, c, lse.clone().requires_grad_()),
             lambda: kv4_key_weights(q, c, lse, out=w),
             lambda: kv4_key_weights(q[:, :0], c, lse[:, :, :0], out=w),
             lambda: kv4_evict(c, w, 8), given)
    was = w.detach().clone()
    for f in calls:
        with pytest.raises(RuntimeError, match="forward-only"):
            f()
    assert torch.equal(w.detach(), was) and c.weights is not w
    with torch.no_grad():
        for f in calls[:1] + calls[3:]:
            f()
    with pytest.raises(ValueError):
        kv4_key_weights(q, c, lse, out=[0.0])


@pytest.mark.parametrize("C,H,D,steps", [(64, 2, 64, (3, 4, 1, 1, 60, 64)),
                                         (96, 1, 128, (1, 1, 1, 1, 1, 1, 1, 70)),
                                         (512, 8, 128, (300, 1, 500, 2))])
def test_a_ring_goes_on_past_the_largest_length(gpu, C, H, D, steps):
    """Every call as over the same rows at the start of a sequence: append by one workgroup
    a sequence and by many, attention of a few and of many rows, key weights, eviction."""
    B, start = 2, torch.tensor([2 ** 30 - C - 5, 2 ** 30 - C - 200])
    c, r = KV4Cache(B, H, D, C), kv4_ref.Ref(B, H, D, C)
    c.lengths.copy_(start)
    total = 0
    for i, T in enumerate((C, *steps)):
        k, v = _rand(3 * i, B, T, H, D), _rand(3 * i + 1, B, T, H, D)
        kv4_append(c, k.cuda(), v.cuda())
        r.append(k, v)
        total += T
        n = c.lengths.cpu().long()
        assert (n <= 2 ** 30).all() and (n >= C).all() and ((n - start - total) % C == 0).all()
        for x, y in zip(kv4_read(c, C), r.read(C)):
            assert torch.equal(x.cpu(), y)
        q = _rand(3 * i + 2, B, T, 2 * H, D)
        o, lse = kv4_attn(q.cuda(), c, 50, return_lse=True)
        _check_attn(r, q, o, lse, 50, None)
        w = kv4_key_weights(q.cuda(), c, lse, 50).double().cpu()
        want = r.key_weights(q, lse, 50)
        for b in range(B):  # the oracle's positions count from 0
            assert torch.allclose(w[b], want[b].roll(int(start[b]) % C, -1), rtol=1e-4, atol=1e-9)
    assert (n < start + total).any()  # a length has dropped
    w = torch.rand(B, H, C, generator=torch.Generator().manual_seed(C))
    new, index, _ = kv4_evict(c, w.cuda(), C // 2, 5)
    at = torch.stack([w[b].roll(-(int(start[b]) % C), -1) for b in range(B)])
    want, _ = r.evict(at, C // 2, 5)
    assert torch.equal(index.cpu() - (n - total)[:, None, None].int(), want)
    for x, y in zip(kv4_read(new, C // 2), r.take(want, C).read(C // 2)):
        assert torch.equal(x.cpu(), y)

"""Rotary embedding at given positions on the GPU against the float64 oracle.

The angle is brought into a quarter turn in 64 bits, rounded to 32 there (2^-25 at most, it
is below 1) and each series is off by a few roundings of its terms: cosine and sine by less
than 2^-22 together, one rounding more with scale. A product and a sum round by 2^-24 of
theirs each. So y is off by at most 2^-21 scale (|x0| + |x1|) before it is rounded to the
type, by half a step u |y| (of f16's smallest, 2^-25)."""
from __future__ import annotations

import pytest
import torch

import ttcd_amd
from oracle import drafted_ref
from ttcd_amd import _lib, rope, rope_frequencies

pytestmark = pytest.mark.gpu

BF, HF, SF = torch.bfloat16, torch.float16, torch.float32
U = {BF: 2.0 ** -8, HF: 2.0 ** -11, SF: 2.0 ** -24}


def _rand(seed, *shape, dtype=BF):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _check(x, y, inv, pos, **kw):
    n = inv.numel()
    want, mag = drafted_ref.rope(x.cpu(), inv.cpu(), pos, **kw)
    limit = U[x.dtype] * want.abs() + 2.0 ** -21 * mag * 1.01 + 2.0 ** -25 * (x.dtype == HF)
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
    bad = ((y.double().cpu() - want).abs() - limit).max().item()
    assert bad <= 0, bad
    assert torch.equal(y[..., 2 * n:], x[..., 2 * n:])


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,n", [(128, 64), (128, 32), (64, 8), (64, 30), (80, 40), (80, 11),
                                 (256, 128), (2, 1), (7, 3), (96, 24), (1024, 512), (64, 7),
                                 (96, 13), (16, 5), (8, 1)])
@pytest.mark.parametrize("B,T", [(1, 1), (3, 37)])
def test_layouts(gpu, dtype, interleaved, D, n, B, T):
    q, k = _rand(1, B, T, 3, D, dtype=dtype).cuda(), _rand(2, B, T, 2, D, dtype=dtype).cuda()
    inv, _ = rope_frequencies(2 * n, 1e4, device="cuda")
    pos = torch.randint(0, 70000, (B, T), generator=torch.Generator().manual_seed(3))
    for inverse, scale in ((False, 1.0), (True, 1.25)):
        got = rope(q, k, inv, pos.int().cuda(), interleaved=interleaved, inverse=inverse,
                   scale=scale)
        for x, y in zip((q, k), got):
            _check(x, y, inv, pos, interleaved=interleaved, inverse=inverse, scale=scale)
        only = rope(q, None, inv, pos.cuda(), interleaved=interleaved, inverse=inverse, scale=scale)
        assert torch.equal(only, got[0])


@pytest.mark.parametrize("T,H", [(1, 1), (5, 1), (511, 1), (600, 16), (1000, 33), (3, 200)])
def test_tasks_that_end_anywhere(gpu, T, H):
    x = _rand(T, 2, T, H, 64).cuda()
    inv, _ = rope_frequencies(64, 1e6, device="cuda")
    _check(x, rope(x, None, inv, offset=7), inv, (7 + torch.arange(T)).expand(2, T))


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_far_positions(gpu, dtype):
    top = 2 ** 31 - 1 if dtype == torch.int32 else 2 ** 40
    pos = torch.tensor([[0, 1, 10 ** 6, 12345678, top, top - 1, -1, -70000]], dtype=dtype)
    x = _rand(1, 1, 8, 2, 128, dtype=SF).cuda()
    inv, _ = rope_frequencies(128, 1e4, device="cuda")
    _check(x, rope(x, None, inv, pos.cuda()), inv, pos)
    if dtype == torch.int64:
        start = 2 ** 33
        _check(x, rope(x, None, inv, offset=start), inv, start + torch.arange(8)[None])


def test_positions_of_every_shape(gpu):
    q = _rand(1, 3, 5, 2, 64).cuda()
    inv, _ = rope_frequencies(64, 1e4, device="cuda")
    pos = torch.tensor([4, 0, 9, 9, 300])
    shared = rope(q, None, inv, pos.cuda())
    _check(q, shared, inv, pos.expand(3, 5))
    assert torch.equal(shared, rope(q, None, inv, pos.expand(3, 5).cuda()))
    assert torch.equal(shared, rope(q, None, inv, pos.int().cuda()[None].expand(3, 5)))
    wide = torch.zeros(3, 10, dtype=torch.int64, device="cuda")
    wide[:, ::2] = pos.cuda()
    assert torch.equal(shared, rope(q, None, inv, wide[:, ::2]))
    assert torch.equal(rope(q, None, inv), rope(q, None, inv, torch.arange(5).cuda()))


@pytest.mark.parametrize("dtype", [BF, SF])
def test_views(gpu, dtype):
    """Heads of a fused projection, transposed heads, rows off 16 bytes, channels apart."""
    inv, _ = rope_frequencies(64, 1e4, device="cuda")
    pos = torch.arange(9).expand(2, 9)
    qkv = _rand(1, 2, 9, 8, 64, dtype=dtype).cuda()
    q, k, _ = qkv.split((4, 2, 2), 2)
    for x in (q, k, qkv.transpose(1, 2).contiguous().transpose(1, 2)):
        _check(x, rope(x, None, inv, pos.cuda()), inv, pos)
    odd = torch.empty(2 * 9 * 3 * 65 + 1, dtype=dtype, device="cuda")[1:].view(2, 9, 3, 65)
    odd.copy_(_rand(5, 2, 9, 3, 65, dtype=dtype))
    for x in (odd[..., :64], odd[..., 1:], qkv.transpose(2, 3).contiguous().transpose(2, 3)):
        _check(x, rope(x, None, inv, pos.cuda()), inv, pos)
    a, b = rope(odd[..., :64], k, inv, pos.cuda())
    _check(odd[..., :64], a, inv, pos)
    _check(k, b, inv, pos)


@pytest.mark.parametrize("interleaved", [False, True])
def test_the_inverse_is_the_gradient(gpu, interleaved):
    """y = R x is linear: <g, R x> = <R' g, x>, R' the inverse at scale 1 and scale times it
    else. Sums of 12288 products of N(0, 1): each side is off by 12288^0.5 2^-20 or so."""
    x, g = (_rand(i, 2, 24, 4, 64, dtype=SF).cuda() for i in (1, 2))
    inv, _ = rope_frequencies(48, 1e4, device="cuda")
    kw = dict(interleaved=interleaved, offset=100)
    y = rope(x, None, inv, **kw)
    back = rope(g, None, inv, inverse=True, **kw)
    assert abs((g.double() * y).sum() - (back.double() * x).sum()) < 12288 ** 0.5 * 2.0 ** -19
    # and by differences, one channel at a time: of a linear map exact but for rounding
    for at in ((0, 0, 0, 0), (1, 23, 3, 47), (0, 7, 2, 63), (1, 5, 1, 24)):
        e = x.clone()
        e[at] += 1
        diff = (g.double() * (rope(e, None, inv, **kw).double() - y.double())).sum()
        assert abs(diff - back[at]) < 1e-4
    assert (rope(y, None, inv, inverse=True, **kw) - x).abs().max() < 8 * 2.0 ** -21 * x.abs().max()


def test_agrees_with_the_prologue(gpu):
    """The prologue's tables hold rounded cosines of angles in 32 bits: near positions agree to
    the tables' rounding."""
    q, k = _rand(1, 1, 64, 4, 128).cuda(), _rand(2, 1, 64, 2, 128).cuda()
    inv = ttcd_amd.rope_inv_freq(128, 1e6, "cuda")
    cos, sin = ttcd_amd.rope_tables(inv, 64)
    for x, y in zip(ttcd_amd.qk_norm_rope(q, k, None, None, 0.0, cos, sin), rope(q, k, inv)):
        # u (|x0| + |x1|) of the tables, u |y| of either result, |y| <= 2 ** 0.5 max |x|
        assert (x.double() - y.double()).abs().max() <= 5 * U[BF] * q.abs().max().double()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,n", [(64, 32), (64, 7), (96, 5), (10, 5)])
def test_outputs_in_place(gpu, interleaved, D, n):
    """The C entry writes over its inputs, the border of what turns within a vector or not."""
    q, k = _rand(1, 2, 33, 3, D).cuda(), _rand(2, 2, 33, 2, D).cuda()
    inv, _ = rope_frequencies(2 * n, 1e4, device="cuda")
    want = rope(q, k, inv, offset=3, interleaved=interleaved)
    qs, ks = (_lib.strides4(x.stride()) for x in (q, k))
    _lib.check(_lib.lib().ttcd_rope_fwd(
        q.data_ptr(), k.data_ptr(), q.data_ptr(), k.data_ptr(), inv.data_ptr(), n, None, 0, None, 3,
        2, 33, 3, 2, D, qs, ks, qs, ks, int(interleaved), 0, 1.0, _lib.DTYPE_BF16, _lib.stream(q)))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_empty_and_another_stream_and_a_graph(gpu):
    inv, _ = rope_frequencies(64, 1e4, device="cuda")
    for shape in ((0, 4, 2, 64), (2, 0, 2, 64)):
        assert rope(torch.empty(shape, dtype=BF, device="cuda"), None, inv).shape == shape
    q, k = _rand(1, 1, 6, 2, 64).cuda(), torch.empty(1, 6, 0, 64, dtype=BF, device="cuda")
    assert rope(q, k, inv)[1].shape == k.shape
    pos = torch.arange(6, device="cuda", dtype=torch.int32)
    want = rope(q, None, inv, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rope(q, None, inv, pos)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = rope(q, None, inv, pos)
    for step in range(3):
        pos.fill_(step)
        q.copy_(_rand(step, 1, 6, 2, 64))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, rope(q, None, inv, pos))


def test_refusals(gpu):
    q, inv = _rand(1, 1, 4, 2, 64).cuda(), torch.ones(32, device="cuda")
    pos = torch.arange(4, device="cuda")
    bad = [lambda: rope(q[0], None, inv), lambda: rope(q, q[:, :2], inv),
           lambda: rope(q, q[..., :32], inv), lambda: rope(q, q.half(), inv),
           lambda: rope(q.double(), None, inv), lambda: rope(q, None, inv.half()),
           lambda: rope(q, None, torch.ones(33, device="cuda")), lambda: rope(q, None, inv[:0]),
           lambda: rope(q, None, inv, pos.float()), lambda: rope(q, None, inv, pos[:3]),
           lambda: rope(q, None, inv.cpu()), lambda: rope(q, None, inv, pos.cpu()),
           lambda: rope(q, None, inv, pos.view(4, 1)), lambda: rope(q, None, inv, scale=float("nan"))]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError, match="forward-only"):
        rope(q.requires_grad_(), None, inv)


@pytest.mark.parametrize("interleaved", [False, True])
def test_the_farthest_positions(gpu, interleaved):
    """Where position * inv_freq passes 53 bits (2^29 with 24 bits of a frequency) the angle is
    exact all the same: the oracle multiplies in integers. The same bounds as near by."""
    pos = torch.tensor([[2 ** 29 + 1, 2 ** 31 + 7, 2 ** 40 - 1, -2 ** 45 + 9, 2 ** 50 + 3,
                         2 ** 52 + 12345, 2 ** 53 - 1, 2 ** 53, -2 ** 53 + 1]])
    x = _rand(1, 1, 9, 2, 128, dtype=SF).cuda()
    for base in (1e4, 1e6):
        inv, _ = rope_frequencies(128, base, device="cuda")
        _check(x, rope(x, None, inv, pos.cuda(), interleaved=interleaved), inv, pos,
               interleaved=interleaved)
    start = 2 ** 53 - 9
    _check(x, rope(x, None, inv, offset=start, interleaved=interleaved), inv,
           start + torch.arange(9)[None], interleaved=interleaved)


def test_offsets_that_are_no_position(gpu):
    q, inv = _rand(1, 1, 4, 2, 64).cuda(), torch.ones(32, device="cuda")
    for offset in (2 ** 53 - 2, 2 ** 53 + 1, 2 ** 64 + 5, -2 ** 53 - 1, -2 ** 70):
        with pytest.raises(ValueError, match="position"):
            rope(q, None, inv, offset=offset)
    rope(q, None, inv, offset=2 ** 53 - 3), rope(q, None, inv, offset=-2 ** 53)


def test_a_scaled_key_is_turned_back(gpu):
    """With a scale (yarn's) inverse=True alone is the gradient, scale times the inverse; a key's
    position comes off with the scale's reciprocal. Two passes, each off by 2^-21 scale
    (|x0| + |x1|) and its rounding, and the reciprocal by 2^-24."""
    inv, s = rope_frequencies(64, 1e4, {"rope_type": "yarn", "factor": 4.0,
                                        "original_max_position_embeddings": 2048}, device="cuda")
    assert s > 1.1
    k = _rand(1, 2, 40, 3, 64, dtype=SF).cuda()
    turned = rope(k, None, inv, offset=70000, scale=s)
    limit = 8 * 2.0 ** -21 * k.abs().max()
    assert (rope(turned, None, inv, offset=70000, inverse=True, scale=1 / s) - k).abs().max() < limit
    grad = rope(turned, None, inv, offset=70000, inverse=True, scale=s)
    assert (grad - s * s * k).abs().max() < 2 * limit

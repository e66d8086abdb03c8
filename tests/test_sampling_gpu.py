"""Sampling and the walk over a tree on the GPU against the oracle. Tokens are equal: weights
and sums are 64 bits on either side, a few 2^-53 apart, so a drawn border is passed
differently once in 10^10 rows or so. A log-probability is rounded to 32 bits once."""
from __future__ import annotations

import math

import pytest
import torch

from oracle import drafted_ref as ref
from ttcd_amd import sample, tree_accept

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
NAN, INF = math.nan, math.inf


def _logits(seed, R, V, dtype, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(R, V, generator=g) * spread).to(dtype)


def _uniform(seed, R):
    return torch.rand(R, generator=torch.Generator().manual_seed(seed))


def _check(x, u, cuda_x=None, **kw):
    """All rows of x (R, V) against the oracle; settings numbers, or lists of one a row."""
    R = x.shape[0]
    gpu = {}
    for name, v in kw.items():
        if isinstance(v, list):
            dt = torch.int32 if name == "top_k" else torch.float32
            v = torch.tensor(v, dtype=dt).cuda()
            kw[name] = v.tolist()
        gpu[name] = v
    tok, lp = sample(x.cuda() if cuda_x is None else cuda_x, u.cuda(), return_logprob=True, **gpu)
    assert tok.dtype == torch.int64 and tok.shape == (R,) and lp.dtype == torch.float32
    for r in range(R):
        row = {n: v[r] if isinstance(v, list) else v for n, v in kw.items()}
        want, wl = ref.sample(x[r].tolist(), float(u[r]), **row)
        assert int(tok[r]) == want, (r, int(tok[r]), want, row)
        got = float(lp[r])
        assert got == wl or abs(got - wl) <= 2.0 ** -24 * abs(wl) + 1e-12, (r, got, wl)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 15, 16, 17, 100, 1000, 4099])
def test_sizes_and_settings(gpu, dtype, V):
    for seed, kw in enumerate((dict(), dict(temperature=0.3), dict(temperature=7.0),
                               dict(temperature=0), dict(top_k=1), dict(top_k=3),
                               dict(top_k=max(1, V // 2)), dict(top_k=V + 5), dict(top_p=0.9),
                               dict(top_p=0.1), dict(top_p=1e-9), dict(top_p=2.0), dict(min_p=0.05),
                               dict(min_p=1.0), dict(top_k=40, top_p=0.8),
                               dict(temperature=0.7, top_k=20, top_p=0.8, min_p=0.1),
                               dict(top_p=0.95, min_p=0.02), dict(top_k=5, min_p=0.3))):
        _check(_logits(seed, 6, V, dtype), _uniform(seed, 6), **kw)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("V", [65535, 65550, 151936])
def test_vocabularies(gpu, dtype, V):
    x = _logits(1, 3, V, dtype)
    x[:, V - 300:] = -INF
    for kw in (dict(), dict(temperature=0.7, top_k=20, top_p=0.8), dict(top_k=50000, top_p=0.97),
               dict(temperature=3.0, min_p=0.01), dict(temperature=0)):
        _check(x, _uniform(V, 3), **kw)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_temperatures_whose_quotient_is_infinite(gpu, dtype):
    """The highest weigh 1 each and nothing else anything, down to the least temperature."""
    x = _logits(7, 4, 1003, dtype)
    x[1, [9, 500, 1002]] = 20.0
    x[2] = -3.0
    x[3, 700] = INF
    u = torch.tensor([0.5, 0.7, 0.999, 0.2])
    for t in (1e-30, 1e-299, 1e-309, 5e-324):
        _check(x, u, temperature=t)
        _check(x, u, temperature=t, top_p=0.9, min_p=0.5)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_few_kept_of_many(gpu, dtype):
    """Rows long enough for a bound under the first top_k: ordinary ones, all equal, all
    negative, one peak beside nothing, the peak in the first vector, few numbers, NaN above."""
    V = 40007
    x = _logits(2, 9, V, dtype)
    x[1] = 1.5
    x[2] = -x[2].abs() - 1
    x[3] = 0.0
    x[3, 30000] = 9.0
    x[4] = x[4].abs() * 0.01
    x[4, 3] = 30.0
    x[5, 100:] = -INF
    x[6, 12345] = NAN
    x[7] = torch.arange(V).flip(0).div(400).floor().to(dtype)
    x[8, 20:] = 0.25
    u = _uniform(3, 9)
    for k in (1, 2, 20, 63, 64, 65, 300, 1023, 1024, 1025):
        _check(x, u, top_k=k)
        _check(x[:, 3:], 1 - u, temperature=0.6, top_k=k, top_p=0.9, min_p=0.01)
    _check(x, u, temperature=0)
    _check(x[:, :32770], u, top_k=[1, 5, 64, 0, 1024, 7, 9, 2000, 33])


@pytest.mark.parametrize("dtype", [BF, HF])
def test_values_that_come_often(gpu, dtype):
    """Counts past 16 bits, in the first stretch and over several: all equal, two values, a
    masked half."""
    V = 250001
    same = torch.zeros(5, V, dtype=dtype)
    same[1] = -3.5
    same[2, ::2] = 1.0
    same[3, 65536:] = -INF
    same[4, :] = -INF
    same[4, 70000] = 0.25
    u = torch.tensor([0.3, 0.999, 0.77, 0.5, 0.9])
    _check(same, u)
    _check(same, u, top_k=140000)
    _check(same, u, top_p=0.6)
    _check(same[:, :200000], u, temperature=0.5, top_k=[70000, 0, 100001, 65535, 1],
           top_p=[0.5, 0.9, 1.0, 0.99, 0.1])
    most = torch.full((1, 1 << 20), 2.0, dtype=dtype)
    tok, lp = sample(most.cuda(), torch.tensor([0.75]).cuda(), return_logprob=True)
    assert tok.item() == 3 << 18 and abs(lp.item() + 20 * math.log(2)) < 1e-6


@pytest.mark.parametrize("dtype", [BF, HF])
def test_no_numbers_and_infinities(gpu, dtype):
    x = _logits(3, 9, 70, dtype)
    x[0] = -INF
    x[1] = NAN
    x[2, ::3] = NAN
    x[3, 5:9] = INF
    x[4] = -x[4].abs()
    x[4, 11] = -NAN
    x[5] = INF
    x[6, 1:] = -INF
    x[7] = torch.tensor([0.0, -0.0] * 35)
    x[8] = torch.where(torch.arange(70) % 3 == 0, -0.0, -1.0)
    x[8, 9] = 0.0
    for seed in range(4):
        for kw in (dict(), dict(temperature=0), dict(top_k=4), dict(top_p=0.7), dict(min_p=0.4)):
            _check(x, _uniform(seed, 9), **kw)


def test_the_least_and_largest_numbers(gpu):
    """Subnormal logits are values of their own; the largest ones' differences overflow no
    weight."""
    for dtype, tiny in ((BF, 2.0 ** -133), (HF, 2.0 ** -24)):
        top = torch.finfo(dtype).max
        x = torch.tensor([[0.0, tiny, 2 * tiny, -tiny, -0.0, 3 * tiny, tiny, -2 * tiny],
                          [top, -top, 0.0, top, 1.0, -top, top, -1.0]]).to(dtype)
        for i in range(8):
            u = torch.full((2,), i / 8 + 0.01)
            for kw in (dict(), dict(top_k=5), dict(top_p=0.6), dict(temperature=1e-3)):
                _check(x, u, **kw)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_zero_without_a_sign_alone_and_nan_above_all(gpu, dtype):
    x = -_logits(4, 6, 3001, dtype).abs() - 0.5
    x[0, 5::7] = -0.0
    x[1, 17] = -0.0
    x[2, 100] = NAN
    x[3] = NAN
    x[3, 2999] = -2.0
    x[4, ::2] = -NAN
    x[5, 1:] = NAN
    for kw in (dict(), dict(top_k=9), dict(top_p=0.5), dict(min_p=0.9), dict(temperature=0)):
        _check(x, _uniform(2, 6), **kw)


def test_ties_go_to_the_lower_index(gpu):
    x = torch.zeros(12, 24, dtype=BF)
    x[:, 3::4] = 1.0
    u = torch.arange(12) / 12.0
    for k in (1, 2, 6, 7, 24):
        _check(x, u, top_k=k)
    for p in (0.2, 0.5, 0.75):
        _check(x, u, top_p=p)


@pytest.mark.parametrize("V", [13, 4096, 5003])
def test_rows_at_any_address(gpu, V):
    wide = _logits(V, 9, V + 11, BF).cuda()
    for start in range(9):
        part = wide[:, start:start + V]
        _check(part.cpu(), _uniform(start, 9), cuda_x=part, top_p=0.9)
    back = wide.T.contiguous().T[:, :V]  # a row's logits apart
    _check(back.cpu(), _uniform(1, 9), cuda_x=back)
    same = wide[:1, :V].expand(9, V)  # every row the same memory
    _check(same.cpu(), _uniform(2, 9), cuda_x=same)


def test_a_setting_a_row(gpu):
    x = _logits(5, 8, 3000, BF)
    _check(x, _uniform(5, 8), temperature=[0.0, 0.5, 1.0, 1.5, 0.2, 3.0, 1.0, 0.0],
           top_k=[0, 7, 3001, 1, 0, 40, 2, 9], top_p=[1.0, 0.5, 0.9, 1.0, 0.99, 0.3, 1.0, 0.5],
           min_p=[0.0, 0.0, 0.02, 0.5, 0.0, 0.1, 0.0, 1.0])
    # out of range, as the header says: a row of each against what it is taken as
    cols = dict(temperature=[-1.0, NAN, 1.0, 1.0, 1.0, 1.0, 1.0, 1.0],
                top_k=[0, 0, -5, 0, 0, 0, 0, 0], top_p=[1.0, 1.0, 1.0, -0.5, NAN, 5.0, 1.0, 1.0],
                min_p=[0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 7.0, -2.0])
    gpu_kw = {n: torch.tensor(v, dtype=torch.int32 if n == "top_k" else torch.float32).cuda()
              for n, v in cols.items()}
    u = _uniform(6, 8)
    tok = sample(x.cuda(), u.cuda(), **gpu_kw)
    taken = [dict(temperature=0), dict(temperature=0), dict(), dict(top_k=1), dict(), dict(),
             dict(min_p=1.0), dict()]
    for r, kw in enumerate(taken):
        assert int(tok[r]) == ref.sample(x[r].tolist(), float(u[r]), **kw)[0]


def test_shapes_and_the_same_token_every_time(gpu):
    x, u = _logits(7, 24, 9001, BF).cuda(), _uniform(7, 24).cuda()
    want = sample(x, u, top_p=0.95)
    assert torch.equal(sample(x.view(2, 3, 4, -1), u.view(2, 3, 4), top_p=0.95), want.view(2, 3, 4))
    assert sample(x[3], u[3], top_p=0.95) == want[3] and sample(x[3], u[3]).shape == ()
    assert sample(x[:0], u[:0]).shape == (0,)
    for _ in range(20):
        assert torch.equal(sample(x, u, top_p=0.95), want)


def test_uniform_at_its_ends(gpu):
    x = _logits(8, 4, 2000, HF)
    for v in (0.0, 1.0 - 2.0 ** -24, 2.0 ** -149):
        _check(x, torch.full((4,), v))
    # out of [0, 1): no access goes by it, and a kept token comes
    tok = sample(x.cuda(), torch.tensor([1.0, 5.0, -3.0, NAN]).cuda(), top_k=3)
    for r in range(4):
        assert int(tok[r]) in x[r].double().topk(6).indices.tolist()


def test_draws_are_spread_as_the_weights_are(gpu):
    """u = (i + 1/2) / n for all i: each token comes n p times, but for one at either end."""
    x = _logits(9, 1, 50, BF)
    n = 4096
    u = (torch.arange(n) + 0.5) / n
    tok = sample(x.expand(n, 50).cuda(), u.cuda())
    got = torch.bincount(tok.cpu(), minlength=50).double()
    assert (got - n * x[0].double().softmax(0)).abs().max() <= 1.0 + 1e-6


def test_another_stream_and_a_graph(gpu):
    x, u = _logits(1, 5, 20000, BF).cuda(), _uniform(1, 5).cuda()
    want = sample(x, u, top_k=50)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sample(x, u, top_k=50)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tok, lp = sample(x, u, top_k=50, return_logprob=True)
    for seed in range(4):
        x.copy_(_logits(seed, 5, 20000, BF))
        u.copy_(_uniform(seed, 5))
        graph.replay()
        torch.cuda.synchronize()
        a, b = sample(x, u, top_k=50, return_logprob=True)
        assert torch.equal(tok, a) and torch.equal(lp, b)


@pytest.mark.parametrize("B,N", [(1, 1), (3, 2), (5, 16), (4, 64), (3, 65), (2, 200), (7, 256)])
def test_walks(gpu, B, N):
    g = torch.Generator().manual_seed(N)
    for turn in range(6):
        parents = torch.stack([torch.tensor([-1] + [
            int(torch.randint(max(0, i - 1 - 5 * turn), i, (1,), generator=g))
            for i in range(1, N)]) for _ in range(B)])
        picked = torch.randint(0, 3, (B, N), generator=g)  # few tokens: several children agree
        tokens = torch.randint(0, 3, (B, N), generator=g)
        if turn == 5:  # chains that agree to their end
            parents = (torch.arange(N) - 1).expand(B, N).clone()
            tokens = picked.gather(1, parents.clamp(min=0))
        counts = torch.tensor([max(0, N - 3 * b) for b in range(B)], dtype=torch.int32)
        for c in (None, counts):
            path, n, following = tree_accept(parents.int().cuda(), tokens.cuda(), picked.cuda(),
                                             counts=None if c is None else c.cuda())
            assert path.dtype == n.dtype == torch.int32 and following.dtype == torch.int64
            for b in range(B):
                want, after = ref.accept(parents[b].tolist(), tokens[b].tolist(),
                                         picked[b].tolist(), N if c is None else int(c[b]))
                assert path[b].tolist() == want + [-1] * (N - len(want))
                assert int(n[b]) == len(want) and int(following[b]) == after


def test_walks_of_malformed_trees_end(gpu):
    """Parents that do not come before their node are none; counts out of range are the nearest."""
    parents = torch.tensor([[3, 0, 2, 1, 99, -7, 4, 6]], dtype=torch.int32).cuda()
    one = torch.ones(1, 8, dtype=torch.int64, device="cuda")
    for c, want in ((None, [0, 1, 3]), (99, [0, 1, 3]), (-4, []), (2, [0, 1])):
        counts = None if c is None else torch.tensor([c], dtype=torch.int32).cuda()
        path, n, following = tree_accept(parents, one, one, counts=counts)
        assert path[0, :len(want)].tolist() == want and n.item() == len(want)
        assert (path[0, len(want):] == -1).all() and following.item() == (1 if want else -1)
    big = torch.tensor([[2 ** 62 + 1, -5]]).cuda()  # tokens are 64 bits
    path, _, following = tree_accept(torch.tensor([[-1, 0]], dtype=torch.int32).cuda(),
                                     big.flip(1), big, counts=None)
    assert path[0].tolist() == [0, 1] and following.item() == -5


def test_refusals(gpu):
    x, u = _logits(0, 2, 16, BF).cuda(), torch.zeros(2, device="cuda")
    ones = torch.ones(2, device="cuda")
    bad = [lambda: sample(x.float(), u), lambda: sample(x, u[:1]), lambda: sample(x, u.double()),
           lambda: sample(x, u.cpu()), lambda: sample(x[:, :0], u),
           lambda: sample(x, u, temperature=-1.0), lambda: sample(x, u, temperature=NAN),
           lambda: sample(x, u, top_k=-1), lambda: sample(x, u, top_k=1.5),
           lambda: sample(x, u, top_p=0.0), lambda: sample(x, u, min_p=1.1),
           lambda: sample(x, u, top_k=ones), lambda: sample(x, u, top_p=ones.cpu()),
           lambda: sample(x, u, temperature=ones[:1]), lambda: sample(x, u, min_p=ones.double())]
    i, t = torch.zeros(2, 4, dtype=torch.int32, device="cuda"), torch.zeros(2, 4, dtype=torch.int64,
                                                                          device="cuda")
    bad += [lambda: tree_accept(i.long(), t, t), lambda: tree_accept(i, i, t),
            lambda: tree_accept(i, t, t[:, :3]), lambda: tree_accept(i[0], t, t),
            lambda: tree_accept(i, t, t.cpu()), lambda: tree_accept(i, t, t, counts=t[:, 0]),
            lambda: tree_accept(i[:, :0], t[:, :0], t[:, :0])]
    for call in bad:
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError, match="forward-only"):
        sample(x.requires_grad_(), u)
    assert [y.shape[0] for y in tree_accept(i[:0], t[:0], t[:0])] == [0, 0, 0]

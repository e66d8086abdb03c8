"""The ipttcdv9 model with drafted tokens over the 4-bit cache on the GPU. A tree's logits are
compared with those of its paths over a bf16 cache that is given the keys and values which the
4-bit one holds (so that both attend over the same numbers, as test_kv4_model_gpu tells), and a
generated text with what the oracle picks from the logits that the model gave on the way."""
from __future__ import annotations

import pytest
import torch

from oracle import drafted_ref as ref
from test_ipttcdv9_gpu import TINY, _ids, _logits_close
from test_kv4_model_gpu import FourBits, HeldCache
from ttcd_amd import IPTTCDv9Cache, ipttcdv9 as M, kv4_read, sample, tree_accept

pytestmark = pytest.mark.gpu
DEV = "cuda"
CFGS = [{}, {"window_size": None}, {"ttt_layers": [], "window_size": 64, "num_heads": 6}]
TREE = [-1, 0, 0, 1, 1, 2, 5, -1, 7, 6]


def _model(cfg, seed=0):
    c = dict(TINY, **cfg)
    return M.IPTTCDv9Prefill(c, M.init_weights(c, DEV, seed=seed))


def _cache(capacity=1024):
    return IPTTCDv9Cache(bits=4, capacity=capacity)


class Drafted(FourBits):
    """`nodes` holds what the drafts hold of each layer's."""

    def __init__(self, **kw):
        super().__init__(**kw)
        self.nodes = {}

    def draft(self, layer, k, v):
        held = super().draft(layer, k, v)
        self.nodes[layer] = kv4_read(self.drafts[layer], k.shape[1])
        return held


class Taken:
    """What HeldCache is given: the nodes of `line`."""

    def __init__(self, four, line):
        self.last = {i: tuple(x[:, line] for x in kv) for i, kv in four.nodes.items()}


def _along(held, four, line):
    """A copy of the bf16 cache that goes on along a path of the tree."""
    out = HeldCache(Taken(four, line))
    out.kv, out.seen, out._shape = dict(held.kv), held.seen, held._shape
    return out


@pytest.mark.parametrize("cfg", CFGS)
@pytest.mark.parametrize("prompt", [1, 97, 300])
def test_a_tree_is_its_paths(cfg, prompt):
    m = _model(cfg)
    ids, tokens = _ids(1, prompt, 3).to(DEV), _ids(1, len(TREE), 5).to(DEV)
    four = Drafted(capacity=1024)
    held = HeldCache(four)
    m.forward(ids, cache=four)
    m.forward(ids, cache=held)
    before = [kv4_read(c, prompt) for c in four.kv4.values()]
    got = m.forward(tokens, cache=four, tree=TREE)
    again = m.forward(tokens, cache=four, tree=torch.tensor(TREE))  # not accepted: as before
    assert got.shape == (1, len(TREE), 1024) and torch.equal(got, again)
    assert four.seen == prompt
    for c, (k, v) in zip(four.kv4.values(), before):
        a, b = kv4_read(c, prompt)
        assert torch.equal(a, k) and torch.equal(b, v)
    for line in ref.lineage(TREE):
        want = m.forward(tokens[:, line], logits_to_keep=1, cache=_along(held, four, line))
        _logits_close(got[:, line[-1]], want[:, 0])


@pytest.mark.parametrize("cfg", CFGS)
def test_accepted_nodes_are_the_next_tokens(cfg):
    """What a tree of which a path is accepted leaves, and the token after it."""
    m = _model(cfg)
    ids, tokens = _ids(1, 60, 1).to(DEV), _ids(1, len(TREE), 2).to(DEV)
    four = Drafted(capacity=1024)
    held = HeldCache(four)
    m.forward(ids, cache=four)
    m.forward(ids, cache=held)
    m.forward(tokens, cache=four, tree=TREE)
    line = [0, 2, 5]
    path = torch.full((1, len(TREE)), -1, dtype=torch.int32, device=DEV)
    path[0, :3] = torch.tensor(line)
    assert four.accept(path, torch.tensor([3], dtype=torch.int32, device=DEV)) == 3
    assert four.seen == four.held == 63
    for i, c in four.kv4.items():
        assert c.lengths.tolist() == [63] and four.drafts[i].lengths.tolist() == [0]
        for x, y in zip(kv4_read(c, 3), four.nodes[i]):
            assert torch.equal(x, y[:, line])
    with pytest.raises(RuntimeError, match="no tree"):
        four.accept(path, path[:, 0])
    bf16 = _along(held, four, line)
    m.forward(tokens[:, line], cache=bf16)
    nxt = _ids(1, 1, 9).to(DEV)
    got = m.forward(nxt, cache=four)
    bf16.four = four
    _logits_close(got, m.forward(nxt, cache=bf16))


def _recorded(m, ids, count, u, kw, draft=None):
    """(the text, what the oracle makes of the logits of its calls, the calls' nodes)."""
    calls = []
    forward = m.forward

    def record(x, **k):
        y = forward(x, **k)
        calls.append((x[0].tolist(), k.get("tree"), y[0].float().cpu(), k["cache"].seen))
        return y
    m.forward = record
    cache = _cache()
    text = m.generate(ids, count, None if u is None else u.to(DEV), draft=draft, cache=cache, **kw)
    m.forward = forward
    assert text.shape == (1, count) and text.dtype == torch.int64
    assert cache.seen == ids.shape[1] + count - 1  # all but the last token
    u = [0.0] * count if u is None else u.tolist()
    want = []
    for tokens, tree, logits, _ in calls:
        def pick(row, place):
            return ref.sample(row.tolist(), u[min(place, count - 1)], **kw)[0]
        if tree is None:
            want.append(pick(logits[-1], len(want)))
            continue
        lines = ref.lineage(tree)
        picked = [pick(row, len(want) + len(line) - 1) for row, line in zip(logits, lines)]
        path, after = ref.accept(tree, tokens, picked, len(tree))
        want += [tokens[i] for i in path[1:]] + [after]
    return text[0].tolist(), want[:count], [len(c[0]) for c in calls[1:]]


@pytest.mark.parametrize("cfg", CFGS)
@pytest.mark.parametrize("kw", [dict(temperature=0), dict(temperature=0.7, top_k=8),
                                dict(temperature=1.0, top_p=0.8, min_p=0.01)])
def test_generated_text_is_what_its_logits_say(cfg, kw):
    m = _model(cfg, seed=2)
    ids = _ids(1, 40, 7).to(DEV)
    u = None if kw["temperature"] == 0 else torch.rand(
        24, generator=torch.Generator().manual_seed(3))
    plain, want, nodes = _recorded(m, ids, 24, u, kw)
    assert plain == want and nodes == [1] * 23
    known = ids[0].tolist() + plain

    def right(text, most):
        """The tokens of the plain text, a wrong one beside each, and a wrong end."""
        parents, tokens, last = [], [], -1
        for t in known[len(text):len(text) + min(most, 4)]:
            parents += [last, last]
            tokens += [(t + 1) % 1024, t]
            last = len(tokens) - 1
        return parents + [last], tokens + [5]

    for draft in (right, lambda t, n: ([-1, 0], [3, 4]),
                  lambda t, n: ([], []) if len(t) % 2 else ([-1] * 300, list(range(300)))):
        text, want, nodes = _recorded(m, ids, 24, u, kw, draft)
        assert text == want
        if draft is right and text == plain:  # every right draft was taken, 5 tokens a call
            assert len(nodes) == 5
    one, want, nodes = _recorded(m, ids, 1, None if u is None else u[:1], kw, right)
    assert one == want and nodes == []


def test_generate_makes_its_own_cache():
    for cfg in CFGS:
        m = _model(cfg, seed=3)
        ids = _ids(1, 300, 8).to(DEV)
        a = m.generate(ids, 6, temperature=0, draft=lambda t, n: ([-1, 0, 1], [1, 2, 3]))
        b = m.generate(ids, 6, temperature=0, draft=lambda t, n: ([-1, 0, 1], [1, 2, 3]),
                       cache=_cache())
        assert torch.equal(a, b)


def test_a_step_by_hand():
    """The calls of a step one by one, twice in a row, the second tree larger than the first
    one's draft."""
    m = _model({"window_size": None}, seed=3)
    cache = _cache()
    logits = m.forward(_ids(1, 20, 8).to(DEV), cache=cache)[:, -1]
    u = torch.rand(1, 40, generator=torch.Generator().manual_seed(1)).to(DEV)
    last = sample(logits, u[0, :1], temperature=0.8)
    seen = 20
    for tree in ([-1, 0, 0, 1], [-1] + [i // 2 for i in range(39)]):
        N = len(tree)
        nodes = torch.cat((last[None], _ids(1, N - 1, N).to(DEV)), 1)
        logits = m.forward(nodes, cache=cache, tree=tree)
        picked = sample(logits, u[:, :N], temperature=0.8, top_p=0.9)
        nodes[0, 2] = picked[0, 0]  # so that it agrees
        parents = torch.tensor([tree], dtype=torch.int32, device=DEV)
        path, n, last = tree_accept(parents, nodes, picked)
        assert path[0, 1] in (1, 2)
        seen += cache.accept(path, n)
        assert cache.seen == seen and all(c.lengths.item() == seen for c in cache.kv4.values())


def test_refusals():
    m = _model({})
    ids, one = _ids(1, 4, 0).to(DEV), [-1, 0, 1, 2]
    with pytest.raises(ValueError, match="IPTTCDv9Cache"):
        m.forward(ids, tree=one)
    with pytest.raises(NotImplementedError, match="4-bit"):
        m.forward(ids, cache=IPTTCDv9Cache(), tree=one)
    with pytest.raises(NotImplementedError, match="one sequence"):
        m.forward(ids.expand(2, 4), cache=_cache(), tree=one)
    full = _model({"window_size": None, "ttt_layers": []})
    with pytest.raises(NotImplementedError, match="keeps"):
        full.forward(ids, cache=IPTTCDv9Cache(bits=4, capacity=1024, keep=64), tree=one)
    for bad in ([-1, 0, 1], [0, 0, 1, 2], [-1, 1, 1, 2], [-1, 0, 1, -2]):
        with pytest.raises(ValueError, match="parents"):
            m.forward(ids, cache=_cache(), tree=bad)
    with pytest.raises(ValueError, match="nodes"):  # ttt_chunk is 256
        m.forward(_ids(1, 256, 0).to(DEV), cache=_cache(), tree=[-1] * 256)
    small = _model({"window_size": None})
    with pytest.raises(ValueError, match="positions"):
        small.forward(_ids(1, 40, 0).to(DEV), cache=_cache(32), tree=[-1] * 40)
    cache = _cache()
    m.forward(ids, cache=cache, tree=one)
    with pytest.raises(ValueError, match="path"):
        cache.accept(torch.zeros(1, 3, dtype=torch.int32, device=DEV), torch.ones(1, device=DEV))
    # nothing was written: the right call still goes
    for p, n in ((torch.zeros(1, 4, device=DEV), torch.ones(1, dtype=torch.int32, device=DEV)),
                 (torch.zeros(1, 4, dtype=torch.int32, device=DEV), torch.ones(1, device=DEV)),
                 (torch.zeros(1, 4, dtype=torch.int32, device=DEV),
                  torch.ones(2, dtype=torch.int32, device=DEV))):
        with pytest.raises(ValueError, match="int32"):
            cache.accept(p, n)
    path, n = torch.zeros(1, 4, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32,
                                                                            device=DEV)
    assert cache.accept(path, n) == 1 and cache.seen == 1
    # a tree that other tokens have passed is of another place
    m.forward(ids, cache=cache, tree=one)
    m.forward(ids, cache=cache)
    with pytest.raises(RuntimeError, match="no tree"):
        cache.accept(path, n)
    assert cache.seen == 5
    u = torch.zeros(3, device=DEV)
    for bad in (lambda: m.generate(ids, 0, u), lambda: m.generate(ids, 3), lambda: m.generate(ids, 4, u),
                lambda: m.generate(ids.expand(2, 4), 3, u),
                lambda: m.generate(ids, 3, u, draft=lambda t, n: ([-1], [])),
                lambda: m.generate(ids, 3, u, draft=lambda t, n: ([-2], [1])),
                lambda: m.generate(ids, 3, u, draft=lambda t, n: ([0], [1])),
                lambda: m.generate(ids, 3, u, draft=lambda t, n: ([-1], [-1])),
                lambda: m.generate(ids, 3, u, draft=lambda t, n: ([-1], [m.cfg["vocab_size"]]))):
        with pytest.raises(ValueError):
            bad()


def test_logits_that_are_no_numbers_end_a_text():
    """A token -1 goes into no embedding."""
    m = _model({"window_size": None})
    m.w = dict(m.w)
    m.w["lm_head.weight"] = torch.full_like(m.w["lm_head.weight"], float("nan"))
    u = torch.zeros(3, device=DEV)
    ids = _ids(1, 4, 0).to(DEV)
    assert m.generate(ids, 1, u[:1]).tolist() == [[-1]]
    for draft in (None, lambda t, n: ([-1], [1])):
        with pytest.raises(RuntimeError, match="no logit"):
            m.generate(ids, 3, u, draft=draft)


def _bush(vocab, nodes):
    """As many drafted tokens after every text, whatever is of use: a chain and leaves."""
    def draft(text, most):
        parents = [-1] + [max(0, i - 1 - i % 3) for i in range(1, nodes)]
        return parents, [(text[-1] + 7 * i) % vocab for i in range(nodes)]
    return draft


@pytest.mark.parametrize("cfg", CFGS[1:])
@pytest.mark.parametrize("prompt,count,capacity,nodes", [
    (40, 25, 64, 16), (40, 24, 64, 60), (4, 29, 32, 60), (30, 3, 32, 31)])
def test_a_text_that_fills_its_cache(monkeypatch, cfg, prompt, count, capacity, nodes):
    """Room for the prompt and all but the last token is enough, whatever is drafted: nodes lie in
    drafts, and only the accepted ones take positions."""
    m = _model(cfg, seed=2)
    ids = _ids(1, prompt, 7).to(DEV)
    monkeypatch.setitem(globals(), "_cache",
                        lambda: IPTTCDv9Cache(bits=4, capacity=capacity))
    kw = dict(temperature=0.7, top_k=8)
    u = torch.rand(count, generator=torch.Generator().manual_seed(3))
    plain, want, _ = _recorded(m, ids, count, u, kw)
    assert plain == want
    known = ids[0].tolist() + plain

    def right(text, most):  # the plain text to its end, then leaves
        tokens = known[len(text):][:nodes]
        n = nodes - len(tokens)
        return (list(range(-1, len(tokens) - 1)) + [-1] * n,
                tokens + [(text[-1] + 5 * i) % 1024 for i in range(n)])
    for draft in (_bush(1024, nodes), right):
        text, want, calls = _recorded(m, ids, count, u, kw, draft)
        assert text == want
        assert max(calls) == min(nodes + 1, capacity)


def test_accepted_nodes_need_room():
    """A tree goes through a full cache; more of its nodes than there is room for are refused
    before any is written, and fewer are taken."""
    m = _model({"window_size": None})
    cache = _cache(32)
    m.forward(_ids(1, 30, 1).to(DEV), cache=cache)
    tree = [-1] + list(range(7))
    m.forward(_ids(1, 8, 2).to(DEV), cache=cache, tree=tree)
    path = torch.arange(8, dtype=torch.int32, device=DEV)[None]
    n = torch.full((1,), 3, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="positions"):
        cache.accept(path, n)
    assert cache.seen == 30 and all(c.lengths.item() == 30 for c in cache.kv4.values())
    assert cache.accept(path, n, most=2) == 2
    assert all(c.lengths.item() == 32 for c in cache.kv4.values())
    m.forward(_ids(1, 8, 3).to(DEV), cache=cache, tree=tree)
    with pytest.raises(ValueError, match="positions"):
        cache.accept(path, n, most=1)
    assert cache.accept(path, n, most=0) == 0 and cache.seen == 32
    with pytest.raises(ValueError, match="positions"):
        m.forward(_ids(1, 1, 4).to(DEV), cache=cache)


def test_trees_over_a_window_that_its_cache_just_holds():
    """The ring wraps: trees, accepted and not, over the last window less one positions."""
    m = _model({"ttt_layers": [], "window_size": 64, "num_heads": 6}, seed=4)
    four = Drafted(capacity=64)
    held = HeldCache(four)
    ids = _ids(1, 60, 1).to(DEV)
    m.forward(ids, cache=four)
    m.forward(ids, cache=held)
    for step in range(4):
        tokens = _ids(1, len(TREE), 10 + step).to(DEV)
        got = m.forward(tokens, cache=four, tree=TREE)
        lines = ref.lineage(TREE)
        for line in lines:
            want = m.forward(tokens[:, line], logits_to_keep=1, cache=_along(held, four, line))
            _logits_close(got[:, line[-1]], want[:, 0])
        line = lines[(6, 9, 4, 8)[step]]
        path = torch.full((1, len(TREE)), -1, dtype=torch.int32, device=DEV)
        path[0, :len(line)] = torch.tensor(line)
        n = torch.tensor([len(line)], dtype=torch.int32, device=DEV)
        held = _along(held, four, line)
        m.forward(tokens[:, line], cache=held)
        assert four.accept(path, n) == len(line)
    assert four.seen > 70
    small = IPTTCDv9Cache(bits=4, capacity=32)  # less than the window: wrong as soon as it wraps
    m.forward(ids[:, :31], cache=small)
    m.forward(tokens, cache=small, tree=TREE)
    with pytest.raises(ValueError, match="positions"):
        small.accept(path, n)


def test_a_refused_accept_changes_nothing():
    """A path on another device than the layers' caches."""
    m = _model({"window_size": None})
    cache, ids = _cache(), _ids(1, 4, 0).to(DEV)
    m.forward(ids, cache=cache, tree=[-1, 0, 1, 2])
    path, n = torch.zeros(1, 4, dtype=torch.int32, device=DEV), torch.ones(1, dtype=torch.int32,
                                                                           device=DEV)
    at = {i: c.device for i, c in cache.kv4.items()}
    for c in cache.kv4.values():
        c.device = torch.device("cuda", 1)
    with pytest.raises(ValueError):
        cache.accept(path, n)
    for i, c in cache.kv4.items():
        c.device = at[i]
    m.forward(ids, cache=cache, tree=[-1, 0, 1, 2])
    assert cache.accept(path, n) == 1 and cache.seen == 1


def test_chunks_of_one_and_two_tokens_take_no_tree():
    """A TTT layer whose update chunk leaves no room for a tree: a token a call."""
    for chunk in (1, 2):
        m = _model({"ttt_chunk": chunk, "ttt_visible_chunks": 64})
        ids = _ids(1, 6, 1).to(DEV)
        plain = m.generate(ids, 5, temperature=0)
        assert torch.equal(plain, m.generate(ids, 5, temperature=0,
                                             draft=lambda t, n: ([-1, 0], [1, 2])))


def test_a_refused_call_sets_no_shape():
    """A batch of two, refused before its first layer, and then the one sequence that goes."""
    m = _model({"window_size": None})
    cache, ids = _cache(), _ids(1, 4, 0).to(DEV)
    with pytest.raises(NotImplementedError, match="one sequence"):
        m.forward(ids.expand(2, 4), cache=cache, tree=[-1, 0, 1, 2])
    m.forward(ids, cache=cache, tree=[-1, 0, 1, 2])
    with pytest.raises(ValueError, match="cache holds"):
        m.forward(ids.expand(2, 4), cache=cache)


def test_generate_refuses_what_is_no_cache():
    m = _model({"window_size": None})
    with pytest.raises(ValueError, match="IPTTCDv9Cache"):
        m.generate(_ids(1, 4, 0).to(DEV), 3, temperature=0, cache={})

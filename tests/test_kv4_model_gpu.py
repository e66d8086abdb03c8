"""An ipttcdv9 prefill and decode over the 4-bit cache on the GPU. The comparator is
the same model over a bf16 cache whose new keys and values are replaced by what the
4-bit one read back for them, so both attend over the same numbers, one with the
prefill kernels.

(Replaced by what 4 bits hold of its own, it would not: its values of the second
layer on differ by d = a bf16 rounding, 2^-8 of them, from the first run's, and where
one lies within d of a border between codes, a share d / step of them, the code is
another, a step of a third of the value: sqrt(d step) = 3 % of it by root mean
square, ten times d.)"""
from __future__ import annotations

import pytest
import torch

from oracle import kv4_ref
from test_ipttcdv9_gpu import TINY, _ids, _logits_close
from ttcd_amd import ipttcdv9 as M, kv4

pytestmark = pytest.mark.gpu
DEV = "cuda"


class FourBits(M.IPTTCDv9Cache):
    """The 4-bit cache; `last` holds what it read back of each layer's newest rows."""

    def __init__(self, **kw):
        super().__init__(bits=4, **kw)
        self.last = {}

    def append(self, layer, k, v):
        held = super().append(layer, k, v)
        self.last[layer] = kv4.kv4_read(held, k.shape[1])
        return held


class HeldCache(M.IPTTCDv9Cache):
    """The bf16 cache of the values that the 4-bit cache `four` holds, a call behind it."""

    def __init__(self, four):
        super().__init__()
        self.four = four

    def extend(self, layer, k, v, keep):
        got = self.four.last[layer]
        for x, y in zip((k, v), got):  # a code apart, a scale apart at most
            assert ((x - y).abs().amax() <= 0.4 * x.abs().amax())
        return super().extend(layer, *got, keep)

    def take(self, layer, index):
        """Keep the rows of index (B, Hkv, n), per head."""
        at = index.long().transpose(1, 2)[..., None]
        self.kv[layer] = tuple(x.gather(1, at.expand(-1, -1, -1, x.shape[-1]).to(x.device))
                               for x in self.kv[layer])


@pytest.mark.parametrize("cfg,chunks", [
    ({}, (300, 700, 256, 1, 1)), ({"window_size": None}, (256, 1, 300, 2, 1)),
    ({"ttt_layers": [], "window_size": 64}, (40, 1, 1, 90, 200, 1))])
def test_chunks_and_tokens_over_4_bits(cfg, chunks):
    cfg = dict(TINY, **cfg)
    w = M.init_weights(cfg, DEV, seed=9)
    T = sum(chunks)
    ids = _ids(2, T, seed=T).to(DEV)
    window = cfg["window_size"]
    room = T if window is None else window + max(chunks) - 1
    for path in M.PATHS:
        model = M.IPTTCDv9Prefill(cfg, w, path=path)
        cache = FourBits(capacity=room)
        same = HeldCache(cache)
        a = 0
        for n in chunks:
            print(f"path {path}: {a}..{a + n}", flush=True)
            got = model.forward(ids[:, a:a + n], logits_to_keep=8, cache=cache)
            want = model.forward(ids[:, a:a + n], logits_to_keep=8, cache=same)
            _logits_close(got, want)
            a += n
            assert cache.seen == a
            assert cache.kv4[0].lengths.tolist() == [a, a]


def test_the_cut_of_a_prompt_does_not_matter():
    """Every row attends over 4-bit keys, its own chunk's among them: one call and many
    give the same rows (without the TTT MLP, which restarts at every call), but for the
    codes that another rounding of a layer's input tips: 3 % of a value by the
    arithmetic above, in each of the layers behind the first, whose noise adds up as
    squares: 3 % sqrt(2) at the mean for the two."""
    cfg = dict(TINY, ttt_layers=[])
    model = M.IPTTCDv9Prefill(cfg, M.init_weights(cfg, DEV, seed=10))
    ids = _ids(1, 700, seed=11).to(DEV)
    whole = model.forward(ids, logits_to_keep=0, cache=M.IPTTCDv9Cache(bits=4, capacity=700))
    cache, a = M.IPTTCDv9Cache(bits=4, capacity=1011), 0
    for n in (450, 50, 1, 1, 198):
        part = model.forward(ids[:, a:a + n], logits_to_keep=0, cache=cache)
        _logits_close(part, whole[:, a:a + n], max_frac=6e-2, mean_frac=4.3e-2)
        a += n


@pytest.mark.parametrize("ttt_layers", [[], [0]])
def test_keys_of_least_weight_are_dropped(monkeypatch, ttt_layers):
    """Full-causal layers cut to 120 keys a head: the dropped ones are the lightest of
    what the layers' attention summed up, and later calls attend over the rest."""
    cfg = dict(TINY, ttt_layers=ttt_layers, window_size=None)
    model = M.IPTTCDv9Prefill(cfg, M.init_weights(cfg, DEV, seed=12))
    ids = _ids(2, 420, seed=13).to(DEV)
    taken = []

    def evict(old, weights, keep, recent, out):
        n = int(old.lengths[0])
        w = old.weights.clone()
        got = real(old, weights, keep, recent, out=out)
        taken.append((w, n, got[1]))
        return got

    real = kv4.kv4_evict
    monkeypatch.setattr(kv4, "kv4_evict", evict)
    cache = FourBits(capacity=420, keep=120, recent=30)
    same = HeldCache(cache)
    a, rows = 0, 0
    for n in (260, 1, 1, 100, 1):
        before = cache.held
        got = model.forward(ids[:, a:a + n], logits_to_keep=4, cache=cache)
        want = model.forward(ids[:, a:a + n], logits_to_keep=4, cache=same)
        _logits_close(got, want)
        a += n
        rows += n
        assert (cache.seen, cache.held) == (a, min(before + n, 120))
        if before + n <= 120:
            assert not taken
            continue
        G = model.Hq // model.Hkv
        for i, (w, held, index) in enumerate(taken):
            assert held == before + n
            # every query's weights are in the sums once, less what was dropped with its keys
            total = w[..., :held].sum(-1)
            assert (total <= rows * G * 1.001).all() and (total >= n * G * 0.999).all()
            ref = kv4_ref.Ref(2, model.Hkv, model.D, cache.capacity)
            ref.rows = [(torch.zeros(held, 1, 1),) * 2] * 2
            assert torch.equal(index.cpu(), ref.evict(w.cpu(), 120, 30)[0])
            same.take(i, index)
        assert len(taken) == cfg["num_hidden_layers"]
        taken.clear()


def test_refusals():
    model = M.IPTTCDv9Prefill(TINY, M.init_weights(TINY, DEV, seed=9))
    ids = _ids(1, 64, seed=1).to(DEV)
    cache = M.IPTTCDv9Cache(bits=4, capacity=64)
    model.forward(ids, cache=cache)
    with pytest.raises(ValueError, match="positions"):
        model.forward(ids[:, :1], cache=cache)
    with pytest.raises(NotImplementedError, match="window"):
        model.forward(ids, cache=M.IPTTCDv9Cache(bits=4, capacity=64, keep=8))
    mask = torch.ones(1, 64, device=DEV)
    mask[0, 0] = 0
    with pytest.raises(NotImplementedError, match="mask"):
        model.forward(ids, cache=M.IPTTCDv9Cache(bits=4, capacity=64), attention_mask=mask)


def _student_rows(monkeypatch, model, ids, chunks, cache):
    """What the student of TTT layer 0 gives in each of the calls."""
    rows, real = [], kv4.kv4_attn

    def attn(q, held, window=None, **kw):
        out = real(q, held, window, **kw)
        if window == model.window_s:
            rows.append(out)
        return out

    monkeypatch.setattr(kv4, "kv4_attn", attn)
    a = 0
    for n in chunks:
        model.forward(ids[:, a:a + n], cache=cache)
        a += n
    monkeypatch.setattr(kv4, "kv4_attn", real)
    return rows


@pytest.mark.parametrize("path", M.PATHS)
def test_the_student_sees_positions_of_its_window_after_an_eviction(monkeypatch, path):
    """Layer 0's queries, keys and values do not depend on attention, so its student over a
    cache that dropped keys has to give what it gives over one that holds all of them, but
    for the order of its sums: a rounding of the probabilities and of the result each, off
    by half a step of 2^-8 on either side, of values of at most max |v|."""
    cfg = dict(TINY, ttt_layers=[0], window_size=None)
    model = M.IPTTCDv9Prefill(cfg, M.init_weights(cfg, DEV, seed=14), path=path)
    span, chunks = model.window_s, (400, 1, 300)
    ids = _ids(1, sum(chunks), seed=15).to(DEV)
    whole = FourBits(capacity=sum(chunks))
    want = _student_rows(monkeypatch, model, ids, chunks, whole)
    cut = FourBits(capacity=sum(chunks), keep=span + 30, recent=span - 1)
    got = _student_rows(monkeypatch, model, ids, chunks, cut)
    assert cut.kv4[0].lengths.tolist() == [span + 30]
    assert [x.shape[1] for x in got] == [400, 300] and len(want) == 2
    top = max(kv4.kv4_read(whole.kv4[0], sum(chunks))[1].abs().max().item(), 1e-6)
    for x, y in zip(got, want):
        assert (x.float() - y.float()).abs().max().item() <= 4 * 2.0 ** -8 * top
    short = FourBits(capacity=sum(chunks), keep=span + 30, recent=span - 2)
    for a, n in ((0, 400), (400, 1)):
        model.forward(ids[:, a:a + n], cache=short)
    held = [c.lengths.tolist() for c in short.kv4.values()]
    with pytest.raises(NotImplementedError, match="student"):
        model.forward(ids[:, 401:], cache=short)
    assert short.seen == 401 and [c.lengths.tolist() for c in short.kv4.values()] == held
    model.forward(ids[:, 401:410], cache=short)  # fewer than a chunk: no student


def test_a_student_window_wider_than_the_teachers_needs_its_room(monkeypatch):
    """With too small a ring the call is refused before it writes. With room, the student
    of layer 0 gives what it gives in one call, but for four half steps as above."""
    cfg = dict(TINY, ttt_layers=[0], window_size=64)  # student window 256
    model = M.IPTTCDv9Prefill(cfg, M.init_weights(cfg, DEV, seed=16), path="stock")
    ids = _ids(1, 768, seed=17).to(DEV)
    cache = M.IPTTCDv9Cache(bits=4, capacity=64 + 256)
    model.forward(ids[:, :256], cache=cache)
    with pytest.raises(ValueError, match="positions"):
        model.forward(ids[:, 256:512], cache=cache)
    assert cache.seen == 256 and cache.kv4[0].lengths.tolist() == [256]
    whole = FourBits(capacity=768)
    want = _student_rows(monkeypatch, model, ids, (768,), whole)[0]
    got = _student_rows(monkeypatch, model, ids, (256,) * 3, FourBits(capacity=511))
    top = max(kv4.kv4_read(whole.kv4[0], 768)[1].abs().max().item(), 1e-6)
    d = (torch.cat(got, 1).float() - want.float()).abs().max().item()
    assert d <= 4 * 2.0 ** -8 * top


def test_a_call_that_raised_between_layers_leaves_no_usable_cache(monkeypatch):
    model = M.IPTTCDv9Prefill(TINY, M.init_weights(TINY, DEV, seed=9))
    ids = _ids(1, 40, seed=1).to(DEV)
    cache = M.IPTTCDv9Cache(bits=4, capacity=128)
    model.forward(ids[:, :20], cache=cache)
    real = M.IPTTCDv9Prefill.layer

    def layer(self, i, *a):
        if i == 1:
            raise MemoryError
        return real(self, i, *a)

    monkeypatch.setattr(M.IPTTCDv9Prefill, "layer", layer)
    with pytest.raises(MemoryError):
        model.forward(ids[:, 20:], cache=cache)
    monkeypatch.setattr(M.IPTTCDv9Prefill, "layer", real)
    with pytest.raises(RuntimeError, match="did not end"):
        model.forward(ids[:, 20:], cache=cache)

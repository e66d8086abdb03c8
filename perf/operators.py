"""The operators of a key / value cache held in 4 bits, as cases that can be timed and compared.

The cache holds values in blocks of 32 channels that share a power of two (2^e, stored as the byte
e + 127), each value as a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6. Position p of a sequence is in
slot p % C of its C slots; `lengths` counts the positions that a sequence has had, the last C of
which are held. Tensors of a cache of B sequences, H key / value heads and D channels:

  k_codes   uint8 (B, H, C, D/2)         channel 2i in the low half of byte i, 2i + 1 in the high one
  k_scales  uint8 (B, H, C, D/32)
  v_codes   uint8 (B, H, C/4, D/8, 4, 4) words of 8 channels, those of 4 slots side by side
  v_scales  uint8 (B, H, C/4, D/32, 4)
  lengths   int32 (B)

Kinds
  append   new keys and values are quantised into the cache and read back
  attn     attention of the newest positions over the cache, a causal window of it
  weights  the attention weight that each held key gets, summed over the queries of its head
  evict    the cache without the keys of least weight, read back

`counts`, where a case has them: a padded batch, sequence b has counts[b] of the T new positions.
Queries are the last positions of their sequence. A window of -1 is none. Sizes are those of the
repository's model configurations, tests and benchmark.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
# the exponents that keep every held value a normal number of the type (f16: any number)
E_RANGE = {"bf16": (-125, 125), "f16": (-23, 13)}


def listed():
    return [
        # a decode step's new token for a batch of 32 sequences, Qwen3-0.6B heads
        _append("append-token", B=32, T=1, Hkv=8, D=128, cap=4096, length=4000, ragged=True),
        # a chunk of a long prompt
        _append("append-chunk", B=1, T=4096, Hkv=8, D=128, cap=12288, length=20000),
        # a padded batch of prompts of odd lengths, SmolLM2 heads, fp16
        _append("append-padded-f16", B=3, T=1777, Hkv=5, D=64, cap=8192, length=3000, ragged=True,
                counts=True, dtype="f16"),
        # one token of a short conversation on the smallest heads: launch and host latency
        _attn("attn", "attn-token-short", B=1, T=1, Hq=4, Hkv=2, D=64, cap=512, length=257),
        # one token each for 32 sequences of mixed length, no window
        _attn("attn", "attn-token-batch", B=32, T=1, Hq=16, Hkv=8, D=128, cap=16384, length=16384,
              ragged=True),
        # one token over a 64K cache, fp16, three query heads per key / value head
        _attn("attn", "attn-token-64k-f16", B=2, T=1, Hq=15, Hkv=5, D=64, cap=65536, length=65001,
              dtype="f16"),
        # a follow-up prompt of 300 tokens onto a full 8192-token window, the ring wrapped
        _attn("attn", "attn-follow-up", B=1, T=300, Hq=16, Hkv=8, D=128, cap=12288, length=40001,
              window=8192, lse=True),
        # a chunk of 4096 tokens of a long prompt onto a full 8192-token window
        _attn("attn", "attn-chunk", B=1, T=4096, Hq=16, Hkv=8, D=128, cap=12288, length=32768,
              window=8192),
        # the weights of a decode step's keys, a batch of 8
        _attn("weights", "weights-token", B=8, T=1, Hq=16, Hkv=8, D=128, cap=16384, length=16000,
              ragged=True),
        # the weights under the last 512 positions of a prompt
        _attn("weights", "weights-chunk", B=1, T=512, Hq=16, Hkv=8, D=128, cap=16384,
              length=16384),
        # a small cache cut to a quarter
        _evict("evict-short", B=1, Hkv=2, D=64, cap=1024, length=1001, keep=256, recent=32),
        # a full 32K cache cut to half, the newest 1024 kept in any case
        _evict("evict-32k", B=2, Hkv=8, D=128, cap=32768, length=32768, keep=16384, recent=1024),
    ]


def _append(name, *, B, T, Hkv, D, cap, length, ragged=False, counts=False, dtype="bf16"):
    case = dict(kind="append", B=B, T=T, Hkv=Hkv, D=D, cap=cap, length=length, ragged=ragged,
                counts=counts, dtype=dtype)
    return case if name is None else dict(case, name=name)


def _attn(kind, name, *, B, T, Hq, Hkv, D, cap, length, window=-1, ragged=False, counts=False,
          lse=False, dtype="bf16"):
    case = dict(kind=kind, B=B, T=T, Hq=Hq, Hkv=Hkv, D=D, cap=cap, length=length, window=window,
                ragged=ragged, counts=counts, lse=lse, dtype=dtype)
    return case if name is None else dict(case, name=name)


def _evict(name, *, B, Hkv, D, cap, length, keep, recent, ragged=False, dtype="bf16"):
    case = dict(kind="evict", B=B, Hkv=Hkv, D=D, cap=cap, length=length, keep=keep, recent=recent,
                ragged=ragged, dtype=dtype)
    return case if name is None else dict(case, name=name)


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(("append", "attn", "attn", "attn", "weights", "evict"))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    Hq, Hkv, D = rng.choice(((16, 8, 128), (16, 8, 128), (15, 5, 64), (4, 2, 64), (8, 2, 128),
                             (4, 4, 128), (9, 3, 64)))
    B = rng.choice((1, 1, 2, 3, 8, 24))
    cap = 32 * _log_int(rng, 2, 2048 // B)
    # at the start of a sequence, up to a full cache, or past it
    length = rng.choice((_log_int(rng, 1, cap), _log_int(rng, 1, cap), cap,
                         cap + _log_int(rng, 1, 3 * cap)))
    ragged = B > 1 and rng.random() < 0.6
    counts = B > 1 and rng.random() < 0.4
    if kind == "append":
        return _append(None, B=B, T=rng.choice((1, _log_int(rng, 1, min(cap, 8192 // B)))),
                       Hkv=Hkv, D=D, cap=cap, length=length, ragged=ragged, counts=counts,
                       dtype=dtype)
    if kind == "evict":
        keep = _log_int(rng, 1, min(cap, 16384))
        return _evict(None, B=min(B, 3), Hkv=Hkv, D=D, cap=cap, length=length, keep=keep,
                      recent=rng.choice((0, keep, _log_int(rng, 1, keep))), ragged=ragged,
                      dtype=dtype)
    window = rng.choice((-1, -1, 8192, 2048, 512, _log_int(rng, 1, cap)))
    top = min(cap, length, 4096 * 12288 * 16 // (B * Hq * cap))
    T = rng.choice((1, 1, _log_int(rng, 1, min(64, top)), _log_int(rng, 1, min(4096, top))))
    return _attn(kind, None, B=B, T=T, Hq=Hq, Hkv=Hkv, D=D, cap=cap, length=length, window=window,
                 ragged=ragged, counts=counts, lse=kind == "attn" and rng.random() < 0.5,
                 dtype=dtype)


def _counts(case):
    """The new positions of each sequence: all T, or T down to none."""
    B, T = case["B"], case["T"]
    return [T - T * b // max(1, B - 1) if case["counts"] else T for b in range(B)]


def _lengths(case):
    """The positions that each sequence has had before the call; for a query, its own among them."""
    B, n = case["B"], case["length"]
    out = [max(1, n - (n - 1) * b // B) if case["ragged"] else n for b in range(B)]
    if case["kind"] in ("attn", "weights"):
        out = [max(a, c) for a, c in zip(out, _counts(case))]
    return out


# ------------------------------------------------------------------- inputs

def _quantise(x, dtype):
    """Codes (one a byte) and scale bytes of x (..., D), in blocks of 32 channels: the least 2^e with
    no value over 6 2^e, then the nearest of the 4-bit values, ties to the even code."""
    lo, hi = E_RANGE[dtype]
    y = x.float().unflatten(-1, (-1, 32))
    top = y.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(top)  # top = m 2^e, m in [0.5, 1); 6 2^e' = 0.75 2^(e' + 3)
    e = torch.where(top > 0, torch.where(m <= 0.75, e - 3, e - 2), lo).clamp(lo, hi)
    y = torch.ldexp(y, -e)
    a = y.abs()
    code = torch.zeros_like(a, dtype=torch.uint8)
    code += (a > 0.25).to(torch.uint8)
    code += (a >= 0.75).to(torch.uint8)
    code += (a > 1.25).to(torch.uint8)
    code += (a >= 1.75).to(torch.uint8)
    code += (a > 2.5).to(torch.uint8)
    code += (a >= 3.5).to(torch.uint8)
    code += (a > 5).to(torch.uint8)
    code += torch.signbit(y).to(torch.uint8) * 8
    return code.flatten(-2), (e.squeeze(-1) + 127).to(torch.uint8)


def _pack(code):
    return code[..., ::2] + 16 * code[..., 1::2]


def _interleave(x):
    """(B, H, C, n, ...) -> (B, H, C/4, n, 4, ...): the rows of 4 slots side by side."""
    return x.unflatten(2, (-1, 4)).transpose(3, 4)


def _filled(case, g):
    """A cache whose slots all hold something, as after earlier sequences."""
    B, H, C, D = case["B"], case["Hkv"], case["cap"], case["D"]
    x = _keys(g, B, H, C, D)
    kc, ks = _quantise(x, case["dtype"])
    x = torch.randn(B, H, C, D, generator=g, device=DEV)
    vc, vs = _quantise(x, case["dtype"])
    return dict(k_codes=_pack(kc), k_scales=ks,
                v_codes=_interleave(_pack(vc).unflatten(-1, (-1, 4))).contiguous(),
                v_scales=_interleave(vs).contiguous(),
                lengths=torch.tensor(_lengths(case), dtype=torch.int32, device=DEV))


def _keys(g, *shape):
    """Keys have a few channels of larger values, as after rotary embedding."""
    x = torch.randn(*shape, generator=g, device=DEV)
    x[..., ::19] *= 3
    return x


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    B, D, dt = case["B"], case["D"], DTYPES[case["dtype"]]
    s = dict(case=case, cache=_filled(case, g), counts=None)
    if case.get("counts"):
        s["counts"] = torch.tensor(_counts(case), dtype=torch.int32, device=DEV)
    if case["kind"] == "append":
        shape = (B, case["T"], case["Hkv"], D)
        s["k"] = _keys(g, *shape).to(dt)
        s["v"] = torch.randn(*shape, generator=g, device=DEV).to(dt)
    elif case["kind"] == "evict":
        # sums of attention weights: most are small, some keys never got any
        w = torch.rand(B, case["Hkv"], case["cap"], generator=g, device=DEV)
        s["weights"] = torch.where(w < 0.05, 0.0, w.log().square())
    else:
        s["q"] = torch.randn(B, case["T"], case["Hq"], D, generator=g, device=DEV).to(dt)
        if case["kind"] == "weights":
            s["lse"] = _scores(s)[1]
    return s


# ---------------------------------------------------------------- plain form

def _values(codes, scales, dtype=torch.float32):
    """What packed codes (..., D/2) and scales (..., D/32) stand for, in float32."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6],
                        dtype=dtype, device=codes.device)
    x = torch.stack((grid[(codes & 15).int()], grid[(codes >> 4).int()]), -1).flatten(-2)
    return torch.ldexp(x.unflatten(-1, (-1, 32)), scales.int().unsqueeze(-1) - 127).flatten(-2)


def _k_values(c):
    return _values(c["k_codes"], c["k_scales"])


def _v_values(c):
    codes = c["v_codes"].transpose(3, 4).flatten(2, 3).flatten(3)
    return _values(codes, c["v_scales"].transpose(3, 4).flatten(2, 3))


def _positions(c):
    """The position that each slot holds (B, C), negative where it holds none."""
    C, n = c["k_codes"].shape[2], c["lengths"].long()[:, None]
    return n - 1 - (n - 1 - torch.arange(C, device=DEV)) % C


def _new_rows(s):
    """(B, T): the position of each new row (after an append: lengths count them), and whether the
    sequence has it."""
    case, c = s["case"], s["cache"]
    t = torch.arange(case["T"], device=DEV)
    n = s["counts"].long()[:, None] if s["counts"] is not None else case["T"]
    return c["lengths"].long()[:, None] - n + t, (t < n).expand(case["B"], -1)


def _scores(s):
    """Masked scores (B, Hkv, G, T, C) in float32, natural, and their log-sum-exp (B, Hq, T)."""
    case, c, q = s["case"], s["cache"], s["q"]
    B, T, Hq, D = q.shape
    H, W = case["Hkv"], case["window"]
    qg = q.float().transpose(1, 2).reshape(B, H, Hq // H * T, D)
    x = (qg @ _k_values(c).transpose(2, 3)).mul_(D ** -0.5).view(B, H, Hq // H, T, -1)
    at, there = _new_rows(s)
    p = _positions(c)[:, None]
    hidden = (p < 0) | (p > at[..., None]) | ~there[..., None]
    if W > 0:
        hidden |= p <= at[..., None] - W
    x.masked_fill_(hidden[:, None, None], -math.inf)
    return x, x.logsumexp(-1).view(B, Hq, T)


def _plain_append(s):
    case, c = s["case"], s["cache"]
    B, T, H, D = s["k"].shape
    n = s["counts"].long()[:, None] if s["counts"] is not None else torch.full((B, 1), T, device=DEV)
    t = torch.arange(T, device=DEV)
    slot = (c["lengths"].long()[:, None] + t) % case["cap"]
    b, t = (t < n).nonzero(as_tuple=True)
    slot = slot[b, t]
    kc, ks = _quantise(s["k"][b, t], case["dtype"])  # (rows, H, D)
    vc, vs = _quantise(s["v"][b, t], case["dtype"])
    c["k_codes"][b, :, slot] = _pack(kc)
    c["k_scales"][b, :, slot] = ks
    c["v_codes"][b, :, slot // 4, :, slot % 4] = _pack(vc).unflatten(-1, (-1, 4))
    c["v_scales"][b, :, slot // 4, :, slot % 4] = vs
    c["lengths"] += n.flatten().int()
    return _plain_read(c, T, case["dtype"])


def _plain_read(c, count, dtype):
    """The last `count` positions of each sequence (B, count, H, D), zeros where it has none."""
    B, C = c["lengths"].shape[0], c["k_codes"].shape[2]
    n = c["lengths"].long()[:, None]
    p = n - count + torch.arange(count, device=DEV)
    none = ((p < 0) | (p < n - C))[:, :, None, None]
    b, slot = torch.arange(B, device=DEV)[:, None], p % C
    k = _values(c["k_codes"][b, :, slot], c["k_scales"][b, :, slot])
    v = _values(c["v_codes"][b, :, slot // 4, :, slot % 4].flatten(3),
                c["v_scales"][b, :, slot // 4, :, slot % 4])
    return tuple(x.masked_fill_(none, 0).to(DTYPES[dtype]) for x in (k, v))


def _plain_attn(s):
    case = s["case"]
    x, lse = _scores(s)
    B, H, G, T, C = x.shape
    top = x.amax(-1, keepdim=True)
    p = x.sub_(top.masked_fill(top == -math.inf, 0)).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp_min_(1e-30)).view(B, H, G * T, C)
    held = (_positions(s["cache"]) >= 0)[:, None, :, None]
    o = p @ _v_values(s["cache"]).masked_fill_(~held, 0)
    o = o.view(B, H * G, T, -1).transpose(1, 2).to(DTYPES[case["dtype"]])
    return (o, lse) if case["lse"] else o


def _plain_weights(s):
    x, _ = _scores(s)
    B, H, G, T, C = x.shape
    lse = s["lse"].view(B, H, G, T, 1)
    return x.sub_(lse.masked_fill(lse == -math.inf, 0)).exp_().sum((2, 3))


def _plain_evict(s):
    case, c = s["case"], s["cache"]
    B, H, C, _ = c["k_codes"].shape
    keep, recent = case["keep"], min(case["recent"], case["keep"])
    n = c["lengths"].long().clamp(max=C)[:, None]  # held
    first = c["lengths"].long()[:, None] - n
    j = torch.arange(C, device=DEV)
    slot = (first + j) % C  # of the j-th oldest held position
    w = s["weights"].gather(2, slot[:, None].expand(B, H, C))
    # the newest before all, then by weight, what is not held last; ties to the lowest position
    newest = ((j >= n - recent) & (j < n))[:, None]
    key = torch.where(newest, math.inf, w).masked_fill_((j >= n)[:, None], -math.inf)
    order = key.sort(dim=-1, descending=True, stable=True).indices
    m = n.clamp(max=keep)[:, None]  # kept
    rank = torch.arange(keep, device=DEV)
    chosen = order[..., :keep].masked_fill(rank >= m, C).sort(-1).values  # by position, none last
    none = chosen == C
    at = chosen.masked_fill(none, 0)
    index = (at + first[:, None]).masked_fill(none, -1).int()
    weights = torch.zeros_like(s["weights"])
    weights[..., :keep] = w.gather(2, at).masked_fill(none, 0)
    # the new cache: kept rows in slots 0.., then read back
    s_at = slot[:, None].expand(B, H, C).gather(2, at)
    b, h = torch.arange(B, device=DEV)[:, None, None], torch.arange(H, device=DEV)[:, None]
    new = dict(
        k_codes=torch.zeros_like(c["k_codes"]), k_scales=torch.zeros_like(c["k_scales"]),
        v_codes=torch.zeros_like(c["v_codes"]), v_scales=torch.zeros_like(c["v_scales"]),
        lengths=m.flatten().int())
    new["k_codes"][:, :, :keep] = c["k_codes"][b, h, s_at]
    new["k_scales"][:, :, :keep] = c["k_scales"][b, h, s_at]
    new["v_codes"][:, :, rank // 4, :, rank % 4] = (
        c["v_codes"][b, h, s_at // 4, :, s_at % 4].permute(2, 0, 1, 3, 4))
    new["v_scales"][:, :, rank // 4, :, rank % 4] = (
        c["v_scales"][b, h, s_at // 4, :, s_at % 4].permute(2, 0, 1, 3))
    return _plain_read(new, keep, case["dtype"]) + (index, weights)


# ----------------------------------------------------------------------- run

def run(s):
    case = s["case"]
    if own:
        return _own(s, case)
    return {"append": _plain_append, "attn": _plain_attn, "weights": _plain_weights,
            "evict": _plain_evict}[case["kind"]](s)


def _own(s, case):
    import ttcd_amd
    c = s["cache"]
    cache = ttcd_amd.KV4Cache.from_parts(c["k_codes"], c["k_scales"], c["v_codes"], c["v_scales"],
                                         c["lengths"], DTYPES[case["dtype"]])
    window = case.get("window")
    if case["kind"] == "append":
        ttcd_amd.kv4_append(cache, s["k"], s["v"], counts=s["counts"])
        return ttcd_amd.kv4_read(cache, case["T"])
    if case["kind"] == "attn":
        return ttcd_amd.kv4_attn(s["q"], cache, window, counts=s["counts"], return_lse=case["lse"])
    if case["kind"] == "weights":
        return ttcd_amd.kv4_key_weights(s["q"], cache, s["lse"], window, counts=s["counts"])
    new, index, weights = ttcd_amd.kv4_evict(cache, s["weights"], case["keep"], case["recent"])
    return ttcd_amd.kv4_read(new, case["keep"]) + (index, weights)


def work(case):
    B, H, D, C = case["B"], case["Hkv"], case["D"], case["cap"]
    row = D // 2 + D // 32  # bytes of one key or value in the cache
    if case["kind"] == "append":
        # read k and v, write their codes; read them again, write the values
        new = sum(_counts(case)) * H
        return {"bytes": 2 * (new * (2 * D + row) + B * case["T"] * H * (row + 2 * D)), "flops": 0}
    if case["kind"] == "evict":
        held = sum(min(n, C) for n in _lengths(case)) * H
        kept = sum(min(n, C, case["keep"]) for n in _lengths(case)) * H
        # weights and kept rows read, rows, index and weights written, rows read again, values written
        return {"bytes": 4 * held + 3 * 2 * kept * row + B * H * case["keep"] * (4 + 4 * D)
                + 4 * B * H * C, "flops": 0}
    Hq, W = case["Hq"], case["window"]
    keys = pairs = 0
    for n, c in zip(_lengths(case), _counts(case)):
        held = max(0, n - C)
        first = [max(held, p - W + 1 if W > 0 else 0) for p in range(n - c, n)]
        pairs += sum(max(0, p + 1 - f) for p, f in zip(range(n - c, n), first))
        keys += n - min(first) if first else 0
    rows = sum(_counts(case)) * Hq
    if case["kind"] == "weights":
        return {"bytes": keys * H * row + rows * (2 * D + 4) + 4 * B * H * C,
                "flops": 2 * Hq * D * pairs}
    return {"bytes": 2 * keys * H * row + rows * 4 * D + (4 * rows if case["lse"] else 0),
            "flops": 4 * Hq * D * pairs}


# --------------------------------------------------------------------- exact

def _exact_values(codes, scales):
    """float64 values of one code a byte (..., D), from the sign, exponent and fraction bits."""
    c = codes.to(torch.int64)
    frac, exp = (c & 1).double(), (c >> 1) & 3
    mag = torch.where(exp == 0, 0.5 * frac, (1 + 0.5 * frac) * torch.exp2((exp - 1).double()))
    sign = 1.0 - 2.0 * (c >> 3).double()
    scale = torch.exp2(scales.double() - 127).repeat_interleave(32, -1)
    return sign * mag * scale


def _exact_rows(c, b, h, slots):
    """Keys and values (len(slots), D) of head h of sequence b, in float64."""
    out = []
    for codes, scales in ((c["k_codes"][b, h, slots], c["k_scales"][b, h, slots]),
                          (c["v_codes"][b, h, slots // 4, :, slots % 4].flatten(1),
                           c["v_scales"][b, h, slots // 4, :, slots % 4])):
        both = torch.stack((codes % 16, codes // 16), -1).flatten(1)
        out.append(_exact_values(both, scales))
    return out


def _exact_round(x, dtype):
    """x (..., D) as the cache holds it, in float64."""
    lo, hi = E_RANGE[dtype]
    y = x.double().unflatten(-1, (-1, 32))
    m, e = torch.frexp(y.abs().amax(-1, keepdim=True) / 1.5)  # the least 2^(e + 2) over it
    e = (torch.where(m > 0.5, e, e - 1) - 2).masked_fill(m == 0, lo).clamp(lo, hi)
    y = y / torch.exp2(e.double())
    step = torch.exp2(torch.frexp(y.abs())[1].clamp(1, 3).double() - 2)
    y = ((y / step).round() * step).clamp(-6, 6)
    return (y * torch.exp2(e.double())).flatten(-2)


def _exact_tail(s, count, keys):
    """The last `count` rows (B, count, H, D) of what keys(b) gives: (n, H, D) rows of k and of v."""
    case = s["case"]
    out = [torch.zeros(case["B"], count, case["Hkv"], case["D"], dtype=torch.float64, device=DEV)
           for _ in range(2)]
    for b in range(case["B"]):
        for o, x in zip(out, keys(b)):
            n = min(count, x.shape[0])
            o[b, count - n:] = x[x.shape[0] - n:]
    return out


def _held(case, n):
    return torch.arange(max(0, n - case["cap"]), n, device=DEV)


def exact(case, seed):
    s = prepare(case, seed)
    c, C, H = s["cache"], case["cap"], case["Hkv"]
    lengths = _lengths(case)
    if case["kind"] == "append":
        counts = _counts(case)

        def keys(b):
            # of the rows held before, the oldest are overwritten by what is appended
            p = _held(case, lengths[b])
            old = [_exact_rows(c, b, h, p % C) for h in range(H)]
            for i, x in enumerate((s["k"], s["v"])):
                rows = torch.stack([o[i] for o in old], 1)
                yield torch.cat((rows, _exact_round(x[b, :counts[b]], case["dtype"])))[-C:]
        return tuple(_exact_tail(s, case["T"], keys))
    if case["kind"] == "evict":
        keep = case["keep"]
        index = torch.full((case["B"], H, keep), -1, dtype=torch.int32, device=DEV)
        weights = torch.zeros(case["B"], H, C, device=DEV)
        rows = {}
        for b in range(case["B"]):
            p = _held(case, lengths[b])
            n, got = len(p), []
            for h in range(H):
                w = s["weights"][b, h, p % C]
                must = min(n, keep, case["recent"])
                # 64-bit keys: the weight's bits (none is negative), then the oldest first
                key = (w.view(torch.int32).long() << 32) + (n - torch.arange(n, device=DEV))
                key[n - must:] = 2 ** 63 - 1
                kept = key.argsort(descending=True)[:min(n, keep)].sort().values
                index[b, h, :len(kept)] = p[kept].int()
                weights[b, h, :len(kept)] = w[kept]
                got.append(_exact_rows(c, b, h, p[kept] % C))
            rows[b] = [torch.stack([g[i] for g in got], 1) for i in range(2)]
        return tuple(_exact_tail(s, keep, rows.__getitem__)) + (index, weights)
    B, T, Hq, D, W = case["B"], case["T"], case["Hq"], case["D"], case["window"]
    G = Hq // H
    o = torch.zeros(B, T, Hq, D, dtype=torch.float64, device=DEV)
    lse = torch.full((B, Hq, T), -math.inf, dtype=torch.float64, device=DEV)
    weights = torch.zeros(B, H, C, dtype=torch.float64, device=DEV)
    for b, (n, new) in enumerate(zip(lengths, _counts(case))):
        if not new:
            continue
        p = _held(case, n)
        at = torch.arange(n - new, n, device=DEV)[:, None]
        seen = (p <= at) & (p > at - (W if W > 0 else n + 1))
        for h in range(H):
            k, v = _exact_rows(c, b, h, p % C)
            for g in range(h * G, h * G + G):
                x = (s["q"][b, :new, g].double() @ k.T * D ** -0.5).masked_fill(~seen, -math.inf)
                if case["kind"] == "weights":
                    weights[b, h, p % C] += torch.exp(x - s["lse"][b, g, :new, None].double()).sum(0)
                    continue
                lse[b, g, :new] = x.logsumexp(-1)
                o[b, :new, g] = torch.exp(x - lse[b, g, :new, None]) @ v
    if case["kind"] == "weights":
        return weights
    return (o, lse) if case["lse"] else o

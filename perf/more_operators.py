"""The operators of a step that verifies drafted tokens, as cases that can be timed and compared.

A step takes a tree of drafted tokens per sequence: node 0 is the token that was picked last, node i
the child of node parents[i] < i (-1: a root). Its nodes go through the model at once, the tokens
that follow each are sampled, and the drafted ones that agree with them stay.

Kinds
  rope     the rotary embedding of queries and keys at given positions
  attn     attention of the nodes over a 4-bit cache and over their ancestors, which a second 4-bit
           cache ("draft") holds, node i in slot i: node i is at position length + depth, sees the
           cache's positions of its window, itself and those of its ancestors that the window reaches
  commit   accepted nodes' keys and values move from the draft into the cache, read back
  sample   a token from every row of logits, and the logarithm of its probability
  accept   the nodes that agree with what was sampled, and the token that follows the last

A 4-bit cache of B sequences, H key / value heads and D channels holds values in blocks of 32
channels that share a power of two (2^e, stored as the byte e + 127), each value as a sign and one of
0, 0.5, 1, 1.5, 2, 3, 4, 6; position p is in slot p % C of C:

  k_codes   uint8 (B, H, C, D/2)         channel 2i in the low half of byte i, 2i + 1 in the high one
  k_scales  uint8 (B, H, C, D/32)
  v_codes   uint8 (B, H, C/4, D/8, 4, 4) words of 8 channels, those of 4 slots side by side
  v_scales  uint8 (B, H, C/4, D/32, 4)
  lengths   int32 (B)

Sampling ranks a row's tokens by logit (ties: the lower index first) and gives each the weight
exp((logit - highest) / temperature). It keeps the first top_k, of those the shortest run with at
least top_p of their sum, of those the ones with at least min_p of the first one's weight, and takes
the first whose running sum exceeds `uniform` times the sum. Temperature 0: the first.

`ragged`: lengths, and numbers of nodes, that differ between the sequences. Sizes are those of the
repository's model configurations, tests and benchmark.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
# the exponents that keep every held value a normal number of the type (f16: any number)
E_RANGE = {"bf16": (-125, 125), "f16": (-23, 13)}


def listed():
    return [
        # the nodes of one drafted step, 32 sequences, Qwen3-0.6B heads
        _rope("rope-step", B=32, T=16, Hq=16, Hkv=8, D=128, rot=128, far=65536),
        # packed prompts of 64K tokens, half of each head in interleaved pairs, stretched frequencies
        _rope("rope-packed", B=1, T=65536, Hq=16, Hkv=8, D=128, rot=64, far=65536, pairs=True,
              packed=True, scaled=True),
        # a few nodes over a short conversation on the smallest heads: launch and host latency
        _attn("attn-short", B=1, N=8, Hq=4, Hkv=2, D=64, cap=512, length=257),
        # 8 sequences of mixed length with 16 nodes each
        _attn("attn-batch", B=8, N=16, Hq=16, Hkv=8, D=128, cap=16384, length=16000, ragged=True),
        # 64 nodes on a full window of 8192, the ring wrapped
        _attn("attn-window", B=4, N=64, Hq=16, Hkv=8, D=128, cap=12288, length=40001, window=8192,
              lse=True),
        # 4 nodes of 64 accepted
        _commit("commit-one", B=1, P=4, N=64, Hkv=8, D=128, cap=16384, length=9000),
        # a large batch, fp16, three query heads a key / value head
        _commit("commit-batch-f16", B=64, P=16, N=256, Hkv=5, D=64, cap=4096, length=4090,
                ragged=True, dtype="f16"),
        # the next token of one sequence, Qwen3 vocabulary
        _sample("sample-token", R=1, V=151936, temperature=0.7, top_k=20, top_p=0.8),
        # those of the 64 nodes of a drafted step, every token a candidate
        _sample("sample-tree-f16", R=64, V=151936, dtype="f16"),
        # a batch of requests, each with settings of its own
        _sample("sample-batch", R=256, V=151936, mixed=True),
        # one drafted step
        _accept("accept-one", B=1, N=16),
        # a large batch of large trees
        _accept("accept-batch", B=256, N=256, ragged=True),
    ]


def _case(kind, name, **case):
    return dict(case, kind=kind) if name is None else dict(case, kind=kind, name=name)


def _rope(name, *, B, T, Hq, Hkv, D, rot, far, pairs=False, packed=False, scaled=False,
          inverse=False, dtype="bf16"):
    return _case("rope", name, B=B, T=T, Hq=Hq, Hkv=Hkv, D=D, rot=rot, far=far, pairs=pairs,
                 packed=packed, scaled=scaled, inverse=inverse, dtype=dtype)


def _attn(name, *, B, N, Hq, Hkv, D, cap, length, window=-1, ragged=False, lse=False,
          dtype="bf16"):
    return _case("attn", name, B=B, N=N, Hq=Hq, Hkv=Hkv, D=D, cap=cap, length=length,
                 window=window, ragged=ragged, lse=lse, dtype=dtype)


def _commit(name, *, B, P, N, Hkv, D, cap, length, ragged=False, dtype="bf16"):
    return _case("commit", name, B=B, P=P, N=N, Hkv=Hkv, D=D, cap=cap, length=length,
                 ragged=ragged, dtype=dtype)


def _sample(name, *, R, V, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mixed=False,
            dtype="bf16"):
    return _case("sample", name, R=R, V=V, temperature=temperature, top_k=top_k, top_p=top_p,
                 min_p=min_p, mixed=mixed, dtype=dtype)


def _accept(name, *, B, N, ragged=False):
    return _case("accept", name, B=B, N=N, ragged=ragged)


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(("rope", "attn", "attn", "commit", "sample", "sample", "accept"))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    ragged = rng.random() < 0.6
    if kind == "accept":
        return _accept(None, B=_log_int(rng, 1, 256), N=_log_int(rng, 1, 256), ragged=ragged)
    if kind == "sample":
        R = rng.choice((1, 1, _log_int(rng, 1, 256)))
        V = rng.choice((151936, 49152, 1024, _log_int(rng, 2, 151936)))
        return _sample(None, R=R, V=V, temperature=rng.choice((0.0, 0.3, 0.7, 1.0, 1.5)),
                       top_k=rng.choice((0, 0, 1, 20, 50, _log_int(rng, 1, V))),
                       top_p=rng.choice((1.0, 1.0, 0.8, 0.95)), min_p=rng.choice((0.0, 0.0, 0.05)),
                       mixed=rng.random() < 0.3, dtype=dtype)
    Hq, Hkv, D = rng.choice(((16, 8, 128), (16, 8, 128), (15, 5, 64), (4, 2, 64), (8, 2, 128),
                             (4, 4, 128), (9, 3, 64)))
    if kind == "rope":
        dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
        D = rng.choice((D, D, 80, 96, 256))
        B = rng.choice((1, 1, 2, 5, 32))
        top = 65536 * 24 * 128 * 2 // (B * (Hq + Hkv) * D * (4 if dtype == "f32" else 2))
        packed = rng.random() < 0.4
        return _rope(None, B=B, T=_log_int(rng, 1, min(top, 65536)), Hq=Hq, Hkv=Hkv, D=D,
                     rot=rng.choice((D, D, D // 2, 2 * rng.randint(1, D // 2))),
                     far=rng.choice((2048, 65536, 1000000)), pairs=rng.random() < 0.5,
                     packed=packed, scaled=rng.random() < 0.3, inverse=rng.random() < 0.3,
                     dtype=dtype)
    N = rng.choice((1, 8, 16, 64, _log_int(rng, 1, 256)))
    if kind == "commit":
        cap = 32 * _log_int(rng, 8, 512)
        return _commit(None, B=_log_int(rng, 1, 64), P=_log_int(rng, 1, N), N=N, Hkv=Hkv, D=D,
                       cap=cap, length=_log_int(rng, 1, 3 * cap), ragged=ragged, dtype=dtype)
    B = rng.choice((1, 1, 2, 3, 8))
    top = 4 * 64 * 16 * 12288 // (B * N * Hq)  # keys of a call as large as the largest listed
    cap = 32 * max(2, _log_int(rng, 2, min(512, top // 32)))
    # from an empty cache on, up to a full one, or past it
    length = rng.choice((0, _log_int(rng, 1, cap), _log_int(rng, 1, cap), cap,
                         cap + _log_int(rng, 1, 3 * cap)))
    return _attn(None, B=B, N=N, Hq=Hq, Hkv=Hkv, D=D, cap=cap, length=length,
                 window=rng.choice((-1, -1, 8192, 2048, 512, _log_int(rng, 1, cap))),
                 ragged=ragged, lse=rng.random() < 0.5, dtype=dtype)


def _counts(case):
    """The nodes of each sequence: all N, or down to none (accepted ones of a commit: all P)."""
    B, n = case["B"], case["P" if case["kind"] == "commit" else "N"]
    return [n - n * b // max(1, B - 1) if case["ragged"] and B > 1 else n for b in range(B)]


def _lengths(case):
    """The positions that each sequence has had before the call."""
    B, n = case["B"], case["length"]
    return [n - n * b // B if case["ragged"] else n for b in range(B)]


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


def _filled(case, g, C, lengths):
    """A cache of C slots that all hold something, as after earlier sequences."""
    B, H, D = case["B"], case["Hkv"], case["D"]
    x = torch.randn(B, H, C, D, generator=g, device=DEV)
    x[..., ::19] *= 3  # keys have a few channels of larger values, as after rotary embedding
    kc, ks = _quantise(x, case["dtype"])
    x = torch.randn(B, H, C, D, generator=g, device=DEV)
    vc, vs = _quantise(x, case["dtype"])
    return dict(k_codes=_pack(kc), k_scales=ks,
                v_codes=_interleave(_pack(vc).unflatten(-1, (-1, 4))).contiguous(),
                v_scales=_interleave(vs).contiguous(),
                lengths=torch.tensor(lengths, dtype=torch.int32, device=DEV))


def _trees(case, g):
    """(B, N) int32: every node's parent is one of the 12 nodes before it."""
    B, N = case["B"], case["N"]
    i = torch.arange(N, device=DEV)
    back = 1 + torch.rand(B, N, generator=g, device=DEV) * i.clamp(max=12)
    parents = (i - back.long()).clamp(min=0)
    parents[:, 0] = -1
    return parents.int()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    kind = case["kind"]
    if kind == "sample":
        return _prepare_sample(case, g)
    B = case["B"]
    s = dict(case=case)
    if kind == "rope":
        T, D, n = case["T"], case["D"], case["rot"] // 2
        dt = DTYPES[case["dtype"]]
        s["q"] = torch.randn(B, T, case["Hq"], D, generator=g, device=DEV).to(dt)
        s["k"] = torch.randn(B, T, case["Hkv"], D, generator=g, device=DEV).to(dt)
        f = 1000000.0 ** -(torch.arange(n, device=DEV, dtype=torch.float32) / n)
        s["inv_freq"] = torch.where(f < 0.01, f / 4, f) if case["scaled"] else f
        s["scale"] = 0.1 * math.log(4) + 1 if case["scaled"] else 1.0
        start = torch.randint(case["far"], (B, T), generator=g, device=DEV)
        if case["packed"]:  # sequences one after the other, each from position 0 on
            i = torch.arange(T, device=DEV).expand(B, T)
            first = (start % 997 == 0).logical_or(i == 0)
            start = i - torch.where(first, i, 0).cummax(-1).values
        s["positions"] = start.int()
        return s
    ragged = case["ragged"] and B > 1
    counts = torch.tensor(_counts(case), dtype=torch.int32, device=DEV)
    if kind == "accept":
        N = case["N"]
        s["parents"] = _trees(case, g)
        # most nodes' token is the one that was picked after their parent
        s["picked"] = torch.randint(151936, (B, N), generator=g, device=DEV)
        drafted = s["picked"].gather(1, s["parents"].clamp(min=0).long())
        wrong = torch.rand(B, N, generator=g, device=DEV) < 0.3
        s["tokens"] = torch.where(wrong, drafted - 1, drafted)
        s["counts"] = counts if ragged else None
        return s
    s["cache"] = _filled(case, g, case["cap"], _lengths(case))
    nodes = 32 * ((case["N"] + 31) // 32)
    if kind == "commit":
        s["draft"] = _filled(case, g, nodes, [case["N"]] * B)
        # P of the N nodes, in their order
        order = torch.rand(B, case["N"], generator=g, device=DEV).argsort(-1)
        s["path"] = order[:, :case["P"]].sort(-1).values.int()
        s["counts"] = counts
        return s
    s["draft"] = _filled(case, g, nodes, _counts(case))
    s["parents"] = _trees(case, g)
    s["counts"] = counts if ragged else None
    s["q"] = torch.randn(B, case["N"], case["Hq"], case["D"], generator=g,
                         device=DEV).to(DTYPES[case["dtype"]])
    return s


def _prepare_sample(case, g):
    R, V = case["R"], case["V"]
    x = torch.randn(R, V, generator=g, device=DEV) * 2
    # a few tokens stand out, and those behind the vocabulary's last are masked
    x.scatter_add_(1, torch.randint(V, (R, min(V, 40)), generator=g, device=DEV),
                   torch.rand(R, min(V, 40), generator=g, device=DEV) * 12)
    x[:, V - V // 600:] = -math.inf
    s = dict(case=case, logits=x.to(DTYPES[case["dtype"]]),
             uniform=torch.rand(R, generator=g, device=DEV))
    for name in ("temperature", "top_k", "top_p", "min_p"):
        s[name] = case[name]
    if case["mixed"]:
        i = torch.arange(R, device=DEV)
        s["temperature"] = (i % 5).float() * 0.3
        s["top_k"] = torch.where(i % 3 == 0, 0, 1 + 7 * i % V).int()
        s["top_p"] = 1 - (i % 4).float() * 0.1
        s["min_p"] = torch.where(i % 6 == 5, 0.02, 0.0).float()
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


def _plain_rope(s):
    case = s["case"]
    n = case["rot"] // 2
    angle = s["positions"].double()[..., None] * s["inv_freq"].double()
    cos = (angle.cos() * s["scale"]).float()[:, :, None]
    sin = (angle.sin() * (-s["scale"] if case["inverse"] else s["scale"])).float()[:, :, None]

    def rotate(x):
        y = x.float()
        r = y[..., :2 * n]
        a, b = (r[..., ::2], r[..., 1::2]) if case["pairs"] else (r[..., :n], r[..., n:])
        a, b = a * cos - b * sin, a * sin + b * cos
        r = torch.stack((a, b), -1).flatten(-2) if case["pairs"] else torch.cat((a, b), -1)
        return torch.cat((r, y[..., 2 * n:]), -1).to(x.dtype)
    return rotate(s["q"]), rotate(s["k"])


def _ancestors(parents):
    """(B, N, N): whether j is i or one of its ancestors."""
    B, N = parents.shape
    i = torch.arange(N, device=DEV)
    up = (parents[..., None] == i) | (i[:, None] == i)
    up = up.float()
    for _ in range(max(1, (N - 1).bit_length())):  # twice the steps each time
        up = (up @ up).clamp_(max=1)
    return up > 0


def _nodes(s, B, N):
    """How many nodes every sequence has, (B, 1)."""
    if s["counts"] is None:
        return torch.full((B, 1), N, device=DEV)
    return s["counts"].long()[:, None]


def _plain_attn(s):
    case, c, d = s["case"], s["cache"], s["draft"]
    B, N, Hq, D = s["q"].shape
    H, C, W = case["Hkv"], case["cap"], case["window"]
    G = Hq // H
    up = _ancestors(s["parents"])
    depth = up.sum(-1) - 1
    length = c["lengths"].long()[:, None]
    slot = torch.arange(C, device=DEV)
    p = length - 1 - (length - 1 - slot) % C  # the position in each slot, negative for none
    p = torch.where(length > 0, p, -1)
    at = length + depth
    seen = (p >= 0)[:, None].expand(B, N, C)
    if W > 0:
        seen = seen & (p[:, None] > at[..., None] - W)
        up = up & (depth[:, None] > depth[..., None] - W)
    node = torch.arange(N, device=DEV)
    there = node < _nodes(s, B, N)
    seen = torch.cat((seen, up), -1) & there[..., None]
    k = torch.cat((_k_values(c), _k_values(d)[:, :, :N]), 2)
    v = torch.cat((_v_values(c).masked_fill((p < 0)[:, None, :, None], 0),
                   _v_values(d)[:, :, :N].masked_fill(~there[:, None, :, None], 0)), 2)
    q = s["q"].float().transpose(1, 2).reshape(B, H, G * N, D)
    x = (q @ k.transpose(2, 3)).mul_(D ** -0.5).view(B, H, G, N, -1)
    x.masked_fill_(~seen[:, None, None], -math.inf)
    lse = x.logsumexp(-1).view(B, Hq, N)
    top = x.amax(-1, keepdim=True)
    e = x.sub_(top.masked_fill(top == -math.inf, 0)).exp_()
    e = e.div_(e.sum(-1, keepdim=True).clamp_min_(1e-30)).view(B, H, G * N, -1)
    o = (e @ v).view(B, Hq, N, D).transpose(1, 2).to(s["q"].dtype)
    return (o, lse) if case["lse"] else o


def _plain_commit(s):
    case, c, d = s["case"], s["cache"], s["draft"]
    C, P, counts = case["cap"], case["P"], s["counts"].long()[:, None]
    b, i = (torch.arange(P, device=DEV) < counts).nonzero(as_tuple=True)
    slot = (c["lengths"].long()[b] + i) % C
    node = s["path"][b, i].long()
    for name in ("k_codes", "k_scales"):
        c[name][b, :, slot] = d[name][b, :, node]
    c["v_codes"][b, :, slot // 4, :, slot % 4] = d["v_codes"][b, :, node // 4, :, node % 4]
    c["v_scales"][b, :, slot // 4, :, slot % 4] = d["v_scales"][b, :, node // 4, :, node % 4]
    c["lengths"] += s["counts"]
    # the last P positions, zeros where a sequence has none
    n = c["lengths"].long()[:, None]
    p = n - P + torch.arange(P, device=DEV)
    none = ((p < 0) | (p < n - C))[:, :, None, None]
    b, slot = torch.arange(case["B"], device=DEV)[:, None], p % C
    k = _values(c["k_codes"][b, :, slot], c["k_scales"][b, :, slot])
    v = _values(c["v_codes"][b, :, slot // 4, :, slot % 4].flatten(3),
                c["v_scales"][b, :, slot // 4, :, slot % 4])
    return tuple(x.masked_fill_(none, 0).to(DTYPES[case["dtype"]]) for x in (k, v))


def _settings(s):
    """temperature, top_k, top_p and min_p as float64 columns."""
    like = s["uniform"].double()
    return [(x.double() if torch.is_tensor(x) else torch.full_like(like, x))[:, None]
            for x in (s["temperature"], s["top_k"], s["top_p"], s["min_p"])]


def _plain_sample(s):
    t, k, p, m = _settings(s)
    V = s["case"]["V"]
    x, order = s["logits"].double().sort(dim=-1, descending=True, stable=True)
    top = x[:, :1]
    w = ((x - top) / t).exp().masked_fill_(x == top, 1).masked_fill_(x == -math.inf, 0)
    rank = torch.arange(V, device=DEV)
    w *= rank < torch.where(t == 0, 1, torch.where(k > 0, k, V))
    run = w.cumsum(-1)
    before = torch.nn.functional.pad(run[:, :-1], (1, 0))
    w *= (before < p * run[:, -1:]) | (p >= 1) | (rank == 0)
    w *= w >= m
    run = w.cumsum(-1)
    total = run[:, -1:]
    j = (run <= s["uniform"].double()[:, None] * total).sum(-1, keepdim=True)
    j = torch.minimum(j, (w > 0).sum(-1, keepdim=True) - 1)
    return order.gather(1, j)[:, 0], (w.gather(1, j) / total).log()[:, 0].float()


def _plain_accept(s):
    B, N = s["parents"].shape
    parents, tokens, picked = s["parents"].long(), s["tokens"], s["picked"]
    node = torch.arange(N, device=DEV)
    there = node < _nodes(s, B, N)
    # a node agrees if its token was picked after its parent; of several children the first
    agrees = (tokens == picked.gather(1, parents.clamp(min=0))) & (parents >= 0) & there
    first = torch.full((B, N), N, device=DEV).scatter_reduce_(
        1, parents.clamp(min=0), torch.where(agrees, node, N), "amin")
    agrees &= first.gather(1, parents.clamp(min=0)) == node
    agrees |= (node == 0) & there
    up = _ancestors(s["parents"])
    stays = (agrees[:, None] | ~up).all(-1)
    accepted = stays.sum(-1)
    path = torch.where(stays, node, N).sort(-1).values
    last = path.gather(1, (accepted[:, None] - 1).clamp(min=0)).clamp(max=N - 1)
    token = torch.where(accepted > 0, picked.gather(1, last)[:, 0], -1)
    return path.masked_fill(path == N, -1).int(), accepted.int(), token


# ----------------------------------------------------------------------- run

def run(s):
    case = s["case"]
    if own:
        return _own(s, case)
    return {"rope": _plain_rope, "attn": _plain_attn, "commit": _plain_commit,
            "sample": _plain_sample, "accept": _plain_accept}[case["kind"]](s)


def _own(s, case):
    import ttcd_amd
    kind = case["kind"]
    if kind == "rope":
        return ttcd_amd.rope(s["q"], s["k"], s["inv_freq"], s["positions"],
                             interleaved=case["pairs"], scale=s["scale"], inverse=case["inverse"])
    if kind == "sample":
        return ttcd_amd.sample(s["logits"], s["uniform"], temperature=s["temperature"],
                               top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                               return_logprob=True)
    if kind == "accept":
        return ttcd_amd.tree_accept(s["parents"], s["tokens"], s["picked"], counts=s["counts"])
    cache, draft = (
        ttcd_amd.KV4Cache.from_parts(c["k_codes"], c["k_scales"], c["v_codes"], c["v_scales"],
                                     c["lengths"], DTYPES[case["dtype"]])
        for c in (s["cache"], s["draft"]))
    if kind == "attn":
        return ttcd_amd.kv4_tree_attn(s["q"], cache, draft, s["parents"], case["window"],
                                      counts=s["counts"], return_lse=case["lse"])
    ttcd_amd.kv4_commit(cache, draft, s["path"], s["counts"])
    return ttcd_amd.kv4_read(cache, case["P"])


def work(case):
    kind = case["kind"]
    if kind == "sample":
        return {"bytes": case["R"] * (2 * case["V"] + 16), "flops": 0}
    B = case["B"]
    if kind == "rope":
        rows, size = B * case["T"], 4 if case["dtype"] == "f32" else 2
        heads = case["Hq"] + case["Hkv"]
        return {"bytes": rows * (2 * heads * case["D"] * size + 4) + 2 * case["rot"],
                "flops": 3 * rows * heads * case["rot"]}
    if kind == "accept":
        return {"bytes": B * case["N"] * (4 + 8 + 8 + 4) + 12 * B, "flops": 0}
    H, D = case["Hkv"], case["D"]
    row = D // 2 + D // 32  # bytes of one key or value in the cache
    if kind == "commit":
        # nodes read and written; the last P positions read, their values written
        return {"bytes": 4 * sum(_counts(case)) * H * row
                + 2 * B * case["P"] * H * (row + 2 * D), "flops": 0}
    # a node sees its window of the cache and, taken as one of a chain, the nodes before it
    Hq, W, C = case["Hq"], case["window"], case["cap"]
    keys = pairs = rows = 0
    for n, c in zip(_lengths(case), _counts(case)):
        held = min(n, C)
        keys += (min(held, W - 1) if W > 0 else held) + c if c else 0
        pairs += sum((min(held, max(0, W - 1)) if W > 0 else held) + 1 for _ in range(c))
        rows += c * Hq
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


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "attn": _exact_attn, "commit": _exact_commit,
            "sample": _exact_sample, "accept": _exact_accept}[case["kind"]](s, case)


def _exact_rope(s, case):
    n = case["rot"] // 2
    turn = torch.polar(torch.full((), s["scale"], dtype=torch.float64, device=DEV),
                       s["positions"].double()[..., None] * s["inv_freq"].double()
                       * (-1 if case["inverse"] else 1))[:, :, None]
    out = []
    re, im = slice(0, n), slice(n, 2 * n)
    if case["pairs"]:
        re, im = slice(0, 2 * n, 2), slice(1, 2 * n, 2)
    for x in (s["q"].double(), s["k"].double()):
        z = torch.complex(x[..., re], x[..., im]) * turn
        x[..., re] = z.real
        x[..., im] = z.imag
        out.append(x)
    return tuple(out)


def _lineage(parents):
    """For every node of one sequence, itself and its ancestors."""
    out = []
    for i, p in enumerate(parents):
        out.append(([] if p < 0 else out[p]) + [i])
    return out


def _exact_attn(s, case):
    B, N, Hq, D = s["q"].shape
    H, C, W = case["Hkv"], case["cap"], case["window"]
    G = Hq // H
    o = torch.zeros(B, N, Hq, D, dtype=torch.float64, device=DEV)
    lse = torch.full((B, Hq, N), -math.inf, dtype=torch.float64, device=DEV)
    parents = s["parents"].tolist()
    for b, (n, count) in enumerate(zip(_lengths(case), _counts(case))):
        if not count:
            continue
        p = torch.arange(max(0, n - C), n, device=DEV)
        lines = _lineage(parents[b][:count])
        at = torch.tensor([n + len(x) - 1 for x in lines], device=DEV)
        tree = torch.zeros(count, count, dtype=torch.bool)
        for i, x in enumerate(lines):
            tree[i, x[-W:] if W > 0 else x] = True
        seen = torch.cat((p > at[:, None] - (W if W > 0 else n + N + 1), tree.to(DEV)), 1)
        nodes = torch.arange(count, device=DEV)
        for h in range(H):
            k, v = (torch.cat(x) for x in zip(_exact_rows(s["cache"], b, h, p % C),
                                              _exact_rows(s["draft"], b, h, nodes)))
            for g in range(h * G, h * G + G):
                x = (s["q"][b, :count, g].double() @ k.T * D ** -0.5).masked_fill(~seen, -math.inf)
                lse[b, g, :count] = x.logsumexp(-1)
                o[b, :count, g] = torch.exp(x - lse[b, g, :count, None]) @ v
    return (o, lse) if case["lse"] else o


def _exact_commit(s, case):
    B, H, C, P, D = case["B"], case["Hkv"], case["cap"], case["P"], case["D"]
    out = [torch.zeros(B, P, H, D, dtype=torch.float64, device=DEV) for _ in range(2)]
    for b, (n, count) in enumerate(zip(_lengths(case), _counts(case))):
        new = s["path"][b, :count].long()
        # the positions before the new ones that are still held
        old = torch.arange(max(0, n - C + count, n + count - P), n, device=DEV)
        for h in range(H):
            rows = zip(_exact_rows(s["cache"], b, h, old % C), _exact_rows(s["draft"], b, h, new))
            for x, (was, now) in zip(out, rows):
                both = torch.cat((was, now))[-P:]
                x[b, P - len(both):, h] = both
    return tuple(out)


def _exact_sample(s, case):
    """By the distinct logits of a row, how often each comes and how many of its tokens stay."""
    tokens = torch.zeros(case["R"], dtype=torch.int64, device=DEV)
    logprob = torch.zeros(case["R"], dtype=torch.float64, device=DEV)
    settings = torch.cat(_settings(s), 1).tolist()
    uniform = s["uniform"].tolist()
    for r, (t, k, p, m) in enumerate(settings):
        x = s["logits"][r].double()
        value, count = x[x > -math.inf].unique(return_counts=True)
        value, count = value.flip(0), count.flip(0)
        if t == 0:
            t, k = 1.0, 1
        w = torch.exp((value - value[0]) / t)
        if k > 0:
            count = torch.minimum(count, (k - (count.cumsum(0) - count)).clamp(min=0).long())
        if p < 1:
            each = w * count
            left = p * each.sum() - (each.cumsum(0) - each)  # of the sum, before each value
            need = (left / w).ceil().clamp(min=0)
            need[0] = need[0].clamp(min=1)
            count = torch.minimum(count, need.long())
        count = torch.where(w >= m, count, 0)
        each = w * count
        run = each.cumsum(0)
        i = int((run <= uniform[r] * run[-1]).sum())
        i = min(i, int((each > 0).sum()) - 1)
        j = int((uniform[r] * run[-1] - (run[i] - each[i])) / w[i])
        j = min(max(j, 0), int(count[i]) - 1)
        tokens[r] = (x == value[i]).nonzero()[j, 0]
        logprob[r] = torch.log(w[i] / run[-1])
    return tokens, logprob


def _exact_accept(s, case):
    B, N = case["B"], case["N"]
    parents, tokens, picked = (s[n].tolist() for n in ("parents", "tokens", "picked"))
    paths, token = [], []
    for b, count in enumerate(_counts(case)):
        path = [0] if count else []
        i = 1
        while path and i < count:  # children come after their parents
            if parents[b][i] == path[-1] and tokens[b][i] == picked[b][path[-1]]:
                path.append(i)
            i += 1
        token.append(picked[b][path[-1]] if path else -1)
        paths.append(path)
    out = torch.tensor([p + [-1] * (N - len(p)) for p in paths], dtype=torch.int32, device=DEV)
    return (out, torch.tensor([len(p) for p in paths], dtype=torch.int32, device=DEV),
            torch.tensor(token, device=DEV))

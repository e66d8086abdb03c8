"""A step that verifies drafted tokens, in plain float64 / integer torch and Python on the
CPU: rotary embedding at given positions, attention of a tree over the 4-bit cache (over
kv4_ref.Ref's rows), sampling, and the walk over the tree."""
from __future__ import annotations

import math

import torch


def _arctan_of_reciprocal(x, one):
    """arctan(1 / x) in units of 1 / one, by its series."""
    total, term, k = 0, one // x, 1
    while term:
        total += term // k if k % 4 == 1 else -(term // k)
        term //= x * x
        k += 2
    return total


_BITS = 240
# 2 pi = 8 (4 arctan(1 / 5) - arctan(1 / 239)), in units of 2^-_BITS
_TURN = 8 * (4 * _arctan_of_reciprocal(5, 1 << _BITS) - _arctan_of_reciprocal(239, 1 << _BITS))


def _angle(p, f):
    """p f modulo 2 pi, the product in integers: it passes 53 bits for positions from 2^29 on."""
    num, den = f.as_integer_ratio()
    a = (p * num << _BITS) // den % _TURN
    return math.ldexp(a - _TURN if 2 * a > _TURN else a, -_BITS)


def rope(x, inv_freq, positions, interleaved=False, scale=1.0, inverse=False):
    """x (B, T, H, D) turned by positions (B, T), float64, and sum |x| |turn| of each pair."""
    n = inv_freq.numel()
    y, mag = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64)
    if positions.numel() and positions.abs().max() >= 2 ** 29:
        a = torch.tensor([[[_angle(p, f) for f in inv_freq.tolist()] for p in row]
                          for row in positions.tolist()], dtype=torch.float64)
    else:
        a = positions.double()[..., None] * inv_freq.double()
    a = a * (-1 if inverse else 1)
    turn = torch.polar(torch.full_like(a, scale), a)[:, :, None]
    i = torch.arange(n)
    re, im = (2 * i, 2 * i + 1) if interleaved else (i, n + i)
    z = torch.complex(y[..., re], y[..., im])
    mag[..., re] = mag[..., im] = scale * (z.real.abs() + z.imag.abs())
    z = z * turn
    y[..., re], y[..., im] = z.real, z.imag
    return y, mag


def lineage(parents):
    """For every node of one sequence, its ancestors and itself, from the root down. A parent
    that does not come before its node is none."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if 0 <= p < i else []) + [i])
    return out


def tree_attn(r, d, q, parents, window=None, counts=None):
    """r, d: the cache's and the draft's kv4_ref.Ref. o (B, N, Hq, D), lse (B, Hq, N), and
    sum_j p_j |v_j| like o."""
    B, N, Hq, D = q.shape
    G = Hq // r.H
    o, mag = (torch.zeros(B, N, Hq, D, dtype=torch.float64) for _ in range(2))
    lse = torch.full((B, Hq, N), -math.inf, dtype=torch.float64)
    for b in range(B):
        n = min(N if counts is None else int(counts[b]), d.length(b))
        if n <= 0:
            continue
        L, first = r.length(b), r.first(b)
        k, v = (torch.cat((r.rows[b][i][first:], d.rows[b][i][:n])).repeat_interleave(G, 1)
                for i in range(2))
        lines = lineage(parents[b, :n].tolist())
        seen = torch.zeros(n, L - first + n, dtype=torch.bool)
        for i, line in enumerate(lines):
            at = L + len(line) - 1
            low = 0 if window is None or window <= 0 else at - window + 1
            seen[i, max(0, low - first):L - first] = True
            for depth, j in enumerate(line):
                seen[i, L - first + j] = L + depth >= low
        x = torch.einsum("thd,lhd->htl", q[b, :n].double().cpu(), k) * D ** -0.5
        x = x.masked_fill(~seen, -math.inf)
        s = x.logsumexp(-1)
        p = torch.exp(x - s[..., None])
        o[b, :n] = torch.einsum("htl,lhd->thd", p, v)
        mag[b, :n] = torch.einsum("htl,lhd->thd", p, v.abs())
        lse[b, :, :n] = s
    return o, lse, mag


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, logprob) of one row: sorted, in Python's fsum where a border is decided."""
    x = [float(v) for v in logits]
    order = sorted((i for i, v in enumerate(x) if v == v and v > -math.inf),
                   key=lambda i: (-x[i], i))
    if not order:
        return -1, -math.inf
    if temperature == 0:
        temperature, top_k = 1.0, 1
    top = x[order[0]]
    w = [1.0 if x[i] == top else math.exp((x[i] - top) / temperature) for i in order]
    n = min(top_k, len(order)) if top_k > 0 else len(order)
    if top_p < 1:
        want, run = top_p * math.fsum(w[:n]), 0.0
        for m in range(n):
            run += w[m]
            if run >= want:
                n = m + 1
                break
    while n > 1 and w[n - 1] < min_p:
        n -= 1
    total = math.fsum(w[:n])
    run = 0.0
    for m in range(n):
        run += w[m]
        if run > u * total:
            break
    return order[m], math.log(w[m] / total)


def accept(parents, tokens, picked, count):
    """(path, next) of one sequence."""
    path = [0] if count > 0 else []
    while path:
        more = [i for i in range(path[-1] + 1, count)
                if parents[i] == path[-1] and tokens[i] == picked[path[-1]]]
        if not more:
            break
        path.append(more[0])
    return path, picked[path[-1]] if path else -1

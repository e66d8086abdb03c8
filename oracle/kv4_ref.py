"""The 4-bit key / value cache of ttcd_amd.kv4 in plain float64 / integer torch on
the CPU: the format, the attention over it, its key weights and its eviction.

`Ref` keeps each sequence's rows as a list over all positions that it has had, of
the values that the cache holds for them; nothing of the device's layout is used
but in `codes_of`, which restates it."""
from __future__ import annotations

import math

import torch

GRID = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64)
E_RANGE = {torch.bfloat16: (-125, 125), torch.float16: (-23, 13)}


def quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes 0..15 like x, exponents (..., D/32)) of x (..., D), by search: the least
    exponent whose 6 2^e reaches the largest magnitude, then the nearest grid value,
    ties to the even code."""
    lo, hi = E_RANGE[x.dtype]
    y = torch.nan_to_num(x.double(), nan=0.0, posinf=math.inf, neginf=-math.inf)
    y = y.unflatten(-1, (-1, 32))
    top = y.abs().amax(-1)
    steps = 6 * torch.exp2(torch.arange(lo, hi + 1, dtype=torch.float64))
    e = torch.searchsorted(steps, top.contiguous()).clamp(max=hi - lo) + lo
    a = (y / torch.exp2(e.double())[..., None]).abs().clamp(max=6)
    d = (a[..., None] - GRID).abs()
    best = d.amin(-1, keepdim=True)
    even = torch.tensor([0, 0, 0, 0, 0, 0, 0, 0]) + torch.arange(8) % 2
    code = torch.where(d == best, even, 2).argmin(-1)
    code = code + 8 * torch.signbit(y)
    return code.flatten(-2), e


def values(code: torch.Tensor, e: torch.Tensor) -> torch.Tensor:
    x = GRID[code % 8] * torch.where(code >= 8, -1.0, 1.0)
    return (x.unflatten(-1, (-1, 32)) * torch.exp2(e.double())[..., None]).flatten(-2)


def held(x: torch.Tensor) -> torch.Tensor:
    """x as the cache holds it, float64."""
    return values(*quantise(x))


def codes_of(k: torch.Tensor, v: torch.Tensor):
    """The cache's four tensors for rows k, v (B, H, C, D) in slots 0 .. C-1."""
    out = []
    for x, is_v in ((k, False), (v, True)):
        code, e = quantise(x)
        packed = (code[..., ::2] + 16 * code[..., 1::2]).to(torch.uint8)
        scale = (e + 127).to(torch.uint8)
        if is_v:
            packed = packed.unflatten(-1, (-1, 4)).unflatten(2, (-1, 4)).transpose(3, 4)
            scale = scale.unflatten(2, (-1, 4)).transpose(3, 4)
        out += [packed.contiguous(), scale.contiguous()]
    return out


class Ref:
    """A cache of B sequences: rows[b] = (k (n, H, D), v), all positions ever appended."""

    def __init__(self, B: int, H: int, D: int, C: int, dtype=torch.bfloat16):
        self.B, self.H, self.D, self.C, self.dtype = B, H, D, C, dtype
        none = torch.zeros(0, H, D, dtype=torch.float64)
        self.rows = [(none, none) for _ in range(B)]

    def append(self, k, v, counts=None):
        for b in range(self.B):
            n = k.shape[1] if counts is None else int(counts[b])
            self.rows[b] = tuple(torch.cat((old, held(x[b, :n].cpu())))
                                 for old, x in zip(self.rows[b], (k, v)))

    def length(self, b):
        return self.rows[b][0].shape[0]

    def first(self, b):
        return max(0, self.length(b) - self.C)

    def read(self, count):
        out = []
        for i in range(2):
            x = torch.zeros(self.B, count, self.H, self.D, dtype=torch.float64)
            for b in range(self.B):
                n = self.length(b)
                rows = self.rows[b][i][max(self.first(b), n - count):]
                x[b, count - len(rows):] = rows
            out.append(x.to(self.dtype))
        return out

    def _scores(self, q, b, window, n):
        """(Hq, n, L) masked scores of sequence b's n queries, over all its positions."""
        L, G = self.length(b), q.shape[2] // self.H
        k = self.rows[b][0].repeat_interleave(G, 1)  # (L, Hq, D)
        x = torch.einsum("thd,lhd->htl", q[b, :n].double().cpu(), k) * self.D ** -0.5
        at = (L - n + torch.arange(n))[:, None]
        p = torch.arange(L)
        hidden = (p > at) | (p < self.first(b))
        if window is not None and window > 0:
            hidden = hidden | (p <= at - window)
        return x.masked_fill(hidden, -math.inf)

    def attn(self, q, window=None, counts=None):
        """o (B, T, Hq, D), lse (B, Hq, T), and sum_j p_j |v_j| like o, in float64."""
        B, T, Hq, D = q.shape
        o, mag = (torch.zeros(B, T, Hq, D, dtype=torch.float64) for _ in range(2))
        lse = torch.full((B, Hq, T), -math.inf, dtype=torch.float64)
        for b in range(B):
            n = T if counts is None else int(counts[b])
            if n == 0 or self.length(b) == 0:
                continue
            x = self._scores(q, b, window, n)
            s = x.logsumexp(-1)
            p = torch.exp(x - s.masked_fill(s == -math.inf, 0)[..., None])
            v = self.rows[b][1].repeat_interleave(Hq // self.H, 1)
            o[b, :n] = torch.einsum("htl,lhd->thd", p, v)
            mag[b, :n] = torch.einsum("htl,lhd->thd", p, v.abs())
            lse[b, :, :n] = s
        return o, lse, mag

    def key_weights(self, q, lse, window=None, counts=None):
        """(B, H, C) by slot, float64."""
        B, T, Hq, _ = q.shape
        out = torch.zeros(B, self.H, self.C, dtype=torch.float64)
        for b in range(B):
            n = T if counts is None else int(counts[b])
            if n == 0 or self.length(b) == 0:
                continue
            x = self._scores(q, b, window, n)
            s = lse[b, :, :n].double().cpu()[..., None]
            w = torch.where(s == -math.inf, 0.0, torch.exp(x - s.masked_fill(s == -math.inf, 0)))
            w = w.sum(1).view(self.H, -1, self.length(b)).sum(1)
            p = torch.arange(self.first(b), self.length(b))
            out[b][:, p % self.C] = w[:, p]
        return out

    def evict(self, weights, keep, recent):
        """(index (B, H, keep) of old positions, -1 behind them; their weights). Sorts
        the old keys by (weight, age) in plain Python."""
        index = torch.full((self.B, self.H, keep), -1, dtype=torch.int32)
        new_w = torch.zeros(self.B, self.H, keep)
        for b in range(self.B):
            p = list(range(self.first(b), self.length(b)))
            kept = min(len(p), keep)
            must = min(recent, kept)
            for h in range(self.H):
                w = {x: float(weights[b, h, x % self.C]) for x in p}
                old = sorted(p[:len(p) - must],
                             key=lambda x: (w[x] != w[x], -w[x] if w[x] == w[x] else 0.0, x))
                stay = sorted(old[:kept - must] + p[len(p) - must:])
                index[b, h, :kept] = torch.tensor(stay, dtype=torch.int32)
                for j, x in enumerate(stay):
                    new_w[b, h, j] = weights[b, h, x % self.C]
        return index, new_w

    def take(self, index, C):
        """The cache of capacity C that holds the positions of index (B, H, keep)."""
        new = Ref(self.B, self.H, self.D, C, self.dtype)
        for b in range(self.B):
            n = int((index[b, 0] >= 0).sum())
            at = index[b, :, :n].long().cpu().T  # (n, H)
            h = torch.arange(self.H)
            new.rows[b] = tuple(x[at, h] for x in self.rows[b])
        return new

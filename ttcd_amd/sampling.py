"""Picking tokens (host side of sample.hip).

    sample(logits, uniform, ...)            a token from every row of logits
    tree_accept(parents, tokens, picked)    the drafted tokens that agree with those

A step that verifies drafted tokens puts all nodes of a tree through the model at once
(kv4_tree_attn), samples what follows each, and keeps the drafted tokens that are what was
sampled: node 0 is the token that was picked last, and its child stays if its token is the
one sampled at node 0, that child's child if .. So with a random number per position the
text is the one that a token at a time would have given. Random numbers are the caller's.
"""
from __future__ import annotations

import torch

from . import _lib

_DT = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}


def _setting(x, name: str, rows: torch.Size, dtype: torch.dtype, device):
    """(the rows' values as a contiguous tensor or None, the value of all)."""
    if isinstance(x, torch.Tensor):
        if x.shape != rows or x.dtype != dtype or x.device != device:
            raise ValueError(f"sample: {name} must be a number or {dtype} {tuple(rows)} on the "
                             f"logits' device, got {tuple(x.shape)} {x.dtype}")
        return x.contiguous(), 0
    return None, x


def _ptr(t):
    return None if t is None else t.data_ptr()


def sample(logits: torch.Tensor, uniform: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0,
           min_p=0.0, return_logprob: bool = False):
    """A token from every row of logits (.., V), bf16 or f16: int64 of the leading shape.

    Tokens rank by logit, of equal ones the lower index first, and weigh exp((logit - highest)
    / temperature). Kept are the first top_k (0: all), of those the shortest run with at least
    top_p (1: all) of their sum, of those the ones with at least min_p (0: all) of the highest
    weight; the token is the first whose running sum exceeds ``uniform`` (fp32, the leading
    shape, numbers in [0, 1)) times the sum of all kept. temperature 0 takes the first.
    -infinity and NaN are no candidates; a row without any gives -1. Each setting is a number,
    or a tensor of the leading shape (fp32, top_k int32) with one for each row; a tensor's
    values are not checked (include/ttcd.h tells what those out of range do).

    With ``return_logprob`` also the fp32 logarithm of the token's share of the kept sum.
    Weights and sums are 64 bits, and none depends on an order of additions that could change:
    the same inputs give the same tokens."""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda or logits.dim() < 1:
        raise ValueError("sample: logits must be a (.., V) tensor on a GPU (HIP) device")
    if logits.dtype not in _DT:
        raise ValueError(f"sample: logits must be bf16 or f16, got {logits.dtype}")
    rows, V, dev = logits.shape[:-1], logits.shape[-1], logits.device
    if (not isinstance(uniform, torch.Tensor) or uniform.shape != rows
            or uniform.dtype != torch.float32 or uniform.device != dev):
        raise ValueError(f"sample: uniform must be fp32 {tuple(rows)} on the logits' device")
    if V < 1:
        raise ValueError("sample: rows of no logits")
    ts, t = _setting(temperature, "temperature", rows, torch.float32, dev)
    ks, k = _setting(top_k, "top_k", rows, torch.int32, dev)
    ps, p = _setting(top_p, "top_p", rows, torch.float32, dev)
    ms, m = _setting(min_p, "min_p", rows, torch.float32, dev)
    if (ts is None and not t >= 0) or (ks is None and (k < 0 or k != int(k))) or (
            ps is None and not p > 0) or (ms is None and not 0 <= m <= 1):
        raise ValueError(f"sample: need temperature >= 0, a whole top_k >= 0, top_p > 0 and min_p "
                         f"in 0 .. 1, got {t}, {k}, {p}, {m}")
    if torch.is_grad_enabled() and logits.requires_grad:
        raise RuntimeError("sample is forward-only: autograd / gradient inputs are not supported; "
                           "call it under torch.no_grad()")
    R = rows.numel()
    if logits.stride(-1) != 1 or logits.dim() > 2:
        logits = logits.reshape(R, V).contiguous()  # leading dimensions that merge: no copy
    uniform = uniform.contiguous()
    tokens = torch.empty_like(uniform, dtype=torch.int64)
    logprobs = torch.empty_like(uniform) if return_logprob else None
    if R:
        _lib.call(logits, _lib.lib().ttcd_sample_fwd, logits.data_ptr(),
                  logits.stride(0) if logits.dim() == 2 else 0, min(R, 2 ** 31 - 1),
                  min(V, 2 ** 31 - 1), uniform.data_ptr(),
                  _ptr(ts), float(t), _ptr(ks), min(int(k), 2 ** 31 - 1), _ptr(ps), float(p),
                  _ptr(ms), float(m), tokens.data_ptr(), _ptr(logprobs), _DT[logits.dtype])
    return (tokens, logprobs) if return_logprob else tokens


def tree_accept(parents: torch.Tensor, tokens: torch.Tensor, picked: torch.Tensor, *,
                counts: torch.Tensor | None = None):
    """The nodes of a tree that agree with what was picked: node 0, whose token is given, its
    first child whose token is picked[b, 0], of that the first child whose token is what was
    picked there, and on. parents int32 (B, N), -1 or a node before; tokens and picked int64
    (B, N): each node's token, and the one that was picked to follow it; counts int32 (B,):
    the first so many are nodes. N <= 256. Returns (path, accepted, next): the nodes in order,
    int32 (B, N), -1 behind the last; how many, int32 (B,); and what was picked at the last,
    int64 (B,) (-1 without nodes)."""
    if not isinstance(parents, torch.Tensor) or not parents.is_cuda or parents.dim() != 2:
        raise ValueError("tree_accept: parents must be (B, N) on a GPU (HIP) device")
    B, N = parents.shape
    dev = parents.device
    for name, t, dtype in (("parents", parents, torch.int32), ("tokens", tokens, torch.int64),
                           ("picked", picked, torch.int64)):
        if (not isinstance(t, torch.Tensor) or t.shape != (B, N) or t.dtype != dtype
                or t.device != dev):
            raise ValueError(f"tree_accept: {name} must be {dtype} ({B}, {N}) on the parents' "
                             "device")
    if counts is not None and (not isinstance(counts, torch.Tensor) or counts.shape != (B,)
                               or counts.dtype != torch.int32 or counts.device != dev):
        raise ValueError(f"tree_accept: counts must be int32 ({B},) on the parents' device")
    if N < 1:
        raise ValueError("tree_accept: trees of no nodes")
    parents, tokens, picked = parents.contiguous(), tokens.contiguous(), picked.contiguous()
    counts = None if counts is None else counts.contiguous()
    path = torch.empty_like(parents)
    accepted = parents.new_empty(B) if counts is None else torch.empty_like(counts)
    following = picked.new_empty(B)
    if B:
        _lib.call(parents, _lib.lib().ttcd_tree_accept, parents.data_ptr(), tokens.data_ptr(),
                  picked.data_ptr(), _ptr(counts), path.data_ptr(), accepted.data_ptr(),
                  following.data_ptr(), min(B, 2 ** 31 - 1),
                  min(N, 2 ** 31 - 1))
    return path, accepted, following

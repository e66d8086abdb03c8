"""Rotary embedding at given positions (host side of rope.hip).

    rope(q, k, inv_freq, positions)              the embedding, or its inverse
    rope_frequencies(dim, base, scaling, ...)    inv_freq and scale for it, plain or
                                                 stretched for long contexts

The attention prologue (ttcd_amd.prologue) rotates what the reference's RotaryEmbedding
rotates: halves of the whole head, by tables of the tensors' type, at consecutive
positions. This is the rotary embedding of other models and of other positions: halves or
interleaved pairs, the first channels of a head, every token at a position of its own (a
padded batch, packed sequences, the nodes of a tree of drafted tokens), without tables: the
angle position * inv_freq is exact, so positions may be far. ``inverse`` turns back: it takes
a cached key's position from it, and a gradient through the embedding.
"""
from __future__ import annotations

import math

import torch

from . import _lib

_DT = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16,
       torch.float32: _lib.DTYPE_F32}


def rope_frequencies(dim: int, base: float, scaling: dict | None = None, device=None,
                     length: int | None = None) -> tuple[torch.Tensor, float]:
    """(inv_freq, scale): the fp32 frequencies base ** (-2 i / dim), i < dim / 2, of a head's
    first `dim` channels, and the factor of cosine and sine. ``scaling`` is a model
    configuration's entry (type under "rope_type" or "type"):

    linear   frequencies / factor
    dynamic  base * (factor * n / m - factor + 1) ** (dim / (dim - 2)) as the base, n the
             larger of `length`, the tokens to come, and m
    yarn     of a pair that turns r times in m positions, frequencies / factor for r up to
             beta_slow (1), the plain ones from beta_fast (32) on, a ramp over the pairs'
             numbers between; scale 0.1 ln factor + 1, or attention_factor, or of
             mscale and mscale_all_dim the quotient of 0.1 mscale ln factor + 1
    llama3   frequencies / factor below low_freq_factor turns, the plain ones above
             high_freq_factor, a ramp over the turns between

    m = original_max_position_embeddings."""
    dim = int(dim)
    if dim < 2 or dim % 2:
        raise ValueError(f"rope_frequencies: dim must be even and >= 2, got {dim}")
    scaling = dict(scaling or {})
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    base = float(base)
    i = torch.arange(0, dim, 2, dtype=torch.float64)
    scale = 1.0

    def need(name):
        if scaling.get(name) is None:
            raise ValueError(f"rope_frequencies: scaling {kind!r} needs {name!r}")
        return float(scaling[name])

    if kind not in ("default", "linear", "dynamic", "yarn", "llama3"):
        raise NotImplementedError(f"rope_frequencies: scaling {kind!r}")
    factor = need("factor") if kind != "default" else 1.0
    if kind == "dynamic":
        m = need("original_max_position_embeddings")
        n = max(float(length or 0), m)
        if dim > 2:
            base *= (factor * n / m - factor + 1) ** (dim / (dim - 2))
    inv = base ** (-i / dim)
    if kind == "linear":
        inv = inv / factor
    elif kind == "yarn":
        m = need("original_max_position_embeddings")

        def pair(turns):  # the pair (a fraction) that turns so many times in m positions
            return dim * math.log(m / (turns * 2 * math.pi)) / (2 * math.log(base))

        low = pair(float(scaling.get("beta_fast") or 32))
        high = pair(float(scaling.get("beta_slow") or 1))
        if scaling.get("truncate", True):
            low, high = math.floor(low), math.ceil(high)
        low, high = max(low, 0), min(high, dim - 1)
        ramp = ((i / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)
        inv = inv / factor * ramp + inv * (1 - ramp)

        def mscale(x):
            return 0.1 * x * math.log(factor) + 1 if factor > 1 else 1.0

        if scaling.get("attention_factor") is not None:
            scale = float(scaling["attention_factor"])
        elif scaling.get("mscale") and scaling.get("mscale_all_dim"):
            scale = mscale(scaling["mscale"]) / mscale(scaling["mscale_all_dim"])
        else:
            scale = mscale(1.0)
    elif kind == "llama3":
        lo, hi = need("low_freq_factor"), need("high_freq_factor")
        turns = need("original_max_position_embeddings") * inv / (2 * math.pi)
        keep = ((turns - lo) / (hi - lo)).clamp(0, 1)
        inv = inv / factor * (1 - keep) + inv * keep
    return inv.to(torch.float32).to(device), scale


def rope(q: torch.Tensor, k: torch.Tensor | None, inv_freq: torch.Tensor,
         positions: torch.Tensor | None = None, *, offset: int = 0, interleaved: bool = False,
         scale: float = 1.0, inverse: bool = False):
    """q (B, T, Hq, D) and k (B, T, Hkv, D) (or None) with the first 2 * len(inv_freq) channels
    of every head turned in pairs, (i, n + i) or ``interleaved`` (2i, 2i + 1), by
    position * inv_freq[i], times scale; the other channels as they are. positions: int32 or
    int64, (B, T) or (T,), on q's device; None: offset .. offset + T - 1. bf16, f16 or f32;
    inv_freq fp32. ``inverse`` turns back. Returns new contiguous (q, k), or q alone."""
    for name, t in (("q", q), ("k", k), ("inv_freq", inv_freq), ("positions", positions)):
        if t is None and name in ("k", "positions"):
            continue
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError(f"rope: {name} must be a tensor on a GPU (HIP) device")
        if t.device != q.device:
            raise ValueError(f"rope: {name} must be on q's device")
        if torch.is_grad_enabled() and t.requires_grad:
            raise RuntimeError("rope is forward-only: autograd / gradient inputs are not supported; "
                               "call it under torch.no_grad() (inverse=True is its gradient)")
    if q.dim() != 4 or (k is not None and (k.dim() != 4 or k.shape[:2] != q.shape[:2]
                                           or k.shape[3] != q.shape[3] or k.dtype != q.dtype)):
        raise ValueError(f"rope: q and k must be (B, T, H, D) of the same B, T, D and dtype, got "
                         f"{tuple(q.shape)}, {None if k is None else tuple(k.shape)}")
    B, T, Hq, D = q.shape
    if q.dtype not in _DT:
        raise ValueError(f"rope: q and k must be bf16, f16 or f32, got {q.dtype}")
    n = inv_freq.numel()
    if inv_freq.dim() != 1 or inv_freq.dtype != torch.float32 or n < 1 or 2 * n > D:
        raise ValueError(f"rope: inv_freq must be fp32 (n,), 1 <= n <= {D // 2}, got "
                         f"{tuple(inv_freq.shape)} {inv_freq.dtype}")
    inv_freq = inv_freq.contiguous()
    steps = None
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64) or tuple(positions.shape) not in (
                (B, T), (T,)):
            raise ValueError(f"rope: positions must be int32 or int64 ({B}, {T}) or ({T},), got "
                             f"{tuple(positions.shape)} {positions.dtype}")
        steps = positions.stride() if positions.dim() == 2 else (0, positions.stride(0))
    q, k = (t if t is None or t.stride(3) == 1 else t.contiguous() for t in (q, k))
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    k_out = None if k is None else torch.empty(k.shape, dtype=k.dtype, device=k.device)
    if k is not None and k.shape[2] and not Hq:
        raise ValueError("rope: q has no heads")
    if q.numel():
        has_k = k is not None and k.shape[2] > 0
        _lib.call(
            q, _lib.lib().ttcd_rope_fwd, q.data_ptr(), k.data_ptr() if has_k else None,
            q_out.data_ptr(), k_out.data_ptr() if has_k else None, inv_freq.data_ptr(), n,
            None if positions is None else positions.data_ptr(),
            int(positions is not None and positions.dtype == torch.int64),
            None if steps is None else _lib.strides2(steps), int(offset), B, T, Hq,
            k.shape[2] if has_k else 0, D, _lib.strides4(q.stride()),
            _lib.strides4(k.stride()) if has_k else None, _lib.strides4(q_out.stride()),
            _lib.strides4(k_out.stride()) if has_k else None, int(bool(interleaved)),
            int(bool(inverse)), float(scale), _DT[q.dtype])
    return q_out if k is None else (q_out, k_out)

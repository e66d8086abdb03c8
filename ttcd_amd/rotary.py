"""Rotary embedding at given positions (host side of rope.hip).

    rope(q, k, inv_freq, positions)              the embedding, or its inverse
    rope_frequencies(dim, base, scaling, ...)    inv_freq and scale for it, plain or
                                                 stretched for long contexts

The attention prologue (ttcd_amd.prologue) rotates what the reference's RotaryEmbedding
rotates: halves of the whole head, by tables of the tensors' type, at consecutive
positions. This is the rotary embedding of other models and of other positions: halves or
interleaved pairs, the first channels of a head, every token at a position of its own (a
padded batch, packed sequences, the nodes of a tree of drafted tokens), without tables: the
angle position * inv_freq is exact (up to 2^53 of either), so positions may be far.
``inverse`` turns back, and multiplies by scale as well: so it takes a gradient through the
embedding. A cached key's position comes off with inverse=True and scale = 1 / the scale that
it was turned with.
"""
from __future__ import annotations

import math
from functools import lru_cache

import torch

from . import _lib

_DT = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16,
       torch.float32: _lib.DTYPE_F32}

# stride arrays (only read) of the last calls: finding one is quicker than making it
_strides4 = lru_cache(maxsize=64)(_lib.strides4)
_strides2 = lru_cache(maxsize=64)(_lib.strides2)


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
    int64, (B, T) or (T,), on q's device; None: offset .. offset + T - 1 (within 2^53). bf16,
    f16 or f32; inv_freq fp32. ``inverse`` turns back, times scale too: the gradient (with
    1 / scale the inverse). Returns new contiguous (q, k), or q alone."""
    if (not isinstance(q, torch.Tensor) or not q.is_cuda or q.dim() != 4
            or not isinstance(inv_freq, torch.Tensor) or not inv_freq.is_cuda):
        raise ValueError("rope: q (B, T, H, D) and inv_freq must be tensors on a GPU (HIP) device")
    B, T, Hq, D = q.shape
    dev, dtype = q.device, q.dtype
    code = _DT.get(dtype)
    if code is None:
        raise ValueError(f"rope: q and k must be bf16, f16 or f32, got {dtype}")
    n = inv_freq.numel()
    if (inv_freq.dim() != 1 or inv_freq.dtype != torch.float32 or inv_freq.device != dev or n < 1
            or 2 * n > D):
        raise ValueError(f"rope: inv_freq must be fp32 (n,), 1 <= n <= {D // 2}, on q's device, got "
                         f"{tuple(inv_freq.shape)} {inv_freq.dtype}")
    Hkv = 0
    if k is not None:
        if (not isinstance(k, torch.Tensor) or k.dim() != 4 or k.dtype != dtype or k.device != dev
                or k.shape[0] != B or k.shape[1] != T or k.shape[3] != D):
            raise ValueError(f"rope: k must be (B, T, H, D) with q's B, T, D = {(B, T, D)}, dtype "
                             f"and device, got {k}")
        Hkv = k.shape[2]
    if torch.is_grad_enabled() and (q.requires_grad or inv_freq.requires_grad
                                    or (k is not None and k.requires_grad)):
        raise RuntimeError("rope is forward-only: autograd / gradient inputs are not supported; "
                           "call it under torch.no_grad() (inverse=True is its gradient)")
    at = steps = None
    wide = 0
    if positions is not None:
        if (not isinstance(positions, torch.Tensor) or positions.device != dev
                or positions.dtype not in (torch.int32, torch.int64)
                or positions.shape not in ((B, T), (T,))):
            raise ValueError(f"rope: positions must be int32 or int64 ({B}, {T}) or ({T},) on q's "
                             "device")
        steps = positions.stride()
        steps = _strides2(steps if len(steps) == 2 else (0,) + steps)
        at, wide = positions.data_ptr(), int(positions.dtype == torch.int64)
    elif not -2 ** 53 <= offset <= 2 ** 53 - max(T - 1, 0):
        raise ValueError(f"rope: offset {offset}: positions must be within 2^53")
    if Hkv and not Hq:
        raise ValueError("rope: q has no heads")
    if q.stride(3) != 1:
        q = q.contiguous()
    if inv_freq.stride(0) != 1:
        inv_freq = inv_freq.contiguous()
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = k_at = k_to = k_strides = k_dense = None
    if k is not None:
        if k.stride(3) != 1:
            k = k.contiguous()
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
        if Hkv:
            k_at, k_to = k.data_ptr(), k_out.data_ptr()
            k_strides, k_dense = _strides4(k.stride()), _strides4(k_out.stride())
    if B and T and Hq:
        _lib.call(q, _lib.lib().ttcd_rope_fwd, q.data_ptr(), k_at, q_out.data_ptr(), k_to,
                  inv_freq.data_ptr(), n, at, wide, steps, offset, B, T, Hq, Hkv, D,
                  _strides4(q.stride()), k_strides, _strides4(q_out.stride()), k_dense,
                  int(interleaved), int(inverse), scale, code)
    return q_out if k is None else (q_out, k_out)

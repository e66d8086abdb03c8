"""A key / value cache held in 4 bits and the calls on it (host side of kv4.hip).

    KV4Cache(batch, kv_heads, head_dim, capacity, dtype)
        the cache: 4.25 bits a value, the last `capacity` positions of each
        sequence, the lengths on the GPU
    kv4_append(cache, k, v)                 new keys and values
    kv4_attn(q, cache, window)              attention of the newest positions
    kv4_key_weights(q, cache, lse, window)  the attention weight of each key
    kv4_evict(cache, weights, keep, recent) the cache without the least of them
    kv4_read(cache, count)                  the held values
    kv4_tree_attn(q, cache, draft, parents) attention of a tree of drafted tokens, whose
        own keys and values are in a second cache
    kv4_commit(cache, draft, path, counts)  accepted ones move into the cache

The reference keeps bf16 keys and values (fla's attn_state, fla/models/utils.py:
35-96) and has no counterpart; window conventions are those of window_attn
(flash-attention's (W-1, 0)), queries sit bottom-right aligned at the last
positions of their sequence, and the softmax scale is head_dim ** -0.5.

A sequence is prefilled and decoded by one append and one attention call per
step and layer; nothing is copied or moved as it grows, a full cache goes on as
a ring, and the calls read the lengths on the GPU, so a step can be captured
into a graph and replayed. ``counts`` (int32, (batch,), on the GPU) makes a call
one of a padded batch: sequence b has the first counts[b] of the T positions
given.

Like the other attention calls these are forward-only, launch on torch's
current stream, allocate only their outputs and workspace and never
synchronise. A call that writes a cache must be ordered (by its stream) against
the others on it.
"""
from __future__ import annotations

import ctypes
from functools import lru_cache

import torch

from . import _lib
from .attn import _DT, _ready as _packed

BLOCK = 32  # channels that share a scale, and what a capacity is a multiple of


class KV4Cache:
    """Keys and values of `batch` sequences in 4 bits: blocks of 32 channels share a
    power of two, a value is one of +-(0, 0.5, 1, 1.5, 2, 3, 4, 6) times that
    (include/ttcd.h tells the layout). `capacity`: positions that are held, a
    multiple of 32. `dtype` (bf16 or f16): that of the keys, values and queries.
    `weights`: also keep ``self.weights``, (batch, kv_heads, capacity) fp32, the
    attention weight of each slot's key, for kv4_key_weights to add to and
    kv4_evict to go by; an append sets it to 0 in the slots it writes."""

    def __init__(self, batch: int, kv_heads: int, head_dim: int, capacity: int,
                 dtype: torch.dtype = torch.bfloat16, device="cuda", weights: bool = False):
        B, H, D, C = int(batch), int(kv_heads), int(head_dim), int(capacity)
        if B < 1 or H < 1:
            raise ValueError(f"KV4Cache: need batch, kv_heads >= 1, got {B}, {H}")
        if D not in (64, 128):
            raise ValueError(f"KV4Cache: head_dim must be 64 or 128, got {D}")
        if C < BLOCK or C % BLOCK:
            raise ValueError(f"KV4Cache: capacity must be a multiple of {BLOCK}, got {C}")
        if dtype not in _DT:
            raise ValueError(f"KV4Cache: dtype {dtype} not supported (bfloat16 or float16)")
        self._alloc(B, H, D, C, dtype, device)
        self.lengths.zero_()
        self.weights = (torch.zeros(B, H, C, dtype=torch.float32, device=self.device)
                        if weights else None)

    def _alloc(self, B, H, D, C, dtype, device) -> None:
        """The parts in one allocation, the lengths not set."""
        n = B * H * C
        codes, scales = n * D // 2, n * D // BLOCK  # multiples of 512 and 32
        blob = torch.empty(2 * (codes + scales) + 4 * B, dtype=torch.uint8, device=device)
        if not blob.is_cuda:
            raise ValueError("KV4Cache: device must be a GPU (HIP) device")
        p = blob.data_ptr()
        self._blob, self._parts = blob, None
        self._bind(p, p + 2 * codes, p + codes, p + 2 * codes + scales,
                   p + 2 * (codes + scales), B, H, D, C, dtype, blob.device)
        self.weights = None

    def _bind(self, kc, ks, vc, vs, lengths, B, H, D, C, dtype, device) -> None:
        self.batch, self.kv_heads, self.head_dim, self.capacity = B, H, D, C
        self.dtype, self.device = dtype, device
        self._c = _lib.KV4CacheStruct(kc, ks, vc, vs, lengths, B, H, D, C)
        self._ref = ctypes.byref(self._c)

    @classmethod
    def from_parts(cls, k_codes: torch.Tensor, k_scales: torch.Tensor, v_codes: torch.Tensor,
                   v_scales: torch.Tensor, lengths: torch.Tensor,
                   dtype: torch.dtype = torch.bfloat16,
                   weights: torch.Tensor | None = None) -> "KV4Cache":
        """The cache that these tensors are (shared, not copied)."""
        if not isinstance(k_codes, torch.Tensor) or k_codes.dim() != 4:
            raise ValueError("KV4Cache: k_codes must be (B, H, C, D / 2)")
        B, H, C, half = k_codes.shape
        D = 2 * half
        if dtype not in _DT:
            raise ValueError(f"KV4Cache: dtype {dtype} not supported (bfloat16 or float16)")
        if D not in (64, 128) or C < BLOCK or C % BLOCK or B < 1 or H < 1:
            raise ValueError(f"KV4Cache: head_dim must be 64 or 128 and capacity a multiple of "
                             f"{BLOCK}, got {tuple(k_codes.shape)}")
        dev, u8 = k_codes.device, torch.uint8
        if (k_scales.shape != (B, H, C, D // 32) or v_codes.shape != (B, H, C // 4, D // 8, 4, 4)
                or v_scales.shape != (B, H, C // 4, D // 32, 4) or lengths.shape != (B,)
                or k_codes.dtype != u8 or k_scales.dtype != u8 or v_codes.dtype != u8
                or v_scales.dtype != u8 or lengths.dtype != torch.int32
                or (weights is not None and (weights.shape != (B, H, C)
                                             or weights.dtype != torch.float32))):
            raise ValueError("KV4Cache: shapes or types of the parts are not those of a cache of "
                             f"(B, H, C, D) = {(B, H, C, D)}")
        parts = (k_codes, k_scales, v_codes, v_scales, lengths)
        for t in parts if weights is None else parts + (weights,):
            if t.device != dev or not t.is_contiguous():
                raise ValueError(f"KV4Cache: the parts must be contiguous and on {dev}")
        if dev.type != "cuda":
            raise ValueError("KV4Cache: the parts must be on a GPU (HIP) device")
        self = cls.__new__(cls)
        self._blob = None
        self._parts = parts
        self._bind(k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(),
                   v_scales.data_ptr(), lengths.data_ptr(), B, H, D, C, dtype, dev)
        self.weights = weights
        return self

    def _part(self, i: int) -> torch.Tensor:
        if self._parts is None:
            B, H, D, C = self.batch, self.kv_heads, self.head_dim, self.capacity
            shapes = ((B, H, C, D // 2), (B, H, C // 4, D // 8, 4, 4), (B, H, C, D // BLOCK),
                      (B, H, C // 4, D // BLOCK, 4))
            sizes = [B * H * C * D // n for n in (2, 2, BLOCK, BLOCK)]
            kc, vc, ks, vs, n = self._blob.split(sizes + [4 * B])
            kc, vc, ks, vs = (t.view(s) for t, s in zip((kc, vc, ks, vs), shapes))
            self._parts = (kc, ks, vc, vs, n.view(torch.int32))
        return self._parts[i]

    @property
    def k_codes(self) -> torch.Tensor:
        return self._part(0)

    @property
    def k_scales(self) -> torch.Tensor:
        return self._part(1)

    @property
    def v_codes(self) -> torch.Tensor:
        return self._part(2)

    @property
    def v_scales(self) -> torch.Tensor:
        return self._part(3)

    @property
    def lengths(self) -> torch.Tensor:
        """Positions that each sequence has had, int32 (batch,); past 2^30 less a multiple
        of the capacity (at least that many remain)."""
        return self._part(4)

    @property
    def weights(self) -> torch.Tensor | None:
        """The slots' attention weights, (batch, kv_heads, capacity) fp32, if they are kept."""
        return self._weights

    @weights.setter
    def weights(self, w: torch.Tensor | None) -> None:
        shape = (self.batch, self.kv_heads, self.capacity)
        if w is not None and (not isinstance(w, torch.Tensor) or w.shape != shape
                              or w.dtype != torch.float32 or w.device != self.device
                              or not w.is_contiguous()):
            raise ValueError(f"KV4Cache: weights must be contiguous fp32 {shape} on {self.device}")
        if w is not None:
            _forward_only(w, "KV4Cache")
        self._weights = w

    def reset(self) -> None:
        """Forget every position."""
        with torch.inference_mode():  # a cache made in inference mode is reset outside it too
            self.lengths.zero_()
            if self.weights is not None:
                self.weights.zero_()


def _cache(cache, fn: str) -> KV4Cache:
    if not isinstance(cache, KV4Cache):
        raise ValueError(f"{fn}: cache must be a KV4Cache")
    return cache


def _forward_only(t: torch.Tensor, fn: str) -> None:
    if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{fn} is forward-only: autograd / gradient inputs are not supported; "
                           "call it under torch.no_grad() or torch.inference_mode()")


def _rows(t, cache: KV4Cache, name: str, fn: str, heads: int | None) -> None:
    """The checks of a (B, T, heads, D) operand (heads None: any multiple of the cache's)."""
    if not isinstance(t, torch.Tensor) or t.dim() != 4:
        raise ValueError(f"{fn}: {name} must be a 4-D tensor (B, T, H, D)")
    B, _, H, D = t.shape
    if B != cache.batch or D != cache.head_dim or (
            H != heads if heads is not None else H < 1 or H % cache.kv_heads):
        raise ValueError(f"{fn}: {name} {tuple(t.shape)} does not match a cache of batch "
                         f"{cache.batch}, {cache.kv_heads} kv heads, head_dim {cache.head_dim}")
    if t.dtype != cache.dtype:
        raise ValueError(f"{fn}: {name} must be {cache.dtype} as the cache, got {t.dtype}")
    if t.device != cache.device:
        raise ValueError(f"{fn}: {name} must be on the cache's device")
    _forward_only(t, fn)


def _counts(counts, cache: KV4Cache, fn: str):
    if counts is None:
        return None
    if (not isinstance(counts, torch.Tensor) or counts.shape != (cache.batch,)
            or counts.dtype != torch.int32 or counts.device != cache.device):
        raise ValueError(f"{fn}: counts must be int32 ({cache.batch},) on the cache's device")
    return counts.contiguous()


def _overlap(a: torch.Tensor, b: torch.Tensor | None) -> bool:
    """Whether two contiguous tensors share memory."""
    if b is None:
        return False
    x, y = a.data_ptr(), b.data_ptr()
    return x < y + b.numel() * b.element_size() and y < x + a.numel() * a.element_size()


def _ptr(t):
    return None if t is None else t.data_ptr()


# stride arrays (only read) of the last calls: finding one is quicker than making it
_strides = lru_cache(maxsize=64)(_lib.strides4)


@lru_cache(maxsize=64)
def _dense(T: int, H: int, D: int):
    return _lib.strides4((T * H * D, H * D, D, 1))


def _operand(t: torch.Tensor):
    """(t, or a copy, with rows as the C entries take them, its stride array). A
    contiguous t's dimensions of 1 may have any stride, and it may start off 16 bytes."""
    if not t.is_contiguous():
        x = _packed(t)
        if x is t:
            return t, _strides(t.stride())
        t = x
    if t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t, _dense(t.shape[1], t.shape[2], t.shape[3])


def _window(window) -> int:
    return 0 if window is None or window < 0 else int(min(window, 2**31 - 1))


def kv4_append(cache: KV4Cache, k: torch.Tensor, v: torch.Tensor, *,
               counts: torch.Tensor | None = None) -> None:
    """Quantise k, v (B, T, Hkv, D) into the cache as the next T positions of every
    sequence (the next counts[b] of sequence b) and add them to its lengths.
    T <= capacity. Any strides; rows of 16-byte alignment are read in place."""
    _cache(cache, "kv4_append")
    _rows(k, cache, "k", "kv4_append", cache.kv_heads)
    _rows(v, cache, "v", "kv4_append", cache.kv_heads)
    if k.shape != v.shape:
        raise ValueError(f"kv4_append: k {tuple(k.shape)} and v {tuple(v.shape)} differ")
    counts = _counts(counts, cache, "kv4_append")
    T = k.shape[1]
    if T > cache.capacity:
        raise ValueError(f"kv4_append: {T} positions into a cache of {cache.capacity}")
    if T == 0:
        return
    (k, ks), (v, vs) = _operand(k), _operand(v)
    _lib.call(cache, _lib.lib().ttcd_kv4_append, cache._ref, k.data_ptr(), v.data_ptr(), T,
          ks, vs, _ptr(counts),
          _ptr(cache.weights), _DT[cache.dtype])


def kv4_read(cache: KV4Cache, count: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(k, v), each (B, count, Hkv, D): the last `count` positions of every sequence
    as the values that the cache holds for them, the newest last; 0 in rows before
    the first held position."""
    _cache(cache, "kv4_read")
    count = int(count)
    if count < 0:
        raise ValueError(f"kv4_read: count must be >= 0, got {count}")
    k = torch.empty(cache.batch, count, cache.kv_heads, cache.head_dim, dtype=cache.dtype,
                    device=cache.device)
    v = torch.empty_like(k)
    if count:
        _lib.call(cache, _lib.lib().ttcd_kv4_read, cache._ref, k.data_ptr(), v.data_ptr(), count,
              _DT[cache.dtype])
    return k, v


def kv4_attn(q: torch.Tensor, cache: KV4Cache, window: int | None = None, *,
             counts: torch.Tensor | None = None, return_lse: bool = False,
             split_keys: bool = True):
    """Attention of q (B, Tq, H, D), the last Tq positions of every sequence (the last
    counts[b] of sequence b, in q's first rows), over the held keys of the `window`
    (None or < 0: all) positions up to each query's own; append their keys first.
    H a multiple of the cache's kv heads. Returns o like q, and with
    ``return_lse`` lse, fp32 natural-log (B, H, Tq). Rows without a key, and rows
    from counts[b] on, get o = 0 and lse = -inf. ``split_keys=False`` keeps every
    row's sums in one workgroup: they then do not depend on the capacity."""
    _cache(cache, "kv4_attn")
    _rows(q, cache, "q", "kv4_attn", None)
    counts = _counts(counts, cache, "kv4_attn")
    if window is not None and window == 0:
        raise ValueError("kv4_attn: window must be >= 1, or None / < 0 for none")
    B, T, H, D = q.shape
    q, qs = _operand(q)
    o = torch.empty(B, T, H, D, dtype=q.dtype, device=q.device)
    lse = torch.empty(B, H, T, dtype=torch.float32, device=q.device) if return_lse else None
    if T > 0:
        L, W = _lib.lib(), _window(window)
        n = L.ttcd_kv4_attn_workspace_bytes(cache._ref, T, H, W) if split_keys else 0
        work = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
        _lib.call(cache, L.ttcd_kv4_attn_fwd, cache._ref, q.data_ptr(), o.data_ptr(), _ptr(lse), T, H,
              qs, _dense(T, H, D), _ptr(counts), W, D ** -0.5,
              _DT[q.dtype], _ptr(work), n)
    return (o, lse) if return_lse else o


def kv4_key_weights(q: torch.Tensor, cache: KV4Cache, lse: torch.Tensor,
                    window: int | None = None, *, counts: torch.Tensor | None = None,
                    out: torch.Tensor | None = None, accumulate: bool = False) -> torch.Tensor:
    """(B, Hkv, capacity) fp32, by slot: the attention weight that each held key got
    from the queries of a kv4_attn call, summed over them and over the query heads of
    its kv head; lse is that call's. ``out`` receives it (``accumulate``: is added
    to, ``out=cache.weights`` for a cache that keeps them)."""
    _cache(cache, "kv4_key_weights")
    _rows(q, cache, "q", "kv4_key_weights", None)
    counts = _counts(counts, cache, "kv4_key_weights")
    if window is not None and window == 0:
        raise ValueError("kv4_key_weights: window must be >= 1, or None / < 0 for none")
    B, T, H, D = q.shape
    if (not isinstance(lse, torch.Tensor) or lse.shape != (B, H, T)
            or lse.dtype != torch.float32 or lse.device != q.device):
        raise ValueError(f"kv4_key_weights: lse must be fp32 ({B}, {H}, {T}) on q's device")
    _forward_only(lse, "kv4_key_weights")
    shape = (B, cache.kv_heads, cache.capacity)
    if out is None:
        if accumulate:
            raise ValueError("kv4_key_weights: accumulate needs out")
        out = torch.empty(shape, dtype=torch.float32, device=q.device)
    elif (not isinstance(out, torch.Tensor) or out.shape != shape or out.dtype != torch.float32
          or out.device != q.device or not out.is_contiguous() or out.data_ptr() % 16):
        raise ValueError(f"kv4_key_weights: out must be contiguous fp32 {shape} on q's device, "
                         "16-byte aligned")
    _forward_only(out, "kv4_key_weights")
    if T == 0:
        with torch.inference_mode():
            return out if accumulate else out.zero_()
    (q, qs), lse = _operand(q), lse.contiguous()
    _lib.call(cache, _lib.lib().ttcd_kv4_key_weights_fwd, cache._ref, q.data_ptr(), lse.data_ptr(),
          out.data_ptr(), T, H, qs, _ptr(counts), _window(window),
          D ** -0.5, int(bool(accumulate)), _DT[q.dtype])
    return out


def kv4_evict(cache: KV4Cache, weights: torch.Tensor | None, keep: int, recent: int = 0, *,
              out: KV4Cache | None = None):
    """The cache without the keys of least weight, per kv head: of n held positions
    min(n, keep) stay, the newest `recent` in any case and of the older ones those of
    the largest weight, ties to the oldest; NaN counts as less than any number.
    weights: (B, Hkv, capacity) fp32 by slot, None for the cache's own.

    Returns (new, index, new_weights): a cache of the same capacity (or ``out``, of
    a capacity >= keep) whose positions 0, 1, .. are the kept ones in their order;
    index (B, Hkv, keep) int32, the position that each had, -1 behind the last;
    and their weights by the new cache's slots, which are also ``new.weights`` if
    either cache keeps weights. The old cache stays as it is."""
    _cache(cache, "kv4_evict")
    weights = cache.weights if weights is None else weights
    keep, recent = int(keep), int(recent)
    B, H, C = cache.batch, cache.kv_heads, cache.capacity
    if (not isinstance(weights, torch.Tensor) or weights.shape != (B, H, C)
            or weights.dtype != torch.float32 or weights.device != cache.device):
        raise ValueError(f"kv4_evict: weights must be fp32 ({B}, {H}, {C}) on the cache's device")
    _forward_only(weights, "kv4_evict")
    if out is None:
        out = KV4Cache.__new__(KV4Cache)
        out._alloc(B, H, cache.head_dim, C, cache.dtype, cache.device)  # the call sets its lengths
    elif (not isinstance(out, KV4Cache) or out.dtype != cache.dtype
          or out.device != cache.device):
        raise ValueError("kv4_evict: out must be a KV4Cache of the cache's dtype and device")
    if keep < 1 or keep > out.capacity or recent < 0:
        raise ValueError(f"kv4_evict: need 1 <= keep <= {out.capacity} and recent >= 0, got "
                         f"{keep}, {recent}")
    weights = weights.contiguous()
    index = torch.empty(B, H, keep, dtype=torch.int32, device=cache.device)
    new_weights = out.weights
    # the weights that are read, and the old cache's, stay as they are
    if (new_weights is None or _overlap(new_weights, weights)
            or _overlap(new_weights, cache.weights)):
        new_weights = torch.empty(B, H, out.capacity, dtype=torch.float32, device=cache.device)
    _lib.call(cache, _lib.lib().ttcd_kv4_evict, cache._ref, weights.data_ptr(), keep,
          min(recent, 2**31 - 1), out._ref, new_weights.data_ptr(), index.data_ptr())
    if cache.weights is not None or out.weights is not None:
        out.weights = new_weights
    return out, index, new_weights


TREE_NODES = 256  # of a sequence, at most


def _draft(draft, cache: KV4Cache, fn: str) -> KV4Cache:
    if not isinstance(draft, KV4Cache):
        raise ValueError(f"{fn}: draft must be a KV4Cache")
    if (draft.batch != cache.batch or draft.kv_heads != cache.kv_heads
            or draft.head_dim != cache.head_dim or draft.dtype != cache.dtype
            or draft.device != cache.device):
        raise ValueError(f"{fn}: draft must have the cache's batch, kv heads, head_dim, dtype and "
                         "device")
    return draft


def _nodes(t, cache: KV4Cache, name: str, fn: str, n: int | None = None) -> torch.Tensor:
    if (not isinstance(t, torch.Tensor) or t.dim() != 2 or t.shape[0] != cache.batch
            or (n is not None and t.shape[1] != n) or t.dtype != torch.int32
            or t.device != cache.device):
        raise ValueError(f"{fn}: {name} must be int32 ({cache.batch}, "
                         f"{'N' if n is None else n}) on the cache's device")
    return t.contiguous()


def kv4_tree_attn(q: torch.Tensor, cache: KV4Cache, draft: KV4Cache, parents: torch.Tensor,
                  window: int | None = None, *, counts: torch.Tensor | None = None,
                  return_lse: bool = False, split_keys: bool = True):
    """Attention of the nodes of a tree of drafted tokens, q (B, N, H, D), N <= 256: node i
    follows node parents[b, i] < i ((B, N) int32; -1: none) and is at position length +
    depth, behind the cache's. It sees the cache's held keys of the `window` (None or < 0:
    all) positions up to its own and, within those, itself and its ancestors, which `draft`
    holds: kv4_append all nodes to an empty second cache first, node i is in its slot i
    (counts[b] of them: the first). So a chain of nodes sees what the same tokens would
    that kv4_append adds to the cache itself, where its capacity holds them beside what their
    windows reach (nodes drop no key), and the cache stays as it is until kv4_commit.
    Returns o like q, and with ``return_lse`` lse, fp32 natural-log (B, H, N); rows behind
    the last node get o = 0 and lse = -inf. ``split_keys`` as in kv4_attn."""
    fn = "kv4_tree_attn"
    _draft(draft, _cache(cache, fn), fn)
    _rows(q, cache, "q", fn, None)
    counts = _counts(counts, cache, fn)
    if window is not None and window == 0:
        raise ValueError(f"{fn}: window must be >= 1, or None / < 0 for none")
    B, N, H, D = q.shape
    parents = _nodes(parents, cache, "parents", fn, N)
    if N > TREE_NODES or N > draft.capacity:
        raise ValueError(f"{fn}: {N} nodes, need at most {min(TREE_NODES, draft.capacity)} (a "
                         f"draft's capacity, and {TREE_NODES})")
    q, qs = _operand(q)
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty(B, H, N, dtype=torch.float32, device=q.device) if return_lse else None
    if N > 0:
        L, W = _lib.lib(), _window(window)
        n = L.ttcd_kv4_tree_attn_workspace_bytes(cache._ref, N, H, W) if split_keys else 0
        work = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
        _lib.call(cache, L.ttcd_kv4_tree_attn_fwd, cache._ref, draft._ref, q.data_ptr(),
                  o.data_ptr(), _ptr(lse), N, H, qs, _dense(N, H, D), parents.data_ptr(),
                  _ptr(counts), W, D ** -0.5, _DT[q.dtype], _ptr(work), n)
    return (o, lse) if return_lse else o


def kv4_commit(cache: KV4Cache, draft: KV4Cache, path: torch.Tensor,
               counts: torch.Tensor | None = None, *, reset: bool = False) -> None:
    """The draft's slots path[b, :counts[b]] ((B, P) int32; counts None: all P) become the
    next positions of sequence b, the same bits, and its lengths count them. path's other
    entries may be anything. P at most the capacity of either. ``reset``: the draft is
    empty afterwards."""
    fn = "kv4_commit"
    _draft(draft, _cache(cache, fn), fn)
    path = _nodes(path, cache, "path", fn)
    counts = _counts(counts, cache, fn)
    P = path.shape[1]
    if P < 1 or P > min(cache.capacity, draft.capacity):
        raise ValueError(f"{fn}: need 1 to {min(cache.capacity, draft.capacity)} nodes (the "
                         f"capacities), got {P}")
    _lib.call(cache, _lib.lib().ttcd_kv4_commit, cache._ref, draft._ref, path.data_ptr(),
              _ptr(counts), P, _ptr(cache.weights), int(bool(reset)))

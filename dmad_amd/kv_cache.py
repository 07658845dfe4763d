"""A paged key-value cache for token-by-token and block-by-block inference on the gfx950 kernels.

``PagedKVCache`` holds the pages and what its sequences hold. Three calls work on it:

  * ``qk_norm_rope_append``: the new tokens' queries and keys are normalised per head and rotated
    (as ``qk_norm_rope_with_tangent`` does), keys and values go into the pages; ``append_kv`` is
    the same without queries, norm and rotation;
  * ``paged_attention``: attention of those queries over the cache, optionally adding up the
    attention weight every slot receives;
  * ``evict_low_weight``: cuts long sequences to their heaviest slots.

They run without derivatives (operands that carry any are refused), put only kernel launches on the current stream and read lengths and
page table on the device, so a captured step follows them. Nothing is copied to the host: what
the device holds is checked by the kernels (see ``PagedKVCache``). Device work only: tensors off
the GPU raise.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from . import _native as nat
from .jvp_attention import _eager_call
from .prologue import HEAD_DIMS, _check_same_device, _norm_weights, _weights_dtype, readable_rows, refuse_forward_mode


# torch.autograd.graph.increment_version of a list
_increment_version = torch._C._increment_version

CACHE_TENSORS = ("k_pages", "v_pages", "page_table", "lengths", "seen", "weight", "position")


def _cache_tensors(cache):
    return [getattr(cache, n) for n in CACHE_TENSORS]


class PagedKVCache:
    """Pages of keys and values, one page list per sequence.

    k_pages, v_pages  [N, Hk, P, D] bf16 or fp16; P a multiple of 16; D one of 16, 32, 64, 128, 256.
                      Any strides with contiguous rows and multiples of 8 elements: an
                      [N, P, Hk, D] pool is passed as its transpose(1, 2)
    page_table        [B, M] int32: slot s of sequence b is slot s % P of page page_table[b, s // P].
                      An id outside [0, N) (-1) marks a page that holds nothing: its slots are not
                      read or written and no query sees them, so a window may drop pages in front
    lengths           [B] int32, slots in use; values outside [0, M * P] count as the nearer end
    seen              [B] int32, tokens appended so far: the position of the next one. Equal to
                      lengths until something is evicted
    weight, position  [N, Hk, P] float32 and int32: each slot's accumulated attention weight and
                      its token's position; both or neither (None: no accumulation, no eviction)

    The tensors are used in place and stay the caller's: pages are handed out, shared or dropped
    by writing to ``page_table`` and ``lengths``. Where a tensor's memory is replaced (``t.data = ...``)
    the next call checks and uses the new one; a captured graph keeps the one it was captured with. A page may appear in several sequences as long
    as it is only read; pages that are appended to, evicted from or whose weights are accumulated
    belong to one sequence, whose row names them once. ``lengths`` and ``seen``, or ``k_pages`` and
    ``v_pages``, may be one memory only where nothing is appended or evicted. Calls that only read a cache may run on several streams at once; one
    that appends, accumulates or evicts is ordered by the caller against all others, as with any
    tensor changed in place. Such calls count as changes in place for autograd: a backward pass that
    needs what they overwrote raises.
    """

    def __init__(self, k_pages, v_pages, page_table, lengths, seen, weight=None, position=None):
        self.k_pages, self.v_pages, self.page_table = k_pages, v_pages, page_table
        self.lengths, self.seen, self.weight, self.position = lengths, seen, weight, position
        self._describe()

    def _describe(self):
        """Checks the tensors and fills the kernels' view of them."""
        op = "PagedKVCache"
        k_pages, v_pages, page_table, lengths, seen, weight, position = _cache_tensors(self)
        device = _check_same_device(op, k_pages, v_pages, page_table, lengths, seen, weight, position)
        if k_pages.dim() != 4 or v_pages.shape != k_pages.shape:
            raise ValueError(f"{op}: k_pages and v_pages must be [N, Hk, P, D], got {tuple(k_pages.shape)} and "
                             f"{tuple(v_pages.shape)}")
        if k_pages.dtype not in (torch.bfloat16, torch.float16) or v_pages.dtype != k_pages.dtype:
            raise NotImplementedError(f"{op}: pages must be bfloat16 or float16, got {k_pages.dtype} and {v_pages.dtype}")
        N, Hk, P, D = k_pages.shape
        if D not in HEAD_DIMS:
            raise NotImplementedError(f"{op}: head dim {D} is not one of {HEAD_DIMS}")
        if P < 16 or P % 16:
            raise NotImplementedError(f"{op}: the page size must be a multiple of 16, got {P}")
        if N < 1 or Hk < 1:
            raise ValueError(f"{op}: an empty pool {tuple(k_pages.shape)}")
        if page_table.dim() != 2 or page_table.dtype != torch.int32 or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
            raise ValueError(f"{op}: page_table must be [B, M] int32 with contiguous rows")
        B, M = page_table.shape
        for name, t in (("lengths", lengths), ("seen", seen)):
            if t.shape != (B,) or t.dtype != torch.int32 or not t.is_contiguous():
                raise ValueError(f"{op}: {name} must be [{B}] int32, contiguous")
        if (weight is None) != (position is None):
            raise ValueError(f"{op}: weight and position together, or neither")
        for name, t, dtype in (("weight", weight, torch.float32), ("position", position, torch.int32)):
            if t is not None and (t.shape != (N, Hk, P) or t.dtype != dtype or not t.is_contiguous() or t.data_ptr() % 16):
                raise ValueError(f"{op}: {name} must be [{N}, {Hk}, {P}] {dtype}, contiguous and 16-byte aligned")

        for name, t in zip(CACHE_TENSORS, (k_pages, v_pages, page_table, lengths, seen, weight, position)):
            if t is not None and (t.is_neg() or (t.numel() and not t.data_ptr())):
                raise ValueError(f"{op}: {name} has no memory that holds its values")

        def strides(name, t):
            if t.stride(3) != 1 or t.data_ptr() % 16:
                raise ValueError(f"{op}: rows of {name} must be contiguous and 16-byte aligned")
            st = [D if n == 1 else s for n, s in zip(t.shape[:3], t.stride()[:3])]
            if any(s % 8 or s < D for s in st):
                raise ValueError(f"{op}: strides of {name} must be multiples of 8 elements and at least {D}, got {t.stride()}")
            return (ctypes.c_int64 * 3)(*st)

        c = nat.KvCache(N, Hk, P, D, B, M, nat.ptr(k_pages), nat.ptr(v_pages), strides("k_pages", k_pages),
                        strides("v_pages", v_pages), nat.ptr(page_table), page_table.stride(0) if B > 1 else M,
                        nat.ptr(lengths), nat.ptr(seen), nat.ptr(weight), nat.ptr(position))
        tensors = [t for t in _cache_tensors(self) if t is not None]
        # one memory for two of them serves a cache that is only read
        shared = ""
        if B and abs(lengths.data_ptr() - seen.data_ptr()) < 4 * B:
            shared = "lengths and seen"
        elif k_pages.data_ptr() == v_pages.data_ptr():
            shared = "k_pages and v_pages"
        described = dict(
            device=device, dtype=k_pages.dtype, batch=B, kv_heads=Hk, page_size=P, head_dim=D, capacity=M * P, _c=c,
            _code=nat.dtype_code(k_pages.dtype), _sizes={}, _pointers=[t.data_ptr for t in tensors],
            _addresses=[t.data_ptr() for t in tensors],
            # their new_empty takes half the host time of torch.empty with a device and a type
            _bytes=torch.empty(0, device=device, dtype=torch.uint8), _floats=torch.empty(0, device=device, dtype=torch.float32),
            # what each call changes, for autograd (which keeps no count of inference tensors)
            _written={by: [t for t in ts if t is not None and not t.is_inference()] for by, ts in (
                ("append", (k_pages, v_pages, lengths, seen, weight, position)), ("attend", (weight,)),
                ("evict", (k_pages, v_pages, lengths, weight, position)))},
            _shared=shared, _ref=ctypes.byref(c))
        self.__dict__.update(described)

    def _settle(self):
        """Follows tensors whose memory was replaced since (``t.data = ...``, a storage that was resized)."""
        if torch.compiler.is_compiling():
            return  # the registered ops describe the tensors that they are given
        if [pointer() for pointer in self._pointers] != self._addresses:
            self._describe()

    def __setattr__(self, name, value):
        if hasattr(self, "_ref"):
            raise AttributeError(f"PagedKVCache.{name} cannot be replaced: write into the tensors in place")
        object.__setattr__(self, name, value)

    @classmethod
    def allocate(cls, batch, capacity, kv_heads, head_dim, dtype=torch.bfloat16, device="cuda", page_size=64,
                 track_weights=True):
        """An empty cache of ``batch`` sequences of up to ``capacity`` slots (rounded up to whole
        pages), each with its own pages in order. ``track_weights``: room for weights and positions."""
        if batch < 1 or capacity < 1 or kv_heads < 1:
            raise ValueError(f"PagedKVCache.allocate: batch {batch}, capacity {capacity}, kv_heads {kv_heads}")
        if page_size < 16 or page_size % 16:
            raise NotImplementedError(f"PagedKVCache: the page size must be a multiple of 16, got {page_size}")
        M = -(-capacity // page_size)
        N = batch * M
        pages = (N, kv_heads, page_size)
        return cls(
            torch.empty((*pages, head_dim), device=device, dtype=dtype),
            torch.empty((*pages, head_dim), device=device, dtype=dtype),
            torch.arange(N, device=device, dtype=torch.int32).view(batch, M),
            torch.zeros(batch, device=device, dtype=torch.int32),
            torch.zeros(batch, device=device, dtype=torch.int32),
            torch.zeros(pages, device=device, dtype=torch.float32) if track_weights else None,
            torch.zeros(pages, device=device, dtype=torch.int32) if track_weights else None,
        )

    def _writable(self, op):
        if self._shared:
            raise ValueError(f"{op}: {self._shared} of the cache share memory, and each is written")

    def _changed(self, by):
        """The launches of an ordinary eager call write through addresses: counted as changes in place here."""
        _increment_version(self._written[by])

    def _workspace(self, query, *args):
        """(pointer, size, owner) of a fresh workspace whose size ``query`` gives, asked once per call's sizes."""
        size = self._sizes.get(args)
        if size is None:
            size = self._sizes[args] = query(self._c, *args)
        if size == 0:
            return None, 0, None
        ws = self._bytes.new_empty(size)
        return ws.data_ptr(), size, ws


def _on_cache(op, cache, t):
    if t is not None and t.device != cache.device:
        _check_same_device(op, t)
        raise ValueError(f"{op}: tensors on {t.device}, the cache on {cache.device}")


def _check_new(op, cache, *named):
    """Shapes of new tokens' q, k, v against the cache."""
    if not isinstance(cache, PagedKVCache):
        raise TypeError(f"{op}: cache must be a PagedKVCache, got {type(cache).__name__}")
    cache._settle()
    tokens = None
    for n, t in named:
        if t is None:
            continue
        _on_cache(op, cache, t)
        shape = t.shape
        if len(shape) == 4:
            B, S, H, D = shape
            tokens = S if tokens is None else tokens
        if len(shape) != 4 or B != cache.batch or D != cache.head_dim or S != tokens:
            raise ValueError(f"{op}: {n} must be [{cache.batch}, S, H, {cache.head_dim}], got {tuple(shape)}")
        if t.dtype != cache.dtype:
            raise ValueError(f"{op}: {n} is {t.dtype}, the cache {cache.dtype}")
        if n != "q" and H != cache.kv_heads:
            raise ValueError(f"{op}: {n} has {H} heads, the cache {cache.kv_heads}")


def _no_grad_only(op, cache, *ts):
    if torch.is_grad_enabled():
        for t in (cache.k_pages, cache.v_pages, cache.weight, *ts):
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{op} has no backward: call it under torch.no_grad()")


# Each call as a registered op, for whatever watches or replaces operators (compilers, dispatch modes, the profiler)
# and for operands whose memory does not hold their values. An ordinary eager call does not go through them.
@torch.library.custom_op("dmad::qk_norm_rope_append",
                         mutates_args=("k_pages", "v_pages", "lengths", "seen", "weight", "position"))
def _append_op(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, q_weight: Optional[torch.Tensor],
               k_weight: Optional[torch.Tensor], eps: float, freqs: Optional[torch.Tensor], k_pages: torch.Tensor,
               v_pages: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, seen: torch.Tensor,
               weight: Optional[torch.Tensor], position: Optional[torch.Tensor]) -> torch.Tensor:
    """q' of ``qk_norm_rope_append`` (0 elements without q)."""
    cache = PagedKVCache(k_pages, v_pages, page_table, lengths, seen, weight, position)
    _check_append(q, k, v, q_weight, k_weight, eps, freqs, cache)
    out = _append(q, k, v, q_weight, k_weight, eps, freqs, cache)
    return k.new_empty((0,)) if out is None else out


@_append_op.register_fake
def _(q, k, v, q_weight, k_weight, eps, freqs, *cache):
    return k.new_empty((0,) if q is None else q.shape)


@torch.library.custom_op("dmad::paged_attn", mutates_args=("weight",))
def _attend_op(q: torch.Tensor, sm_scale: float, causal: bool, k_pages: torch.Tensor, v_pages: torch.Tensor,
               page_table: torch.Tensor, lengths: torch.Tensor, seen: torch.Tensor, weight: Optional[torch.Tensor],
               position: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor]:
    """(o, lse) of ``paged_attention``; adds to ``weight`` where it is given."""
    cache = PagedKVCache(k_pages, v_pages, page_table, lengths, seen, weight, position)
    return _attend(q, cache, _check_attend(q, cache, sm_scale, weight is not None), causal, weight is not None)


@_attend_op.register_fake
def _(q, sm_scale, causal, *cache):
    B, S, Hq, _ = q.shape
    return q.new_empty(q.shape), q.new_empty((B, Hq, S), dtype=torch.float32)


@torch.library.custom_op("dmad::kv_evict", mutates_args=("k_pages", "v_pages", "lengths", "weight", "position"))
def _evict_op(keep: int, recent: int, sink: int, k_pages: torch.Tensor, v_pages: torch.Tensor, page_table: torch.Tensor,
              lengths: torch.Tensor, seen: torch.Tensor, weight: torch.Tensor, position: torch.Tensor) -> None:
    """``evict_low_weight``."""
    cache = PagedKVCache(k_pages, v_pages, page_table, lengths, seen, weight, position)
    _check_evict(cache, keep, recent, sink)
    _evict(cache, keep, recent, sink)


@_evict_op.register_fake
def _(keep, recent, sink, *cache):
    return None


_APPEND = "qk_norm_rope_append"


def _check_append(q, k, v, q_weight, k_weight, eps, freqs, cache):
    """Refuses what an append does not take (the weights' types apart, which the launch looks at)."""
    op = _APPEND
    if k is None or v is None:
        raise ValueError(f"{op}: k and v must be given")
    _check_new(op, cache, ("k", k), ("v", v), ("q", q))
    cache._writable(op)
    for t in (q_weight, k_weight, freqs):
        _on_cache(op, cache, t)
    _no_grad_only(op, cache, q, k, v, q_weight, k_weight, freqs)
    if not eps >= 0:
        raise ValueError(f"{op}: eps must be non-negative, got {eps}")
    if q is None and q_weight is not None:
        raise ValueError(f"{op}: q_weight without q")
    D = cache.head_dim
    if freqs is not None and (freqs.dim() != 2 or freqs.shape[1] != D // 2 or freqs.shape[0] < 1):
        raise ValueError(f"{op}: freqs must be [positions, {D // 2}], got {tuple(freqs.shape)}")


def qk_norm_rope_append(q, k, v, q_weight, k_weight, eps, freqs, cache):
    """Appends S new tokens to every sequence of the cache and returns their queries.

    q [B, S, Hq, D] comes back normalised per head and rotated, k [B, S, Hk, D] goes into the cache
    so, v [B, S, Hk, D] as it is. The tokens take the slots after ``cache.lengths`` and the positions
    from ``cache.seen`` on; then both advance by S. ``freqs`` [T, D/2] are angles by position, shared
    by the sequences: a token whose position has no row gets NaN in q and k. A weight of None skips
    that norm, freqs None the rotation. New slots start with weight 0. Tokens beyond the capacity
    are dropped (``lengths`` stays at it, ``seen`` advances), and those whose page holds nothing.
    """
    eps = float(eps)
    _check_append(q, k, v, q_weight, k_weight, eps, freqs, cache)
    if _eager_call(q, k, v, q_weight, k_weight, freqs):
        out = _append(q, k, v, q_weight, k_weight, eps, freqs, cache)
        cache._changed("append")
        return out
    _weights_dtype(_APPEND, k, cache.head_dim, q_weight, k_weight)
    refuse_forward_mode(_APPEND, q, k, v, q_weight, k_weight, freqs, *_cache_tensors(cache))
    out = torch.ops.dmad.qk_norm_rope_append(q, k, v, q_weight, k_weight, eps, freqs, *_cache_tensors(cache))
    return None if q is None else out


def _append(q, k, v, q_weight, k_weight, eps, freqs, cache):
    """The launch."""
    S, Hq = k.shape[1], 0 if q is None else q.shape[2]
    cq, ck, wcode = _norm_weights(_APPEND, k, cache.head_dim, q_weight, k_weight)
    if freqs is not None and (freqs.dtype != torch.float32 or not freqs.is_contiguous()):
        freqs = freqs.to(torch.float32).contiguous()
    out = None if q is None else torch.empty_like(q, memory_format=torch.contiguous_format)
    if Hq == 0:
        q = None
    ops = [(None, None) if t is None else readable_rows(t) for t in (q, k, v)]
    with nat.on_device(cache.device):
        nat.check(nat.lib().dmad_qk_norm_rope_append(
            cache._code, wcode, S, Hq, *(nat.ptr(t) for t, _ in ops), *(s for _, s in ops),
            nat.ptr(cq if q is not None else None), nat.ptr(ck), nat.ptr(freqs), 0 if freqs is None else freqs.shape[0],
            eps, nat.ptr(out), cache._ref, nat.stream_ptr(cache.device)))
    return out


def append_kv(k, v, cache):
    """Appends k and v [B, S, Hk, D] to the cache as they are (see ``qk_norm_rope_append``)."""
    qk_norm_rope_append(None, k, v, None, None, 0.0, None, cache)


def _check_attend(q, cache, sm_scale, accumulate):
    """Refuses what the attention does not take; the scale."""
    op = "paged_attention"
    _check_new(op, cache, ("q", q))
    _no_grad_only(op, cache, q)
    Hq = q.shape[2]
    if Hq < 1 or Hq % cache.kv_heads:
        raise ValueError(f"{op}: {Hq} query heads are not a multiple of the cache's {cache.kv_heads}")
    scale = cache.head_dim ** -0.5 if sm_scale is None else float(sm_scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise NotImplementedError(f"{op}: sm_scale must be positive and finite, got {sm_scale}")
    if accumulate and cache.weight is None:
        raise ValueError(f"{op}: the cache keeps no weights to accumulate")
    return scale


def paged_attention(q, cache, sm_scale=None, causal=False, accumulate=False, return_lse=False):
    """Attention of q [B, S, Hq, D] over each sequence's cache: o [B, S, Hq, D] (and lse [B, Hq, S]).

    Made for few new tokens (S = 1, a draft of a few, a small block): the work is split over the
    cache's length, and K and V are read once per 32 query rows (16 at 256-wide heads) of a key
    head. Up to 32 rows that costs what one does; a block of 1560 tokens takes 20 times as long.
    The softmax weights are rounded to the operands' type for their product with V (their sum, the
    scores and lse are float32). Hq is a multiple of the cache's heads; query head h reads key head
    h // (Hq // Hk). ``sm_scale`` defaults to D^-1/2. Every token sees all slots in use;
    with ``causal`` the S tokens are the last S slots (just appended, none dropped for want of room,
    nothing evicted since) and each sees the slots up to its own. A token that sees no slot gets o = 0 and lse = -inf, and so
    does one whose scores are all -inf. What a slot that a token does not see holds, infinities and
    NaN among it, does not reach the token.

    ``accumulate`` adds to ``cache.weight`` what each slot receives: its softmax weight summed over
    the S tokens and the query heads of its key head. It takes scratch of 4 bytes per query row and
    slot of the cache's whole capacity, written and read back: made for few rows (1560 tokens of 40
    heads over 32760 slots: 8.2 GB and 6.3 ms).
    """
    scale = _check_attend(q, cache, sm_scale, accumulate)
    causal, accumulate = bool(causal), bool(accumulate)
    if _eager_call(q):
        o, lse = _attend(q, cache, scale, causal, accumulate)
        if accumulate:
            cache._changed("attend")
    else:
        refuse_forward_mode("paged_attention", q, *_cache_tensors(cache))
        tensors = _cache_tensors(cache)
        if not accumulate:
            tensors[-2:] = None, None
        o, lse = torch.ops.dmad.paged_attn(q, scale, causal, *tensors)
    return (o, lse) if return_lse else o


def _attend(q, cache, scale, causal, accumulate):
    """The launch: (o, lse)."""
    S, Hq = q.shape[1], q.shape[2]
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = cache._floats.new_empty((cache.batch, Hq, S))
    q, strides = readable_rows(q)
    ws_ptr, ws_size, ws = cache._workspace(nat.paged_attn_workspace_bytes, S, Hq, accumulate)
    with nat.on_device(cache.device):
        nat.check(nat.lib().dmad_paged_attn(
            cache._code, cache._ref, S, Hq, nat.ptr(q), strides, int(causal), int(accumulate), scale,
            nat.ptr(o), nat.ptr(lse), ws_ptr, ws_size, nat.stream_ptr(cache.device)))
    return o, lse


def _check_evict(cache, keep, recent, sink):
    """Refuses what the eviction does not take."""
    op = "evict_low_weight"
    if not isinstance(cache, PagedKVCache):
        raise TypeError(f"{op}: cache must be a PagedKVCache, got {type(cache).__name__}")
    cache._settle()
    if cache.weight is None:
        raise ValueError(f"{op}: the cache keeps no weights and positions")
    if keep < 1 or recent < 0 or sink < 0 or recent + sink > keep:
        raise ValueError(f"{op}: keep must be at least 1, recent and sink non-negative and together at most keep; got "
                         f"keep={keep}, recent={recent}, sink={sink}")
    cache._writable(op)
    _no_grad_only(op, cache)


def evict_low_weight(cache, keep, recent=0, sink=0):
    """Cuts every sequence of more than ``keep`` slots to ``keep``, in place, each key head by itself.

    Slots of the first ``sink`` positions and of the last ``recent`` ones (of ``cache.seen``) stay,
    then those with the largest accumulated weight; of equal ones the lower slots. A NaN weight
    counts as the largest. The sequence then ends behind its ``keep``-th slot; slots before that
    end that go are filled, in order, with those beyond that stay, with their weights and
    positions: slots are in no order of position afterwards, and a key head's slot holds another
    token than another head's. Pages beyond ``cache.lengths`` are free then. Slots of missing pages
    hold nothing: they do not count towards ``keep`` and none is filled, so a window whose front
    pages were dropped keeps ``keep`` of the slots it still has (``cache.lengths`` is then larger
    than ``keep`` by the missing ones; without any it is ``keep``).
    """
    keep, recent, sink = int(keep), int(recent), int(sink)
    _check_evict(cache, keep, recent, sink)
    if keep >= cache.capacity or cache.batch == 0:
        return  # no sequence can be longer
    if _eager_call():
        _evict(cache, keep, recent, sink)
        cache._changed("evict")
    else:
        refuse_forward_mode("evict_low_weight", *_cache_tensors(cache))
        torch.ops.dmad.kv_evict(keep, recent, sink, *_cache_tensors(cache))


def _evict(cache, keep, recent, sink):
    """The launches."""
    ws_ptr, ws_size, ws = cache._workspace(nat.kv_evict_workspace_bytes, keep)
    with nat.on_device(cache.device):
        nat.check(nat.lib().dmad_kv_evict(cache._code, cache._ref, keep, recent, sink, ws_ptr, ws_size,
                                          nat.stream_ptr(cache.device)))

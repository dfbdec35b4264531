"""The paged K/V cache in 8 bits: its append, its attention, and the attention over the pages that score best.

A :class:`PagedKV8Cache` holds codes of one byte (int8 or float8_e4m3fn) with an FP32 scale per block -- a page of one KV
head -- for K and for V: half the bytes of a 16-bit cache, and so up to twice the speed of what reads it.  A decode step over it is

    q = rope_gqa_paged_kv8_append(q, k, v, cos, sin, positions, page_table, sequence_ids, cache, rope_dim=..., interleaved=...)
    out = paged_kv8_decode_attention(q, cache, positions, page_table, sequence_ids)

or, over the ``top_pages`` pages of each context whose mean keys score best,

    pages = select_kv8_pages(q, cache, positions, page_table, sequence_ids, top_pages=...)
    out = paged_kv8_sparse_attention(q, cache, pages, positions, page_table, sequence_ids)

Not part of upstream, whose cache has the type of its values.  As everywhere: ValueError for what an op does not take, the tensors' device,
torch's current stream, no synchronisation, safe under graph capture; index values are trusted, but for positions below 0, which mark
padding.  These ops have no gradient.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import _native
from .contracts import storage_overlaps
from .ops import _RMS_DTYPES, _flags, _gate, _need

HEAD_DIMS = (64, 128, 256)
MAX_PAGE_SIZE = 1024
MAX_GROUP = 8  # query heads that share a KV head
MAX_SELECT_PAGES = 51200  # pages of a sequence that select_kv8_pages can choose from
MAX_TOKENS = 65535  # of a call that reads the cache
MAX_APPEND_TOKENS = 1 << 26  # and tokens * kv_heads of one that reads it
_LARGEST = 3.4028234663852886e38  # of float32
_CODES = {torch.int8: _native.XDK_KV8_INT8, torch.float8_e4m3fn: _native.XDK_KV8_E4M3}


@dataclass(frozen=True)
class PagedKV8Cache:
    """Codes, scales and mean keys of a paged cache; the tensors are the caller's and are written in place.

    ``k``, ``v``: int8 or float8_e4m3fn, [pages, page_size, kv_heads, head_dim] ("NHD") or [pages, kv_heads, page_size, head_dim]
    ("HND"); ``k_scale``, ``v_scale``: float32 [pages, kv_heads], a value is code * scale, and no scale is negative; ``k_mean``: int8 [pages, kv_heads,
    head_dim], the mean key of each full block in units of its scale (e4m3: of its scale * 448 / 127), both as the call left them that
    wrote the block's last position, or None for a cache from which no pages are selected."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor
    k_mean: torch.Tensor | None = None
    kv_layout: str = "NHD"

    def __post_init__(self):
        layout = self.kv_layout.upper()
        _need(layout in ("NHD", "HND"), "kv_layout must be NHD or HND")
        object.__setattr__(self, "kv_layout", layout)
        k, v = self.k, self.v
        _need(k.dtype in _CODES, "k must be int8 or float8_e4m3fn")
        _need(v.dtype == k.dtype, "k and v must have one dtype")
        _need(k.dim() == 4 and k.shape == v.shape, "k and v must be 4D paged tensors of one shape")
        _need(k.numel() > 0, "pages, page_size, kv_heads and head_dim must be positive")
        _need(self.head_dim in HEAD_DIMS, "head_dim must be 64, 128 or 256")
        _need(self.page_size <= MAX_PAGE_SIZE, f"page_size must be at most {MAX_PAGE_SIZE}")
        _need(self.kv_heads <= 65535, "kv_heads must be at most 65535")
        for name, t in (("k_scale", self.k_scale), ("v_scale", self.v_scale)):
            _need(t.dtype == torch.float32 and tuple(t.shape) == (self.pages, self.kv_heads), f"{name} must be float32 [pages, kv_heads]")
        if self.k_mean is not None:
            _need(self.k_mean.dtype == torch.int8 and tuple(self.k_mean.shape) == (self.pages, self.kv_heads, self.head_dim),
                  "k_mean must be int8 [pages, kv_heads, head_dim]")
        for t in self.tensors():
            _need(t.device == k.device, "the cache's tensors must share one device")
            _need(t.is_contiguous(), "the cache's tensors must be contiguous")
            _need(not t.requires_grad, "the cache has no gradient; detach its tensors")
            _need(t.dtype == torch.float32 or t.data_ptr() % 16 == 0, "k, v and k_mean must be 16-byte aligned")
        every = self.tensors()
        _need(not any(storage_overlaps(a, b) for i, a in enumerate(every) for b in every[:i]), "the cache's tensors must not overlap")

    @classmethod
    def empty(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, *, dtype=torch.int8, kv_layout: str = "NHD",
              means: bool = True, device="cuda") -> "PagedKV8Cache":
        """A cache of zeros.  ``means=False``: without the mean keys, for a cache from which no pages are selected."""
        shape = (pages, page_size, kv_heads, head_dim) if kv_layout.upper() == "NHD" else (pages, kv_heads, page_size, head_dim)
        return cls(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device),
                   torch.zeros(pages, kv_heads, device=device), torch.zeros(pages, kv_heads, device=device),
                   torch.zeros(pages, kv_heads, head_dim, dtype=torch.int8, device=device) if means else None, kv_layout)

    @property
    def hnd(self) -> bool:
        return self.kv_layout == "HND"

    @property
    def pages(self) -> int:
        return self.k.shape[0]

    @property
    def page_size(self) -> int:
        return self.k.shape[2 if self.hnd else 1]

    @property
    def kv_heads(self) -> int:
        return self.k.shape[1 if self.hnd else 2]

    @property
    def head_dim(self) -> int:
        return self.k.shape[3]

    def tensors(self) -> tuple:
        every = (self.k, self.v, self.k_scale, self.v_scale)
        return every if self.k_mean is None else (*every, self.k_mean)

    def dequantized(self) -> tuple:
        """(k, v) in float32, in the cache's layout: what the codes stand for (to look at or to export; an ordinary torch expression)."""
        per = (slice(None), slice(None), None, None) if self.hnd else (slice(None), None, slice(None), None)
        return self.k.float() * self.k_scale[per], self.v.float() * self.v_scale[per]


def _indices(q, cache, positions, page_table, sequence_ids):
    """The checks that the four ops share; returns (tokens, q_heads)."""
    _need(isinstance(cache, PagedKV8Cache), "cache must be a PagedKV8Cache")
    _gate(q)
    _need(q.dtype in _RMS_DTYPES, "q must be float32, bfloat16 or float16")
    _need(q.dim() == 3 and q.numel() > 0, "q must be [tokens, q_heads, head_dim]")
    _need(not q.requires_grad, "these ops have no gradient; detach q")
    _need(cache.k.device == q.device, "the cache must be on the same CUDA device as q")
    tokens, q_heads, head_dim = q.shape
    _need(head_dim == cache.head_dim, "q and the cache must have one head_dim")
    _need(q_heads % cache.kv_heads == 0, "q_heads must be divisible by kv_heads")
    for name, t in (("positions", positions), ("page_table", page_table), ("sequence_ids", sequence_ids)):
        _need(t.is_cuda and t.device == q.device, f"{name} must be on the same CUDA device as q")
        _need(t.dtype == torch.int64, f"{name} must be int64")
        _need(t.is_contiguous(), f"{name} must be contiguous")
    _need(positions.dim() == 1 and sequence_ids.dim() == 1 and page_table.dim() == 2, "index tensors have the wrong rank")
    _need(positions.shape[0] == tokens and sequence_ids.shape[0] == tokens, "index vectors must have one entry per token")
    _need(page_table.shape[0] > 0 and page_table.shape[1] > 0, "page_table must contain at least one page per sequence row")
    return tokens, q_heads


def rope_gqa_paged_kv8_append(q, k, v, cos, sin, positions, page_table, sequence_ids, cache: PagedKV8Cache, *, rope_dim: int,
                              interleaved: bool, dependent_launch: bool = False):
    """Rotate Q and K, write rotated K and V into their blocks as codes, return rotated Q.

    The arguments are those of :func:`cross_dsl_kernels_b200.ops.rope_gqa_paged_kv_append`.  A block's scale is the largest
    |value| it was given since its first position was written, / 127 (int8) or 448 (e4m3); where a call makes it grow, the block's
    other codes are rounded to the new scale.  A block whose last position is written gets its mean key; a call that writes others
    of its positions anew leaves that as it is, until the last one is written again, too.  Tokens may come in any order, several
    for one page, and of several for one slot the last one counts.  A token with a position below 0 is padding: nothing is written
    for it, and its row of the result is 0.  A value that is not finite makes its block read as NaN until the page is begun anew."""
    done = _native.host().kv8_append(q, k, v, cos, sin, positions, page_table, sequence_ids, *_parts(cache), rope_dim, interleaved,
                                     dependent_launch)
    if done is not None:
        return done
    tokens, q_heads = _indices(q, cache, positions, page_table, sequence_ids)
    _need(tokens <= MAX_APPEND_TOKENS, f"at most {MAX_APPEND_TOKENS} tokens per call")
    _need(q_heads <= 65535, "q_heads must be at most 65535")
    kv_heads, head_dim = cache.kv_heads, cache.head_dim
    for name, t, want in (("k", k, q.dtype), ("v", v, q.dtype), ("cos", cos, torch.float32), ("sin", sin, torch.float32)):
        _need(t.is_cuda and t.device == q.device, f"{name} must be on the same CUDA device as q")
        _need(t.dtype == want, f"{name} has an unexpected dtype")
        _need(not t.requires_grad, f"these ops have no gradient; detach {name}")
    _need(k.dim() == 3 and v.dim() == 3, "q, k, v must be [tokens, heads, head_dim]")
    _need(tuple(k.shape) == (tokens, kv_heads, head_dim) and k.shape == v.shape, "k and v must be [tokens, kv_heads, head_dim] of the cache")
    for name, t in (("q", q), ("k", k), ("v", v)):
        dense = t.stride(2) == 1 and t.stride(1) == t.shape[2] and t.stride(0) >= t.shape[1] * t.shape[2]
        _need(t.is_contiguous() or dense, f"{name} must be contiguous or a column slice of a row-major matrix")
    _need(cos.dim() == 2 and cos.is_contiguous() and sin.is_contiguous(), "cos and sin must be contiguous [max_position, >= rope_dim / 2]")
    _need(type(rope_dim) is int and rope_dim > 0 and rope_dim % 2 == 0, "rope_dim must be a positive even integer")
    _need(rope_dim <= head_dim, "rope_dim cannot exceed head_dim")
    _need(cos.shape[0] > 0 and cos.shape[1] >= rope_dim // 2 and sin.shape == cos.shape, "cos/sin need >= rope_dim / 2 columns and equal shapes")
    inputs = (q, k, v, cos, sin, positions, page_table, sequence_ids)
    _need(not any(storage_overlaps(c, t) for c in cache.tensors() for t in inputs), "the cache must not overlap the input tensors")
    with torch.cuda.device(q.device):
        lib = _native.lib()
        q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        # the groups of a long batch by page: a fresh block per call, as the scratch of the other ops
        need = lib.xdk_kv8_append_scratch_bytes(tokens, kv_heads)
        scratch = torch.empty(need, device=q.device, dtype=torch.uint8) if need else None
        status = lib.xdk_kv8_append(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), cos.data_ptr(), sin.data_ptr(), positions.data_ptr(), page_table.data_ptr(),
            sequence_ids.data_ptr(), q_out.data_ptr(), cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(),
            cache.v_scale.data_ptr(), cache.k_mean.data_ptr() if cache.k_mean is not None else None, tokens, q_heads, kv_heads, head_dim,
            cos.shape[1], page_table.shape[1], cache.page_size, rope_dim,
            q.stride(0) if tokens > 1 else q_heads * head_dim, k.stride(0) if tokens > 1 else kv_heads * head_dim,
            v.stride(0) if tokens > 1 else kv_heads * head_dim, int(bool(interleaved)), int(cache.hnd), _native.dtype_code(q.dtype),
            _CODES[cache.k.dtype], scratch.data_ptr() if need else None, need, _flags(dependent_launch), _native.stream_ptr(q.device))
    _native.check(status, "xdk_kv8_append")
    return q_out


def _parts(cache) -> tuple:
    """What the native half takes of a cache; of anything else, what it declines."""
    if type(cache) is not PagedKV8Cache:
        return (None,) * 6
    return cache.k, cache.v, cache.k_scale, cache.v_scale, cache.k_mean, cache.kv_layout


def _read(q, cache, positions, page_table, sequence_ids, scale):
    tokens, q_heads = _indices(q, cache, positions, page_table, sequence_ids)
    _need(q.is_contiguous(), "q must be contiguous [tokens, q_heads, head_dim]")
    _need(q_heads // cache.kv_heads <= MAX_GROUP, f"q_heads / kv_heads must be at most {MAX_GROUP}")
    scale = float(cache.head_dim) ** -0.5 if scale is None else float(scale)
    _need(abs(scale) <= _LARGEST, "scale must be finite in float32")
    _need(tokens <= MAX_TOKENS, f"at most {MAX_TOKENS} tokens per call")
    _need(tokens * cache.kv_heads <= MAX_APPEND_TOKENS, f"tokens * kv_heads must be at most {MAX_APPEND_TOKENS}")
    return tokens, q_heads, scale


def _destination(q, peer_out):
    width = q.shape[1] * q.shape[2]
    if peer_out is not None:
        _need(peer_out.ld >= peer_out.col0 + width, "peer_out is narrower than col0 + q_heads * head_dim")
        return None, peer_out
    out = torch.empty_like(q)
    dst = _native.PeerOutStruct()
    dst.ptr[0], dst.world, dst.ld, dst.col0 = out.data_ptr(), 1, width, 0
    return out, dst


def paged_kv8_decode_attention(q, cache: PagedKV8Cache, positions, page_table, sequence_ids, *, scale=None, context_hint: int = 0,
                               dependent_launch: bool = False, peer_out=None):
    """Decode attention of one query token per sequence over an 8-bit cache (the token's own K/V included): softmax(scale * q.K) . V per
    head, softmax and sums in FP32, any q_heads / kv_heads up to 8.  A token with a position below 0 has no context: zeros.

    ``context_hint`` and ``peer_out`` as for :func:`cross_dsl_kernels_b200.ops.paged_decode_attention`."""
    if peer_out is None:
        done = _native.host().kv8_attention(q, *_parts(cache), positions, page_table, sequence_ids, scale, context_hint, dependent_launch)
        if done is not None:
            return done
    tokens, q_heads, scale = _read(q, cache, positions, page_table, sequence_ids, scale)
    with torch.cuda.device(q.device):
        lib = _native.lib()
        out, dst = _destination(q, peer_out)
        hint = int(context_hint)
        if hint <= 0:  # no bound: that of a page table row
            hint = page_table.shape[1] * cache.page_size
        hint = min(hint, 2 ** 62)
        need = lib.xdk_kv8_decode_attention_scratch_bytes(tokens, q_heads, cache.kv_heads, cache.head_dim, hint)
        scratch = torch.empty(need, device=q.device, dtype=torch.uint8)
        status = lib.xdk_kv8_decode_attention(
            q.data_ptr(), cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), positions.data_ptr(),
            page_table.data_ptr(), sequence_ids.data_ptr(), ctypes.byref(dst), tokens, q_heads, cache.kv_heads, cache.head_dim,
            page_table.shape[1], cache.page_size, int(cache.hnd), scale, hint, _native.dtype_code(q.dtype), _CODES[cache.k.dtype],
            scratch.data_ptr(), need, _flags(dependent_launch), _native.stream_ptr(q.device))
    _native.check(status, "xdk_kv8_decode_attention")
    return out


def select_kv8_pages(q, cache: PagedKV8Cache, positions, page_table, sequence_ids, *, top_pages: int, dependent_launch: bool = False):
    """The pages that :func:`paged_kv8_sparse_attention` reads for each token and KV head: int32 [tokens, kv_heads, top_pages],
    logical pages in ascending order, -1 behind the last one.

    The last page of the context is always among them, the others are those in front of it with the best scores, the lowest page first
    among equals: score = max over the query heads of the group of the product of the head's codes (q in 8 bits) with the block's mean key.
    Products of whole numbers, so the choice does not depend on an order of summation.  Shorter contexts: all of their pages; a position
    below 0: none.  ``cache`` has to have its mean keys (``k_mean``); rotated q, as the attention takes it."""
    done = _native.host().kv8_select(q, *_parts(cache), positions, page_table, sequence_ids, top_pages, dependent_launch)
    if done is not None:
        return done
    tokens, q_heads, _ = _read(q, cache, positions, page_table, sequence_ids, None)
    _need(cache.k_mean is not None, "the cache has no mean keys to select pages by (k_mean)")
    _need(type(top_pages) is int and 0 < top_pages < 2 ** 31, "top_pages must be a positive integer")
    _need(page_table.shape[1] <= MAX_SELECT_PAGES, f"page_table may have at most {MAX_SELECT_PAGES} pages per sequence row")
    with torch.cuda.device(q.device):
        pages = torch.empty((tokens, cache.kv_heads, top_pages), dtype=torch.int32, device=q.device)
        status = _native.lib().xdk_kv8_select_pages(
            q.data_ptr(), cache.k_mean.data_ptr(), cache.k_scale.data_ptr(), positions.data_ptr(), page_table.data_ptr(),
            sequence_ids.data_ptr(), pages.data_ptr(), tokens, q_heads, cache.kv_heads, cache.head_dim, page_table.shape[1],
            cache.page_size, top_pages, _native.dtype_code(q.dtype), _flags(dependent_launch), _native.stream_ptr(q.device))
    _native.check(status, "xdk_kv8_select_pages")
    return pages


def paged_kv8_sparse_attention(q, cache: PagedKV8Cache, pages, positions, page_table, sequence_ids, *, scale=None,
                               dependent_launch: bool = False, peer_out=None):
    """:func:`paged_kv8_decode_attention` over the positions in the listed pages only.  ``pages``: int32 [tokens, kv_heads, n],
    logical pages in ascending order, from :func:`select_kv8_pages` or any other choice (a window, the first pages); an
    entry that is negative, not above the one before it, or behind the token's context adds nothing."""
    if peer_out is None:
        done = _native.host().kv8_sparse(q, *_parts(cache), pages, positions, page_table, sequence_ids, scale, dependent_launch)
        if done is not None:
            return done
    tokens, q_heads, scale = _read(q, cache, positions, page_table, sequence_ids, scale)
    _need(pages.is_cuda and pages.device == q.device, "pages must be on the same CUDA device as q")
    _need(pages.dtype == torch.int32 and pages.is_contiguous(), "pages must be contiguous int32")
    _need(pages.dim() == 3 and tuple(pages.shape[:2]) == (tokens, cache.kv_heads) and pages.shape[2] > 0, "pages must be [tokens, kv_heads, n]")
    _need(pages.shape[2] <= (2 ** 31 - 1) // MAX_PAGE_SIZE, "too many pages per token")
    with torch.cuda.device(q.device):
        lib = _native.lib()
        out, dst = _destination(q, peer_out)
        need = lib.xdk_kv8_sparse_attention_scratch_bytes(tokens, q_heads, cache.kv_heads, cache.head_dim, cache.page_size, pages.shape[2])
        scratch = torch.empty(need, device=q.device, dtype=torch.uint8)
        status = lib.xdk_kv8_sparse_attention(
            q.data_ptr(), cache.k.data_ptr(), cache.v.data_ptr(), cache.k_scale.data_ptr(), cache.v_scale.data_ptr(), pages.data_ptr(),
            positions.data_ptr(), page_table.data_ptr(), sequence_ids.data_ptr(), ctypes.byref(dst), tokens, q_heads, cache.kv_heads,
            cache.head_dim, page_table.shape[1], cache.page_size, pages.shape[2], int(cache.hnd), scale, _native.dtype_code(q.dtype),
            _CODES[cache.k.dtype], scratch.data_ptr(), need, _flags(dependent_launch), _native.stream_ptr(q.device))
    _native.check(status, "xdk_kv8_sparse_attention")
    return out

"""
A paged key / value cache for serving a decoder: which pages a request has, where its new tokens go, and the attention of one new token per request
over the pages (``csrc/paged.cu``, ``csrc/paged_attention.cu``). All of it is on the GPU: a decoding step asks the host for nothing and can be
captured in a CUDA graph.

A cache is ``[pages, key heads, page size, D]`` for keys and one for values; its layers share one block table. ``block_table[i, b]`` is the page
of tokens ``b * page_size .. `` of request ``i``. Free pages lie in a ring ``free_pages`` (of as many places as there are pages), from place
``free_range[0]`` to before ``free_range[1]``, both counted on without end and taken modulo the size of the ring. A step of a serving loop::

    new = append_tokens(block_table, lengths, counts, free_pages, free_range, page_size=16, max_tokens=total)
    for each layer:
        q = norm_rope_to_cache(q, k, v, new.positions, frequencies, k_cache, v_cache, new.slots)      # ops/norm_rope.py
        out = paged_attention(q, k_cache, v_cache, block_table, new.lengths)
    lengths, free_range = new.lengths, new.free_range
    ...
    lengths, free_range = release_pages(block_table, lengths, finished, free_pages, free_range, page_size=16)

The reference has no counterpart: its step-wise states grow by concatenation (returnn/frontend/attention.py:289).
"""

from __future__ import annotations
from typing import NamedTuple, Optional
import ctypes
import math
import torch
from . import _lib, nodes
from .gemm import status_tensor

__all__ = ["AppendedTokens", "ReleasedPages", "append_tokens", "release_pages", "paged_attention", "append_tokens_reference",
           "release_pages_reference", "paged_attention_reference"]

_vp, _i32, _i64, _f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float


class AppendedTokens(NamedTuple):
    """
    what :func:`append_tokens` returns. On the GPU the tensors may share one allocation: one that is kept keeps the memory of all (copy it to keep it alone).
    """

    slots: torch.Tensor  # [max_tokens] int32, page * page size + place in the page; -1: no place (request not granted, or room without a token)
    positions: torch.Tensor  # [max_tokens] int32 position in the request; 0 in room without a token
    requests: torch.Tensor  # [max_tokens] int32; -1 in room without a token
    offsets: torch.Tensor  # [requests + 1] int32: the first token of each request, and their number
    lengths: torch.Tensor  # [requests] int32 after the call (unchanged where not granted)
    free_range: torch.Tensor  # [2] int64 after the call
    granted: torch.Tensor  # [requests] bool: the new tokens have their place


class ReleasedPages(NamedTuple):
    """what :func:`release_pages` returns; see :class:`AppendedTokens` about their memory"""

    lengths: torch.Tensor  # [requests] int32, 0 where finished
    free_range: torch.Tensor  # [2] int64


def _check_table(what, block_table, lengths, per_request, per_type, free_pages, free_range, page_size):
    dev = block_table.device
    if block_table.dim() != 2 or block_table.dtype != torch.int32 or (block_table.stride(1) != 1 and block_table.shape[1] > 1):
        raise ValueError("%s: the block table must be int32 [requests, blocks] with unit stride over the blocks" % what)
    for t, kind in ((lengths, torch.int32), (per_request, per_type)):
        if t.shape != block_table.shape[:1] or t.dtype != kind or t.device != dev:
            raise ValueError("%s: expected %s [%i] on %s, got %s %s on %s" % (what, kind, block_table.shape[0], dev, t.dtype, tuple(t.shape), t.device))
    if free_pages.dim() != 1 or free_pages.dtype != torch.int32 or not free_pages.is_contiguous() or free_pages.device != dev or not free_pages.numel():
        raise ValueError("%s: free_pages must be a contiguous int32 [pages] on %s" % (what, dev))
    if free_range.shape != (2,) or free_range.dtype != torch.int64 or free_range.device != dev:
        raise ValueError("%s: free_range must be int64 [2] on %s" % (what, dev))
    if page_size < 1:
        raise ValueError("%s: page size %r" % (what, page_size))


def append_tokens(block_table: torch.Tensor, lengths: torch.Tensor, counts: torch.Tensor, free_pages: torch.Tensor, free_range: torch.Tensor, *,
                  page_size: int, max_tokens: int) -> AppendedTokens:
    """
    Room for ``counts[i]`` more tokens of each request ``i``: pages from the ring where the last one of the request is full, their entries in the block
    table (written in place), and slot, position and request of every new token, the requests one after another.

    Requests are served in their order as long as the sum of the pages they need is there. One that comes too late, or whose row of the table
    is too short, is not granted: its length stays and its tokens have no slot. Lengths, counts, ring and range are not changed; the same call again has the same result.

    :param block_table: [requests, blocks] int32
    :param lengths: [requests] int32 tokens so far
    :param counts: [requests] int32 new tokens, 0 where there are none
    :param free_pages: [pages] int32, the ring; pages times page size at most 2^31
    :param free_range: [2] int64
    :param max_tokens: room for new tokens, at least ``counts.sum()`` (tokens beyond it are left out of the lists, not of the lengths)
    """
    what = "append_tokens"
    mod = nodes.of(block_table)
    if mod is not None:
        res = mod.append_tokens(block_table, lengths, counts, free_pages, free_range, page_size, max_tokens)
        if res is not None:
            return AppendedTokens(*res)
    _check_table(what, block_table, lengths, counts, torch.int32, free_pages, free_range, page_size)
    if max_tokens < 0:
        raise ValueError("%s: max_tokens %r" % (what, max_tokens))
    if free_pages.shape[0] * page_size > 2**31:
        raise ValueError("%s: %i pages of %i tokens, slots have 31 bits" % (what, free_pages.shape[0], page_size))
    if not (block_table.is_cuda and _lib.use_native(block_table)):
        return append_tokens_reference(block_table, lengths, counts, free_pages, free_range, page_size=page_size, max_tokens=max_tokens)
    with torch.cuda.device_of(block_table):
        dev = block_table.device
        n, blocks = block_table.shape
        lengths, counts, free_range = lengths.contiguous(), counts.contiguous(), free_range.contiguous()
        lists = torch.empty(3, (max_tokens + 3) // 4 * 4, dtype=torch.int32, device=dev)
        offsets = torch.empty(n + 1, dtype=torch.int32, device=dev)
        new_lengths = torch.empty(n, dtype=torch.int32, device=dev)
        new_range = torch.empty(2, dtype=torch.int64, device=dev)
        granted = torch.empty(n, dtype=torch.bool, device=dev)
        fn = _lib.bind("rb200_paged_append", [_vp, _i64, _i32, _vp, _vp, _i32, _vp, _i64, _vp, _i32, _i64, _vp, _vp, _vp, _vp, _vp, _vp, _vp, _vp])
        slots, positions, requests = lists[:, :max_tokens].unbind(0)
        _lib.check(fn(block_table.data_ptr(), block_table.stride(0), blocks, lengths.data_ptr(), counts.data_ptr(), n, free_pages.data_ptr(), free_pages.shape[0],
                      free_range.data_ptr(), page_size, max_tokens, slots.data_ptr(), positions.data_ptr(), requests.data_ptr(), offsets.data_ptr(),
                      new_lengths.data_ptr(), new_range.data_ptr(), granted.data_ptr(), _lib.stream_ptr()), what)
        _lib.count_launch()
        nodes.written(block_table)
    return AppendedTokens(slots, positions, requests, offsets, new_lengths, new_range, granted)


def release_pages(block_table: torch.Tensor, lengths: torch.Tensor, finished: torch.Tensor, free_pages: torch.Tensor, free_range: torch.Tensor, *,
                  page_size: int) -> ReleasedPages:
    """
    The pages of finished requests go to the tail of the ring (written in place), in the order of requests and blocks; their lengths become 0.
    Lengths, table and range are not changed.

    :param finished: [requests] bool
    """
    what = "release_pages"
    mod = nodes.of(block_table)
    if mod is not None:
        res = mod.release_pages(block_table, lengths, finished, free_pages, free_range, page_size)
        if res is not None:
            return ReleasedPages(*res)
    _check_table(what, block_table, lengths, finished, torch.bool, free_pages, free_range, page_size)
    if not (block_table.is_cuda and _lib.use_native(block_table)):
        return release_pages_reference(block_table, lengths, finished, free_pages, free_range, page_size=page_size)
    with torch.cuda.device_of(block_table):
        dev = block_table.device
        n, blocks = block_table.shape
        lengths, finished, free_range = lengths.contiguous(), finished.contiguous(), free_range.contiguous()
        new_lengths = torch.empty(n, dtype=torch.int32, device=dev)
        new_range = torch.empty(2, dtype=torch.int64, device=dev)
        fn = _lib.bind("rb200_paged_release", [_vp, _i64, _i32, _vp, _vp, _i32, _vp, _i64, _vp, _i32, _vp, _vp, _vp])
        _lib.check(fn(block_table.data_ptr(), block_table.stride(0), blocks, lengths.data_ptr(), finished.data_ptr(), n, free_pages.data_ptr(), free_pages.shape[0],
                      free_range.data_ptr(), page_size, new_lengths.data_ptr(), new_range.data_ptr(), _lib.stream_ptr()), what)
        _lib.count_launch()
        nodes.written(free_pages)
    return ReleasedPages(new_lengths, new_range)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, *,
                    scale: Optional[float] = None) -> torch.Tensor:
    """
    Attention of one query per request over its cached tokens (the newest among them: ``lengths`` counts it), without gradient.

    The waits in the kernel are bounded. One that runs out leaves its code on the status board (:mod:`returnn_b200.ops.status`), and the result is not valid: programs of their own
    look at the board with :class:`returnn_b200.ops.status.StatusPoller` or :func:`returnn_b200.ops.status.check_now`.

    :param q: [requests, heads, D] bf16 or fp32, unit stride over D
    :param k_cache: [pages, key heads, page size, D] of the same type, D a multiple of 8 up to 256; any strides with unit stride over D
        that are multiples of 16 bytes. ``heads`` is a multiple of the key heads; query head ``h`` reads key head ``h // (heads / key heads)``.
    :param v_cache: the same for the values
    :param block_table: [requests, blocks] int32. An entry that is no page counts as tokens that are not there.
    :param lengths: [requests] int32; a request of length 0 gets zeros
    :param scale: of the scores, default ``D ** -0.5``
    :return: [requests, heads, D], contiguous
    """
    what = "paged_attention"
    mod = nodes.of(q)
    if mod is not None:
        res = mod.paged_attention(q, k_cache, v_cache, block_table, lengths, q.shape[-1] ** -0.5 if scale is None else scale, status_tensor(q.device))
        if res is not None:
            return res
    if q.dim() != 3 or k_cache.dim() != 4 or v_cache.shape != k_cache.shape or k_cache.shape[3] != q.shape[2]:
        raise ValueError("%s: q %s must be [requests, heads, D], the caches [pages, key heads, page size, D], got %s and %s" % (
            what, tuple(q.shape), tuple(k_cache.shape), tuple(v_cache.shape)))
    if not (q.dtype == k_cache.dtype == v_cache.dtype) or not (q.device == k_cache.device == v_cache.device == block_table.device == lengths.device):
        raise TypeError("%s: all of one type and device, got %s / %s / %s on %s / %s / %s" % (
            what, q.dtype, k_cache.dtype, v_cache.dtype, q.device, k_cache.device, v_cache.device))
    n, heads, d = q.shape
    pages, kv_heads, page, _ = k_cache.shape
    if kv_heads < 1 or heads % kv_heads or page < 1:
        raise ValueError("%s: %i query heads over %i key heads, page size %i" % (what, heads, kv_heads, page))
    if block_table.dim() != 2 or block_table.shape[0] != n or block_table.dtype != torch.int32 or (block_table.stride(1) != 1 and block_table.shape[1] > 1):
        raise ValueError("%s: the block table must be int32 [%i, blocks] with unit stride over the blocks" % (what, n))
    if lengths.shape != (n,) or lengths.dtype != torch.int32:
        raise ValueError("%s: lengths must be int32 [%i]" % (what, n))
    if torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad):
        raise RuntimeError("%s has no gradient: call it under torch.no_grad()" % what)
    if nodes.has_tangent(q, k_cache, v_cache):
        raise RuntimeError("%s has no derivative" % what)
    scale = float(d) ** -0.5 if scale is None else float(scale)
    if not (q.is_cuda and _lib.use_native(q)):
        return paged_attention_reference(q, k_cache, v_cache, block_table, lengths, scale=scale)
    if q.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError("%s: bf16 and fp32 on the GPU, got %s" % (what, q.dtype))
    for c in (k_cache, v_cache):
        unit = 16 // c.element_size()
        if c.stride(3) != 1 or any(s % unit for s, m in zip(c.stride()[:3], c.shape) if m > 1) or c.data_ptr() % 16:
            raise ValueError("%s: a cache starts on 16 bytes and has unit stride over D and other strides of whole 16 bytes, got %s" % (what, c.stride()))
    with torch.cuda.device_of(q):
        if q.stride(2) != 1:
            q = q.contiguous()
        lengths = lengths.contiguous()
        bf16 = 1 if q.dtype == torch.bfloat16 else 0
        size = _lib.bind("rb200_paged_attention_workspace", [_i32, _i32, _i32, _i32, _i32])
        size.restype = _i64
        work = torch.empty(size(n, heads, kv_heads, d, bf16), dtype=torch.uint8, device=q.device)
        out = torch.empty(n, heads, d, dtype=q.dtype, device=q.device)
        # (the stride of an axis of one element is never used)
        st = (_i64 * 8)(q.stride(0), q.stride(1), *(s if m > 1 else 0 for c in (k_cache, v_cache) for s, m in zip(c.stride()[:3], c.shape)))
        fn = _lib.bind("rb200_paged_attention", [_vp, _vp, _vp, _vp, _i64, _vp, _vp, _vp, _vp, _i32, _i32, _i32, _i32, _i32, _i32, _i32, _f32, _i32, _vp, _vp])
        _lib.check(fn(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(), block_table.stride(0), lengths.data_ptr(), out.data_ptr(),
                      work.data_ptr(), st, n, heads, kv_heads, d, page, block_table.shape[1], pages, scale, bf16, status_tensor(q.device).data_ptr(), _lib.stream_ptr()), what)
        _lib.count_launch(2)
    return out


# ---- plain torch: what runs on the CPU, and the oracle of the kernels


def append_tokens_reference(block_table, lengths, counts, free_pages, free_range, *, page_size, max_tokens):
    """plain torch"""
    dev = block_table.device
    n, blocks = block_table.shape
    size = free_pages.shape[0]
    lens, add = lengths.long().clamp(min=0), counts.long().clamp(min=0)
    head, tail = free_range[0], free_range[1]
    have = (lens + page_size - 1) // page_size
    fits = lens + add <= blocks * page_size
    need = torch.where(fits, (lens + add + page_size - 1) // page_size - have, 0)
    granted = fits & ((need == 0) | (torch.cumsum(need, 0) <= (tail - head).clamp(0, size)))
    take = torch.where(granted, need, 0)
    first = torch.cumsum(take, 0) - take
    at = torch.arange(blocks, device=dev)[None, :]
    fresh = free_pages[(head + first[:, None] + at - have[:, None]) % size]
    block_table.copy_(torch.where((at >= have[:, None]) & (at < (have + take)[:, None]), fresh, block_table))
    offsets = torch.cat([add.new_zeros(1), torch.cumsum(add, 0)])
    token = torch.arange(max_tokens, device=dev)
    request = torch.searchsorted(offsets[1:].contiguous(), token, right=True)
    real = request < n
    i32 = torch.int32
    new_lengths = torch.where(granted, lens + add, lengths.long()).to(i32)
    new_range = torch.stack([head + take.sum(), tail])
    if not n:
        none = torch.full((max_tokens,), -1, dtype=i32, device=dev)
        return AppendedTokens(none, torch.zeros_like(none), none.clone(), offsets.to(i32), new_lengths, new_range, granted)
    request = request.clamp(max=n - 1)
    position = lens[request] + token - offsets[request]
    placed = real & granted[request]
    page = block_table[request, (position // page_size).clamp(max=blocks - 1)] if blocks else torch.zeros_like(request)
    slot = torch.where(placed, page.long() * page_size + position % page_size, -1)
    return AppendedTokens(slot.to(i32), torch.where(real, position, 0).to(i32), torch.where(real, request, -1).to(i32), offsets.to(i32), new_lengths,
                          new_range, granted)


def release_pages_reference(block_table, lengths, finished, free_pages, free_range, *, page_size):
    """plain torch"""
    dev = block_table.device
    size = free_pages.shape[0]
    head, tail = free_range[0], free_range[1]
    count = torch.where(finished, ((lengths.long().clamp(min=0) + page_size - 1) // page_size).clamp(max=block_table.shape[1]), 0)
    last = torch.cumsum(count, 0)
    total = (last[-1] if len(last) else torch.zeros_like(tail)).minimum((size - (tail - head).clamp(min=0)).clamp(min=0))
    if block_table.numel():
        number = (torch.arange(size, device=dev) - tail) % size  # of the page that would get a place of the ring
        request = torch.searchsorted(last, number, right=True).clamp(max=len(last) - 1)
        block = (number - (last - count)[request]).clamp(0, block_table.shape[1] - 1)
        free_pages.copy_(torch.where(number < total, block_table[request, block], free_pages))
    return ReleasedPages(torch.where(finished, 0, lengths), torch.stack([head, tail + total]))


def paged_attention_reference(q, k_cache, v_cache, block_table, lengths, *, scale=None):
    """plain torch, in fp32 or the wider type of the input"""
    n, heads, d = q.shape
    pages, kv_heads, page, _ = k_cache.shape
    t = block_table.shape[1] * page
    wide = torch.promote_types(q.dtype, torch.float32)
    if not t or not pages or not n:
        return torch.zeros_like(q, memory_format=torch.contiguous_format)
    real = (block_table >= 0) & (block_table < pages)
    there = real.repeat_interleave(page, dim=1) & (torch.arange(t, device=q.device)[None, :] < lengths[:, None])
    at = block_table.clamp(0, pages - 1).long()
    k, v = (c[at].to(wide).transpose(2, 3).reshape(n, t, kv_heads, d).transpose(1, 2) for c in (k_cache, v_cache))
    mask = there[:, None, :, None]
    k, v = torch.where(mask, k, 0.0), torch.where(mask, v, 0.0)  # (what lies in unused places may be anything)
    s = torch.matmul(q.to(wide).reshape(n, kv_heads, heads // kv_heads, d), k.transpose(-1, -2)) * (d ** -0.5 if scale is None else scale)
    s = torch.where(there[:, None, None, :], s, -math.inf)
    top = s.amax(dim=-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = e.sum(dim=-1, keepdim=True)
    return (torch.matmul(e, v) / torch.where(total == 0, 1.0, total)).reshape(n, heads, d).to(q.dtype)

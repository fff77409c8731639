"""Pages: the tables of a step, rows written by slot, and a cache in 8 bits with a scale for each block of tokens.

A paged cache is a pool of pages of `page_size` tokens.  A request's tokens lie in the pages that its row of the
block_table (batch, max_pages) int32 names; the slot of a token is page * page_size + its place in the page.

    pages_resize             lengths before and after a step -> table, positions and slots of the new tokens
    cache_write              bf16 keys and values to their slots: the caches that infllmv2_attn_with_kvcache,
                             infllmv2_attn_varlen_func and infllmv2_attn_stage1 read through a block_table
    cache_write_b8           the same into a cache in 8 bits
    infllmv2_attn_paged_b8   any number of new tokens per sequence over that cache

The cache in 8 bits is kept head by head, with one scale for 64 tokens of a head:
    k_cache, v_cache  (pages, nheads_k, page_size, 128)  torch.float8_e4m3fn or torch.float8_e5m2
    k_scale, v_scale  (pages, nheads_k, page_size / 64)  torch.float8_e8m0fnu
A value is code * scale.  The scale is the smallest power of two (at least 2^-127) with which the largest magnitude of
the block's rows fits the codes (448 or 57344); codes are rounded to nearest even.  Where a later token of a block
is larger than what the scale fits, the scale grows and the codes that are there are rounded to it.  A block that an
infinity or a NaN was written to is NaN, until it is begun anew.  Without a block_table a page is a sequence."""
import functools
from typing import Optional, Tuple

import torch

from . import _lib
from .attention import BLOCK_N, GROUP, HEAD_DIM, _status_words
from .ops import _on, _require_cuda, _stream
from .quant_cache import _cu, _ints, _no_gradient, _no_tangent, _ptr, _table
from .rotary import _rows

_CODES = {torch.float8_e4m3fn: 0, torch.float8_e5m2: 1}
_MAX_REQUESTS = 16384


def page_pool(num_pages: int, device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """The ring of a pool whose pages are all free: free_pages (num_pages,) int32 and free_range (2,) int32, the place
    of the first free page in it and their number."""
    return (torch.arange(num_pages, dtype=torch.int32, device=device),
            torch.tensor([0, num_pages], dtype=torch.int32, device=device))


def pages_resize(seqlens: torch.Tensor, targets: torch.Tensor, block_table: torch.Tensor, free_pages: torch.Tensor,
                 free_range: torch.Tensor, page_size: int, total: int
                 ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Block tables and slots of a step, from the lengths of all requests before and after it.  One launch.

    seqlens, targets: (batch,) int32, at most 16384.  A request whose target is larger gets pages from the front of the
    ring (free_pages, free_range; see `page_pool`), written behind those of its row of block_table (batch, max_pages)
    int32, in place; requests get theirs in order.  One whose target is smaller gives pages back behind the ring's end
    (target 0: all of them); its row keeps what stood there.  Pages given back can be taken by the next call.
    total: the number of new tokens, sum(max(targets - seqlens, 0)); positions and slots get this many rows.
    A request that would need more pages than its row has is refused, and where the ring runs out, that request and all
    behind it that need a page: they keep their length, and the slots of their tokens are -1.  Their tokens are counted in
    cu_seqlens all the same, and rows that an attention over this step gives for them mean nothing (their keys are not
    there, and the edge is set as if they were): drop the rows whose slot is -1.

    Returns (seqlens, free_range, cu_seqlens, positions, slots): lengths after the step, the ring's new range, (batch + 1,)
    int32 first rows of the requests' new tokens, and per new token its position (int32) and slot (int64); rows behind
    the last request have position 0 and slot -1.  seqlens and free_range are new tensors: pass them to the next call
    (a captured step copies them back into those that it was captured with)."""
    what = "pages_resize"
    _require_cuda(seqlens, "seqlens")
    shape, dev = seqlens.shape, seqlens.device
    batch = shape[0] if len(shape) == 1 else 0
    if not 1 <= batch <= _MAX_REQUESTS:
        raise ValueError(f"{what}: seqlens must be (batch,) int32 of 1 to {_MAX_REQUESTS} requests")
    seqlens, targets = _ints(what, "seqlens", seqlens, shape, dev), _ints(what, "targets", targets, shape, dev)
    width = block_table.shape[1] if block_table.dim() == 2 else 0
    if block_table.dtype is not torch.int32 or width < 1 or block_table.shape[0] != batch or block_table.device != dev:
        raise ValueError(f"{what}: block_table must be ({batch}, max_pages) int32 on {dev}")
    row, one = block_table.stride()
    if (one != 1 and width > 1) or (row < width and batch > 1):
        raise ValueError(f"{what}: block_table is written in place, its rows must be dense and apart")
    num_pages = free_pages.numel()
    if free_pages.dtype is not torch.int32 or free_pages.dim() != 1 or num_pages < 1 or free_pages.device != dev \
            or not free_pages.is_contiguous():
        raise ValueError(f"{what}: free_pages must be contiguous (num_pages,) int32 on {dev}")
    free_range = _ints(what, "free_range", free_range, (2,), dev)
    if page_size < 1 or total < 0 or width * page_size >= 2 ** 31 or total >= 2 ** 31:
        raise ValueError(f"{what}: page_size and total must be positive, a row's positions and total below 2^31")
    # (the results of 32 bits are one allocation: three less are 4 us of a call that takes 17)
    lens, left, cu, positions = torch.empty(2 * batch + 3 + total, dtype=torch.int32, device=dev).split_with_sizes(
        (batch, 2, batch + 1, total))
    slots = torch.empty(total, dtype=torch.int64, device=dev)
    with _on(dev):
        at = lens.data_ptr()
        _lib.call("ifv2_pages_resize", seqlens.data_ptr(), targets.data_ptr(), block_table.data_ptr(), row, width,
                  free_pages.data_ptr(), num_pages, free_range.data_ptr(), at, at + 4 * batch, at + 4 * batch + 8,
                  at + 8 * batch + 12, slots.data_ptr(), batch, page_size, total, _stream(dev))
    return lens, left, cu, positions, slots


def _new_rows(what, k, v, slots, heads, dev):
    """(k, its strides, v, its strides, slots) of rows that go to a cache."""
    shape = k.shape
    if (k.dtype is not torch.bfloat16 or v.dtype is not torch.bfloat16 or len(shape) != 3 or shape[1] != heads or shape[2] != HEAD_DIM
            or v.shape != shape or k.device != dev or v.device != dev):
        raise ValueError(f"{what}: k and v must be (total, {heads}, {HEAD_DIM}) bf16 on {dev}")
    _no_gradient(what, k, v)
    if slots.dtype is not torch.int64 or slots.shape != shape[:1] or slots.device != dev:
        raise ValueError(f"{what}: slots must be ({shape[0]},) int64 on {dev}")
    return (*_rows(k), *_rows(v), slots if slots.is_contiguous() else slots.contiguous())


def cache_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor) -> None:
    """Write keys and values (total, nheads_k, 128) bf16 to their slots (total,) int64 of a paged cache (pages, page_size,
    nheads_k, 128) bf16, in place.  A token whose slot is negative or not in the cache goes nowhere; a slot that two
    tokens of one call have is undefined.  One launch."""
    what = "cache_write"
    _require_cuda(k_cache, "k_cache")
    shape, dev = k_cache.shape, k_cache.device
    if k_cache.dtype is not torch.bfloat16 or v_cache.dtype is not torch.bfloat16 or len(shape) != 4 or shape[3] != HEAD_DIM \
            or v_cache.shape != shape or v_cache.device != dev or not k_cache.is_contiguous() or not v_cache.is_contiguous():
        raise ValueError(f"{what}: caches must be contiguous (pages, page_size, nheads_k, {HEAD_DIM}) bf16 on one device")
    if (k_cache.data_ptr() | v_cache.data_ptr()) & 15:
        raise ValueError(f"{what}: caches must begin at a multiple of 16 bytes")
    k, k_token, k_head, v, v_token, v_head, slots = _new_rows(what, k, v, slots, shape[2], dev)
    if k.shape[0] == 0 or shape[0] == 0 or shape[1] == 0 or shape[2] == 0:
        return
    with _on(dev):
        _lib.call("ifv2_cache_write", k.data_ptr(), v.data_ptr(), k_token, k_head, v_token, v_head, k_cache.data_ptr(),
                  v_cache.data_ptr(), slots.data_ptr(), shape[0], shape[1], k.shape[0], shape[2], HEAD_DIM, _stream(dev))


def b8_cache(pages: int, page_size: int, heads_k: int, dtype: torch.dtype = torch.float8_e4m3fn, device="cuda"):
    """An empty cache in 8 bits with block scales (k_cache, v_cache, k_scale, v_scale): zeros of the smallest scale."""
    if dtype not in _CODES:
        raise ValueError("b8_cache: dtype must be torch.float8_e4m3fn or torch.float8_e5m2")
    if page_size < BLOCK_N or page_size % BLOCK_N:
        raise ValueError(f"b8_cache: page_size must be a positive multiple of {BLOCK_N}")
    codes = [torch.zeros(pages, heads_k, page_size, HEAD_DIM, dtype=torch.uint8, device=device).view(dtype) for _ in range(2)]
    scales = [torch.zeros(pages, heads_k, page_size // BLOCK_N, dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu)
              for _ in range(2)]
    return (*codes, *scales)


def _check_b8(what, k_cache, v_cache, k_scale, v_scale):
    """(pages, heads_k, page_size, code, device) of a cache in 8 bits with block scales."""
    _require_cuda(k_cache, "k_cache")
    dtype, shape, dev = k_cache.dtype, k_cache.shape, k_cache.device
    code = _CODES.get(dtype)
    if code is None or v_cache.dtype is not dtype or k_scale.dtype is not torch.float8_e8m0fnu or v_scale.dtype is not torch.float8_e8m0fnu:
        raise ValueError(f"{what}: the caches must be float8_e4m3fn or float8_e5m2, their scales float8_e8m0fnu")
    if len(shape) != 4 or shape[3] != HEAD_DIM or shape[2] % BLOCK_N or shape[2] == 0 or v_cache.shape != shape:
        raise ValueError(f"{what}: caches must be (pages, nheads_k, page_size, {HEAD_DIM}), page_size a multiple of {BLOCK_N}")
    scales = (shape[0], shape[1], shape[2] // BLOCK_N)
    if k_scale.shape != scales or v_scale.shape != scales:
        raise ValueError(f"{what}: scales must be (pages, nheads_k, page_size / {BLOCK_N})")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()):
        raise ValueError(f"{what}: caches and scales must be contiguous")
    if v_cache.device != dev or k_scale.device != dev or v_scale.device != dev:
        raise ValueError(f"{what}: caches and scales must be on one device")
    if (k_cache.data_ptr() | v_cache.data_ptr()) & 15:
        raise ValueError(f"{what}: caches must begin at a multiple of 16 bytes")
    return shape[0], shape[1], shape[2], code, dev


def cache_write_b8(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                   v_scale: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantise keys and values (total, nheads_k, 128) bf16 to their slots (total,) int64 of a cache in 8 bits with block
    scales, in place.  One launch.

    The rows that a call writes into one block are consecutive tokens of the call at consecutive slots, as `pages_resize`
    gives them; a block that a call writes in two pieces is undefined.  Rows that begin a block (place 0 of its 64) give
    it their scale; rows behind others may only raise it, and the earlier codes of the block are then rounded to the new
    one.  What stands behind the written rows of a block is no longer valid.  Tokens whose slot is negative or not in
    the cache go nowhere."""
    what = "cache_write_b8"
    pages, heads, page_size, code, dev = _check_b8(what, k_cache, v_cache, k_scale, v_scale)
    k, k_token, k_head, v, v_token, v_head, slots = _new_rows(what, k, v, slots, heads, dev)
    if k.shape[0] == 0 or pages == 0 or heads == 0:
        return
    with _on(dev):
        _lib.call("ifv2_b8_write", k.data_ptr(), v.data_ptr(), k_token, k_head, v_token, v_head, k_cache.data_ptr(),
                  v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), slots.data_ptr(), pages, page_size, code, k.shape[0],
                  heads, HEAD_DIM, _stream(dev))


@functools.lru_cache(maxsize=256)
def _workspace_bytes(total_q, batch, heads, max_seqlen_q, capacity):
    return int(_lib.load().ifv2_b8_attn_workspace_bytes(total_q, batch, heads, HEAD_DIM, max_seqlen_q, capacity))


def infllmv2_attn_paged_b8(
    q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
    cu_seqlens_q: torch.Tensor, max_seqlen_q: int, cache_seqlens: torch.Tensor, block_table: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None, causal: bool = True, topk_idx: Optional[torch.Tensor] = None,
    block_mask: Optional[torch.Tensor] = None, return_softmax_lse: bool = False,
):
    """Attention of packed query tokens over a cache in 8 bits with block scales: a decode step, drafted tokens, a
    prompt's chunk, or (causal=False) the states of an encoder.

    q: (total_q, nheads, 128) bf16, nheads = 16 * nheads_k; cu_seqlens_q (batch + 1,) int32; max_seqlen_q: no sequence
    has more query tokens.  cache_seqlens (batch,) int32: keys of each sequence, its query tokens' own included.
    causal: the last query token sees all of them, the one before it all but the last, and so on; otherwise every token
    sees all.  block_table (batch, max_pages) int32, or None: sequence b is page b.  topk_idx: int32 (nheads_k, total_q,
    topk) 64-token blocks that a token attends, -1 unused, or block_mask: the same packed, int64 (nheads_k, total_q,
    words) with a word per 64 blocks of a sequence's capacity; None = all.
    Tokens that see no key get 0 (softmax_lse +inf), and so do rows behind the last sequence.  A token that sees a key of a
    NaN block, or of a page that the cache does not have, gets NaN.  Codes are finite (cache_write_b8 writes no others).
    A sequence with more than max_seqlen_q tokens has rows that are not written, and rows of a request that `pages_resize`
    refused (slots -1) mean nothing.  Blocks are selected among at most 524288 keys of capacity.  Weights are rounded to 9 bits
    (2^-9 + 2^-11 of each) where max_seqlen_q is 1 or 2, to fp16 (2^-11) elsewhere, queries to 2^-17.8 of the row's largest
    element; scores must stay in fp32's range.  Where max_seqlen_q is 1 or 2, values of a block that are more than 2^90 below
    the largest block's of those that the token attends (without a selection: the sequence's tokens) count as 0.
    Returns out (total_q, nheads, 128) [, softmax_lse (total_q, nheads) fp32].  Forward only."""
    what = "infllmv2_attn_paged_b8"
    pages, hk, length, code, dev = _check_b8(what, k_cache, v_cache, k_scale, v_scale)
    heads, shape = hk * GROUP, q.shape
    if q.dtype is not torch.bfloat16 or len(shape) != 3 or shape[1] != heads or shape[2] != HEAD_DIM or q.device != dev:
        raise ValueError(f"{what}: q must be (total_q, {heads}, {HEAD_DIM}) bf16 ({GROUP} heads per KV head) on the cache's device")
    if q.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(f"{what}: forward only, as infllmv2_attn_with_kvcache")
    _no_tangent(what, q)
    total = shape[0]
    cu_seqlens_q, batch = _cu(what, cu_seqlens_q, dev)
    cache_seqlens = _ints(what, "cache_seqlens", cache_seqlens, (batch,), dev)
    if not 1 <= max_seqlen_q < 2 ** 31:
        raise ValueError(f"{what}: max_seqlen_q must be positive and below 2^31")
    width, cap = 0, length
    if block_table is not None:
        block_table, width = _table(what, block_table, batch, dev)
        cap = width * length
    elif pages < batch:
        raise ValueError(f"{what}: {batch} sequences need as many pages, or a block_table")
    words = (cap + 64 * BLOCK_N - 1) // (64 * BLOCK_N)
    if block_mask is not None:
        if topk_idx is not None or block_mask.dtype is not torch.int64 or block_mask.device != dev or block_mask.shape != (hk, total, words):
            raise ValueError(f"{what}: block_mask must be ({hk}, {total}, {words}) int64 on {dev} and excludes topk_idx")
        block_mask = block_mask.contiguous()
    elif topk_idx is not None:
        if topk_idx.dtype is not torch.int32 or topk_idx.device != dev or topk_idx.dim() != 3 or topk_idx.shape[:2] != (hk, total):
            raise ValueError(f"{what}: topk_idx must be ({hk}, {total}, topk) int32 on {dev}")
        topk_idx = topk_idx.contiguous()
        if topk_idx.shape[2] == 0:                     # (a list of no entries has no address)
            topk_idx = torch.full((hk, total, 1), -1, dtype=torch.int32, device=dev)
    q = q.contiguous()
    if q.data_ptr() & 15:
        q = q.clone()
    out = torch.empty_like(q)
    lse = torch.empty(total, heads, dtype=torch.float32, device=dev) if return_softmax_lse else None
    if total and hk:
        ws_bytes = _workspace_bytes(total, batch, heads, max_seqlen_q, cap)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        with _on(dev):
            _lib.call("ifv2_b8_attn", q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                      out.data_ptr(), _ptr(lse), cu_seqlens_q.data_ptr(), cache_seqlens.data_ptr(), _ptr(block_table), width,
                      _ptr(topk_idx), topk_idx.shape[2] if topk_idx is not None else 0, _ptr(block_mask),
                      words if block_mask is not None else 0, batch, total, max_seqlen_q, pages, length, code, heads,
                      hk, HEAD_DIM, HEAD_DIM ** -0.5 if softmax_scale is None else float(softmax_scale), 1 if causal else 0,
                      ws.data_ptr(), ws_bytes, _status_words(dev).data_ptr(), _stream(dev))
    return (out, lse) if return_softmax_lse else out

"""A key-value cache in 8 bits: writing, reading back, and the attention of one new token over it.

Counterparts of `cache_fill`, `decode_append` and `infllmv2_attn_with_kvcache` for a cache whose rows are 128 codes
(torch.float8_e4m3fn or torch.int8) and one power-of-two scale (torch.float8_e8m0fnu): 129 bytes instead of 256.

The cache is kept head by head, so that a block of keys of one head is one run of memory:
    k_cache, v_cache  (slots, nheads_k, length, 128)        k_scale, v_scale  (slots, nheads_k, length)
A slot is a sequence of up to `length` tokens, or with a block_table (batch, max_pages) int32 a page of `length`.
A row's value is code * scale.  The scale is the smallest power of two (at least 2^-127) with which the row's largest
magnitude fits the codes (448 or 127), codes are rounded to nearest even, and reading back is exact.  A row with an
infinity or a NaN reads back as NaN.  Writes to pages, slots or positions that the cache does not have are dropped,
reads of them give NaN.  Where two tokens of one call go to the same row (a page twice in a block_table, sequences that
share a slot at one length) that row is undefined: codes and scale may come from different tokens.  No other row is
touched."""
import functools
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _lib
from .attention import BLOCK_N, GROUP, HEAD_DIM
from .ops import _on, _require_cuda, _stream
from .rotary import _no_gradient as _no_table_gradient, _rows, _tables

_LIST = 256      # longest block list that the attention takes without a mask
_CODES = {torch.float8_e4m3fn: 0, torch.int8: 1}


def q8_cache(slots: int, length: int, heads_k: int, dtype: torch.dtype = torch.float8_e4m3fn, device="cuda"):
    """An empty cache (k_cache, v_cache, k_scale, v_scale): zeros of the smallest scale."""
    if dtype not in _CODES:
        raise ValueError("q8_cache: dtype must be torch.float8_e4m3fn or torch.int8")
    codes = [torch.zeros(slots, heads_k, length, HEAD_DIM, dtype=torch.uint8, device=device).view(dtype) for _ in range(2)]
    scales = [torch.zeros(slots, heads_k, length, dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu) for _ in range(2)]
    return (*codes, *scales)


def _check_cache(what, k_cache, v_cache, k_scale, v_scale):
    """(slots, heads_k, length, code, device) of a cache."""
    _require_cuda(k_cache, "k_cache")
    dtype, shape, dev = k_cache.dtype, k_cache.shape, k_cache.device
    code = _CODES.get(dtype)
    if code is None or v_cache.dtype is not dtype or k_scale.dtype is not torch.float8_e8m0fnu or v_scale.dtype is not torch.float8_e8m0fnu:
        raise ValueError(f"{what}: the caches must be float8_e4m3fn or int8, their scales float8_e8m0fnu")
    rows = shape[:3]
    if len(shape) != 4 or shape[3] != HEAD_DIM or v_cache.shape != shape or k_scale.shape != rows or v_scale.shape != rows:
        raise ValueError(f"{what}: caches must be (slots, heads_k, length, {HEAD_DIM}), their scales (slots, heads_k, length)")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()):
        raise ValueError(f"{what}: caches and scales must be contiguous")
    if v_cache.device != dev or k_scale.device != dev or v_scale.device != dev:
        raise ValueError(f"{what}: caches and scales must be on one device")
    return shape[0], shape[1], shape[2], code, dev


def _ints(what, name, t, shape, dev):
    """An int32 tensor of the given shape on dev, contiguous."""
    if t is None:
        return None
    if t.dtype is not torch.int32 or t.shape != shape or t.device != dev:
        raise ValueError(f"{what}: {name} must be {shape} int32 on {dev}")
    return t if t.is_contiguous() else t.contiguous()


def _table(what, block_table, batch, dev):
    if block_table is None:
        return None, 0
    shape = block_table.shape
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError(f"{what}: block_table must be (batch, max_pages) int32")
    return _ints(what, "block_table", block_table, (batch, shape[1]), dev), shape[1]


@functools.lru_cache(maxsize=256)
def _workspace_bytes(batch, heads):
    return int(_lib.load().ifv2_q8_decode_workspace_bytes(batch, heads, HEAD_DIM))


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _cu(what, cu_seqlens, dev):
    shape = cu_seqlens.shape
    if cu_seqlens.dtype is not torch.int32 or len(shape) != 1 or shape[0] < 2 or cu_seqlens.device != dev:
        raise ValueError(f"{what}: cu_seqlens must be (batch + 1,) int32 on {dev}")
    return cu_seqlens if cu_seqlens.is_contiguous() else cu_seqlens.contiguous(), shape[0] - 1


def _no_gradient(what, k, v):
    if (k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
        raise NotImplementedError(f"{what}: nothing flows back from a cache (pass k.detach() and v.detach())")


def cache_fill_q8(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                  v_scale: torch.Tensor, cu_seqlens: torch.Tensor, start: Optional[torch.Tensor] = None,
                  block_table: Optional[torch.Tensor] = None, seqlens_out: Optional[torch.Tensor] = None) -> None:
    """Quantise the packed rows of every sequence (k, v: (total, nheads_k, 128) bf16, cu_seqlens (batch + 1,) int32)
    into positions start[b], start[b] + 1, ... of its slot or pages, in place.  start (batch,) int32, default 0;
    seqlens_out (batch,) int32, optional: min(start[b] + len_b, capacity).  One launch."""
    what = "cache_fill_q8"
    slots, hk, length, code, dev = _check_cache(what, k_cache, v_cache, k_scale, v_scale)
    shape = k.shape
    if (k.dtype is not torch.bfloat16 or v.dtype is not torch.bfloat16 or len(shape) != 3 or shape[1] != hk or shape[2] != HEAD_DIM
            or v.shape != shape or k.device != dev or v.device != dev):
        raise ValueError(f"{what}: k and v must be (total, {hk}, {HEAD_DIM}) bf16 on {dev}")
    _no_gradient(what, k, v)
    cu_seqlens, batch = _cu(what, cu_seqlens, dev)
    block_table, pages = _table(what, block_table, batch, dev)
    if block_table is None and slots < batch:
        raise ValueError(f"{what}: {batch} sequences need as many slots")
    start = _ints(what, "start", start, (batch,), dev)
    if seqlens_out is not None and (_ints(what, "seqlens_out", seqlens_out, (batch,), dev) is not seqlens_out
                                    or (start is not None and seqlens_out.data_ptr() == start.data_ptr())):
        raise ValueError(f"{what}: seqlens_out must be contiguous and not start itself")
    (k, k_token, k_head), (v, v_token, v_head) = _rows(k), _rows(v)
    with _on(dev):
        _lib.call("ifv2_q8_fill", k.data_ptr(), v.data_ptr(), k_token, k_head, v_token, v_head,
                  k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), cu_seqlens.data_ptr(),
                  _ptr(start), _ptr(block_table), pages, _ptr(seqlens_out), slots, length, code, batch, shape[0], hk,
                  HEAD_DIM, _stream(dev))


def cache_read_q8(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                  cu_seqlens: torch.Tensor, total: int, start: Optional[torch.Tensor] = None,
                  block_table: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows of the cache as packed keys and values (total, nheads_k, 128) bf16, exactly: cu_seqlens[b + 1] -
    cu_seqlens[b] rows of every sequence from position start[b] (default 0) on.  total: their number (rows past
    cu_seqlens[-1] are zeros).  What the next chunk of a prompt attends through infllmv2_attn_varlen_func."""
    what = "cache_read_q8"
    slots, hk, length, code, dev = _check_cache(what, k_cache, v_cache, k_scale, v_scale)
    cu_seqlens, batch = _cu(what, cu_seqlens, dev)
    block_table, pages = _table(what, block_table, batch, dev)
    if block_table is None and slots < batch:
        raise ValueError(f"{what}: {batch} sequences need as many slots")
    start = _ints(what, "start", start, (batch,), dev)
    if total < 0:
        raise ValueError(f"{what}: total must not be negative")
    k = torch.empty_strided((total, hk, HEAD_DIM), (hk * HEAD_DIM, HEAD_DIM, 1), dtype=torch.bfloat16, device=dev)
    v = torch.empty_like(k)
    with _on(dev):
        _lib.call("ifv2_q8_read", k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), k.data_ptr(),
                  v.data_ptr(), cu_seqlens.data_ptr(), _ptr(start), _ptr(block_table), pages, slots, length, code, batch,
                  total, hk, HEAD_DIM, _stream(dev))
    return k, v


def decode_append_q8(k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                     k_scale: torch.Tensor, v_scale: torch.Tensor, cache_seqlens: torch.Tensor,
                     positions: Optional[torch.Tensor] = None, kc_cache: Optional[torch.Tensor] = None,
                     n_comp: Optional[torch.Tensor] = None, kernel_size: int = 32, kernel_stride: int = 16,
                     kc2_cache: Optional[torch.Tensor] = None, n_comp2: Optional[torch.Tensor] = None,
                     kernel2_size: int = 128, kernel2_stride: int = 64) -> None:
    """`decode_append` for a cache in 8 bits (slots): k_new / v_new (batch, nheads_k, 128) are quantised into
    position cache_seqlens[b], completed windows of compressed keys become the mean of the keys as the cache holds
    them (kc_cache (batch, c_capacity, nheads_k, 128) bf16), lengths advance in place.  One launch."""
    what = "decode_append_q8"
    slots, hk, cap, code, dev = _check_cache(what, k_cache, v_cache, k_scale, v_scale)
    b = cache_seqlens.numel()
    for name, t in (("k_new", k_new), ("v_new", v_new)):
        if t.dtype != torch.bfloat16 or t.device != dev or not t.is_contiguous() or t.numel() != b * hk * HEAD_DIM:
            raise ValueError(f"{what}: {name} must be contiguous ({b}, {hk}, {HEAD_DIM}) bf16 on {dev}")
    _no_gradient(what, k_new, v_new)
    if slots < b:
        raise ValueError(f"{what}: {b} sequences need as many slots")
    for name, t in (("cache_seqlens", cache_seqlens), ("positions", positions), ("n_comp", n_comp), ("n_comp2", n_comp2)):
        if t is not None and (t.dtype != torch.int32 or t.device != dev or not t.is_contiguous() or t.numel() != b):
            raise ValueError(f"{what}: {name} must be contiguous ({b},) int32 on {dev}")
    for c in (kc_cache, kc2_cache):
        if c is not None and (c.dtype != torch.bfloat16 or c.device != dev or not c.is_contiguous() or c.dim() != 4
                              or c.shape[0] != b or c.shape[2:] != (hk, HEAD_DIM)):
            raise ValueError(f"{what}: a compressed cache must be contiguous ({b}, c_capacity, {hk}, {HEAD_DIM}) bf16")
    with _on(dev):
        _lib.call("ifv2_q8_append", k_new.data_ptr(), v_new.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                  k_scale.data_ptr(), v_scale.data_ptr(), _ptr(kc_cache), _ptr(kc2_cache), cache_seqlens.data_ptr(),
                  _ptr(positions), _ptr(n_comp), _ptr(n_comp2), code, b, slots, cap,
                  kc_cache.shape[1] if kc_cache is not None else 0, kc2_cache.shape[1] if kc2_cache is not None else 0, hk,
                  HEAD_DIM, kernel_size, kernel_stride, kernel2_size, kernel2_stride, _stream(dev))


def infllmv2_attn_with_kvcache_q8(
    q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
    k: Optional[torch.Tensor] = None, v: Optional[torch.Tensor] = None, rotary_cos: Optional[torch.Tensor] = None,
    rotary_sin: Optional[torch.Tensor] = None, rotary_positions: Optional[torch.Tensor] = None,
    rotary_sections: Optional[Sequence[int]] = None, cache_seqlens: Optional[Union[int, torch.Tensor]] = None,
    cache_batch_idx: Optional[torch.Tensor] = None, block_table: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None, rotary_interleaved: bool = True, return_softmax_lse: bool = False,
    topk_idx: Optional[torch.Tensor] = None, block_mask: Optional[torch.Tensor] = None,
):
    """`infllmv2_attn_with_kvcache` over a cache in 8 bits: one new query token per sequence.

    q: (batch, 1, nheads, 128) bf16, nheads = 16 * nheads_k.  k, v: optional (batch, 1, nheads_k, 128), quantised
    into position cache_seqlens[b] first, in place.  cache_seqlens: int or (batch,) int32 (default: the whole
    capacity).  cache_batch_idx (batch,) int32: the slot each sequence uses.  block_table (batch, max_pages) int32:
    slots are pages, of a multiple of 16 positions.  topk_idx: int32 (batch, nheads_k, 1, topk) 64-token blocks to
    attend (None = all), or block_mask: the same packed, int64 (batch, nheads_k, 1, words); the 1 may be missing.
    rotary_cos / rotary_sin (positions, rotary_dim / 2) fp32 rotate the query and the appended key, as `rotary_axes`
    does, at rotary_positions ((batch,) or (axes, batch) int32 with rotary_sections; default: cache_seqlens); without
    an append nothing is rotated.  The rotated rows are not rounded to bf16 in between.
    A new token without room in the cache is neither written nor attended.  A sequence without keys gets 0
    (softmax_lse +inf), one that attends a key in a page or slot that the cache does not have NaN (softmax_lse too).
    Returns out (batch, 1, nheads, 128) [, softmax_lse (batch, nheads, 1) fp32].  Forward only."""
    what = "infllmv2_attn_with_kvcache_q8"
    slots, hk, length, code, dev = _check_cache(what, k_cache, v_cache, k_scale, v_scale)
    shape = q.shape
    batch, heads = shape[0], hk * GROUP
    if q.dtype is not torch.bfloat16 or shape != (batch, 1, heads, HEAD_DIM) or q.device != dev:
        raise ValueError(f"{what}: q must be (batch, 1, {heads}, {HEAD_DIM}) bf16 ({GROUP} heads per KV head) on the "
                         "cache's device")
    if q.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(f"{what}: forward only, as infllmv2_attn_with_kvcache")
    k_ptr = v_ptr = None
    if k is not None and v is not None:
        new = (batch, 1, hk, HEAD_DIM)
        if (k.dtype is not torch.bfloat16 or v.dtype is not torch.bfloat16 or k.shape != new or v.shape != new
                or k.device != dev or v.device != dev):
            raise ValueError(f"{what}: k and v must be {new} bf16 on {dev}")
        _no_gradient(what, k, v)
        k, v = k.contiguous(), v.contiguous()
        k_ptr, v_ptr = k.data_ptr(), v.data_ptr()
    elif k is not None or v is not None:
        raise ValueError(f"{what}: pass both k and v, or neither")
    if (rotary_cos is None) != (rotary_sin is None):
        raise ValueError(f"{what}: pass both rotary_cos and rotary_sin, or neither")
    pages, cap = 0, length
    if block_table is not None:
        block_table, pages = _table(what, block_table, batch, dev)
        if cache_batch_idx is not None:
            raise NotImplementedError(f"{what}: a paged cache takes no cache_batch_idx")
        if length % 16 != 0:
            raise NotImplementedError(f"{what}: page size must be a multiple of 16")
        cap = pages * length
    elif cache_batch_idx is not None:
        cache_batch_idx = _ints(what, "cache_batch_idx", cache_batch_idx, (batch,), dev)
    elif slots < batch:
        raise ValueError(f"{what}: {batch} sequences need as many slots, or cache_batch_idx")
    if cache_seqlens is None:
        cache_seqlens = cap
    if isinstance(cache_seqlens, int):
        cache_seqlens = torch.full((batch,), cache_seqlens, dtype=torch.int32, device=dev)
    cache_seqlens = _ints(what, "cache_seqlens", cache_seqlens, (batch,), dev)
    mask_ptr, idx_ptr, words, topk = None, None, 0, 0
    if block_mask is not None:
        words = (cap + 64 * BLOCK_N - 1) // (64 * BLOCK_N)
        if topk_idx is not None or block_mask.dtype is not torch.int64 or block_mask.device != dev \
                or block_mask.shape not in ((batch, hk, 1, words), (batch, hk, words)):
            raise ValueError(f"{what}: block_mask must be ({batch}, {hk}, 1, {words}) int64 on {dev} and excludes topk_idx")
        block_mask = block_mask.contiguous()
        mask_ptr = block_mask.data_ptr()
    elif topk_idx is not None:
        words = (cap + 64 * BLOCK_N - 1) // (64 * BLOCK_N)
        shape = topk_idx.shape
        if topk_idx.dtype is not torch.int32 or topk_idx.device != dev or len(shape) not in (3, 4) \
                or shape[:-1] not in ((batch, hk, 1), (batch, hk)):
            raise ValueError(f"{what}: topk_idx must be ({batch}, {hk}, 1, topk) int32 on {dev}")
        topk_idx, topk = topk_idx.contiguous(), shape[-1]
        idx_ptr = topk_idx.data_ptr()
        if topk > _LIST or topk == 0:                    # (shorter lists are walked as they are; one of no entries has no address)
            block_mask = (torch.zeros if topk == 0 else torch.empty)(batch, hk, 1, words, dtype=torch.int64, device=dev)
            mask_ptr = block_mask.data_ptr()
    rotary = (None, None, None, 0, None, 0, 0, 0)
    if rotary_cos is not None and k is not None:
        _no_table_gradient(what, rotary_cos, rotary_sin)
        if rotary_sections is not None and type(rotary_sections) is not tuple:
            rotary_sections = tuple(rotary_sections)
        cos, sin, at, axis_stride, pair_axis, axes, rows, pairs = _tables(
            what, rotary_cos, rotary_sin, cache_seqlens if rotary_positions is None else rotary_positions, rotary_sections,
            batch, dev)
        rotary = (cos.data_ptr(), sin.data_ptr(), at.data_ptr(), axis_stride, pair_axis, axes, 2 * pairs, rows)
    q = q.contiguous()
    out = torch.empty_like(q)
    lse = torch.empty_strided((batch, heads, 1), (heads, 1, 1), dtype=torch.float32, device=dev) if return_softmax_lse else None
    ws_bytes = _workspace_bytes(batch, heads)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    with _on(dev):
        _lib.call("ifv2_q8_decode", q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(),
                  v_scale.data_ptr(), k_ptr, v_ptr, *rotary, 1 if rotary_interleaved else 0, idx_ptr, topk, mask_ptr, words,
                  out.data_ptr(), _ptr(lse), cache_seqlens.data_ptr(), _ptr(cache_batch_idx), _ptr(block_table), pages,
                  slots, length, code, batch, heads, hk, HEAD_DIM, HEAD_DIM ** (-0.5) if softmax_scale is None else float(softmax_scale),
                  ws.data_ptr(), ws_bytes, _stream(dev))
    return (out, lse) if return_softmax_lse else out

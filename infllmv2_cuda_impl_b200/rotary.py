"""Rotary positions over several axes, for the packed queries and keys in front of the attention operators.

The reference rotates by one axis, inside its decode (rotary_cos / rotary_sin of
infllm_v2/infllmv2_sparse_attention.py:609-630); `rotary_axes` is the operator for prompts and training, and for
tokens whose position has several coordinates (time, height and width of images and video)."""
import functools
from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from .ops import _on, _plain_eager, _require_cuda, _stream

_forward_ad = torch.autograd.forward_ad
_profiled = torch.autograd._profiler_enabled
HEAD_DIM = 128
MAX_AXES = 4


@functools.lru_cache(maxsize=256)
def _pair_axis(sections, pairs: int, axes: int) -> Optional[bytes]:
    """Axis number of every pair, from the number of pairs of each axis; None for one axis."""
    if sections is None:
        if axes != 1:
            raise ValueError("rotary: positions on several axes need sections")
        return None
    if len(sections) != axes or sum(sections) != pairs or min(sections) < 0 or any(type(n) is not int for n in sections):
        raise ValueError(f"rotary: sections must be {axes} counts (one per axis of positions) that sum up to {pairs} pairs, "
                         f"got {sections}")
    return b"".join(bytes([a]) * n for a, n in enumerate(sections))


def _no_gradient(what, rotary_cos, rotary_sin):
    """(Of the caller's own tensors: below the registered operator, and where a compiler traces it, nobody would ask.)"""
    if rotary_cos.requires_grad or rotary_sin.requires_grad:
        raise NotImplementedError(f"{what}: the tables get no gradient")


def _tables(what, rotary_cos, rotary_sin, positions, sections, tokens, device):
    """Checks of the arguments that every rotating call takes; (cos, sin, positions, axis_stride, pair_axis, axes, rows,
    pairs).  (These calls are bound by their host time where tokens are few, so a check costs one attribute.)"""
    shape, at = rotary_cos.shape, positions.shape
    if (rotary_cos.dtype is not torch.float32 or rotary_sin.dtype is not torch.float32 or len(shape) != 2
            or rotary_sin.shape != shape or rotary_cos.device != device or rotary_sin.device != device):
        raise ValueError(f"{what}: rotary_cos and rotary_sin must be (positions, rotary_dim / 2) fp32 on {device}, of one shape")
    rows, pairs = shape
    if pairs < 8 or pairs > HEAD_DIM // 2 or pairs % 8 != 0 or rows < 1:
        raise ValueError(f"{what}: rotary_dim must be a positive multiple of 16 up to {HEAD_DIM}, and the tables hold a position")
    if positions.dtype is not torch.int32 or len(at) not in (1, 2) or at[-1] != tokens or positions.device != device:
        raise ValueError(f"{what}: positions must be ({tokens},) or (axes, {tokens}) int32 on {device}")
    axes, axis_stride = 1, 0
    if len(at) == 2:
        axes = at[0]
        if not 1 <= axes <= MAX_AXES:
            raise ValueError(f"{what}: 1 to {MAX_AXES} axes, got {axes}")
        strides = positions.stride()
        if strides[1] != 1 and tokens > 1:
            positions = positions.contiguous()
            strides = positions.stride()
        axis_stride = strides[0]
    elif not positions.is_contiguous():
        positions = positions.contiguous()
    return (rotary_cos.contiguous(), rotary_sin.contiguous(), positions, axis_stride, _pair_axis(tuple(sections) if type(sections) is list else sections, pairs, axes), axes, rows,
            pairs)


def _rows(x):
    """(x, its first two strides) with unit stride in the features and rows on 16-byte boundaries; copied only where it
    has to be."""
    a, b, c = x.stride()
    if c != 1 or (a | b) & 7 or x.data_ptr() & 15:
        x = x.clone(memory_format=torch.contiguous_format)
        a, b, c = x.stride()
    return x, a, b


def _dense_like(x):
    """An empty (tokens, heads, 128) tensor of x's kind, dense in this order.  (torch.empty takes twice the time.)"""
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _turn(q, k, tables, interleaved, back):
    """(q, k) rotated, dense; k may be None.  tables: what `_tables` returns."""
    cos, sin, positions, axis_stride, pair_axis, axes, rows, pairs = tables
    dev, (tokens, heads, _) = q.device, q.shape
    q, q_token, q_head = _rows(q)
    q_out = _dense_like(q)
    k_out = k_ptr = k_out_ptr = None
    heads_k = k_token = k_head = 0
    if k is not None:
        k, k_token, k_head = _rows(k)
        heads_k = k.shape[1]
        k_out = _dense_like(k)
        k_ptr, k_out_ptr = k.data_ptr(), k_out.data_ptr()
    with _on(dev):
        _lib.call("ifv2_rotary_axes", q.data_ptr(), k_ptr, q_out.data_ptr(), k_out_ptr, cos.data_ptr(), sin.data_ptr(),
                  positions.data_ptr(), axis_stride, pair_axis, axes, tokens, heads, heads_k, HEAD_DIM, q_token, q_head,
                  k_token, k_head, 2 * pairs, rows, interleaved, back, _stream(dev))
    return q_out, k_out


@torch.library.custom_op("infllmv2_attn::_rotary_axes", mutates_args=(), device_types="cuda")
def _rotary_axes(q: torch.Tensor, k: Optional[torch.Tensor], rotary_cos: torch.Tensor, rotary_sin: torch.Tensor,
                 positions: torch.Tensor, sections: Optional[Sequence[int]], interleaved: bool,
                 back: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    """`_turn` as a registered operator (an empty second result without k)."""
    tables = _tables("rotary_axes", rotary_cos, rotary_sin, positions, None if sections is None else tuple(sections), q.shape[0],
                     q.device)
    q_out, k_out = _turn(q, k, tables, interleaved, back)
    return q_out, k_out if k_out is not None else q_out.new_empty(0)


@_rotary_axes.register_fake
def _(q, k, rotary_cos, rotary_sin, positions, sections, interleaved, back):
    return q.new_empty(q.shape), k.new_empty(k.shape) if k is not None else q.new_empty(0)


def _direct(*tensors) -> bool:
    """True where nothing watches operators: the body is called then, the registered operator elsewhere."""
    return not torch.compiler.is_compiling() and not _profiled() and _plain_eager(*tensors)


def _registered(q, k, rotary_cos, rotary_sin, positions, sections, interleaved, back):
    q, k_out = _rotary_axes(q, k, rotary_cos, rotary_sin, positions, None if sections is None else list(sections), interleaved, back)
    return q, k_out if k is not None else None


class RotaryAxesFunc(torch.autograd.Function):
    """A rotation is linear: its gradient is the rotation by minus the angle, and so on to any order."""

    @staticmethod
    def forward(ctx, q, k, rotary_cos, rotary_sin, positions, sections, interleaved, back):
        ctx.sections, ctx.interleaved, ctx.back = sections, interleaved, back
        ctx.set_materialize_grads(False)
        if _direct(q, k, rotary_cos, rotary_sin, positions):
            tables = _tables("rotary_axes", rotary_cos, rotary_sin, positions, sections, q.shape[0], q.device)
            ctx.save_for_backward(*tables[:3])
            return _turn(q, k, tables, interleaved, back)
        ctx.save_for_backward(rotary_cos, rotary_sin, positions)
        return _registered(q, k, rotary_cos, rotary_sin, positions, sections, interleaved, back)

    @staticmethod
    def backward(ctx, dq, dk):
        dq = dq if ctx.needs_input_grad[0] else None
        dk = dk if ctx.needs_input_grad[1] else None
        one, other = (dk, None) if dq is None else (dq, dk)      # the body wants a first tensor
        if one is None:
            return (None,) * 8
        # (a saved-tensor hook may give a saved tensor back with other strides: nothing that the forward pass knew of
        # their layout holds here)
        one, other = _rotary_maybe_grad(one, other, *ctx.saved_tensors, ctx.sections, ctx.interleaved, not ctx.back)
        return ((None, one) if dq is None else (one, other)) + (None,) * 6


class RotaryAxesDualFunc(RotaryAxesFunc):
    """The same where a forward-mode level is open: a tangent turns as the rows do.  (Apart, because torch.compile takes
    no Function with a jvp.)"""

    @staticmethod
    def forward(ctx, q, k, rotary_cos, rotary_sin, positions, sections, interleaved, back):
        ctx.save_for_forward(rotary_cos, rotary_sin, positions)
        ctx.shapes = q.shape, None if k is None else k.shape
        return RotaryAxesFunc.forward(ctx, q, k, rotary_cos, rotary_sin, positions, sections, interleaved, back)

    @staticmethod
    def jvp(ctx, tq, tk, t_cos, t_sin, *_):
        if t_cos is not None or t_sin is not None:
            raise NotImplementedError("rotary_axes: the tables get no gradient")
        one, other = (tk, None) if tq is None else (tq, tk)
        turned, other = _rotary_maybe_grad(one, other, *ctx.saved_tensors, ctx.sections, ctx.interleaved, ctx.back)
        both = (None, turned) if tq is None else (turned, other)
        # (a result that is a tensor needs a tangent)
        return tuple(turned.new_zeros(n) if t is None and n is not None else t for t, n in zip(both, ctx.shapes))


def _rotary_maybe_grad(q, k, rotary_cos, rotary_sin, positions, sections, interleaved, back):
    if _forward_ad._current_level >= 0:                # (a tensor with a tangent need not require a gradient)
        return RotaryAxesDualFunc.apply(q, k, rotary_cos, rotary_sin, positions, sections, interleaved, back)
    if (q.requires_grad or (k is not None and k.requires_grad)) and torch.is_grad_enabled():
        return RotaryAxesFunc.apply(q, k, rotary_cos, rotary_sin, positions, sections, interleaved, back)
    if _direct(q, k, rotary_cos, rotary_sin, positions):
        return _turn(q, k, _tables("rotary_axes", rotary_cos, rotary_sin, positions, sections, q.shape[0], q.device),
                     interleaved, back)
    return _registered(q, k, rotary_cos, rotary_sin, positions, sections, interleaved, back)


def rotary_axes(q: torch.Tensor, k: Optional[torch.Tensor], rotary_cos: torch.Tensor, rotary_sin: torch.Tensor,
                positions: torch.Tensor, sections: Optional[Sequence[int]] = None, interleaved: bool = True):
    """Rotary positions of packed queries and keys, differentiable in q and k.

    q: (tokens, nheads, 128), k: (tokens, nheads_k, 128) or None, bf16; slices of one projection are taken as they
    are (rows on 16-byte boundaries).  rotary_cos / rotary_sin: (positions, rotary_dim / 2) fp32, rotary_dim a
    multiple of 16 up to 128.  positions: (tokens,) int32, or (axes, tokens) for up to four axes; sections: with
    several axes, how many of the rotary_dim / 2 pairs turn by the position on each (in order).  Pairs are features
    (2i, 2i+1) if interleaved, else (i, i + rotary_dim / 2); features from rotary_dim on pass through.  The
    arithmetic is fp32, the results are rounded once.  A position outside the tables takes their first or last row.
    Returns (q, k) rotated (k None without one), dense.

    A backward pass that is captured into a CUDA graph must not share its leaves with an eager graph that is still alive
    (as for any operator: autograd would end the process)."""
    shape = q.shape
    if q.dtype is not torch.bfloat16 or len(shape) != 3 or shape[2] != HEAD_DIM:
        raise ValueError(f"rotary_axes: q must be (tokens, nheads, {HEAD_DIM}) bf16")
    _require_cuda(q, "q")
    if k is not None:
        other = k.shape
        if k.dtype is not torch.bfloat16 or len(other) != 3 or other[2] != HEAD_DIM or other[0] != shape[0] or k.device != q.device:
            raise ValueError(f"rotary_axes: k must be (tokens, nheads_k, {HEAD_DIM}) bf16, with the tokens and on the device of q")
    _no_gradient("rotary_axes", rotary_cos, rotary_sin)
    if sections is not None and type(sections) is not tuple:
        sections = tuple(sections)
    return _rotary_maybe_grad(q, k, rotary_cos, rotary_sin, positions, sections, bool(interleaved), False)

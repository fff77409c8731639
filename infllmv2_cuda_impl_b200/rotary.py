"""Rotary positions over several axes, for the packed queries and keys in front of the attention operators.

The reference rotates by one axis, inside its decode (rotary_cos / rotary_sin of
infllm_v2/infllmv2_sparse_attention.py:609-630); `rotary_axes` is the operator for prompts and training, and for
tokens whose position has several coordinates (time, height and width of images and video)."""
import functools
from typing import Optional, Sequence, Tuple

import torch

from . import _lib
from .ops import _on, _plain_eager, _require_cuda, _stream

HEAD_DIM = 128
MAX_AXES = 4


@functools.lru_cache(maxsize=256)
def _pair_axis(sections, pairs: int, axes: int) -> Optional[bytes]:
    """Axis number of every pair, from the number of pairs of each axis; None for one axis."""
    if sections is None:
        if axes != 1:
            raise ValueError("rotary: positions on several axes need sections")
        return None
    if len(sections) != axes or sum(sections) != pairs or min(sections) < 0:
        raise ValueError(f"rotary: sections must be {axes} counts (one per axis of positions) that sum up to {pairs} pairs, "
                         f"got {tuple(sections)}")
    return b"".join(bytes([a]) * n for a, n in enumerate(sections))


def _tables(what, rotary_cos, rotary_sin, positions, sections, tokens, device):
    """Checks of the arguments that every rotating call takes; (cos, sin, positions, axis_stride, pair_axis, axes)."""
    for name, t in (("rotary_cos", rotary_cos), ("rotary_sin", rotary_sin)):
        if t.dtype != torch.float32 or t.dim() != 2 or t.shape != rotary_cos.shape or t.device != device:
            raise ValueError(f"{what}: {name} must be (positions, rotary_dim / 2) fp32 on {device}, as the other table")
        if t.requires_grad:
            raise NotImplementedError(f"{what}: the tables get no gradient")
    pairs = rotary_cos.shape[1]
    if pairs < 8 or pairs > HEAD_DIM // 2 or pairs % 8 != 0 or rotary_cos.shape[0] < 1:
        raise ValueError(f"{what}: rotary_dim must be a positive multiple of 16 up to {HEAD_DIM}, and the tables hold a position")
    if positions.dtype != torch.int32 or positions.device != device or positions.dim() not in (1, 2) or positions.shape[-1] != tokens:
        raise ValueError(f"{what}: positions must be ({tokens},) or (axes, {tokens}) int32 on {device}")
    axes = positions.shape[0] if positions.dim() == 2 else 1
    if not 1 <= axes <= MAX_AXES:
        raise ValueError(f"{what}: 1 to {MAX_AXES} axes, got {axes}")
    if positions.stride(-1) != 1 and tokens > 1:
        positions = positions.contiguous()
    pair_axis = _pair_axis(None if sections is None else tuple(sections), pairs, axes)
    return (rotary_cos.contiguous(), rotary_sin.contiguous(), positions, positions.stride(0) if positions.dim() == 2 else 0,
            pair_axis, axes)


def _rows(x):
    """x with unit stride in the features and rows on 16-byte boundaries; copied only where it has to be."""
    if x.stride(-1) == 1 and (x.stride(0) | x.stride(1)) % 8 == 0 and x.data_ptr() % 16 == 0:
        return x
    return x.contiguous() if not x.is_contiguous() else x.clone()


def _rotate(q, k, rotary_cos, rotary_sin, positions, sections, interleaved, back):
    """Returns (q, k) rotated, dense; k may be None."""
    tokens, dev = q.shape[0], q.device
    cos, sin, positions, axis_stride, pair_axis, axes = _tables("rotary_axes", rotary_cos, rotary_sin, positions, sections, tokens, dev)
    q = _rows(q)
    q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    k_out = None
    k_args = (None, None, 0, 0, 0)
    if k is not None:
        k = _rows(k)
        k_out = torch.empty(k.shape, dtype=k.dtype, device=dev)
        k_args = (k.data_ptr(), k_out.data_ptr(), k.shape[1], k.stride(0), k.stride(1))
    with _on(dev):
        _lib.call("ifv2_rotary_axes", q.data_ptr(), k_args[0], q_out.data_ptr(), k_args[1], cos.data_ptr(), sin.data_ptr(),
                  positions.data_ptr(), axis_stride, pair_axis, axes, tokens, q.shape[1], k_args[2], HEAD_DIM, q.stride(0),
                  q.stride(1), k_args[3], k_args[4], 2 * cos.shape[1], cos.shape[0], int(bool(interleaved)), int(bool(back)),
                  _stream(dev))
    return q_out, k_out


@torch.library.custom_op("infllmv2_attn::_rotary_axes", mutates_args=(), device_types="cuda")
def _rotary_axes(q: torch.Tensor, k: Optional[torch.Tensor], rotary_cos: torch.Tensor, rotary_sin: torch.Tensor,
                 positions: torch.Tensor, sections: Optional[Sequence[int]], interleaved: bool,
                 back: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    """`_rotate` as a registered operator (an empty second result without k)."""
    q_out, k_out = _rotate(q, k, rotary_cos, rotary_sin, positions, sections, interleaved, back)
    return q_out, k_out if k_out is not None else q_out.new_empty(0)


@_rotary_axes.register_fake
def _(q, k, rotary_cos, rotary_sin, positions, sections, interleaved, back):
    return q.new_empty(q.shape), k.new_empty(k.shape) if k is not None else q.new_empty(0)


def _call(q, k, rotary_cos, rotary_sin, positions, sections, interleaved, back):
    """The body where nothing watches operators, the registered operator elsewhere."""
    if not torch.compiler.is_compiling() and not torch.autograd._profiler_enabled() and _plain_eager(q, k, rotary_cos, rotary_sin, positions):
        return _rotate(q, k, rotary_cos, rotary_sin, positions, sections, interleaved, back)
    q, k_out = _rotary_axes(q, k, rotary_cos, rotary_sin, positions, None if sections is None else list(sections), interleaved, back)
    return q, k_out if k is not None else None


class RotaryAxesFunc(torch.autograd.Function):
    """A rotation is linear: its gradient is the rotation by minus the angle, and so on to any order."""

    @staticmethod
    def forward(ctx, q, k, rotary_cos, rotary_sin, positions, sections, interleaved, back):
        ctx.save_for_backward(rotary_cos, rotary_sin, positions)
        ctx.sections, ctx.interleaved, ctx.back = sections, interleaved, back
        ctx.set_materialize_grads(False)
        return _call(q, k, rotary_cos, rotary_sin, positions, sections, interleaved, back)

    @staticmethod
    def backward(ctx, dq, dk):
        cos, sin, positions = ctx.saved_tensors
        args = (cos, sin, positions, ctx.sections, ctx.interleaved, not ctx.back)
        dq = dq if ctx.needs_input_grad[0] else None
        dk = dk if ctx.needs_input_grad[1] else None
        if dq is None:
            return (None, _rotary_maybe_grad(dk, None, *args)[0] if dk is not None else None) + (None,) * 6
        return _rotary_maybe_grad(dq, dk, *args) + (None,) * 6


def _rotary_maybe_grad(q, k, *args):
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return RotaryAxesFunc.apply(q, k, *args)
    return _call(q, k, *args)


def rotary_axes(q: torch.Tensor, k: Optional[torch.Tensor], rotary_cos: torch.Tensor, rotary_sin: torch.Tensor,
                positions: torch.Tensor, sections: Optional[Sequence[int]] = None, interleaved: bool = True):
    """Rotary positions of packed queries and keys, differentiable in q and k.

    q: (tokens, nheads, 128), k: (tokens, nheads_k, 128) or None, bf16; slices of one projection are taken as they
    are (rows on 16-byte boundaries).  rotary_cos / rotary_sin: (positions, rotary_dim / 2) fp32, rotary_dim a
    multiple of 16 up to 128.  positions: (tokens,) int32, or (axes, tokens) for up to four axes; sections: with
    several axes, how many of the rotary_dim / 2 pairs turn by the position on each (in order).  Pairs are features
    (2i, 2i+1) if interleaved, else (i, i + rotary_dim / 2); features from rotary_dim on pass through.  The
    arithmetic is fp32, the results are rounded once.  A position outside the tables takes their first or last row.
    Returns (q, k) rotated (k None without one), dense."""
    for name, t in (("q", q), ("k", k)):
        if t is None and name == "k":
            continue
        _require_cuda(t, name)
        if t.dtype != torch.bfloat16 or t.dim() != 3 or t.shape[-1] != HEAD_DIM:
            raise ValueError(f"rotary_axes: {name} must be (tokens, heads, {HEAD_DIM}) bf16")
    if k is not None and (k.shape[0] != q.shape[0] or k.device != q.device):
        raise ValueError("rotary_axes: q and k must have the same tokens, on one device")
    sections = None if sections is None else tuple(int(n) for n in sections)
    return _rotary_maybe_grad(q, k, rotary_cos, rotary_sin, positions, sections, bool(interleaved), False)

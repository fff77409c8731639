"""CPU: which tensors and strides `rotary_axes` and its derivatives launch with.  The launch itself is replaced by the
formula in tensor arithmetic, which reads its arguments by the strides that it is given, as the kernel does."""
import pytest
import torch

import infllm_v2
from infllmv2_cuda_impl_b200 import rotary

BF = torch.bfloat16


def _body(seen):
    def turn(q, k, tables, interleaved, back):
        cos, sin, positions, axis_stride, pair_axis, axes, rows, pairs = tables
        tokens = q.shape[0]
        at = [a * axis_stride + tokens for a in range(axes)]
        assert max(at) <= positions.untyped_storage().nbytes() // 4 - positions.storage_offset(), "positions are read out of range"
        assert cos.is_contiguous() and sin.is_contiguous()
        seen.append((positions.shape, axis_stride))
        pos = torch.as_strided(positions, (axes, tokens), (axis_stride, 1)).long()
        axis = torch.tensor(list(pair_axis) if pair_axis is not None else [0] * pairs)
        i = torch.arange(pairs)
        c, s = cos[pos[axis].t(), i][:, None], sin[pos[axis].t(), i][:, None] * (-1.0 if back else 1.0)
        f0 = 2 * i if interleaved else i
        f1 = f0 + 1 if interleaved else f0 + pairs

        def one(x):
            y = x.detach().float().clone()
            y[..., f0], y[..., f1] = x[..., f0].float() * c - x[..., f1].float() * s, x[..., f0].float() * s + x[..., f1].float() * c
            return y.to(BF)
        return one(q), one(k) if k is not None else None
    return turn


@pytest.fixture
def launches(monkeypatch):
    seen = []
    monkeypatch.setattr(rotary, "_require_cuda", lambda t, name: None)
    monkeypatch.setattr(rotary, "_turn", _body(seen))
    return seen


def _inputs(n=6, total=100, axes=3, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k = torch.randn(n, 16, 128, generator=g).to(BF), torch.randn(n, 2, 128, generator=g).to(BF)
    ang = 6.3 * torch.rand(40, 64, generator=g)
    pos = torch.randint(0, 40, (axes, total), generator=g, dtype=torch.int32)
    return q, k, ang.cos(), ang.sin(), pos


HOOKS = {
    "save_on_cpu": lambda: torch.autograd.graph.save_on_cpu(),
    "clone": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t),
    "transposed": lambda: torch.autograd.graph.saved_tensors_hooks(
        lambda t: t, lambda t: t.t().contiguous().t() if t.dim() == 2 else t),
    "spread": lambda: torch.autograd.graph.saved_tensors_hooks(
        lambda t: t, lambda t: torch.stack([t, torch.full_like(t, 39)], -1)[..., 0]),
}


@pytest.mark.parametrize("hook", sorted(HOOKS))
@pytest.mark.parametrize("axes", [1, 3])
def test_saved_tensors_may_come_back_with_other_strides(launches, hook, axes):
    q, k, cos, sin, wide = _inputs(axes=axes)
    pos = wide[:, 20:26]                                  # (axes, 6) in rows of 100
    sections = (20, 20, 24) if axes == 3 else None
    grads = []
    for context in (torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t), HOOKS[hook]()):
        x, y = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
        with context:
            out = infllm_v2.rotary_axes(x, y, cos, sin, pos, sections=sections)
        grads.append(torch.autograd.grad(out, (x, y), (q, k)))
    assert torch.equal(grads[0][0], grads[1][0]) and torch.equal(grads[0][1], grads[1][1])

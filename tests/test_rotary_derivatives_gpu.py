"""GPU: gradients of `rotary_axes` where autograd keeps its tensors elsewhere or runs the forward pass twice.  The
rotation is the same work in every form, so the bits are the same."""
import pytest
import torch

import infllm_v2
from helpers import det_tensor
from test_rotary_gpu import DEV, _positions, _tables

pytestmark = pytest.mark.gpu

CONTEXTS = {
    "save_on_cpu": lambda: torch.autograd.graph.save_on_cpu(),
    "pinned": lambda: torch.autograd.graph.save_on_cpu(pin_memory=True),
    "clone": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t),
    "transposed": lambda: torch.autograd.graph.saved_tensors_hooks(
        lambda t: t, lambda t: t.t().contiguous().t() if t.dim() == 2 else t),
}


def _inputs(n, axes, wide=1000, rows=300):
    cos, sin = (t.to(DEV) for t in _tables(rows, 128))
    q, k = det_tensor((n, 32, 128), 1).to(DEV), det_tensor((n, 2, 128), 2).to(DEV)
    pos = _positions(axes, wide, rows, 3).to(DEV)[:, 400:400 + n]         # a slice of wider rows
    sections = {1: None, 3: (20, 20, 24)}[axes]
    return q, k, cos, sin, pos, sections


@pytest.mark.parametrize("context", sorted(CONTEXTS))
@pytest.mark.parametrize("n,axes", [(1, 3), (77, 3), (301, 1)])
def test_saved_tensors_kept_elsewhere(context, n, axes):
    q, k, cos, sin, pos, sections = _inputs(n, axes)
    want = infllm_v2.rotary_axes(q, k, cos, sin, pos.contiguous(), sections=sections)
    grads = []
    for inside, at in ((False, pos.contiguous()), (True, pos)):
        x, y = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
        if inside:
            with CONTEXTS[context]():
                out = infllm_v2.rotary_axes(x, y, cos, sin, at, sections=sections)
        else:
            out = infllm_v2.rotary_axes(x, y, cos, sin, at, sections=sections)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        grads.append(torch.autograd.grad(out, (x, y), (q, k)))
    assert torch.equal(grads[0][0], grads[1][0]) and torch.equal(grads[0][1], grads[1][1])


@pytest.mark.parametrize("reentrant", [False, True])
def test_checkpointed_forward(reentrant):
    from torch.utils.checkpoint import checkpoint
    q, k, cos, sin, pos, sections = _inputs(77, 3)
    grads = []
    for again in (False, True):
        x, y = q.clone().requires_grad_(True), k.clone().requires_grad_(True)
        f = lambda a, b: infllm_v2.rotary_axes(a * 2, b * 3, cos, sin, pos, sections=sections)
        out = checkpoint(f, x, y, use_reentrant=reentrant) if again else f(x, y)
        torch.autograd.backward(out, (q, k))
        grads.append((x.grad, y.grad))
    assert torch.equal(grads[0][0], grads[1][0]) and torch.equal(grads[0][1], grads[1][1])


@pytest.mark.parametrize("grad", [False, True])
def test_forward_mode(grad):
    """A rotation is linear: the tangent of the result is the rotated tangent."""
    from torch.autograd import forward_ad
    q, k, cos, sin, pos, sections = _inputs(77, 3)
    tq, tk = det_tensor(q.shape, 7).to(DEV), det_tensor(k.shape, 8).to(DEV)
    want = infllm_v2.rotary_axes(tq, tk, cos, sin, pos, sections=sections)
    x, y = q.clone().requires_grad_(grad), k.clone().requires_grad_(grad)
    with forward_ad.dual_level():
        out = infllm_v2.rotary_axes(forward_ad.make_dual(x, tq), forward_ad.make_dual(y, tk), cos, sin, pos, sections=sections)
        out = [forward_ad.unpack_dual(t) for t in out]
        alone = infllm_v2.rotary_axes(forward_ad.make_dual(x, tq), y, cos, sin, pos, sections=sections)
        alone = [forward_ad.unpack_dual(t).tangent for t in alone]
    plain = infllm_v2.rotary_axes(q, k, cos, sin, pos, sections=sections)
    for i in range(2):
        assert torch.equal(out[i].primal, plain[i]) and torch.equal(out[i].tangent, want[i])
    assert torch.equal(alone[0], want[0]) and (alone[1] is None or not alone[1].any())

"""GPU: rotary positions over several axes against the 64-bit formula, forward and backward.

Tolerance: the result is an fp32 sum of two products, rounded once to bf16.  That is half a step of bf16, 2^-8 of
the value, and three fp32 roundings of terms no larger than the row's largest magnitude: 2 * 2^-24 each way, with
room 2^-21 of it."""
import pytest
import torch

import infllm_v2
from oracle.rotary import rotary_axes as exact
from helpers import det_tensor

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _tables(rows, dim):
    i = torch.arange(dim // 2, dtype=torch.float64)
    ang = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-2 * i / dim)
    return ang.cos().float(), ang.sin().float()


def _positions(axes, n, rows, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, rows, (axes, n), generator=g, dtype=torch.int32)


def _near(got, want, x):
    tol = 2.0 ** -8 * want.abs() + 2.0 ** -21 * x.double().abs().amax(-1, keepdim=True)
    assert got.shape == want.shape
    assert bool(((got.cpu().double() - want).abs() <= tol).all())


SECTIONS = {1: lambda p: (p,), 2: lambda p: (p // 2, p - p // 2), 3: lambda p: (p // 4, p // 4 + 1, p - 2 * (p // 4) - 1),
            4: lambda p: (1, 0, p - 3, 2)}


@pytest.mark.parametrize("tokens,hq,hk,dim,axes,interleaved", [
    (1, 16, 1, 128, 1, True), (1, 32, 2, 128, 3, False), (64, 32, 2, 128, 3, True), (77, 16, 1, 96, 2, False),
    (130, 128, 8, 64, 4, True), (513, 48, 3, 16, 3, False), (300, 5, 7, 112, 3, True), (9, 1, 1, 128, 4, False)])
def test_rotation_forward_and_backward(tokens, hq, hk, dim, axes, interleaved):
    rows = 700
    q, k = det_tensor((tokens, hq, 128), 1, 1.0), det_tensor((tokens, hk, 128), 2, 3.0)
    cos, sin = _tables(rows, dim)
    pos, sections = _positions(axes, tokens, rows, 3), SECTIONS[axes](dim // 2)
    qd, kd = q.to(DEV).requires_grad_(True), k.to(DEV).requires_grad_(True)
    args = (cos.to(DEV), sin.to(DEV), pos.to(DEV))
    qo, ko = infllm_v2.rotary_axes(qd, kd, *args, sections=sections, interleaved=interleaved)
    for got, x in ((qo.detach(), q), (ko.detach(), k)):
        _near(got, exact(x, cos, sin, pos, sections, interleaved), x)
    gq, gk = det_tensor(q.shape, 4, 1.0), det_tensor(k.shape, 5, 0.1)
    dq, dk = torch.autograd.grad((qo, ko), (qd, kd), (gq.to(DEV), gk.to(DEV)))
    for got, x in ((dq, gq), (dk, gk)):
        _near(got, exact(x, cos, sin, pos, sections, interleaved, back=True), x)
    # one of the two gradients alone
    qo, ko = infllm_v2.rotary_axes(qd, kd, *args, sections=sections, interleaved=interleaved)
    assert torch.equal(torch.autograd.grad(qo, qd, gq.to(DEV), retain_graph=True)[0], dq)
    assert torch.equal(torch.autograd.grad(ko, kd, gk.to(DEV))[0], dk)


def test_gradient_against_differences():
    """A rotation is linear in its input: f(x + d) - f(x) = f(d), whose product with the upstream gradient is the
    product of the gradient with d.  Each side carries half a bf16 step per element."""
    n, rows = 33, 50
    cos, sin = _tables(rows, 128)
    pos = _positions(3, n, rows, 1)
    sections = (16, 24, 24)
    x = det_tensor((n, 16, 128), 1, 1.0).to(DEV).requires_grad_(True)
    d, g = det_tensor((n, 16, 128), 2, 1.0), det_tensor((n, 16, 128), 3, 1.0)
    args = (cos.to(DEV), sin.to(DEV), pos.to(DEV))
    grad = torch.autograd.grad(infllm_v2.rotary_axes(x, None, *args, sections=sections)[0], x, g.to(DEV))[0].cpu().double()
    diff = infllm_v2.rotary_axes(d.to(DEV), None, *args, sections=sections)[0].cpu().double()
    a, b = (grad * d.double()).sum(), (g.double() * diff).sum()
    bound = 2.0 ** -8 * ((grad * d.double()).abs().sum() + (g.double() * diff).abs().sum()) * 1.01
    assert float((a - b).abs()) <= float(bound)


def test_second_derivative_is_the_rotation_again():
    cos, sin = _tables(40, 128)
    args = (cos.to(DEV), sin.to(DEV), _positions(1, 20, 40, 1)[0].to(DEV))
    x = det_tensor((20, 16, 128), 1).to(DEV).requires_grad_(True)
    g = det_tensor((20, 16, 128), 2).to(DEV).requires_grad_(True)
    y = infllm_v2.rotary_axes(x, None, *args)[0]
    dx, = torch.autograd.grad(y, x, g, create_graph=True)
    u = det_tensor((20, 16, 128), 3).to(DEV)
    dg, = torch.autograd.grad(dx, g, u)
    assert torch.equal(dg, infllm_v2.rotary_axes(u, None, *args)[0])


def test_slices_of_one_projection_and_other_strides():
    """Rows that are not dense, or not on 16-byte boundaries, give the bits of their dense copies."""
    n, hq, hk, rows = 65, 32, 2, 90
    cos, sin = (t.to(DEV) for t in _tables(rows, 128))
    pos = _positions(3, n, rows, 5).to(DEV)
    kw = dict(sections=(20, 20, 24), interleaved=False)
    qkv = det_tensor((n, (hq + 2 * hk), 128), 1).to(DEV)
    q, k = qkv[:, :hq], qkv[:, hq:hq + hk]
    ref = infllm_v2.rotary_axes(q.contiguous(), k.contiguous(), cos, sin, pos, **kw)
    for a, b in ((q, k), (q.transpose(0, 1).contiguous().transpose(0, 1), k)):
        got = infllm_v2.rotary_axes(a, b, cos, sin, pos, **kw)
        assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    odd = torch.empty(q.numel() + 3, dtype=q.dtype, device=DEV)[3:].view(q.shape).copy_(q)
    apart = torch.stack([k, k], -1)[..., 0]                          # features two elements apart
    got = infllm_v2.rotary_axes(odd, apart, cos, sin, pos.t().contiguous().t(), **kw)
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    one = k[:1].expand(n, hk, 128)                                   # a broadcast key
    got = infllm_v2.rotary_axes(q, one, cos, sin, pos, **kw)[1]
    assert torch.equal(got, infllm_v2.rotary_axes(q, one.contiguous(), cos, sin, pos, **kw)[1])


def test_positions_outside_the_tables_take_the_nearest_row():
    cos, sin = (t.to(DEV) for t in _tables(10, 128))
    x = det_tensor((3, 16, 128), 1).to(DEV)
    at = torch.tensor([-5, 10, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    near = torch.tensor([0, 9, 9], dtype=torch.int32, device=DEV)
    assert torch.equal(infllm_v2.rotary_axes(x, None, cos, sin, at)[0], infllm_v2.rotary_axes(x, None, cos, sin, near)[0])


def test_no_tokens_and_no_heads():
    cos, sin = (t.to(DEV) for t in _tables(10, 128))
    pos = torch.zeros(0, dtype=torch.int32, device=DEV)
    q, k = infllm_v2.rotary_axes(torch.empty(0, 16, 128, dtype=torch.bfloat16, device=DEV), None, cos, sin, pos)
    assert q.shape == (0, 16, 128) and k is None
    q = det_tensor((2, 16, 128), 1).to(DEV)
    q, k = infllm_v2.rotary_axes(q, q[:, :0], cos, sin, torch.zeros(2, dtype=torch.int32, device=DEV))
    assert k.shape == (2, 0, 128)


def test_same_bits_as_fp32_arithmetic():
    """Products and sums are rounded one by one, so fp32 tensor arithmetic gives the same bits."""
    n, rows = 257, 300
    cos, sin = (t.to(DEV) for t in _tables(rows, 128))
    pos = _positions(1, n, rows, 5)[0].to(DEV)
    x = det_tensor((n, 16, 128), 1, 5.0).to(DEV)
    c, s = cos[pos.long()][:, None], sin[pos.long()][:, None]
    x0, x1 = x[..., :64].float(), x[..., 64:].float()
    ref = torch.cat([x0 * c - x1 * s, x0 * s + x1 * c], -1).to(torch.bfloat16)
    assert torch.equal(infllm_v2.rotary_axes(x, None, cos, sin, pos, interleaved=False)[0], ref)


def test_registered_form_and_graph_capture():
    n, rows = 40, 60
    cos, sin = (t.to(DEV) for t in _tables(rows, 128))
    pos = _positions(2, n, rows, 5).to(DEV)
    q, k = det_tensor((n, 16, 128), 1).to(DEV), det_tensor((n, 1, 128), 2).to(DEV)
    ref = infllm_v2.rotary_axes(q, k, cos, sin, pos, sections=(30, 34))

    class Pass(torch.overrides.TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    with Pass():
        got = infllm_v2.rotary_axes(q, k, cos, sin, pos, sections=(30, 34))
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        infllm_v2.rotary_axes(q, k, cos, sin, pos, sections=(30, 34))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = infllm_v2.rotary_axes(q, k, cos, sin, pos, sections=(30, 34))
    q.mul_(0.5)
    pos.add_(1)
    graph.replay()
    ref = infllm_v2.rotary_axes(q, k, cos, sin, pos, sections=(30, 34))
    assert torch.equal(out[0], ref[0]) and torch.equal(out[1], ref[1])


def test_compiled_form():
    n, rows = 20, 60
    cos, sin = (t.to(DEV) for t in _tables(rows, 128))
    pos = _positions(1, n, rows, 5)[0].to(DEV)
    q = det_tensor((n, 16, 128), 1).to(DEV)
    f = torch.compile(lambda x: infllm_v2.rotary_axes(x, None, cos, sin, pos)[0], backend="eager", fullgraph=True)
    ref = infllm_v2.rotary_axes(q, None, cos, sin, pos)[0]
    assert torch.equal(f(q), ref)
    x = q.clone().requires_grad_(True)
    f = torch.compile(lambda x: infllm_v2.rotary_axes(x, None, cos, sin, pos)[0], backend="aot_eager", fullgraph=True)
    y = f(x)
    assert torch.equal(y.detach(), ref)
    eager = infllm_v2.rotary_axes(x, None, cos, sin, pos)[0]
    assert torch.equal(torch.autograd.grad(y, x, q)[0], torch.autograd.grad(eager, x, q)[0])

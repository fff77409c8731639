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


def _rotated(x, cos, sin, pos, sections):
    return infllm_v2.rotary_axes(x, None, cos, sin, pos, sections=sections)[0]


@pytest.mark.parametrize("with_k", [None, "plain", "dual"])
@pytest.mark.parametrize("q_dual", [True, False])
def test_forward_mode_turns_the_tangents(launches, with_k, q_dual):
    """A rotation is linear: the tangent of the result is the rotated tangent."""
    from torch.autograd import forward_ad
    if not q_dual and with_k != "dual":
        return
    q, k, cos, sin, wide = _inputs()
    pos, sections = wide[:, 20:26], (20, 20, 24)
    tq, tk = torch.randn(q.shape).to(BF), torch.randn(k.shape).to(BF)
    for grad in (None, False, True):                      # (None: without gradient mode, which forward mode does not ask)
        x, y = q.clone().requires_grad_(bool(grad)), k.clone().requires_grad_(bool(grad))
        with forward_ad.dual_level(), torch.set_grad_enabled(grad is not None):
            a = forward_ad.make_dual(x, tq) if q_dual else x
            b = None if with_k is None else forward_ad.make_dual(y, tk) if with_k == "dual" else y
            out = infllm_v2.rotary_axes(a, b, cos, sin, pos, sections=sections)
            (po, to), (pk, tk_out) = (forward_ad.unpack_dual(t) if t is not None else (None, None) for t in out)
            assert torch.equal(po.detach(), _rotated(q, cos, sin, pos, sections))
            for dual, got, tangent in ((q_dual, to, tq), (with_k == "dual", tk_out, tk)):
                if dual:
                    assert torch.equal(got.detach(), _rotated(tangent, cos, sin, pos, sections))
                else:
                    assert got is None or not got.any()


def test_forward_over_reverse_and_reverse_over_forward(launches):
    from torch.autograd import forward_ad
    q, _, cos, sin, wide = _inputs()
    pos, sections = wide[:, 20:26], (20, 20, 24)
    g, tg, t = (torch.randn(q.shape).to(BF) for _ in range(3))
    x = q.clone().requires_grad_(True)
    with forward_ad.dual_level():
        y = infllm_v2.rotary_axes(x, None, cos, sin, pos, sections=sections)[0]
        dx = torch.autograd.grad(y, x, forward_ad.make_dual(g, tg))[0]
        u = q.clone().requires_grad_(True)
        want = torch.autograd.grad(infllm_v2.rotary_axes(u, None, cos, sin, pos, sections=sections)[0], u, tg)[0]
        assert torch.equal(forward_ad.unpack_dual(dx).tangent, want)
    t.requires_grad_(True)
    with forward_ad.dual_level():
        y = infllm_v2.rotary_axes(forward_ad.make_dual(q, t), None, cos, sin, pos, sections=sections)[0]
        got = torch.autograd.grad(forward_ad.unpack_dual(y).tangent, t, tg)[0]
    assert torch.equal(got, want)


def test_tables_with_a_tangent_are_refused(launches):
    from torch.autograd import forward_ad
    q, _, cos, sin, wide = _inputs()
    pos, sections = wide[:, 20:26], (20, 20, 24)
    with forward_ad.dual_level():
        for c, s in ((forward_ad.make_dual(cos, sin), sin), (cos, forward_ad.make_dual(sin, cos))):
            with pytest.raises(NotImplementedError, match="tables"):
                infllm_v2.rotary_axes(q, None, c, s, pos, sections=sections)


def test_function_transforms_lose_no_derivative(launches):
    """torch.func.jvp and vjp want more of an autograd.Function than this one has, and say so."""
    q, _, cos, sin, wide = _inputs()
    f = lambda x: _rotated(x, cos, sin, wide[:, 20:26], (20, 20, 24))
    for call in (lambda: torch.func.jvp(f, (q,), (q,)), lambda: torch.func.vjp(f, q),
                 lambda: torch.func.grad(lambda x: f(x).float().sum())(q)):
        with pytest.raises(RuntimeError, match="setup_context"):
            call()


def test_compilation_traces_the_differentiable_form(launches):
    """In one piece (fullgraph); the compiled code itself, which would launch, is replaced."""
    q, k, cos, sin, wide = _inputs()
    pos, sections, graphs = wide[:, 20:26].contiguous(), (20, 20, 24), []

    def backend(graph, inputs):
        graphs.append(graph)
        return lambda *args: (q * 2, k * 3)

    f = torch.compile(lambda x, y: infllm_v2.rotary_axes(x, y, cos, sin, pos, sections=sections), backend=backend, fullgraph=True)
    for grad in (False, True):
        a, b = f(q.clone().requires_grad_(grad), k)
        assert torch.equal(a, q * 2) and torch.equal(b, k * 3)
    assert len(graphs) == 2 and not launches


@pytest.mark.parametrize("grad", [False, True])
def test_tables_that_require_a_gradient_are_refused_in_every_form(launches, grad):
    q, k, cos, sin, wide = _inputs()
    pos, sections = wide[:, 20:26].contiguous(), (20, 20, 24)
    q.requires_grad_(grad)

    class Pass(torch.overrides.TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    def call(c, s):
        return infllm_v2.rotary_axes(q, k, c, s, pos, sections=sections)

    def under_a_mode(c, s):
        with Pass():
            return call(c, s)

    compiled = torch.compile(call, backend=lambda graph, inputs: lambda *args: (q * 2, k * 3))
    for f in (call, under_a_mode, compiled):
        for c, s in ((cos.clone().requires_grad_(True), sin), (cos, sin.clone().requires_grad_(True))):
            with pytest.raises(NotImplementedError, match="tables"):
                f(c, s)
    assert not launches

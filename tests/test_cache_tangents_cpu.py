"""CPU: the calls over caches in 8 bits and over pages have no forward-mode derivative, and say so where a row has a tangent."""
import pytest
import torch
from torch.autograd import forward_ad

import infllm_v2
from infllmv2_cuda_impl_b200 import _lib, paged, quant_cache

BF, I32 = torch.bfloat16, torch.int32


@pytest.fixture
def launches(monkeypatch):
    seen = []
    for module in (quant_cache, paged):
        monkeypatch.setattr(module, "_require_cuda", lambda t, name: None)
        monkeypatch.setattr(module, "_stream", lambda dev: 0)
        monkeypatch.setattr(module, "_on", lambda dev: torch.no_grad())
    monkeypatch.setattr(paged, "_status_words", lambda dev: torch.zeros(4, dtype=I32))
    monkeypatch.setattr(_lib, "call", lambda name, *args: seen.append(name))
    return seen


def _calls(k, v, q):
    q8, b8 = infllm_v2.q8_cache(3, 64, 2, torch.int8, "cpu"), infllm_v2.b8_cache(3, 64, 2, torch.float8_e4m3fn, "cpu")
    rows, lens, slots = torch.zeros(3, 64, 2, 128, dtype=BF), torch.zeros(3, dtype=I32), torch.arange(3)
    cu = torch.arange(4, dtype=I32)
    return ((lambda: infllm_v2.cache_write(k, v, rows, rows.clone(), slots)), (lambda: infllm_v2.cache_write_b8(k, v, *b8, slots)),
            (lambda: infllm_v2.cache_fill_q8(k, v, *q8, cu)), (lambda: infllm_v2.decode_append_q8(k, v, *q8, lens)),
            (lambda: infllm_v2.infllmv2_attn_with_kvcache_q8(q[:, None], *q8, k=k[:, None], v=v[:, None], cache_seqlens=lens)),
            (lambda: infllm_v2.infllmv2_attn_paged_b8(q, *b8, cu, 1, lens)))


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("which", ["k", "v", "q"])
def test_rows_with_a_tangent(launches, which, grad_mode):
    t = dict(k=torch.zeros(3, 2, 128, dtype=BF), v=torch.zeros(3, 2, 128, dtype=BF), q=torch.zeros(3, 32, 128, dtype=BF))
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        for f in _calls(**t):                                      # (an open level alone does not matter)
            f()
        assert len(launches) == 6
        dual = dict(t, **{which: forward_ad.make_dual(t[which], torch.ones_like(t[which]))})
        calls = _calls(**dual)
        for f in calls[:5] if which != "q" else calls[4:]:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                f()
        assert len(launches) == 6
        for f in _calls(**{n: forward_ad.unpack_dual(x).primal for n, x in dual.items()}):
            f()
        assert len(launches) == 12


@pytest.mark.parametrize("which", ["k", "v", "q"])
def test_function_transforms(launches, which):
    t = dict(k=torch.zeros(3, 2, 128, dtype=BF), v=torch.zeros(3, 2, 128, dtype=BF), q=torch.zeros(3, 32, 128, dtype=BF))
    for i in range(5) if which != "q" else (4, 5):
        def f(x):
            _calls(**dict(t, **{which: x}))[i]()
            return x.sum()
        with pytest.raises((NotImplementedError, RuntimeError)):
            torch.func.jvp(f, (t[which],), (torch.ones_like(t[which]),))
        with pytest.raises((NotImplementedError, RuntimeError)):
            torch.func.grad(f)(t[which])
        with pytest.raises((NotImplementedError, RuntimeError, ValueError)):
            torch.func.vmap(f)(t[which].expand(2, *t[which].shape))
    assert not launches

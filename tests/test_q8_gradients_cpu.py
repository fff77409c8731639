"""CPU: the calls that write keys and values into an 8-bit cache refuse rows that require a gradient, all by one rule."""
import pytest
import torch

import infllm_v2
from infllmv2_cuda_impl_b200 import _lib, quant_cache

BF = torch.bfloat16


@pytest.fixture
def launches(monkeypatch):
    seen = []
    monkeypatch.setattr(quant_cache, "_require_cuda", lambda t, name: None)
    monkeypatch.setattr(quant_cache, "_stream", lambda dev: 0)
    monkeypatch.setattr(quant_cache, "_on", lambda dev: torch.no_grad())
    monkeypatch.setattr(_lib, "call", lambda name, *args: seen.append(name))
    return seen


def _calls(k, v, q):
    cache = infllm_v2.q8_cache(3, 32, 2, torch.int8, "cpu")
    lens = torch.zeros(3, dtype=torch.int32)
    return (lambda: infllm_v2.cache_fill_q8(k, v, *cache, torch.arange(4, dtype=torch.int32)),
            lambda: infllm_v2.decode_append_q8(k, v, *cache, lens),
            lambda: infllm_v2.infllmv2_attn_with_kvcache_q8(q, *cache, k=k[:, None], v=v[:, None], cache_seqlens=lens))


@pytest.mark.parametrize("which", ["k", "v", "q"])
def test_rows_that_require_a_gradient(launches, which):
    t = dict(k=torch.zeros(3, 2, 128, dtype=BF), v=torch.zeros(3, 2, 128, dtype=BF), q=torch.zeros(3, 1, 32, 128, dtype=BF))
    t[which] = t[which].requires_grad_(True)
    calls = _calls(**t)
    for f in calls if which != "q" else calls[2:]:
        with pytest.raises(NotImplementedError):
            f()
        assert not launches
    with torch.no_grad():
        for f in calls:
            f()
    for f in _calls(**{n: x.detach() for n, x in t.items()}):
        f()
    assert launches == 2 * ["ifv2_q8_fill", "ifv2_q8_append", "ifv2_q8_decode"]

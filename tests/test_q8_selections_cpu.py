"""CPU: block lists and masks of the 8-bit decode are taken in the order that is documented, batch before heads, and in no
other that has as many numbers."""
import pytest
import torch

import infllm_v2
from infllmv2_cuda_impl_b200 import _lib, quant_cache

Q = torch.zeros(3, 1, 32, 128, dtype=torch.bfloat16)


@pytest.fixture
def launches(monkeypatch):
    seen = []
    monkeypatch.setattr(quant_cache, "_require_cuda", lambda t, name: None)
    monkeypatch.setattr(quant_cache, "_stream", lambda dev: 0)
    monkeypatch.setattr(quant_cache, "_on", lambda dev: torch.no_grad())
    monkeypatch.setattr(_lib, "call", lambda name, *args: seen.append(name))
    return seen


def _attend(**kw):
    cache = infllm_v2.q8_cache(3, 8192, 2, torch.int8, "cpu")
    return infllm_v2.infllmv2_attn_with_kvcache_q8(Q, *cache, **kw)


@pytest.mark.parametrize("shape", [(2, 3, 1, 4), (2, 3, 4), (3, 1, 2, 4), (6, 1, 1, 4), (1, 3, 2, 4), (3, 2, 2, 2), (3, 2, 4, 1), (6, 4), (24,)])
def test_other_orders_are_refused(launches, shape):
    with pytest.raises(ValueError):
        _attend(topk_idx=torch.zeros(shape, dtype=torch.int32))
    words = tuple(n if n != 4 else 2 for n in shape)
    with pytest.raises(ValueError):
        _attend(block_mask=torch.zeros(words, dtype=torch.int64))
    assert not launches


@pytest.mark.parametrize("shape", [(3, 2, 1, 4), (3, 2, 4), (3, 2, 1, 0), (3, 2, 300)])
def test_lists(launches, shape):
    assert _attend(topk_idx=torch.zeros(shape, dtype=torch.int32)).shape == Q.shape
    assert launches == ["ifv2_q8_decode"]


@pytest.mark.parametrize("shape", [(3, 2, 1, 2), (3, 2, 2)])
def test_masks(launches, shape):
    assert _attend(block_mask=torch.zeros(shape, dtype=torch.int64)).shape == Q.shape
    assert launches == ["ifv2_q8_decode"]

"""CPU: what the operators of a paged cache refuse, in Python (the device check put aside) and in the C ABI, and what has nothing to
do.  Nothing is launched: a call that got as far as the library fails the test."""
import math

import pytest
import torch

import infllm_v2
from infllmv2_cuda_impl_b200 import _lib, paged

E4M3, E5M2, E8M0, BF = torch.float8_e4m3fn, torch.float8_e5m2, torch.float8_e8m0fnu, torch.bfloat16
I32, I64 = torch.int32, torch.int64


@pytest.fixture
def no_launch(monkeypatch):
    monkeypatch.setattr(paged, "_require_cuda", lambda t, name: None)

    def call(name, *args):
        raise AssertionError(f"{name} was called")

    monkeypatch.setattr(_lib, "call", call)


def _ints(*shape):
    return torch.zeros(*shape, dtype=I32)


def _b8(pages=3, page=128, hk=2, dtype=E4M3):
    return dict(zip(("k_cache", "v_cache", "k_scale", "v_scale"), infllm_v2.b8_cache(pages, page, hk, dtype, "cpu")))


def test_cpu_tensors_are_refused():
    ring, left = infllm_v2.page_pool(4, "cpu")
    assert ring.tolist() == [0, 1, 2, 3] and left.tolist() == [0, 4] and ring.dtype == left.dtype == I32
    k, cache = torch.zeros(4, 2, 128, dtype=BF), _b8()
    rows = torch.zeros(2, 64, 2, 128, dtype=BF)
    for f in (lambda: infllm_v2.pages_resize(_ints(2), _ints(2), _ints(2, 4), ring, left, 16, 0),
              lambda: infllm_v2.cache_write(k, k, rows, rows.clone(), torch.zeros(4, dtype=I64)),
              lambda: infllm_v2.cache_write_b8(k, k, *cache.values(), torch.zeros(4, dtype=I64)),
              lambda: infllm_v2.infllmv2_attn_paged_b8(torch.zeros(2, 32, 128, dtype=BF), *cache.values(), _ints(3), 1, _ints(2))):
        with pytest.raises(RuntimeError, match="CUDA"):
            f()


def test_empty_cache_is_zeros():
    for dtype in (E4M3, E5M2):
        k, v, ks, vs = infllm_v2.b8_cache(2, 192, 3, dtype, "cpu")
        assert k.shape == v.shape == (2, 3, 192, 128) and ks.shape == vs.shape == (2, 3, 3)
        assert k.dtype == v.dtype == dtype and ks.dtype == vs.dtype == E8M0
        assert not any(t.view(torch.uint8).any() for t in (k, v, ks, vs))
    for page, dtype in ((0, E4M3), (65, E4M3), (-64, E4M3), (64, BF), (64, torch.int8)):
        with pytest.raises(ValueError):
            infllm_v2.b8_cache(2, page, 3, dtype, "cpu")


RESIZE = dict(seqlens=_ints(2), targets=_ints(2), block_table=_ints(2, 4), free_pages=_ints(8), free_range=_ints(2), page_size=16, total=5)


@pytest.mark.parametrize("change", [
    dict(seqlens=_ints(0), targets=_ints(0), block_table=_ints(0, 4)), dict(seqlens=_ints(2, 1)), dict(seqlens=_ints(2).long()),
    dict(targets=_ints(3)), dict(targets=_ints(2).long()), dict(block_table=_ints(2, 4).long()), dict(block_table=_ints(3, 4)),
    dict(block_table=_ints(2, 0)), dict(block_table=_ints(8)), dict(block_table=_ints(2, 8)[:, ::2]), dict(block_table=_ints(1, 4).expand(2, 4)),
    dict(block_table=_ints(4, 2).t()), dict(free_pages=_ints(8).long()), dict(free_pages=_ints(0)), dict(free_pages=_ints(2, 4)),
    dict(free_pages=_ints(16)[::2]), dict(free_range=_ints(3)), dict(free_range=_ints(2).long()), dict(page_size=0), dict(total=-1),
    dict(page_size=2 ** 29), dict(total=2 ** 31),
    dict(seqlens=_ints(16385), targets=_ints(16385), block_table=_ints(16385, 1)),
], ids=lambda c: " ".join(c))
def test_resize(no_launch, change):
    with pytest.raises(ValueError):
        infllm_v2.pages_resize(**{**RESIZE, **change})


WRITE = dict(k=torch.zeros(4, 2, 128, dtype=BF), v=torch.zeros(4, 2, 128, dtype=BF), slots=torch.zeros(4, dtype=I64))
BAD_ROWS = [dict(k=torch.zeros(4, 2, 128)), dict(v=torch.zeros(4, 2, 128, dtype=torch.float16)), dict(k=torch.zeros(4, 3, 128, dtype=BF)),
            dict(v=torch.zeros(5, 2, 128, dtype=BF)), dict(k=torch.zeros(4, 2, 64, dtype=BF)), dict(k=torch.zeros(4, 256, dtype=BF)),
            dict(slots=torch.zeros(4, dtype=I32)), dict(slots=torch.zeros(5, dtype=I64)), dict(slots=torch.zeros(4, 1, dtype=I64))]


@pytest.mark.parametrize("change", BAD_ROWS + [
    dict(k_cache=torch.zeros(3, 128, 2, 128)), dict(v_cache=torch.zeros(3, 64, 2, 128, dtype=BF)), dict(k_cache=torch.zeros(3, 256, 128, dtype=BF)),
    dict(v_cache=torch.zeros(3, 2, 128, 128, dtype=BF).transpose(1, 2)), dict(k_cache=torch.zeros(3 * 256 * 128 + 1, dtype=BF)[1:].view(3, 128, 2, 128)),
    dict(k_cache=torch.zeros(3, 128, 2, 64, dtype=BF), v_cache=torch.zeros(3, 128, 2, 64, dtype=BF))], ids=lambda c: " ".join(c))
def test_write(no_launch, change):
    args = {**WRITE, "k_cache": torch.zeros(3, 128, 2, 128, dtype=BF), "v_cache": torch.zeros(3, 128, 2, 128, dtype=BF), **change}
    with pytest.raises(ValueError):
        infllm_v2.cache_write(**args)


BAD_B8 = [dict(k_cache=torch.zeros(3, 2, 128, 128, dtype=torch.uint8)), dict(v_cache=_b8(dtype=E5M2)["v_cache"]), dict(k_scale=torch.zeros(3, 2, 2)),
          dict(k_scale=_b8(page=64)["k_scale"]), dict(v_scale=_b8(pages=2)["v_scale"]), dict(v_cache=_b8(page=64)["v_cache"]),
          dict(k_cache=_b8(page=64)["k_cache"].view(torch.uint8)[:, :, :32].contiguous().view(E4M3)),
          dict(k_cache=_b8(3, 128, 128)["k_cache"].view(torch.uint8)[:, :2].view(E4M3)),
          dict(v_scale=torch.zeros(3, 4, 2, dtype=torch.uint8)[:, ::2].view(E8M0)),
          dict(k_cache=torch.zeros(3 * 2 * 128 * 128 + 8, dtype=torch.uint8)[8:].view(E4M3).view(3, 2, 128, 128))]


@pytest.mark.parametrize("change", BAD_ROWS + BAD_B8, ids=lambda c: " ".join(c))
def test_write_b8(no_launch, change):
    with pytest.raises(ValueError):
        infllm_v2.cache_write_b8(**{**_b8(), **WRITE, **change})


ATTEND = dict(q=torch.zeros(4, 32, 128, dtype=BF), cu_seqlens_q=_ints(3), max_seqlen_q=2, cache_seqlens=_ints(2), block_table=_ints(2, 3))


@pytest.mark.parametrize("change", BAD_B8 + [
    dict(q=torch.zeros(4, 32, 128)), dict(q=torch.zeros(4, 16, 128, dtype=BF)), dict(q=torch.zeros(4, 32, 64, dtype=BF)), dict(q=torch.zeros(32, 128, dtype=BF)),
    dict(cu_seqlens_q=_ints(1)), dict(cu_seqlens_q=_ints(3).long()), dict(cu_seqlens_q=_ints(4)), dict(cache_seqlens=_ints(3)),
    dict(cache_seqlens=_ints(2).long()), dict(max_seqlen_q=0), dict(max_seqlen_q=2 ** 31), dict(block_table=_ints(3, 3)), dict(block_table=_ints(2, 0)),
    dict(block_table=_ints(2, 3).long()), dict(block_table=_ints(6)), dict(cu_seqlens_q=_ints(5), cache_seqlens=_ints(4), block_table=None),
    dict(topk_idx=_ints(2, 4, 3).long()), dict(topk_idx=_ints(1, 4, 3)), dict(topk_idx=_ints(2, 3, 3)), dict(topk_idx=_ints(2, 4)),
    dict(block_mask=_ints(2, 4, 1)), dict(block_mask=torch.zeros(2, 4, 2, dtype=I64)), dict(block_mask=torch.zeros(4, 2, 1, dtype=I64)),
    dict(block_mask=torch.zeros(2, 4, 1, dtype=I64), topk_idx=_ints(2, 4, 3))], ids=lambda c: " ".join(c))
def test_attend(no_launch, change):
    with pytest.raises(ValueError):
        infllm_v2.infllmv2_attn_paged_b8(**{**_b8(), **ATTEND, **change})


def test_gradients_are_refused(no_launch):
    q = torch.zeros(4, 32, 128, dtype=BF, requires_grad=True)
    with pytest.raises(NotImplementedError):
        infllm_v2.infllmv2_attn_paged_b8(**{**_b8(), **ATTEND, "q": q})
    k = torch.zeros(4, 2, 128, dtype=BF, requires_grad=True)
    rows = torch.zeros(3, 128, 2, 128, dtype=BF)
    for change in (dict(k=k), dict(v=k)):
        with pytest.raises(NotImplementedError):
            infllm_v2.cache_write_b8(**{**_b8(), **WRITE, **change})
        with pytest.raises(NotImplementedError):
            infllm_v2.cache_write(**{**WRITE, "k_cache": rows, "v_cache": rows.clone(), **change})


def test_nothing_to_do(no_launch):
    none = torch.zeros(0, 2, 128, dtype=BF)
    infllm_v2.cache_write_b8(none, none, *_b8().values(), torch.zeros(0, dtype=I64))
    infllm_v2.cache_write(none, none, torch.zeros(3, 128, 2, 128, dtype=BF), torch.zeros(3, 128, 2, 128, dtype=BF), torch.zeros(0, dtype=I64))
    infllm_v2.cache_write_b8(WRITE["k"], WRITE["v"], *_b8(pages=0).values(), WRITE["slots"])
    out, lse = infllm_v2.infllmv2_attn_paged_b8(**{**_b8(), **ATTEND, "q": torch.zeros(0, 32, 128, dtype=BF)}, return_softmax_lse=True)
    assert out.shape == (0, 32, 128) and lse.shape == (0, 32)


# ---------------------------------------------------------------------------------- the C ABI --
P = 0x10000                                        # an address that nothing reads: every call here is refused


def _c(name, defaults, **change):
    args = {**defaults, **change}
    _lib.call(name, *args.values())


C_RESIZE = dict(seqlens=P, targets=P, table=P, stride=4, width=4, ring=P, pages=8, range=P, lens=P, left=P, cu=P, positions=P, slots=P,
                batch=2, page=16, total=5, stream=None)
C_WRITE = dict(k=P, v=P, kt=256, kh=128, vt=256, vh=128, kc=P, vc=P, slots=P, pages=3, page=64, total=4, heads=2, dim=128, stream=None)
C_B8 = dict(k=P, v=P, kt=256, kh=128, vt=256, vh=128, kc=P, vc=P, ks=P, vs=P, slots=P, pages=3, page=64, code=0, total=4, heads=2, dim=128,
            stream=None)
C_ATTN = dict(q=P, kc=P, vc=P, ks=P, vs=P, out=P, lse=None, cu=P, lens=P, table=P, width=3, lists=None, topk=0, mask=None, words=0, batch=2, total=4,
              most=2, pages=3, length=64, code=0, heads=32, hk=2, dim=128, scale=0.1, causal=1, ws=P, bytes=1 << 30, status=P, stream=None)


@pytest.mark.parametrize("change", [dict(batch=0), dict(width=0), dict(pages=0), dict(page=0), dict(total=-1), dict(batch=16385),
                                    dict(page=2 ** 30), dict(total=2 ** 31), dict(stride=3), dict(seqlens=None), dict(slots=None), dict(range=None)])
def test_c_resize(change):
    with pytest.raises((ValueError, RuntimeError)):
        _c("ifv2_pages_resize", C_RESIZE, **change)


@pytest.mark.parametrize("change", [dict(dim=64), dict(pages=-1), dict(page=0), dict(total=-1), dict(heads=0), dict(heads=4097), dict(k=None),
                                    dict(slots=None), dict(kt=4), dict(vh=1), dict(k=P + 8), dict(vc=P + 2), dict(total=2 ** 31)])
def test_c_write(change):
    with pytest.raises((ValueError, RuntimeError, NotImplementedError)):
        _c("ifv2_cache_write", C_WRITE, **change)
    _c("ifv2_cache_write", C_WRITE, total=0)
    _c("ifv2_cache_write", C_WRITE, pages=0)


@pytest.mark.parametrize("change", [dict(dim=64), dict(code=2), dict(code=-1), dict(page=96), dict(page=0), dict(pages=-1), dict(total=-1), dict(heads=0),
                                    dict(heads=32768), dict(total=2 ** 31), dict(v=None), dict(ks=None), dict(kh=4), dict(v=P + 4), dict(kc=P + 4)])
def test_c_b8_write(change):
    with pytest.raises((ValueError, RuntimeError, NotImplementedError)):
        _c("ifv2_b8_write", C_B8, **change)
    _c("ifv2_b8_write", C_B8, total=0)
    _c("ifv2_b8_write", C_B8, pages=0)


@pytest.mark.parametrize("change", [
    dict(dim=64), dict(heads=16), dict(hk=0, heads=0), dict(code=3), dict(batch=-1), dict(batch=0), dict(total=-1), dict(most=-1), dict(pages=-1),
    dict(pages=0), dict(length=0), dict(length=96), dict(width=0), dict(words=-1), dict(topk=-1), dict(lists=P, topk=2 ** 30), dict(lists=P, topk=3, mask=P, words=1),
    dict(q=None), dict(out=None), dict(cu=None), dict(lens=None), dict(ws=None), dict(status=None), dict(kc=None), dict(vs=None), dict(table=None, batch=4),
    dict(total=2 ** 31), dict(width=2 ** 25), dict(pages=2 ** 25), dict(mask=P, words=2), dict(lists=P, topk=3, width=8193), dict(mask=P, words=129, width=8193),
    dict(bytes=1000), dict(q=P + 8), dict(out=P + 2), dict(ws=P + 4), dict(kc=P + 8)])
def test_c_attend(change):
    with pytest.raises((ValueError, RuntimeError, NotImplementedError)):
        _c("ifv2_b8_attn", C_ATTN, **change)
    _c("ifv2_b8_attn", C_ATTN, total=0)


def test_workspace_sizes():
    """What a call needs grows with its tiles and does not depend on the lengths; nonsense needs nothing."""
    f = _lib.load().ifv2_b8_attn_workspace_bytes
    assert 0 < f(1, 1, 16, 128, 1, 4096) == f(64, 64, 128, 128, 1, 65536)
    assert f(64, 32, 32, 128, 2, 65536) > f(32, 32, 32, 128, 1, 65536)
    assert f(4096, 1, 32, 128, 4096, 32768) > f(8, 1, 32, 128, 8, 32768)
    assert f(4, 2, 32, 64, 2, 192) == f(-1, 2, 32, 128, 2, 192) == f(4, 2, 32, 128, 2, -64) == 0
    # a call whose costs pass 2^30 has its tiles listed, whatever the tokens
    assert f(64, 64, 32, 128, 1, 2 ** 30) > f(64, 64, 32, 128, 1, 2 ** 20)
    assert math.gcd(f(1, 1, 16, 128, 1, 4096), 256) == 256

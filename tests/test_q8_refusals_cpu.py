"""CPU: what the rotary and 8-bit cache operators refuse, in Python (the device check put aside) and in the C ABI.
Nothing is launched: a call that got as far as the library fails the test."""
import pytest
import torch

import infllm_v2
from infllmv2_cuda_impl_b200 import _lib, quant_cache, rotary

E4M3, INT8, E8M0 = torch.float8_e4m3fn, torch.int8, torch.float8_e8m0fnu
BF = torch.bfloat16


@pytest.fixture
def no_launch(monkeypatch):
    for m in (rotary, quant_cache):
        monkeypatch.setattr(m, "_require_cuda", lambda t, name: None)

    def call(name, *args):
        raise AssertionError(f"{name} was called")

    monkeypatch.setattr(_lib, "call", call)


def _ints(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def _cache(slots=3, length=32, hk=2, dtype=E4M3):
    return list(infllm_v2.q8_cache(slots, length, hk, dtype, "cpu"))


def test_cpu_tensors_are_refused():
    q = torch.zeros(2, 16, 128, dtype=BF)
    with pytest.raises(RuntimeError, match="CUDA"):
        infllm_v2.rotary_axes(q, None, torch.zeros(4, 64), torch.zeros(4, 64), _ints(2))
    cache = _cache()
    k = torch.zeros(4, 2, 128, dtype=BF)
    for f in (lambda: infllm_v2.cache_fill_q8(k, k, *cache, _ints(2)),
              lambda: infllm_v2.cache_read_q8(*cache, _ints(2), 4),
              lambda: infllm_v2.decode_append_q8(k[:3], k[:3], *cache, _ints(3)),
              lambda: infllm_v2.infllmv2_attn_with_kvcache_q8(torch.zeros(3, 1, 32, 128, dtype=BF), *cache)):
        with pytest.raises(RuntimeError, match="CUDA"):
            f()


def test_empty_cache_is_zeros():
    for dtype in (E4M3, INT8):
        k, v, ks, vs = _cache(2, 5, 3, dtype)
        assert k.shape == v.shape == (2, 3, 5, 128) and ks.shape == vs.shape == (2, 3, 5)
        assert k.dtype == dtype and ks.dtype == E8M0 and not k.view(torch.uint8).any() and not ks.view(torch.uint8).any()
    with pytest.raises(ValueError):
        infllm_v2.q8_cache(2, 5, 3, torch.float8_e5m2, "cpu")
    with pytest.raises(ValueError):
        infllm_v2.DecodeCache(2, 64, 2, infllm_v2.SparseConfig(), "cpu", kv_dtype=torch.float16)
    with pytest.raises(NotImplementedError):
        infllm_v2.DecodeCache(2, 64, 2, infllm_v2.SparseConfig(), "cpu").read(_ints(3), 0)


@pytest.mark.parametrize("change", [
    dict(q=torch.zeros(4, 16, 128)), dict(q=torch.zeros(4, 16, 64, dtype=BF)), dict(q=torch.zeros(64, 128, dtype=BF)),
    dict(k=torch.zeros(5, 2, 128, dtype=BF)), dict(cos=torch.zeros(9, 64, dtype=BF)), dict(cos=torch.zeros(8, 64)),
    dict(cos=torch.zeros(9, 60), sin=torch.zeros(9, 60)), dict(cos=torch.zeros(9, 72), sin=torch.zeros(9, 72)),
    dict(cos=torch.zeros(0, 64), sin=torch.zeros(0, 64)), dict(cos=torch.zeros(9, 0), sin=torch.zeros(9, 0)),
    dict(pos=torch.zeros(4, dtype=torch.int64)), dict(pos=_ints(5)), dict(pos=_ints(3, 5)), dict(pos=_ints(5, 4)),
    dict(pos=_ints(0, 4)), dict(pos=_ints(1, 2, 4)), dict(pos=_ints(3, 4)), dict(pos=_ints(3, 4), sections=(32, 32)),
    dict(pos=_ints(3, 4), sections=(32, 16, 15)), dict(pos=_ints(3, 4), sections=(65, -1, 0)), dict(sections=(32, 32))])
def test_rotary_refusals(no_launch, change):
    args = dict(q=torch.zeros(4, 16, 128, dtype=BF), k=torch.zeros(4, 2, 128, dtype=BF), cos=torch.zeros(9, 64),
                sin=torch.zeros(9, 64), pos=_ints(4), sections=None)
    args.update(change)
    with pytest.raises(ValueError):
        infllm_v2.rotary_axes(args["q"], args["k"], args["cos"], args["sin"], args["pos"], sections=args["sections"])


def test_tables_get_no_gradient(no_launch):
    with pytest.raises(NotImplementedError):
        infllm_v2.rotary_axes(torch.zeros(4, 16, 128, dtype=BF), None, torch.zeros(9, 64, requires_grad=True), torch.zeros(9, 64), _ints(4))


def _bad_caches():
    yield "types differ", lambda c: c.__setitem__(1, c[1].view(torch.uint8).view(INT8))
    yield "bf16", lambda c: c.__setitem__(0, torch.zeros(c[0].shape, dtype=BF))
    yield "scale type", lambda c: c.__setitem__(2, c[2].view(torch.uint8))
    yield "scale shape", lambda c: c.__setitem__(3, c[3][:, :, :-1].contiguous())
    yield "head dim", lambda c: c.__setitem__(0, c[0][..., :64].contiguous())
    yield "not contiguous", lambda c: c.__setitem__(0, c[0].transpose(1, 2).contiguous().transpose(1, 2))


@pytest.mark.parametrize("name,spoil", list(_bad_caches()))
def test_caches_that_do_not_fit(no_launch, name, spoil):
    cache = _cache()
    spoil(cache)
    k = torch.zeros(3, 2, 128, dtype=BF)
    for f in (lambda: infllm_v2.cache_fill_q8(k, k, *cache, _ints(4)), lambda: infllm_v2.cache_read_q8(*cache, _ints(4), 3),
              lambda: infllm_v2.decode_append_q8(k, k, *cache, _ints(3)),
              lambda: infllm_v2.infllmv2_attn_with_kvcache_q8(torch.zeros(3, 1, 32, 128, dtype=BF), *cache)):
        with pytest.raises(ValueError):
            f()


@pytest.mark.parametrize("change", [
    dict(k=torch.zeros(4, 2, 128)), dict(k=torch.zeros(4, 3, 128, dtype=BF)), dict(v=torch.zeros(5, 2, 128, dtype=BF)),
    dict(cu=torch.zeros(3, dtype=torch.int64)), dict(cu=_ints(1)), dict(cu=_ints(2, 2)), dict(cu=_ints(5)), dict(start=_ints(3)),
    dict(start=torch.zeros(2, dtype=torch.int64)), dict(table=_ints(3, 2)), dict(table=_ints(2)), dict(table=_ints(2, 0)),
    dict(out=_ints(3)), dict(out=_ints(2, 2)[:, 0])])
def test_fill_and_read_refusals(no_launch, change):
    args = dict(k=torch.zeros(4, 2, 128, dtype=BF), v=torch.zeros(4, 2, 128, dtype=BF), cu=_ints(3), start=None, table=None, out=None)
    args.update(change)
    with pytest.raises(ValueError):
        infllm_v2.cache_fill_q8(args["k"], args["v"], *_cache(), args["cu"], args["start"], args["table"], args["out"])
    if not {"k", "v", "out"} & set(change):
        with pytest.raises(ValueError):
            infllm_v2.cache_read_q8(*_cache(), args["cu"], 4, args["start"], args["table"])


def test_fill_refuses_gradients_and_shared_outputs(no_launch):
    k = torch.zeros(4, 2, 128, dtype=BF, requires_grad=True)
    with pytest.raises(NotImplementedError):
        infllm_v2.cache_fill_q8(k, k.detach(), *_cache(), _ints(3))
    start = _ints(2)
    with pytest.raises(ValueError):
        infllm_v2.cache_fill_q8(k.detach(), k.detach(), *_cache(), _ints(3), start=start, seqlens_out=start)
    with pytest.raises(ValueError):
        infllm_v2.cache_read_q8(*_cache(), _ints(3), -1)


@pytest.mark.parametrize("change", [
    dict(k=torch.zeros(3, 2, 128)), dict(k=torch.zeros(2, 2, 128, dtype=BF)), dict(lens=torch.zeros(3, dtype=torch.int64)), dict(lens=_ints(4)),
    dict(positions=_ints(2)), dict(kc=torch.zeros(3, 2, 2, 128)), dict(kc=torch.zeros(2, 2, 2, 128, dtype=BF)), dict(n_comp=_ints(1))])
def test_append_refusals(no_launch, change):
    args = dict(k=torch.zeros(3, 2, 128, dtype=BF), lens=_ints(3), positions=None, kc=torch.zeros(3, 2, 2, 128, dtype=BF), n_comp=None)
    args.update(change)
    with pytest.raises(ValueError):
        infllm_v2.decode_append_q8(args["k"], torch.zeros(3, 2, 128, dtype=BF), *_cache(), args["lens"], args["positions"],
                                   args["kc"], args["n_comp"])


Q = torch.zeros(3, 1, 32, 128, dtype=BF)
KV = torch.zeros(3, 1, 2, 128, dtype=BF)


@pytest.mark.parametrize("change,error", [
    (dict(q=Q.float()), ValueError), (dict(q=Q[:, 0]), ValueError), (dict(q=Q.expand(3, 2, 32, 128)), ValueError),
    (dict(q=torch.zeros(3, 1, 30, 128, dtype=BF)), ValueError), (dict(q=Q.clone().requires_grad_(True)), NotImplementedError),
    (dict(q=torch.zeros(4, 1, 32, 128, dtype=BF)), ValueError), (dict(k=KV), ValueError), (dict(k=KV, v=KV.float()), ValueError),
    (dict(k=KV[:, 0], v=KV[:, 0]), ValueError), (dict(cache_seqlens=torch.zeros(3, dtype=torch.int64)), ValueError),
    (dict(cache_seqlens=_ints(2)), ValueError), (dict(cache_batch_idx=_ints(2)), ValueError),
    (dict(cache_batch_idx=torch.zeros(3, dtype=torch.int64)), ValueError),
    (dict(block_table=_ints(3, 2), cache_batch_idx=_ints(3)), NotImplementedError), (dict(block_table=_ints(2, 2)), ValueError),
    (dict(topk_idx=torch.zeros(3, 2, 1, 4)), ValueError), (dict(topk_idx=_ints(3, 1, 1, 4)), ValueError),
    (dict(topk_idx=_ints(3, 2, 1, 1), block_mask=torch.zeros(3, 2, 1, 1, dtype=torch.int64)), ValueError),
    (dict(block_mask=_ints(3, 2, 1, 1)), ValueError), (dict(block_mask=torch.zeros(3, 2, 1, 2, dtype=torch.int64)), ValueError),
    (dict(rotary_cos=torch.zeros(4, 64)), ValueError), (dict(k=KV, v=KV, rotary_cos=torch.zeros(4, 64, dtype=BF), rotary_sin=torch.zeros(4, 64, dtype=BF)), ValueError),
    (dict(k=KV, v=KV, rotary_cos=torch.zeros(4, 64), rotary_sin=torch.zeros(4, 64), rotary_positions=_ints(3, 3)), ValueError),
    (dict(k=KV, v=KV, rotary_cos=torch.zeros(4, 64), rotary_sin=torch.zeros(4, 64), rotary_positions=_ints(2)), ValueError)])
def test_attention_refusals(no_launch, change, error):
    args = dict(q=Q)
    args.update(change)
    with pytest.raises(error):
        infllm_v2.infllmv2_attn_with_kvcache_q8(args.pop("q"), *_cache(), **args)


def test_page_size_refusal(no_launch):
    with pytest.raises(NotImplementedError):
        infllm_v2.infllmv2_attn_with_kvcache_q8(Q, *_cache(4, 24), block_table=_ints(3, 2))


P = 1 << 20                                                                       # an aligned address that nothing reads


def _rotary_args(**kw):
    a = dict(q=P, k=P, qo=P, ko=P, cos=P, sin=P, pos=P, ax=0, pair=None, axes=1, n=4, hq=16, hk=1, d=128, s0=2048, s1=128, s2=128, s3=128,
             dim=128, rows=9, il=1, back=0, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("change,code", [
    (dict(d=64), -2), (dict(n=-1), -1), (dict(dim=0), -1), (dict(dim=24), -1), (dict(dim=144), -1), (dict(axes=0), -1), (dict(axes=5), -1),
    (dict(rows=0), -1), (dict(cos=None), -1), (dict(pos=None), -1), (dict(q=None), -1), (dict(q=P + 8), -1), (dict(s0=4), -1),
    (dict(cos=P + 4), -1), (dict(axes=2, pair=b"\0" * 63 + b"\2"), -1)])
def test_c_rotary_refusals(lib, change, code):
    assert lib.ifv2_rotary_axes(*_rotary_args(**change)) == code and lib.ifv2_last_error()


def test_c_rotary_without_tokens(lib):
    assert lib.ifv2_rotary_axes(*_rotary_args(n=0)) == 0


def _fill_args(**kw):
    a = dict(k=P, v=P, s0=128, s1=128, s2=128, s3=128, kc=P, vc=P, ks=P, vs=P, cu=P, start=None, table=None, pages=0, out=None, slots=2,
             length=16, code=0, batch=2, total=4, hk=1, d=128, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("change,code", [
    (dict(d=64), -2), (dict(code=2), -1), (dict(batch=0), -1), (dict(total=-1), -1), (dict(length=0), -1), (dict(kc=None), -1),
    (dict(slots=1), -1), (dict(table=P, pages=0), -1), (dict(k=None), -1), (dict(kc=P + 8), -1), (dict(s2=12), -1), (dict(k=P + 2), -1),
    (dict(start=P, out=P), -1), (dict(total=1 << 31), -3), (dict(hk=70000), -3)])
def test_c_fill_refusals(lib, change, code):
    assert lib.ifv2_q8_fill(*_fill_args(**change)) == code and lib.ifv2_last_error()


def _append_args(**kw):
    a = dict(k=P, v=P, kc=P, vc=P, ks=P, vs=P, c1=P, c2=None, lens=P, pos=None, n1=None, n2=None, code=0, batch=2, slots=2, cap=16, cc=4,
             cc2=0, hk=1, d=128, k1=32, s1=16, k2=0, s2=0, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("change,code", [
    (dict(d=64), -2), (dict(code=-1), -1), (dict(slots=1), -1), (dict(k=None), -1), (dict(lens=P, pos=P), -1), (dict(k1=0), -1),
    (dict(c2=P), -1), (dict(n2=P), -1), (dict(v=P + 4), -1)])
def test_c_append_refusals(lib, change, code):
    assert lib.ifv2_q8_append(*_append_args(**change)) == code and lib.ifv2_last_error()


def _decode_args(**kw):
    a = dict(q=P, kc=P, vc=P, ks=P, vs=P, k=None, v=None, cos=None, sin=None, pos=None, ax=0, pair=None, axes=0, dim=0, rows=0, il=0,
             idx=None, topk=0, mask=None, words=0, out=P, lse=None, lens=P, bidx=None, table=None, pages=0, slots=2, length=64, code=0,
             batch=2, hq=16, hk=1, d=128, scale=0.1, ws=P, bytes=1 << 40, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("change,code", [
    (dict(d=64), -2), (dict(hq=32), -2), (dict(code=7), -1), (dict(length=0), -1), (dict(q=None), -1), (dict(k=P), -1), (dict(cos=P, sin=P), -1),
    (dict(k=P, v=P, cos=P), -1), (dict(k=P, v=P, cos=P, sin=P, dim=128, rows=4, axes=0), -1), (dict(idx=P, topk=257), -1), (dict(idx=P, topk=-1), -1), (dict(mask=P), -1),
    (dict(idx=P, topk=300, mask=P, words=5000), -3), (dict(table=P, pages=2, length=24), -1), (dict(table=P, pages=2, bidx=P), -2),
    (dict(slots=1), -1), (dict(slots=1 << 20, length=1 << 20), -3), (dict(table=P, pages=1 << 30), -3), (dict(bytes=16), -1),
    (dict(q=P + 8), -1), (dict(batch=70000, slots=70000), -3)])
def test_c_decode_refusals(lib, change, code):
    assert lib.ifv2_q8_decode(*_decode_args(**change)) == code and lib.ifv2_last_error()


def test_c_decode_without_sequences(lib):
    assert lib.ifv2_q8_decode(*_decode_args(batch=0)) == 0

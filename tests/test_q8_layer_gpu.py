"""GPU: DecodeCache and SparseAttention over an 8-bit cache, and a run of the operators together: rotate a prompt,
write it, attend its next token, read it back for the next chunk."""
import pytest
import torch

import infllm_v2
from oracle.q8 import attend, dequantise, quantise
from helpers import det_tensor, cu

pytestmark = pytest.mark.gpu
DEV = "cuda"
HQ, HK = 32, 2
E4M3, INT8 = torch.float8_e4m3fn, torch.int8


def _raw(t):
    return t.view(torch.uint8).cpu() if t.dtype != torch.uint8 else t.cpu()


def _prefill(lens, cap, dtype, cfg):
    layer = infllm_v2.SparseAttention(cfg)
    cache = infllm_v2.DecodeCache(len(lens), cap, HK, cfg, DEV, kv_dtype=dtype)
    q, k, v = det_tensor((sum(lens), HQ, 128), 1, 0.5), det_tensor((sum(lens), HK, 128), 2, 0.5), det_tensor((sum(lens), HK, 128), 3)
    out = layer.prefill(q.to(DEV), k.to(DEV), v.to(DEV), cu(lens, DEV), max(lens), lens, cache=cache)
    return layer, cache, out, k, v


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("coarse", [False, True])
def test_prefill_fills_and_decode_selects_over_the_cache(dtype, coarse):
    lens, cap = [700, 130, 1000], 1100
    cfg = infllm_v2.SparseConfig(topk=4, init_blocks=1, local_blocks=1, dense_len=0, coarse_lse=coarse)
    layer, cache, out, k, v = _prefill(lens, cap, dtype, cfg)
    plain = infllm_v2.DecodeCache(len(lens), cap, HK, cfg, DEV)
    q0 = det_tensor((sum(lens), HQ, 128), 1, 0.5)
    assert torch.equal(out, layer.prefill(q0.to(DEV), k.to(DEV), v.to(DEV), cu(lens, DEV), max(lens), lens, cache=plain))
    assert cache.seqlens.tolist() == lens and torch.equal(cache.kc, plain.kc) and torch.equal(cache.n_comp, plain.n_comp)
    kr, vr = cache.read(cu(lens, DEV), sum(lens))
    for x, got in ((k, kr), (v, vr)):
        assert torch.equal(got.cpu(), dequantise(*quantise(x, dtype)).to(torch.bfloat16))
    for step in range(40):
        q, kn, vn = (det_tensor((3, h, 128), 50 + 3 * step + i, 0.5).to(DEV) for i, h in enumerate((HQ, HK, HK)))
        got = layer.decode(q, kn, vn, cache)
        max_c = cfg.windows(cache.max_len)
        kc = cache.kc.view(-1, HK, 128)
        if coarse:
            score = infllm_v2.infllmv2_attn_stage1(q, kc, cache.kc2.view(-1, HK, 128), cache.cu_q, cache.cu_c, cache.cu_c2, 1,
                                                   max_c, causal=False, seqused_k=cache.n_comp, seqused_v=cache.n_comp2)
            mask, idx = infllm_v2.decode_select(score, cache.positions, 4, cap, 1, 1, seqused_c=cache.n_comp, return_topk=True)
        else:
            mask, idx = infllm_v2.infllmv2_stage1_decode_select(q, kc, cache.cu_c, cache.positions, max_c, cap, 4, 1, 1,
                                                                seqused_k=cache.n_comp, return_topk=True)
        again = infllm_v2.infllmv2_attn_with_kvcache_q8(q[:, None], cache.k, cache.v, cache.k_scale, cache.v_scale,
                                                        cache_seqlens=cache.seqlens, block_mask=mask)
        assert torch.equal(got, again)
    assert cache.seqlens.tolist() == [n + 40 for n in lens]
    # the last step against 64 bits: half a bf16 step and weights off by 2^-9 (see the tests of the operator)
    args = [t.cpu() for t in (cache.k, cache.v)] + [_raw(t) for t in (cache.k_scale, cache.v_scale)]
    want, _ = attend(q.cpu(), *args, [n + 40 for n in lens], topk_idx=idx.cpu())
    avg, _ = attend(q.cpu(), args[0], args[1].float().abs(), *args[2:], [n + 40 for n in lens], topk_idx=idx.cpu())
    assert bool(((got[:, 0].cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -9 * avg).all())


@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_captured_decode_equals_eager(dtype):
    lens, cap = [500, 64], 600
    cfg = infllm_v2.SparseConfig(topk=4, init_blocks=1, local_blocks=1, dense_len=200)
    layer, a, *_ = _prefill(lens, cap, dtype, cfg)
    _, b, *_ = _prefill(lens, cap, dtype, cfg)
    step = layer.capture_decode(a)
    for i in range(35):
        q, k, v = (det_tensor((2, h, 128), 900 + 3 * i + j, 0.5).to(DEV) for j, h in enumerate((HQ, HK, HK)))
        assert torch.equal(step(q, k, v), layer.decode(q, k, v, b, static_shapes=True))
    for name in ("k", "v", "k_scale", "v_scale", "kc", "seqlens", "n_comp"):
        assert torch.equal(_raw(getattr(a, name).contiguous().view(torch.uint8)), _raw(getattr(b, name).contiguous().view(torch.uint8)))


def test_a_full_cache_is_refused():
    cfg = infllm_v2.SparseConfig(dense_len=0)
    layer, cache, *_ = _prefill([64, 32], 64, E4M3, cfg)
    x = torch.zeros(2, HQ, 128, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="full"):
        layer.decode(x, x[:, :HK], x[:, :HK], cache)


@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_rotate_write_attend_and_read_for_the_next_chunk(dtype):
    lens, page, rows = [150, 33], 16, 400
    table = torch.randperm(30, generator=torch.Generator().manual_seed(1))[:28].view(2, 14).to(torch.int32)
    i = torch.arange(64, dtype=torch.float64)
    ang = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-i / 64)
    cos, sin = ang.cos().float().to(DEV), ang.sin().float().to(DEV)
    sections = (16, 24, 24)
    cache = infllm_v2.q8_cache(30, page, HK, dtype, DEV)
    q, k, v = (det_tensor((sum(lens), h, 128), s, 1.0).to(DEV) for s, h in ((1, HQ), (2, HK), (3, HK)))
    pos = torch.stack([torch.arange(sum(lens)) // d for d in (1, 3, 7)]).to(torch.int32).to(DEV)
    q_r, k_r = infllm_v2.rotary_axes(q, k, cos, sin, pos, sections=sections)
    length = torch.zeros(2, dtype=torch.int32, device=DEV)
    infllm_v2.cache_fill_q8(k_r, v, *cache, cu(lens, DEV), block_table=table.to(DEV), seqlens_out=length)
    assert length.tolist() == lens
    q1, k1, v1 = (det_tensor((2, 1, h, 128), s, 1.0).to(DEV) for s, h in ((4, HQ), (5, HK), (6, HK)))
    pos1 = torch.tensor([[150, 33], [60, 20], [30, 10]], dtype=torch.int32, device=DEV)
    out = infllm_v2.infllmv2_attn_with_kvcache_q8(
        q1, *cache, k=k1, v=v1, rotary_cos=cos, rotary_sin=sin, rotary_positions=pos1, rotary_sections=sections,
        cache_seqlens=length, block_table=table.to(DEV))
    grown = [n + 1 for n in lens]
    kr, vr = infllm_v2.cache_read_q8(*cache, cu(grown, DEV), sum(grown), block_table=table.to(DEV))
    # what was read back is what the token attended: the same token through the varlen attention over it.  Both round
    # their weights (2^-9 of bf16 weights there) and their results once; the varlen query is rounded to bf16 after its
    # rotation, which moves a score by at most 2^-8 sum |q k| / sqrt(128).
    q1_r = infllm_v2.rotary_axes(q1[:, 0], None, cos, sin, pos1, sections=sections)[0]
    ref = infllm_v2.infllmv2_attn_varlen_func(q1_r, kr, vr, cu([1, 1], DEV), cu(grown, DEV), 1, max(grown), causal=True)
    at = 0
    for b, n in enumerate(grown):
        kk, vv = kr[at:at + n].cpu().double(), vr[at:at + n].cpu().double()
        for h in range(HQ):
            qa = q1_r[b, h].cpu().double()
            ds = 2.0 ** -8 * float((kk[:, h // 16].abs() @ qa.abs()).max()) / 128 ** 0.5
            w = torch.softmax(kk[:, h // 16] @ qa / 128 ** 0.5, 0)
            avg = w @ vv[:, h // 16].abs()
            x, y = out[b, 0, h].cpu().double(), ref[b, h].cpu().double()
            assert bool(((x - y).abs() <= 2.0 ** -8 * (x.abs() + y.abs()) + avg * (2.0 ** -7 + 4 * ds)).all())
        at += n


def test_second_device_and_streams():
    """Tensors of another device than the current one, and calls on a stream of the caller's."""
    stream = torch.cuda.Stream()
    cache = infllm_v2.q8_cache(1, 64, 1, E4M3, DEV)
    k = det_tensor((64, 1, 128), 1).to(DEV)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        infllm_v2.cache_fill_q8(k, k, *cache, cu([64], DEV))
        out = infllm_v2.infllmv2_attn_with_kvcache_q8(k[:1].expand(16, 1, 128).reshape(1, 1, 16, 128), *cache)
    stream.synchronize()
    assert torch.equal(out, infllm_v2.infllmv2_attn_with_kvcache_q8(k[:1].expand(16, 1, 128).reshape(1, 1, 16, 128), *cache))
    if torch.cuda.device_count() > 1:
        other = [t.to("cuda:1") for t in cache]
        q = k[:1].expand(16, 1, 128).reshape(1, 1, 16, 128).to("cuda:1")
        assert torch.equal(infllm_v2.infllmv2_attn_with_kvcache_q8(q, *other).cpu(), out.cpu())

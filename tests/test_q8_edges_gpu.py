"""GPU: edges of the 8-bit cache and of the attention over it, next to the tests of each operator."""
import pytest
import torch

import infllm_v2
from oracle.q8 import attend, quantise
from helpers import det_tensor, cu
from test_q8_decode_gpu import DEV, E4M3, INT8, _cache, _check, _to_gpu

pytestmark = pytest.mark.gpu


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("page,topk", [(0, False), (16, False), (32, False), (64, False), (16, True), (64, True)])
def test_log_sum_exp_of_places_that_do_not_exist_is_nan(dtype, page, topk):
    """Scores against rows that the cache does not have are NaN, whatever the SM's memory held before."""
    q = det_tensor((3, 1, 32, 128), 7)
    if page:
        per = 192 // page
        cache = _cache(3 * per, page, 2, dtype, 3)
        table = torch.randperm(3 * per, generator=torch.Generator().manual_seed(1)).view(3, per).to(torch.int32)
        table[1, 1], table[2, per - 1] = 3 * per, -1
        lens, where = [192, 2 * page + 5, 192 - page], dict(block_table=table.to(DEV))       # the third does not reach its bad page
    else:
        cache = _cache(3, 190, 2, dtype, 3)
        table = torch.tensor([0, 3, 2], dtype=torch.int32)
        lens, where = [190, 77, 64], dict(cache_batch_idx=table.to(DEV))
    idx = torch.arange(3, dtype=torch.int32).expand(3, 2, 1, 3).contiguous() if topk else None
    junk = _to_gpu(_cache(64, 640, 2, dtype, 5))
    for _ in range(3):
        infllm_v2.infllmv2_attn_with_kvcache_q8(det_tensor((64, 1, 32, 128), 7).to(DEV), *junk)
        out, lse = infllm_v2.infllmv2_attn_with_kvcache_q8(
            q.to(DEV), *_to_gpu(cache), cache_seqlens=_ints(lens), topk_idx=None if idx is None else idx.to(DEV),
            return_softmax_lse=True, **where)
        assert bool(torch.isnan(out[1].float()).all()) and bool(torch.isnan(lse[1]).all())
        assert not torch.isnan(lse[::2]).any()
        _check(out[::2], lse[::2], q[::2], cache, lens[::2], table[::2] if page else None, None if page else table[::2])


@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_long_lists_that_change_from_call_to_call(dtype):
    """Lists of more than 256 entries are packed by a kernel beside which the attention starts: every call attends its own
    list, although the packed words lie where those of the call before lay."""
    n, k = 20000, 260
    cache = _cache(1, n, 1, dtype, 3)
    dev, q = _to_gpu(cache), det_tensor((1, 1, 16, 128), 7)
    lists = []
    for first in (0, 25, 50, 100, 0):
        idx = torch.full((1, 1, 1, k), -1, dtype=torch.int32)
        blocks = torch.arange(first, 313, 2 + first // 25)
        idx[0, 0, 0, :len(blocks)] = blocks
        lists.append(idx)
    outs = [infllm_v2.infllmv2_attn_with_kvcache_q8(q.to(DEV), *dev, topk_idx=idx.to(DEV), return_softmax_lse=True)
            for idx in lists]
    for (out, lse), idx in zip(outs, lists):
        _check(out, lse, q, cache, [n], topk_idx=idx)
    graph, idx = torch.cuda.CUDAGraph(), lists[0].to(DEV)
    qd = q.to(DEV)
    with torch.cuda.graph(graph):
        out, lse = infllm_v2.infllmv2_attn_with_kvcache_q8(qd, *dev, topk_idx=idx, return_softmax_lse=True)
    for (want, want_lse), other in zip(outs, lists):
        idx.copy_(other)
        for _ in range(3):
            graph.replay()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_two_tokens_of_one_row_touch_no_other_row(dtype):
    """Such a row is undefined; the rows around it, and what the other sequences attend, are not."""
    hk, page, lens = 2, 16, [20, 36, 9]
    table = torch.tensor([[0, 1, 2], [3, 1, 4], [5, 6, 7]], dtype=torch.int32)          # page 1 twice
    k, v = det_tensor((sum(lens), hk, 128), 1), det_tensor((sum(lens), hk, 128), 2)
    cache = infllm_v2.q8_cache(8, page, hk, dtype, DEV)
    for t in cache:
        t.view(torch.uint8).fill_(0xA5)
    infllm_v2.cache_fill_q8(k.to(DEV), v.to(DEV), *cache, cu(lens, DEV), block_table=table.to(DEV))
    new_k, new_v = det_tensor((3, 1, hk, 128), 3), det_tensor((3, 1, hk, 128), 4)
    # the appends of the first two sequences: position 20 is in page 1 as well, offset 4, and so is 16 + 4 of the second
    q = det_tensor((3, 1, 16 * hk, 128), 5)
    out, lse = infllm_v2.infllmv2_attn_with_kvcache_q8(
        q.to(DEV), *cache, k=new_k.to(DEV), v=new_v.to(DEV), cache_seqlens=_ints([20, 20, 9]), block_table=table.to(DEV),
        return_softmax_lse=True)
    want = [torch.full(t.shape, 0xA5, dtype=torch.uint8) for t in cache]
    both = torch.zeros(8, page, dtype=torch.bool)
    both[1, :5] = True
    at = 0
    for b, n in enumerate(lens):
        for i in range(n):
            p, o = int(table[b, i // page]), i % page
            for x, j in ((k, 0), (v, 1)):
                y, e = quantise(x[at + i], dtype)
                want[j][p, :, o], want[j + 2][p, :, o] = y.view(torch.uint8), e
        at += n
    for x, j in ((new_k, 0), (new_v, 1)):
        y, e = quantise(x[2, 0], dtype)
        want[j][5, :, 9], want[j + 2][5, :, 9] = y.view(torch.uint8), e
    for got, ref in zip(cache, want):
        got, ref = got.view(torch.uint8).cpu().movedim(1, 2), ref.movedim(1, 2)
        if got.dim() == 4 and dtype == E4M3:                                            # (a zero may have either sign)
            got, ref = got.view(E4M3).float().nan_to_num(1000.0), ref.view(E4M3).float().nan_to_num(1000.0)
        assert torch.equal(got[~both], ref[~both])
    kc, vc, kb, vb = (t.cpu() for t in cache)
    _check(out[2:], lse[2:], q[2:], (kc, vc, kb.view(torch.uint8), vb.view(torch.uint8)), [10], table[2:])


def test_lengths_next_to_the_border_of_32_bits():
    """start + rows is a number of more than 32 bits: the length is the capacity, as for any start past it."""
    cache = infllm_v2.q8_cache(3, 16, 1, INT8, DEV)
    k = det_tensor((6, 1, 128), 1).to(DEV)
    lens = torch.zeros(3, dtype=torch.int32, device=DEV)
    infllm_v2.cache_fill_q8(k, k, *cache, cu([2, 2, 2], DEV), start=_ints([2 ** 31 - 1, -2 ** 31, 15]), seqlens_out=lens)
    assert lens.tolist() == [16, 0, 16]
    seen = cache[0].view(torch.uint8).any(-1).any(1).nonzero().tolist()
    assert seen == [[2, 15]]


@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_first_keys_whose_scores_leave_the_range(dtype):
    """The first two blocks score -inf in 32 bits (-2^130), the others about -28: they alone have weight, and their weights
    are held against their own maximum.  One CTA attends all of a head, so that every warp begins in such a block."""
    batch, hk, n = 64, 8, 512
    k, v = det_tensor((batch, hk, n, 128), 3, 1.0), det_tensor((batch, hk, n, 128), 4, 1.0)
    q = (det_tensor((batch, 1, hk * 16, 128), 5, 1.0) * 8).round() / 8                   # (exact next to 2^10)
    q[..., :8], q[..., 8] = -2.0 ** 10, 16.0
    k[:, :, :128] = 0
    k[:, :, :128, :8] = 2.0 ** 120
    k[:, :, 128:, :8], k[:, :, 128:, 8] = 0, -20.0
    (kc, kb), (vc, vb) = quantise(k, dtype), quantise(v, dtype)
    idx = torch.arange(8, dtype=torch.int32, device=DEV).expand(batch, hk, 1, 8)
    out, lse = infllm_v2.infllmv2_attn_with_kvcache_q8(q.to(DEV), *_to_gpu((kc, vc, kb, vb)), topk_idx=idx, return_softmax_lse=True)
    rest = (kc[:, :, 128:], vc[:, :, 128:], kb[:, :, 128:], vb[:, :, 128:])
    _check(out, lse, q, rest, [n - 128] * batch)


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("vexp", [-120, -125, -128])
def test_results_among_the_subnormal_numbers(dtype, vexp):
    """A bf16 number below 2^-126 has steps of 2^-133, so a rounding is off by 2^-134; 2^-133 leaves as much for fp32 sums of
    subnormal numbers (2^-149 each).  Weights: 2^-11, and scores off by 130 * 2^-24 * sum |q k| / sqrt(128) < 2^-13."""
    k, v, q = det_tensor((1, 1, 100, 128), 3, 1.0), det_tensor((1, 1, 100, 128), 4, 1.0), det_tensor((1, 1, 16, 128), 5, 1.0)
    v = (v.double() * 2.0 ** vexp).to(torch.bfloat16)
    v[0, 0, 7] = 0
    (kc, kb), (vc, vb) = quantise(k, dtype), quantise(v, dtype)
    out = infllm_v2.infllmv2_attn_with_kvcache_q8(q.to(DEV), *_to_gpu((kc, vc, kb, vb)), cache_seqlens=100).cpu().double()[:, 0]
    want, _ = attend(q[:, 0], kc, vc, kb, vb, [100])
    avg, _ = attend(q[:, 0], kc, vc.float().abs(), kb, vb, [100])
    tol = 2.0 ** -8 * want.abs() + 2.0 ** -10 * avg + 2.0 ** -133
    assert bool(((out - want).abs() <= tol).all())
    assert float((out == 0).double().mean()) <= float((want.abs() <= 2.0 ** -134 + 2.0 ** -10 * avg).double().mean())

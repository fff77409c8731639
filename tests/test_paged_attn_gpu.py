"""GPU: attention of new tokens over a cache in 8 bits with block scales, against the formula in 64 bits on the same codes.

Tolerances (`_check`), from the kernel's own roundings: the result is rounded to bf16 (2^-8 of it).  A weight is three e5m2
terms of its fp16 rounding (2^-9 + 2^-11 of it, and 2^-24 of the largest one, an eighth more for the sums' fp32), so that
the result moves by that much of the attention over |v|.  A query is two e4m3 terms, off by at most 2^-18 of its largest
element, and scores are rounded to fp32 a few times, so that one moves by at most 2^-18 d max|q| max|k| scale, written as
`slack` below; a weight moves by that much of itself, the log-sum-exp by that much."""
import math

import pytest
import torch

import infllm_v2
from oracle import paged
from helpers import cu, det_tensor

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


def make(lens, hk, page, dtype, seed, k_size=1.0, v_size=1.0, extra=2):
    """A cache on the GPU that holds random rows of every sequence (sizes: a number, or one per token position), its
    table, and (k, v) in float64."""
    g = torch.Generator().manual_seed(seed)
    most = max(max(lens), 1)
    if page:
        per = (most + page - 1) // page
        pages, length = per * len(lens) + extra, page
        table = torch.randperm(pages, generator=g)[:per * len(lens)].view(len(lens), per).to(torch.int32)
    else:
        pages, length, table = len(lens) + extra, (most + 63) // 64 * 64, None
    cache = infllm_v2.b8_cache(pages, length, hk, dtype, "cpu")
    cache = [c.view(torch.uint8) for c in cache]
    cache[0].fill_(0x7F), cache[1].fill_(0x7F)                     # NaN codes wherever nothing is written
    cache[2].fill_(130), cache[3].fill_(130)
    cache = [c.view(t) for c, t in zip(cache, (dtype, dtype, torch.float8_e8m0fnu, torch.float8_e8m0fnu))]
    for b, n in enumerate(lens):
        if n == 0:
            continue
        pos = torch.arange(n)
        pg = torch.full_like(pos, b) if table is None else table[b].long()[pos // length]
        slots = pg * length + pos % length
        for i, size in ((0, k_size), (1, v_size)):
            x = torch.randn(n, hk, 128, generator=g, dtype=torch.float64)
            size = size(pos) if callable(size) else torch.full((n,), size, dtype=torch.float64)
            x = (x * size[:, None, None]).to(torch.bfloat16)
            y, e = paged.write(x, cache[i], cache[2 + i].view(torch.uint8), slots)
            keep = cache[i].double().isnan() & y.isnan()
            cache[i] = torch.where(keep, torch.full_like(y, float("nan")), y).float().to(dtype)
            cache[2 + i] = e.to(torch.uint8).view(torch.float8_e8m0fnu)
    k, v = (paged.numbers(cache[i], cache[2 + i].view(torch.uint8)) for i in (0, 1))
    return [c.to(DEV) for c in cache], table, k, v


def check(got, q, k, v, cu_q, lens, table, causal=True, lists=None, scale=None):
    out, lse = (x.cpu() for x in got)
    ref, ref_lse, size, reach = paged.attend(q, k, v, cu_q.tolist(), lens, table, causal, lists, scale)
    amax = q.double().abs().amax(-1)
    k_max = k[~k.isnan()].abs().max() if k.numel() else torch.zeros(())
    slack = amax * float(k_max) * 128 * (128 ** -0.5 if scale is None else abs(scale)) * 2.0 ** -18 + (reach + 1) * 2.0 ** -20
    nan = ref.isnan()
    assert torch.equal(nan, out.isnan()) and torch.equal(ref_lse.isnan(), lse.isnan())
    none = ref_lse == math.inf
    assert torch.equal(none, lse == math.inf) and bool((out[none] == 0).all())
    ok = ~ref_lse.isnan() & ~none
    err = (lse.double() - ref_lse).abs()
    assert bool((err <= slack + 2.0 ** -21 * ref_lse.abs())[ok].all()), float(err[ok].max())
    tol = 2.0 ** -8 * ref.abs() + size * (2.0 ** -9 + 2.0 ** -11) * 1.125 + size * (2 * slack)[..., None] + _floor(v, size) + 2.0 ** -133
    err = (out.double() - ref).abs()
    bad = (err > tol) & ~nan
    assert not bool(bad.any()), (float(err[bad].max()), float((err / tol)[~nan].max()), bad.nonzero()[:4].tolist())
    return err


def _floor(v, size):
    """What is lost of weights below the least e5m2 number: 2^-17 of 2^10 in units of the largest contribution of a code's
    top, for every key."""
    return size.amax(-1, keepdim=True) * 2.0 ** -12


def queries(lens_q, hk, seed, size=1.0):
    return det_tensor((max(sum(lens_q), 1), 16 * hk, 128), seed, size)[:sum(lens_q)]


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("lens,new,hk,page", [
    ([1], [1], 1, 64), ([64], [1], 2, 64), ([65], [1], 1, 128), ([128], [1], 1, 0), ([129, 1, 700], [1, 1, 1], 2, 64),
    ([300, 5], [2, 1], 2, 64), ([200, 130, 63], [4, 1, 3], 1, 192), ([90], [90], 2, 64), ([150, 40], [17, 33], 1, 0),
    ([1000, 0, 3, 513], [1, 1, 1, 1], 3, 256), ([257], [6], 1, 64), ([2, 3], [5, 3], 1, 64)])
def test_against_the_formula(dtype, lens, new, hk, page):
    cache, table, k, v = make(lens, hk, page, dtype, 3)
    q = queries(new, hk, 5)
    cu_q = cu(new)
    got = infllm_v2.infllmv2_attn_paged_b8(q.to(DEV), *cache, cu_q.to(DEV), max(new), torch.tensor(lens, dtype=torch.int32, device=DEV),
                                           block_table=None if table is None else table.to(DEV), return_softmax_lse=True)
    check(got, q, k, v, cu_q, lens, table)


@pytest.mark.parametrize("new", [[1, 1], [3, 2], [9, 40]])
def test_every_key_for_every_token(new):
    lens = [333, 70]
    cache, table, k, v = make(lens, 2, 64, E4M3, 7)
    q, cu_q = queries(new, 2, 8), cu(new)
    got = infllm_v2.infllmv2_attn_paged_b8(q.to(DEV), *cache, cu_q.to(DEV), max(new), torch.tensor(lens, dtype=torch.int32, device=DEV),
                                           block_table=table.to(DEV), causal=False, softmax_scale=0.2, return_softmax_lse=True)
    check(got, q, k, v, cu_q, lens, table, False, None, 0.2)


def _lists(lens, new, hk, n, seed):
    """Lists with duplicates left out, some empty, some naming blocks that the token does not reach."""
    g = torch.Generator().manual_seed(seed)
    rows = []
    for b, (m, t) in enumerate(zip(lens, new)):
        for i in range(t):
            blocks = (m + 63) // 64 + 1
            x = torch.stack([torch.cat([torch.randperm(blocks, generator=g)[:n].sort().values, torch.full((max(n - blocks, 0),), -1)])
                             for _ in range(hk)])
            if (b + i) % 5 == 3:
                x[:] = -1
            rows.append(x)
    return torch.stack(rows, 1).to(torch.int32)


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("lens,new,page", [([900, 700, 5, 2000], [1, 1, 1, 1], 64), ([900, 300], [2, 2], 128), ([700, 64, 65], [4, 3, 1], 64),
                                           ([800, 100], [20, 11], 0)])
def test_selected_blocks(dtype, lens, new, page):
    hk = 2
    cache, table, k, v = make(lens, hk, page, dtype, 11)
    q, cu_q, lists = queries(new, hk, 12), cu(new), _lists(lens, new, hk, 4, 13)
    more = dict(block_table=None if table is None else table.to(DEV), return_softmax_lse=True)
    args = (q.to(DEV), *cache, cu_q.to(DEV), max(new), torch.tensor(lens, dtype=torch.int32, device=DEV))
    got = infllm_v2.infllmv2_attn_paged_b8(*args, topk_idx=lists.to(DEV), **more)
    check(got, q, k, v, cu_q, lens, table, True, lists)
    cap = cache[0].shape[2] * (1 if table is None else table.shape[1])
    mask, _ = infllm_v2.topk_to_uint64(lists.to(DEV), cap, 64)
    # (not bit for bit the same: a mask row counts for another cost than a list, so that tiles are cut elsewhere)
    check(infllm_v2.infllmv2_attn_paged_b8(*args, block_mask=mask, **more), q, k, v, cu_q, lens, table, True, lists)


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("new", [[1], [3], [30]])
def test_blocks_of_very_different_sizes(dtype, new):
    """Values that grow, shrink, vanish and come back; keys whose blocks differ."""
    lens = [64 * 11 + 7]
    sizes = torch.tensor([1.0, 0.0, 2.0 ** -30, 2.0 ** 20, 2.0 ** -60, 3.0, 2.0 ** 50, 1.0, 0.0, 2.0 ** -20, 2.0 ** 49, 5.0], dtype=torch.float64)
    for order in (sizes, sizes.flip(0), torch.cat([torch.zeros(3, dtype=torch.float64), sizes[5:6].repeat(9)])):
        cache, table, k, v = make(lens, 1, 64, dtype, 17, lambda p: 1.0 + (p // 64 % 3).double(), lambda p: order[p // 64])
        q, cu_q = queries(new, 1, 18), cu(new)
        got = infllm_v2.infllmv2_attn_paged_b8(q.to(DEV), *cache, cu_q.to(DEV), max(new), torch.tensor(lens, dtype=torch.int32, device=DEV),
                                               block_table=table.to(DEV), return_softmax_lse=True)
        check(got, q, k, v, cu_q, lens, table)


@pytest.mark.parametrize("new", [[1], [4], [9]])
def test_scores_that_keep_growing(new):
    """Every block's scores are far above those before it (the reference moves with each of them), and the other way."""
    lens = [64 * 9 + 30]
    for up in (True, False):
        cache, table, k, v = make(lens, 1, 64, E4M3, 19, lambda p: 6.0 * (1.0 + (p if up else lens[0] - p) // 64).double())
        q, cu_q = queries(new, 1, 20, 2.0), cu(new)
        got = infllm_v2.infllmv2_attn_paged_b8(q.to(DEV), *cache, cu_q.to(DEV), max(new), torch.tensor(lens, dtype=torch.int32, device=DEV),
                                               block_table=table.to(DEV), return_softmax_lse=True)
        check(got, q, k, v, cu_q, lens, table)


def test_queries_of_any_size():
    lens, new = [200, 100, 70], [1, 1, 1]
    cache, table, k, v = make(lens, 1, 64, E4M3, 23)
    q = queries(new, 1, 24)
    q[0] *= 2.0 ** -100
    q[1] *= 2.0 ** 3
    q[2, 3] = 0
    cu_q = cu(new)
    got = infllm_v2.infllmv2_attn_paged_b8(q.to(DEV), *cache, cu_q.to(DEV), 1, torch.tensor(lens, dtype=torch.int32, device=DEV),
                                           block_table=table.to(DEV), return_softmax_lse=True)
    check(got, q, k, v, cu_q, lens, table)


@pytest.mark.parametrize("new", [[1, 1, 1, 1], [3, 2, 4, 1], [10, 20, 9, 11]])
def test_nan_blocks_and_missing_pages(new):
    """NaN reaches the tokens that see the block, and no others; so do pages that the cache does not have."""
    lens = [300, 200, 150, 130]
    cache, table, k, v = make(lens, 2, 64, E4M3, 29)
    bytes_k, bytes_v = cache[2].view(torch.uint8), cache[3].view(torch.uint8)
    bytes_k[table[0, 1].item(), 0] = 255
    bytes_v[table[1, 3].item(), 1] = 255                           # holds the last tokens: some of a chunk do not see it
    k[table[0, 1].item(), 0], v[table[1, 3].item(), 1] = math.nan, math.nan
    table = table.clone()
    table[2, 2] = -1
    table[3, 0] = 10 ** 6
    q, cu_q = queries(new, 2, 30), cu(new)
    got = infllm_v2.infllmv2_attn_paged_b8(q.to(DEV), *cache, cu_q.to(DEV), max(new), torch.tensor(lens, dtype=torch.int32, device=DEV),
                                           block_table=table.to(DEV), return_softmax_lse=True)
    out, lse = (x.cpu() for x in got)
    ref, ref_lse, *_ = paged.attend(q, k, v, cu_q.tolist(), lens, table)
    assert torch.equal(out.isnan(), ref.isnan()) and torch.equal(lse.isnan(), ref_lse.isnan())
    assert bool(ref.isnan().any()) and not bool(ref.isnan().all())


def test_rows_behind_the_last_sequence_are_zeros():
    lens, new = [100, 300], [2, 3]
    cache, table, k, v = make(lens, 1, 64, E5M2, 31)
    q, cu_q = queries([2, 3, 6], 1, 32), cu(new)
    out, lse = infllm_v2.infllmv2_attn_paged_b8(q.to(DEV), *cache, cu_q.to(DEV), 3, torch.tensor(lens, dtype=torch.int32, device=DEV),
                                                block_table=table.to(DEV), return_softmax_lse=True)
    assert bool((out[5:] == 0).all()) and bool((lse[5:] == math.inf).all())
    check((out[:5], lse[:5]), q[:5], k, v, cu_q, lens, table)


def test_long_walks_are_split_and_joined():
    """Thousands of keys in few tiles, so that every CTA has a piece; the answer is that of one piece per tile."""
    lens, new, hk = [5000, 3333], [1, 1], 1
    cache, table, k, v = make(lens, hk, 256, E4M3, 37)
    q, cu_q = queries(new, hk, 38), cu(new)
    args = (q.to(DEV), *cache, cu_q.to(DEV), 1, torch.tensor(lens, dtype=torch.int32, device=DEV))
    got = infllm_v2.infllmv2_attn_paged_b8(*args, block_table=table.to(DEV), return_softmax_lse=True)
    check(got, q, k, v, cu_q, lens, table)
    again = infllm_v2.infllmv2_attn_paged_b8(*args, block_table=table.to(DEV), return_softmax_lse=True)
    assert all(torch.equal(a, b) for a, b in zip(got, again))

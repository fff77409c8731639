"""GPU: rows written by slot into a cache in 8 bits with block scales.  Codes and scales are equal to the definition in 64 bits:
with a power of two the product is exact, so that only a value's place decides its code, also where codes are rounded
to a larger scale."""
import pytest
import torch

import infllm_v2
from oracle import paged
from helpers import det_tensor

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


def cache_of(pages, page, hk, dtype, mark=0x35):
    cache = infllm_v2.b8_cache(pages, page, hk, dtype, DEV)
    for t in cache:
        t.view(torch.uint8).fill_(mark)
    return list(cache)


def write_and_check(cache, k, v, slots):
    """Writes and compares all of the cache, what the call has no business with included.  (Codes as numbers: -0 is 0.)"""
    before = [t.cpu() for t in cache]
    infllm_v2.cache_write_b8(k.to(DEV), v.to(DEV), *cache, slots.to(DEV))
    for i, x in ((0, k), (1, v)):
        y, e = paged.write(x, before[i], before[2 + i].view(torch.uint8), slots)
        assert torch.equal(cache[2 + i].view(torch.uint8).cpu().long(), e)
        got = cache[i].cpu().double()
        assert torch.equal(got.nan_to_num(1e9), y.nan_to_num(1e9)), (got - y).abs().max()


def values(total, hk, seed):
    """Tokens of many sizes: ordinary, tiny, huge, subnormal, zero, one element alone."""
    x = det_tensor((total, hk, 128), seed).float()
    size = torch.tensor([1.0, 2.0 ** -20, 2.0 ** 60, 2.0 ** -128, 0.0, 2.0 ** -133, 3.0])
    x = x * size[(torch.arange(total) // 70) % 7][:, None, None]
    if total > 8:
        x[8, 0] = 0
        x[8, 0, 77] = -448.0
    return x.to(torch.bfloat16)


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("lens,start,hk,page", [
    ([1], [0], 1, 64), ([1], [63], 1, 64), ([64], [0], 2, 64), ([65, 3], [10, 130], 2, 128), ([500, 1, 17, 16], [0, 200, 5, 64], 2, 64),
    ([300, 15, 130], [63, 64, 1], 3, 192), ([1] * 40, list(range(40)), 8, 64), ([20, 2, 33], [40, 62, 31], 5, 256)])
def test_prompts_and_what_follows_them(dtype, lens, start, hk, page):
    """Rows at any place, first into marked pages, then the same length again right behind."""
    most = max(2 * n + s for n, s in zip(lens, start))
    per = (most + page - 1) // page
    g = torch.Generator().manual_seed(len(lens))
    table = torch.randperm(per * len(lens) + 2, generator=g)[:per * len(lens)].view(len(lens), per)
    cache = cache_of(per * len(lens) + 2, page, hk, dtype)
    total = sum(lens)
    for turn in range(2):
        slots = []
        for b, (n, s) in enumerate(zip(lens, start)):
            pos = torch.arange(n) + s + turn * n
            slots.append(table[b][pos // page] * page + pos % page)
        slots = torch.cat(slots)
        write_and_check(cache, values(total, hk, 1 + turn), values(total, hk, 7 + turn).flip(0), slots)


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
def test_token_by_token_with_scales_that_grow(dtype):
    """One token at a time through two blocks: each raises the scale of its block or fits it."""
    hk, page = 2, 128
    cache = cache_of(1, page, hk, dtype)
    g = torch.Generator().manual_seed(3)
    for pos in range(page):
        size = 2.0 ** (pos % 64 // 3 - 8) * (1.0 if pos % 5 else 0.01)
        k, v = ((torch.randn(1, hk, 128, generator=g) * size).to(torch.bfloat16) for _ in range(2))
        write_and_check(cache, k, v, torch.tensor([pos]))


@pytest.mark.parametrize("dtype,top", [(E4M3, 448.0), (E5M2, 57344.0)])
def test_borders_of_the_scale(dtype, top):
    """The largest code itself, the next bf16 number above it, the smallest scale, and every bf16 exponent as a block's largest."""
    for x in (top, top * (1 + 2.0 ** -7), 2.0 ** -133, 0.0, -top):
        k = torch.full((1, 1, 128), 0.25 * x, dtype=torch.bfloat16)
        k[0, 0, 5] = x
        write_and_check(cache_of(1, 64, 1, dtype), k, -k, torch.tensor([0]))
    n = 64 * 250
    k = torch.randn(n, 1, 128, generator=torch.Generator().manual_seed(1), dtype=torch.float64).clamp(-1.9, 1.9)
    k = (k * 2.0 ** (torch.arange(n) // 64 - 126).double()[:, None, None]).to(torch.bfloat16)
    write_and_check(cache_of(250, 64, 1, dtype), k, k.flip(0), torch.arange(n))


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
def test_every_code_rounds_to_a_larger_scale(dtype):
    """A block that holds all codes, then a token that needs the scale 1, 2, 5, 20 and 200 powers of two larger."""
    finite = torch.arange(256, dtype=torch.uint8).view(dtype).double()
    finite = torch.where(finite.isfinite(), finite, torch.zeros_like(finite))
    for up in (1, 2, 5, 20, 200):
        cache = cache_of(1, 64, 1, dtype)
        codes = finite.repeat(63 * 128 // 256 + 1)[:63 * 128].view(63, 128).float().to(dtype)
        for i in (0, 1):
            cache[i].view(torch.uint8)[0, 0, :63] = codes.view(torch.uint8).to(DEV)
            cache[2 + i].view(torch.uint8)[0, 0, 0] = 20
        x = torch.full((1, 1, 128), paged.TOP[dtype] * 2.0 ** (20 - 127 + up), dtype=torch.float64).to(torch.bfloat16)
        write_and_check(cache, x, x, torch.tensor([63]))


def test_infinities_and_nans_make_the_block_nan_until_it_begins_anew():
    hk, page = 2, 64
    cache = cache_of(2, page, hk, E4M3)
    k, v = det_tensor((30, hk, 128), 1), det_tensor((30, hk, 128), 2)
    k[4, 0, 3], v[7, 1, 0] = float("inf"), float("nan")
    write_and_check(cache, k, v, torch.arange(30))
    write_and_check(cache, det_tensor((10, hk, 128), 3), det_tensor((10, hk, 128), 4), torch.arange(30, 40))      # stays NaN
    write_and_check(cache, det_tensor((70, hk, 128), 5), det_tensor((70, hk, 128), 6), torch.arange(70))


def test_slots_that_the_cache_does_not_have():
    cache = cache_of(2, 64, 1, E5M2)
    slots = torch.tensor([-1, 128, 5, 6, 7, -1, 2 ** 40, 64, 65])
    write_and_check(cache, det_tensor((9, 1, 128), 1), det_tensor((9, 1, 128), 2), slots)


def test_runs_end_where_slots_jump_and_at_segments():
    """Long and short runs in one call, most of them across the borders of 64 tokens, more than the CTAs of a small call."""
    hk, page = 2, 256
    g = torch.Generator().manual_seed(4)
    slots, at = [], 0
    while at < 40 * page - 300:
        n = int(torch.randint(1, 150, (1,), generator=g))
        slots.append(torch.arange(at, at + n))
        at += n + int(torch.randint(1, 4, (1,), generator=g)) * 64
    slots = torch.cat(slots)
    write_and_check(cache_of(40, page, hk, E4M3), det_tensor((len(slots), hk, 128), 1), det_tensor((len(slots), hk, 128), 2), slots)


def test_fused_rows_other_stream_and_graph():
    hk, total = 4, 100
    x = det_tensor((total, 16 + 2 * hk, 128), 9).to(DEV)
    k, v = x[:, 16:16 + hk], x[:, 16 + hk:]
    slots = torch.arange(20, 20 + total)
    want = cache_of(3, 64, hk, E4M3)
    infllm_v2.cache_write_b8(k, v, *want, slots.to(DEV))
    side = torch.cuda.Stream()
    cache = cache_of(3, 64, hk, E4M3)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        infllm_v2.cache_write_b8(k, v, *cache, slots.to(DEV))
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, want))
    cache, slots_d = cache_of(3, 64, hk, E4M3), slots.to(DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        infllm_v2.cache_write_b8(k, v, *cache, slots_d)
    for _ in range(2):
        graph.replay()
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, want))
    odd = torch.zeros(total * hk * 128 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(total, hk, 128).copy_(k)      # off a 16-byte boundary
    cache = cache_of(3, 64, hk, E4M3)
    infllm_v2.cache_write_b8(odd, v, *cache, slots_d)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, want))

"""GPU: writing an 8-bit cache and reading it back.  Codes and scales are equal to the definition in 64 bits, value
by value: with a power-of-two scale every product is exact and only the place of a value decides its code."""
import pytest
import torch

import infllm_v2
from oracle.q8 import quantise, dequantise, rows_of
from helpers import det_tensor, cu

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3, INT8 = torch.float8_e4m3fn, torch.int8


def _bytes(x):
    return x.view(torch.uint8).cpu()


def _cache(slots, length, hk, dtype, fill=0xA5):
    """A cache whose bytes are all `fill`, so that a row that is touched without need shows."""
    cache = infllm_v2.q8_cache(slots, length, hk, dtype, DEV)
    for t in cache:
        t.view(torch.uint8).fill_(fill)
    return cache


def _values(total, hk, seed):
    """Rows of many sizes: ordinary, tiny, huge, subnormal, zero, one element alone."""
    x = det_tensor((total, hk, 128), seed, 1.0)
    scale = torch.tensor([1.0, 2.0 ** -20, 2.0 ** 60, 2.0 ** -128, 0.0, 2.0 ** -133, 3.0], dtype=torch.float32)
    x = (x.float() * scale[torch.arange(total) % 7][:, None, None]).to(torch.bfloat16)
    if total > 8:
        x[8, 0] = 0
        x[8, 0, 77] = -448.0                     # the largest code itself
    if total > 9:
        x[9, 0, :] = 1.0
        x[9, 0, 5] = 1.984375 * 64               # 127, the largest int8 code
    if total > 10:
        x[10, 0, 0] = 450.0                      # just above: the next exponent
    return x


def _check(cache, k, v, lens, start, table, length, untouched=0xA5):
    kc, vc, ks, vs = (t.cpu() for t in cache)
    seen = torch.zeros(ks.shape, dtype=torch.bool)
    at = 0
    for b, n in enumerate(lens):
        slot, off = rows_of(table, None, length, b, start[b] + n)
        slot, off = slot[start[b]:], off[start[b]:]
        for x, codes, scale in ((k, kc, ks), (v, vc, vs)):
            y, e = quantise(x[at:at + n], codes.dtype)
            assert torch.equal(scale.view(torch.uint8)[slot, :, off], e)
            assert torch.equal(codes[slot, :, off].float(), y.float())
        seen[slot, :, off] = True
        at += n
    for t in (kc, vc):
        assert bool((t.view(torch.uint8)[~seen] == untouched).all())
    for t in (ks, vs):
        assert bool((t.view(torch.uint8)[~seen] == untouched).all())


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("lens,hk,page,start", [
    ([1], 1, 0, [0]), ([37, 1, 0, 64], 2, 0, [0, 5, 3, 1]), ([37, 1, 0, 64], 2, 16, [0, 5, 3, 1]),
    ([300, 129], 8, 64, [0, 63]), ([11, 300], 3, 5, [2, 0]), ([1, 1, 1], 4, 256, [255, 256, 0])])
def test_write_and_read_back(dtype, lens, hk, page, start):
    total = sum(lens)
    k, v = _values(total, hk, 1), _values(total, hk, 2).flip(0)
    most = max(s + n for s, n in zip(start, lens))
    table = None
    if page:
        per = (most + page - 1) // page
        table = torch.randperm(len(lens) * per + 2, generator=torch.Generator().manual_seed(1))[:len(lens) * per]
        table = table.view(len(lens), per).to(torch.int32)
        cache = _cache(len(lens) * per + 2, page, hk, dtype)
    else:
        cache = _cache(len(lens) + 1, most, hk, dtype)
    cu_d, start_d = cu(lens, DEV), torch.tensor(start, dtype=torch.int32, device=DEV)
    table_d = None if table is None else table.to(DEV)
    seqlens = torch.zeros(len(lens), dtype=torch.int32, device=DEV)
    infllm_v2.cache_fill_q8(k.to(DEV), v.to(DEV), *cache, cu_d, start=start_d, block_table=table_d, seqlens_out=seqlens)
    assert seqlens.tolist() == [s + n for s, n in zip(start, lens)]
    _check(cache, k, v, lens, start, table, page or most)
    kr, vr = infllm_v2.cache_read_q8(*cache, cu_d, total + 3, start=start_d, block_table=table_d)
    assert not kr[total:].any() and not vr[total:].any()           # rows behind the last sequence
    for x, got in ((k, kr), (v, vr)):
        want = dequantise(*quantise(x, dtype)).to(torch.bfloat16)   # exact but for values below 2^-133
        assert torch.equal(got[:total].cpu(), want)


@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_every_bf16_number_as_the_largest_of_a_row(dtype):
    """65536 rows, one for each bit pattern, with random smaller numbers beside it: codes and scales are the oracle's."""
    g = torch.Generator().manual_seed(1)
    top = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = torch.randint(0, 65536, (65536, 1, 128), generator=g, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = torch.where(x.abs().float() <= top.abs().float()[:, None, None], x, torch.zeros_like(x))   # (not below a NaN)
    x[torch.arange(65536), 0, torch.randint(0, 128, (65536,), generator=g)] = top
    kc, vc, ks, vs = infllm_v2.q8_cache(1, 65536, 1, dtype)
    infllm_v2.cache_fill_q8(x.to(DEV), x.to(DEV), kc, vc, ks, vs, cu([65536], DEV))
    codes, scales = quantise(x[:, 0], dtype)
    assert torch.equal(ks.view(torch.uint8).cpu().flatten(), scales.view(torch.uint8).flatten())
    assert torch.equal(kc.float().cpu().flatten(), codes.float().flatten())              # (a zero may have either sign)
    assert torch.equal(kc.view(torch.uint8), vc.view(torch.uint8)) and torch.equal(ks.view(torch.uint8), vs.view(torch.uint8))


@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_infinities_and_nan_make_the_row_nan(dtype):
    k = det_tensor((4, 2, 128), 1)
    v = k.clone()
    k[1, 0, 3], k[2, 1, 127], v[3, 1, 0] = float("inf"), float("nan"), float("-inf")
    cache = _cache(1, 4, 2, dtype)
    infllm_v2.cache_fill_q8(k.to(DEV), v.to(DEV), *cache, cu([4], DEV))
    kr, vr = (t.cpu().float() for t in infllm_v2.cache_read_q8(*cache, cu([4], DEV), 4))
    bad = torch.zeros(4, 2, dtype=torch.bool)
    bad[1, 0] = bad[2, 1] = True
    assert torch.equal(torch.isnan(kr).all(-1), bad) and torch.equal(torch.isnan(kr).any(-1), bad)
    assert torch.isnan(vr[3, 1]).all() and not torch.isnan(vr[:3]).any()
    assert _bytes(cache[2])[0, 0, 1] == 255


def test_largest_and_smallest_numbers():
    big = torch.finfo(torch.bfloat16).max
    k = torch.zeros(3, 1, 128, dtype=torch.bfloat16)
    k[0, 0, 0], k[0, 0, 1], k[1, 0, 9], k[2, 0, 2] = big, 1.5 * 2.0 ** 127, 2.0 ** -133, -(2.0 ** -118)
    for dtype in (E4M3, INT8):
        cache = _cache(1, 3, 1, dtype)
        infllm_v2.cache_fill_q8(k.to(DEV), k.to(DEV), *cache, cu([3], DEV))
        y, e = quantise(k, dtype)
        assert torch.equal(_bytes(cache[2])[0, 0], e[:, 0]) and torch.equal(cache[0][0, 0].cpu().float(), y[:, 0].float())


def test_rows_without_a_place_are_dropped_and_read_as_nan():
    """Pages that the cache does not have, positions past the table and below 0, and an unused tail."""
    page, hk = 16, 2
    table = torch.tensor([[1, -1], [3, 7], [0, 4]], dtype=torch.int32)    # pages 0 .. 4
    lens, start = [20, 40, 5], [0, 0, -3]
    k = _values(sum(lens), hk, 1)
    for dtype in (E4M3, INT8):
        cache = _cache(5, page, hk, dtype)
        args = dict(start=torch.tensor(start, dtype=torch.int32, device=DEV), block_table=table.to(DEV))
        seqlens = torch.zeros(3, dtype=torch.int32, device=DEV)
        infllm_v2.cache_fill_q8(k.to(DEV), k.to(DEV), *cache, cu(lens, DEV), seqlens_out=seqlens, **args)
        assert seqlens.tolist() == [20, 32, 2]
        got = infllm_v2.cache_read_q8(*cache, cu(lens, DEV), sum(lens), **args)[0].cpu()
        there = torch.tensor([True] * 16 + [False] * 4 + [True] * 16 + [False] * 24 + [False] * 3 + [True] * 2)
        want = dequantise(*quantise(k, dtype)).to(torch.bfloat16)
        assert torch.equal(got[there], want[there]) and torch.isnan(got[~there].float()).all()
        used = torch.zeros(5, page, dtype=torch.bool)
        used[1], used[3], used[0, :2] = True, True, True
        assert bool((_bytes(cache[0]).movedim(1, 2)[~used] == 0xA5).all())


def test_slices_of_one_projection():
    hk, lens = 2, [33, 20]
    qkv = det_tensor((53, 36, 128), 1).to(DEV)
    k, v = qkv[:, 32:34], qkv[:, 34:36]
    a, b = _cache(2, 40, hk, E4M3), _cache(2, 40, hk, E4M3)
    infllm_v2.cache_fill_q8(k, v, *a, cu(lens, DEV))
    infllm_v2.cache_fill_q8(k.contiguous(), v.contiguous(), *b, cu(lens, DEV))
    for x, y in zip(a, b):
        assert torch.equal(_bytes(x), _bytes(y))


def test_no_tokens():
    cache = _cache(2, 16, 1, INT8)
    seqlens = torch.full((2,), 9, dtype=torch.int32, device=DEV)
    none = torch.empty(0, 1, 128, dtype=torch.bfloat16, device=DEV)
    start = torch.tensor([3, 20], dtype=torch.int32, device=DEV)
    infllm_v2.cache_fill_q8(none, none, *cache, cu([0, 0], DEV), start=start, seqlens_out=seqlens)
    assert seqlens.tolist() == [3, 16]
    k, v = infllm_v2.cache_read_q8(*cache, cu([0, 0], DEV), 0)
    assert k.shape == (0, 1, 128) and v.shape == (0, 1, 128)


@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_append_matches_fill_and_recompression(dtype):
    """70 appends leave the cache as one fill of the grown sequences does; windows that they complete are the means
    of the keys as the cache holds them (one bf16 rounding of an fp32 sum of 32 or 128 terms)."""
    lens, cap, hk, steps = [100, 31, 0, 257], 320, 2, 70
    k_all = [_values(n + steps, hk, 10 + n) for n in lens]
    v_all = [_values(n + steps, hk, 20 + n) for n in lens]
    cache, ref = _cache(4, cap, hk, dtype), _cache(4, cap, hk, dtype)
    seqlens = torch.zeros(4, dtype=torch.int32, device=DEV)
    positions, n_comp, n_comp2 = (torch.zeros(4, dtype=torch.int32, device=DEV) for _ in range(3))
    kc, kc2 = torch.zeros(4, 19, hk, 128, dtype=torch.bfloat16, device=DEV), torch.zeros(4, 4, hk, 128, dtype=torch.bfloat16, device=DEV)
    infllm_v2.cache_fill_q8(torch.cat([k[:n] for k, n in zip(k_all, lens)]).to(DEV),
                            torch.cat([v[:n] for v, n in zip(v_all, lens)]).to(DEV), *cache, cu(lens, DEV), seqlens_out=seqlens)
    for s in range(steps):
        kn, vn = (torch.stack([x[min(n + s, x.shape[0] - 1)] for x, n in zip(xs, lens)]).to(DEV) for xs in (k_all, v_all))
        infllm_v2.decode_append_q8(kn, vn, *cache, seqlens, positions, kc, n_comp, 32, 16, kc2, n_comp2, 128, 64)
    grown = [min(n + steps, cap) for n in lens]                  # the last sequence runs into its capacity
    assert seqlens.tolist() == grown and positions.tolist() == [99 + steps, 30 + steps, steps - 1, cap]
    infllm_v2.cache_fill_q8(torch.cat([k[:n] for k, n in zip(k_all, grown)]).to(DEV),
                            torch.cat([v[:n] for v, n in zip(v_all, grown)]).to(DEV), *ref, cu(grown, DEV))
    for x, y in zip(cache, ref):
        assert torch.equal(_bytes(x), _bytes(y))
    kr = infllm_v2.cache_read_q8(*cache, cu(grown, DEV), sum(grown))[0].cpu().double()
    at = 0
    for b, n in enumerate(grown):
        for comp, count, size, step in ((kc, n_comp, 32, 16), (kc2, n_comp2, 128, 64)):
            assert int(count[b]) == (n - size) // step + 1
            for j in range((n - size) // step + 1):
                if step * j + size <= lens[b]:
                    continue                                     # (a window of the prefill: not the append's)
                rows = kr[at + step * j:at + step * j + size]
                want, got = rows.mean(0), comp[b, j].cpu().double()
                tol = 2.0 ** -8 * want.abs() + 2.0 ** -24 * size * rows.abs().mean(0) + 2.0 ** -133
                assert bool(((got - want).abs() <= tol).all())
        at += n


def test_two_calls_at_once_on_two_streams():
    hk, n = 2, 3000
    k, v = det_tensor((n, hk, 128), 1).to(DEV), det_tensor((n, hk, 128), 2).to(DEV)
    caches = [_cache(1, n, hk, d) for d in (E4M3, INT8, E4M3, INT8)]
    cu_d = cu([n], DEV)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for i in range(2):
        with torch.cuda.stream(streams[i]):
            infllm_v2.cache_fill_q8(k, v, *caches[i], cu_d)
            back = infllm_v2.cache_read_q8(*caches[i], cu_d, n)
        infllm_v2.cache_fill_q8(k, v, *caches[i + 2], cu_d)
        streams[i].synchronize()
        torch.cuda.synchronize()
        assert torch.equal(back[0], infllm_v2.cache_read_q8(*caches[i + 2], cu_d, n)[0])


def test_rows_beyond_32_bit_offsets():
    """The last slot of a cache of more than 2^31 bytes of codes."""
    slots, length, hk = 9, 131072, 16
    cache = infllm_v2.q8_cache(slots, length, hk, E4M3, DEV)
    assert cache[0].numel() > 2 ** 31
    k = _values(21, hk, 1)
    lens = [0] * (slots - 1) + [21]
    start = torch.full((slots,), length - 21, dtype=torch.int32, device=DEV)
    infllm_v2.cache_fill_q8(k.to(DEV), k.to(DEV), *cache, cu(lens, DEV), start=start)
    y, e = quantise(k, E4M3)
    assert torch.equal(cache[0][-1, :, -21:].cpu().float().transpose(0, 1), y.float())
    got = infllm_v2.cache_read_q8(*cache, cu(lens, DEV), 21, start=start)[1].cpu()
    assert torch.equal(got, dequantise(y, e).to(torch.bfloat16))

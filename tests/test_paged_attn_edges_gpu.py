"""GPU: attention over 8-bit blocks where its calls can go wrong: shares and joins, empty sequences, lists of any order, queries of
any stride, streams and graphs.  Tolerances: tests/test_paged_attn_gpu.py."""
import math

import pytest
import torch

import infllm_v2
from oracle import paged
from helpers import cu, det_tensor
from test_paged_attn_gpu import E4M3, E5M2, check, make, queries

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def attend(q, cache, cu_q, most, lens, table, **more):
    return infllm_v2.infllmv2_attn_paged_b8(q.to(DEV), *cache, cu_q.to(DEV), most, ints(lens),
                                            block_table=None if table is None else table.to(DEV), return_softmax_lse=True, **more)


@pytest.mark.parametrize("most,new_of", [(1, lambda i: 1), (2, lambda i: i % 3), (8, lambda i: i % 6), (20, lambda i: (i * 7) % 21)])
def test_more_tiles_than_shares(most, new_of):
    """Hundreds of short sequences, some without keys and some without tokens: a CTA has many tiles, a tile two CTAs."""
    batch = 400 if most == 1 else 90
    lens = [(i * 37) % 300 if i % 11 else 0 for i in range(batch)]
    new = [new_of(i) for i in range(batch)]
    cache, table, k, v = make(lens, 1, 64, E4M3, 41)
    q, cu_q = queries(new, 1, 42), cu(new)
    check(attend(q, cache, cu_q, most, lens, table), q, k, v, cu_q, lens, table)


@pytest.mark.parametrize("hk", [1, 3, 8])
def test_heads(hk):
    lens, new = [400, 77], [1, 1]
    for new in ([1, 1], [2, 1], [5, 9]):
        cache, table, k, v = make(lens, hk, 128, E5M2, 43)
        q, cu_q = queries(new, hk, 44), cu(new)
        check(attend(q, cache, cu_q, max(new), lens, table), q, k, v, cu_q, lens, table)


@pytest.mark.parametrize("said", [1, 2, 3, 8, 9, 500])
def test_a_larger_bound_on_the_tokens(said):
    """max_seqlen_q is a bound: what is said decides which kernel runs, not the result."""
    lens, new = [333, 64, 1], [1, 1, 1]
    cache, table, k, v = make(lens, 2, 64, E4M3, 45)
    q, cu_q = queries(new, 2, 46), cu(new)
    check(attend(q, cache, cu_q, said, lens, table), q, k, v, cu_q, lens, table)


def test_costs_past_32_bits():
    """A table so wide that the cost of what it has room for passes 2^30: tiles are listed by a kernel of their own."""
    length, width, batch = 65536, 16384, 64
    lens = [70 + i for i in range(batch)]
    table = torch.full((batch, width), -1, dtype=torch.int32)
    table[:, 0] = torch.arange(batch) % 2
    cache, _, k, v = make([200, 210], 2, 0, E4M3, 47, extra=0)
    grown = infllm_v2.b8_cache(2, length, 2, E4M3, DEV)
    for big, small in zip(grown, cache):
        big.view(torch.uint8)[:, :, :small.shape[2]] = small.view(torch.uint8)
    new = [1] * batch
    q, cu_q = queries(new, 2, 48), cu(new)
    wide = torch.zeros(2, 2, length, 128, dtype=torch.float64)
    kk, vv = wide.clone(), wide
    kk[:, :, :k.shape[2]], vv[:, :, :v.shape[2]] = k.nan_to_num(0.0), v.nan_to_num(0.0)
    check(attend(q, grown, cu_q, 1, lens, table), q, kk, vv, cu_q, lens, table)


@pytest.mark.parametrize("new", [[1, 1], [2, 2], [4, 3], [12, 9]])
def test_lists_of_any_order(new):
    """Unsorted, with entries twice, unused ones in between, blocks past the sequence and past the capacity, long and empty lists."""
    lens, hk = [1500, 300], 2
    cache, table, k, v = make(lens, hk, 64, E4M3, 49)
    q, cu_q = queries(new, hk, 50), cu(new)
    g = torch.Generator().manual_seed(51)
    for n in (1, 7, 300, 0):
        lists = torch.randint(-3, 40, (hk, sum(new), n), generator=g).to(torch.int32)
        if n > 3:
            lists[:, 0, 1], lists[:, 0, 2] = 2 ** 31 - 1, -2 ** 31
        check(attend(q, cache, cu_q, max(new), lens, table, topk_idx=lists.to(DEV)), q, k, v, cu_q, lens, table, True, lists)


def test_masks_as_wide_as_they_may_be():
    lens, new, hk = [5000], [1], 1
    cache, table, k, v = make(lens, hk, 64, E4M3, 52)
    wide = torch.full((1, 8192), -1, dtype=torch.int32)
    wide[0, :table.shape[1]] = table[0]
    q, cu_q = queries(new, hk, 53), cu(new)
    lists = torch.tensor([[[0, 3, 63, 64, 65, 77, 78, 8191]]], dtype=torch.int32)
    mask, _ = infllm_v2.topk_to_uint64(lists.to(DEV), 8192 * 64, 64)
    check(attend(q, cache, cu_q, 1, lens, wide, block_mask=mask), q, k, v, cu_q, lens, wide, True, lists)
    check(attend(q, cache, cu_q, 1, lens, wide, topk_idx=lists.to(DEV)), q, k, v, cu_q, lens, wide, True, lists)
    with pytest.raises(RuntimeError, match="524288"):
        attend(q, cache, cu_q, 1, lens, torch.cat([wide, wide[:, :1]], 1), topk_idx=lists.to(DEV))


@pytest.mark.parametrize("new", [[1], [2], [10]])
def test_scales_of_any_sign(new):
    lens = [300]
    cache, table, k, v = make(lens, 1, 64, E4M3, 54)
    q, cu_q = queries(new, 1, 55), cu(new)
    for scale in (-0.1, 1e-6, 0.7):
        check(attend(q, cache, cu_q, max(new), lens, table, softmax_scale=scale), q, k, v, cu_q, lens, table, True, None, scale)
    out, lse = attend(q, cache, cu_q, max(new), lens, table, softmax_scale=0.0)
    ref, ref_lse, size, _ = paged.attend(q, k, v, cu_q.tolist(), lens, table, True, None, 0.0)
    assert bool(((out.cpu().double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -8 * size).all())
    assert bool(((lse.cpu().double() - ref_lse).abs() <= 1e-5).all())


@pytest.mark.parametrize("new", [[1, 1], [2, 2], [10, 20]])
def test_a_nan_in_a_query_stays_in_its_row(new):
    lens = [200, 130]
    cache, table, k, v = make(lens, 1, 64, E4M3, 56)
    q, cu_q = queries(new, 1, 57), cu(new)
    q[0, 3, 7], q[-1, 5, 0] = float("nan"), float("inf")
    out, lse = (x.cpu() for x in attend(q, cache, cu_q, max(new), lens, table))
    rows = torch.zeros(lse.shape, dtype=torch.bool)
    rows[0, 3], rows[-1, 5] = True, True
    assert torch.equal(lse.isnan(), rows) and torch.equal(out.isnan().all(-1), rows) and torch.equal(out.isnan().any(-1), rows)


def test_queries_of_other_strides():
    lens, new, hk = [150, 90], [1, 1], 2
    cache, table, k, v = make(lens, hk, 64, E4M3, 58)
    x = det_tensor((2, 16 * hk + 4, 257), 59).to(DEV)
    for q in (x[:, 2:2 + 16 * hk, 1:129], x[:, :16 * hk, ::2][..., :128]):
        check(attend(q, cache, cu(new), 1, lens, table), q.cpu().contiguous(), k, v, cu(new), lens, table)
    flat = torch.zeros(2 * 32 * 128 + 1, dtype=torch.bfloat16, device=DEV)
    odd = flat[1:].view(2, 32, 128)
    odd.copy_(x[:, :32, :128])
    check(attend(odd, cache, cu(new), 1, lens, table), odd.cpu(), k, v, cu(new), lens, table)


@pytest.mark.parametrize("new", [[1, 1, 1], [2, 1, 2], [8, 3, 5], [40, 3, 17]])
def test_streams_graphs_and_calls_at_once(new):
    """The same bits from the current stream, from another, from two at once, and from graphs whose inputs change."""
    lens, hk = [2000, 64, 700], 2
    cache, table, k, v = make(lens, hk, 64, E4M3, 60)
    q, cu_q = queries(new, hk, 61).to(DEV), cu(new, DEV)
    args = lambda x: (x, *cache, cu_q, max(new), ints(lens))       # noqa: E731
    more = dict(block_table=table.to(DEV), return_softmax_lse=True)
    want = infllm_v2.infllmv2_attn_paged_b8(*args(q), **more)
    want2 = infllm_v2.infllmv2_attn_paged_b8(*args(-q), **more)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for st, x in zip(streams, (q, -q)):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                got.append(infllm_v2.infllmv2_attn_paged_b8(*args(x), **more))
        torch.cuda.synchronize()
        for g, w in zip(got, (want, want2)):
            assert all(torch.equal(a, b) for a, b in zip(g, w))
    held = q.clone()
    inputs = args(held)
    graphs, outs = [], []
    torch.cuda.synchronize()
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(infllm_v2.infllmv2_attn_paged_b8(*inputs, **more))
        graphs.append(graph)
    for x, w in ((q, want), (-q, want2), (q, want)):
        held.copy_(x)
        for graph, out in zip(graphs, outs):
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(out, w))


def test_without_a_table_pages_are_sequences():
    """More pages than sequences, a capacity that no length reaches, lengths past it."""
    lens = [64, 200]
    cache, _, k, v = make(lens, 2, 0, E4M3, 62, extra=5)
    q, cu_q = queries([1, 1], 2, 63), cu([1, 1])
    check(attend(q, cache, cu_q, 1, lens, None), q, k, v, cu_q, lens, None)
    cap = cache[0].shape[2]
    full = [cap, cap]
    for c in cache[:2]:
        c.view(torch.uint8)[:2, :, 200:] = 0
        c.view(torch.uint8)[0, :, 64:] = 0
    k, v = (paged.numbers(cache[i].cpu(), cache[2 + i].view(torch.uint8).cpu()) for i in (0, 1))
    check(attend(q, cache, cu_q, 1, [cap + 100, 10 ** 9], None), q, k, v, cu_q, full, None)
    out, lse = attend(q, cache, cu_q, 1, [-3, 0], None)
    assert bool((out == 0).all()) and bool((lse == math.inf).all())
    empty = infllm_v2.infllmv2_attn_paged_b8(q.to(DEV)[:0], *cache, torch.zeros(3, dtype=torch.int32, device=DEV), 1, ints(lens))
    assert empty.shape == (0, 32, 128)


def test_keys_past_32_bits():
    """Blocks whose bytes are past 2^32 from the start of the cache, written and attended."""
    pages, page, hk = 2500, 4096, 4                                # 5.2 GB a cache
    cache = [torch.empty(pages, hk, page, 128, dtype=torch.uint8, device=DEV).view(E4M3) for _ in range(2)]
    cache += [torch.zeros(pages, hk, page // 64, dtype=torch.uint8, device=DEV).view(torch.float8_e8m0fnu) for _ in range(2)]
    n, own = 5000, [2499, 2100]
    k, v = det_tensor((n, hk, 128), 64), det_tensor((n, hk, 128), 65)
    pos = torch.arange(n)
    slots = torch.tensor(own)[pos // page] * page + pos % page
    infllm_v2.cache_write_b8(k.to(DEV), v.to(DEV), *cache, slots.to(DEV))
    kk, vv = (paged.numbers(cache[i].view(torch.uint8)[own].cpu().view(E4M3), cache[2 + i].view(torch.uint8)[own].cpu()) for i in (0, 1))
    kk[1, :, n - page:], vv[1, :, n - page:] = 0, 0                # (never written)
    for new in ([1], [10]):
        q, cu_q = queries(new, hk, 66), cu(new)
        got = attend(q, cache, cu_q, max(new), [n], torch.tensor([own], dtype=torch.int32))
        check(got, q, kk, vv, cu_q, [n], torch.tensor([[0, 1]]))


@pytest.mark.parametrize("most", [1, 2, 8, 20])
@pytest.mark.parametrize("batch", [3, 400])
def test_no_sequence_has_a_token(most, batch):
    """Rows, but none of a sequence: no tile for anyone, whichever way tiles are dealt."""
    lens = [100] * batch
    cache, table, _, _ = make([100], 2, 64, E4M3, 67)
    table = table.expand(batch, -1).contiguous()
    q = queries([5], 2, 68)
    for more in (dict(), dict(topk_idx=ints([[[0, 1]] * 5] * 2))):
        out, lse = attend(q, cache, torch.zeros(batch + 1, dtype=torch.int32), most, lens, table, **more)
        assert bool((out == 0).all()) and bool((lse == math.inf).all())
    infllm_v2.check_device_status()


@pytest.mark.parametrize("new", [[1, 1], [4, 3], [12, 9]])
def test_lists_longer_than_the_blocks_there_are(new):
    lens, hk = [700, 300], 2
    cache, table, k, v = make(lens, hk, 64, E4M3, 69)
    q, cu_q = queries(new, hk, 70), cu(new)
    lists = (torch.arange(20001, dtype=torch.int32) * 7 % 30000).expand(hk, sum(new), -1).contiguous()
    lists[1] = lists[1] % 5
    check(attend(q, cache, cu_q, max(new), lens, table, topk_idx=lists.to(DEV)), q, k, v, cu_q, lens, table, True, lists)


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("new", [[1], [2], [10]])
def test_blocks_of_the_smallest_scale(new, dtype):
    """Values whose block has the exponent -127, alone and before a block of the usual size.  Results stay above 2^-126 where it is
    alone: below, 32-bit arithmetic may give 0, so that is what they may be off by."""
    for lens, v_size in (([3], 2.0 ** -122), ([130], lambda pos: torch.where(pos < 64, 2.0 ** -122, 1.0).double())):
        cache, table, k, v = make(lens, 1, 64, dtype, 71, v_size=v_size)
        assert int(cache[3].view(torch.uint8)[int(table[0, 0])]) == 0
        q, cu_q = queries(new, 1, 72), cu(new)
        out, lse = (x.cpu() for x in attend(q, cache, cu_q, max(new), lens, table))
        ref, ref_lse, size, _ = paged.attend(q, k, v, cu_q.tolist(), lens, table, True, None, None)
        none = ref_lse == math.inf
        assert torch.equal(none, lse == math.inf)
        assert bool(((out.double() - ref).abs() <= 2.0 ** -8 * ref.abs() + 2.0 ** -7 * size + 2.0 ** -126).all())
        assert not bool((out.double()[~none] == 0).all())


@pytest.mark.parametrize("most", [1, 2, 5])
def test_thousands_of_sequences(most):
    """More sequences than a CTA has threads, over pages that they share."""
    batch = 2500
    cache, table, k, v = make([128] * 5, 1, 64, E4M3, 73)
    lens = [(i * 29) % 129 for i in range(batch)]
    new = [1 + (i * 7) % most if i % 13 else 0 for i in range(batch)]
    table = table[torch.arange(batch) % 5].contiguous()
    q, cu_q = queries(new, 1, 74), cu(new)
    check(attend(q, cache, cu_q, most, lens, table), q, k, v, cu_q, lens, table)

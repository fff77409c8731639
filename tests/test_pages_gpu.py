"""GPU: page tables of a step against the definition request by request, and rows written by slot.  Whole numbers and copies:
everything is equal."""
import random

import pytest
import torch

import infllm_v2
from oracle import paged
from helpers import det_tensor

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def problem(seed, batch, most, page, spare, grow, shrink, width_slack=2, big=0):
    """Lengths before and after, a table of used pages with a mark (-7) everywhere else, and a ring that begins anywhere."""
    rng = random.Random(seed)
    old = [rng.randint(0, most) for _ in range(batch)]
    new = []
    for n in old:
        x = rng.random()
        new.append(n + rng.randint(1, max(2, big or most)) if x < grow else rng.choice([0, rng.randint(0, n)]) if x < grow + shrink else n)
    pages = lambda n: -(-n // page)                                # noqa: E731
    width = max(pages(n) for n in old + new) + width_slack
    width = max(width, 1)
    used = sum(pages(n) for n in old)
    ids = list(range(used + spare + 5))
    rng.shuffle(ids)
    table, at = [], 0
    for n in old:
        table.append(ids[at:at + pages(n)] + [-7] * (width - pages(n)))
        at += pages(n)
    size = len(ids)
    first = rng.randrange(size)
    ring = [-9] * size
    for i in range(spare):
        ring[(first + i) % size] = ids[at + i]
    return old, new, table, ring, [first, spare]


def run(old, new, table, ring, free_range, page, total):
    table_d, ring_d = ints(table), ints(ring)
    got = infllm_v2.pages_resize(ints(old), ints(new), table_d, ring_d, ints(free_range), page, total)
    return [x.tolist() for x in got] + [table_d.tolist(), ring_d.tolist()]


def check(old, new, table, ring, free_range, page, total):
    want = paged.resize(old, new, table, ring, free_range, page, total)
    got = run(old, new, table, ring, free_range, page, total)
    for name, g, w in zip(("seqlens", "free_range", "cu_seqlens", "positions", "slots", "block_table", "free_pages"), got, want):
        assert g == w, name


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("batch,most,page,spare,grow,shrink", [
    (1, 10, 64, 3, 1.0, 0.0), (1, 300, 16, 40, 0.0, 1.0), (7, 100, 16, 60, 0.6, 0.3), (64, 1000, 64, 900, 0.5, 0.3),
    (255, 50, 1, 9000, 0.5, 0.5), (257, 40, 7, 700, 0.4, 0.4), (600, 30, 64, 400, 0.3, 0.3), (33, 700, 80, 0, 0.5, 0.5),
    (40, 300, 16, 50, 0.9, 0.05), (300, 200, 16, 300, 0.7, 0.2)])
def test_against_the_definition(seed, batch, most, page, spare, grow, shrink):
    p = problem(seed, batch, most, page, spare, grow, shrink)
    check(*p, page, sum(max(b - a, 0) for a, b in zip(p[0], p[1])))


@pytest.mark.parametrize("batch", [5, 300])
def test_rows_behind_and_totals_that_are_not_the_sum(batch):
    p = problem(5, batch, 60, 16, 2000, 0.7, 0.1)
    total = sum(max(b - a, 0) for a, b in zip(p[0], p[1]))
    for n in (0, 1, total // 2, total + 1, total + 999):
        check(*p, 16, n)


def test_requests_wider_than_their_rows_are_refused():
    old, new, table, ring, free_range = problem(3, 20, 100, 16, 300, 0.0, 0.0, width_slack=0)
    width = len(table[0])
    new = [n + (1000 if i % 3 == 0 else 5) for i, n in enumerate(old)]
    assert any(-(-n // 16) > width for n in new)
    check(old, new, table, ring, free_range, 16, sum(new) - sum(old))


def test_a_long_prompt_among_many():
    p = problem(9, 200, 3000, 64, 9000, 0.3, 0.2, big=20000)
    check(*p, 64, sum(max(b - a, 0) for a, b in zip(p[0], p[1])))


def test_negative_lengths_are_none():
    table, ring = [[-7, -7]] * 3, list(range(9))
    got = run([-5, 0, 3], [4, -1, -8], [r[:] for r in table[:2]] + [[8, -7]], ring[:8] + [-1], [0, 8], 4, 4)
    assert got[0] == [4, 0, 0] and got[2] == [0, 4, 4, 4] and got[3] == [0, 1, 2, 3] and got[4] == [0, 1, 2, 3]
    assert got[1] == [1, 8] and got[6] == list(range(8)) + [8]


def test_table_rows_of_another_stride_and_a_second_call():
    old, new, table, ring, free_range = problem(11, 30, 200, 16, 600, 0.6, 0.2)
    wide = torch.full((30, len(table[0]) + 9), -5, dtype=torch.int32, device=DEV)
    view = wide[:, 3:3 + len(table[0])]
    view.copy_(ints(table))
    total = sum(max(b - a, 0) for a, b in zip(old, new))
    args = (ints(old), ints(new), view, ints(ring), ints(free_range), 16, total)
    want = paged.resize(old, new, table, ring, free_range, 16, total)
    for _ in range(2):                                             # (nothing that is read is written)
        got = infllm_v2.pages_resize(*args)
        assert [x.tolist() for x in got] == [list(x) for x in want[:5]]
        assert view.tolist() == want[5] and args[3].tolist() == want[6]
    assert bool((wide[:, :3] == -5).all()) and bool((wide[:, 3 + len(table[0]):] == -5).all())


def test_pages_go_round():
    """Requests come and go for a while: no page is ever in two places, and all come back."""
    batch, page, width, pages = 13, 16, 12, 90
    rng = random.Random(2)
    ring, left = infllm_v2.page_pool(pages, DEV)
    table = torch.full((batch, width), -1, dtype=torch.int32, device=DEV)
    lens = ints([0] * batch)
    for step in range(60):
        now = lens.tolist()
        new = [0 if rng.random() < 0.15 else min(n + rng.randint(0, 30), width * page) for n in now]
        if step == 59:
            new = [0] * batch
        total = sum(max(b - a, 0) for a, b in zip(now, new))
        lens, left, cu, pos, slots = infllm_v2.pages_resize(lens, ints(new), table, ring, left, page, total)
        held = [p for row, n in zip(table.tolist(), lens.tolist()) for p in row[:-(-n // page)]]
        first, count = left.tolist()
        free = [ring.tolist()[(first + i) % pages] for i in range(count)]
        assert sorted(held + free) == list(range(pages))
        got = [s for s in slots.tolist() if s >= 0]
        assert len(set(got)) == len(got) and all(s // page in held for s in got)
    assert lens.tolist() == [0] * batch and left.tolist()[1] == pages


def test_captured_step():
    """A step in a CUDA graph, whose state is copied back within it: ten replays are ten steps."""
    batch, page, width = 5, 16, 8
    ring, left = infllm_v2.page_pool(50, DEV)
    table = torch.full((batch, width), -1, dtype=torch.int32, device=DEV)
    lens = ints([3, 0, 16, 31, 15])
    want_lens, want_range, want_table, want_ring = [0] * batch, left.tolist(), table.tolist(), ring.tolist()
    r = paged.resize(want_lens, lens.tolist(), want_table, want_ring, want_range, page, 0)
    lens0, left, *_ = infllm_v2.pages_resize(ints([0] * batch), lens, table, ring, left, page, 0)
    lens, left = lens0.clone(), left.clone()
    want_lens, want_range, want_table, want_ring = list(r[0]), list(r[1]), r[5], r[6]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        infllm_v2.pages_resize(lens, lens + 1, table.clone(), ring.clone(), left, page, batch)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        after, rest, cu, pos, slots = infllm_v2.pages_resize(lens, lens + 1, table, ring, left, page, batch)
        lens.copy_(after)
        left.copy_(rest)
    for _ in range(10):
        graph.replay()
        r = paged.resize(want_lens, [n + 1 for n in want_lens], want_table, want_ring, want_range, page, batch)
        assert pos.tolist() == r[3] and slots.tolist() == r[4]
        want_lens, want_range, want_table, want_ring = list(r[0]), list(r[1]), r[5], r[6]
    assert lens.tolist() == want_lens and left.tolist() == want_range and table.tolist() == want_table


@pytest.mark.parametrize("total,hk,page,fused", [(1, 1, 16, False), (7, 2, 64, True), (8, 3, 1, False), (9, 8, 256, True), (1000, 2, 16, True),
                                                 (333, 5, 80, False)])
def test_rows_by_slot(total, hk, page, fused):
    g = torch.Generator().manual_seed(total)
    pages = total // page + 3
    slots = torch.randperm(pages * page, generator=g)[:total]
    slots[torch.rand(total, generator=g) < 0.1] = -1
    if total > 5:
        slots[3], slots[4] = pages * page, 2 ** 40
    k, v = det_tensor((total, hk, 128), 1), det_tensor((total, hk, 128), 2)
    kc, vc = (torch.full((pages, page, hk, 128), x, dtype=torch.bfloat16, device=DEV) for x in (3.0, 5.0))
    kd, vd = k.to(DEV), v.to(DEV)
    if fused:
        qkv = torch.zeros(total, 4 + 2 * hk, 128, dtype=torch.bfloat16, device=DEV)
        qkv[:, 4:4 + hk], qkv[:, 4 + hk:] = kd, vd
        kd, vd = qkv[:, 4:4 + hk], qkv[:, 4 + hk:]
    assert infllm_v2.cache_write(kd, vd, kc, vc, slots.to(DEV)) is None
    ok = (slots >= 0) & (slots < pages * page)
    for x, cache, mark in ((k, kc, 3.0), (v, vc, 5.0)):
        want = torch.full((pages * page, hk, 128), mark, dtype=torch.bfloat16)
        want[slots[ok]] = x[ok]
        assert torch.equal(cache.cpu().view(-1, hk, 128), want)


def test_rows_of_other_strides():
    """Features that are not side by side, rows that begin off a 16-byte boundary, no rows at all."""
    k = det_tensor((20, 2, 256), 3).to(DEV)
    kc, vc = torch.zeros(3, 16, 2, 128, dtype=torch.bfloat16, device=DEV), torch.zeros(3, 16, 2, 128, dtype=torch.bfloat16, device=DEV)
    slots = torch.arange(20, device=DEV) * 2
    infllm_v2.cache_write(k[..., ::2], k[..., 3:131], kc, vc, slots)
    assert torch.equal(kc.view(-1, 2, 128)[slots], k[..., ::2]) and torch.equal(vc.view(-1, 2, 128)[slots], k[..., 3:131])
    infllm_v2.cache_write(k[:0, :, :128], k[:0, :, :128], kc, vc, slots[:0])


def test_rows_past_32_bits():
    """Slots whose bytes are past 2^32 from the start of the cache."""
    pages, page, hk = 9, 2 ** 20, 4                                # 9.7 GB a cache
    kc = torch.empty(pages, page, hk, 128, dtype=torch.bfloat16, device=DEV)
    vc = torch.empty_like(kc)
    slots = torch.tensor([0, 5 * page + 7, 9 * page - 1], device=DEV)
    kc.view(-1, hk, 128)[slots], vc.view(-1, hk, 128)[slots] = 0, 0
    k, v = det_tensor((3, hk, 128), 5).to(DEV), det_tensor((3, hk, 128), 6).to(DEV)
    infllm_v2.cache_write(k, v, kc, vc, slots)
    assert torch.equal(kc.view(-1, hk, 128)[slots], k) and torch.equal(vc.view(-1, hk, 128)[slots], v)

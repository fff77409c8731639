"""GPU: a serving loop over pages, from lengths to attention, as an engine would run it: tables and slots, rotation, rows written by
slot, prompts in chunks, decode steps, drafts, requests that end and others that begin; for the cache in 8 bits (against
the formula on the codes that the definition gives) and for the bf16 one."""
import pytest
import torch

import infllm_v2
from oracle import paged
from helpers import det_tensor
from test_paged_attn_gpu import check

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
PAGE, HK, BATCH, WIDTH = 64, 2, 4, 12


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def tables(rows):
    i = torch.arange(64, dtype=torch.float64)
    ang = torch.arange(rows, dtype=torch.float64)[:, None] * (10000.0 ** (-2.0 * i / 128))[None]
    return ang.cos().float().to(DEV), ang.sin().float().to(DEV)


# lengths after each step: prompts in one piece and in two, single tokens, drafts of three taken back to one, an end, a new request
STEPS = [[100, 0, 70, 0], [160, 301, 71, 0], [161, 302, 72, 1], [162, 303, 0, 2], [165, 306, 90, 5], [163, 304, 88, 3], [164, 305, 89, 4]]


class Engine:
    def __init__(self, pages=40):
        self.ring, self.left = infllm_v2.page_pool(pages, DEV)
        self.table = torch.full((BATCH, WIDTH), -1, dtype=torch.int32, device=DEV)
        self.lens = ints([0] * BATCH)
        self.cos, self.sin = tables(WIDTH * PAGE)
        self.seed = 0

    def step(self, target):
        old = self.lens.tolist()
        new = [max(b - a, 0) for a, b in zip(old, target)]
        self.lens, self.left, cu, pos, slots = infllm_v2.pages_resize(self.lens, ints(target), self.table, self.ring, self.left, PAGE, sum(new))
        self.seed += 3
        q, k, v = (det_tensor((max(sum(new), 1), n * HK, 128), self.seed + i)[:sum(new)].to(DEV) for i, n in ((0, 16), (1, 1), (2, 1)))
        q, k = infllm_v2.rotary_axes(q, k, self.cos, self.sin, pos)
        return new, cu, slots, q, k, v


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
def test_serving_in_8_bits(dtype):
    e = Engine()
    cache = list(infllm_v2.b8_cache(40, PAGE, HK, dtype, DEV))
    mine = [t.cpu() for t in cache]
    for target in STEPS:
        new, cu, slots, q, k, v = e.step(target)
        infllm_v2.cache_write_b8(k, v, *cache, slots)
        for i, x in ((0, k), (1, v)):
            y, b = paged.write(x.cpu(), mine[i], mine[2 + i].view(torch.uint8), slots.cpu())
            mine[i], mine[2 + i] = y.float().to(dtype), b.to(torch.uint8).view(torch.float8_e8m0fnu)
            assert torch.equal(cache[i].cpu().double(), y) and torch.equal(cache[2 + i].view(torch.uint8).cpu().long(), b)
        if sum(new) == 0:
            continue
        got = infllm_v2.infllmv2_attn_paged_b8(q, *cache, cu, max(new), e.lens, block_table=e.table, return_softmax_lse=True)
        numbers = [paged.numbers(mine[i], mine[2 + i].view(torch.uint8)) for i in (0, 1)]
        check(got, q.cpu(), *numbers, cu.cpu(), e.lens.tolist(), e.table.cpu())
    assert e.lens.tolist() == STEPS[-1]


def test_serving_in_bf16():
    """The framework's attention over bf16 pages reads what cache_write and pages_resize put there."""
    e = Engine()
    kc, vc = (torch.full((40, PAGE, HK, 128), float("nan"), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    kept = [[], []]
    rows = {}
    for target in STEPS:
        new, cu, slots, q, k, v = e.step(target)
        infllm_v2.cache_write(k, v, kc, vc, slots)
        at = 0
        for b, n in enumerate(new):
            rows[b] = [x[:e.lens.tolist()[b] - n] for x in rows.get(b, (k[:0], v[:0]))]
            rows[b] = [torch.cat([x, y[at:at + n]]) for x, y in zip(rows[b], (k, v))]
            at += n
        if max(new) != 1 or min(new) != 1:
            continue
        out = infllm_v2.infllmv2_attn_with_kvcache(q.view(BATCH, 1, 16 * HK, 128), kc, vc, cache_seqlens=e.lens, block_table=e.table)
        for b in range(BATCH):
            kk, vv = (x.double().transpose(0, 1).repeat_interleave(16, 0) for x in rows[b])
            p = torch.softmax(torch.einsum("hd,hkd->hk", q[b].double(), kk) * 128 ** -0.5, -1)
            ref, size = torch.einsum("hk,hkd->hd", p, vv), torch.einsum("hk,hkd->hd", p, vv.abs())
            # bf16 of the result and of the weights, and a little for the scores' fp32
            assert bool(((out[b, 0].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -12) * size).all())
            kept[0].append(b)
    assert kept[0]


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
def test_captured_step_of_all_calls(dtype):
    """One decode step in a graph: tables, rotation, write, attention; ten replays against ten eager steps, bit for bit."""
    def state():
        e = Engine()
        cache = list(infllm_v2.b8_cache(40, PAGE, HK, dtype, DEV))
        new, cu, slots, q, k, v = e.step([60, 130, 1, 64])
        infllm_v2.cache_write_b8(k, v, *cache, slots)
        return e, cache

    def step(e, cache, q, k, v):
        lens, left, cu, pos, slots = infllm_v2.pages_resize(e.lens, e.lens + 1, e.table, e.ring, e.left, PAGE, BATCH)
        q, k = infllm_v2.rotary_axes(q, k, e.cos, e.sin, pos)
        infllm_v2.cache_write_b8(k, v, *cache, slots)
        out = infllm_v2.infllmv2_attn_paged_b8(q, *cache, cu, 1, lens, block_table=e.table)
        e.lens.copy_(lens)
        e.left.copy_(left)
        return out

    inputs = [[det_tensor((BATCH, n * HK, 128), 100 + 3 * t + i).to(DEV) for i, n in ((0, 16), (1, 1), (2, 1))] for t in range(10)]
    e, cache = state()
    e.lens, e.left = e.lens.clone(), e.left.clone()
    want = [step(e, cache, *x).clone() for x in inputs]
    e2, cache2 = state()
    e2.lens, e2.left = e2.lens.clone(), e2.left.clone()
    held = [x.clone() for x in inputs[0]]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(e2, cache2, *held)
    for x, w in zip(inputs, want):
        for a, b in zip(held, x):
            a.copy_(b)
        graph.replay()
        assert torch.equal(out, w)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache, cache2))


def test_states_of_an_encoder():
    """Cross attention: decoder tokens over the states of another length, written once, attended without an order."""
    lens, new = [333, 64, 150], [5, 1, 20]
    ring, left = infllm_v2.page_pool(20, DEV)
    table = torch.full((3, 6), -1, dtype=torch.int32, device=DEV)
    lens_d, left, cu, pos, slots = infllm_v2.pages_resize(ints([0, 0, 0]), ints(lens), table, ring, left, 64, sum(lens))
    cache = list(infllm_v2.b8_cache(20, 64, HK, E4M3, DEV))
    infllm_v2.cache_write_b8(det_tensor((sum(lens), HK, 128), 1).to(DEV), det_tensor((sum(lens), HK, 128), 2).to(DEV), *cache, slots)
    numbers = [paged.numbers(cache[i].cpu(), cache[2 + i].view(torch.uint8).cpu()) for i in (0, 1)]
    q = det_tensor((sum(new), 16 * HK, 128), 3)
    cu_q = torch.tensor([0, 5, 6, 26], dtype=torch.int32)
    got = infllm_v2.infllmv2_attn_paged_b8(q.to(DEV), *cache, cu_q.to(DEV), 20, lens_d, block_table=table, causal=False, return_softmax_lse=True)
    check(got, q, *numbers, cu_q, lens, table.cpu(), False)

"""GPU: what pages_resize and the writes by slot give to the calls that read pages: prompts' chunks over bf16 pages, block scores over pages
of compressed keys (bit for bit as over packed rows), and a step in which a request is refused."""
import pytest
import torch

import infllm_v2
import oracle
from oracle import paged
from helpers import cu, det_tensor, local_topk
from test_paged_attn_gpu import E4M3, check
from test_paged_serve_gpu import BATCH, HK, PAGE, STEPS, Engine

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("selected", [False, True])
def test_chunks_over_bf16_pages(selected):
    """Every step of a serving loop through infllmv2_attn_varlen_func: prompts in pieces, drafts, single tokens, requests without any."""
    e = Engine()
    kc, vc = (torch.full((40, PAGE, HK, 128), float("nan"), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    rows = {b: [torch.zeros(0, HK, 128, dtype=torch.bfloat16, device=DEV)] * 2 for b in range(BATCH)}
    for n, target in enumerate(STEPS):
        new, cu_q, slots, q, k, v = e.step(target)
        infllm_v2.cache_write(k, v, kc, vc, slots)
        lens, at = e.lens.tolist(), 0
        for b in range(BATCH):
            rows[b] = [torch.cat([x[:lens[b] - new[b]], y[at:at + new[b]]]) for x, y in zip(rows[b], (k, v))]
            at += new[b]
        if sum(new) == 0:
            continue
        packed = [torch.cat([rows[b][i] for b in range(BATCH)]) for i in (0, 1)]
        lists = local_topk(HK, new, lens, 2, 100 + n).to(DEV) if selected else None
        more = dict(causal=True, topk_idx=lists, return_attn_probs=True)
        cu_k = cu(lens, DEV)
        want = infllm_v2.infllmv2_attn_varlen_func(q, *packed, cu_q, cu_k, max(new), max(lens), **more)
        got = infllm_v2.infllmv2_attn_varlen_func(q, kc, vc, cu_q, cu_k, max(new), max(lens), block_table=e.table, **more)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and not bool(got[0].isnan().any())
        infllm_v2.check_device_status()
        if selected:
            ref, _ = oracle.sparse_attention_fwd(q.cpu(), *(x.cpu() for x in packed), cu_q.cpu(), cu_k.cpu(), lists.cpu(), causal=True)
            size, _ = oracle.sparse_attention_fwd(q.cpu(), packed[0].cpu(), packed[1].cpu().abs(), cu_q.cpu(), cu_k.cpu(), lists.cpu(), causal=True)
            # bf16 of the result and of the weights, and a little for the scores' fp32
            assert bool(((got[0].cpu().float() - ref).abs() <= 2.0 ** -8 * ref.abs() + (2.0 ** -8 + 2.0 ** -12) * size).all())


def test_block_scores_over_pages_of_compressed_keys():
    lens, page = [700, 4200, 40], 128
    k = det_tensor((sum(lens), HK, 128), 1, 0.5)
    q = det_tensor((sum(lens), 16 * HK, 128), 2, 0.5).to(DEV)
    kc, cu_c = oracle.compress_keys(k, cu(lens).tolist())
    n = [b - a for a, b in zip(cu_c, cu_c[1:])]
    ring, left = infllm_v2.page_pool(9, DEV)
    ring.copy_(ring.flip(0))
    table = torch.full((3, 3), -1, dtype=torch.int32, device=DEV)
    after, left, cu_new, _, slots = infllm_v2.pages_resize(ints([0, 0, 0]), ints(n), table, ring, left, page, sum(n))
    assert cu_new.tolist() == cu_c and after.tolist() == n
    pages, spare = (torch.full((9, page, HK, 128), 1e4, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    kc = kc.to(DEV)
    infllm_v2.cache_write(kc, -kc, pages, spare, slots)
    cu_q = cu(lens, DEV)
    want = infllm_v2.infllmv2_attn_stage1(q, kc, kc, cu_q, cu_new, cu_new, max(lens), max(n), causal=True)
    got = infllm_v2.infllmv2_attn_stage1(q, pages, pages, cu_q, cu_new, cu_new, max(lens), max(n), causal=True, block_table=table)
    assert torch.equal(got, want)
    rows = [r for i in range(3) for r in (int(table[i, j // page]) * page + j % page for j in range(n[i]))]
    assert torch.equal(spare.view(-1, HK, 128)[rows], -kc) and int((spare == 1e4).all(-1).all(-1).sum()) == 9 * page - sum(n)


@pytest.mark.parametrize("which", [0, 1, 2])
def test_a_step_with_a_refused_request(which):
    """The refused request's tokens are counted in cu_seqlens and go nowhere; the others' results are what they are without it."""
    lens, grow = [100, 50, 70], [30, 5, 1]
    ring, left = infllm_v2.page_pool(12, DEV)
    table = torch.full((3, 3), -1, dtype=torch.int32, device=DEV)
    cache = list(infllm_v2.b8_cache(12, 64, HK, E4M3, DEV))
    mine = [t.cpu() for t in cache]
    seq = ints([0, 0, 0])
    for step in range(2):
        new = lens if step == 0 else [200 if b == which else g for b, g in enumerate(grow)]
        targets = ints([a + b for a, b in zip(seq.tolist(), new)])
        seq, left, cu_q, _, slots = infllm_v2.pages_resize(seq, targets, table, ring, left, 64, sum(new))
        q, k, v = (det_tensor((sum(new), m * HK, 128), 10 * step + i).to(DEV) for i, m in ((0, 16), (1, 1), (2, 1)))
        infllm_v2.cache_write_b8(k, v, *cache, slots)
        for i, x in ((0, k), (1, v)):
            y, b = paged.write(x.cpu(), mine[i], mine[2 + i].view(torch.uint8), slots.cpu())
            mine[i], mine[2 + i] = y.float().to(E4M3), b.to(torch.uint8).view(torch.float8_e8m0fnu)
    assert seq.tolist() == [n if b == which else n + g for b, (n, g) in enumerate(zip(lens, grow))]
    assert cu_q.tolist() == cu(new).tolist() and bool((slots[int(cu_q[which]):int(cu_q[which + 1])] == -1).all())
    assert torch.equal(cache[0].cpu().view(torch.uint8), mine[0].view(torch.uint8))
    out, lse = infllm_v2.infllmv2_attn_paged_b8(q, *cache, cu_q, max(new), seq, block_table=table, return_softmax_lse=True)
    rows = torch.cat([torch.arange(int(cu_q[b]), int(cu_q[b + 1])) for b in range(3) if b != which])
    others = [b for b in range(3) if b != which]
    numbers = [paged.numbers(mine[i], mine[2 + i].view(torch.uint8)) for i in (0, 1)]
    check((out[rows], lse[rows]), q.cpu()[rows], *numbers, cu([new[b] for b in others]), [seq.tolist()[b] for b in others],
          table.cpu()[others])

"""GPU: blocks that are NaN and pages that are not there, beside blocks that are neither.  Tolerances: tests/test_paged_attn_gpu.py.

Many sequences read the same pages, so that a thread block has whole tiles and its units follow one another in one share."""
import math

import pytest
import torch

import infllm_v2
from oracle import paged
from helpers import cu
from test_paged_attn_gpu import E4M3, E5M2, check, make, queries

pytestmark = pytest.mark.gpu
DEV = "cuda"


def attend(q, cache, cu_q, most, lens, table, **more):
    return infllm_v2.infllmv2_attn_paged_b8(q.to(DEV), *cache, cu_q.to(DEV), most, torch.tensor(lens, dtype=torch.int32, device=DEV),
                                            block_table=table.to(DEV), return_softmax_lse=True, **more)


def many(length, new, hk, dtype, seed, k_size=1.0, v_size=1.0, sequences=None):
    """`sequences` sequences of one table's pages: (cache, table, k, v, lens, q, cu_q)."""
    cache, table, k, v = make([length], hk, 64, dtype, seed, k_size, v_size)
    n = sequences or (150 if new <= 2 else 80)
    q = queries([new] * n, hk, seed + 1)
    return cache, table.expand(n, -1).contiguous(), k, v, [length] * n, q, cu([new] * n)


def check_some(got, q, k, v, cu_q, lens, table, causal=True, lists=None):
    """`check` of the first, a middle and the last sequence."""
    some = [0, len(lens) // 2, len(lens) - 1]
    rows = torch.cat([torch.arange(int(cu_q[b]), int(cu_q[b + 1])) for b in some])
    check([x.cpu()[rows] for x in got], q[rows], k, v, cu([int(cu_q[b + 1] - cu_q[b]) for b in some]), [lens[b] for b in some],
          table[some], causal, None if lists is None else lists[:, rows])


def spoil(cache, numbers, which, table, blocks):
    """Blocks of sequence 0 become NaN: their scale bytes, and what the formula reads."""
    for block in blocks:
        page = int(table[0, block])
        cache[2 + which].view(torch.uint8)[page] = 255
        numbers[page] = math.nan


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("new", [1, 2, 3, 20])
@pytest.mark.parametrize("size", [1.0, 2.0 ** -60, 2.0 ** 60])
def test_lse_behind_nan_values(dtype, new, size):
    """The values of a tile's first two units are NaN, the keys are not: the sums go on as if nothing were wrong with the values."""
    cache, table, k, v, lens, q, cu_q = many(64 * 11 + 7, new, 1, dtype, 81, v_size=size, sequences=60 if new == 20 else None)
    spoil(cache, v, 1, table, range(4))
    got = attend(q, cache, cu_q, new, lens, table)
    check_some(got, q, k, v, cu_q, lens, table)
    assert bool(got[0].isnan().all()) and not bool(got[1].isnan().any())


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("new", [2, 5, 12])
@pytest.mark.parametrize("size", [2.0 ** -100, 2.0 ** 70])
def test_a_neighbour_of_nan_values_keeps_its_own(dtype, new, size):
    """The first token of each sequence selects blocks of NaN values in front of the others' blocks of very small or large ones."""
    cache, table, k, v, lens, q, cu_q = many(64 * 10, new, 1, dtype, 83, v_size=size, sequences=150 if new == 2 else 40)
    spoil(cache, v, 1, table, range(4))
    lists = torch.tensor([4, 5, 6, 8], dtype=torch.int32).repeat(1, q.shape[0], 1)
    lists[0, ::new] = torch.tensor([0, 1, 2, 3], dtype=torch.int32)
    got = attend(q, cache, cu_q, new, lens, table, topk_idx=lists.to(DEV), causal=False)
    check_some(got, q, k, v, cu_q, lens, table, False, lists)
    nan = got[0].isnan().all(-1).all(-1)
    assert bool(nan[::new].all()) and int(nan.sum()) == len(lens)


@pytest.mark.parametrize("new", [1, 2, 3, 20])
@pytest.mark.parametrize("nan_unit,high_unit", [(0, 1), (1, 0), (0, 2), (2, 1), (1, 4)])
def test_nan_values_of_the_lowest_weight(new, nan_unit, high_unit):
    """A NaN block reaches every token that sees it, however far its keys' scores are below those of another unit."""
    cache, table, k, v, lens, q, cu_q = many(64 * 10, new, 1, E4M3, 85, lambda p: torch.where(p // 128 == high_unit, 300.0, 0.01).double(),
                                             sequences=60 if new == 20 else None)
    spoil(cache, v, 1, table, [2 * nan_unit])
    out, lse = attend(q, cache, cu_q, new, lens, table)
    assert bool(out.isnan().all()) and not bool(lse.isnan().any())
    # (far enough apart that even the square root of a weight of the one is nothing beside the other's: 252 log(2))
    assert float(lse.min()) > 200


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("new", [2, 8, 13])
@pytest.mark.parametrize("missing", [-1, 10 ** 6])
def test_missing_pages_of_a_neighbour(dtype, new, missing):
    """Tokens that see nothing of a page which the cache does not have keep their result, whatever lies in page 0."""
    lens = [64 * 5 + 1, 64 * 7 + 30]
    cache, table, k, v = make(lens, 2, 64, dtype, 87)
    cache = [torch.cat([torch.full_like(c.view(torch.uint8)[:1], 0x7F if i < 2 else 130), c.view(torch.uint8)]).view(c.dtype)
             for i, c in enumerate(cache)]                         # (a page of NaN codes in front)
    k, v = (torch.cat([torch.zeros_like(x[:1]), x]) for x in (k, v))
    table = table + 1
    table[0, 5] = missing                                          # of one key: only the last token sees it
    q, cu_q = queries([new, new], 2, 88), cu([new, new])
    out, lse = attend(q, cache, cu_q, new, lens, table)
    check((out, lse), q, k, v, cu_q, lens, table)
    assert not bool(out[:new - 1].isnan().any()) and bool(out[new - 1].isnan().all()) and not bool(out[new:].isnan().any())
    table[1, 3] = missing                                          # a whole block that one token selects
    lists = torch.tensor([0, 1, 6], dtype=torch.int32).repeat(2, 2 * new, 1)
    lists[:, new + 1, 1] = 3
    out, lse = attend(q, cache, cu_q, new, lens, table, topk_idx=lists.to(DEV))
    check((out, lse), q, k, v, cu_q, lens, table, True, lists)
    assert bool(out[new + 1].isnan().all()) and int(out.isnan().all(-1).all(-1).sum()) == 1

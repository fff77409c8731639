"""GPU: attention over 8-bit blocks at the edges of its arithmetic: queries and keys of the largest and smallest sizes, scores that
move the references, walks of many selected blocks.  Tolerances: tests/test_paged_attn_gpu.py, and `check_exact`."""
import math

import pytest
import torch

import infllm_v2
from oracle import paged
from helpers import cu
from test_paged_attn_gpu import E4M3, E5M2, _floor, check, make, queries

pytestmark = pytest.mark.gpu
DEV = "cuda"


def attend(q, cache, cu_q, most, lens, table, **more):
    return infllm_v2.infllmv2_attn_paged_b8(q.to(DEV), *cache, cu_q.to(DEV), most, torch.tensor(lens, dtype=torch.int32, device=DEV),
                                            block_table=table.to(DEV), return_softmax_lse=True, **more)


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("new", [1, 2, 5, 20])
@pytest.mark.parametrize("q_log,k_log", [(-123, 120), (-119, 122), (-100, 100), (100, -100), (118, -121), (122, -124)])
def test_large_keys_and_small_queries(dtype, new, q_log, k_log):
    """Products of ordinary size of factors at the ends of bf16's range: no step on the way leaves fp32's.

    Queries are multiples of 2^-6 of at most 2, times a power of two; where they are subnormal they lose bits, and the formula reads
    what is left.  Keys go to the cache through the definition, so their codes are what they are."""
    lens = [300, 90]
    cache, table, k, v = make(lens, 1, 64, dtype, 91, 2.0 ** k_log)
    q = (queries([new, new], 1, 92).double() * 2.0 ** q_log).to(torch.bfloat16)
    cu_q = cu([new, new])
    check(attend(q, cache, cu_q, new, lens, table), q, k, v, cu_q, lens, table)


def check_exact(got, q, k, v, cu_q, lens, table, **more):
    """`check` for queries that two e4m3 terms hold exactly: scores are off by the fp32 rounding of their 128 products alone, 2^-20 of
    the sum of their magnitudes, and so are results and log-sum-exps."""
    x = q.double().abs().amax(-1, keepdim=True)
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64), 8.0 - torch.floor(torch.log2(x)))
    step = torch.where(x * step > 448, step / 2, step)
    y = q.double() * step * 4                                      # the second term's least step is 2^-9, a first one's rest of 2^-2 x 8 bits
    assert bool((y == y.round()).all()) and float((x * step).max()) <= 448
    out, lse = (t.cpu()[:q.shape[0]] for t in got)
    ref, ref_lse, size, reach = paged.attend(q, k, v, cu_q.tolist(), lens, table, **more)
    slack = (reach + 1) * 2.0 ** -20
    assert float(slack.max()) < 2.0 ** -8
    err = (lse.double() - ref_lse).abs()
    assert bool((err <= slack + 2.0 ** -21 * ref_lse.abs()).all()), float((err - slack).max())
    tol = 2.0 ** -8 * ref.abs() + size * (2.0 ** -9 + 2.0 ** -11) * 1.125 + size * (2 * slack)[..., None] + _floor(v, size) + 2.0 ** -133
    err = (out.double() - ref).abs()
    assert bool((err <= tol).all()), (float((err / tol).max()), (err > tol).nonzero()[:4].tolist())


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("new", [1, 2, 4, 9, 40])
@pytest.mark.parametrize("up", [True, False])
def test_references_that_move(dtype, new, up):
    """Every block's scores above those before it, or below, and values whose blocks differ: what is rescaled on the way is off by no
    more than what is not."""
    length = 64 * 13 + 30
    grow = lambda p: 2.0 * (1.0 + (p if up else length - p) // 64).double()        # noqa: E731
    cache, table, k, v = make([length], 1, 64, dtype, 95, grow, lambda p: torch.pow(2.0, (p // 64 % 5 - 2).double()))
    n = 1 if new > 9 else 60
    q = queries([new] * n, 1, 96, 2.0)
    table = table.expand(n, -1).contiguous()
    got = attend(q, cache, cu([new] * n), new, [length] * n, table)
    few = min(n, 3)
    check_exact(got, q[:few * new], k, v, cu([new] * few), [length] * few, table)


@pytest.mark.parametrize("new", [[1, 1], [2, 1], [3, 2], [9, 4]])
@pytest.mark.parametrize("causal", [True, False])
def test_masks_of_many_blocks(new, causal):
    """Hundreds of selected blocks a token, other ones for every token, as lists and as masks, with an order and without."""
    lens, hk = [10000, 3000], 2
    cache, table, k, v = make(lens, hk, 256, E4M3, 97)
    cap = table.shape[1] * 256
    g = torch.Generator().manual_seed(98)
    lists = torch.stack([torch.stack([torch.randperm(cap // 64, generator=g)[:120].sort().values for _ in range(sum(new))]) for _ in range(hk)])
    lists = lists.to(torch.int32)
    q, cu_q = queries(new, hk, 99), cu(new)
    mask, _ = infllm_v2.topk_to_uint64(lists.to(DEV), cap, 64)
    for more in (dict(topk_idx=lists.to(DEV)), dict(block_mask=mask)):
        got = attend(q, cache, cu_q, max(new), lens, table, causal=causal, **more)
        check(got, q, k, v, cu_q, lens, table, causal, lists)
    everything = torch.full_like(mask, -1)
    check(attend(q, cache, cu_q, max(new), lens, table, causal=causal, block_mask=everything), q, k, v, cu_q, lens, table, causal)


def check_underflow(got, q, k, v, cu_q, lens, table, causal, lists, pieces=4):
    """`check`, for results that may be subnormal.  fp32 arithmetic may give 0 for any number below 2^-126: for the result of a
    piece of a tile, for what it adds to the row's sum, and for the row's result.  A share is three units of 128 keys at least, and
    a tile's start counts as two, so that 1536 keys have four pieces at most."""
    out, lse = (t.cpu() for t in got)
    ref, ref_lse, size, reach = paged.attend(q, k, v, cu_q.tolist(), lens, table, causal, lists)
    slack = q.double().abs().amax(-1) * float(k[~k.isnan()].abs().max()) * 128 ** 0.5 * 2.0 ** -18 + (reach + 1) * 2.0 ** -20
    none = ref_lse == torch.inf
    assert torch.equal(none, lse == torch.inf) and bool((out[none] == 0).all())
    assert bool(((lse.double() - ref_lse).abs() <= slack + 2.0 ** -21 * ref_lse.abs())[~none].all())
    tol = 2.0 ** -8 * ref.abs() + size * (2.0 ** -9 + 2.0 ** -11) * 1.125 + size * (2 * slack)[..., None] + _floor(v, size) + (2 * pieces + 1) * 2.0 ** -126
    err = (out.double() - ref).abs()
    assert bool((err <= tol)[~none].all()), (float((err / tol)[~none].max()), (err > tol).nonzero()[:4].tolist())


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("new", [1, 2, 3, 9])
@pytest.mark.parametrize("order", [0, 1, 2, 3, 4])
def test_values_of_every_size(dtype, new, order):
    """Values whose blocks are up to 2^227 apart, in blocks that the tokens of a tile select for themselves: a token's sums and its
    result are those of its own blocks, whatever the others' are."""
    logs = [[60, -120, 60, 60, -120, 100], [-118, 0, 100, -118, 100, -118], [100, -100, 0, -118, 60, -60], [0, 55, -80, -118, 57, 30],
            [0, -118, 55, 0, 110, 0]][order]
    logs = torch.tensor(logs * 2, dtype=torch.float64)
    length = 64 * len(logs) - 5
    cache, table, k, v = make([length], 1, 64, dtype, 101, 1.0, lambda p: torch.pow(2.0, logs[p // 64]))
    n = 150 if new <= 2 else 60
    table, lens, cu_q = table.expand(n, -1).contiguous(), [length] * n, cu([new] * n)
    q = queries([new] * n, 1, 102)
    g = torch.Generator().manual_seed(103 + order)
    lists = torch.stack([torch.randperm(len(logs), generator=g)[:3].sort().values for _ in range(new * n)]).to(torch.int32)[None]
    few = torch.arange(4 * new)
    for some in (lists, None):
        out, lse = attend(q, cache, cu_q, new, lens, table, causal=False, **({} if some is None else dict(topk_idx=some.to(DEV))))
        check_underflow((out[few], lse[few]), q[few], k, v, cu([new] * 4), lens[:4], table[:4], False, None if some is None else some[:, few])


@pytest.mark.parametrize("dtype", [E4M3, E5M2])
@pytest.mark.parametrize("new", [3, 9])
@pytest.mark.parametrize("high_first", [False, True])
def test_pieces_far_apart(dtype, new, high_first):
    """Half of the keys score 2^128 times the others and have values 2^-128 of theirs, so that both halves count alike, in pieces
    of one tile that are joined."""
    length, hk = 64 * 60, 1
    q = torch.full((new, 16, 128), 0.5, dtype=torch.bfloat16)
    high = (torch.arange(length) < length // 2) == high_first
    size = 128 * math.log(2.0) / (0.5 * 128 ** 0.5)                # what every feature of a high key is: 128 log(2) = 128 q k 128^-1/2
    k = torch.where(high, size, 0.0).double()[:, None, None].expand(length, hk, 128).to(torch.bfloat16)
    g = torch.Generator().manual_seed(105)
    v = (torch.randn(length, hk, 128, generator=g, dtype=torch.float64) * torch.where(high, 2.0 ** -108, 2.0 ** 20).double()[:, None, None]).to(torch.bfloat16)
    cache = [c.view(torch.uint8) for c in infllm_v2.b8_cache(60, 64, hk, dtype, "cpu")]
    codes = []
    for i, x in ((0, k), (1, v)):
        y, e = paged.write(x, cache[i].view(dtype), cache[2 + i], torch.arange(length))
        codes.append(y.float().to(dtype)), cache[2 + i].copy_(e)
    cache = codes + [c.view(torch.float8_e8m0fnu) for c in cache[2:]]
    kk, vv = (paged.numbers(cache[i], cache[2 + i].view(torch.uint8)) for i in (0, 1))
    table, cu_q = torch.arange(60, dtype=torch.int32)[None], cu([new])
    got = attend(q, [c.to(DEV) for c in cache], cu_q, new, [length], table, causal=False)
    _, _, size, _ = paged.attend(q, kk, vv, cu_q.tolist(), [length], table, False)
    _, _, low, _ = paged.attend(q, kk, torch.where(high.view(60, 64)[:, None, :, None], 0.0, vv), cu_q.tolist(), [length], table, False)
    assert float((low / size).mean()) > 2.0 ** -4                  # (the low half counts)
    check_underflow(got, q, kk, vv, cu_q, [length], table, False, None, pieces=11)

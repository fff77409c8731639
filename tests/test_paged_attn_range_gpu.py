"""GPU: attention over 8-bit blocks at the edges of its arithmetic: queries and keys of the largest and smallest sizes, scores that
move the references, walks of many selected blocks.  Tolerances: tests/test_paged_attn_gpu.py, and `check_exact`."""
import math

import pytest
import torch

import infllm_v2
from oracle import paged
from helpers import cu, det_tensor
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

"""GPU: attention of one new token over an 8-bit cache against the same codes in 64 bits.

Tolerance of an output: half a bf16 step of it (2^-8 of the value), and weights that are off by at most w relative to
each other, which moves the average by w times the average of |v|.  w: a weight rounded to fp16 (2^-11, and for weights
below 2^-14 of the largest 2^-25 of it), exponentials and sums in fp32 (2^-20 with room), and scores off by
ds = 130 * 2^-24 * sum |q_i k_i| * scale from 128 fp32 additions of exact products, twice (a weight and the sum).
The log-sum-exp is off by ds and by fp32 roundings of itself (2^-20 with room)."""
import pytest
import torch

import infllm_v2
from oracle.q8 import attend, dequantise, quantise, rows_of
from oracle.rotary import rotary_axes as exact_rotary
from helpers import det_tensor

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3, INT8 = torch.float8_e4m3fn, torch.int8


def _cache(slots, length, hk, dtype, seed, junk=True):
    """Codes and scales of quantised rows, NaN bytes in a copy's unused places are the callers' business."""
    k, v = det_tensor((slots, hk, length, 128), seed, 1.0), det_tensor((slots, hk, length, 128), seed + 1, 1.0)
    grow = torch.exp2(torch.randint(-6, 7, (slots, hk, length, 1), generator=torch.Generator().manual_seed(seed)).float())
    v = (v.float() * grow).to(torch.bfloat16)
    (kc, kb), (vc, vb) = quantise(k, dtype), quantise(v, dtype)
    return kc, vc, kb, vb


def _spoil(cache, lens, table, length):
    """NaN codes and scales in every place that no sequence uses."""
    used = torch.zeros(cache[2].shape[0], length, dtype=torch.bool)
    for b, n in enumerate(lens):
        slot, off = rows_of(table, None, length, b, n)
        used[slot, off] = True
    for t in cache:
        raw = t.view(torch.uint8).movedim(1, 2)          # (slots, length, hk[, 128])
        raw[~used] = 255


def _to_gpu(cache):
    kc, vc, kb, vb = cache
    return (kc.to(DEV), vc.to(DEV), kb.view(torch.float8_e8m0fnu).to(DEV), vb.view(torch.float8_e8m0fnu).to(DEV))


def _check(out, lse, q, cache, lens, table=None, batch_idx=None, topk_idx=None, scale=None):
    kc, vc, kb, vb = cache
    q3 = q.reshape(q.shape[0], -1, 128)
    want, want_lse = attend(q3, kc, vc, kb, vb, lens, table, batch_idx, topk_idx, scale)
    mag = lambda c: c.float().abs() if c.dtype != E4M3 else c.float().abs()  # noqa: E731
    avg, _ = attend(q3, kc, mag(vc), kb, vb, lens, table, batch_idx, topk_idx, scale)
    # sum |q_i k_i| scale is at most the largest over the keys in use
    top = 0.0
    for b, n in enumerate(lens):
        slot, off = rows_of(table, batch_idx, kc.shape[2], b, n)
        if n:
            k = dequantise(kc[slot, :, off], kb[slot, :, off]).abs()                     # (n, hk, 128)
            qa = q3[b].double().abs().view(kc.shape[1], -1, 128)
            top = max(top, float(torch.einsum("nhd,hgd->hgn", k, qa).max()))
    ds = 130 * 2.0 ** -24 * top * abs(128 ** -0.5 if scale is None else scale)
    tol = 2.0 ** -8 * want.abs() + avg * (2.0 ** -11 + 2.0 ** -20 + 4 * ds) + 1e-30
    got = out.cpu().double().view(want.shape)
    assert bool(((got - want).abs() <= tol).all()), float(((got - want).abs() / tol).max())
    if lse is not None:
        g, w = lse.cpu().double().view(want_lse.shape), want_lse
        assert torch.equal(torch.isinf(g), torch.isinf(w))
        fine = ~torch.isinf(w)
        assert bool(((g - w).abs()[fine] <= 2 * ds + 2.0 ** -20 * (1 + w.abs()[fine])).all())


def _table(batch, pages, slots, seed):
    return torch.randperm(slots, generator=torch.Generator().manual_seed(seed))[:batch * pages].view(batch, pages).to(torch.int32)


def _lists(lens, hk, k, seed, dup=False):
    g = torch.Generator().manual_seed(seed)
    idx = torch.full((len(lens), hk, 1, k), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        for h in range(hk):
            pick = torch.randperm((n + 63) // 64, generator=g)[:k].sort().values if n else torch.zeros(0)
            idx[b, h, 0, :len(pick)] = pick
            if dup and len(pick) > 1:
                idx[b, h, 0, 0] = pick[-1]                       # out of order and twice
    return idx


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("lens,hk,page,topk", [
    ([1], 1, 0, 0), ([0, 1, 31, 32, 33, 63, 64, 65], 2, 0, 0), ([700, 0, 130], 2, 16, 0), ([513, 100, 1000], 1, 48, 0),
    ([300], 8, 64, 0), ([2000], 1, 256, 0), ([129, 1000, 64], 2, 0, 3), ([900, 1, 77, 0], 2, 16, 4), ([4097], 2, 64, 70),
    ([90] * 40, 4, 0, 0), ([640] * 9, 16, 64, 5),
    ([20011, 300], 1, 0, 300), ([16500], 1, 16, 256), ([700] * 30, 8, 0, 9),
    ([4200] * 5 + [64, 0, 700, 4097], 17, 0, 60), ([300] * 28, 8, 16, 50)])
def test_attention(dtype, lens, hk, page, topk):
    batch, most = len(lens), max(lens)
    table = None
    if page:
        pages = max((most + page - 1) // page, 1)
        cache = _cache(batch * pages + 2, page, hk, dtype, 3)
        table = _table(batch, pages, batch * pages + 2, 4)
    else:
        cache = _cache(batch, most + 3, hk, dtype, 3)
    _spoil(cache, lens, table, cache[0].shape[2])
    q = det_tensor((batch, 1, hk * 16, 128), 7, 1.5)
    idx = _lists(lens, hk, topk, 5, dup=True) if topk else None
    args = dict(cache_seqlens=torch.tensor(lens, dtype=torch.int32, device=DEV), return_softmax_lse=True,
                block_table=None if table is None else table.to(DEV))
    dev = _to_gpu(cache)
    out, lse = infllm_v2.infllmv2_attn_with_kvcache_q8(q.to(DEV), *dev, topk_idx=None if idx is None else idx.to(DEV), **args)
    assert out.shape == q.shape and lse.shape == (batch, hk * 16, 1)
    _check(out, lse, q, cache, lens, table, topk_idx=idx)
    if topk:
        cap = cache[0].shape[2] * (table.shape[1] if page else 1)
        mask = infllm_v2.topk_to_uint64(idx.to(DEV), cap, 64)[0]
        got = infllm_v2.infllmv2_attn_with_kvcache_q8(q.to(DEV), *dev, block_mask=mask, **args)
        if batch * hk <= 148:            # (shared by the same number of CTAs, whatever the mask selects)
            assert torch.equal(got[0], out) and torch.equal(got[1], lse)
        _check(*got, q, cache, lens, table, topk_idx=idx)


@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_lists_in_any_order(dtype):
    """Lists that are not ascending, hold entries twice, past the keys, or unused ones in between."""
    cache = _cache(3, 2000, 2, dtype, 3)
    q = det_tensor((3, 1, 32, 128), 7, 1.5)
    lens = [2000, 900, 64]
    idx = torch.tensor([[5, 3, 3, 31, 0, 40, -1, 7], [14, -1, 2, 13, 14, 0, -1, 2], [0, 0, -1, 1, 9, 0, 0, -1]], dtype=torch.int32)
    idx = torch.stack([idx, idx.flip(1)], 1)[:, :, None].contiguous()
    args = dict(cache_seqlens=torch.tensor(lens, dtype=torch.int32, device=DEV), return_softmax_lse=True)
    out, lse = infllm_v2.infllmv2_attn_with_kvcache_q8(q.to(DEV), *_to_gpu(cache), topk_idx=idx.to(DEV), **args)
    _check(out, lse, q, cache, lens, topk_idx=idx)
    mask = infllm_v2.topk_to_uint64(idx.to(DEV), 2000, 64)[0]
    got = infllm_v2.infllmv2_attn_with_kvcache_q8(q.to(DEV), *_to_gpu(cache), block_mask=mask, **args)
    assert torch.equal(got[0], out) and torch.equal(got[1], lse)


@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_mask_that_leaves_nothing(dtype):
    cache = _cache(2, 200, 1, dtype, 3)
    q = det_tensor((2, 1, 16, 128), 7, 1.5)
    idx = torch.tensor([[[[-1, -1]]], [[[3, 2]]]], dtype=torch.int32)        # nothing; blocks past the 100 keys and block 2
    lens = [150, 100]
    out, lse = infllm_v2.infllmv2_attn_with_kvcache_q8(
        q.to(DEV), *_to_gpu(cache), cache_seqlens=torch.tensor(lens, dtype=torch.int32, device=DEV), topk_idx=idx.to(DEV),
        return_softmax_lse=True)
    assert not out.any() and bool(torch.isinf(lse).all())


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("page,axes,interleaved,dim", [(0, 0, True, 128), (16, 1, True, 128), (0, 3, False, 128), (64, 2, False, 96),
                                                       (0, 3, True, 64)])
def test_append_and_rotation(dtype, page, axes, interleaved, dim):
    """The new row is what fp32 arithmetic makes of it, bit for bit; the attention is that over the grown cache."""
    hk, lens, cap = 2, [0, 63, 64, 127, 192, 5], 192                          # the fifth cache is full
    batch = len(lens)
    table = None
    if page:
        pages = cap // page
        cache, table = _cache(batch * pages, page, hk, dtype, 3), _table(batch, pages, batch * pages, 4)
    else:
        cache = _cache(batch, cap, hk, dtype, 3)
    q, k, v = det_tensor((batch, 1, hk * 16, 128), 7, 1.5), det_tensor((batch, 1, hk, 128), 8, 2.0), det_tensor((batch, 1, hk, 128), 9)
    lens_t = torch.tensor(lens, dtype=torch.int32)
    more, q_rot, k_rot = {}, q.double(), k.float()
    if axes:
        i = torch.arange(dim // 2, dtype=torch.float64)
        ang = torch.arange(300, dtype=torch.float64)[:, None] * 10000.0 ** (-2 * i / dim)
        cos, sin = ang.cos().float(), ang.sin().float()
        sections = {1: (dim // 2,), 2: (dim // 2 - 5, 5), 3: (dim // 2 - 12, 4, 8)}[axes]
        pos = torch.stack([(lens_t + 40 * a).clamp(0, 299) for a in range(axes)]).to(torch.int32)
        more = dict(rotary_cos=cos.to(DEV), rotary_sin=sin.to(DEV), rotary_sections=sections, rotary_interleaved=interleaved)
        if axes > 1:
            more["rotary_positions"] = pos.to(DEV)
        q_rot = exact_rotary(q[:, 0], cos, sin, pos, sections, interleaved)[:, None]
        axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)])
        c, s = cos[pos.long()[axis].t(), torch.arange(dim // 2)], sin[pos.long()[axis].t(), torch.arange(dim // 2)]
        kk = k[:, 0].float()
        f0 = torch.arange(0, dim, 2) if interleaved else torch.arange(dim // 2)
        f1 = f0 + 1 if interleaved else f0 + dim // 2
        k_rot = kk.clone()
        k_rot[..., f0] = kk[..., f0] * c[:, None] - kk[..., f1] * s[:, None]
        k_rot[..., f1] = kk[..., f0] * s[:, None] + kk[..., f1] * c[:, None]
        k_rot = k_rot[:, None]
    dev = _to_gpu(cache)
    out, lse = infllm_v2.infllmv2_attn_with_kvcache_q8(
        q.to(DEV), *dev, k=k.to(DEV), v=v.to(DEV), cache_seqlens=lens_t.to(DEV), return_softmax_lse=True,
        block_table=None if table is None else table.to(DEV), **more)
    grown = [t.clone() for t in cache]
    for b, n in enumerate(lens):
        if n >= cap:
            continue
        slot, off = (b, n) if table is None else (int(table[b, n // page]), n % page)
        for j, x in ((0, k_rot), (1, v.float())):
            y, e = quantise(x[b, 0], dtype)
            grown[j][slot, :, off], grown[j + 2][slot, :, off] = y, e
    for got, want in zip(dev, grown):
        assert torch.equal(got.view(torch.uint8).cpu() & 0x7F if got.dtype == E4M3 else got.view(torch.uint8).cpu(),
                           want.view(torch.uint8) & 0x7F if want.dtype == E4M3 else want.view(torch.uint8))
        if got.dtype == E4M3:                                                # (a zero may have either sign)
            assert torch.equal(got.float().cpu(), want.float())
    _check(out, lse, q_rot, grown, [min(n + 1, cap) for n in lens], table)


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("page", [0, 64])
def test_append_with_block_lists(dtype, page):
    """The new row is written whether its block is selected or not, and attended only if it is."""
    hk, lens, cap = 2, [0, 63, 64, 500, 511, 130], 512
    batch = len(lens)
    table = _table(batch, cap // 64, batch * cap // 64, 4) if page else None
    cache = _cache(batch * cap // 64, 64, hk, dtype, 3) if page else _cache(batch, cap, hk, dtype, 3)
    q, k, v = det_tensor((batch, 1, hk * 16, 128), 7, 1.5), det_tensor((batch, 1, hk, 128), 8, 2.0), det_tensor((batch, 1, hk, 128), 9)
    idx = _lists([n + 1 for n in lens], hk, 3, 5)
    idx[3, 0, 0] = torch.tensor([0, 2, 7])          # 500 is in block 7
    idx[3, 1, 0] = torch.tensor([0, 2, 6])
    idx[4, 0, 0] = torch.tensor([-1, -1, -1])
    idx[5, 1, 0] = torch.tensor([2, -1, -1])        # 130 is in block 2: one key and the new one
    dev = _to_gpu(cache)
    out, lse = infllm_v2.infllmv2_attn_with_kvcache_q8(
        q.to(DEV), *dev, k=k.to(DEV), v=v.to(DEV), cache_seqlens=torch.tensor(lens, dtype=torch.int32, device=DEV),
        block_table=None if table is None else table.to(DEV), topk_idx=idx.to(DEV), return_softmax_lse=True)
    grown = [t.clone() for t in cache]
    for b, n in enumerate(lens):
        slot, off = (b, n) if table is None else (int(table[b, n // 64]), n % 64)
        for j, x in ((0, k), (1, v)):
            grown[j][slot, :, off], grown[j + 2][slot, :, off] = quantise(x[b, 0], dtype)
    for got, want in zip(dev, grown):
        if got.dtype == E4M3:
            assert torch.equal(got.float().cpu(), want.float())              # (a zero may have either sign)
        else:
            assert torch.equal(got.view(torch.uint8).cpu(), want.view(torch.uint8))
    _check(out, lse, q, grown, [n + 1 for n in lens], table, topk_idx=idx)


def test_sequences_that_share_a_slot_are_appended_before_any_attends():
    cache = _cache(2, 200, 1, E4M3, 3)
    dev = _to_gpu(cache)
    q, k = det_tensor((2, 1, 16, 128), 7), det_tensor((2, 1, 1, 128), 8)
    slot = torch.tensor([1, 1], dtype=torch.int32)
    lens = [150, 151]
    out = infllm_v2.infllmv2_attn_with_kvcache_q8(q.to(DEV), *dev, k=k.to(DEV), v=k.to(DEV), cache_batch_idx=slot.to(DEV),
                                                  cache_seqlens=torch.tensor(lens, dtype=torch.int32, device=DEV))
    grown = [t.clone() for t in cache]
    for b, n in enumerate(lens):
        for j in (0, 1):
            grown[j][1, :, n], grown[j + 2][1, :, n] = quantise(k[b, 0], E4M3)
    _check(out, None, q, grown, [151, 152], batch_idx=slot)


def test_lengths_past_the_capacity_and_below_zero():
    cache = _cache(3, 70, 1, E4M3, 3)
    q, k = det_tensor((3, 1, 16, 128), 7), det_tensor((3, 1, 1, 128), 8)
    dev = _to_gpu(cache)
    lens = torch.tensor([100, -3, 70], dtype=torch.int32, device=DEV)
    out, lse = infllm_v2.infllmv2_attn_with_kvcache_q8(q.to(DEV), *dev, k=k.to(DEV), v=k.to(DEV), cache_seqlens=lens,
                                                       return_softmax_lse=True)
    for got, was in zip(dev, cache):
        assert torch.equal(got.view(torch.uint8).cpu(), was.view(torch.uint8))   # nothing had room
    _check(out, lse, q, cache, [70, 0, 70])
    out = infllm_v2.infllmv2_attn_with_kvcache_q8(q.to(DEV), *dev)                # the whole capacity
    _check(out, None, q, cache, [70, 70, 70])
    out = infllm_v2.infllmv2_attn_with_kvcache_q8(q.to(DEV), *dev, cache_seqlens=65, softmax_scale=0.3)
    _check(out, None, q, cache, [65, 65, 65], scale=0.3)


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("page", [0, 16, 32])
@pytest.mark.parametrize("at_k,at_v", [(0, 0), (1, 0), (7, 9), (15, 15), (16, 3), (0, 16)])
def test_scales_at_every_alignment(dtype, page, at_k, at_v):
    """Scale bytes at any address, rows of any number, the first and the last row of the cache attended, NaN around them."""
    lens = [77, 33, 128] if page else [77, 33, 99]
    length = page or 99
    slots = 12 if page else 3
    cache = _cache(slots, length, 2, dtype, 3)
    q = det_tensor((3, 1, 32, 128), 7)
    table = None
    if page:                                                                     # (the first and the last page are used)
        per = 128 // page
        table = torch.arange(3 * per).flip(0).view(3, per).to(torch.int32) % slots
    kc, vc, kb, vb = _to_gpu(cache)
    args = dict(cache_seqlens=torch.tensor(lens, dtype=torch.int32, device=DEV), return_softmax_lse=True,
                block_table=None if table is None else table.to(DEV))

    def moved(scale, at):
        buf = torch.full((scale.numel() + 64,), 255, dtype=torch.uint8, device=DEV)
        buf[at:at + scale.numel()] = scale.view(torch.uint8).flatten()
        return buf[at:at + scale.numel()].view(torch.float8_e8m0fnu).view(scale.shape)

    out, lse = infllm_v2.infllmv2_attn_with_kvcache_q8(q.to(DEV), kc, vc, moved(kb, at_k), moved(vb, at_v), **args)
    _check(out, lse, q, cache, lens, table)


def test_slots_of_other_sequences():
    cache = _cache(5, 90, 2, INT8, 3)
    q = det_tensor((3, 1, 32, 128), 7)
    idx = torch.tensor([4, 0, 4], dtype=torch.int32)
    lens = [90, 33, 64]
    out, lse = infllm_v2.infllmv2_attn_with_kvcache_q8(
        q.to(DEV), *_to_gpu(cache), cache_seqlens=torch.tensor(lens, dtype=torch.int32, device=DEV),
        cache_batch_idx=idx.to(DEV), return_softmax_lse=True)
    _check(out, lse, q, cache, lens, batch_idx=idx)


@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_places_that_do_not_exist_give_nan(dtype):
    """A page or a slot that the cache does not have is never read; its sequence's result is NaN, the others' are not."""
    cache = _cache(6, 32, 1, dtype, 3)
    q = det_tensor((3, 1, 16, 128), 7)
    table = torch.tensor([[0, 1], [2, 6], [4, -1]], dtype=torch.int32)
    lens = [64, 40, 32]                                                          # the third does not reach its bad page
    out = infllm_v2.infllmv2_attn_with_kvcache_q8(q.to(DEV), *_to_gpu(cache), block_table=table.to(DEV),
                                                  cache_seqlens=torch.tensor(lens, dtype=torch.int32, device=DEV)).cpu()
    assert torch.isnan(out[1].float()).all() and not torch.isnan(out[::2].float()).any()
    _check(out[::2], None, q[::2], cache, [64, 32], table[::2])
    k = det_tensor((3, 1, 1, 128), 8)
    dev = _to_gpu(cache)
    idx = torch.tensor([5, 6, -1], dtype=torch.int32)
    out = infllm_v2.infllmv2_attn_with_kvcache_q8(
        q.to(DEV), *dev, k=k.to(DEV), v=k.to(DEV), cache_batch_idx=idx.to(DEV),
        cache_seqlens=torch.tensor([10, 10, 10], dtype=torch.int32, device=DEV)).cpu()
    assert torch.isnan(out[1:].float()).all() and not torch.isnan(out[0].float()).any()
    changed = [s for s in range(6) if not torch.equal(dev[0][s].view(torch.uint8).cpu(), cache[0][s].view(torch.uint8))]
    assert changed == [5]


@pytest.mark.parametrize("dtype", [E4M3, INT8])
def test_nan_rows(dtype):
    """A NaN scale of a key or a value that is attended shows in its head's output, one that is masked does not."""
    cache = _cache(1, 192, 2, dtype, 3)
    for t, byte, row in ((0, 2, 5), (1, 3, 70)):
        cache[t].view(torch.uint8)[0, 0, row] = 0
        cache[byte][0, 0, row] = 255
    q = det_tensor((1, 1, 32, 128), 7)
    lists = {0: [0], 1: [1], 2: [2]}
    for blocks, bad in ((lists[0], True), (lists[1], True), (lists[2], False)):
        idx = torch.tensor(blocks, dtype=torch.int32).view(1, 1, 1, 1).expand(1, 2, 1, 1).contiguous()
        out = infllm_v2.infllmv2_attn_with_kvcache_q8(q.to(DEV), *_to_gpu(cache), cache_seqlens=192, topk_idx=idx.to(DEV)).cpu().float()
        assert bool(torch.isnan(out[0, 0, :16]).all()) == bad and not torch.isnan(out[0, 0, 16:]).any()
    q[0, 0, 3, 9] = float("nan")                                                  # one query head
    idx = torch.tensor([2], dtype=torch.int32).view(1, 1, 1, 1).expand(1, 2, 1, 1).contiguous()
    out = infllm_v2.infllmv2_attn_with_kvcache_q8(q.to(DEV), *_to_gpu(cache), cache_seqlens=192, topk_idx=idx.to(DEV)).cpu().float()
    assert torch.isnan(out[0, 0, 3]).all() and not torch.isnan(out[0, 0, [0, 1, 2, 4, 15, 16, 31]]).any()


@pytest.mark.parametrize("dtype", [E4M3, INT8])
@pytest.mark.parametrize("kexp,vexp,qexp", [(0, -100, 0), (0, 110, 0), (-60, 0, 60), (40, 0, -40), (0, -125, 0), (115, 0, -115), (-112, 0, 112), (100, -60, -100),
                                            (0, 0, -120), (-126, 0, 60)])
def test_extreme_sizes(dtype, kexp, vexp, qexp):
    """Scores and values of an ordinary kind from factors far from 1."""
    k, v = det_tensor((1, 1, 100, 128), 3, 1.0), det_tensor((1, 1, 100, 128), 4, 1.0)
    q = det_tensor((1, 1, 16, 128), 5, 1.0)
    k, v, q = ((x.double() * 2.0 ** e).to(torch.bfloat16) for x, e in ((k, kexp), (v, vexp), (q, qexp)))
    v[0, 0, 7] = 0
    (kc, kb), (vc, vb) = quantise(k, dtype), quantise(v, dtype)
    cache = (kc, vc, kb, vb)
    out, lse = infllm_v2.infllmv2_attn_with_kvcache_q8(q.to(DEV), *_to_gpu(cache), cache_seqlens=100, return_softmax_lse=True)
    # a bf16 result below 2^-126 is subnormal: its step is 2^-133
    want, _ = attend(q[:, 0], *cache, [100])
    if float(want.abs().max()) < 2.0 ** -110:
        avg, _ = attend(q[:, 0], kc, vc.float().abs(), kb, vb, [100])
        assert bool(((out.cpu().double()[:, 0] - want).abs() <= 2.0 ** -8 * want.abs() + avg * 2.0 ** -9 + 2.0 ** -126).all())
    else:
        _check(out, lse, q, cache, [100])


@pytest.mark.parametrize("append", [False, True])
def test_lists_without_an_entry_attend_nothing(append):
    cache = _to_gpu(_cache(2, 70, 1, INT8, 3))
    q = det_tensor((2, 1, 16, 128), 7).to(DEV)
    new = dict(k=det_tensor((2, 1, 1, 128), 8).to(DEV), v=det_tensor((2, 1, 1, 128), 9).to(DEV)) if append else {}
    before = cache[1].clone()
    idx = torch.empty(2, 1, 1, 0, dtype=torch.int32, device=DEV)
    out, lse = infllm_v2.infllmv2_attn_with_kvcache_q8(
        q, *cache, topk_idx=idx, cache_seqlens=torch.tensor([69, 5], dtype=torch.int32, device=DEV), return_softmax_lse=True, **new)
    assert bool((out == 0).all()) and bool((lse == float("inf")).all())
    changed = (cache[1] != before).any(dim=-1).nonzero().tolist()
    assert changed == ([[0, 0, 69], [1, 0, 5]] if append else [])


@pytest.mark.parametrize("scale", [0.0, -0.2])
def test_scales_of_zero_and_below(scale):
    cache = _cache(2, 130, 1, INT8, 3)
    q = det_tensor((2, 1, 16, 128), 7, 1.5)
    lens = [130, 77]
    out, lse = infllm_v2.infllmv2_attn_with_kvcache_q8(q.to(DEV), *_to_gpu(cache), softmax_scale=scale, return_softmax_lse=True,
                                                       cache_seqlens=torch.tensor(lens, dtype=torch.int32, device=DEV))
    _check(out, lse, q, cache, lens, scale=scale)


def test_values_that_differ_by_many_orders():
    """One token with values 2^60 times the others' and next to no weight does not cost the others their bits."""
    n = 200
    k, v = det_tensor((1, 1, n, 128), 3, 1.0), det_tensor((1, 1, n, 128), 4, 1.0)
    q = det_tensor((1, 1, 16, 128), 5, 1.0)
    v[0, 0, 50] *= 2.0 ** 60
    k[0, 0, 50] = (-40.0 * q.float().sum((0, 1, 2)).sign()).to(torch.bfloat16)
    for dtype in (E4M3, INT8):
        (kc, kb), (vc, vb) = quantise(k, dtype), quantise(v, dtype)
        out, lse = infllm_v2.infllmv2_attn_with_kvcache_q8(q.to(DEV), *_to_gpu((kc, vc, kb, vb)), cache_seqlens=n,
                                                           return_softmax_lse=True)
        _check(out, lse, q, (kc, vc, kb, vb), [n])


def test_large_scores():
    """Scores of thousands: one key takes all the weight."""
    for dtype in (E4M3, INT8):
        cache = _cache(2, 300, 1, dtype, 3)
        q = det_tensor((2, 1, 16, 128), 7, 400.0)
        out, lse = infllm_v2.infllmv2_attn_with_kvcache_q8(q.to(DEV), *_to_gpu(cache), return_softmax_lse=True)
        _check(out, lse, q, cache, [300, 300])


def test_many_splits_of_a_long_sequence_and_repeatability():
    n, hk = 20011, 1
    cache = _cache(1, n, hk, E4M3, 3)
    q = det_tensor((1, 1, 16, 128), 7, 1.5)
    dev = _to_gpu(cache)
    out, lse = infllm_v2.infllmv2_attn_with_kvcache_q8(q.to(DEV), *dev, return_softmax_lse=True)
    _check(out, lse, q, cache, [n])
    for _ in range(3):
        again = infllm_v2.infllmv2_attn_with_kvcache_q8(q.to(DEV), *dev, return_softmax_lse=True)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)


def test_strided_query_and_new_rows():
    cache = _cache(3, 80, 2, E4M3, 3)
    qkv = det_tensor((3, 1, 36, 128), 7).to(DEV)
    q, k, v = qkv[:, :, :32], qkv[:, :, 32:34], qkv[:, :, 34:]
    lens = torch.tensor([5, 64, 20], dtype=torch.int32, device=DEV)
    a, b = _to_gpu(cache), _to_gpu(cache)
    x = infllm_v2.infllmv2_attn_with_kvcache_q8(q, *a, k=k, v=v, cache_seqlens=lens)
    y = infllm_v2.infllmv2_attn_with_kvcache_q8(q.contiguous(), *b, k=k.contiguous(), v=v.contiguous(), cache_seqlens=lens)
    assert torch.equal(x, y) and all(torch.equal(s.view(torch.uint8), t.view(torch.uint8)) for s, t in zip(a, b))


def test_captured_step_follows_lengths_and_two_graphs_run_at_once():
    hk, cap = 2, 500
    caches = [_cache(4, cap, hk, d, 3) for d in (E4M3, INT8)]
    dev = [_to_gpu(c) for c in caches]
    q, k, v = (det_tensor((4, 1, h, 128), s, 1.0).to(DEV) for h, s in ((32, 7), (2, 8), (2, 9)))
    lens = torch.tensor([100, 0, 64, 400], dtype=torch.int32, device=DEV)

    def step(i):
        return infllm_v2.infllmv2_attn_with_kvcache_q8(q, *dev[i], k=k, v=v, cache_seqlens=lens, return_softmax_lse=True)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(0), step(1)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for i in range(2):
        with torch.cuda.graph(graphs[i]):
            outs.append(step(i))
    for shift in (0, 37):
        lens.add_(shift)
        q.mul_(0.9)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        got = [(o.clone(), l.clone()) for o, l in outs]
        for i in range(2):
            want = step(i)
            assert torch.equal(got[i][0], want[0]) and torch.equal(got[i][1], want[1])


def test_rows_beyond_32_bit_offsets():
    slots, length, hk = 9, 131072, 16
    dev = infllm_v2.q8_cache(slots, length, hk, E4M3, DEV)
    assert dev[0].numel() > 2 ** 31
    small = _cache(1, 150, hk, E4M3, 3)
    for t, s in zip(dev, small):
        t.view(torch.uint8)[-1, :, :150] = s.view(torch.uint8)[0].to(DEV)
    q = det_tensor((1, 1, 256, 128), 7)
    out, lse = infllm_v2.infllmv2_attn_with_kvcache_q8(
        q.to(DEV), *dev, cache_seqlens=150, cache_batch_idx=torch.tensor([slots - 1], dtype=torch.int32, device=DEV),
        return_softmax_lse=True)
    _check(out, lse, q, small, [150])

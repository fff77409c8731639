"""Rows of 8-bit codes with power-of-two scales, and attention of one token over them, in 64 bits."""
import math

import torch

TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def quantise(x: torch.Tensor, dtype: torch.dtype):
    """Rows (..., 128) -> (codes in dtype, scale bytes uint8), from the definition.  float64 throughout."""
    x = x.double()
    amax = x.abs().amax(-1)
    fine = torch.isfinite(amax)
    e = torch.full(amax.shape, -127, dtype=torch.int64)
    for at in (amax > 0).logical_and(fine).nonzero().tolist():
        m, p = math.frexp(float(amax[tuple(at)]))            # amax = m 2^p, m in [0.5, 1)
        tm, tp = math.frexp(TOP[dtype])
        e[tuple(at)] = max(p - tp + (1 if m > tm else 0), -127)
    y = torch.where(fine[..., None], x, torch.zeros_like(x)) * torch.pow(torch.tensor(2.0, dtype=torch.float64), -e)[..., None]
    if dtype == torch.int8:
        codes = torch.round(y).to(torch.int8)
    else:
        # spacing of e4m3 around y: 2^(floor(log2 |y|) - 3), 2^-9 below 2^-6
        step = torch.pow(torch.tensor(2.0, dtype=torch.float64), torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
        codes = (torch.round(y / step) * step).float().to(torch.float8_e4m3fn)       # (exact: y is on the grid)
    return codes, torch.where(fine, e + 127, torch.full_like(e, 255)).to(torch.uint8)


def dequantise(codes: torch.Tensor, byte: torch.Tensor):
    """Rows in float64; NaN for byte 255."""
    s = torch.pow(torch.tensor(2.0, dtype=torch.float64), byte.double() - 127)
    s = torch.where(byte == 255, torch.full_like(s, float("nan")), s)
    return codes.float().double() * s[..., None]


def rows_of(block_table, batch_idx, length, b, n):
    """Slots and offsets of positions 0 .. n - 1 of sequence b."""
    pos = torch.arange(n)
    if block_table is not None:
        return block_table[b].long()[pos // length], pos % length
    slot = b if batch_idx is None else int(batch_idx[b])
    return torch.full((n,), slot), pos


def attend(q, k_codes, v_codes, k_byte, v_byte, lens, block_table=None, batch_idx=None, topk_idx=None, scale=None):
    """q (batch, heads_q, 128) over the first lens[b] keys, or those in the listed 64-key blocks.  Returns float64
    (out (batch, heads_q, 128), lse (batch, heads_q)); 0 and +inf without a key."""
    batch, hq, d = q.shape
    hk, length = k_codes.shape[1], k_codes.shape[2]
    group = hq // hk
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(batch, hq, d, dtype=torch.float64)
    lse = torch.full((batch, hq), float("inf"), dtype=torch.float64)
    for b in range(batch):
        slot, off = rows_of(block_table, batch_idx, length, b, int(lens[b]))
        for h in range(hk):
            s, o = slot, off
            if topk_idx is not None:
                blocks = {int(i) for i in topk_idx[b, h].flatten().tolist() if i >= 0}
                keep = torch.tensor([p // 64 in blocks for p in range(int(lens[b]))], dtype=torch.bool)
                s, o = slot[keep], off[keep]
            if s.numel() == 0:
                continue
            k = dequantise(k_codes[s, h, o], k_byte[s, h, o])
            v = dequantise(v_codes[s, h, o], v_byte[s, h, o])
            x = q[b, h * group:(h + 1) * group].double() @ k.t() * scale
            lse[b, h * group:(h + 1) * group] = torch.logsumexp(x, -1)
            out[b, h * group:(h + 1) * group] = torch.softmax(x, -1) @ v
    return out, lse

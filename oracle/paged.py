"""Page tables of a step, rows written by slot, 8-bit blocks with a power-of-two scale each, and attention over them, in
whole numbers and 64 bits, one request, block and token at a time."""
import math

import torch

TOP = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}
BLOCK = 64


def resize(seqlens, targets, table, ring, free_range, page, total):
    """Lists of ints (table: a list of rows) -> (seqlens, range, cu, positions, slots, table, ring)."""
    table, ring = [list(r) for r in table], list(ring)
    size, width = len(ring), len(table[0])
    first, count = free_range
    pages = lambda n: -(-n // page)                                # noqa: E731
    before, lens, back, cu, positions, slots, asked, taken = list(ring), [], [], [0], [], [], 0, 0
    for b, (old, new) in enumerate(zip(seqlens, targets)):
        need = max(pages(new) - pages(old), 0) if pages(new) <= width else 0
        granted = pages(new) <= width and (need == 0 or asked + need <= count)
        if granted:
            for i in range(need):
                table[b][pages(old) + i] = before[(first + asked + i) % size]
            for i in range(pages(new), pages(old)):
                back.append(table[b][i])
            taken += need
        asked += need
        for pos in range(old, max(new, old)):
            positions.append(pos)
            slots.append(table[b][pos // page] * page + pos % page if granted else -1)
        lens.append(new if granted else old)
        cu.append(cu[-1] + max(new - old, 0))
    for i, x in enumerate(back):
        ring[(first + count + i) % size] = x
    fill = max(total - len(positions), 0)
    return (lens, [(first + taken) % size, count - taken + len(back)], cu, (positions + [0] * fill)[:total],
            (slots + [-1] * fill)[:total], table, ring)


def round_to(y, dtype):
    """float64 numbers in the type's range, to the nearest of its numbers, ties to the even one."""
    bits, low = (3, -6) if dtype == torch.float8_e4m3fn else (2, -14)
    e = torch.frexp(y)[1] - 1
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64), torch.clamp(e, min=low).double() - bits)
    return torch.round(y / step) * step


def exponent(amax, dtype):
    m, e = math.frexp(amax)
    tm, te = math.frexp(TOP[dtype])
    return -127 if amax == 0 else max(e - te + (1 if m > tm else 0), -127)


def write(x, cache, scale, slots):
    """Rows x (n, heads, 128) to their slots of cache (pages, heads, page, 128) and scale (pages, heads, page / 64) uint8:
    returns (codes float64, bytes int64).  Consecutive tokens at consecutive slots of a block are one run."""
    dtype, y, byte = cache.dtype, cache.double(), scale.long()
    length, slots = cache.shape[2], slots.tolist()
    limit = cache.shape[0] * length
    i = 0
    while i < len(slots):
        n = 1
        while i + n < len(slots) and slots[i + n] == slots[i] + n and slots[i + n] % BLOCK:
            n += 1
        if 0 <= slots[i] < limit:
            page, place = divmod(slots[i], length)
            part, off = divmod(place, BLOCK)
            for h in range(x.shape[1]):
                rows = x[i:i + n, h].double()
                old = int(byte[page, h, part]) if off else 0
                if not torch.isfinite(rows).all() or old == 255:
                    new, rows = 255, torch.zeros_like(rows)
                else:
                    new = max(exponent(float(rows.abs().max()), dtype) + 127, old)
                    if off and new > old:
                        y[page, h, place - off:place] = round_to(y[page, h, place - off:place] * 2.0 ** max(old - new, -64), dtype)
                    rows = round_to(rows * 2.0 ** (127 - new), dtype)
                y[page, h, place:place + n], byte[page, h, part] = rows, new
        i += n
    return y, byte


def numbers(cache, scale):
    """The cache's values in float64, NaN in NaN blocks."""
    s = torch.pow(torch.tensor(2.0, dtype=torch.float64), scale.double() - 127)
    s = torch.where(scale == 255, torch.full_like(s, float("nan")), s)
    return cache.double() * s.repeat_interleave(BLOCK, -1)[..., None]


def attend(q, k, v, cu, lens, table=None, causal=True, lists=None, scale=None):
    """q (total, heads, 128) over k, v (pages, heads_k, page, 128) float64.  lists (heads_k, total, n) blocks or None.
    Returns float64 (out, lse, size): size is the attention over |v|, what errors of the weights are relative to; and
    the largest sum of |q_i k_i| scale that a token's row meets, for errors of the scores, (total, heads)."""
    total, hq, d = q.shape
    hk, length = k.shape[1], k.shape[2]
    group = hq // hk
    scale = d ** -0.5 if scale is None else scale
    out, size = torch.zeros(total, hq, d, dtype=torch.float64), torch.zeros(total, hq, d, dtype=torch.float64)
    lse, reach = torch.full((total, hq), math.inf, dtype=torch.float64), torch.zeros(total, hq, dtype=torch.float64)
    for b, n in enumerate(lens):
        new = int(cu[b + 1]) - int(cu[b])
        for i in range(new):
            t, seen = int(cu[b]) + i, max(n - new + i + 1, 0) if causal else n
            for h in range(hk):
                pos = torch.arange(seen)
                if lists is not None:
                    mine = {int(x) for x in lists[h, t].tolist() if x >= 0}
                    pos = pos[torch.tensor([int(p) // BLOCK in mine for p in pos], dtype=torch.bool)]
                if pos.numel() == 0:
                    continue
                page = torch.full_like(pos, b) if table is None else table[b].long()[pos // length]
                there = (page >= 0) & (page < k.shape[0])
                page = torch.where(there, page, torch.zeros_like(page))
                kk, vv = k[page, h, pos % length].clone(), v[page, h, pos % length].clone()
                kk[~there], vv[~there] = math.nan, math.nan
                g = slice(h * group, (h + 1) * group)
                x = q[t, g].double() @ kk.t() * scale
                p = torch.softmax(x, -1)
                lse[t, g], out[t, g], size[t, g] = torch.logsumexp(x, -1), p @ vv, p @ vv.abs()
                reach[t, g] = (q[t, g].double().abs() @ kk.abs().t()).amax(-1) * abs(scale)
    return out, lse, size, reach

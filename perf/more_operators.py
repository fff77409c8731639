"""Pages of a key-value cache, rows written into them, and a cache in 8 bits with a scale for each block of tokens.

Each case is one pass of a serving step's work around attention, in two forms.  The plain form is elementary
tensor arithmetic in 32 bits; with `own` the same pass goes through the package's public entry points.

kinds
    tables   request lengths before and after a step: pages are taken from a ring of free ones or given back to it,
             the block table gets the new pages, every new token its position and its slot
    rows     bf16 keys and values written into the pages of a cache by slot, (pages, page, heads, 128)
    codes    keys and values quantised into the pages of a cache in 8 bits by slot: (pages, heads, page, 128) codes,
             one power-of-two scale per 64 tokens and head, (pages, heads, page / 64)
    attend   one or more new tokens per sequence over such a cache, all of it or the selected blocks

A block whose scale has to grow because a later token is larger has its earlier codes rounded to the new scale.
"""
import math
import random

import torch

own = False

D, GROUP, BLOCK = 128, 16, 64
DEV = "cuda"
TOP = {"e4m3": 448.0, "e5m2": 57344.0}                          # largest code
TOP_EXP = {"e4m3": 8, "e5m2": 15}                               # 1.75 2^TOP_EXP = TOP
CODE = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}


# ------------------------------------------------------------------------------- the cases --

def listed():
    return [
        # one token more for each of 64 running requests: launch latency is what counts
        dict(name="tables_step_b64", kind="tables", batch=64, most=131072, page=64, tokens=64, prompts=0, done=0, short=False),
        # a busy engine's step: 256 rows, a third of them done, prompts of 131072 tokens in all admitted
        dict(name="tables_mixed_b256", kind="tables", batch=256, most=16384, page=64, tokens=131072, prompts=40, done=80, short=False),
        # short prompts and single tokens mixed, odd lengths, into pages of 64
        dict(name="rows_pages_ragged", kind="rows", lens="1,77,1300,1,2049,5003,1", hk=2, page=64, start=37),
        # half of a 131072-token prompt of a model with 8 KV heads
        dict(name="rows_65536", kind="rows", lens="65536", hk=8, page=256, start=0),
        # the tokens of one decode step appended to blocks in progress
        dict(name="codes_step_b64", kind="codes", lens=",".join(["1"] * 64), hk=2, code="e4m3", page=64, start=1000),
        # the next chunks of a few prompts, which begin inside a block
        dict(name="codes_chunks_ragged", kind="codes", lens="900,3,2500,4097,64", hk=2, code="e5m2", page=128, start=333),
        # a whole 131072-token prompt of a model with 8 KV heads
        dict(name="codes_131072", kind="codes", lens="131072", hk=8, code="e4m3", page=256, start=0),
        # a chat session on one card
        dict(name="attend_b1", kind="attend", batch=1, lo=12001, hi=12001, new_lo=1, new_hi=1, hk=2, code="e4m3", page=64,
             topk=0, causal=True),
        # an engine's decode step over uneven sequences, all of the cache attended
        dict(name="attend_pages_b16", kind="attend", batch=16, lo=1000, hi=32000, new_lo=1, new_hi=1, hk=2, code="e5m2",
             page=64, topk=0, causal=True),
        # the batch-64 decode of the benchmark over 64 selected blocks, caches of 32768 .. 131072 tokens
        dict(name="attend_b64_selected", kind="attend", batch=64, lo=32768, hi=131072, new_lo=1, new_hi=1, hk=2, code="e4m3",
             page=256, topk=64, causal=True),
        # drafted tokens of 12 requests checked at once, 128 query heads
        dict(name="attend_drafts_b12", kind="attend", batch=12, lo=900, hi=30000, new_lo=2, new_hi=5, hk=8, code="e4m3",
             page=128, topk=0, causal=True),
        # a prompt's next chunk over what the cache holds of it
        dict(name="attend_chunk_4096_of_32768", kind="attend", batch=1, lo=32768, hi=32768, new_lo=4096, new_hi=4096, hk=2,
             code="e4m3", page=64, topk=0, causal=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _ragged(rng, total, most):
    """`total` tokens in 1 .. most sequences of uneven length."""
    n = rng.randint(1, min(most, total))
    cuts = sorted(rng.sample(range(1, total), n - 1)) if n > 1 else []
    return ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [total]))


def draw(rng):
    kind = rng.choice(["tables", "rows", "codes", "attend", "attend", "attend"])
    page = rng.choice([64, 64, 128, 192, 256])
    if kind == "tables":
        batch = _log_int(rng, 1, 512)
        prompts = rng.randint(0, max(1, batch // 3))
        return dict(kind=kind, batch=batch, most=_log_int(rng, 300, 131072 if batch < 128 else 16384),
                    page=rng.choice([16, 64, 80, 128, 256]), tokens=_log_int(rng, 2, 131072), prompts=prompts,
                    done=rng.randint(0, max(0, batch - prompts) // 2), short=rng.random() < 0.25)
    hk = rng.choice([1, 2, 2, 4, 8])
    code = rng.choice(["e4m3", "e5m2"])
    if kind in ("rows", "codes"):
        most = (131072 if kind == "codes" else 65536) * 8 // hk
        case = dict(kind=kind, lens=_ragged(rng, _log_int(rng, 2, min(most, 131072)), rng.choice([12, 100])), hk=hk, page=page,
                    start=rng.choice([0, rng.randint(1, 500)]))
        return case if kind == "rows" else dict(case, code=code)
    new = rng.choice([1, 1, rng.randint(2, 8), _log_int(rng, 9, 4096)])
    causal = rng.random() < 0.85
    batch, hi = _log_int(rng, 1, 64), _log_int(rng, 2, 131072)
    if new > 8:
        batch = min(batch, 6)
    while batch * hi * hk > 12 * 30000 * 8:
        hi = hi // 2
    hi = max(hi, new, 1)
    while batch * new * hi * hk > 4096 * 28000 * 2 and batch > 1:
        batch = batch // 2
    while batch * new * hi * hk > 4096 * 28000 * 2 and hk > 1:
        hk = hk // 2
    return dict(kind=kind, batch=batch, lo=max(new, int(hi * rng.uniform(0.05, 1.0))), hi=hi, new_lo=rng.randint(1, new) if new > 1 else 1,
                new_hi=new, hk=hk, code=code, page=rng.choice([0, page]), topk=rng.choice([0, 0, 16, 64]) if causal else 0,
                causal=causal)


# --------------------------------------------------------------------------------- inputs --

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _rand(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g, dtype=torch.bfloat16)


def _keys(g, n, hk):
    """(n, hk, 128) keys that drift from segment to segment of 192 tokens, with some large features."""
    seg = _rand(g, n // 192 + 1, hk, D)
    k = _rand(g, n, hk, D).mul_(0.8).add_(seg[torch.arange(n, device=DEV) // 192], alpha=0.6)
    k[..., ::37] *= 4.0
    return k


def _values(g, n, hk):
    """(n, hk, 128) values whose tokens differ in size."""
    return _rand(g, n, hk, D) * torch.exp(0.7 * _rand(g, n, hk, 1))


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _cu(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return _ints(out)


def _lens(case):
    return [int(x) for x in case["lens"].split(",")]


def _pages(n, page):
    return (n + page - 1) // page


def _prepare_tables(case, seed):
    """Lengths of all requests before and after, a table of their pages, and the ring of the pages that nobody has."""
    rng = random.Random(int(seed))
    b, most, page, prompts, done = case["batch"], case["most"], case["page"], case["prompts"], case["done"]
    order = rng.sample(range(b), b)
    old = [rng.randint(most // 4, most) for _ in range(b)]
    new = [n + 1 for n in old]
    for i in order[:done]:
        new[i] = 0                                                 # this request has ended
    left = case["tokens"]
    for j, i in enumerate(order[done:done + prompts]):
        old[i] = 0 if j % 3 else rng.randint(0, most)              # a whole prompt, or a prompt's next chunk
        n = left if j == prompts - 1 else max(1, left * 2 // (prompts - j + 1))
        new[i], left = old[i] + n, max(1, left - n)
    width = _pages(most + case["tokens"], page)
    used = sum(_pages(n, page) for n in old)
    need = sum(max(0, _pages(m, page) - _pages(n, page)) for n, m in zip(old, new))
    free = need // 2 if case["short"] else need + 17
    g = _gen(seed)
    size = b * (_pages(most, page) + 2) + _pages(case["tokens"], page) + 17     # pages of the whole cache
    ids = torch.randperm(size, device=DEV, generator=g).to(torch.int32)
    have = _ints([_pages(n, page) for n in old])[:, None] > torch.arange(width, device=DEV)
    table = torch.full((b, width), -1, dtype=torch.int32, device=DEV)
    table[have] = ids[:used]
    first = rng.randint(0, size - 1)
    ring = torch.full((size,), -1, dtype=torch.int32, device=DEV)
    ring[(first + torch.arange(free, device=DEV)) % size] = ids[used:used + free]
    return dict(case=case, old=_ints(old), new=_ints(new), table=table, ring=ring, range=_ints([first, free]),
                total=sum(max(0, m - n) for n, m in zip(old, new)))


def _cache_of(case, lens, g):
    """Zeroed pages for sequences of `lens` tokens, and their table (None: a sequence's rows are one page)."""
    hk, page = case["hk"], case["page"]
    most = max(lens)
    if page:
        per = _pages(most, page)
        slots, length = len(lens) * per + 3, page
        table = torch.randperm(slots, device=DEV, generator=g)[:len(lens) * per].view(len(lens), per).to(torch.int32)
    else:
        slots, length, table = len(lens), _pages(most, BLOCK) * BLOCK, None
    s = dict(table=table)
    for name in "kv":
        if case["kind"] == "rows":
            s[name + "_cache"] = torch.zeros(slots, length, hk, D, dtype=torch.bfloat16, device=DEV)
            continue
        s[name + "_cache"] = torch.zeros(slots, hk, length, D, dtype=torch.uint8, device=DEV).view(CODE[case["code"]])
        s[name + "_scale"] = torch.zeros(slots, hk, length // BLOCK, dtype=torch.uint8, device=DEV).view(torch.float8_e8m0fnu)
    return s


def _slots(s, b, pos):
    """Slots (n,) of tokens at positions `pos` of sequence b: page * page size + place in it."""
    length = s["length"]
    page = torch.full_like(pos, b) if s["table"] is None else s["table"][b, pos // length].long()
    return page * length + pos % length


def _fill(s, case, lens, g):
    """Puts keys and values of every sequence into the empty cache, a sequence at a time."""
    for b, n in enumerate(lens):
        if n:
            slots = _slots(s, b, torch.arange(n, device=DEV))
            for name, x in (("k", _keys(g, n, case["hk"])), ("v", _values(g, n, case["hk"]))):
                if case["kind"] == "rows":
                    s[name + "_cache"].view(-1, case["hk"], D)[slots] = x
                else:
                    _store(s, name, x, slots, case["code"])


def prepare(case, seed):
    if case["kind"] == "tables":
        return _prepare_tables(case, seed)
    g, hk = _gen(seed), case["hk"]
    if case["kind"] in ("rows", "codes"):
        lens, start = _lens(case), case["start"]
        before = [start - start // 2 * (b % 2) - b % 3 * (start > 2) for b in range(len(lens))]
        s = dict(case=case, length=case["page"], **_cache_of(case, [n + m for n, m in zip(lens, before)], g))
        _fill(s, case, before, g)
        s["slots"] = torch.cat([_slots(s, b, torch.arange(m, m + n, device=DEV)) for b, (n, m) in enumerate(zip(lens, before))])
        qkv = _rand(g, sum(lens), (GROUP + 2) * hk, D)             # keys and values cut out of one projection
        qkv[:, GROUP * hk:(GROUP + 1) * hk] = _keys(g, sum(lens), hk)
        qkv[:, (GROUP + 1) * hk:] = _values(g, sum(lens), hk) * 1.5
        s["k"], s["v"] = qkv[:, GROUP * hk:(GROUP + 1) * hk], qkv[:, (GROUP + 1) * hk:]
        return s
    rng = random.Random(int(seed))
    b, lo, hi = case["batch"], case["lo"], case["hi"]
    lens = [rng.randint(lo, hi) for _ in range(b)]
    lens[0] = hi                                                   # (the work of a case does not hang on the seed)
    same = random.Random(b * 131 + hi)
    new = [same.randint(case["new_lo"], case["new_hi"]) for _ in lens]
    new[0] = case["new_hi"]
    s = dict(case=case, **_cache_of(case, lens, g))
    s["length"] = s["k_cache"].shape[2]
    _fill(s, case, lens, g)
    s.update(lens=_ints(lens), cu=_cu(new), most=max(new), total=sum(new), host_lens=lens, host_new=new)
    s["q"] = 1.5 * _rand(g, sum(new), GROUP * hk, D)
    s["idx"] = _lists(g, s, hk, case["topk"]) if case["topk"] else None
    return s


def _lists(g, s, hk, topk):
    """(hk, tokens, topk) int32: block 0, the newest blocks and others that neighbouring tokens mostly agree on, ascending,
    -1 in the unused tail."""
    n = _pages(max(s["host_lens"]), BLOCK)
    last = torch.cat([torch.arange(m - t, m, device=DEV) for m, t in zip(s["host_lens"], s["host_new"])]) // BLOCK
    at, shared = torch.arange(n, device=DEV), torch.arange(s["total"], device=DEV) // 32
    out = torch.empty(hk, s["total"], topk, dtype=torch.int32, device=DEV)
    for h in range(hk):
        score = torch.rand(s["total"] // 32 + 1, n, device=DEV, generator=g)[shared]
        score = score + 0.1 * torch.rand(s["total"], n, device=DEV, generator=g)
        score = torch.where((at == 0) | (at > last[:, None] - topk // 2), torch.full_like(score, 2.0), score)
        val, idx = score.masked_fill(at > last[:, None], -1.0).topk(min(topk, n), dim=-1)
        idx = torch.where(val >= 0, idx, torch.full_like(idx, n)).sort(-1).values
        idx = torch.where(idx == n, torch.full_like(idx, -1), idx)
        out[h] = torch.cat([idx, idx.new_full((s["total"], topk - idx.shape[-1]), -1)], -1).to(torch.int32)
    return out


# ------------------------------------------------------------------------- the plain form --

def _resize(s):
    """A step of the tables, whole numbers throughout."""
    page, table, ring = s["case"]["page"], s["table"], s["ring"]
    b, width = table.shape
    old, new = s["old"].long(), s["new"].long()
    had, want = _pages(old, page), _pages(new, page)
    need = torch.where(want <= width, want - had, torch.zeros_like(had)).clamp(min=0)
    upto = need.cumsum(0)
    first, free = s["range"].long()
    granted = (want <= width) & ((need == 0) | (upto <= free))
    kept = torch.where(granted, new, old)
    taken = torch.where(granted, need, torch.zeros_like(need))
    back = (had - _pages(kept, page)).clamp(min=0)
    i = torch.arange(width, device=DEV)
    # pages that end with this step go behind the last free one, request by request
    gone = (i >= (had - back)[:, None]) & (i < had[:, None])
    at = (first + free + (back.cumsum(0) - back)[:, None] + i - (had - back)[:, None]) % ring.numel()
    ring[at[gone]] = table[gone]
    # pages that begin with it come from the front
    fresh = (i >= had[:, None]) & (i < (had + taken)[:, None])
    at = (first + (upto - need)[:, None] + i - had[:, None]) % ring.numel()
    table[fresh] = ring[at[fresh]]
    grow = (new - old).clamp(min=0)
    cu = torch.cat([grow.new_zeros(1), grow.cumsum(0)])
    t = torch.arange(s["total"], device=DEV)
    who = torch.searchsorted(cu, t, right=True) - 1
    pos = old[who] + t - cu[who]
    ok = granted[who]
    slot = table[who, torch.where(ok, pos // page, torch.zeros_like(pos))].long() * page + pos % page
    left = torch.stack([(first + taken.sum()) % ring.numel(), free - taken.sum() + back.sum()])
    return dict(lens=kept.int(), range=left.int(), cu=cu.int(), positions=pos.int(),
                slots=torch.where(ok, slot, torch.full_like(slot, -1)), table=table, ring=ring)


def _exponent(amax, code):
    """The smallest e >= -127 with amax 2^-e <= the largest code."""
    m, e = torch.frexp(amax)                                       # amax = m 2^e, m in [0.5, 1)
    e = e - 1 - TOP_EXP[code] + (m > 0.875)
    return torch.where(amax > 0, e, torch.full_like(e, -127)).clamp_(min=-127)


def _store(s, name, x, slots, code):
    """Quantises rows (n, hk, 128) at slots that are runs of neighbours, a run within a block or blocks in one piece."""
    cache, scale = s[name + "_cache"].view(torch.uint8), s[name + "_scale"].view(torch.uint8)
    hk, length = cache.shape[1], cache.shape[2]
    x = x.float()
    per = length // BLOCK
    block = slots // BLOCK                                         # (page, block of the page)
    ids, inv = torch.unique_consecutive(block, return_inverse=True)
    n = ids.numel()
    amax = x.new_zeros(n, hk).index_reduce_(0, inv, x.abs().amax(-1), "amax", include_self=True)
    off = slots.new_full((n,), BLOCK).index_reduce_(0, inv, slots % BLOCK, "amin", include_self=True)
    page, part = ids // per, ids % per
    e = _exponent(amax, code)
    before = scale[page, :, part].int() - 127                      # (n, hk)
    e = torch.where(off[:, None] > 0, torch.maximum(e, before), e)
    rows = (page[:, None] * hk + torch.arange(hk, device=DEV)) * length + part[:, None] * BLOCK        # (n, hk)
    codes = cache.view(-1, D)
    grown = ((off[:, None] > 0) & (e > before)).nonzero()          # earlier rows that need the new scale
    if grown.numel():
        i, h = grown.unbind(1)
        at = rows[i, h][:, None] + torch.arange(BLOCK, device=DEV)
        y = codes[at].view(CODE[code]).float() * torch.exp2((before - e)[i, h].clamp(min=-64).float())[:, None, None]
        mine = torch.arange(BLOCK, device=DEV) < off[i, None]
        codes[at[mine]] = y[mine].to(CODE[code]).view(torch.uint8)
    scale[page, :, part] = (e + 127).to(torch.uint8)
    y = torch.ldexp(x, -e[inv][:, :, None]).to(CODE[code]).view(torch.uint8)
    codes[rows[inv] + (slots % BLOCK)[:, None]] = y


def _load(s, name, rows):
    """Rows of the flattened cache as 32-bit numbers."""
    code, scale = s[name + "_cache"], s[name + "_scale"].view(torch.uint8)
    e = scale.view(-1)[rows // BLOCK].int()
    return code.view(torch.uint8).view(-1, D)[rows].view(code.dtype).float() * torch.ldexp(torch.ones_like(e, dtype=torch.float32), e - 127)[..., None]


def _softmax_av(x, v):
    """Output and log-sum-exp of scores (..., keys) with -inf in masked places; rows that see nothing give 0 and +inf."""
    m = x.amax(-1, keepdim=True)
    none = m == -math.inf
    p = torch.exp(x - torch.where(none, torch.zeros_like(m), m))
    l = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(none, torch.ones_like(l), l)
    return out, torch.where(none, torch.full_like(m, math.inf), m + l.log()).squeeze(-1)


def _rows(s, b, h, pos):
    length, hk = s["length"], s["k_cache"].shape[1]
    page = b + torch.zeros_like(pos) if s["table"] is None else s["table"][b, pos // length].long()
    return (page * hk + h) * length + pos % length


def _attend_steps(s):
    """A few tokens per sequence, all sequences and heads at once."""
    case, most, b = s["case"], s["most"], s["case"]["batch"]
    hk, cu, lens = case["hk"], s["cu"].long(), s["lens"].long()
    t = torch.arange(most, device=DEV)
    news = cu[1:] - cu[:-1]
    real = t < news[:, None]                                       # (b, most)
    tok = torch.where(real, cu[:-1, None] + t, torch.zeros_like(cu[:-1, None]))
    q = s["q"].float()[tok].view(b, most, hk, GROUP, D).permute(0, 2, 1, 3, 4)          # (b, hk, most, 16, 128)
    limit = lens[:, None] - news[:, None] + 1 + t if case["causal"] else lens[:, None].expand(-1, most)
    bb, hh = torch.arange(b, device=DEV)[:, None, None, None], torch.arange(hk, device=DEV)[None, :, None, None]
    if s["idx"] is None:
        pos = torch.arange(max(s["host_lens"]), device=DEV).expand(b, 1, 1, -1)
        seen = pos < limit[:, None, :, None]
    else:
        idx = s["idx"][:, tok].permute(1, 0, 2, 3).long()          # (b, hk, most, topk)
        pos = (idx[..., None] * BLOCK + torch.arange(BLOCK, device=DEV)).flatten(3)
        seen = (idx >= 0)[..., None].expand(-1, -1, -1, -1, BLOCK).flatten(3) & (pos < limit[:, None, :, None])
        pos = torch.where(seen, pos, torch.zeros_like(pos))
    here = pos < lens[:, None, None, None]
    rows = _rows(s, bb, hh, torch.where(here, pos, torch.zeros_like(pos)))              # (b, hk, 1 or most, keys)
    x = torch.matmul(q, _load(s, "k", rows).transpose(-1, -2)) * D ** -0.5
    x = x.masked_fill(~seen[:, :, :, None, :], -math.inf)
    out, lse = _softmax_av(x, _load(s, "v", rows))
    pick = real.nonzero()                                          # (tokens, 2), in order
    out = out.permute(0, 2, 1, 3, 4)[pick[:, 0], pick[:, 1]].reshape(-1, hk * GROUP, D)
    lse = lse.permute(0, 2, 1, 3)[pick[:, 0], pick[:, 1]].reshape(-1, hk * GROUP)
    return dict(out=out.to(torch.bfloat16), lse=lse)


def _attend_chunks(s):
    """Sequence by sequence and head by head, 256 tokens at a time."""
    case = s["case"]
    hk, out, lse, at = case["hk"], torch.empty_like(s["q"]), s["q"].new_empty(s["total"], case["hk"] * GROUP, dtype=torch.float32), 0
    for b, (n, t) in enumerate(zip(s["host_lens"], s["host_new"])):
        pos = torch.arange(n, device=DEV)
        for h in range(hk):
            rows, heads = _rows(s, b, h, pos), slice(h * GROUP, (h + 1) * GROUP)
            k, v = _load(s, "k", rows), _load(s, "v", rows)
            for t0 in range(0, t, 256):
                t1 = min(t, t0 + 256)
                part = slice(at + t0, at + t1)
                limit = n - t + 1 + torch.arange(t0, t1, device=DEV) if case["causal"] else torch.full((t1 - t0,), n, device=DEV)
                seen = pos < limit[:, None]
                if s["idx"] is not None:
                    keep = torch.zeros(t1 - t0, _pages(n, BLOCK) + 1, dtype=torch.bool, device=DEV)
                    idx = s["idx"][h, part].long()
                    keep.scatter_(1, torch.where(idx >= 0, idx, torch.full_like(idx, keep.shape[1] - 1)), True)
                    seen = seen & keep[:, pos // BLOCK]
                x = torch.matmul(s["q"][part, heads].float(), k.t()) * D ** -0.5
                y, z = _softmax_av(x.masked_fill_(~seen[:, None], -math.inf), v)
                out[part, heads], lse[part, heads] = y.to(torch.bfloat16), z
        at += t
    return dict(out=out, lse=lse)


def _caches(s):
    if s["case"]["kind"] == "rows":
        return dict(k_cache=s["k_cache"], v_cache=s["v_cache"])
    return dict(k_cache=s["k_cache"], v_cache=s["v_cache"], k_scale=s["k_scale"].view(torch.uint8), v_scale=s["v_scale"].view(torch.uint8))


def _run_plain(s):
    case = s["case"]
    if case["kind"] == "tables":
        return _resize(s)
    if case["kind"] == "rows":
        for name in "kv":
            s[name + "_cache"].view(-1, case["hk"], D)[s["slots"]] = s[name]
        return _caches(s)
    if case["kind"] == "codes":
        for name in "kv":
            _store(s, name, s[name], s["slots"], case["code"])
        return _caches(s)
    return _attend_steps(s) if s["most"] <= 8 else _attend_chunks(s)


# --------------------------------------------------------------------- the package's calls --

def _run_own(s):
    import infllm_v2 as iv
    case = s["case"]
    if case["kind"] == "tables":
        lens, left, cu, positions, slots = iv.pages_resize(s["old"], s["new"], s["table"], s["ring"], s["range"], case["page"], s["total"])
        return dict(lens=lens, range=left, cu=cu, positions=positions, slots=slots, table=s["table"], ring=s["ring"])
    if case["kind"] == "rows":
        iv.cache_write(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"])
        return _caches(s)
    cache = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    if case["kind"] == "codes":
        iv.cache_write_b8(s["k"], s["v"], *cache, s["slots"])
        return _caches(s)
    out, lse = iv.infllmv2_attn_paged_b8(s["q"], *cache, s["cu"], s["most"], s["lens"], block_table=s["table"],
                                         causal=case["causal"], topk_idx=s["idx"], return_softmax_lse=True)
    return dict(out=out, lse=lse)


def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return _run_plain(s)


# ---------------------------------------------------------------------------------- work --

def work(case):
    kind = case["kind"]
    if kind == "tables":
        # lengths in and out; a new page's number read and written; a position and a slot per token
        n = case["tokens"] + case["batch"] - case["done"] if case["prompts"] else case["batch"] - case["done"]
        back = case["done"] * case["most"] * 5 / 8 / case["page"]
        return dict(bytes=16 * case["batch"] + 12 * n + 8 * (n / case["page"] + back), flops=0)
    hk = case["hk"]
    if kind in ("rows", "codes"):
        rows = 2 * sum(_lens(case)) * hk
        return dict(bytes=rows * 2 * D + 4 * rows // hk + (rows * 2 * D if kind == "rows" else rows * (D + 1 / BLOCK)),
                    flops=0 if kind == "rows" else 3 * rows * D)
    b, new = case["batch"], (case["new_lo"] + case["new_hi"]) / 2
    keys = (case["lo"] + case["hi"]) / 2
    seen = keys - (new - 1) / 2 if case["causal"] else keys        # keys that a token sees
    if case["topk"]:
        seen = min(seen, BLOCK * case["topk"])
        keys = seen if case["new_hi"] == 1 else keys
    return dict(bytes=2 * b * hk * keys * (D + 1 / BLOCK) + b * new * hk * GROUP * (4 * D + 4),
                flops=4 * b * new * seen * hk * GROUP * D)


# ------------------------------------------------------------------------ 64-bit answers --

def _exact_round(y, code):
    """Numbers rounded to the nearest code, ties to the even one, from the definition of the type."""
    bits, low = (3, -6) if code == "e4m3" else (2, -14)
    _, e = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), torch.clamp(e - 1, min=low) - bits)
    return torch.round(y / step) * step


def _exact_codes(s, name):
    """Codes of the cache after the write, as numbers, block by block over the runs that the call's slots are."""
    code = s["case"]["code"]
    y = s[name + "_cache"].double()
    e = s[name + "_scale"].view(torch.uint8).double() - 127
    hk, length = y.shape[1], y.shape[2]
    x, slots = s[name].double(), s["slots"].tolist()
    runs, at = [], 0
    for i in range(1, len(slots) + 1):
        if i == len(slots) or slots[i] // BLOCK != slots[at] // BLOCK:
            runs.append((at, i))
            at = i
    amax = x.abs().amax(-1).cpu()
    for a, z in runs:
        page, place = divmod(slots[a], length)
        part, off = divmod(place, BLOCK)
        top = amax[a:z].amax(0)                                    # (hk)
        want = torch.where(top > 0, torch.ceil(torch.log2(top / TOP[code])), torch.full_like(top, -127.0))
        want = torch.where(top > TOP[code] * torch.exp2(want), want + 1, want)      # (the logarithm is rounded)
        want = torch.where(top <= TOP[code] * torch.exp2(want - 1), want - 1, want).clamp(min=-127)
        want = want.to(DEV)
        if off:
            now = torch.maximum(want, e[page, :, part])
            grow = torch.exp2(e[page, :, part] - now)[:, None, None]
            old = y[page, :, place - off:place]
            y[page, :, place - off:place] = torch.where(grow < 1, _exact_round(old * grow, code), old)
            want = now
        e[page, :, part] = want
        y[page, :, place:place + z - a] = _exact_round(x[a:z].transpose(0, 1) * torch.exp2(-want)[:, None, None], code)
    return y


def _exact_attend(s):
    case, outs, lses, at = s["case"], [], [], 0
    length = s["length"]

    def numbers(name, page, h, off):
        return (s[name + "_cache"].view(torch.uint8)[page, h, off].view(s[name + "_cache"].dtype).double()
                * torch.exp2(s[name + "_scale"].view(torch.uint8)[page, h, off // BLOCK].double() - 127)[:, None])

    for b, (n, t) in enumerate(zip(s["host_lens"], s["host_new"])):
        pos = torch.arange(n, device=DEV)
        page = torch.full_like(pos, b) if s["table"] is None else s["table"][b].long()[pos // length]
        heads_o, heads_l = [], []
        for h in range(case["hk"]):
            k, v = numbers("k", page, h, pos % length), numbers("v", page, h, pos % length)
            parts_o, parts_l = [], []
            for i in range(t) if t <= 8 or s["idx"] is not None else range(0, t, 512):
                j = i + 1 if t <= 8 or s["idx"] is not None else min(t, i + 512)
                q = s["q"][at + i:at + j, h * GROUP:(h + 1) * GROUP].double()
                last = torch.arange(n - t + i, n - t + j, device=DEV) if case["causal"] else torch.full((j - i,), n, device=DEV)
                use = pos
                if s["idx"] is not None:
                    mine = s["idx"][h, at + i].long()
                    use = (mine[mine >= 0][:, None] * BLOCK + torch.arange(BLOCK, device=DEV)).flatten()
                    use = use[use <= last[0]]
                x = torch.einsum("tgd,kd->tgk", q, k[use]) / math.sqrt(D)
                x = torch.where(use <= last[:, None, None], x, torch.full_like(x, -math.inf))
                parts_l.append(torch.logsumexp(x, -1))
                parts_o.append(torch.softmax(x, -1) @ v[use])
            heads_o.append(torch.cat(parts_o))
            heads_l.append(torch.cat(parts_l))
        outs.append(torch.cat(heads_o, 1))
        lses.append(torch.cat(heads_l, 1))
        at += t
    return dict(out=torch.cat(outs), lse=torch.cat(lses))


def _exact_cost(case):
    if case["kind"] == "rows":
        return 0
    if case["kind"] == "codes":
        return sum(_lens(case)) / 8000                             # (the runs are walked one by one)
    per = case["new_hi"] * (1.0 if case["topk"] else 1 / 512 if case["new_hi"] > 8 else 1.0)
    return (case["batch"] * case["hk"] * per * 4e-4 + case["batch"] * case["hk"] * case["new_hi"] * case["hi"] * 8192 / 2e13
            + case["batch"] * case["hk"] * case["hi"] / 1e8)


def exact(case, seed):
    if case["kind"] == "tables":
        return None                                                # whole numbers
    if _exact_cost(case) > 18:
        return None
    s = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "rows":
            for name in "kv":
                s[name + "_cache"].view(-1, case["hk"] * D).index_copy_(0, s["slots"], s[name].reshape(-1, case["hk"] * D))
            return {name + "_cache": s[name + "_cache"].double() for name in "kv"}
        if case["kind"] == "codes":
            return dict(k_cache=_exact_codes(s, "k"), v_cache=_exact_codes(s, "v"), k_scale=None, v_scale=None)
        return _exact_attend(s)

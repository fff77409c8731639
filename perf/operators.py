"""Rotary positions over several axes, and a key-value cache in 8 bits: written, read back, attended.

Each case is one pass of work around attention, in two forms.  The plain form is elementary tensor
arithmetic in 32 bits; with `own` the same pass goes through the package's public entry points.

kinds
    rotary   positions (one axis, or time / height / width) rotated into queries and keys
    train    the same, forward and backward
    write    keys and values of packed sequences quantised into a cache (slots or pages)
    read     rows of such a cache read back as packed bf16 tensors
    attend   one new token per sequence over the cache, optionally rotated and appended first
    serve    a prompt from rotation over the cache write to the attention of its next token

A cache is kept head by head: codes (slots, heads_k, length, 128) and a power-of-two scale per row,
(slots, heads_k, length), where a slot is a sequence or a page of a block table.
"""
import math

import torch

own = False

D, GROUP, BLOCK = 128, 16, 64
DEV = "cuda"
TOP = {"e4m3": 1.75 * 2.0 ** 8, "int8": 127.0}                 # largest code
CODE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


# ------------------------------------------------------------------------------- the cases --

def listed():
    return [
        # positions of one decode step of 64 sequences: launch latency is what counts
        dict(name="rotary_step_b64", kind="rotary", tokens=64, hk=2, dim=128, axes=1, halves=True, fused=True),
        # a 32768-token prompt with images, three axes, queries and keys cut out of one projection
        dict(name="rotary_prompt_32768", kind="rotary", tokens=32768, hk=2, dim=128, axes=3, halves=True, fused=True),
        # a training step over an odd number of tokens, partial rotation of neighbouring pairs
        dict(name="rotary_train_8191", kind="train", tokens=8191, hk=2, dim=96, axes=3, halves=False, fused=False),
        # a batch of short prompts of odd lengths into pages of 64 tokens
        dict(name="write_pages_ragged", kind="write", lens="1,77,1300,2049,5003", hk=2, code="e4m3", page=64, start=37),
        # a whole 131072-token prompt of a model with 8 KV heads into its slot
        dict(name="write_131072", kind="write", lens="131072", hk=8, code="int8", page=0, start=0),
        # a few sequences read back from small pages before their next chunk
        dict(name="read_pages_ragged", kind="read", lens="900,3,2500,4097", hk=2, code="int8", page=16, start=5),
        # a long prompt read back
        dict(name="read_65536", kind="read", lens="65536", hk=8, code="e4m3", page=0, start=0),
        # a chat session on one card: one sequence, rotated and appended
        dict(name="attend_b1_append", kind="attend", batch=1, lo=12001, hi=12001, hk=2, code="e4m3", page=0, topk=0, axes=1,
             append=True),
        # an engine with pages of 16 tokens and uneven sequences, all of the cache attended
        dict(name="attend_pages_b16", kind="attend", batch=16, lo=1000, hi=32000, hk=2, code="e4m3", page=16, topk=0, axes=0,
             append=False),
        # a server batch with 128 query heads, images among the prompts, 8-bit integers
        dict(name="attend_b12_append", kind="attend", batch=12, lo=900, hi=30000, hk=8, code="int8", page=0, topk=0, axes=3,
             append=True),
        # the batch-64 decode of the benchmark over 64 selected blocks, caches of 32768 .. 131072 tokens
        dict(name="attend_b64_selected", kind="attend", batch=64, lo=32768, hi=131072, hk=2, code="e4m3", page=0, topk=64,
             axes=0, append=False),
        # three prompts with images: rotate, write, attend the next token
        dict(name="serve_prompts", kind="serve", lens="700,45,2100", hk=2, code="e4m3", page=64, axes=3),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _ragged(rng, total, most):
    """`total` tokens in 1 .. most sequences of uneven length."""
    n = rng.randint(1, min(most, total))
    cuts = sorted(rng.sample(range(1, total), n - 1)) if n > 1 else []
    return ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [total]))


def draw(rng):
    kind = rng.choice(["rotary", "train", "write", "read", "attend", "attend", "serve"])
    hk = rng.choice([1, 2, 2, 4, 8])
    code = rng.choice(["e4m3", "int8"])
    if kind in ("rotary", "train"):
        most = 32768 * 2 // hk if kind == "rotary" else 16384 // hk
        return dict(kind=kind, tokens=_log_int(rng, 1, min(most, 32768)), hk=hk, dim=rng.choice([64, 96, 128, 128]),
                    axes=rng.choice([1, 2, 3, 3]), halves=rng.random() < 0.5, fused=rng.random() < 0.5)
    if kind in ("write", "read"):
        most = (131072 if kind == "write" else 65536) * 8 // hk
        return dict(kind=kind, lens=_ragged(rng, _log_int(rng, 2, min(most, 131072)), 12), hk=hk, code=code,
                    page=rng.choice([0, 16, 64, 80, 256]), start=rng.choice([0, rng.randint(1, 500)]))
    if kind == "serve":
        return dict(kind=kind, lens=_ragged(rng, _log_int(rng, 2, 8000), 6), hk=hk, code=code, page=rng.choice([16, 64, 256]),
                    axes=rng.choice([1, 3]))
    batch, hi = _log_int(rng, 1, 64), _log_int(rng, 2, 131072)
    while batch * hi * hk > 12 * 30000 * 8:
        hi = hi // 2
    append = rng.random() < 0.5
    return dict(kind=kind, batch=batch, lo=max(1, int(hi * rng.uniform(0.05, 1.0))), hi=max(1, hi), hk=hk, code=code,
                page=rng.choice([0, 16, 48, 64, 256]), topk=rng.choice([0, 0, 16, 64]), axes=rng.choice([0, 1, 3]) if append else 0,
                append=append)


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


def _cu(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device=DEV)


def _lens(case):
    return [int(x) for x in case["lens"].split(",")]


def _sections(case):
    """Pairs of each axis: a quarter (three axes) or half (two) of them to the first."""
    pairs, axes = case.get("dim", D) // 2, case["axes"]
    if axes == 1:
        return (pairs,)
    first = pairs // 4 if axes == 3 else pairs // 2
    return (first, pairs - first) if axes == 2 else (first, (pairs - first) // 2, pairs - first - (pairs - first) // 2)


def _positions(n, axes, offset=0):
    """(axes, n) int32: runs of 512 text tokens, whose axes agree, between images of 16 rows of 32 tokens."""
    i = torch.arange(n, device=DEV) + offset
    image, cell = (i // 512) % 2 == 1, i % 512
    base = i - cell
    per_axis = [i, torch.where(image, base + cell // 32, i), torch.where(image, base + cell % 32, i)]
    if axes == 3:
        per_axis[0] = torch.where(image, base, i)
    return torch.stack(per_axis[:axes] if axes < 3 else per_axis).to(torch.int32)


def _tables(rows, dim):
    """cos and sin of position x 10000^(-2i/dim), worked out in 64 bits."""
    i = torch.arange(dim // 2, device=DEV, dtype=torch.float64)
    ang = torch.arange(rows, device=DEV, dtype=torch.float64)[:, None] * (10000.0 ** (-2.0 * i / dim))[None, :]
    return ang.cos().float(), ang.sin().float()


def _empty_cache(case, lens, g):
    """Codes and scales of zeros for sequences of up to max(lens) tokens, and the block table."""
    hk, page = case["hk"], case["page"]
    b, most = len(lens), max(lens)
    if page:
        per = (most + page - 1) // page
        slots, length = b * per + 3, page
        table = torch.randperm(slots, device=DEV, generator=g)[:b * per].view(b, per).to(torch.int32)
    else:
        slots, length, table = b, most, None
    s = dict(table=table)
    for name in ("k", "v"):
        s[name + "_cache"] = torch.zeros(slots, hk, length, D, dtype=torch.uint8, device=DEV).view(CODE[case["code"]])
        s[name + "_scale"] = torch.zeros(slots, hk, length, dtype=torch.uint8, device=DEV).view(torch.float8_e8m0fnu)
    return s


def _fill(s, case, lens, g):
    """Puts keys and values of every sequence into the cache, a sequence at a time."""
    for b, n in enumerate(lens):
        pos = torch.arange(n, device=DEV)
        rows = _rows(s, torch.full_like(pos, b), pos)
        _store(s, "k", _keys(g, n, case["hk"]), rows, case["code"])
        _store(s, "v", _values(g, n, case["hk"]), rows, case["code"])


def prepare(case, seed):
    g = _gen(seed)
    kind, hk = case["kind"], case["hk"]
    s = dict(case=case)
    if kind in ("rotary", "train"):
        n, dim = case["tokens"], case["dim"]
        if case["fused"]:
            qkv = _rand(g, n, (GROUP + 2) * hk, D)
            s["q"], s["k"] = qkv[:, :GROUP * hk], qkv[:, GROUP * hk:(GROUP + 1) * hk]
        else:
            s["q"], s["k"] = _rand(g, n, GROUP * hk, D), _rand(g, n, hk, D)
        offset = 4000 + int(seed) % 1000
        s["pos"], s["sections"] = _positions(n, case["axes"], offset), _sections(case)
        s["cos"], s["sin"] = _tables(n + offset + 32, dim)
        if kind == "train":
            s["q"], s["k"] = s["q"].detach().requires_grad_(True), s["k"].detach().requires_grad_(True)
            s["dq"], s["dk"] = _rand(g, n, GROUP * hk, D), _rand(g, n, hk, D)
        return s
    if kind in ("write", "read"):
        lens, start = _lens(case), case["start"]
        s.update(_empty_cache(case, [n + start for n in lens], g))
        s.update(cu=_cu(lens), total=sum(lens))
        s["start"] = torch.tensor([start - start // 2 * (b % 2) for b in range(len(lens))], dtype=torch.int32, device=DEV)
        if kind == "write":
            s["k"], s["v"] = _keys(g, sum(lens), hk), _values(g, sum(lens), hk)
        else:
            _fill(s, case, [n + start for n in lens], g)
        return s
    if kind == "attend":
        b, lo, hi = case["batch"], case["lo"], case["hi"]
        lens = torch.randint(lo, hi + 1, (b,), device=DEV, generator=g)
        lens[0] = hi                                    # (the work of a case does not hang on the seed)
        s["lens"] = lens.to(torch.int32)
        room = 1 if case["append"] else 0
        s.update(_empty_cache(case, [n + room for n in [hi] * b], g))
        _fill(s, case, lens.tolist(), g)
        s["q"] = 1.5 * _rand(g, b, 1, GROUP * hk, D)
        s["idx"] = _lists(g, s["lens"] + room, hi + room, hk, case["topk"]) if case["topk"] else None
        if case["append"]:
            s["k"], s["v"] = _keys(g, b, hk).view(b, 1, hk, D), _values(g, b, hk).view(b, 1, hk, D)
            if case["axes"]:
                s["cos"], s["sin"] = _tables(hi + 64, D)
                s["sections"] = _sections(case)
                back = torch.tensor([0, 9, 20], device=DEV)[:case["axes"], None]
                s["pos"] = (s["lens"][None, :] - back).clamp_(min=0).to(torch.int32) if case["axes"] > 1 else None
        return s
    lens = _lens(case)                                  # serve
    n, b = sum(lens), len(lens)
    s.update(_empty_cache(case, [x + 1 for x in lens], g))
    s.update(cu=_cu(lens), lens=torch.tensor(lens, dtype=torch.int32, device=DEV), sections=_sections(case))
    s["q"], s["k"], s["v"] = _rand(g, n, GROUP * hk, D), _keys(g, n, hk), _values(g, n, hk)
    s["pos"] = torch.cat([_positions(x, case["axes"]) for x in lens], 1)
    s["cos"], s["sin"] = _tables(max(lens) + 64, D)
    s["q1"], s["k1"] = 1.5 * _rand(g, b, 1, GROUP * hk, D), _keys(g, b, hk).view(b, 1, hk, D)
    s["v1"] = _values(g, b, hk).view(b, 1, hk, D)
    s["pos1"] = s["lens"].repeat(case["axes"], 1)
    return s


def _lists(g, lens, most, hk, topk):
    """(batch, hk, 1, topk) int32: block 0, the newest blocks and random others, ascending, -1 in the unused tail."""
    n = (most + BLOCK - 1) // BLOCK
    last = (lens.long() - 1).div(BLOCK, rounding_mode="floor")[:, None, None]
    at = torch.arange(n, device=DEV)
    score = torch.rand(lens.numel(), hk, n, device=DEV, generator=g)
    score = torch.where((at == 0) | (at > last - topk // 2), torch.full_like(score, 2.0), score).masked_fill(at > last, -1.0)
    val, idx = score.topk(min(topk, n), dim=-1)
    idx = torch.where(val >= 0, idx, torch.full_like(idx, n)).sort(-1).values
    idx = torch.where(idx == n, torch.full_like(idx, -1), idx)
    idx = torch.cat([idx, idx.new_full(idx.shape[:-1] + (topk - idx.shape[-1],), -1)], -1)
    return idx.to(torch.int32)[:, :, None, :].contiguous()


# ------------------------------------------------------------------------- the plain form --

def _rotate(x, cos, sin, halves, back=False):
    """Rows (n, heads, 128) rotated by the angles of (n, dim / 2) cos and sin, in 32 bits."""
    half = cos.shape[-1]
    x, cos, sin = x.float(), cos[:, None, :], sin[:, None, :] * (-1.0 if back else 1.0)
    turn, rest = x[..., :2 * half], x[..., 2 * half:]
    x0, x1 = (turn[..., :half], turn[..., half:]) if halves else (turn[..., 0::2], turn[..., 1::2])
    y0, y1 = x0 * cos - x1 * sin, x0 * sin + x1 * cos
    y = torch.cat([y0, y1], -1) if halves else torch.stack([y0, y1], -1).flatten(-2)
    return torch.cat([y, rest], -1)


def _angles(s, pos):
    """cos and sin (n, dim / 2) of tokens at positions (axes, n): each pair at the position of its axis."""
    sections = torch.tensor(s["sections"], device=DEV)
    axis = torch.arange(len(s["sections"]), device=DEV).repeat_interleave(sections, output_size=sum(s["sections"]))
    at = pos.long()[axis].t()                           # (n, dim / 2)
    pair = torch.arange(at.shape[1], device=DEV)
    return s["cos"][at, pair], s["sin"][at, pair]


def _rows(s, b, pos):
    """Rows (n, hk) of the flattened cache for tokens at position `pos` of sequences `b`."""
    hk, length = s["k_cache"].shape[1], s["k_cache"].shape[2]
    slot = b if s["table"] is None else s["table"][b, pos // length].long()
    off = pos if s["table"] is None else pos % length
    return (slot[:, None] * hk + torch.arange(hk, device=DEV)) * length + off[:, None]


def _quantise(x, code):
    """Codes and biased exponents of rows (..., 128): the smallest power of two that fits the largest value."""
    x = x.float()
    amax = x.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(amax)                            # amax = m 2^e, m in [0.5, 1)
    e = e - (9 if code == "e4m3" else 7) + (m > TOP[code] / (512 if code == "e4m3" else 128))
    e = torch.where(amax > 0, e, torch.full_like(e, -127)).clamp_(min=-127)
    y = torch.ldexp(x, -e)
    y = y.to(torch.float8_e4m3fn) if code == "e4m3" else y.round().to(torch.int8)
    return y.view(torch.uint8), (e + 127).to(torch.uint8).squeeze(-1)


def _store(s, name, x, rows, code):
    y, e = _quantise(x, code)
    s[name + "_cache"].view(torch.uint8).view(-1, D)[rows] = y
    s[name + "_scale"].view(torch.uint8).view(-1)[rows] = e


def _load(s, name, rows):
    """Rows of the cache as 32-bit numbers."""
    code = s[name + "_cache"]
    y = code.view(torch.uint8).view(-1, D)[rows].view(code.dtype).float()
    e = s[name + "_scale"].view(torch.uint8).view(-1)[rows].int()
    return y * (e << 23).view(torch.float32)[..., None]


def _token_rows(s, total):
    i = torch.arange(total, device=DEV)
    b = torch.searchsorted(s["cu"], i, right=True) - 1
    start = s["start"][b].long() if "start" in s else 0
    return _rows(s, b, i - s["cu"][b].long() + start)


def _attend(s, q, lens):
    """q (batch, hk, 16, 128) in 32 bits over the first `lens` keys of every sequence, or over its listed blocks."""
    b, hk = q.shape[:2]
    if s.get("idx") is not None:
        idx = s["idx"].view(b, hk, -1, 1).long()
        pos = (idx * BLOCK + torch.arange(BLOCK, device=DEV)).flatten(2)
        seen = (idx >= 0).expand(-1, -1, -1, BLOCK).flatten(2) & (pos < lens[:, None, None])
        pos = torch.where(seen, pos, torch.zeros_like(pos))
    else:
        length = s["k_cache"].shape[2]
        most = length if s["table"] is None else s["table"].shape[1] * length
        pos = torch.arange(most, device=DEV).expand(b, hk, -1)
        seen = pos < lens[:, None, None]
    bb, hh = torch.arange(b, device=DEV)[:, None, None], torch.arange(hk, device=DEV)[None, :, None]
    length = s["k_cache"].shape[2]
    slot = bb if s["table"] is None else s["table"][bb, pos // length].long()
    rows = (slot * hk + hh) * length + (pos if s["table"] is None else pos % length)
    x = torch.matmul(q, _load(s, "k", rows).transpose(-1, -2)) * D ** -0.5
    x = x.masked_fill(~seen[:, :, None, :], -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - m)
    l = p.sum(-1, keepdim=True)
    v = _load(s, "v", rows).masked_fill(~seen[..., None], 0.0)
    out = torch.matmul(p, v) / l
    return out.to(torch.bfloat16).view(b, 1, hk * GROUP, D), (m + l.log()).view(b, hk * GROUP, 1)


def _attend_plain(s, q, k=None, v=None, pos=None):
    case = s["case"]
    b, hk = q.shape[0], case["hk"]
    lens, q = s["lens"], q.view(b, hk * GROUP, D).float()
    if k is not None:
        k = k.view(b, hk, D).float()
        if "cos" in s:
            cos, sin = _angles(s, pos if pos is not None else lens[None])
            q, k = _rotate(q, cos, sin, True), _rotate(k, cos, sin, True)
        rows = _rows(s, torch.arange(b, device=DEV), lens.long())
        _store(s, "k", k, rows, case["code"])
        _store(s, "v", v.view(b, hk, D), rows, case["code"])
        lens = lens + 1
    return _attend(s, q.view(b, hk, GROUP, D), lens)


def _cache(s):
    return dict(k_cache=s["k_cache"], v_cache=s["v_cache"], k_scale=s["k_scale"].view(torch.uint8),
                v_scale=s["v_scale"].view(torch.uint8))


def _run_plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind in ("rotary", "train"):
        cos, sin = _angles(s, s["pos"])
        bf = torch.bfloat16
        turn = lambda x, back=False: _rotate(x.detach(), cos, sin, case["halves"], back).to(bf)  # noqa: E731
        r = dict(q=turn(s["q"]), k=turn(s["k"]))
        if kind == "train":
            r.update(dq=turn(s["dq"], True), dk=turn(s["dk"], True))
        return r
    if kind == "write":
        rows = _token_rows(s, s["total"])
        _store(s, "k", s["k"], rows, case["code"])
        _store(s, "v", s["v"], rows, case["code"])
        return _cache(s)
    if kind == "read":
        rows = _token_rows(s, s["total"])
        return dict(k=_load(s, "k", rows).to(torch.bfloat16), v=_load(s, "v", rows).to(torch.bfloat16))
    if kind == "attend":
        out, lse = _attend_plain(s, s["q"], s.get("k"), s.get("v"), s.get("pos"))
        return dict(out=out, lse=lse, **(_cache(s) if case["append"] else {}))
    cos, sin = _angles(s, s["pos"])
    q, k = (_rotate(x, cos, sin, True).to(torch.bfloat16) for x in (s["q"], s["k"]))
    rows = _token_rows(s, q.shape[0])
    _store(s, "k", k, rows, case["code"])
    _store(s, "v", s["v"], rows, case["code"])
    out, lse = _attend_plain(s, s["q1"], s["k1"], s["v1"], s["pos1"])
    return dict(q=q, k=k, out=out, lse=lse, **_cache(s))


# --------------------------------------------------------------------- the package's calls --

def _run_own(s):
    import infllm_v2 as iv
    case = s["case"]
    kind = case["kind"]
    if kind in ("rotary", "train"):
        q, k = iv.rotary_axes(s["q"], s["k"], s["cos"], s["sin"], s["pos"], sections=s["sections"],
                              interleaved=not case["halves"])
        if kind == "rotary":
            return dict(q=q, k=k)
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return dict(q=q.detach(), k=k.detach(), dq=dq, dk=dk)
    cache = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    if kind == "write":
        iv.cache_fill_q8(s["k"], s["v"], *cache, s["cu"], start=s["start"], block_table=s["table"])
        return _cache(s)
    if kind == "read":
        k, v = iv.cache_read_q8(*cache, s["cu"], s["total"], start=s["start"], block_table=s["table"])
        return dict(k=k, v=v)
    if kind == "attend":
        more = {}
        if "cos" in s:
            more = dict(rotary_cos=s["cos"], rotary_sin=s["sin"], rotary_positions=s["pos"], rotary_sections=s["sections"],
                        rotary_interleaved=False)
        out, lse = iv.infllmv2_attn_with_kvcache_q8(s["q"], *cache, k=s.get("k"), v=s.get("v"), cache_seqlens=s["lens"],
                                                    block_table=s["table"], topk_idx=s["idx"], return_softmax_lse=True, **more)
        return dict(out=out, lse=lse, **(_cache(s) if case["append"] else {}))
    q, k = iv.rotary_axes(s["q"], s["k"], s["cos"], s["sin"], s["pos"], sections=s["sections"], interleaved=False)
    iv.cache_fill_q8(k, s["v"], *cache, s["cu"], block_table=s["table"])
    out, lse = iv.infllmv2_attn_with_kvcache_q8(
        s["q1"], *cache, k=s["k1"], v=s["v1"], rotary_cos=s["cos"], rotary_sin=s["sin"], rotary_positions=s["pos1"],
        rotary_sections=s["sections"], rotary_interleaved=False, cache_seqlens=s["lens"], block_table=s["table"],
        return_softmax_lse=True)
    return dict(q=q, k=k, out=out, lse=lse, **_cache(s))


def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return _run_plain(s)


# ---------------------------------------------------------------------------------- work --

def work(case):
    kind, hk = case["kind"], case["hk"]
    row = 2 * D                                         # a bf16 row; one of the cache takes D codes and a scale
    if kind in ("rotary", "train", "serve"):
        n = case["tokens"] if "tokens" in case else sum(_lens(case))
        rows = n * hk * (GROUP + 1)
        dim = case.get("dim", D)
        turn = dict(bytes=2 * row * rows + 4 * case["axes"] * n + 4 * dim * n, flops=3 * dim * rows)
        if kind == "rotary":
            return turn
        if kind == "train":
            return {k: 2 * v for k, v in turn.items()}
        write = 2 * n * hk * (D + 1) + n * hk * row
        keys = (n + len(_lens(case))) * hk
        return dict(bytes=turn["bytes"] + write + 2 * keys * (D + 1), flops=turn["flops"] + 4 * n * hk * D + 4 * keys * D * GROUP)
    if kind in ("write", "read"):
        rows = 2 * sum(_lens(case)) * hk
        return dict(bytes=rows * (row + D + 1), flops=2 * rows * D)
    b = case["batch"]
    keys = b * (case["lo"] + case["hi"]) / 2
    if case["topk"]:
        keys = min(keys, b * BLOCK * case["topk"])
    keys *= hk
    return dict(bytes=2 * keys * (D + 1) + 2 * b * hk * GROUP * row, flops=4 * keys * D * GROUP)


# ------------------------------------------------------------------------ 64-bit answers --

def _exact_turn(x, s, halves, back=False):
    """Rotation of rows (n, heads, 128) as complex numbers."""
    half = s["cos"].shape[1]
    x = x.detach().double()
    axis = [a for a, n in enumerate(s["sections"]) for _ in range(n)]
    z = torch.stack([torch.complex(s["cos"].double()[s["at"][a].long(), i], s["sin"].double()[s["at"][a].long(), i])
                     for i, a in enumerate(axis)], 1)[:, None, :]
    z = z.conj() if back else z
    first = list(range(half)) if halves else list(range(0, 2 * half, 2))
    second = [i + half for i in first] if halves else [i + 1 for i in first]
    y, w = x.clone(), torch.complex(x[..., first], x[..., second]) * z
    y[..., first], y[..., second] = w.real, w.imag
    return y


def _exact_codes(x, code):
    """Codes (as numbers) and exponents of rows, from the definition: spacing 2^(floor(log2 |y|) - 3), at least 2^-9."""
    x = x.double()
    amax = x.abs().amax(-1)
    e = torch.full_like(amax, -127.0)
    some = amax > 0
    e[some] = torch.ceil(torch.log2(amax[some] / TOP[code])).clamp_(min=-127)
    e = torch.where(some & (amax * torch.exp2(-e) > TOP[code]), e + 1, e)
    e = torch.where(some & (e > -127) & (amax * torch.exp2(1 - e) <= TOP[code]), e - 1, e)
    y = x * torch.exp2(-e)[..., None]
    if code == "int8":
        return y.round(), e
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return (y / step).round() * step, e


class _ExactCache:
    """The cache of a state as 64-bit codes and exponents."""

    def __init__(self, s, code):
        self.s, self.code = s, code
        self.y = {n: s[n + "_cache"].double() for n in "kv"}
        self.e = {n: s[n + "_scale"].view(torch.uint8).double() - 127 for n in "kv"}

    def at(self, b, pos):
        length = self.s["k_cache"].shape[2]
        return (b, pos) if self.s["table"] is None else (self.s["table"][b].long()[pos // length], pos % length)

    def put(self, n, b, pos, x):
        slot, off = self.at(b, pos)
        y, e = _exact_codes(x, self.code)
        if not torch.is_tensor(slot):
            slot = torch.full_like(off, slot)
        self.y[n][slot, :, off], self.e[n][slot, :, off] = y, e

    def get(self, n, b, pos):
        slot, off = self.at(b, pos)
        if not torch.is_tensor(slot):
            slot = torch.full_like(off, slot)
        return self.y[n][slot, :, off] * torch.exp2(self.e[n][slot, :, off])[..., None]       # (n, hk, 128)

    def codes(self):
        keep = self.code == "e4m3"
        return dict(k_cache=self.y["k"] if keep else None, v_cache=self.y["v"] if keep else None, k_scale=None, v_scale=None)


def _exact_attend(s, cache, q, lens):
    outs, lses = [], []
    hk = s["k_cache"].shape[1]
    for b, n in enumerate(lens.tolist()):
        pos = torch.arange(n, device=DEV)
        heads_o, heads_l = [], []
        for h in range(hk):
            at = pos
            if s.get("idx") is not None:
                keep = torch.zeros(n // BLOCK + 1, dtype=torch.bool, device=DEV)
                own_list = s["idx"][b, h, 0].long()
                keep[own_list[own_list >= 0]] = True
                at = pos[keep[pos // BLOCK]]
            k, v = cache.get("k", b, at)[:, h], cache.get("v", b, at)[:, h]
            x = q[b].view(hk, GROUP, D)[h] @ k.t() / math.sqrt(D)
            heads_l.append(torch.logsumexp(x, -1))
            heads_o.append(torch.softmax(x, -1) @ v)
        outs.append(torch.cat(heads_o))
        lses.append(torch.cat(heads_l))
    return torch.stack(outs)[:, None], torch.stack(lses)[..., None]


def _exact_step(s, cache, q, k, v, pos):
    b, hk = q.shape[0], s["k_cache"].shape[1]
    q, lens = q.view(b, hk * GROUP, D).double(), s["lens"].long()
    if k is not None:
        k, v = k.view(b, hk, D).double(), v.view(b, hk, D).double()
        if "cos" in s:
            s["at"] = pos if pos is not None else lens[None]
            q, k = _exact_turn(q, s, True), _exact_turn(k, s, True)
        for i in range(b):
            cache.put("k", i, lens[i:i + 1], k[i:i + 1])
            cache.put("v", i, lens[i:i + 1], v[i:i + 1])
        lens = lens + 1
    return _exact_attend(s, cache, q, lens)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    with torch.no_grad():
        if kind in ("rotary", "train"):
            s["at"] = s["pos"]
            r = dict(q=_exact_turn(s["q"], s, case["halves"]), k=_exact_turn(s["k"], s, case["halves"]))
            if kind == "train":
                r.update(dq=_exact_turn(s["dq"], s, case["halves"], True), dk=_exact_turn(s["dk"], s, case["halves"], True))
            return r
        cache = _ExactCache(s, case["code"])
        if kind == "attend":
            out, lse = _exact_step(s, cache, s["q"], s.get("k"), s.get("v"), s.get("pos"))
            return dict(out=out, lse=lse, **(cache.codes() if case["append"] else {}))
        cu = s["cu"].tolist()
        spans = [(b, torch.arange(n, device=DEV) + (int(s["start"][b]) if "start" in s else 0), slice(cu[b], cu[b] + n))
                 for b, n in enumerate(_lens(case))]
        if kind == "read":
            return {n: torch.cat([cache.get(n, b, pos) for b, pos, _ in spans]) for n in "kv"}
        k = s["k"]
        if kind == "serve":
            s["at"] = s["pos"]
            q, k = _exact_turn(s["q"], s, True), _exact_turn(s["k"], s, True)
            rounded = k.to(torch.bfloat16)              # (what the rotation returns is what is written)
        for b, pos, rows in spans:
            cache.put("k", b, pos, (rounded if kind == "serve" else k)[rows])
            cache.put("v", b, pos, s["v"][rows])
        if kind == "write":
            return cache.codes() if case["code"] == "e4m3" else None
        out, lse = _exact_step(s, cache, s["q1"], s["k1"], s["v1"], s["pos1"])
        return dict(q=q, k=k, out=out, lse=lse, **cache.codes())

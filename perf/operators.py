"""Cases that time the paged 4-bit KV cache: the attention that reads it, the append that
quantises into it, and the page operations (fork with copy-on-write, compaction).

Where ``own`` is false the operators run in their plain form, elementary torch operations in
32 bits; where it is true, the engine's entry points run on the same state.

Storage the operators agree on.  A pool is uint8 [pages, kv heads, block] (page operations take
[layers, pages, kv heads, block]); the block of one page and head holds, one after the other,

    K nibbles [page_size, D/2] | K scales fp16 [page_size, D/32] | V nibbles | V scales

One scale serves 32 channels of one token and head: x ~ n * scale with n in [-7, 7] stored as the
nibble n + 8.  A row is D/8 little-endian 32-bit words; word t * (D/32) + g holds the channels
32 g + 8 t + e in nibble e.  scale = max|x| / 7 rounded up to 5 significant bits and held in
[2^-20, 9216], so n * scale is exact in bf16 and fp16; x / scale rounds half to even.
A page table is int32 [rows, slots], -1 where a row has no page.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SCALE_MIN, SCALE_MAX = 2.0 ** -20, 9216.0


def engine():
    """The package's array-level entry points (only where ``own`` is true)."""
    root = os.path.join(os.getcwd(), "custom-ml-library_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from tensorsmith_b200 import engine as entry_points

    return entry_points


# -- cases -----------------------------------------------------------------------------------


def listed():
    attn = dict(op="attention", q_len=1, causal=True)
    return [
        # The first tokens of one conversation on a small model: latency alone counts.
        dict(attn, name="attn_short", dtype="bf16", rows=1, q_heads=4, kv_heads=4, dim=64, lo=37, hi=37, page=16),
        # A full serving batch, one token a row, every head its own cache: the cache's bytes count.
        dict(attn, name="attn_batch", dtype="f16", rows=64, q_heads=32, kv_heads=32, dim=128, lo=1024, hi=8192,
             page=64),
        # Two users with very long documents and shared heads: few rows, so the keys are split.
        dict(attn, name="attn_long", dtype="f16", rows=2, q_heads=16, kv_heads=2, dim=128, lo=60001, hi=131072,
             page=64),
        # Five draft tokens checked at once over ragged grouped-query rows.
        dict(attn, name="attn_draft", dtype="bf16", rows=16, q_heads=32, kv_heads=8, dim=128, q_len=5, lo=5, hi=8192,
             page=32),
        # A small fp32 evaluation with an uneven head size and odd lengths.
        dict(attn, name="attn_f32", dtype="f32", rows=3, q_heads=6, kv_heads=3, dim=96, lo=1, hi=701, page=32),
        # The second chunk of two long prompts against what the first ones left in the cache.
        dict(attn, name="attn_prompt", dtype="bf16", rows=2, q_heads=32, kv_heads=8, dim=128, q_len=1000, lo=5000,
             hi=8192, page=64),
        # One token of every row of a serving batch written to the cache.
        dict(op="append", name="append_token", dtype="bf16", rows=64, kv_heads=8, dim=128, steps=1, lo=0, hi=8191,
             page=64),
        # Prompts written to the cache.
        dict(op="append", name="append_prompt", dtype="bf16", rows=8, kv_heads=8, dim=128, steps=2047, lo=0, hi=300,
             page=64),
        # A beam-search step of a small model: beams reordered, shared last pages copied.
        dict(op="beam", name="beam_small", rows=8, beams=4, layers=4, kv_heads=4, dim=64, lo=100, hi=250, page=16,
             spare=64),
        # The same for a large batch and model: 64 prompts of 4 beams.
        dict(op="beam", name="beam_large", rows=256, beams=4, layers=16, kv_heads=8, dim=128, lo=500, hi=4000,
             page=64, spare=512),
        # A small pool closed up after a few rows left.
        dict(op="compact", name="compact_small", rows=8, layers=4, kv_heads=4, dim=64, lo=20, hi=200, page=16,
             pages=160),
        # A large pool closed up: about a gigabyte of pages moves.
        dict(op="compact", name="compact_large", rows=128, layers=8, kv_heads=8, dim=128, lo=500, hi=4100, page=64,
             pages=9001),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "append", "beam", "compact"])
    page = rng.choice([16, 32, 64])
    dim = rng.choice([32, 64, 64, 96, 128, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8, 16, 32])
    if op == "attention":
        group = rng.choice([1, 1, 2, 4, 5, 8])
        q_len = 1 if rng.random() < 0.6 else _log(rng, 2, 600)
        rows = _log(rng, 1, 64)
        # the largest: about 0.3e9 cached values on one side, 2e11 score products
        hi = _log(rng, 1, 131072)
        hi = min(hi, int(2.4e9 / (rows * kv_heads * dim)),
                 max(1, int(1.5e11 / (4.0 * rows * kv_heads * group * q_len * dim))) if q_len > 1 else hi)
        q_len = max(1, min(q_len, hi))
        return dict(op=op, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), rows=rows, q_heads=kv_heads * group,
                    kv_heads=kv_heads, dim=dim, q_len=q_len, causal=rng.random() < 0.8, lo=rng.randint(0, hi), hi=hi,
                    page=page)
    if op == "append":
        rows, steps = _log(rng, 1, 64), _log(rng, 1, 2000)
        rows = max(1, min(rows, int(1.6e7 / (steps * kv_heads * dim))))
        lo = rng.randint(0, 500)
        return dict(op=op, dtype=rng.choice(["bf16", "f16", "f32"]), rows=rows, kv_heads=kv_heads, dim=dim,
                    steps=steps, lo=lo, hi=lo + rng.randint(0, 1000), page=page)
    layers = _log(rng, 1, 16)
    block = kv_heads * page * dim * 9 // 8 * layers
    if op == "beam":
        beams = rng.choice([2, 3, 4, 8])
        rows = beams * max(1, min(_log(rng, 1, 64), int(3e8 / (block * beams))))
        lo = _log(rng, 1, 500)
        hi = lo + _log(rng, 1, 2000)
        hi = max(lo, min(hi, int(4e9 / block / rows * page)))
        return dict(op=op, rows=rows, beams=beams, layers=layers, kv_heads=kv_heads, dim=dim, lo=lo, hi=hi,
                    page=page, spare=rows + rng.randint(1, 400))
    pages = max(2, min(_log(rng, 2, 20000), int(4e9 / block)))
    rows = max(1, min(_log(rng, 1, 128), pages // 2))
    hi = max(1, min(4000, pages * page // (2 * rows)))
    return dict(op=op, rows=rows, layers=layers, kv_heads=kv_heads, dim=dim, lo=rng.randint(1, hi), hi=hi, page=page,
                pages=pages)


def _lengths(case):
    """One length a row, evenly spread over [lo, hi]."""
    n, lo, hi = case["rows"], case["lo"], case["hi"]
    return [lo + (hi - lo) * i // max(1, n - 1) if n > 1 else hi for i in range(n)]


def _row_bytes(dim):
    return dim // 2 + dim // 16


# -- inputs ----------------------------------------------------------------------------------


def _pool(case, layers, pages, gen):
    """Pages as quantised activations fill them: bell-shaped nibbles, scales of 5 significant bits."""
    dim, page, heads = case["dim"], case["page"], case["kv_heads"]
    pool = torch.empty(layers, pages, heads, 2, page * _row_bytes(dim), dtype=torch.uint8, device="cuda")
    for part in pool.unbind(0):
        part.random_(0, 256, generator=gen)
        part.bitwise_and_(0x77)
        more = torch.empty_like(part).random_(0, 256, generator=gen).bitwise_and_(0x77)
        part.add_(more).add_(0x11)
        scales = torch.randint(16, 32, (pages, heads, 2, page * dim // 32), generator=gen, device="cuda",
                               dtype=torch.int32)
        part[..., page * dim // 2:] = (scales.float() / 64).half().view(torch.uint8)
    return pool.view(layers, pages, heads, 2 * page * _row_bytes(dim))


def _shuffled(lens, gen):
    order = torch.randperm(len(lens), generator=gen, device="cuda")
    return torch.tensor(lens, dtype=torch.int32, device="cuda")[order]


def _table(lens, page, slots, pages, gen):
    """Every row's pages, scattered over the pool."""
    need = (lens + page - 1) // page
    place = torch.randperm(pages, generator=gen, device="cuda").int()
    first = torch.cumsum(need, 0) - need
    slot = torch.arange(slots, device="cuda")
    at = (first[:, None] + slot).clamp(max=pages - 1)
    return torch.where(slot < need[:, None], place[at.long()], -1).int().contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, page = case["op"], case["page"]
    lens = _shuffled(_lengths(case), gen)
    state = dict(case)
    if op in ("attention", "append"):
        dtype = DTYPES[case["dtype"]]
        steps = case.get("steps", 0)
        most = case["hi"] + steps
        slots = max(1, -(-most // page))
        pages = sum(-(-(n + steps) // page) for n in _lengths(case)) + 3
        state.update(pool=_pool(case, 1, pages, gen)[0], table=_table(lens + steps, page, slots, pages, gen),
                     lens=lens, most=most)
        if op == "attention":
            # [rows, tokens, heads, dim] projections seen as [rows, heads, tokens, dim]
            q = torch.randn(case["rows"], case["q_len"], case["q_heads"], case["dim"], generator=gen, device="cuda")
            state["q"] = q.to(dtype).permute(0, 2, 1, 3)
        else:
            shape = (case["rows"], steps, case["kv_heads"], case["dim"])
            loud = 1 + 7 * (torch.rand(case["dim"], generator=gen, device="cuda") < 0.03)  # outlier channels
            for name in ("key", "value"):
                x = torch.randn(shape, generator=gen, device="cuda") * loud
                state[name] = x.to(dtype).permute(0, 2, 1, 3)
        return state
    if op == "beam":
        rows, beams = case["rows"], case["beams"]
        lens = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda").view(-1, beams)[:, :1]
        lens = lens.expand(-1, beams).reshape(-1).contiguous()
        need = (lens + page - 1) // page
        slots = case["hi"] // page + 2
        pages = sum(-(-n // page) for n in _lengths(case)) + case["spare"]
        state.update(table=_table(lens, page, slots, pages, gen), lens=lens)
        state["pool"] = _pool(case, case["layers"], pages, gen)
        pick = torch.randint(0, beams, (rows,), generator=gen, device="cuda", dtype=torch.int32)
        state["index"] = torch.arange(rows, device="cuda", dtype=torch.int32) // beams * beams + pick
        state["pages"] = pages
    else:
        pages = case["pages"]
        slots = -(-case["hi"] // page) + 1
        state.update(table=_table(lens, page, slots, pages, gen), lens=lens)
        state["pool"] = _pool(case, case["layers"], pages, gen)
    # References to each page, and (free pages, a page below which none is free, error, unused).
    refs = torch.zeros(pages + 1, dtype=torch.int32, device="cuda")
    refs.scatter_add_(0, torch.where(state["table"] < 0, pages, state["table"]).long().view(-1),
                      torch.ones_like(state["table"]).view(-1))
    state["refs"] = refs[:pages].clone()
    counters = torch.zeros(4, dtype=torch.int32, device="cuda")
    counters[0] = (state["refs"] == 0).sum()
    state["counters"] = counters
    return state


# -- the plain forms -------------------------------------------------------------------------


def _read(pool, table, dim, page):
    """Keys and values [rows, kv heads, slots * page, D] in 32 bits of the pages a table names."""
    rows, slots = table.shape
    heads = pool.shape[1]
    taken = pool.view(torch.int64)[table.clamp(min=0).long()].view(torch.uint8)  # [rows, slots, heads, block]
    taken = taken.view(rows, slots, heads, 2, page * _row_bytes(dim))
    nib = taken[..., : page * dim // 2].reshape(rows, slots, heads, 2, page, 4, dim // 32, 4)
    value = torch.stack((nib & 15, nib >> 4), -1).float() - 8  # [.., chunk t, group g, byte, nibble of the byte]
    value = value.flatten(-2).transpose(-2, -3)  # [.., page, g, t, e]
    scale = taken[..., page * dim // 2:].contiguous().view(torch.float16).float().view(
        rows, slots, heads, 2, page, dim // 32, 1, 1)
    value = (value * scale).reshape(rows, slots, heads, 2, page, dim).permute(3, 0, 2, 1, 4, 5)
    value = value.reshape(2, rows, heads, slots * page, dim)
    return value[0], value[1]


def _attention(s):
    k, v = _read(s["pool"], s["table"], s["dim"], s["page"])
    q = s["q"].float()
    rows, q_heads, q_len, dim = q.shape
    kv_heads, keys = k.shape[1], k.shape[2]
    q = q.reshape(rows, kv_heads, -1, dim)  # the query heads and tokens of one key head together
    score = q @ k.transpose(-1, -2) / math.sqrt(dim)
    score = score.view(rows, q_heads, q_len, keys)
    key = torch.arange(keys, device=q.device)
    seen = key < s["lens"][:, None, None]
    if s["causal"]:
        at = s["lens"][:, None] - q_len + torch.arange(q_len, device=q.device)
        seen = seen & (key <= at[:, :, None])
    seen = seen[:, None]
    score = torch.where(seen, score, -torch.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -torch.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    v = torch.where((key < s["lens"][:, None])[:, None, :, None], v, 0.0)
    out = (p.view(rows, kv_heads, -1, keys) @ v).view(rows, q_heads, q_len, dim)
    return (out / torch.where(total == 0, 1.0, total)).to(s["q"].dtype)


def _quantise(x):
    """Nibbles (uint8, 0..15) and fp16 scales of x [.., D] in 32 bits."""
    x = x.view(*x.shape[:-1], -1, 32)
    most = x.abs().amax(-1, keepdim=True)
    step = (most / torch.full_like(most, 7)).clamp(max=SCALE_MAX)  # a division, not a product with 1/7
    bits = step.view(torch.int32)
    step = ((bits + 0x7FFFF) & ~0x7FFFF).view(torch.float32).clamp(SCALE_MIN, SCALE_MAX)
    n = torch.round(x / step).clamp(-7, 7) + 8
    return n.to(torch.uint8), step.half()


def _append(s):
    dim, page, steps = s["dim"], s["page"], s["steps"]
    pos = s["lens"][:, None] + torch.arange(steps, device="cuda")  # [rows, steps]
    place = s["table"].gather(1, (pos // page).long()).long()
    at = (pos % page).long()
    pool = s["pool"].view(s["pool"].shape[0], s["kv_heads"], 2, page * _row_bytes(dim))
    nibbles = pool[..., : page * dim // 2].unflatten(-1, (page, dim // 2))
    scales = pool[..., page * dim // 2:].unflatten(-1, (page, dim // 16))
    n, step = _quantise(torch.stack((s["key"], s["value"]), 3).permute(0, 2, 1, 3, 4).float().contiguous())
    n = n.unflatten(-1, (4, 8)).transpose(-2, -3).flatten(-3)  # [rows, steps, heads, 2, (t, g, e)]
    nibbles[place, :, :, at] = n[..., 0::2] | (n[..., 1::2] << 4)
    scales[place, :, :, at] = step[..., 0].contiguous().view(torch.uint8)
    # what the written nibbles stand for, from the pool
    back = nibbles[place, :, :, at]
    value = torch.stack((back & 15, back >> 4), -1).float() - 8
    value = value.view(*back.shape[:-1], 4, dim // 32, 8).transpose(-2, -3).flatten(-2)
    value = value * scales[place, :, :, at].contiguous().view(torch.float16).float()[..., None]
    value = value.flatten(-2).permute(3, 0, 2, 1, 4).to(s["key"].dtype)
    return value[0], value[1]


def _count(table, pages):
    n = torch.zeros(pages + 1, dtype=torch.int32, device=table.device)
    at = torch.where(table < 0, pages, table).long().view(-1)
    return n.scatter_add_(0, at, torch.ones_like(at, dtype=torch.int32))[:pages]


def _beam(s):
    """Rows become copies of the rows that ``index`` names, sharing their pages; then every row
    gets a page of its own to write its next token to, in the order of rows and slots, the
    lowest free pages first.  Of a shared page's writers the last keeps it if nobody else has it."""
    table, lens, refs, page, pages = s["table"], s["lens"], s["refs"], s["page"], s["pages"]
    pool = s["pool"].view(torch.int64)
    src = s["index"].long()
    slot = torch.arange(table.shape[1], device="cuda")
    new_lens = lens[src]
    new = torch.where(slot < ((new_lens + page - 1) // page)[:, None], table[src], -1)
    refs += _count(new, pages) - _count(table, pages)
    row = torch.arange(len(src), device="cuda", dtype=torch.int32)
    first = (new_lens // page).long()[:, None]
    partial = new_lens % page != 0
    held = new.gather(1, first)[:, 0]
    writer = torch.where(partial, held, pages).long()
    writers = torch.zeros(pages + 1, dtype=torch.int32, device="cuda").scatter_add_(0, writer, torch.ones_like(row))
    last = torch.full((pages + 1,), -1, dtype=torch.int32, device="cuda").scatter_reduce_(0, writer, row, "amax")
    copies = partial & ((refs[held.clamp(min=0).long()] > writers[writer]) | (row < last[writer]))
    wanted = (slot == first) & (copies[:, None] | (new < 0))
    rank = torch.cumsum(wanted.view(-1).int(), 0).view(wanted.shape) - 1
    free = torch.nonzero(refs == 0)[:, 0].int()
    got = torch.where(wanted, free[rank.clamp(min=0)], new)
    src_page, dst_page = held[copies].long(), got.gather(1, first)[:, 0][copies].long()
    pool[:, dst_page] = pool[:, src_page]
    refs += _count(got, pages) - _count(new, pages)
    s["table"].copy_(got)
    s["lens"].copy_(new_lens)
    return s["table"], s["lens"], refs, (refs == 0).sum().int(), pool


def _compact(s):
    """Live pages move down until they fill the pool's start: the lowest hole takes the highest page."""
    table, refs, pool = s["table"], s["refs"], s["pool"].view(torch.int64)
    live = refs > 0
    count = live.sum()
    place = torch.arange(len(refs), device="cuda")
    movers = place[live & (place >= count)].flip(0)
    holes = place[~live & (place < count)]
    pool[:, holes] = pool[:, movers]
    to = place.clone()
    to[movers] = holes
    new_refs = refs.clone()
    new_refs[holes] = refs[movers]
    new_refs[movers] = 0
    return torch.where(table < 0, table, to[table.clamp(min=0).long()].int()), new_refs, pool


def run(s):
    op = s["op"]
    if not own:
        return {"attention": _attention, "append": _append, "beam": _beam, "compact": _compact}[op](s)
    e = engine()
    if op == "attention":
        return e.attention_int4(s["q"], s["pool"], s["table"], s["lens"], page_size=s["page"], max_len=s["most"],
                                is_causal=s["causal"])[0]
    if op == "append":
        e.kv_append_int4(s["key"], s["value"], s["pool"], s["table"], page_size=s["page"], positions=s["lens"])
        return e.kv_gather_int4(s["pool"], s["table"], s["steps"], page_size=s["page"], dtype=s["key"].dtype,
                                starts=s["lens"])
    if op == "beam":
        table, lens = e.kv_pages_fork(s["table"], s["lens"], s["index"], s["refs"], s["counters"],
                                      page_size=s["page"])
        e.kv_pages_reserve(s["pool"], table, lens, 1, s["refs"], s["counters"], page_size=s["page"])
        s["table"], s["lens"] = table, lens
        return table, lens, s["refs"], s["counters"][0], s["pool"].view(torch.int64)
    table, refs = e.kv_pages_compact(s["pool"], s["table"], s["refs"], s["counters"],
                                     table_out=torch.empty_like(s["table"]), refs_out=torch.empty_like(s["refs"]))
    return table, refs, s["pool"].view(torch.int64)


# -- what a pass cannot do without -----------------------------------------------------------


def work(case):
    op, page = case["op"], case["page"]
    lens = _lengths(case)
    size = {"f32": 4, "f16": 2, "bf16": 2}.get(case.get("dtype"), 0)
    if op == "attention":
        io = 2 * case["rows"] * case["q_heads"] * case["q_len"] * case["dim"] * size
        cache = sum(lens) * case["kv_heads"] * 2 * _row_bytes(case["dim"])
        pairs = 0
        for n in lens:  # keys seen by the q_len queries of a row
            first = max(0, n - case["q_len"])
            fewer = case["q_len"] - (n - first)
            tokens = case["q_len"] - fewer
            pairs += (tokens * (first + 1 + n) // 2) if case["causal"] else n * case["q_len"]
        return {"bytes": io + cache, "flops": 4 * case["dim"] * case["q_heads"] * pairs}
    if op == "append":
        values = 2 * case["rows"] * case["steps"] * case["kv_heads"]
        # read, quantised and written, and read back as values
        return {"bytes": values * (2 * case["dim"] * size + 2 * _row_bytes(case["dim"])),
                "flops": 4 * values * case["dim"]}
    page_bytes = case["layers"] * case["kv_heads"] * 2 * page * _row_bytes(case["dim"])
    if op == "beam":
        # of the beams of a prompt that share a partial page all but one copy it: with random
        # parents beams * (1 - 1/beams)^beams parents have no child
        share = (1 - 1 / case["beams"]) ** case["beams"]
        copied = sum(share for n in lens[:: case["beams"]] for _ in range(case["beams"]) if n % page)
        slots = case["hi"] // page + 2
        return {"bytes": 2 * copied * page_bytes + 8 * case["rows"] * slots, "flops": 0}
    live = sum(-(-n // page) for n in lens)
    moved = live * (1 - live / case["pages"])  # live pages are spread evenly over the pool
    return {"bytes": 2 * moved * page_bytes + 8 * case["pages"], "flops": 0}


# -- the operators in 64 bits ----------------------------------------------------------------


def _exact_rows(block, kind, dim, page):
    """fp64 [page, D] rows of one page's and head's block: kind 0 keys, 1 values (vectorised over leading axes)."""
    size = page * (dim // 2 + dim // 16)
    part = block[..., kind * size:(kind + 1) * size]
    words = part[..., : page * dim // 2].contiguous().view(torch.int32)
    words = words.view(*part.shape[:-1], page, dim // 8)
    scales = part[..., page * dim // 2:].contiguous().view(torch.float16).double()
    scales = scales.view(*part.shape[:-1], page, dim // 32)
    channel = torch.arange(dim, device=block.device)
    group, rest = channel // 32, channel % 32
    word = rest // 8 * (dim // 32) + group
    nibble = (words[..., word] >> (4 * (rest % 8)).int()) & 15
    return (nibble.double() - 8) * scales[..., group]


def exact(case, seed):
    op = case["op"]
    if op in ("beam", "compact"):
        return None  # whole numbers and moved bytes
    s = prepare(case, seed)
    dim, page = case["dim"], case["page"]
    if op == "append":
        out = []
        for x in (s["key"], s["value"]):
            x = x.double()
            groups = x.unflatten(-1, (-1, 32))
            least = groups.abs().amax(-1) / 7
            power = torch.floor(torch.log2(least.clamp(min=1e-300)))
            unit = torch.exp2(power - 4)  # the fifth significant bit
            scale = (torch.ceil(least / unit) * unit).clamp(SCALE_MIN, SCALE_MAX)
            n = torch.round(groups / scale[..., None]).clamp(-7, 7)
            out.append((n * scale[..., None]).flatten(-2))
        return tuple(out)
    q = s["q"].double()
    group = case["q_heads"] // case["kv_heads"]
    if sum(_lengths(case)) * case["q_heads"] * case["q_len"] * dim > 2e12:
        return None
    out = torch.zeros_like(q)
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        blocks = s["pool"][s["table"][b, : -(-n // page)].long()]
        for h in range(case["kv_heads"]):
            k = _exact_rows(blocks[:, h], 0, dim, page).flatten(0, 1)[:n]
            v = _exact_rows(blocks[:, h], 1, dim, page).flatten(0, 1)[:n]
            mine = q[b, h * group:(h + 1) * group]
            score = mine @ k.T * dim ** -0.5
            if case["causal"]:
                limit = n - case["q_len"] + torch.arange(case["q_len"], device="cuda")
                hidden = torch.arange(n, device="cuda") > limit[:, None]
                score = score.masked_fill(hidden, -math.inf)
            p = torch.softmax(score, -1)
            out[b, h * group:(h + 1) * group] = torch.where(torch.isnan(p), 0.0, p) @ v
    return out

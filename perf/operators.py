"""Performance cases of the operators on a paged key/value cache that is held in 8 bits: writing rows into it, reading them back, attention
over it, the attention weight that every cached token gets, and the eviction of the lightest tokens.

The cache: pages of 16 tokens.  `codes` [pages, 2, kv_heads, 16 * dim] (keys, then values) of float8_e4m3fn or int8, `scales` fp32
[pages, 2, kv_heads], a power of two for each page and head.  A key block is laid out [dim / 64][16 tokens][64], a value block
[dim / 64][4 quads of tokens][64][4 tokens of the quad].  Page 0 is the padding page.  `row0` [entries + 1] says which rows are an
entry's, `starts` how many tokens it has in the cache before them, `indptr` / `ids` which pages are its.

Every case is a call that a server makes: `append` and `evict` cases read back what they wrote, as the values it stands for.
Sizes are those of the repository's Qwen shapes (8 kv heads of 128 with 32 query heads, 4 of 256 with 16), contexts those of its benchmark
(1024, 10 000) and longer ones.
"""
import math
import random

import torch

own = False

PAGE = 16
FORMATS = {"e4m3": (torch.float8_e4m3fn, 448.0), "int8": (torch.int8, 127.0)}
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
SINKS = 4            # first tokens that an eviction always keeps


def _case(name, op, entries, ctx, rows, kv, group, dim, fmt, dtype="bf16", budget=0, keep=1.0):
    c = {"op": op, "entries": entries, "ctx": ctx, "rows": rows, "kv": kv, "group": group, "dim": dim, "fmt": fmt, "dtype": dtype,
         "budget": budget, "keep": keep}
    return {"name": name, **c} if name else c


def listed():
    return [
        # a decode step of a server's batch: one token each joins 16 caches, most of them in the middle of a page
        _case("append-step", "append", 16, 1024, 1, 8, 4, 128, "e4m3"),
        # prompts of all lengths enter the cache behind a shared system prompt
        _case("append-prompts", "append", 4, 100, 8000, 8, 4, 128, "int8"),
        # one session's context is taken out of the cache for another server
        _case("read-session", "read", 1, 0, 1000, 4, 4, 256, "e4m3"),
        # a batch of long documents leaves the cache in full precision
        _case("read-batch", "read", 8, 0, 10000, 8, 4, 128, "int8", "fp32"),
        # the headline's decode step: one request with 1024 tokens
        _case("attend-single", "attend", 1, 1023, 1, 8, 4, 128, "e4m3"),
        # a decode step of a full batch with contexts of all lengths
        _case("attend-batch", "attend", 32, 8191, 1, 8, 4, 128, "int8"),
        # one request over a very long context, queries kept in fp32
        _case("attend-long", "attend", 1, 131071, 1, 4, 4, 256, "e4m3", "fp32"),
        # portions of two long prompts, each over what came before it
        _case("attend-portion", "attend", 2, 9000, 1000, 8, 4, 128, "e4m3"),
        # a decode step that also adds up what each cached token was worth
        _case("weigh-step", "weigh", 16, 4095, 1, 8, 4, 128, "e4m3"),
        # whole prompts, weights counted from nothing, before they are cut to a budget
        _case("weigh-prompt", "weigh", 3, 0, 2000, 4, 4, 256, "int8", keep=0.0),
        # one chat goes back to half its tokens
        _case("evict-chat", "evict", 1, 2000, 0, 8, 4, 128, "e4m3", budget=1000),
        # a batch of long sessions is cut to a quarter
        _case("evict-batch", "evict", 8, 32000, 0, 8, 4, 128, "int8", budget=8000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "read", "attend", "attend", "weigh", "evict"])
    kv, dim = rng.choice([(8, 128), (4, 256), (2, 256), (8, 64), (1, 128), (3, 64)])
    group, fmt, dtype = rng.choice([1, 2, 4, 5, 8]), rng.choice(["e4m3", "int8"]), rng.choice(["bf16", "bf16", "fp32"])
    entries, budget, keep = _log(rng, 1, 32), 0, 1.0
    if op == "append":
        ctx, rows = _log(rng, 1, 2000) - 1, 1 if rng.random() < 0.4 else _log(rng, 2, 8000)
        entries = min(entries, max(1, 30000 // rows))
    elif op == "read":
        ctx, rows = 0, _log(rng, 1, 10000)
        entries = min(entries, max(1, 60000 // rows))
    elif op == "evict":
        ctx, rows = _log(rng, 40, 32000), 0
        budget = max(16, int(ctx * rng.uniform(0.1, 0.9)))
        entries = min(entries, max(1, 200000 // ctx), max(1, 60000000 // (budget * kv * dim)))
    elif rng.random() < 0.6:                                    # a decode step
        ctx, rows = _log(rng, 1, 130000) - 1, 1
        entries = min(entries, max(1, 250000 // (ctx + 1)))
    else:                                                       # a portion of a prompt
        ctx, rows = rng.choice([0, _log(rng, 1, 8000)]), _log(rng, 2, 1000)
        entries = max(1, min(entries, 300000000 // (rows * kv * group * (ctx + rows))))
        keep = rng.choice([0.0, 1.0, 0.9])
    return _case("", op, entries, ctx, rows, kv, group, dim, fmt, dtype, budget, keep)


def _lengths(case):
    """(tokens in the cache, rows of this call) of every entry: the first has the most, the others from a tenth of it on"""
    rng = random.Random("lengths %s" % sorted((k, v) for k, v in case.items() if k != "name"))
    some = lambda n: max(min(n, 1), int(n * rng.uniform(0.1, 1.0)))  # noqa: E731
    return [(case["ctx"], case["rows"])] + [(some(case["ctx"]), some(case["rows"])) for _ in range(case["entries"] - 1)]


def work(case):
    n, kv, D, group = _lengths(case), case["kv"], case["dim"], case["group"]
    s = 2 if case["dtype"] == "bf16" else 4
    rows, tokens = sum(r for _, r in n), sum(c + r for c, r in n)
    pair = 2 * kv * D                                            # values of a token
    if case["op"] == "append":                                   # rows in, codes out; the touched blocks' codes in, their values out
        back = sum((c + r) - c // PAGE * PAGE for c, r in n)
        return {"bytes": rows * pair * (s + 1) + back * pair * 3, "flops": (rows + back) * pair}
    if case["op"] == "read":
        return {"bytes": rows * pair * (1 + s), "flops": rows * pair}
    if case["op"] == "evict":
        kept = sum(min(c, case["budget"]) for c, _ in n)
        return {"bytes": tokens * kv * 4 + kept * (pair * 5 + kv * 8), "flops": 2 * kept * pair}
    pairs = sum(r * c + r * (r + 1) // 2 for c, r in n) * kv * group
    by = tokens * pair + 2 * rows * kv * group * D * s + (tokens * kv * 8 if case["op"] == "weigh" else 0)
    return {"bytes": by, "flops": 4 * pairs * D}


# ---- the cache's layout and formats in elementary operations ----
def _exponent(amax, top):
    """least e with amax <= top * 2^e; -100 at the least"""
    m, x = torch.frexp(amax / 2)                                 # amax = m * 2^(x + 1), m in [1/2, 1)
    edge = top / 2.0 ** (math.floor(math.log2(top)) + 1)
    e = x + 1 - (math.floor(math.log2(top)) + 1) + (m > edge).to(x.dtype)
    return torch.where(amax > 0, e.clamp(min=-100), torch.full_like(e, -100))


def _encode(x, e, fmt):
    """values -> codes at the scale 2^e"""
    y = torch.ldexp(x, -e)
    return (y.round() if fmt == "int8" else y).to(FORMATS[fmt][0])


def _bytes(codes):
    return codes.view(torch.uint8)


def _pack(k, v):
    """[n, 2 x (kv, 16, dim)] codes of blocks -> [n, 2, kv, 16 * dim]"""
    n, kv, _, D = k.shape
    a = _bytes(k).view(n, kv, PAGE, D // 64, 64).transpose(2, 3)
    b = _bytes(v).view(n, kv, 4, 4, D // 64, 64).permute(0, 1, 4, 2, 5, 3)
    return torch.stack([a.reshape(n, kv, PAGE * D), b.reshape(n, kv, PAGE * D)], 1).view(k.dtype)


def _unpack(codes):
    """[n, 2, kv, 16 * dim] -> keys, values as numbers [n, kv, 16, dim]"""
    n, _, kv, m = codes.shape
    D = m // PAGE
    a = _bytes(codes)[:, 0].view(n, kv, D // 64, PAGE, 64).transpose(2, 3).reshape(n, kv, PAGE, D)
    b = _bytes(codes)[:, 1].view(n, kv, D // 64, 4, 64, 4).permute(0, 1, 3, 5, 2, 4).reshape(n, kv, PAGE, D)
    return a.view(codes.dtype).float(), b.view(codes.dtype).float()


class _State:
    pass


def prepare(case, seed):
    """Caches with what came before, the rows of the call, and the index tables that a server has of its batch"""
    s, dev = _State(), "cuda"
    n, kv, D, fmt, B = _lengths(case), case["kv"], case["dim"], case["fmt"], case["entries"]
    gen = torch.Generator(device=dev).manual_seed(seed)
    normal = lambda *d: torch.randn(*d, generator=gen, device=dev)  # noqa: E731
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    sums = lambda v: [sum(v[:i]) for i in range(len(v) + 1)]  # noqa: E731
    s.op, s.fmt, s.type, s.kv, s.dim, s.entries = case["op"], fmt, TYPES[case["dtype"]], kv, D, B
    s.row0, s.starts, s.lens = i32(sums([r for _, r in n])), i32([c for c, _ in n]), i32([c + r for c, r in n])
    s.rows, s.max_rows, s.max_len = sum(r for _, r in n), max(r for _, r in n), max(c + r for c, r in n)
    pages = [(c + r + PAGE - 1) // PAGE for c, r in n]
    dst = [(min(c, case["budget"]) + PAGE - 1) // PAGE for c, _ in n] if case["op"] == "evict" else []
    order = 1 + torch.randperm(sum(pages) + sum(dst), generator=gen, device=dev).to(torch.int32)      # pages in no order; 0 is the padding page
    s.indptr, s.ids = i32(sums(pages)), order[:sum(pages)].contiguous()
    total = 1 + order.numel()
    # keys have a few strong channels, as after a rotation of normed heads; values do not; pages differ in size
    strong = 1 + 3 * (torch.rand(2, kv, 1, D, generator=gen, device=dev) < 0.05).float()
    strong[1] = 1
    size = torch.exp(0.5 * normal(total, 2, kv, 1, 1))
    s.codes = torch.empty(total, 2, kv, PAGE * D, dtype=FORMATS[fmt][0], device=dev)
    s.scales = torch.empty(total, 2, kv, dtype=torch.float32, device=dev)
    for p in range(0, total, 1024):                              # in runs: whole caches in fp32 would not fit beside each other
        x = normal(min(1024, total - p), 2, kv, PAGE, D) * strong * size[p:p + 1024]
        e = _exponent(x.abs().amax((3, 4)), FORMATS[fmt][1])
        c = _encode(x, e[..., None, None], fmt)
        s.codes[p:p + 1024] = _pack(c[:, 0], c[:, 1])
        s.scales[p:p + 1024] = torch.ldexp(torch.ones_like(x[:, :, :, 0, 0]), e)
    if s.op == "append":
        s.k, s.v = ((normal(s.rows, kv, D) * torch.exp(0.5 * normal(s.rows, 1, 1)) * strong[i, :, 0]).to(s.type) for i in (0, 1))
        back = [(c // PAGE * PAGE, (c + r) - c // PAGE * PAGE) for c, r in n]
        s.back0, s.back_starts, s.back_rows, s.back_most = i32(sums([r for _, r in back])), i32([c for c, _ in back]), sum(r for _, r in back), max(r for _, r in back)
    if s.op in ("attend", "weigh"):
        s.q, s.scale = normal(s.rows, kv * case["group"], D).to(s.type), D ** -0.5
    if s.op in ("weigh", "evict"):                               # what the tokens were worth so far: few heavy ones
        s.mass = 1e-3 * torch.exp(2 * normal(total, kv, PAGE))
        s.mass[0] = 0
        s.mass_out, s.keep = s.mass.clone(), case["keep"]
    if s.op == "evict":
        s.budget, s.last = case["budget"], case["budget"] // 4
        kept = [min(c, s.budget) for c, _ in n]
        s.dst_indptr, s.dst_ids = i32(sums(dst)), order[sum(pages):].contiguous()
        s.back0, s.back_starts, s.back_rows, s.back_most = i32(sums(kept)), i32([0] * B), sum(kept), max(kept)
    return s


def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from pegainfer_amd import ops_blocks as B
    if s.op == "append":
        B.kv8_append(s.k, s.v, s.codes, s.scales, s.row0, s.starts, s.indptr, s.ids, max_rows=s.max_rows)
        return B.kv8_read(s.codes, s.scales, s.back0, s.back_starts, s.indptr, s.ids, s.back_rows, max_rows=s.back_most)
    if s.op == "read":
        return B.kv8_read(s.codes, s.scales, s.row0, s.starts, s.indptr, s.ids, s.rows, dtype=s.type, max_rows=s.max_rows)
    if s.op == "attend":
        return B.kv8_attention(s.q, s.codes, s.scales, s.row0, s.starts, s.indptr, s.ids, s.scale, max_rows=s.max_rows, max_len=s.max_len)
    if s.op == "weigh":
        out = B.kv8_attention(s.q, s.codes, s.scales, s.row0, s.starts, s.indptr, s.ids, s.scale, max_rows=s.max_rows, max_len=s.max_len,
                              mass=s.mass, mass_out=s.mass_out, mass_keep=s.keep)
        return out, s.mass_out
    kept = B.kv8_evict(s.codes, s.scales, s.mass, s.lens, s.indptr, s.ids, s.dst_indptr, s.dst_ids, s.budget, keep_first=SINKS, keep_last=s.last,
                       max_len=s.max_len)
    k, v = B.kv8_read(s.codes, s.scales, s.back0, s.back_starts, s.dst_indptr, s.dst_ids, s.back_rows, max_rows=s.back_most)
    return kept, k, v, s.mass


# ---- the plain forms ----
def _pages(indptr, ids, block, there):
    """pages [entries, n] of the entries' blocks; the padding page where there is none"""
    at = (indptr[:-1, None] + block).clamp(0, ids.numel() - 1)
    return torch.where(there, ids[at], torch.zeros_like(ids[at])).long()


def _owner(row0, rows):
    r = torch.arange(rows, device=row0.device, dtype=torch.int32)
    e = torch.searchsorted(row0, r, right=True) - 1
    return e, r - row0[e]


def _read_plain(codes, scales, row0, starts, indptr, ids, rows, dtype):
    e, i = _owner(row0, rows)
    slot = starts[e] + i
    page, t = ids[indptr[e] + slot // PAGE].long(), (slot % PAGE).long()
    n, _, kv, m = codes.shape
    raw = _bytes(codes)
    k = raw.view(n, 2, kv, m // 1024, PAGE, 64)[page, 0, :, :, t].reshape(rows, kv, m // PAGE)
    v = raw.view(n, 2, kv, m // 1024, 4, 64, 4)[page, 1, :, :, t // 4, :, t % 4].reshape(rows, kv, m // PAGE)
    return tuple((x.view(codes.dtype).float() * scales[page, i][..., None]).to(dtype) for i, x in enumerate((k, v)))


def _append_plain(s):
    dev, top = s.k.device, FORMATS[s.fmt][1]
    most = (s.max_rows + PAGE - 2) // PAGE + 1
    first = s.starts // PAGE
    rows = s.row0[1:] - s.row0[:-1]
    block = first[:, None] + torch.arange(most, device=dev, dtype=torch.int32)
    there = (block * PAGE < (s.starts + rows)[:, None]) & (rows[:, None] > 0)
    page = _pages(s.indptr, s.ids, block, there)                                      # [B, most]
    slot = block[..., None] * PAGE + torch.arange(PAGE, device=dev, dtype=torch.int32)  # [B, most, 16]
    new = (slot >= s.starts[:, None, None]) & (slot < (s.starts + rows)[:, None, None])
    old = slot < s.starts[:, None, None]
    row = (s.row0[:-1, None, None] + slot - s.starts[:, None, None]).clamp(0, s.rows - 1).long()
    x = torch.stack([s.k.float()[row], s.v.float()[row]], 2).transpose(3, 4)           # [B, most, 2, kv, 16, D]
    n, o = new[:, :, None, None, :, None], old[:, :, None, None, :, None]
    e = _exponent(torch.where(n, x.abs(), torch.zeros_like(x)).amax((4, 5)), top)
    was = s.scales[page]
    has_old = old.any(-1)[..., None, None]
    e = torch.where(has_old, torch.maximum(e, torch.frexp(was)[1] - 1), e)
    shape = x.shape
    k, v = _unpack(s.codes.view(torch.uint8)[page.reshape(-1)].view(s.codes.dtype))
    before = torch.stack([k, v], 1).view(shape) * was[..., None, None]
    x = torch.where(n, x, torch.where(o, before, torch.zeros_like(x)))
    c = _encode(x, e[..., None, None], s.fmt).view(-1, *shape[2:])
    _bytes(s.codes)[page.reshape(-1)] = _bytes(_pack(c[:, 0].contiguous(), c[:, 1].contiguous()))
    s.scales[page] = torch.ldexp(torch.ones_like(was), e)
    return _read_plain(s.codes, s.scales, s.back0, s.back_starts, s.indptr, s.ids, s.back_rows, torch.bfloat16)


def _attend_plain(s):
    dev, kv, D, B = s.q.device, s.kv, s.dim, s.entries
    blocks = (s.max_len + PAGE - 1) // PAGE
    block = torch.arange(blocks, device=dev, dtype=torch.int32)[None]
    page = _pages(s.indptr, s.ids, block, block * PAGE < s.lens[:, None])
    k, v = _unpack(s.codes.view(torch.uint8)[page.reshape(-1)].view(s.codes.dtype))
    scale = s.scales[page.reshape(-1)]
    flat = lambda x, i: (x * scale[:, i, :, None, None]).view(B, blocks, kv, PAGE, D).transpose(1, 2).reshape(B, kv, blocks * PAGE, D)  # noqa: E731
    k, v = flat(k, 0), flat(v, 1)
    i = torch.arange(s.max_rows, device=dev, dtype=torch.int32)
    row = (s.row0[:-1, None] + i).clamp(0, s.rows - 1).long()                            # [B, R]
    real = i < (s.row0[1:] - s.row0[:-1])[:, None]
    q = s.q.float()[row].view(B, s.max_rows, kv, -1, D).transpose(1, 2)                # [B, kv, R, group, D]
    p = (q.reshape(B, kv, -1, D) @ k.transpose(2, 3).contiguous()).view(B, kv, s.max_rows, -1, blocks * PAGE) * s.scale
    seen = torch.arange(blocks * PAGE, device=dev, dtype=torch.int32) <= (s.starts[:, None] + i)[..., None]
    p = p.masked_fill_(~seen[:, None, :, None], -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True))
    o = (p.view(B, kv, -1, blocks * PAGE) @ v).view(B, kv, s.max_rows, -1, D)
    e, local = _owner(s.row0, s.rows)
    out = o[e, :, local.long()].reshape(s.rows, -1, D).to(s.q.dtype)
    if s.op == "attend":
        return out
    new = (p * real[:, None, :, None, None]).sum((2, 3))                                # [B, kv, L]
    new = new.view(B, kv, blocks, PAGE).transpose(1, 2)
    slot = block[..., None] * PAGE + torch.arange(PAGE, device=dev, dtype=torch.int32)
    was = s.mass[page]
    s.mass_out[page] = torch.where((slot < s.lens[:, None, None])[:, :, None], s.keep * was + new, s.mass_out[page])
    s.mass_out[0] = 0
    return out, s.mass_out


def _evict_plain(s):
    dev, kv, D, B, top = s.codes.device, s.kv, s.dim, s.entries, s.budget
    blocks, out_blocks = (s.max_len + PAGE - 1) // PAGE, (top + PAGE - 1) // PAGE
    block = torch.arange(blocks, device=dev, dtype=torch.int32)[None]
    page = _pages(s.indptr, s.ids, block, block * PAGE < s.lens[:, None])
    mass = s.mass[page].transpose(1, 2).reshape(B, kv, blocks * PAGE)
    slot = torch.arange(blocks * PAGE, device=dev, dtype=torch.int32)
    lens = s.lens[:, None, None]
    always = (slot < SINKS) | (slot >= lens - s.last) | (lens <= top)
    rank = torch.where(always, torch.full_like(mass, math.inf), mass).masked_fill(slot >= lens, -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True)[1]
    order = torch.nn.functional.pad(order, (0, max(0, top - order.shape[-1])), value=blocks * PAGE)[..., :top]
    order = torch.where(order < lens, order, torch.full_like(order, 1 << 30))            # fewer than the budget: what is not there goes last
    kept = torch.sort(order, -1)[0]
    there = kept < (1 << 30)
    at = torch.nn.functional.pad(torch.where(there, kept, torch.zeros_like(kept)), (0, out_blocks * PAGE - top))       # [B, kv, 16 * out_blocks]
    real = torch.nn.functional.pad(there, (0, out_blocks * PAGE - top))
    src = page.gather(1, (at // PAGE).view(B, -1)).view(at.shape)
    head, t = torch.arange(kv, device=dev)[None, :, None], at % PAGE
    n, _, _, m = s.codes.shape
    raw = _bytes(s.codes)
    k = raw.view(n, 2, kv, D // 64, PAGE, 64)[src, 0, head, :, t].reshape(B, kv, -1, D).view(s.codes.dtype).float()
    v = raw.view(n, 2, kv, D // 64, 4, 64, 4)[src, 1, head, :, t // 4, :, t % 4].reshape(B, kv, -1, D).view(s.codes.dtype).float()
    x = torch.stack([k, v], 1).view(B, 2, kv, out_blocks, PAGE, D)
    was = torch.stack([s.scales[src, 0, head], s.scales[src, 1, head]], 1).view(B, 2, kv, out_blocks, PAGE)
    r = real.view(B, 1, kv, out_blocks, PAGE)
    e = torch.frexp(torch.where(r, was, torch.full_like(was, 2.0 ** -100)).amax(-1))[1] - 1
    c = _encode(torch.where(r[..., None], x * was[..., None], torch.zeros_like(x)), e[..., None, None], s.fmt)          # [B, 2, kv, blocks, 16, D]
    c = c.view(torch.uint8).permute(0, 3, 1, 2, 4, 5).reshape(B * out_blocks, 2, kv, PAGE, D).view(s.codes.dtype)
    to = torch.arange(out_blocks, device=dev, dtype=torch.int32)[None]
    to = _pages(s.dst_indptr, s.dst_ids, to, to * PAGE < s.lens[:, None].clamp(max=top))
    _bytes(s.codes)[to.reshape(-1)] = _bytes(_pack(c[:, 0].contiguous(), c[:, 1].contiguous()))
    s.scales[to] = torch.ldexp(torch.ones_like(was[..., 0]), e).permute(0, 3, 1, 2).contiguous()
    moved = torch.where(real, s.mass[src, head, t], torch.zeros_like(mass[..., :1])).view(B, kv, out_blocks, PAGE)
    s.mass[to] = moved.transpose(1, 2).contiguous()
    s.mass[0] = 0
    k, v = _read_plain(s.codes, s.scales, s.back0, s.back_starts, s.dst_indptr, s.dst_ids, s.back_rows, torch.bfloat16)
    return torch.where(there, kept, torch.full_like(kept, -1)).to(torch.int32), k, v, s.mass


def _plain(s):
    if s.op == "read":
        return _read_plain(s.codes, s.scales, s.row0, s.starts, s.indptr, s.ids, s.rows, s.type)
    return {"append": _append_plain, "attend": _attend_plain, "weigh": _attend_plain, "evict": _evict_plain}[s.op](s)


# ---- the definition in 64 bits, entry by entry ----
def _e4m3_table():
    out = []
    for b in range(256):
        x, m = b >> 3 & 15, b & 7
        v = m * 2.0 ** -9 if x == 0 else (8 + m) * 2.0 ** (x - 10)
        out.append(math.nan if b & 127 == 127 else -v if b & 128 else v)
    return torch.tensor(out, dtype=torch.float64, device="cuda")


def _token(s, side, pages, slots):
    """the tokens at `slots` of an entry [n, kv, D], and their scales [n, kv]"""
    D = s.dim
    d, t, page = torch.arange(D, device="cuda"), slots % PAGE, pages[slots // PAGE]
    tt = t[:, None]
    at = d // 64 * 1024 + (tt * 64 + d % 64 if side == 0 else tt // 4 * 256 + d % 64 * 4 + tt % 4)        # [n, D]
    raw = s.codes.view(torch.uint8)[page, side].gather(2, at[:, None].expand(-1, s.kv, -1)).long()
    value = (raw - 256 * (raw > 127)).double() if s.fmt == "int8" else _e4m3_table()[raw]
    return value, s.scales[page, side].double()


def _least(amax, top):
    """least power of two that amax / top does not pass"""
    x = torch.ceil(torch.log2(amax.double() / top))
    x = torch.where(top * torch.exp2(x - 1) >= amax, x - 1, x)
    x = torch.where(top * torch.exp2(x) < amax, x + 1, x)
    return torch.exp2(x.clamp(min=-100))


def _most(x):
    """the largest of each run of 16 rows [n, kv]"""
    return torch.nn.functional.pad(x, (0, 0, 0, -x.shape[0] % PAGE)).view(-1, PAGE, x.shape[1]).amax(1)


def _rounded(x, scale, fmt):
    y = x / scale
    if fmt == "int8":
        return torch.round(y) * scale
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step * scale


def exact(case, seed):
    s = prepare(case, seed)
    top, B = FORMATS[s.fmt][1], s.entries
    lens, starts, row0 = s.lens.tolist(), s.starts.tolist(), s.row0.tolist()
    pages = [s.ids[s.indptr[e]:s.indptr[e + 1]].long() for e in range(B)]
    slots = [torch.arange(lens[e], device="cuda") for e in range(B)]
    both = (0, 1)
    if s.op == "read":
        every = [[(lambda c, w: c * w[..., None])(*_token(s, i, pages[e], slots[e])) for e in range(B)] for i in both]
        return tuple(torch.cat(x) for x in every)
    if s.op == "append":
        got = []
        for i, x in zip(both, (s.k, s.v)):
            parts = []
            for e in range(B):
                low = starts[e] // PAGE * PAGE
                c, w = _token(s, i, pages[e], torch.arange(low, starts[e], device="cuda"))
                rows = torch.cat([c * w[..., None], x[row0[e]:row0[e + 1]].double()])
                n, older = rows.shape[0], starts[e] - low
                block = torch.arange(n, device="cuda") // PAGE
                amax = rows.abs().amax(-1)
                amax[:older] = 0
                scale = _least(_most(amax), top)
                if older:
                    scale[0] = torch.maximum(scale[0], w[0])
                parts.append(_rounded(rows, scale[block][..., None], s.fmt))
            got.append(torch.cat(parts))
        return tuple(got)
    if s.op == "evict":
        kept_all, ks, mass = [], ([], []), s.mass.double()
        for e in range(B):
            n = min(lens[e], s.budget)
            m = s.mass[pages[e]].transpose(1, 2).reshape(-1, s.kv)[:lens[e]]
            kept = slots[e][:, None].expand(-1, s.kv)
            if lens[e] > s.budget:
                lo, hi = SINKS, lens[e] - s.last
                between = lo + torch.sort(-m[lo:hi], dim=0, stable=True)[1][:s.budget - SINKS - s.last]
                kept = torch.cat([kept[:lo], torch.sort(between, 0)[0], kept[hi:]])
            kept_all.append(torch.nn.functional.pad(kept.T.int(), (0, s.budget - n), value=-1))
            block = torch.arange(n, device="cuda") // PAGE
            for i in both:
                c, w = _token(s, i, pages[e], slots[e])
                c, w = c.gather(0, kept[..., None].expand(-1, -1, s.dim)), w.gather(0, kept)
                ks[i].append(_rounded(c * w[..., None], _most(w)[block][..., None], s.fmt))
            to = s.dst_ids[s.dst_indptr[e]:s.dst_indptr[e + 1]].long()
            moved = torch.zeros(to.numel() * PAGE, s.kv, dtype=torch.float64, device="cuda")
            moved[:n] = m.double().gather(0, kept)
            mass[to] = moved.view(-1, PAGE, s.kv).transpose(1, 2)
        return torch.stack(kept_all), torch.cat(ks[0]), torch.cat(ks[1]), mass
    H = s.q.shape[1]
    out = torch.zeros(s.rows, H, s.dim, dtype=torch.float64, device="cuda")
    mass = s.mass.double() if s.op == "weigh" else None
    for e in range(B):
        k, v = ((lambda c, w: (c * w[..., None]).transpose(0, 1).contiguous())(*_token(s, i, pages[e], slots[e])) for i in both)      # [kv, L, D]
        weight = torch.zeros(s.kv, lens[e], dtype=torch.float64, device="cuda")
        for r in range(row0[e], row0[e + 1], 128):
            m = min(128, row0[e + 1] - r)
            q = s.q[r:r + m].double().view(m, s.kv, -1, s.dim).transpose(0, 1).reshape(s.kv, -1, s.dim)
            z = torch.bmm(q, k.transpose(1, 2).contiguous()) * s.scale
            far = (starts[e] + r - row0[e] + torch.arange(m, device="cuda")).repeat_interleave(H // s.kv)
            p = torch.softmax(z.masked_fill(slots[e] > far[:, None], -math.inf), -1)
            out[r:r + m] = torch.bmm(p, v).view(s.kv, m, -1, s.dim).transpose(0, 1).reshape(m, H, s.dim)
            weight += p.sum(1)
        if mass is not None:
            had = mass[pages[e]].transpose(1, 2).reshape(-1, s.kv)
            had[:lens[e]] = s.keep * had[:lens[e]] + weight.T
            mass[pages[e]] = had.view(-1, PAGE, s.kv).transpose(1, 2)
    return out if mass is None else (out, mass)

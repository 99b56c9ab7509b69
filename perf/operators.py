"""Cases of the packed KV cache's windowed decode, chunk attention and page operators.

Four operators over one page arena (16-token pages, FP16 / INT8 / INT4 records):

* ``window``:  one query token per sequence attends the last ``window`` tokens
  and the first ``sinks`` tokens of its pages;
* ``chunk``:   the last ``rows`` tokens of every sequence attend its pages
  causally (a prompt's next chunk, or drafted tokens to verify), optionally
  with the same window and sinks;
* ``fork``:    new sequences continue given parents: page tables are gathered,
  a half-filled last page is copied into a fresh slot;
* ``compact``: the pages that a table refers to are copied, in table order,
  into another arena, and the table follows.

The page format: a page holds ``kv_heads`` records back to back, each
``[K payload][V payload][K scales][V scales][pad to 16 bytes]``; payloads are 16
rows of ``dim`` values (fp16, int8 or nibbles, the even element low), V's 16-byte
units permuted inside each 128-byte line; scales are fp16, one per ``group``
consecutive elements.  A table entry is an int64: mode in bits 0-1 (0 skip,
1 INT4, 2 INT8, 3 FP16), valid tokens - 1 in bits 2-5, byte offset from bit 8.
"""

import math
import sys

import torch

own = False

BLOCK = 16


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one user's chat reply with a local-attention layer: the smallest call, where latency counts
        dict(name="window_single", op="window", batch=1, q_heads=16, kv_heads=8, dim=128, group=2048,
             tokens=512, ragged=False, rows=1, window=128, sinks=4, fp16=25, int8=25, int4=50, gone=0),
        # a serving batch at the batched-decode geometry, half of each context inside the window
        dict(name="window_batch", op="window", batch=64, q_heads=16, kv_heads=8, dim=128, group=2048,
             tokens=8192, ragged=False, rows=1, window=4096, sinks=16, fp16=15, int8=35, int4=40, gone=10),
        # one sequence of a million tokens of which a local layer sees the last eighth
        dict(name="window_long", op="window", batch=1, q_heads=32, kv_heads=8, dim=128, group=2048,
             tokens=1048576, ragged=False, rows=1, window=131072, sinks=128, fp16=5, int8=25, int4=70, gone=0),
        # requests of uneven age, head_dim 64, three query heads a KV head, a window that ends inside pages
        dict(name="window_ragged", op="window", batch=37, q_heads=24, kv_heads=8, dim=64, group=64,
             tokens=5003, ragged=True, rows=1, window=1000, sinks=5, fp16=20, int8=30, int4=45, gone=5),
        # drafted tokens of a speculative decoder, verified in one pass over the cache
        dict(name="chunk_verify", op="chunk", batch=16, q_heads=16, kv_heads=8, dim=128, group=2048,
             tokens=8192, ragged=False, rows=5, window=0, sinks=0, fp16=15, int8=35, int4=40, gone=10),
        # a short follow-up question to a short chat
        dict(name="chunk_short", op="chunk", batch=1, q_heads=16, kv_heads=8, dim=128, group=64,
             tokens=612, ragged=False, rows=100, window=0, sinks=0, fp16=25, int8=25, int4=50, gone=0),
        # the last chunk of a long document's prompt, four query heads a KV head
        dict(name="chunk_long", op="chunk", batch=1, q_heads=32, kv_heads=8, dim=128, group=2048,
             tokens=32768, ragged=False, rows=2048, window=0, sinks=0, fp16=10, int8=20, int4=65, gone=5),
        # chunks of uneven requests through a local-attention layer with sinks, odd sizes, head_dim 64
        dict(name="chunk_window", op="chunk", batch=4, q_heads=24, kv_heads=8, dim=64, group=64,
             tokens=12001, ragged=True, rows=1000, window=2048, sinks=4, fp16=20, int8=30, int4=45, gone=5),
        # one step of a beam search over every layer of a small model: table gather and a few pages, latency
        dict(name="fork_beams", op="fork", layers=28, batch=4, children=4, kv_heads=8, dim=128, group=64,
             tokens=519, fp16=5, int8=0, int4=95),
        # sixteen prompts sampled four times each: every child shares the prompt's pages
        dict(name="fork_samples", op="fork", layers=28, batch=16, children=64, kv_heads=8, dim=128, group=64,
             tokens=2055, fp16=5, int8=0, int4=95),
        # a small model's pages moved together after its beams have ended: planning counts as much as copying
        dict(name="compact_beams", op="compact", layers=28, batch=4, columns=33, kv_heads=8, dim=128,
             group=64, fp16=10, int8=0, int4=70, gone=20, shared=50),
        # a whole store moved into a fresh arena, sequence after sequence, after requests have ended
        dict(name="compact_store", op="compact", layers=28, batch=16, columns=128, kv_heads=8, dim=128,
             group=64, fp16=10, int8=30, int4=50, gone=10, shared=20),
    ]


def draw(rng):
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    op = rng.choice(["window", "window", "chunk", "chunk", "chunk", "fork", "compact"])
    dim = rng.choice([64, 128])
    if op in ("window", "chunk"):
        kv = rng.choice([1, 2, 4, 8])
        fp16, int8 = rng.randint(5, 30), rng.randint(5, 40)
        gone = rng.choice([0, 5, 10])
        case = dict(op=op, q_heads=kv * rng.choice([1, 2, 3, 4, 8]), kv_heads=kv, dim=dim,
                    group=rng.choice([32, 64, 128, 16 * dim]), ragged=rng.random() < 0.5,
                    fp16=fp16, int8=int8, int4=100 - fp16 - int8 - gone, gone=gone)
        if op == "window":
            batch = log(1, 64)
            tokens = log(17, min(131072, 524288 // batch))
            return dict(case, batch=batch, tokens=tokens, rows=1, window=log(1, tokens), sinks=rng.choice([0, 1, 4, 37, 128]))
        batch = log(1, 16)
        rows = log(2, 1024)
        tokens = rows + log(1, min(16384, 65536 // batch))
        rows = max(2, min(rows, int(8e11 / (4 * batch * case["q_heads"] * dim * tokens))))
        local = rng.random() < 0.4
        return dict(case, batch=batch, tokens=tokens, rows=rows, window=log(1, tokens) if local else 0,
                    sinks=rng.choice([0, 4, 64]) if local else 0)
    kv = rng.choice([2, 4, 8])
    group = rng.choice([32, 64, 128])
    if group > dim:
        group = dim
    layers, batch = rng.randint(1, 28), log(1, 16)
    if op == "fork":
        return dict(op="fork", layers=layers, batch=batch, children=log(1, 64), kv_heads=kv, dim=dim, group=group,
                    tokens=log(1, 2048), fp16=rng.randint(2, 20), int8=0, int4=80)
    fp16, int8 = rng.randint(5, 30), rng.randint(5, 40)
    return dict(op="compact", layers=layers, batch=batch, columns=log(1, 128), kv_heads=kv, dim=dim, group=group,
                fp16=fp16, int8=int8, int4=90 - fp16 - int8, gone=10, shared=rng.choice([0, 20, 50]))


# ------------------------------------------------------------- page format
MODE_BITS = {1: 4, 2: 8, 3: 16}


def _record(dim, group, bits):
    """(payload bytes, scales, record bytes) of one (page, head)."""
    payload = BLOCK * dim * bits // 8
    scales = 0 if bits == 16 else BLOCK * dim // group
    return payload, scales, (2 * payload + 4 * scales + 15) // 16 * 16


def _v_order(dim, bits, device):
    """Stored position of each row-major byte of a V payload (its own inverse)."""
    row = dim * bits // 8
    o = torch.arange(BLOCK * row, device=device)
    if row == 256:
        key = ((o >> 9) & 1) | (((o >> 10) & 1) << 2)
    elif row == 128:
        key = (o >> 7) & 6
    elif row == 64:
        key = (o >> 6) & 6
    else:
        key = (o >> 6) & 2
    return o ^ (key << 4)


def _layout(case, counts):
    """Byte base of each size class (16, 8, 4) in an arena of ``counts`` slots, and the arena's bytes."""
    base, cursor = {}, 0
    for bits in (16, 8, 4):
        base[bits] = cursor
        cursor += counts[bits] * case["kv_heads"] * _record(case["dim"], case["group"], bits)[2]
    return base, max(cursor, 16)


def _shares(case, n):
    """How many of ``n`` pages are FP16, INT8, INT4 and evicted."""
    total = case["fp16"] + case["int8"] + case["int4"] + case.get("gone", 0)
    n8, n4 = n * case["int8"] // total, n * case["int4"] // total
    gone = n * case.get("gone", 0) // total
    return n - n8 - n4 - gone, n8, n4, gone


def _fill(case, arena, base, bits, count, g):
    """Write ``count`` quantized pages of one precision: K and V are N(0, 1), four channels a head eight times that."""
    heads, dim, group = case["kv_heads"], case["dim"], case["group"]
    payload, scales, rec = _record(dim, group, bits)
    size = heads * rec
    dev = arena.device
    order = _v_order(dim, bits, dev)
    step = max(1, (1 << 26) // (heads * BLOCK * dim))
    for lo in range(0, count, step):
        n = min(step, count - lo)
        page = arena[base + lo * size:base + (lo + n) * size].view(n, heads, rec)
        page.zero_()
        for kv in range(2):
            x = torch.randn(n, heads, BLOCK, dim, device=dev, generator=g)
            x[..., 3::dim // 4] *= 8
            if bits == 16:
                raw = x.half().view(torch.uint8).reshape(n, heads, payload)
            else:
                top = 127 if bits == 8 else 7
                x = x.half().float().view(n, heads, scales, group)
                s = (x.abs().amax(-1, keepdim=True) / top).clamp_min(2.0 ** -14).half()
                q = (x / s.float()).round().clamp(-top, top).to(torch.int32)
                if bits == 8:
                    raw = q.to(torch.int8).view(torch.uint8).reshape(n, heads, payload)
                else:
                    q = (q & 15).view(n, heads, payload, 2)
                    raw = (q[..., 0] | (q[..., 1] << 4)).to(torch.uint8)
                at = 2 * payload + kv * 2 * scales
                page[..., at:at + 2 * scales] = s.view(n, heads, scales).view(torch.uint8)
            page[..., kv * payload:(kv + 1) * payload] = raw[..., order] if kv else raw


def _descriptors(case, modes, ntok, base, g):
    """Table entries of pages of ``modes`` (0 skip), each class at a random permutation of its slots."""
    dev = modes.device
    flat = modes.reshape(-1)
    off = torch.zeros(flat.numel(), dtype=torch.int64, device=dev)
    for mode, bits in MODE_BITS.items():
        where = (flat == mode).nonzero().view(-1)
        size = case["kv_heads"] * _record(case["dim"], case["group"], bits)[2]
        off[where] = base[bits] + torch.randperm(where.numel(), device=dev, generator=g) * size
    d = (off << 8) | ((ntok.reshape(-1).to(torch.int64) - 1) << 2) | flat
    return torch.where(flat == 0, torch.zeros_like(d), d).view(modes.shape)


def _counts(modes):
    return {bits: int((modes == mode).sum()) for mode, bits in MODE_BITS.items()}


def _random_modes(case, n, g, dev):
    n16, n8, n4, gone = _shares(case, n)
    codes = torch.cat([torch.full((m,), c, dtype=torch.int64, device=dev)
                       for c, m in ((3, n16), (2, n8), (1, n4), (0, gone))])
    return codes[torch.randperm(n, device=dev, generator=g)]


# ----------------------------------------------------------------- prepare
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)
    return {"window": _prepare_attention, "chunk": _prepare_attention,
            "fork": _prepare_fork, "compact": _prepare_compact}[case["op"]](case, g)


def _prepare_attention(case, g):
    dev = torch.device("cuda")
    batch, rows, most = case["batch"], case["rows"], case["tokens"]
    tokens = torch.full((batch,), most, dtype=torch.int64, device=dev)
    if case["ragged"]:  # requests of uneven age, the oldest of the full length
        least = max(1, most // 3)
        tokens = torch.randint(least, most + 1, (batch,), device=dev, generator=g)
        tokens[0] = most
    blocks = -(-most // BLOCK)
    modes = _random_modes(case, batch * blocks, g, dev).view(batch, blocks)
    column = torch.arange(blocks, device=dev)
    used = (tokens + BLOCK - 1) // BLOCK
    fresh = ((tokens - rows).clamp_min(0) // BLOCK - 1).clamp_min(0)  # this step's tokens and the page before are FP16
    modes = torch.where(column >= fresh[:, None], 3, modes)
    modes = torch.where(column >= used[:, None], 0, modes)
    ntok = (tokens[:, None] - column * BLOCK).clamp(1, BLOCK)
    counts = _counts(modes)
    base, size = _layout(case, counts)
    arena = torch.empty(size, dtype=torch.uint8, device=dev)
    for bits in (16, 8, 4):
        _fill(case, arena, base[bits], bits, counts[bits], g)
    query = torch.randn(batch, case["q_heads"], rows, case["dim"], device=dev, generator=g).half()
    return dict(case=case, arena=arena, base=base, counts=counts, table=_descriptors(case, modes, ntok, base, g),
                tokens=tokens.to(torch.int32), query=query, scale=1 / math.sqrt(case["dim"]))


def _prepare_fork(case, g):
    dev = torch.device("cuda")
    layers, batch, children, tokens = case["layers"], case["batch"], case["children"], case["tokens"]
    blocks = -(-tokens // BLOCK)
    room = blocks + 8  # columns for the tokens still to come
    modes = torch.zeros(layers, batch, room, dtype=torch.int64, device=dev)
    old = max(0, blocks - 2)  # the newest pages are FP16
    modes[..., :old] = _random_modes(case, layers * batch * old, g, dev).view(layers, batch, old)
    modes[..., old:blocks] = 3
    ntok = (tokens - torch.arange(room, device=dev) * BLOCK).clamp(1, BLOCK).expand(layers, batch, room)
    counts = _counts(modes)
    spare = layers * children
    base, _ = _layout(case, counts)
    slots = dict(counts)
    slots[16] += spare
    base, size = _layout(case, slots)
    arena = torch.zeros(size, dtype=torch.uint8, device=dev)
    for bits in (16, 8, 4):
        _fill(case, arena, base[bits], bits, counts[bits], g)
    parents = torch.randint(0, batch, (children,), device=dev, generator=g)
    size16 = case["kv_heads"] * _record(case["dim"], case["group"], 16)[2]
    free = base[16] + (counts[16] + torch.randperm(spare, device=dev, generator=g)) * size16
    fresh = ((free << 8) | 3).view(layers, children)
    # a parent's first child goes on with the parent's own last page
    index = torch.arange(children, device=dev)
    first = (parents[None, :] == parents[:, None]).to(torch.int64).argmax(1) == index
    fresh = torch.where(first, torch.zeros_like(fresh), fresh)
    return dict(case=case, arena=arena, base=base, counts=slots, table=_descriptors(case, modes, ntok, base, g),
                parents=parents, fresh=fresh, tokens=torch.full((batch,), tokens, dtype=torch.int32, device=dev))


def _prepare_compact(case, g):
    dev = torch.device("cuda")
    shape = (case["layers"], case["batch"], case["columns"])
    n = math.prod(shape)
    modes = _random_modes(case, n, g, dev)
    counts = _counts(modes)
    base, size = _layout(case, counts)
    arena = torch.empty(size, dtype=torch.uint8, device=dev)
    for bits in (16, 8, 4):
        _fill(case, arena, base[bits], bits, counts[bits], g)
    ntok = torch.full((n,), BLOCK, dtype=torch.int64, device=dev)
    table = _descriptors(case, modes, ntok, base, g).view(shape)
    # forked sequences: a share of the columns refer to sequence 0's page
    same = torch.rand(shape[0], 1, shape[2], device=dev, generator=g) * 100 < case["shared"]
    table = torch.where(same, table[:, :1], table).contiguous()
    live = {bits: int((torch.unique(table[(table & 3) == mode]).numel())) for mode, bits in MODE_BITS.items()}
    return dict(case=case, arena=arena, base=base, counts=counts, table=table, live=live,
                target=torch.zeros(size, dtype=torch.uint8, device=dev))


# --------------------------------------------------------------------- run
def run(s):
    c = s["case"]
    if own:
        if "dynamic-quantization_b200" not in sys.path:
            sys.path.insert(0, "dynamic-quantization_b200")
        import anchorkv_b200 as akv

        if c["op"] == "compact":
            pool = akv.PagePool.over(s["arena"], c["kv_heads"], c["dim"], group=c["group"])
            into = akv.PagePool.over(s["target"], c["kv_heads"], c["dim"], group=c["group"], pages=s["counts"])
            return akv.compact_pages(pool, s["table"], into), s["target"]
        pool = akv.PagePool.over(s["arena"], c["kv_heads"], c["dim"], group=c["group"])
        if c["op"] == "fork":
            return akv.fork_pages(pool, s["table"], s["parents"], s["fresh"], tokens=s["tokens"]), s["arena"]
        store = akv.PagedBatch.over(pool, s["table"], tokens=s["tokens"])
        if c["op"] == "window":
            return akv.packed_attention(s["query"], store, s["scale"], window=c["window"], sinks=c["sinks"])
        return akv.chunk_attention(s["query"], store, s["scale"], window=c["window"] or None, sinks=c["sinks"])
    if c["op"] == "fork":
        return _plain_fork(s)
    if c["op"] == "compact":
        return _plain_compact(s)
    return _plain_attention(s)


def _class_pages(s, d, bits):
    """fp32 K and V ``[n, heads, 16, dim]`` of entries ``d`` read as pages of one precision."""
    c, n = s["case"], d.numel()
    heads, dim, group = c["kv_heads"], c["dim"], c["group"]
    payload, scales, rec = _record(dim, group, bits)
    count = s["counts"][bits]
    if count == 0:
        return None
    slots = s["arena"][s["base"][bits]:s["base"][bits] + count * heads * rec].view(count, heads, rec)
    page = slots[(((d >> 8) - s["base"][bits]) // (heads * rec)).clamp(0, count - 1)]
    k = _values(page[..., :payload], page[..., 2 * payload:2 * payload + 2 * scales], bits, group)
    v = _values(page[..., payload:2 * payload][..., _v_order(dim, bits, d.device)],
                page[..., 2 * payload + 2 * scales:2 * payload + 4 * scales], bits, group)
    shape = (n, heads, BLOCK, dim)
    return k.view(shape), v.view(shape)


def _values(raw, scale_bytes, bits, group):
    """fp32 values of a payload as the cache's readers see them: integers times their scale, rounded once to fp16."""
    raw = raw.contiguous()
    if bits == 16:
        return raw.view(torch.float16).float()
    if bits == 8:
        q = raw.view(torch.int8).float()
    else:
        q = torch.stack([raw & 15, raw >> 4], -1).flatten(-2).float()
        q = q - 16 * (q > 7).float()
    s = scale_bytes.contiguous().view(torch.float16).float()
    x = q.view(*s.shape, group) * s.unsqueeze(-1)
    return x.half().float().flatten(-2)


def _plain_attention(s):
    c, table, query = s["case"], s["table"], s["query"]
    dev = table.device
    batch, blocks = table.shape
    heads, dim, rows = c["kv_heads"], c["dim"], query.shape[2]
    tokens = s["tokens"].to(torch.int64)
    at = tokens[:, None] - rows + torch.arange(rows, device=dev)  # [batch, rows]: positions of the query rows
    if c["window"]:  # the columns that hold sinks, then those from the oldest window's page on
        lead = min(blocks, -(-c["sinks"] // BLOCK))
        near = min(blocks - lead, -(-(c["window"] + rows + BLOCK) // BLOCK))
        first = ((at[:, :1] - c["window"] + 1).clamp_min(0) // BLOCK).clamp_min(lead)
        column = torch.cat([torch.arange(lead, device=dev).expand(batch, lead),
                            first + torch.arange(near, device=dev)], 1)
    else:
        column = torch.arange(blocks, device=dev).expand(batch, blocks)
    d = torch.where(column < blocks, table.gather(1, column.clamp_max(blocks - 1)), 0)
    mode = (d & 3).reshape(-1)
    n = d.numel()
    k = torch.zeros(n, heads, BLOCK, dim, device=dev)
    v = torch.zeros(n, heads, BLOCK, dim, device=dev)
    k, v = _take(s, d, mode, 3, k, v)
    k, v = _take(s, d, mode, 2, k, v)
    k, v = _take(s, d, mode, 1, k, v)
    span = column.shape[1] * BLOCK
    k = k.view(batch, -1, heads, BLOCK, dim).transpose(1, 2).reshape(batch, heads, span, dim)
    v = v.view(batch, -1, heads, BLOCK, dim).transpose(1, 2).reshape(batch, heads, span, dim)
    pos = (column[:, :, None] * BLOCK + torch.arange(BLOCK, device=dev)).view(batch, 1, span)
    there = ((d & 3) != 0).repeat_interleave(BLOCK, 1).view(batch, 1, span) & (pos < tokens.view(batch, 1, 1))
    v = v * there.view(batch, 1, span, 1)
    here = at[:, :, None]
    seen = there & (pos <= here) & (here >= 0)
    if c["window"]:
        seen = seen & ((pos > here - c["window"]) | (pos < c["sinks"]))
    gqa = c["q_heads"] // heads
    q = query.float().view(batch, heads, gqa * rows, dim)
    score = (q @ k.transpose(2, 3)).view(batch, heads, gqa, rows, span).mul_(s["scale"])
    score.masked_fill_(~seen.view(batch, 1, 1, rows, span), -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(batch, heads, gqa * rows, span) @ v).view(batch, heads, gqa, rows, dim)
    out = torch.where(total > 0, out / total, 0.0)
    return out.view(batch, c["q_heads"], rows, dim).half()


def _take(s, d, mode, code, k, v):
    got = _class_pages(s, d.reshape(-1), MODE_BITS[code])
    if got is None:
        return k, v
    hit = (mode == code).view(-1, 1, 1, 1)
    return torch.where(hit, got[0], k), torch.where(hit, got[1], v)


def _plain_fork(s):
    c, table, parents, fresh, arena = s["case"], s["table"], s["parents"], s["fresh"], s["arena"]
    size = c["kv_heads"] * _record(c["dim"], c["group"], 16)[2]
    new = table.index_select(1, parents)
    tokens = s["tokens"].to(torch.int64)[parents]
    column = (tokens // BLOCK).clamp_max(table.shape[2] - 1).view(1, -1, 1).expand(table.shape[0], -1, 1)
    old = new.gather(2, column).squeeze(2)
    copied = (fresh != 0) & (tokens % BLOCK != 0)
    pages = arena[s["base"][16]:s["base"][16] + s["counts"][16] * size].view(-1, size)
    src = torch.where(copied, (old >> 8) - s["base"][16], 0).view(-1) // size
    dst = torch.where(copied, (fresh >> 8) - s["base"][16], 0).view(-1) // size
    pages.index_copy_(0, dst, pages.index_select(0, torch.where(copied.view(-1), src, 0)))
    entry = torch.where(copied, (fresh >> 8 << 8) | (old & 255), old)
    new.scatter_(2, column, entry.unsqueeze(2))
    return new, arena


def _plain_compact(s):
    table = s["table"]
    flat = table.reshape(-1)
    new = torch.zeros_like(flat)
    new = _move(s, flat, new, 3)
    new = _move(s, flat, new, 2)
    new = _move(s, flat, new, 1)
    return new.view(table.shape), s["target"]


def _move(s, flat, new, code):
    """Copy the pages of one precision in the order in which the table first names them; their new entries."""
    c, bits = s["case"], MODE_BITS[code]
    count, live = s["counts"][bits], s["live"][bits]
    if live == 0:
        return new
    size = c["kv_heads"] * _record(c["dim"], c["group"], bits)[2]
    hit = (flat & 3) == code
    slot = torch.where(hit, ((flat >> 8) - s["base"][bits]) // size, count)
    index = torch.arange(flat.numel(), device=flat.device)
    first = torch.full((count + 1,), flat.numel(), device=flat.device).scatter_reduce(0, slot, index, "amin")
    owner = hit & (first[slot] == index)
    rank = (owner.cumsum(0) - 1)
    place = torch.zeros(count + 1, dtype=torch.int64, device=flat.device).scatter(0, torch.where(owner, slot, count), rank)
    src = torch.zeros(live + 1, dtype=torch.int64, device=flat.device).scatter(0, torch.where(owner, rank, live), slot.clamp_max(count - 1))
    pages = s["arena"][s["base"][bits]:s["base"][bits] + count * size].view(-1, size)
    target = s["target"][s["base"][bits]:s["base"][bits] + live * size].view(-1, size)
    torch.index_select(pages, 0, src[:live], out=target)
    entry = ((s["base"][bits] + place[slot] * size) << 8) | (flat & 255)
    return torch.where(hit, entry, new)


# -------------------------------------------------------------------- work
def _visible(case, tokens, at):
    """Tokens that the query row at position ``at`` sees, evicted pages left in."""
    n = min(at + 1, tokens)
    if not case["window"]:
        return n
    near = min(n, case["window"])
    return near + min(case["sinks"], n - near)


def work(case):
    page = lambda bits: case["kv_heads"] * _record(case["dim"], case["group"], bits)[2]  # noqa: E731
    if case["op"] == "compact":
        n = case["layers"] * case["batch"] * case["columns"]
        n16, n8, n4, _ = _shares(case, n)
        kept = 1 - case["shared"] / 100 * (1 - 1 / case["batch"])
        return {"bytes": 2 * kept * (n16 * page(16) + n8 * page(8) + n4 * page(4)) + 16 * n, "flops": 0}
    if case["op"] == "fork":
        blocks = -(-case["tokens"] // BLOCK) + 8
        held = case["batch"] * (1 - (1 - 1 / case["batch"]) ** case["children"])  # parents that have a child
        copies = max(0, case["children"] - held) * case["layers"] if case["tokens"] % BLOCK else 0
        return {"bytes": 8 * case["layers"] * blocks * (held + case["children"]) + 2 * copies * page(16) +
                8 * case["layers"] * case["children"], "flops": 0}
    batch, rows, tokens = case["batch"], case["rows"], case["tokens"]
    mean = tokens * 2 // 3 if case["ragged"] else tokens
    kept = 1 - case["gone"] / 100
    pairs = sum(_visible(case, mean, mean - rows + i) for i in range(rows) if mean - rows + i >= 0)
    union = mean if not case["window"] else min(mean, case["window"] + rows - 1 + case["sinks"])
    blocks = -(-union // BLOCK)
    late = min(blocks, -(-rows // BLOCK) + 1)  # this step's own pages are FP16
    n16, n8, n4, _ = _shares(case, blocks - late)
    pages = (n16 + late) * page(16) + n8 * page(8) + n4 * page(4)
    return {"bytes": batch * (pages + 8 * blocks + 4 * case["q_heads"] * rows * case["dim"]),
            "flops": 4.0 * batch * case["q_heads"] * case["dim"] * pairs * kept}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "fork":
        return _exact_fork(s)
    if case["op"] == "compact":
        return _exact_compact(s)
    return _exact_attention(s)


def _exact_page_values(s, offsets, mode):
    """float64 K, V ``[pages, heads, 16, dim]`` of the pages at byte ``offsets``, element by element."""
    c, bits = s["case"], MODE_BITS[mode]
    heads, dim, group = c["kv_heads"], c["dim"], c["group"]
    payload, scales, rec = _record(dim, group, bits)
    dev = s["arena"].device
    element = torch.arange(BLOCK * dim, device=dev)
    record = offsets[:, None, None] + torch.arange(heads, device=dev)[None, :, None] * rec
    out = []
    for kv in range(2):
        byte = element * bits // 8
        if kv:
            byte = payload + _v_order(dim, bits, dev)[byte]
        low = s["arena"][record + byte].to(torch.int64)
        if bits == 16:
            high = s["arena"][record + byte + 1].to(torch.int64)
            word = (low | (high << 8)).to(torch.int32).to(torch.int16)
            x = word.view(torch.float16).double()
        else:
            if bits == 4:
                low = torch.where(element % 2 == 0, low % 16, low // 16)
            q = torch.where(low >= 1 << (bits - 1), low - (1 << bits), low).double()
            at = record + 2 * payload + kv * 2 * scales + element // group * 2
            word = (s["arena"][at].to(torch.int64) | (s["arena"][at + 1].to(torch.int64) << 8)).to(torch.int32)
            x = (q * word.to(torch.int16).view(torch.float16).double()).half().double()
        out.append(x.view(-1, heads, BLOCK, dim))
    return out


def _exact_attention(s):
    c = s["case"]
    dev = s["arena"].device
    heads, dim, gqa = c["kv_heads"], c["dim"], c["q_heads"] // c["kv_heads"]
    rows = s["query"].shape[2]
    out = torch.zeros(s["query"].shape, dtype=torch.float64, device=dev)
    lengths = s["tokens"].tolist()
    for b, length in enumerate(lengths):
        d = s["table"][b]
        column = torch.arange(d.numel(), device=dev)
        want = ((d & 3) != 0) & (column * BLOCK < length)
        if c["window"]:
            oldest = max(0, length - rows) - c["window"] + 1
            want &= (column * BLOCK < c["sinks"]) | (column * BLOCK + BLOCK > oldest)
        held = want.nonzero().view(-1)
        if not held.numel():
            continue
        k = torch.zeros(held.numel(), heads, BLOCK, dim, dtype=torch.float64, device=dev)
        v = torch.zeros_like(k)
        for mode in MODE_BITS:
            of = ((d[held] & 3) == mode).nonzero().view(-1)
            for part in of.split(1 << 11):
                k[part], v[part] = _exact_page_values(s, d[held[part]] >> 8, mode)
        pos = (held[:, None] * BLOCK + torch.arange(BLOCK, device=dev)).view(-1)
        k = k.transpose(0, 1).reshape(heads, -1, dim)
        v = v.transpose(0, 1).reshape(heads, -1, dim)
        v = v * (pos < length).view(1, -1, 1)
        step = max(1, (1 << 27) // (heads * gqa * pos.numel()))
        for lo in range(0, rows, step):
            at = length - rows + torch.arange(lo, min(rows, lo + step), device=dev)[:, None]
            seen = (pos < length) & (pos <= at) & (at >= 0)
            if c["window"]:
                seen &= (at - pos < c["window"]) | (pos < c["sinks"])
            q = s["query"][b, :, lo:lo + step].double().view(heads, gqa, -1, dim)
            score = torch.einsum("hgrd,htd->hgrt", q, k) * s["scale"]
            score = torch.where(seen, score, -math.inf)
            top = score.amax(-1, keepdim=True)
            weight = torch.where(seen, (score - torch.where(top == -math.inf, 0.0, top)).exp(), 0.0)
            total = weight.sum(-1, keepdim=True)
            got = torch.einsum("hgrt,htd->hgrd", weight / torch.where(total > 0, total, 1.0), v)
            out[b, :, lo:lo + step] = got.reshape(c["q_heads"], -1, dim)
    return out


def _exact_fork(s):
    c = s["case"]
    size = c["kv_heads"] * _record(c["dim"], c["group"], 16)[2]
    table, fresh, parents = s["table"].cpu(), s["fresh"].cpu().tolist(), s["parents"].cpu().tolist()
    tokens = s["tokens"].cpu().tolist()
    new = torch.zeros(table.shape[0], len(parents), table.shape[2], dtype=torch.int64)
    for layer in range(table.shape[0]):
        for i, p in enumerate(parents):
            new[layer, i] = table[layer, p]
            if tokens[p] % BLOCK and fresh[layer][i]:
                column = tokens[p] // BLOCK
                old, to = int(table[layer, p, column]), fresh[layer][i] >> 8
                s["arena"][to:to + size] = s["arena"][old >> 8:(old >> 8) + size]
                new[layer, i, column] = (to << 8) | (old & 255)
    return new, s["arena"]


def _exact_compact(s):
    c = s["case"]
    size = {m: c["kv_heads"] * _record(c["dim"], c["group"], b)[2] for m, b in MODE_BITS.items()}
    table = s["table"].cpu()
    place, entries = {}, []
    taken = {m: s["base"][b] for m, b in MODE_BITS.items()}
    for d in table.reshape(-1).tolist():
        mode, off = d & 3, d >> 8
        if mode == 0:
            entries.append(0)
            continue
        if off not in place:
            place[off] = taken[mode]
            taken[mode] += size[mode]
            s["target"][place[off]:place[off] + size[mode]] = s["arena"][off:off + size[mode]]
        entries.append((place[off] << 8) | (d & 255))
    return torch.tensor(entries).view(table.shape), s["target"]

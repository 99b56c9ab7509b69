"""Windowed decode and chunk attention where calls go wrong: layouts, scales,
tokens nobody sees, rows that see nothing, far offsets, streams, captured graphs,
and the borders between the two ways that a chunk runs."""

import numpy as np
import pytest
import torch

import anchorkv_b200 as akv
from anchorkv_b200 import pool as P
from position_reference import assert_rows_close, attention_rows_torch

pytestmark = pytest.mark.gpu

# rows, tokens: a chunk that runs on the decode, and one on the operand tiles
SMALL, LARGE = (5, [150, 70]), (2100, [2500, 2150])
SIZES = pytest.mark.parametrize("rows,lengths", [SMALL, LARGE], ids=["decode", "tiles"])
HQ, HKV = 16, 2


def _normal(cuda, seed, shape, dtype=torch.float16):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(cuda)


def _fp16_store(cuda, lengths, dim=128, heads=HKV, seed=0, bits=16):
    """Pages of one precision and the values that they hold (those of FP16 pages exactly)."""
    span = -(-max(max(lengths), 1) // 16) * 16
    k, v = (_normal(cuda, seed + i, (len(lengths), heads, span, dim)) for i in (1, 2))
    nblk = span // 16
    pool = P.PagePool(heads, dim, pages={bits: len(lengths) * nblk}, device=cuda, shuffle_seed=seed)
    store = P.pack_dense(pool, k, v, np.full((len(lengths), nblk), bits), lengths=lengths)
    return store, k, v


def _expected(q, k, v, lengths, scale, window=None, sinks=0, held=None):
    parts = []
    for b, n in enumerate(lengths):
        there = torch.arange(k.shape[2], device=k.device) < n if held is None else held[b]
        parts.append(attention_rows_torch(q[b], k[b], v[b], there, n, scale, window, sinks))
    return np.stack([p[0] for p in parts]), np.stack([p[1] for p in parts])


def _clean(cuda):
    assert akv.take_device_status(cuda) == 0


@SIZES
def test_layouts_of_queries_and_outputs(cuda, rows, lengths):
    store, k, v = _fp16_store(cuda, lengths)
    batch, scale = len(lengths), .09
    q = _normal(cuda, 5, (batch, HQ, rows, 128))
    want = _expected(q, k, v, lengths, scale, 100, 3)
    call = lambda query, **kw: akv.chunk_attention(query, store, scale, window=100, sinks=3, **kw)  # noqa: E731
    token_major = q.transpose(1, 2).contiguous().transpose(1, 2)   # [batch, rows, heads, dim] in memory
    padded = torch.zeros((batch, HQ, rows, 192), dtype=torch.float16, device=cuda)[..., 24:152]
    padded.copy_(q)
    odd = torch.zeros(q.numel() + 1, dtype=torch.float16, device=cuda)[1:].view(q.shape)  # 2-byte aligned
    odd.copy_(q)
    spread = torch.zeros((batch, HQ, rows, 256), dtype=torch.float16, device=cuda)[..., ::2]
    spread.copy_(q)
    for query in (q, token_major, padded, odd, spread):
        assert_rows_close(call(query), *want)
    same = q[:1, :1].expand(batch, HQ, rows, 128)
    assert_rows_close(call(same), *_expected(same, k, v, lengths, scale, 100, 3))
    # outputs: token-major, rows of an odd pitch, an odd address; what lies around them stays
    for shape, cut in (((batch, rows, HQ, 128), lambda t: t.transpose(1, 2)),
                       ((batch, HQ, rows + 2, 131), lambda t: t[:, :, 1:-1, 1:129]),
                       ((batch, HQ + 1, rows, 136), lambda t: t[:, :HQ, :, 8:])):
        whole = torch.full(shape, 7.0, dtype=torch.float16, device=cuda)
        out = cut(whole)
        assert call(q, out=out) is out
        assert_rows_close(out, *want)
        mask = torch.zeros(shape, dtype=torch.bool, device=cuda)
        cut(mask).fill_(True)
        assert (whole[~mask] == 7).all()
    _clean(cuda)


@SIZES
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("scale", [0.0, -0.09, 1e-8, 3.0])
def test_scales_of_any_sign(cuda, rows, lengths, dim, scale):
    store, k, v = _fp16_store(cuda, lengths, dim)
    q = _normal(cuda, 5, (len(lengths), HQ, rows, dim))
    if scale == 3.0:
        q = q / 32  # scores stay where fp32 sums carry the tolerance's 2^-13
    out = akv.chunk_attention(q, store, scale, window=200, sinks=1)
    assert_rows_close(out, *_expected(q, k, v, lengths, scale, 200, 1))
    one = akv.packed_attention(q[:, :, -1:].contiguous(), store, scale, window=200, sinks=1)
    assert_rows_close(one, *(x[:, :, -1:] for x in _expected(q, k, v, lengths, scale, 200, 1)))
    _clean(cuda)


@SIZES
@pytest.mark.parametrize("dim,bits", [(64, 16), (128, 16), (128, 8), (64, 4)])
def test_tokens_nobody_sees_hold_anything(cuda, rows, lengths, dim, bits):
    """Page bytes of tokens outside every row's window, past a page's count, of evicted
    pages and of the free slots are NaN patterns; the output is as without them."""
    store, k, v = _fp16_store(cuda, lengths, dim, bits=bits)
    q = _normal(cuda, 5, (len(lengths), HQ, rows, dim))
    table = store.table.clone()
    table[:, 2] = 0  # evicted
    pool = store.pool
    clean = P.PagedBatch.over(pool, table, tokens=store.tokens)
    window, sinks = 40, 5
    want = [akv.chunk_attention(q, clean, .1, window=window, sinks=sinks),
            akv.packed_attention(q[:, :, -1:], clean, .1, window=window, sinks=sinks)]
    before = pool.arena.clone()
    arena = torch.full_like(pool.arena, 0xFF)  # NaN as fp16, and scales of NaN
    rec = pool.page_bytes[bits] // HKV
    payload = 16 * dim * bits // 8
    row_bytes = dim * bits // 8
    order = P.v_order(dim, bits, "cpu").numpy()
    for b, n in enumerate(lengths):
        for j in range(-(-n // 16)):
            pos = 16 * j + np.arange(16)
            seen = (pos < n) & ((pos >= max(n - rows - window + 1, 0)) | (pos < sinks))
            if j == 2 or not seen.any():
                continue
            off = int(table[b, j]) >> 8
            for h in range(HKV):
                at = off + h * rec
                keep = np.zeros(rec, bool)
                keep[:payload] = np.repeat(seen, row_bytes)
                keep[payload:2 * payload] = np.repeat(seen, row_bytes)[order]
                keep[2 * payload:] = True  # scales of a page that is seen
                m = torch.from_numpy(keep).to(cuda)
                arena[at:at + rec] = torch.where(m, before[at:at + rec], arena[at:at + rec])
    pool.arena.copy_(arena)
    got = [akv.chunk_attention(q, clean, .1, window=window, sinks=sinks),
           akv.packed_attention(q[:, :, -1:], clean, .1, window=window, sinks=sinks)]
    for g, w in zip(got, want):
        assert torch.equal(g, w) and torch.isfinite(g).all()
    _clean(cuda)


@SIZES
def test_a_nan_key_stays_with_the_rows_that_see_it(cuda, rows, lengths):
    store, k, v = _fp16_store(cuda, lengths)
    at = lengths[0] - 3  # the last three rows of sequence 0 see it
    off = int(store.table[0, at // 16]) >> 8
    record = store.pool.arena[off:off + store.pool.page_bytes[16] // HKV].view(torch.float16)
    record[at % 16 * 128] = float("nan")
    q = _normal(cuda, 5, (len(lengths), HQ, rows, 128))
    out = akv.chunk_attention(q, store, .09)
    group = HQ // HKV
    assert torch.isnan(out[0, :group, -3:]).all()
    out[0, :group, -3:] = 0
    want, tol = _expected(q, k, v, lengths, .09)
    want[0, :group, -3:] = 0
    assert_rows_close(out, want, tol)
    _clean(cuda)


@pytest.mark.parametrize("dim", [64, 128])
def test_rows_that_see_nothing_are_zero(cuda, dim):
    store, k, v = _fp16_store(cuda, [40, 0, 1, 16], dim)
    empty = P.PagedBatch.over(store.pool, torch.zeros_like(store.table), tokens=store.tokens)
    for rows in (1, 3, 17, 200, 3000 + 7):
        q = _normal(cuda, rows, (4, HQ, rows, dim))
        out = akv.chunk_attention(q, store, .1, out=torch.full_like(q, 3))
        assert_rows_close(out, *_expected(q, k, v, [40, 0, 1, 16], .1))
        assert not akv.chunk_attention(q, empty, .1, out=torch.full_like(q, 3)).any()
        assert not akv.chunk_attention(q, empty, .1, window=9, sinks=2, out=torch.full_like(q, 3)).any()
    q = _normal(cuda, 7, (4, HQ, 1, dim))
    assert not akv.packed_attention(q, empty, .1, window=9, out=torch.full_like(q, 3)).any()
    # a window that only evicted pages fall into, with a sink that is there
    table = store.table.clone()
    table[0, 1:] = 0
    only = P.PagedBatch.over(store.pool, table, tokens=store.tokens)
    held = torch.zeros((4, 48), dtype=torch.bool, device=cuda)
    for b, n in enumerate((16, 0, 1, 16)):
        held[b, :n] = True
    for sinks in (0, 2):
        out = akv.packed_attention(q, only, .1, window=8, sinks=sinks)
        assert_rows_close(out, *_expected(q, k, v, [40, 0, 1, 16], .1, 8, sinks, held))
    assert akv.chunk_attention(q[:, :, :0], store, .1).shape == (4, HQ, 0, dim)
    _clean(cuda)


@SIZES
def test_token_counts_of_every_form(cuda, rows, lengths):
    """A tensor, one int, counts beyond the pages or below zero, a PagedLayer, and a table of several
    sequences' common pages."""
    store, k, v = _fp16_store(cuda, lengths)
    q = _normal(cuda, 5, (len(lengths), HQ, rows, 128))
    one = P.PagedBatch.over(store.pool, store.table, tokens=400)
    want = _expected(q, k, v, [400, 400], .1)
    if lengths[1] >= 400:
        assert_rows_close(akv.chunk_attention(q, one, .1), *want)
    span = store.table.shape[1] * 16
    full = P.PagedBatch.over(store.pool, store.table[:1], tokens=torch.tensor([2 ** 31 - 1], dtype=torch.int32,
                                                                              device=cuda))
    held = [torch.arange(span, device=cuda) < lengths[0]]
    assert_rows_close(akv.chunk_attention(q[:1], full, .1), *_expected(q[:1], k[:1], v[:1], [span], .1, held=held))
    below = P.PagedBatch.over(store.pool, store.table, tokens=torch.tensor([-5, -2 ** 31], dtype=torch.int32,
                                                                          device=cuda))
    assert not akv.chunk_attention(q, below, .1, window=30, out=torch.full_like(q, 2)).any()
    unknown = P.PagedBatch.over(store.pool, store.table)
    for call in (lambda: akv.chunk_attention(q, unknown, .1),
                 lambda: akv.packed_attention(q[:, :, :1], unknown, .1, window=5)):
        with pytest.raises(ValueError, match="token counts"):
            call()
    layer = akv.PagedLayer(HKV, 128, lengths[0], device=cuda)
    layer.append(k[:1, :, :lengths[0]], v[:1, :, :lengths[0]])
    lk, lv = layer.dense()
    assert_rows_close(akv.chunk_attention(q[:1], layer, .1, window=64, sinks=20),
                      *_expected(q[:1], lk, lv, lengths[:1], .1, 64, 20))
    _clean(cuda)


def test_python_refusals(cuda):
    store, _, _ = _fp16_store(cuda, [40, 16])
    q = torch.zeros((2, HQ, 3, 128), dtype=torch.float16, device=cuda)
    chunk = lambda query=q, layer=store, **kw: akv.chunk_attention(query, layer, kw.pop("scale", .1), **kw)  # noqa: E731
    for kw in (dict(window=0), dict(window=-3), dict(sinks=2), dict(window=4, sinks=-1)):
        with pytest.raises(ValueError, match="window"):
            chunk(**kw)
        with pytest.raises(ValueError, match="window"):
            akv.packed_attention(q[:, :, :1], store, .1, **kw)
    for bad in (q.float(), q.cpu(), q.bfloat16()):
        with pytest.raises(ValueError, match="FP16"):
            chunk(bad)
    with pytest.raises(ValueError, match="divisible"):
        chunk(q[:, :15])
    with pytest.raises(ValueError, match="rows, head_dim"):
        chunk(q[:1])
    for out in (q.float(), q[:, :, :2], q.cpu(), torch.zeros((2, HQ, 3, 256), dtype=torch.float16, device=cuda)[..., ::2]):
        with pytest.raises(ValueError, match="out must"):
            chunk(out=out)
    for scale in (float("nan"), float("inf")):
        with pytest.raises(ValueError):
            chunk(scale=scale)
    for tokens in (torch.zeros(2, dtype=torch.int64, device=cuda), torch.zeros(3, dtype=torch.int32, device=cuda),
                   torch.zeros(2, dtype=torch.int32), torch.zeros(4, dtype=torch.int32, device=cuda)[::2], -1, 1 << 31):
        with pytest.raises(ValueError, match="token"):
            chunk(layer=P.PagedBatch.over(store.pool, store.table, tokens=tokens))
    for table in (store.table.int(), store.table.t().contiguous().t()):
        with pytest.raises(ValueError, match="page table"):
            chunk(layer=P.PagedBatch.over(store.pool, table, tokens=16))
    with pytest.raises(ValueError, match="one device"):
        chunk(layer=P.PagedBatch.over(store.pool, store.table.cpu(), tokens=16))
    with pytest.raises(ValueError):  # one row of pages for both sequences: their strides are not a table's
        chunk(layer=P.PagedBatch.over(store.pool, store.table[:1].expand(2, -1), tokens=16))
    with pytest.raises(ValueError, match="nonempty"):
        chunk(layer=P.PagedBatch.over(store.pool, store.table[:, :0], tokens=16))
    _clean(cuda)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("columns", [250, 1000, 1051, 1052, 1053, 1054, 4000])
def test_a_long_sequence_with_many_rows(cuda, dim, columns):
    """Both ways of running a chunk, over lengths around where one takes over."""
    n = 16 * columns - 7
    store, k, v = _fp16_store(cuda, [n], dim, heads=1, seed=columns)
    q = _normal(cuda, 3, (1, 8, 44, dim))
    for window, sinks in ((None, 0), (16 * 600, 33)):
        out = akv.chunk_attention(q, store, dim ** -.5, window=window, sinks=sinks)
        assert_rows_close(out, *_expected(q, k, v, [n], dim ** -.5, window, sinks))
    _clean(cuda)


def test_a_batch_in_slices(cuda):
    """Operand tiles of 2.7 GB in all: the batch goes in slices of whole sequences."""
    heads, columns, batch, rows = 8, 1024, 40, 17
    small, k, v = _fp16_store(cuda, [1024], heads=heads)
    order = torch.stack([torch.randperm(columns, generator=torch.Generator().manual_seed(b)) % 64 for b in range(batch)])
    table = small.table[0][order.to(cuda)].contiguous()
    tokens = torch.randint(8000, 16 * columns + 1, (batch,), generator=torch.Generator().manual_seed(1))
    store = P.PagedBatch.over(small.pool, table, tokens=tokens.int().to(cuda))
    q = _normal(cuda, 4, (batch, 16, rows, 128))
    out = akv.chunk_attention(q, store, .1)
    _clean(cuda)
    for b in (0, 1, 15, 29, 30, 31, 38, 39):
        at = (16 * order[b][:, None] + torch.arange(16)).reshape(-1).to(cuda)
        there = torch.ones(16 * columns, dtype=torch.bool, device=cuda)
        want = attention_rows_torch(q[b], k[0][:, at], v[0][:, at], there, int(tokens[b]), .1)
        assert_rows_close(out[b], *want)


def test_offsets_beyond_32_bits(cuda):
    """Pages that start past 4 GiB of an arena, and the slots that forks and compaction use there."""
    size = (4 << 30) + (64 << 20)
    store, k, v = _fp16_store(cuda, [700, 100])
    arena = torch.empty(size, dtype=torch.uint8, device=cuda)
    far = (4 << 30) + 4096
    arena[far:far + store.pool.nbytes].copy_(store.pool.arena)
    pool = akv.PagePool.over(arena, HKV, 128)
    table = torch.where(store.table != 0, store.table + (far << 8), 0)
    moved = P.PagedBatch.over(pool, table, tokens=store.tokens)
    for rows in (1, 4, 600):
        q = _normal(cuda, rows, (2, HQ, rows, 128))
        got = akv.chunk_attention(q, moved, .1, window=200, sinks=4)
        assert torch.equal(got, akv.chunk_attention(q, store, .1, window=200, sinks=4))
    q = _normal(cuda, 1, (2, HQ, 1, 128))
    assert torch.equal(akv.packed_attention(q, moved, .1, window=50), akv.packed_attention(q, store, .1, window=50))
    fresh = torch.tensor([0, P.encode(16, 1, size - store.pool.page_bytes[16])], device=cuda)
    forked = akv.fork_pages(pool, table, torch.tensor([0, 0], device=cuda), fresh, tokens=700)
    pair = P.PagedBatch.over(pool, forked, tokens=700)
    out = akv.packed_attention(q[:1].expand(2, -1, -1, -1), pair, .1, window=50)
    assert torch.equal(out[0], out[1])
    into = P.PagePool(HKV, 128, pages={16: store.table.numel()}, device=cuda)
    near = akv.compact_pages(pool, table, into)
    assert torch.equal(akv.packed_attention(q, P.PagedBatch.over(into, near, tokens=store.tokens), .1, window=50),
                       akv.packed_attention(q, store, .1, window=50))
    _clean(cuda)


@SIZES
def test_streams_at_once(cuda, rows, lengths):
    """The same calls on two streams at a time, each waiting only for its own inputs."""
    stores = [_fp16_store(cuda, lengths, seed=10 * i) for i in range(2)]
    qs = [_normal(cuda, 5 + i, (len(lengths), HQ, rows, 128)) for i in range(2)]
    want = [akv.chunk_attention(q, s[0], .1, window=300) for q, s in zip(qs, stores)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                late = torch.zeros_like(qs[i])
                torch.cuda._sleep(200_000)
                late.copy_(qs[i])
                got[i].append(akv.chunk_attention(late, stores[i][0], .1, window=300))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])
    _clean(cuda)


@SIZES
def test_captured_graphs(cuda, rows, lengths):
    """Two graphs captured on one stream, replayed in turn, on two streams at once, and with eager calls
    between; token counts and table entries are read at replay."""
    store, k, v = _fp16_store(cuda, [n + 40 for n in lengths])
    tokens = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    view = P.PagedBatch.over(store.pool, store.table, tokens=tokens)
    qs = [_normal(cuda, 5 + i, (len(lengths), HQ, rows, 128)) for i in range(2)]
    calls = [lambda q: akv.chunk_attention(q, view, .1), lambda q: akv.chunk_attention(q, view, .1, window=77, sinks=9)]
    for call, q in zip(calls, qs):
        call(q)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for call, q in zip(calls, qs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(call(q))
        graphs.append(graph)
    masks = [(None, 0), (77, 9)]
    for step in range(3):
        tokens.copy_(torch.tensor([n + 13 * step for n in lengths], dtype=torch.int32))
        for q in qs:
            q.copy_(_normal(cuda, 50 + step, q.shape))
        torch.cuda.synchronize()
        if step < 2:
            for g in graphs:
                g.replay()
        else:
            streams = [torch.cuda.Stream() for _ in graphs]
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        eager = akv.chunk_attention(qs[0], view, .1, window=20)
        torch.cuda.synchronize()
        now = [n + 13 * step for n in lengths]
        held = [torch.arange(k.shape[2], device=cuda) < n + 40 for n in lengths]
        for out, q, (window, sinks) in zip(outs, qs, masks):
            assert_rows_close(out, *_expected(q, k, v, now, .1, window, sinks, held))
        assert_rows_close(eager, *_expected(qs[0], k, v, now, .1, 20, 0, held))
    _clean(cuda)


def test_captured_forks_and_compactions(cuda):
    store, _, _ = _fp16_store(cuda, [100, 37])
    pool, table = store.pool, store.table
    spare = P.PagePool.over(torch.empty(pool.nbytes + 4 * pool.page_bytes[16], dtype=torch.uint8, device=cuda), HKV, 128)
    spare.arena[:pool.nbytes].copy_(pool.arena)
    slots = [pool.nbytes + i * pool.page_bytes[16] for i in range(4)]
    tokens = torch.tensor([100, 37], dtype=torch.int32, device=cuda)
    parents = torch.tensor([0, 0, 1], device=cuda)
    fresh = torch.tensor([0, P.encode(16, 1, slots[0]), P.encode(16, 1, slots[1])], device=cuda)
    targets = [P.PagePool(HKV, 128, pages={16: n}, device=cuda) for n in (40, 40)]
    side = torch.cuda.Stream()
    graphs, forked, compacted = [], [], []
    for target in targets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            forked.append(akv.fork_pages(spare, table, parents, fresh, tokens=tokens))
            compacted.append(akv.compact_pages(spare, forked[-1], target))
        graphs.append(graph)
    q = _normal(cuda, 2, (3, HQ, 1, 128))
    for order in ([0, 0, 1], [1, 0, 1]):
        parents.copy_(torch.tensor(order))
        counts = torch.tensor([[100, 37][p] for p in order], dtype=torch.int32, device=cuda)
        for graph, target, t in zip(graphs, targets, compacted):
            graph.replay()
            torch.cuda.synchronize()
            got = akv.packed_attention(q, P.PagedBatch.over(target, t, tokens=counts), .1, window=60, sinks=5)
            plain = P.PagedBatch.over(pool, table[parents].contiguous(), tokens=counts)
            assert torch.equal(got, akv.packed_attention(q, plain, .1, window=60, sinks=5))
    _clean(cuda)


def test_a_store_under_visibility_rules_has_no_positions(cuda):
    """Its decode view names visible blocks, whose columns are no positions: refused."""
    cache = akv.DeclarativeKVCache(16)
    k, v = (_normal(cuda, i, (1, HKV, 32, 128)) for i in (1, 2))
    cache.add_segment(0, k, v, token_start=0, role=akv.SegmentRole.CONTEXT)
    q = _normal(cuda, 3, (1, HQ, 1, 128))
    assert akv.packed_attention(q, cache, .1).shape == q.shape
    with pytest.raises(ValueError, match="token counts"):
        akv.packed_attention(q, cache, .1, window=8)
    with pytest.raises(ValueError, match="token counts"):
        akv.chunk_attention(q, cache, .1)
    _clean(cuda)


@pytest.mark.parametrize("dim,hq,hkv,window,sinks", [(128, 16, 8, 30000, 77), (64, 24, 2, 20001, 0),
                                                     (128, 4, 4, 40000, 5), (64, 8, 8, 9000, 8000)])
def test_long_windows_of_single_tokens(cuda, dim, hq, hkv, window, sinks):
    """Items of many pages, cut between warps and joined by the merge."""
    lengths = [33000, 20007, 5]
    store, k, v = _fp16_store(cuda, lengths, dim, heads=hkv, seed=window)
    q = _normal(cuda, 3, (3, hq, 1, dim))
    out = akv.packed_attention(q, store, dim ** -.5, window=window, sinks=sinks)
    assert_rows_close(out, *_expected(q, k, v, lengths, dim ** -.5, window, sinks))
    several = _normal(cuda, 4, (3, hq, 3, dim))
    out = akv.chunk_attention(several, store, dim ** -.5, window=window, sinks=sinks)
    assert_rows_close(out, *_expected(several, k, v, lengths, dim ** -.5, window, sinks))
    _clean(cuda)

"""Windowed decode, chunk attention, forking and compaction: what needs no GPU.

Argument checks of the C entry points (none reaches the CUDA runtime), of their
Python counterparts as far as they come before a device is needed, and the host
bookkeeping of page slots."""

import ctypes

import numpy as np
import pytest
import torch

import anchorkv_b200 as akv
from anchorkv_b200 import _lib, live
from anchorkv_b200 import pool as P

OK, INVALID, UNSUPPORTED = _lib.OK, _lib.ERR_INVALID, _lib.ERR_UNSUPPORTED
VP = ctypes.c_void_p
A, A8 = VP(0x1000), VP(0x1008)  # an aligned and a misaligned buffer, never looked at
NAN, INF = float("nan"), float("inf")


def _chunk(arena=A, arena_bytes=1 << 20, table=A, table_stride=64, columns=64, tokens=None, uniform=1000, q=A,
           strides=(4096, 1024, 128), batch=2, rows=8, q_heads=16, kv_heads=8, dim=128, group=64, scale=.1, window=0,
           sinks=0, splits=4, out=A, ws=A, ws_bytes=1 << 30):
    return _lib.load().akv_chunk_attention(arena, arena_bytes, table, table_stride, None, columns, tokens, uniform, q,
                                           *strides, batch, rows, q_heads, kv_heads, dim, group, scale, window, sinks,
                                           splits, out, *strides, ws, ws_bytes, None, None)


@pytest.mark.parametrize("wrong", [
    dict(arena=None), dict(table=None), dict(q=None), dict(out=None), dict(ws=None), dict(arena=A8), dict(q=A8),
    dict(ws=A8), dict(arena_bytes=-1), dict(scale=NAN), dict(scale=INF), dict(strides=(4100, 1024, 128)),
    dict(strides=(4096, 1028, 128)), dict(strides=(4096, 1024, 132)), dict(table_stride=63), dict(uniform=-1),
    dict(batch=0), dict(batch=65536), dict(rows=0), dict(q_heads=12), dict(kv_heads=0), dict(columns=-1),
    dict(sinks=-1), dict(window=0, sinks=1), dict(window=-1, sinks=1)],
    ids=lambda w: "-".join(f"{k}" for k in w))
@pytest.mark.parametrize("large", [False, True], ids=["decode", "tiles"])
def test_chunk_entry_refuses(wrong, large):
    size = dict(rows=512, table_stride=4096, columns=4096) if large else {}
    if large and "table_stride" in wrong:
        wrong = dict(table_stride=4095)
    assert _chunk(**{**size, **wrong}) == INVALID


def test_chunk_entry_refuses_geometry():
    assert _chunk(dim=96) == UNSUPPORTED and _chunk(group=48) == UNSUPPORTED and _chunk(group=16) == UNSUPPORTED
    assert _chunk(dim=64, group=2048) == UNSUPPORTED
    assert _chunk(rows=1 << 28) == UNSUPPORTED                                     # rows of a call: 31 bits
    assert _chunk(columns=(1 << 26) + 1, table_stride=1 << 27) == UNSUPPORTED      # positions: 30 bits
    size = _lib.load().akv_chunk_workspace_bytes
    assert size(0, 1, 16, 8, 128, 64, 0, 0, 4) == -1 and size(1, 0, 16, 8, 128, 64, 0, 0, 4) == -1
    assert size(1, 1, 12, 8, 128, 64, 0, 0, 4) == -1 and size(1, 1, 16, 8, 96, 64, 0, 0, 4) == -1
    assert size(1, 1, 16, 8, 128, -1, 0, 0, 4) == -1 and size(1, 1, 16, 8, 128, 64, 0, 3, 4) == -1
    assert size(1, 1, 16, 8, 128, 64, 9, -1, 4) == -1


def test_fork_entry_refuses():
    def fork(table=A, layer_stride=128, seq_stride=64, layers=2, batch=2, columns=64, tokens=None, uniform=10,
             parents=A, children=3, out=VP(0x100000), arena=A, arena_bytes=1 << 20, heads=2, dim=128, group=64):
        return _lib.load().akv_fork_pages(table, layer_stride, seq_stride, layers, batch, columns, tokens, uniform,
                                          parents, children, None, out, arena, arena_bytes, heads, dim, group, None,
                                          None)

    for wrong in (dict(table=None), dict(parents=None), dict(out=None), dict(arena=None), dict(arena=A8),
                  dict(layers=0), dict(batch=0), dict(children=-1), dict(columns=-1), dict(arena_bytes=-1),
                  dict(seq_stride=63), dict(layer_stride=-1), dict(uniform=-1), dict(heads=0),
                  dict(out=VP(0x1000 + 8 * 255))):  # the table's last entry
        assert fork(**wrong) == INVALID, wrong
    assert fork(dim=96) == UNSUPPORTED and fork(group=48) == UNSUPPORTED
    assert fork(children=0) == OK and fork(columns=0) == OK  # nothing to write: no launch


def test_compact_entry_refuses():
    size = _lib.load().akv_compact_workspace_bytes
    page = 2 * P.record_bytes(128, 64, 4)
    room = size(10, 64 * page, 2, 128, 64)
    assert room > 0 and size(-1, page, 2, 128, 64) == -1 and size(10, -1, 2, 128, 64) == -1
    assert size(1 << 31, page, 2, 128, 64) == -1 and size(1, page, 2, 96, 64) == -1 and size(1, page, 0, 128, 64) == -1

    def compact(table=A, entries=10, out=VP(0x2000), arena=VP(0x100000), arena_bytes=64 * page, into=VP(0x1000000),
                into_bytes=4 * page, slots=(0, 4, 0, 0, 0, 0), heads=2, dim=128, group=64, ws=A, ws_bytes=room):
        given = None if slots is None else (ctypes.c_int64 * 6)(*slots)
        return _lib.load().akv_compact_pages(table, entries, out, arena, arena_bytes, into, into_bytes, given, heads,
                                             dim, group, ws, ws_bytes, None, None)

    for wrong in (dict(table=None), dict(out=None), dict(arena=None), dict(into=None), dict(slots=None), dict(ws=None),
                  dict(entries=-1), dict(entries=1 << 31), dict(arena=A8), dict(into=A8), dict(ws=A8),
                  dict(arena_bytes=-1), dict(into_bytes=-1), dict(ws_bytes=room - 1), dict(heads=0),
                  dict(into=VP(0x100010)), dict(out=VP(0x1008)),                  # arenas, tables overlap
                  dict(slots=(0, 5, 0, 0, 0, 0)), dict(slots=(8, 1, 0, 0, 0, 0)),  # past the arena, unaligned
                  dict(slots=(-16, 1, 0, 0, 0, 0)), dict(slots=(0, -1, 0, 0, 0, 0)),
                  dict(slots=(0, 1 << 62, 0, 0, 0, 0))):
        assert compact(**wrong) == INVALID, wrong
    assert compact(dim=96) == UNSUPPORTED and compact(group=16) == UNSUPPORTED
    assert compact(entries=0) == OK


def test_python_refusals_before_a_device():
    pool = P.PagePool(2, 128, group=64, pages={16: 4}, device="cpu")
    batch = P.PagedBatch.over(pool, torch.zeros(1, 4, dtype=torch.int64), tokens=64)
    query = torch.zeros(1, 4, 3, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        akv.chunk_attention(query, batch, .1)
    for shape in ((4, 3, 128), (2, 4, 3, 128), (1, 4, 3, 64)):
        with pytest.raises(ValueError, match="batch, heads, rows, head_dim"):
            akv.chunk_attention(torch.zeros(shape, dtype=torch.float16), batch, .1)
    with pytest.raises(ValueError, match="CUDA"):
        akv.packed_attention(query[:, :, :1], batch, .1, window=4)
    for table in (batch.table, batch.table.to(torch.int32)):
        with pytest.raises(ValueError, match="page table"):
            akv.fork_pages(pool, table, torch.zeros(1, dtype=torch.int64))
        with pytest.raises(ValueError, match="page table"):
            akv.compact_pages(pool, table, P.PagePool(2, 128, group=64, pages={16: 4}, device="cpu"))


def test_pool_over_refusals():
    arena = torch.zeros(1 << 16, dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA"):
        akv.PagePool.over(arena, 2, 128)
    for kw in (dict(dim=96), dict(dim=128, group=48)):
        with pytest.raises(ValueError, match="geometry"):
            akv.PagePool.over(arena, 2, **kw)


def test_free_slots_stack_over_runs():
    s = P._FreeSlots()
    s.add_run(160, 16, 4)
    s.add_run(1000, 10, 2)
    s.add_run(7, 7, 0)
    assert len(s) == 6 and not s.untouched(160, 6)
    assert s.take(0).tolist() == []
    assert s.take(2).tolist() == [160, 176]
    s.give(np.array([160, 176]))
    assert s.take(3).tolist() == [176, 160, 192]  # last in first out, then the runs
    assert s.take(3).tolist() == [208, 1000, 1010] and len(s) == 0
    s.give(np.arange(100))
    assert len(s) == 100 and s.take(100).tolist() == list(range(99, -1, -1))

    fresh = P._FreeSlots()
    assert fresh.untouched(0, 0)
    fresh.add_run(64, 32, 5)
    assert fresh.untouched(64, 5) and not fresh.untouched(0, 5)
    fresh.skip(2)
    assert not fresh.untouched(64, 5) and fresh.take(3).tolist() == [128, 160, 192] and len(fresh) == 0


def test_pool_slots_and_growth():
    pool = P.PagePool(2, 64, group=64, pages={16: 2, 4: 3}, device="cpu")
    assert pool.untouched
    big, small = pool.page_bytes[16], pool.page_bytes[4]
    assert pool.alloc_many(4, 3).tolist() == [2 * big + i * small for i in range(3)]
    with pytest.raises(MemoryError):
        pool.alloc(4)
    with pytest.raises(MemoryError):
        pool.alloc_many(16, 3)
    assert pool.free_slots(16) == 2 and not pool.untouched
    before = pool.nbytes
    pool.reserve(4, 5)
    assert pool.nbytes == before + 64 * small and pool.alloc(4) == before
    shuffled = P.PagePool(2, 64, group=64, pages={16: 50}, device="cpu", shuffle_seed=3)
    assert sorted(shuffled.alloc_many(16, 50).tolist()) == [i * big for i in range(50)]


def test_store_refuses_before_any_change():
    store = live.PagedKVStore(2, 3, 2, 64, 64, device="cpu")
    for parents in ([], [[0]], [3], [-1], [0.5], [True, False, True]):
        with pytest.raises(ValueError, match="parents"):
            store.fork(parents)
    for tokens in (-1, 1):
        with pytest.raises(ValueError, match="crop"):
            store.crop(tokens)
    store.crop(0)  # nothing to drop
    store.lengths[1] = 5
    with pytest.raises(ValueError, match="between steps"):
        store.fork([0])
    with pytest.raises(ValueError, match="between steps"):
        store.crop(0)
    assert store.batch == 3 and store.tables.shape == (2, 3, 4)

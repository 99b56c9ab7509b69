"""Forking and compacting pages: every byte and every table entry."""

import numpy as np
import pytest
import torch

import anchorkv_b200 as akv
from anchorkv_b200 import _lib
from anchorkv_b200 import pool as P

pytestmark = pytest.mark.gpu


def _pool(cuda, heads, dim, group, pages, seed):
    """A pool whose arena holds random bytes."""
    pool = P.PagePool(heads, dim, group=group, pages=pages, device=cuda, shuffle_seed=seed)
    g = torch.Generator(device=cuda).manual_seed(seed)
    pool.arena.copy_(torch.randint(0, 256, (pool.nbytes,), dtype=torch.uint8, device=cuda, generator=g))
    return pool


def _page(pool, desc):
    bits, _, offset = P.decode(int(desc))
    return pool.arena[offset:offset + pool.page_bytes[bits]]


GEOMETRIES = [(8, 128, 64), (1, 64, 32), (3, 64, 1024), (2, 128, 2048)]


@pytest.mark.parametrize("heads,dim,group", GEOMETRIES)
@pytest.mark.parametrize("tokens", [1, 15, 16, 17, 47, 64])
def test_fork_copies_the_half_filled_page_and_shares_the_rest(cuda, heads, dim, group, tokens):
    layers, batch, columns = 3, 3, 6
    parents = [2, 0, 0, 2, 2]
    rng = np.random.default_rng(tokens)
    used = -(-tokens // 16)
    n = layers * batch * used
    pool = _pool(cuda, heads, dim, group, {16: n + layers * 5, 8: n, 4: n}, tokens)
    table = np.zeros((layers, batch, columns), np.int64)
    for layer in range(layers):
        for b in range(batch):
            for j in range(used):
                last = j == used - 1
                bits = 16 if last else int(rng.choice([16, 8, 4]))
                table[layer, b, j] = P.encode(bits, (tokens - 1) % 16 + 1 if last else 16, pool.alloc(bits))
    table[0, 0, 0] = table[0, 0, 0] if used == 1 else 0  # an evicted page stays one
    fresh = np.zeros((layers, 5), np.int64)
    for layer in range(layers):
        for child in (2, 3, 4):  # children 0 and 1 go on with their parents' own pages
            fresh[layer, child] = P.encode(16, 1, pool.alloc(16))
    before = pool.arena.clone()
    t = torch.from_numpy(table).to(cuda)
    got = akv.fork_pages(pool, t, torch.tensor(parents, device=cuda), torch.from_numpy(fresh).to(cuda), tokens=tokens)
    want = table[:, parents].copy()
    expected = before.clone()
    if tokens % 16:
        for layer in range(layers):
            for child in (2, 3, 4):
                old, new = int(want[layer, child, used - 1]), int(fresh[layer, child])
                want[layer, child, used - 1] = (new >> 8 << 8) | (old & 255)
                size = pool.page_bytes[16]
                expected[new >> 8:(new >> 8) + size] = before[old >> 8:(old >> 8) + size]
    assert torch.equal(got.cpu(), torch.from_numpy(want))
    assert torch.equal(pool.arena, expected)
    assert torch.equal(t.cpu(), torch.from_numpy(table))
    assert akv.take_device_status(cuda) == 0
    # without fresh slots everything is shared; a layer of a strided table forks alone
    assert torch.equal(akv.fork_pages(pool, t, torch.tensor(parents, device=cuda)).cpu(),
                       torch.from_numpy(table[:, parents]))
    view = t[1, :, :used]
    assert torch.equal(akv.fork_pages(pool, view, torch.tensor([1], device=cuda)).cpu(),
                       torch.from_numpy(table[1, [1], :used]))


def test_fork_takes_each_parents_own_count_and_refuses_bad_entries_on_the_device(cuda):
    pool = _pool(cuda, 2, 128, 64, {16: 10, 8: 2, 4: 2}, 5)
    slot = lambda bits, n=16: P.encode(bits, n, pool.alloc(bits))  # noqa: E731
    table = np.array([[slot(16), slot(16, 3)], [slot(16, 9), 0], [slot(4), slot(8, 2)]])
    tokens = torch.tensor([19, 9, 18], dtype=torch.int32, device=cuda)
    fresh = np.array([slot(16), slot(16), slot(16), 0])
    t, parents = torch.from_numpy(table).to(cuda), torch.tensor([0, 1, 2, 1], device=cuda)
    before = pool.arena.clone()
    got = akv.fork_pages(pool, t, parents, torch.from_numpy(fresh).to(cuda), tokens=tokens).cpu().numpy()
    assert got[0].tolist() == [table[0, 0], (fresh[0] >> 8 << 8) | (table[0, 1] & 255)]
    assert got[1].tolist() == [(fresh[1] >> 8 << 8) | (table[1, 0] & 255), 0]
    assert got[2].tolist() == table[2].tolist()  # an FP16 slot cannot take an INT8 page: it stays shared
    assert got[3].tolist() == table[1].tolist()
    assert akv.take_device_status(cuda) == _lib.DEV_BAD_DESCRIPTOR
    for child, old in ((0, table[0, 1]), (1, table[1, 0])):
        assert torch.equal(_page(pool, fresh[child]), before[old >> 8:(old >> 8) + pool.page_bytes[16]])
    out = akv.fork_pages(pool, t, torch.tensor([3, 1, -1], device=cuda)).cpu().numpy()
    assert out[0].tolist() == [0, 0] and out[2].tolist() == [0, 0] and out[1].tolist() == table[1].tolist()
    assert akv.take_device_status(cuda) == _lib.DEV_BAD_PARENT


@pytest.mark.parametrize("heads,dim,group", GEOMETRIES)
@pytest.mark.parametrize("entries", [1, 31, 1024, 1025, 5000])
def test_compaction_moves_each_page_once_in_table_order(cuda, heads, dim, group, entries):
    rng = np.random.default_rng(entries + heads)
    counts = {16: entries // 6 + 1, 8: entries // 5 + 1, 4: entries // 4 + 1}
    pool = _pool(cuda, heads, dim, group, counts, entries)
    pages = [P.encode(b, int(rng.integers(1, 17)), int(o)) for b in (16, 8, 4) for o in pool.alloc_many(b, counts[b])]
    table = np.array(pages)[rng.integers(0, len(pages), entries)]  # some shared, some left out
    table[rng.random(entries) < .1] = 0
    live = {b: len({d >> 8 for d in table.tolist() if P.decode(d)[0] == b}) for b in (16, 8, 4)}
    into = P.PagePool(heads, dim, group=group, pages={b: live[b] + 2 for b in live}, device=cuda)
    t = torch.from_numpy(table).to(cuda)
    before = pool.arena.clone()
    got = akv.compact_pages(pool, t, into, live)
    place, want = {}, []
    taken = dict(into.base)
    expected = torch.zeros_like(into.arena)
    for d in table.tolist():
        bits, _, off = P.decode(d)
        if bits is None:
            want.append(0)
            continue
        if off not in place:
            place[off] = taken[bits]
            expected[taken[bits]:taken[bits] + pool.page_bytes[bits]] = before[off:off + pool.page_bytes[bits]]
            taken[bits] += pool.page_bytes[bits]
        want.append((place[off] << 8) | (d & 255))
    assert got.cpu().tolist() == want
    assert torch.equal(into.arena, expected) and torch.equal(pool.arena, before)
    assert [into.free_slots(b) for b in (16, 8, 4)] == [2, 2, 2]
    assert into.alloc(16) == into.base[16] + live[16] * into.page_bytes[16]
    assert akv.take_device_status(cuda) == 0


def test_compaction_reports_what_it_cannot_move(cuda):
    pool = _pool(cuda, 2, 64, 64, {16: 3, 8: 3, 4: 3}, 8)
    good = [P.encode(16, 16, int(o)) for o in pool.alloc_many(16, 3)]
    far = P.encode(16, 16, (pool.nbytes + 64) // 16 * 16)
    odd = good[1] + (8 << 8)
    into = P.PagePool(2, 64, group=64, pages={16: 2}, device=cuda)
    t = torch.tensor([[good[0], far, good[1]], [odd, good[0], good[2]]], device=cuda)
    got = akv.compact_pages(pool, t, into).cpu()
    size = pool.page_bytes[16]
    assert got.tolist() == [[P.encode(16, 16, 0), 0, P.encode(16, 16, size)], [0, P.encode(16, 16, 0), 0]]
    assert akv.take_device_status(cuda) == _lib.DEV_BAD_DESCRIPTOR


def test_compaction_keeps_to_the_counted_slots(cuda):
    """More pages than the caller counted: the rest stay behind, and no free slot of the target is written."""
    pool = _pool(cuda, 2, 128, 64, {16: 4, 4: 3}, 3)
    pages = [P.encode(16, 16, int(o)) for o in pool.alloc_many(16, 4)] + [P.encode(4, 7, int(o)) for o in pool.alloc_many(4, 3)]
    for entries in (len(pages), 9000):  # one CTA's plan, and the plan of many
        table = torch.tensor((pages * (entries // len(pages) + 1))[:entries], device=cuda)
        into = P.PagePool(2, 128, group=64, pages={16: 6, 4: 6}, device=cuda)
        got = akv.compact_pages(pool, table, into, {16: 2, 4: 1}).cpu().tolist()
        size = pool.page_bytes
        want = [P.encode(16, 16, 0), P.encode(16, 16, size[16]), 0, 0, P.encode(4, 7, into.base[4]), 0, 0]
        assert got == (want * (entries // len(want) + 1))[:entries]
        assert akv.take_device_status(cuda) == _lib.DEV_BAD_DESCRIPTOR
        assert not into.arena[2 * size[16]:into.base[4]].any() and not into.arena[into.base[4] + size[4]:].any()
        assert [into.free_slots(b) for b in (16, 8, 4)] == [4, 0, 5]

"""A store that decodes, forks, crops, compacts and decodes on, against the token
histories of its sequences; the same through a model's cache and attention route."""

import numpy as np
import pytest
import torch

import anchorkv_b200 as akv
from anchorkv_b200 import live
from anchorkv_b200 import pool as P
from paged_reference import block_values
from position_reference import assert_rows_close, attention_rows_f64

pytestmark = pytest.mark.gpu
HEADS, LAYERS, HQ = 2, 2, 8


class _Histories:
    """The store's twin: per sequence the ids of its tokens, whose keys and values lie in a bank."""

    def __init__(self, cuda, dim, group, archive, recent, protected=(), batch=2, capacity=400):
        gen = torch.Generator().manual_seed(dim + archive)
        self.bank = torch.randn((2, LAYERS, 4000, HEADS, dim), generator=gen).half()
        self.dim, self.group, self.recent, self.protected, self.cuda = dim, group, recent, protected, cuda
        self.store = live.PagedKVStore(LAYERS, batch, HEADS, dim, capacity, group=group, archive_bits=archive,
                                       recent_pages=recent, protected=protected, device=cuda)
        self.tokens = [[] for _ in range(batch)]
        self.used = 0
        self.archive, self.old = archive, -1  # pages up to `old` have left the recent window

    def _new(self, n):
        ids = np.arange(self.used, self.used + len(self.tokens) * n).reshape(len(self.tokens), n)
        self.used += ids.size
        return ids

    def _kv(self, ids, layer):
        k, v = (self.bank[i, layer][torch.from_numpy(ids)].transpose(1, 2).contiguous().to(self.cuda) for i in (0, 1))
        return k, v  # [batch, heads, n, dim]

    def prefill(self, n):
        ids = self._new(n)
        for layer in range(LAYERS):
            self.store.prefill(layer, *self._kv(ids, layer))
        self._grown(ids)

    def append(self, n):
        ids = self._new(n)
        for layer in range(LAYERS):
            self.store.append(layer, *self._kv(ids, layer))
        self._grown(ids)

    def _grown(self, ids):
        self.tokens = [t + i.tolist() for t, i in zip(self.tokens, ids)]
        self.old = max(self.old, len(self.tokens[0]) // 16 - self.recent - 1)

    def fork(self, parents):
        self.store.fork(parents)
        self.tokens = [list(self.tokens[p]) for p in parents]

    def crop(self, n):
        self.store.crop(n)
        self.tokens = [t[:n] for t in self.tokens]
        self.old = min(self.old, n // 16 - 1)

    def values(self, layer):
        """What the pages have to hold by their precision: float64 K, V [batch, heads, tokens, dim]."""
        bits, n = self.store.bits(layer), len(self.tokens[0])
        out = np.zeros((2, len(self.tokens), HEADS, -(-n // 16) * 16, self.dim))
        for b, ids in enumerate(self.tokens):
            for which in (0, 1):
                rows = self.bank[which, layer][ids].numpy().transpose(1, 0, 2)  # [heads, n, dim]
                for j in range(-(-n // 16)):
                    part = rows[:, 16 * j:16 * j + 16]
                    for h in range(HEADS):
                        out[which, b, h, 16 * j:16 * j + part.shape[1]] = (
                            part[h] if bits[b, j] == 16 else block_values(part[h], int(bits[b, j]), self.group, "page"))
        return out[:, :, :, :n]

    def check(self):
        """Bytes, precisions, tables, sharing and slot counts agree with the histories."""
        store, n = self.store, len(self.tokens[0])
        pages = -(-n // 16)
        assert store.lengths == [n] * LAYERS and store.batch == len(self.tokens)
        assert torch.equal(store.tables.cpu(), torch.from_numpy(store._desc))
        assert not store._desc[:, :, pages:].any()
        archived = [j for j in range(min(self.old + 1, pages)) if j not in self.protected]
        want_bits = np.full(pages, 16)
        want_bits[archived] = self.archive
        names = {4: set(), 8: set(), 16: set()}
        for layer in range(LAYERS):
            got = store.dense(layer)
            for g, want in zip(got, self.values(layer)):
                assert np.array_equal(g.double().cpu().numpy(), want)
            bits = store.bits(layer)
            assert pages == 0 or (bits == want_bits).all()
            for b in range(store.batch):
                for j in range(pages):
                    d = int(store._desc[layer, b, j])
                    assert ((d >> 2) & 15) + 1 == min(16, n - 16 * j)
                    # one page for two entries only where the histories agree up to its end
                    for other in range(b):
                        if int(store._desc[layer, other, j]) == d:
                            assert self.tokens[other][:16 * j + 16] == self.tokens[b][:16 * j + 16]
                            assert n >= 16 * j + 16, "a half-filled page has one sequence"
                    names[int(bits[b, j])].add(d >> 8)
        for b_ in (4, 8, 16):  # every slot is free or named
            assert store.pool.free_slots(b_) + len(names[b_]) == store.pool.capacity[b_], b_
        assert store.payload_bytes == sum(
            len(names[b_]) * HEADS * P.algorithmic_record_bytes(self.dim, self.group, b_) for b_ in names)
        assert akv.take_device_status(self.cuda) == 0

    def attend(self, rows, window=None, sinks=0):
        scale, n = self.dim ** -.5, len(self.tokens[0])
        q = torch.randn((len(self.tokens), HQ, rows, self.dim), generator=torch.Generator().manual_seed(n + rows)).half()
        held = np.ones((len(self.tokens), n), bool)
        for layer in range(LAYERS):
            view = self.store.batch_view(layer)
            k, v = self.values(layer)
            want = attention_rows_f64(q, k, v, held, [n] * len(self.tokens), scale, window, sinks)
            if rows == 1:
                out = akv.packed_attention(q.to(self.cuda), view, scale, window=window, sinks=sinks)
                assert_rows_close(out, *want)
            assert_rows_close(akv.chunk_attention(q.to(self.cuda), view, scale, window=window, sinks=sinks), *want)


@pytest.mark.parametrize("dim,group,archive,recent,protected", [
    (128, 64, 4, 1, (1,)), (64, 32, 8, 2, ()), (128, 128, 16, 2, ()), (64, 64, 4, 0, (0, 5))])
def test_operators_together(cuda, dim, group, archive, recent, protected):
    """Beams, drafts and samples over one store: every step checked against the histories."""
    h = _Histories(cuda, dim, group, archive, recent, protected)
    h.prefill(45)
    h.check()
    h.fork([0, 1, 1, 0, 1])        # half-filled pages copied, the rest shared
    h.check()
    h.append(1)
    h.check()
    h.attend(1, window=20, sinks=3)
    h.fork([4, 2, 2])              # beams change places, two sequences end
    h.check()
    h.append(30)                   # pages are archived, shared ones once
    h.check()
    h.attend(30)
    h.append(8)
    h.crop(81)                     # drafts not accepted: inside the last page
    h.check()
    h.append(2)
    h.check()
    h.fork([2, 2, 0, 2, 1, 1])
    h.crop(64)                     # a page border: shared pages end
    h.check()
    h.fork([0, 0, 4])              # nothing half-filled: all is shared
    h.check()
    assert (h.store._desc[:, 0] == h.store._desc[:, 1]).all()
    before = h.store.pool.nbytes
    assert h.store.compact() == before - h.store.pool.nbytes
    h.check()
    assert h.store.pool.free_slots(16) == LAYERS * 3  # every sequence's next page
    h.attend(17, window=33)
    h.append(1)
    h.check()
    h.append(50)
    h.check()
    h.attend(5, window=40, sinks=16)
    h.fork([1])                    # one sequence is left
    h.check()
    assert h.store.compact() > 0
    h.append(100)
    h.check()
    h.attend(100, window=64)
    h.crop(0)
    h.check()
    h.prefill(33)
    h.check()
    h.attend(33)


def test_cropping_into_a_shared_full_page_gives_each_its_own(cuda):
    h = _Histories(cuda, 64, 64, 16, 1)
    h.prefill(80)
    h.fork([0, 0, 1, 0])
    h.check()
    h.crop(70)  # page 4 was full and shared by three
    h.check()
    h.append(3)
    h.check()
    h.attend(3)


def test_archived_pages_are_not_reopened(cuda):
    h = _Histories(cuda, 128, 64, 4, 1)
    h.prefill(100)
    desc, free = h.store._desc.copy(), [h.store.pool.free_slots(b) for b in (4, 8, 16)]
    with pytest.raises(ValueError, match="archived page"):
        h.store.crop(40)
    assert np.array_equal(h.store._desc, desc) and [h.store.pool.free_slots(b) for b in (4, 8, 16)] == free
    h.check()
    h.crop(48)  # its border is fine
    h.check()
    h.append(60)
    h.check()


def test_a_store_of_full_capacity_forks_and_compacts(cuda):
    h = _Histories(cuda, 64, 64, 4, 1, capacity=64)
    h.prefill(64)
    h.fork([1, 0, 1])
    h.check()
    h.store.compact()
    h.check()
    with pytest.raises(ValueError, match="capacity"):
        h.append(1)
    h.used = 3000
    h.crop(63)
    h.append(1)
    h.check()


def test_fork_and_compact_refusals(cuda):
    pool = P.PagePool(HEADS, 128, pages={16: 4, 4: 2}, device=cuda)
    table = torch.zeros((2, 3, 4), dtype=torch.int64, device=cuda)
    one = torch.zeros(1, dtype=torch.int64, device=cuda)
    for t in (table.cpu(), table.int(), table[0, 0]):
        with pytest.raises(ValueError, match="page table"):
            akv.fork_pages(pool, t, one)
    for parents in (one.int(), one.cpu(), one.view(1, 1), torch.zeros(4, dtype=torch.int64, device=cuda)[::2]):
        with pytest.raises(ValueError, match="parents"):
            akv.fork_pages(pool, table, parents)
    fresh = torch.zeros(2, dtype=torch.int64, device=cuda)
    for bad in (fresh[:1], fresh.int(), fresh.cpu()):
        with pytest.raises(ValueError, match="fresh"):
            akv.fork_pages(pool, table, one, bad, tokens=5)
    counts = torch.zeros(3, dtype=torch.int32, device=cuda)
    for tokens in (None, -1, 1 << 31, counts.long(), counts[:2], counts.cpu()):
        with pytest.raises(ValueError, match="token"):
            akv.fork_pages(pool, table, one, fresh, tokens=tokens)
    with pytest.raises(ValueError, match="no sequence"):
        akv.fork_pages(pool, table[:, :0], one)
    assert akv.fork_pages(pool, table, one[:0]).shape == (2, 0, 4)
    assert akv.fork_pages(pool, table[..., :0], one).shape == (2, 1, 0)
    # a transposed table, and one whose rows lie apart, are read as they are
    pages = torch.arange(24, device=cuda).view(4, 3, 2) << 8
    assert torch.equal(akv.fork_pages(pool, pages.permute(2, 1, 0), one), pages.permute(2, 1, 0)[:, :1])
    assert torch.equal(akv.fork_pages(pool, pages.transpose(0, 1)[..., :1], one), pages.transpose(0, 1)[:, :1, :1])

    other = lambda heads=HEADS, dim=128, group=64, **kw: P.PagePool(heads, dim, group=group, pages={16: 4, 4: 2},  # noqa: E731
                                                                    device=cuda, **kw)
    for into in (other(heads=1), other(dim=64), other(group=32)):
        with pytest.raises(ValueError, match="geometry"):
            akv.compact_pages(pool, table, into)
    used, grown = other(), other()
    used.alloc(16)
    grown.reserve(16, 50)
    for into in (used, grown, other(shuffle_seed=1)):
        with pytest.raises(ValueError, match="new one"):
            akv.compact_pages(pool, table, into)
    with pytest.raises(MemoryError):
        akv.compact_pages(pool, table, other(), {16: 5})
    with pytest.raises(ValueError, match="non-negative"):
        akv.compact_pages(pool, table, other(), {4: -1})
    same = P.PagePool.over(pool.arena, HEADS, 128, pages={16: 4, 4: 2})
    with pytest.raises(ValueError, match="of its own"):
        akv.compact_pages(pool, table, same)
    assert akv.compact_pages(pool, table[:, :0], other()).shape == (2, 0, 4)
    into = other()
    assert not akv.compact_pages(pool, table, into, {}).any() and into.untouched
    with pytest.raises(ValueError, match="do not fit"):
        P.PagePool.over(pool.arena, HEADS, 128, pages={16: 5, 4: 2})
    for arena in (pool.arena[8:], pool.arena[::2], pool.arena.view(torch.int8), pool.arena.view(2, -1)):
        with pytest.raises(ValueError, match="16-byte aligned"):
            P.PagePool.over(arena, HEADS, 128)
    with pytest.raises(MemoryError):
        same.reserve(16, 5)
    assert akv.take_device_status(cuda) == 0


def _model(cuda, sliding=None):
    from transformers import Qwen3Config, Qwen3ForCausalLM

    torch.manual_seed(3)
    extra = {} if sliding is None else dict(use_sliding_window=True, sliding_window=sliding, max_window_layers=0)
    config = Qwen3Config(vocab_size=512, hidden_size=512, intermediate_size=512, num_hidden_layers=2,
                         num_attention_heads=8, num_key_value_heads=2, head_dim=64, max_position_embeddings=4096,
                         attn_implementation="sdpa", **extra)
    return Qwen3ForCausalLM(config).to(device=cuda, dtype=torch.float16).eval()


def _prefilled(model, ids, archive, cuda, **kw):
    from transformers import DynamicCache

    cache = DynamicCache()
    model(input_ids=ids, past_key_values=cache, use_cache=True, logits_to_keep=1)
    source = [(layer.keys, layer.values) for layer in cache.layers]
    assert source[0][0].shape[2] == ids.shape[1]
    return live.batched_live_cache(source, max_tokens=512, archive_bits=archive, device=cuda, **kw)


@pytest.mark.parametrize("sliding", [None, 50])
def test_a_model_takes_several_tokens_and_windows(cuda, sliding):
    """Chunks, drafts that are cropped away and single tokens give the logits of the whole
    text at once (the tolerance of the FP16 decode test: the same model arithmetic in fp16)."""
    model = _model(cuda, sliding)
    ids = torch.randint(0, 512, (3, 160), generator=torch.Generator().manual_seed(4)).to(cuda)
    with torch.inference_mode():
        want = model(input_ids=ids, use_cache=False).logits.float()
        for backend in ("packed", "dense"):
            cache = _prefilled(model, ids[:, :70], 16, cuda)
            with live.paged_route(model, cache, backend):
                got = live.decode_step(model, cache, ids[:, 70:107]).float()
                torch.testing.assert_close(got, want[:, 70:107], atol=.05, rtol=.01)
                live.decode_step(model, cache, ids[:, :5])  # drafts
                cache.crop(107)
                got = live.decode_step(model, cache, ids[:, 107]).float()
                torch.testing.assert_close(got, want[:, 107], atol=.05, rtol=.01)
                cache.crop(-1)
                got = live.decode_step(model, cache, ids[:, 107:160]).float()
                torch.testing.assert_close(got, want[:, 107:160], atol=.05, rtol=.01)
            assert cache.get_seq_length() == 160
    assert akv.take_device_status(cuda) == 0


def test_a_models_beams_change_places(cuda):
    """The cache's reordering against fresh caches over the same histories."""
    model = _model(cuda)
    ids = torch.randint(0, 512, (6, 120), generator=torch.Generator().manual_seed(5)).to(cuda)
    with torch.inference_mode():
        cache = _prefilled(model, ids[:2, :75], 4, cuda, recent_pages=1)
        twin = [0, 0, 0, 1, 1, 1]
        cache.batch_repeat_interleave(3)
        fresh = _prefilled(model, ids[twin, :75], 4, cuda, recent_pages=1)
        beams = torch.tensor([3, 1, 1, 0, 5, 5], device=cuda)
        for c, order in ((cache, beams), (fresh, None)):
            with live.paged_route(model, c):
                first = live.decode_step(model, c, ids[:, 80])
                if c is cache:
                    cache.reorder_cache(order)
                    assert cache.store.payload_bytes < fresh.store.payload_bytes
                    kept = first
        torch.testing.assert_close(kept.float(), first.float(), atol=.05, rtol=.01)
        whole = [list(x) for x in (torch.tensor(twin)[beams.cpu()].tolist(), beams.tolist())]
        history = torch.cat([ids[whole[0], :75], ids[whole[1], 80:81]], 1)
        again = _prefilled(model, history[:, :75], 4, cuda, recent_pages=1)
        with live.paged_route(model, again):
            live.decode_step(model, again, history[:, 75])
            want = live.decode_step(model, again, ids[:, 81:95]).float()
        with live.paged_route(model, cache):
            got = live.decode_step(model, cache, ids[:, 81:95]).float()
        torch.testing.assert_close(got, want, atol=.05, rtol=.01)
        cache.batch_select_indices(torch.tensor([4, 0], device=cuda))
        cache.store.compact()
        again.batch_select_indices([4, 0])
        results = []
        for c in (cache, again):
            with live.paged_route(model, c):
                results.append(live.decode_step(model, c, ids[:2, 95]).float())
        torch.testing.assert_close(results[0], results[1], atol=.05, rtol=.01)
    assert akv.take_device_status(cuda) == 0

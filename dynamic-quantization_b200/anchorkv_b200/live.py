"""Batched Hugging Face decode over the packed store.

The reference decodes one sequence at a time: its ``LiveCache`` holds one
``PagedLayer`` per layer and its attention route calls the packed kernel per
layer (``src/anchorkv/colab_experiment.py:92-148``).  That route runs
unchanged on this package: its ``PagedLayer``, ``dense_attention`` and
``packed_attention`` are drop-ins (see the integration notes), and the tests
run the reference's own route, model gate and controlled-decode harness
(``src/anchorkv/benchmark_suite.py:155-264``) with them substituted.

What is new here is a batch: :class:`PagedKVStore` keeps the pages of
``batch`` sequences for every layer in one shared :class:`PagePool`, one page
table per layer that :func:`packed_attention` reads as a ``PagedBatch``:

* prefill packs every layer's prefix in one ``akv_pack_pages`` launch, pages
  older than the recent window straight to the archive precision (pack_page
  rounding, the same bytes the reference's append-then-demote gives);
* a decode step appends each layer's new K/V rows for all sequences in one
  ``akv_append_rows`` launch, which also advances the pages' valid-token
  counts on the device; a fresh page's descriptors reach the table through
  the same launch (one pinned, non-blocking copy of ``batch`` descriptors);
* when a page leaves the recent window it is demoted for all sequences at
  once (``akv_repack_pages``) and its FP16 slots return to the pool; pages of a
  step of several tokens stay FP16 until the step after it, so that its rows
  attend them as written and rejected drafts can be cropped away;
* sequences may share pages: ``fork`` gives every new sequence its parent's
  page tables in one ``akv_fork_pages`` launch over all layers and copies only
  half-filled last pages (beam search, several samples of one prompt), ``crop``
  drops the newest tokens (drafts that were not accepted), ``compact`` moves the
  live pages into an arena of their size.

:func:`batched_live_cache` wraps the store as a transformers ``DynamicCache``
and :func:`paged_route` registers an attention function that decodes through
it, so a batched ``model(...)`` step runs two kernel launches per layer for
attention (decode, merge) plus one append.  Several query tokens per sequence (a
prompt's next chunk, drafted tokens) go through :func:`chunk_attention`, and a
layer's ``sliding_window`` becomes the attention's window.

Model code (``transformers``) is imported lazily: it is needed only when a
model runs.
"""

from __future__ import annotations

from contextlib import contextmanager

import numpy as np
import torch

from . import _lib
from . import pool as P
from .decode import chunk_attention, packed_attention
from .pages import compact_pages, fork_pages

# Name the batched attention function is registered under.
ROUTE = "anchorkv_b200_batched"


class PagedKVStore:
    """Pages of ``batch`` sequences for ``layers`` layers over one shared pool.

    Sequences of a batch advance together (one decode token each per step).
    Pages start FP16; a complete page older than the ``recent_pages`` most
    recent ones is demoted to ``archive_bits`` unless its index is in
    ``protected`` (the lifecycle of the reference's PagedLayer,
    packed_decode.py:135-179, for every sequence at once)."""

    def __init__(self, layers: int, batch: int, heads: int, dim: int, max_tokens: int, *, group: int = 64,
                 archive_bits: int = 4, recent_pages: int = 2, protected=(), device="cuda"):
        if archive_bits not in (4, 8, 16):
            raise ValueError("archive_bits must be 4, 8 or 16")
        if dim not in (64, 128) or not P.group_ok(dim, group) or group > dim:
            raise ValueError("supported geometry: head dim 64/128, group 32/64/128 dividing it")
        self.layers, self.batch, self.heads, self.dim, self.group = layers, batch, heads, dim, group
        self.archive_bits, self.recent_pages = archive_bits, recent_pages
        self.protected = frozenset(int(p) for p in protected)
        self.device = torch.device(device)
        self.capacity = -(-max_tokens // P.BLOCK)
        hot = self.capacity if archive_bits == 16 else min(self.capacity, recent_pages + 2 + len(self.protected))
        sizes = {16: layers * batch * hot}
        if archive_bits != 16:
            sizes[archive_bits] = layers * batch * self.capacity
        self.pool = P.PagePool(heads, dim, group=group, pages=sizes, device=self.device, zero=False)
        self.tables = torch.zeros((layers, batch, self.capacity), dtype=torch.int64, device=self.device)
        self._desc = np.zeros((layers, batch, self.capacity), np.int64)  # host mirror of the tables
        # holder[b, j]: the first sequence that names sequence b's page j (b itself where it is
        # not shared); every layer forks alike, so one map serves them all
        self._holder = np.repeat(np.arange(batch)[:, None], self.capacity, 1)
        self.lengths = [0] * layers
        self._archived = [-1] * layers
        self.demotions = 0

    # ------------------------------------------------------------- writes
    def prefill(self, layer: int, key: torch.Tensor, value: torch.Tensor) -> None:
        """Store a prefix ``[batch, heads, tokens, dim]`` of an empty layer."""
        if self.lengths[layer]:
            raise ValueError("prefill needs an empty layer; decode steps go through append")
        batch, heads, tokens, dim = key.shape
        if (batch, heads, dim) != (self.batch, self.heads, self.dim) or value.shape != key.shape:
            raise ValueError("key/value geometry does not match the store")
        if tokens > self.capacity * P.BLOCK:
            raise ValueError("cache geometry or capacity exceeded")
        _lib.require_cuda(key, "key")
        if not any(self.lengths):  # an emptied store: nothing is shared any more
            self._holder[:] = np.arange(batch)[:, None]
        status, stream = _lib.status_ptr(self.device), _lib.stream_of(self.device)  # raises before any change
        n = -(-tokens // P.BLOCK)
        eligible = tokens // P.BLOCK - self.recent_pages  # complete pages older than the recent window
        bits = np.full(n, 16)
        if self.archive_bits != 16:
            old = np.arange(n) < eligible
            old[list(p for p in self.protected if p < n)] = False
            bits[old] = self.archive_bits
        ntok = np.minimum(P.BLOCK, tokens - P.BLOCK * np.arange(n))
        desc = np.zeros((batch, n), np.int64)
        for b_ in (16, 8, 4):
            cols = np.nonzero(bits == b_)[0]
            if cols.size:
                self.pool.reserve(b_, batch * cols.size)
                offs = self.pool.alloc_many(b_, batch * cols.size).reshape(batch, cols.size)
                desc[:, cols] = P.encode_array(np.full(offs.shape, P.BITS_TO_MODE[b_]),
                                               np.broadcast_to(ntok[cols], offs.shape), offs)
        pad = n * P.BLOCK - tokens
        k = torch.nn.functional.pad(key.half(), (0, 0, 0, pad)).contiguous()
        v = torch.nn.functional.pad(value.half(), (0, 0, 0, pad)).contiguous()
        d = P.to_device(desc.reshape(-1), self.device)
        _lib.call("akv_pack_pages", k.data_ptr(), v.data_ptr(), heads * n * P.BLOCK * dim, n * P.BLOCK * dim, n,
                  batch * n, d.data_ptr(), self.pool.arena.data_ptr(), self.pool.nbytes, heads, dim, self.group,
                  _lib.SEM_PAGE, status, stream)
        self.tables[layer, :, :n].copy_(d.view(batch, n))
        self.demotions += batch * int((bits != 16).sum())  # the reference appends, then demotes, these pages
        self._desc[layer, :, :n] = desc
        self.lengths[layer] = tokens
        self._archived[layer] = max(eligible - 1, -1)

    def append(self, layer: int, key: torch.Tensor, value: torch.Tensor, *, archive: bool = True) -> None:
        """Append ``[batch, heads, rows, dim]`` decode-step K/V to every sequence.

        Pages that leave the recent window are demoted within the call.  With
        ``archive=False`` only those that earlier steps pushed out of it are; the
        pages that this step completes or pushes out keep FP16 until the layer's
        next append, so that the step's rows attend them as they were written and
        ``crop`` can take the step back.  FP16 slots grow to hold the step."""
        if key.shape != value.shape or key.shape[0] != self.batch or key.shape[1] != self.heads \
                or key.shape[-1] != self.dim:
            raise ValueError("key/value geometry does not match the store")
        rows = key.shape[2]
        if self.lengths[layer] + rows > self.capacity * P.BLOCK:
            raise ValueError("cache geometry or capacity exceeded")
        key, value = P.as_fp16_rows(key), P.as_fp16_rows(value)
        status, stream = _lib.status_ptr(self.device), _lib.stream_of(self.device)
        if not archive:
            self._archive(layer)
            self.pool.reserve(16, self.batch * (-(-(self.lengths[layer] + rows) // P.BLOCK) - self.pages(layer)))
        done = 0
        while done < rows:
            page, row = divmod(self.lengths[layer], P.BLOCK)
            take = min(P.BLOCK - row, rows - done)
            fresh = None
            if row == 0:  # a new FP16 page for every sequence
                self.pool.reserve(16, self.batch)
                offs = self.pool.alloc_many(16, self.batch)
                new = P.encode_array(np.full(self.batch, _lib.MODE_FP16), np.full(self.batch, take), offs)
                fresh = P.to_device(new, self.device)
                self._desc[layer, :, page] = new
                self._holder[:, page] = np.arange(self.batch)
            else:
                self._desc[layer, :, page] = (self._desc[layer, :, page] & ~np.int64(15 << 2)) | ((row + take - 1) << 2)
            k, v = key[:, :, done:done + take], value[:, :, done:done + take]
            tbl = self.tables[layer]
            _lib.call("akv_append_rows", k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2),
                      self.batch, take, row, tbl.data_ptr(), tbl.stride(0), page,
                      None if fresh is None else fresh.data_ptr(), self.pool.arena.data_ptr(), self.pool.nbytes,
                      self.heads, self.dim, status, stream)
            self.lengths[layer] += take
            done += take
            if archive:
                self._archive(layer)

    def _archive(self, layer: int) -> None:
        last = self.lengths[layer] // P.BLOCK - self.recent_pages - 1
        pages = [p for p in range(self._archived[layer] + 1, last + 1) if p not in self.protected]
        if self.archive_bits == 16 or not pages:
            self._archived[layer] = max(self._archived[layer], last)
            return
        status, stream = _lib.status_ptr(self.device), _lib.stream_of(self.device)  # raises before any change
        self._archived[layer] = max(self._archived[layer], last)
        holder = self._holder[:, pages]
        own = holder == np.arange(self.batch)[:, None]  # a shared page is repacked once
        src = self._desc[layer][:, pages][own]
        self.pool.reserve(self.archive_bits, src.size)
        offs = self.pool.alloc_many(self.archive_bits, src.size)
        dst = np.zeros(holder.shape, np.int64)
        dst[own] = P.encode_array(np.full(src.size, P.BITS_TO_MODE[self.archive_bits]), ((src >> 2) & 15) + 1, offs)
        packed = dst[own]
        dst = dst[holder, np.arange(len(pages))]  # every sequence's entry names its holder's page
        s_dev, d_dev = P.to_device(src, self.device), P.to_device(packed, self.device)
        entries = d_dev.view(dst.shape) if own.all() else P.to_device(dst, self.device)
        _lib.call("akv_repack_pages", s_dev.data_ptr(), d_dev.data_ptr(), src.size, self.pool.arena.data_ptr(),
                  self.pool.nbytes, self.heads, self.dim, self.group, _lib.SEM_PAGE, status, stream)
        self.tables[layer].index_copy_(1, P.to_device(pages, self.device), entries)
        self._desc[layer][:, pages] = dst
        self.pool.free_many(16, src >> 8)  # stream order: later writes to these slots follow the repack
        self.demotions += src.size

    # ------------------------------------------------- sequences and pages
    def _even_length(self, what: str) -> int:
        if len(set(self.lengths)) > 1:
            raise ValueError(f"{what} works between steps: the layers hold {sorted(set(self.lengths))} tokens")
        return self.lengths[0]

    def _free_pages(self, sequences: np.ndarray, columns: np.ndarray) -> None:
        """Return the pages (sequences[i], columns[i]) of every layer to the pool."""
        desc = self._desc[:, sequences, columns]
        for bits, mode in P.BITS_TO_MODE.items():
            self.pool.free_many(bits, desc[(desc & 3) == mode] >> 8)

    def fork(self, parents) -> None:
        """Make the batch the sequences that continue ``parents`` (indices of
        present sequences, any number of each; the new batch may be larger or
        smaller).  A child shares its parent's pages; where several children
        continue one half-filled page, all but the first get a copy of it (one
        launch over all layers).  Pages that no child holds return to the pool."""
        length = self._even_length("fork")
        index = np.asarray(parents.tolist() if isinstance(parents, torch.Tensor) else parents)
        if index.ndim != 1 or index.size == 0 or index.dtype.kind not in "iu":
            raise ValueError("parents must be a non-empty list of sequence indices")
        if (index < 0).any() or (index >= self.batch).any():
            raise ValueError(f"parents must lie in [0, {self.batch})")
        index = index.astype(np.int64)
        _lib.raise_pending(self.device)  # an earlier kernel's error, before any change
        children, n = index.size, self.pages()
        columns = np.arange(n)
        held = self._holder[index, :n]  # [children, n]: the old holder of each child's page
        first = np.full((self.batch, n), children)
        for child in range(children - 1, -1, -1):  # the first child of each old page wins
            first[held[child], columns] = child
        holder = np.repeat(np.arange(children)[:, None], self.capacity, 1)
        holder[:, :n] = first[held, columns]
        last = length // P.BLOCK
        copied = np.nonzero(holder[:, last] != np.arange(children))[0] if length % P.BLOCK else np.zeros(0, np.int64)
        desc = self._desc[:, index]
        fresh = None
        if copied.size:
            self.pool.reserve(16, self.layers * copied.size)
            offs = self.pool.alloc_many(16, self.layers * copied.size).reshape(self.layers, copied.size)
            new = np.zeros((self.layers, children), np.int64)
            new[:, copied] = (offs << 8) | (desc[:, copied, last] & 255)
            desc[:, copied, last] = new[:, copied]
            holder[copied, last] = copied
            fresh = P.to_device(new, self.device)
        tables = fork_pages(self.pool, self.tables, P.to_device(index, self.device), fresh, tokens=length)
        gone = (self._holder[:, :n] == np.arange(self.batch)[:, None]) & (first == children)
        self._free_pages(*np.nonzero(gone))  # stream order: later writes to these slots follow the copies
        self.batch, self.tables, self._desc, self._holder = children, tables, desc, holder

    def crop(self, tokens: int) -> None:
        """Keep the first ``tokens`` tokens of every sequence; the pages behind
        them return to the pool.  A cut inside a page needs that page in FP16 (the
        next tokens are written there), and gives each sequence its own copy of
        it where it was shared."""
        length = self._even_length("crop")
        if not 0 <= tokens <= length:
            raise ValueError(f"crop must keep between 0 and {length} tokens")
        if tokens == length:
            return
        _lib.raise_pending(self.device)  # an earlier kernel's error, before any change
        keep, old = -(-tokens // P.BLOCK), self.pages()
        own = self._holder == np.arange(self.batch)[:, None]
        if tokens % P.BLOCK:
            last = keep - 1
            if ((self._desc[:, :, last] & 3) != _lib.MODE_FP16).any():
                raise ValueError(f"token {tokens} lies inside an archived page: crop to a page's first token")
            self._reopen(last, tokens, own[:, last])
        sequences, columns = np.nonzero(own[:, keep:old])
        self._free_pages(sequences, columns + keep)
        self._desc[:, :, keep:] = 0
        self._holder[:, keep:] = np.arange(self.batch)[:, None]
        self.tables[:, :, keep:].zero_()
        for layer in range(self.layers):
            self.lengths[layer] = tokens
            self._archived[layer] = min(self._archived[layer], tokens // P.BLOCK - 1)

    def _reopen(self, page: int, tokens: int, own: np.ndarray) -> None:
        """Make ``page`` the half-filled last page of every sequence, a copy where it is shared."""
        fresh = np.zeros((self.layers, self.batch), np.int64)
        count = (tokens % P.BLOCK - 1) << 2
        self._desc[:, :, page] = (self._desc[:, :, page] & ~np.int64(15 << 2)) | count
        self.tables[:, :, page].copy_(P.to_device(self._desc[:, :, page], self.device))
        if own.all():
            return
        copied = np.nonzero(~own)[0]
        self.pool.reserve(16, self.layers * copied.size)
        offs = self.pool.alloc_many(16, self.layers * copied.size).reshape(self.layers, copied.size)
        fresh[:, copied] = (offs << 8) | (self._desc[:, copied, page] & 255)
        self.tables = fork_pages(self.pool, self.tables, P.to_device(np.arange(self.batch), self.device),
                                 P.to_device(fresh, self.device), tokens=tokens)
        self._desc[:, copied, page] = fresh[:, copied]
        self._holder[copied, page] = copied

    def compact(self) -> int:
        """Move the live pages into an arena of their number, with FP16 room for
        every sequence's next page, and drop the old arena.  Returns the bytes by
        which the arena shrank (negative where that room is more than was free)."""
        _lib.raise_pending(self.device)  # an earlier kernel's error, before any change
        n = max(self.pages(layer) for layer in range(self.layers))
        own = self._holder[:, :n] == np.arange(self.batch)[:, None]
        modes = self._desc[:, :, :n] & 3
        live = {bits: int(((modes == mode) & own).sum()) for bits, mode in P.BITS_TO_MODE.items()}
        room = dict(live)
        room[16] += self.layers * self.batch
        into = P.PagePool(self.heads, self.dim, group=self.group, pages=room, device=self.device, zero=False)
        tables = compact_pages(self.pool, self.tables, into, live)
        # the same order on the host: pages by first naming, (layer, sequence, column), within a precision
        desc = np.zeros_like(self._desc)
        for bits, mode in P.BITS_TO_MODE.items():
            mine = (modes == mode) & own
            place = into.base[bits] + np.arange(int(mine.sum()), dtype=np.int64) * into.page_bytes[bits]
            desc[:, :, :n][mine] = (place << 8) | (self._desc[:, :, :n][mine] & 255)
        desc[:, :, :n] = desc[:, self._holder[:, :n], np.arange(n)]
        shrunk = self.pool.nbytes - into.nbytes
        self.pool, self.tables, self._desc = into, tables, desc
        return shrunk

    # -------------------------------------------------------------- reads
    def pages(self, layer: int = 0) -> int:
        return -(-self.lengths[layer] // P.BLOCK)

    def batch_view(self, layer: int) -> P.PagedBatch:
        """Layer ``layer``'s page table for :func:`packed_attention` (query ``[batch, Hq, 1, D]``)."""
        return P.PagedBatch.over(self.pool, self.tables[layer, :, :self.pages(layer)], tokens=self.lengths[layer])

    def bits(self, layer: int = 0) -> np.ndarray:
        """Precision of every page, ``[batch, pages]``."""
        modes = self._desc[layer, :, :self.pages(layer)] & 3
        return np.vectorize(P.MODE_TO_BITS.get, otypes=[np.int64])(modes)

    @property
    def payload_bytes(self) -> int:
        """Payload + scale bytes of every page, a shared page counted once (QuantizedPage.nbytes of K and V,
        packed_decode.py:28-32)."""
        total = 0
        own = self._holder == np.arange(self.batch)[:, None]
        for layer in range(self.layers):
            bits = self.bits(layer)[own[:, :self.pages(layer)]]
            for b_ in (16, 8, 4):
                per_page = self.heads * (2 * P.BLOCK * self.dim * b_ // 8 +
                                         (0 if b_ == 16 else 4 * P.BLOCK * self.dim // self.group))
                total += int((bits == b_).sum()) * per_page
        return total

    @property
    def resident_bytes(self) -> int:
        """Payload + scales + the page tables (8 bytes per page slot)."""
        return self.payload_bytes + self.tables.numel() * 8

    def dense(self, layer: int) -> tuple[torch.Tensor, torch.Tensor]:
        """fp16 K, V ``[batch, heads, tokens, dim]`` as the pages hold them."""
        n = self.pages(layer)
        desc = self.tables[layer, :, :n].contiguous()
        k = torch.empty((self.heads, self.batch * n * P.BLOCK, self.dim), dtype=torch.float16, device=self.device)
        v = torch.empty_like(k)
        if n:
            _lib.call("akv_unpack_pages", desc.data_ptr(), self.batch * n, self.pool.arena.data_ptr(),
                      self.pool.nbytes, self.heads, self.dim, self.group, k.data_ptr(), v.data_ptr(), _lib.DTYPE_F16,
                      _lib.status_ptr(self.device), _lib.stream_of(self.device))
        shape = (self.heads, self.batch, n * P.BLOCK, self.dim)
        length = self.lengths[layer]
        return (k.view(shape).transpose(0, 1)[:, :, :length], v.view(shape).transpose(0, 1)[:, :, :length])

    def report(self) -> dict:
        return {"resident_bytes": self.resident_bytes, "payload_bytes": self.payload_bytes,
                "demotions": self.demotions, "tokens": self.lengths[0], "batch": self.batch}


_CACHE_CLASS = None


def batched_live_cache(source, *, max_tokens: int, group: int = 64, archive_bits: int = 4, recent_pages: int = 2,
                       protected=(), device="cuda"):
    """A transformers ``DynamicCache`` over a :class:`PagedKVStore`, prefilled
    from ``source`` = [(key, value)] per layer, each ``[batch, heads, tokens,
    dim]`` (e.g. a stock cache's layers after a batched prefill).  ``update``
    appends the step's keys/values to the store and hands them back unchanged;
    the routed attention (:func:`paged_route`) reads the store."""
    global _CACHE_CLASS
    if _CACHE_CLASS is None:
        from transformers import DynamicCache

        class BatchedLiveCache(DynamicCache):
            def __init__(self, store: PagedKVStore):
                super().__init__()
                self.store = store

            def get_seq_length(self, layer_idx=0):
                return self.store.lengths[layer_idx]

            def update(self, key_states, value_states, layer_idx, cache_kwargs=None):
                self.store.append(layer_idx, key_states, value_states, archive=key_states.shape[2] == 1)
                return key_states, value_states

            # the model library's names for what the store does (beam search, samples, drafts)
            def reorder_cache(self, beam_idx):
                self.store.fork(beam_idx)

            def batch_repeat_interleave(self, repeats):
                self.store.fork(np.repeat(np.arange(self.store.batch), repeats))

            def batch_select_indices(self, indices):
                self.store.fork(indices)

            def crop(self, max_length):
                length = self.store.lengths[0]
                keep = length + max_length if max_length < 0 else min(max_length, length)
                self.store.crop(keep)

            def report(self):
                return self.store.report()

        _CACHE_CLASS = BatchedLiveCache
    key0 = source[0][0]
    store = PagedKVStore(len(source), key0.shape[0], key0.shape[1], key0.shape[-1], max_tokens, group=group,
                         archive_bits=archive_bits, recent_pages=recent_pages, protected=protected, device=device)
    for layer, (key, value) in enumerate(source):
        store.prefill(layer, key.to(device), value.to(device))
    return _CACHE_CLASS(store)


def _route_mask(q_length: int, attention_mask=None, **_) -> None:
    """The route's mask function (the model library calls it once per kind of layer
    and forward): there is no mask to make.  Only here does a padding mask
    ``[batch, tokens]`` show itself; several rows whose padding would be attended are refused."""
    if q_length > 1 and attention_mask is not None and not bool(attention_mask.all()):
        raise ValueError("the paged route attends every stored token up to a row's own: a padding mask with hidden "
                         "tokens cannot be honoured for several query tokens")


@contextmanager
def paged_route(model, cache, backend: str = "packed"):
    """Route ``model``'s attention over ``cache``'s pages for the duration of the
    block: ``backend="packed"`` decodes one query token per sequence with
    :func:`packed_attention` and several with :func:`chunk_attention`,
    ``"dense"`` dequantises the pages and runs SDPA (the reference route's two
    backends, colab_experiment.py:123-148).  The step's keys and values are in the
    pages by then: those of several tokens in FP16, with the pages that were recent
    before the step; a single token that completes a page demotes the page that
    leaves the recent window first.  A layer with a ``sliding_window`` attends
    that many last positions.

    Rows are causal over every stored token, padding included, and take no other
    mask: a step of several tokens with an explicit mask (``[batch, heads, rows,
    tokens]``) or with a padding mask that hides a token raises ValueError.  A step
    of one token ignores its mask.

    On exit the model's attention implementation is restored and the registry entries
    point back at SDPA, so they keep no reference to the cache."""
    from transformers.masking_utils import ALL_MASK_ATTENTION_FUNCTIONS
    from transformers.modeling_utils import ALL_ATTENTION_FUNCTIONS

    if backend not in ("packed", "dense"):
        raise ValueError("backend must be 'packed' or 'dense'")
    sdpa, sdpa_mask = ALL_ATTENTION_FUNCTIONS["sdpa"], ALL_MASK_ATTENTION_FUNCTIONS["sdpa"]
    store = cache.store

    def attention(module, query, key, value, attention_mask, scaling, **kwargs):
        if query.shape[2] > 1 and attention_mask is not None:
            raise ValueError("the paged route's rows are causal: an explicit attention mask cannot be honoured for "
                             "several query tokens")
        view = store.batch_view(module.layer_idx)
        window = kwargs.get("sliding_window")
        if backend == "dense":
            k, v = store.dense(module.layer_idx)
            g = query.shape[1] // k.shape[1]
            rows, length = query.shape[2], k.shape[2]
            mask = None
            if rows > 1 or window is not None:
                at = torch.arange(length - rows, length, device=query.device)[:, None]
                pos = torch.arange(length, device=query.device)
                mask = (pos <= at) & (pos > at - (window or length))
            out = torch.nn.functional.scaled_dot_product_attention(
                query, k.repeat_interleave(g, 1), v.repeat_interleave(g, 1), attn_mask=mask, scale=scaling)
        elif query.shape[2] == 1:
            out = packed_attention(query, view, scaling, window=window)
        else:
            out = chunk_attention(query, view, scaling, window=window)
        return out.transpose(1, 2), None

    previous = model.config._attn_implementation
    ALL_ATTENTION_FUNCTIONS.register(ROUTE, attention)
    ALL_MASK_ATTENTION_FUNCTIONS.register(ROUTE, _route_mask)
    model.config._attn_implementation = ROUTE
    try:
        yield
    finally:
        model.config._attn_implementation = previous
        ALL_ATTENTION_FUNCTIONS.register(ROUTE, sdpa)
        ALL_MASK_ATTENTION_FUNCTIONS.register(ROUTE, sdpa_mask)


def decode_step(model, cache, tokens: torch.Tensor):
    """One batched step.  ``tokens`` ``[batch]`` (a decoded token per sequence, in any
    shape of as many elements) gives last-position logits ``[batch, vocab]``; ``[batch, n]`` (a
    prompt's next chunk, or drafted tokens to verify) logits ``[batch, n, vocab]``."""
    position = cache.get_seq_length()
    rows = tokens.shape[1] if tokens.dim() == 2 and tokens.numel() != cache.store.batch else 1
    out = model(input_ids=tokens.reshape(-1, rows), past_key_values=cache,
                cache_position=torch.arange(position, position + rows, device=tokens.device),
                attention_mask={"full_attention": None, "sliding_attention": None}, use_cache=True,
                logits_to_keep=rows)
    return out.logits if rows > 1 else out.logits[:, -1]

"""Physical page storage: one HBM arena, three record size classes, page tables.

A page is 16 tokens of K and V for every KV head of one (sequence, layer).  It
is stored as ``heads`` head records back to back; a head record is
``[K payload][V payload][K scales][V scales][pad to 16 B]`` with the reference
byte layout for the payload (fp16, int8, or two's-complement nibbles with the
even element low, as ``packed_decode.pack_page`` writes them,
packed_decode.py:48-67) and fp16 scales.  K payloads are row-major; V payloads
hold the same bytes with 16-byte units permuted inside each 128-byte line
(:func:`v_swizzle`), the order the decode kernel reads without shared-memory
bank conflicts.  Pages live at 16-byte aligned offsets so one bulk copy moves a
head record from HBM into shared memory.

A page table entry (descriptor) is an int64: mode in bits 0-1 (0 = skip:
evicted or not visible, 1 = INT4, 2 = INT8, 3 = FP16), valid tokens - 1 in
bits 2-5, byte offset in bits 8-63.

:class:`PagePool` owns the arena and hands out page slots per size class.
Allocation is host bookkeeping (a free-list per class); only descriptors and
payloads live on the device.  :class:`PagedBatch` is the page table of a batch
of sequences of one layer over a shared pool, the batched counterpart of the
reference's batch-one ``PagedLayer`` table (packed_decode.py:122-133).
"""

from __future__ import annotations

from functools import cached_property

import numpy as np
import torch

from . import _lib

BLOCK = 16
BITS_TO_MODE = {4: _lib.MODE_INT4, 8: _lib.MODE_INT8, 16: _lib.MODE_FP16}
MODE_TO_BITS = {v: k for k, v in BITS_TO_MODE.items()}


def record_bytes(dim: int, group: int, bits: int) -> int:
    """Bytes of one (page, KV head) record; mirrors akv_record_bytes."""
    payload = BLOCK * dim * bits // 8
    scales = 0 if bits == 16 else BLOCK * dim // group
    return (2 * payload + 4 * scales + 15) // 16 * 16


def v_swizzle(dim: int, bits: int, offsets) -> np.ndarray:
    """Stored byte offset of each row-major byte offset of a V payload, and
    back (the map is an involution); mirrors ``v_swizzle`` in akv_common.cuh.

    The 16-byte units of a V payload are permuted inside each 128-byte line by
    an XOR keyed on the line's token row, so the decode kernel's V fragment
    loads hit distinct shared-memory banks.  K payloads and scales are
    row-major."""
    o = np.asarray(offsets, np.int64)
    row = dim * bits // 8
    if row == 256:
        key = ((o >> 9) & 1) | (((o >> 10) & 1) << 2)
    elif row == 128:
        key = (o >> 7) & 6
    elif row == 64:
        key = (o >> 6) & 6
    elif row == 32:
        key = (o >> 6) & 2
    else:
        raise ValueError(f"no V payload layout for head_dim {dim} at {bits} bits")
    return o ^ (key << 4)


_V_ORDER: dict = {}


def v_order(dim: int, bits: int, device) -> torch.Tensor:
    """int64 index over one V payload's bytes: ``stored[i] == row_major[order[i]]``
    (and ``row_major[i] == stored[order[i]]``)."""
    key = (dim, bits, str(device))
    if key not in _V_ORDER:
        n = BLOCK * dim * bits // 8
        _V_ORDER[key] = torch.from_numpy(v_swizzle(dim, bits, np.arange(n))).to(device)
    return _V_ORDER[key]


def encode(bits: int | None, ntok: int, offset: int) -> int:
    """Descriptor for a page; ``bits=None`` gives a skip entry."""
    if bits is None:
        return 0
    if not 1 <= ntok <= BLOCK or offset % 16:
        raise ValueError("descriptor needs 1..16 valid tokens and a 16-byte aligned offset")
    return (offset << 8) | ((ntok - 1) << 2) | BITS_TO_MODE[bits]


def encode_array(mode_codes: np.ndarray, ntok: np.ndarray, offsets: np.ndarray) -> np.ndarray:
    """Vectorised :func:`encode`; mode code 0 (skip) yields 0."""
    d = (offsets.astype(np.int64) << 8) | ((ntok.astype(np.int64) - 1) << 2) | mode_codes.astype(np.int64)
    return np.where(mode_codes == 0, 0, d)


def decode(desc: int) -> tuple[int | None, int, int]:
    """(bits or None for skip, valid tokens, byte offset)."""
    mode = desc & 3
    return (MODE_TO_BITS.get(mode), ((desc >> 2) & 15) + 1, desc >> 8)


def to_device(array, device) -> torch.Tensor:
    """An int64 host array on ``device`` through pinned memory, without blocking
    the host (torch keeps the pinned block until the copy has run)."""
    return torch.from_numpy(np.ascontiguousarray(array, np.int64)).pin_memory().to(device, non_blocking=True)


def as_fp16_rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as fp16 with head_dim contiguous, 8-byte aligned rows and strides in
    whole 4-element units (the layout akv_append_rows reads)."""
    t = t.to(torch.float16)
    if t.stride(-1) != 1 or t.data_ptr() % 8 or any(s % 4 for s in t.stride()[:-1]):
        t = t.contiguous()
    return t


def group_ok(dim: int, group: int) -> bool:
    return group in (32, 64, 128, BLOCK * dim)


class _FreeSlots:
    """Free byte offsets of one size class: a stack of returned slots over runs of
    never used ones (first, step, count), so a pool of any size is set up at
    once and slots move by whole arrays.  Slots come back last in, first out;
    then the runs in ascending order."""

    __slots__ = ("_stack", "_top", "_runs", "_in_runs")
    _NONE = np.zeros(0, np.int64)

    def __init__(self):
        self._stack, self._top = self._NONE, 0
        self._runs, self._in_runs = [], 0

    def __len__(self) -> int:
        return self._top + self._in_runs

    def add_run(self, first: int, step: int, count: int) -> None:
        if count > 0:
            self._runs.append([first, step, count])
            self._in_runs += count

    def take(self, n: int) -> np.ndarray:
        out = np.empty(n, np.int64)
        got = min(n, self._top)
        out[:got] = self._stack[self._top - got:self._top][::-1]
        self._top -= got
        while got < n:
            run = self._runs[0]
            k = min(n - got, run[2])
            out[got:got + k] = run[0] + run[1] * np.arange(k, dtype=np.int64)
            run[0] += run[1] * k
            run[2] -= k
            if run[2] == 0:
                self._runs.pop(0)
            got += k
            self._in_runs -= k
        return out

    def untouched(self, first: int, count: int) -> bool:
        """Whether every slot of a class of ``count`` from byte ``first`` is free, in ascending order."""
        if count == 0:
            return len(self) == 0
        return self._top == 0 and len(self._runs) == 1 and self._runs[0][0] == first and self._runs[0][2] == count

    def skip(self, n: int) -> None:
        """Take the first ``n`` slots of an untouched class (no array of them is made)."""
        if n:
            run = self._runs[0]
            run[0], run[2] = run[0] + run[1] * n, run[2] - n
            self._in_runs -= n
            if run[2] == 0:
                self._runs.pop()

    def give(self, offsets: np.ndarray) -> None:
        need = self._top + offsets.size
        if need > self._stack.size:
            grown = np.empty(max(need, 2 * self._stack.size), np.int64)
            grown[:self._top] = self._stack[:self._top]
            self._stack = grown
        self._stack[self._top:need] = offsets
        self._top = need


_PAGE_BYTES: dict = {}


def _page_bytes(heads: int, dim: int, group: int) -> dict:
    """Bytes of a page by precision, one dict per geometry."""
    key = (heads, dim, group)
    if key not in _PAGE_BYTES:
        _PAGE_BYTES[key] = {b: heads * record_bytes(dim, group, b) for b in (4, 8, 16)}
    return _PAGE_BYTES[key]


class PagePool:
    """An arena of page slots in three size classes (FP16 / INT8 / INT4).

    ``pages`` maps bits -> number of slots.  Slots of a class are contiguous;
    ``alloc`` pops from a free list (optionally shuffled, which gives the
    random physical placement of a long-lived shared pool).
    """

    fixed = False  # over(): the arena is the caller's and never grows

    def __init__(self, heads: int, dim: int, *, group: int = 64, pages: dict | None = None,
                 device="cuda", shuffle_seed: int | None = None, zero: bool = True):
        if dim not in (64, 128):
            raise ValueError("supported geometry: head dim 64 or 128")
        if not group_ok(dim, group):
            raise ValueError(f"supported scale groups for head dim {dim}: 32, 64, 128, {BLOCK * dim}")
        self.device = torch.device(device)
        self._lay_out(heads, dim, group, pages)
        if shuffle_seed is not None:
            rng = np.random.default_rng(shuffle_seed)
            for bits in (16, 8, 4):
                slots = np.arange(self.capacity[bits], dtype=np.int64)
                rng.shuffle(slots)
                self._free[bits] = _FreeSlots()
                # the stack gives its last entry first: reverse so slot order is allocation order
                self._free[bits].give((self.base[bits] + slots * self.page_bytes[bits])[::-1])
        alloc = torch.zeros if zero else torch.empty
        self.arena = alloc(self.nbytes, dtype=torch.uint8, device=self.device)

    def _lay_out(self, heads: int, dim: int, group: int, pages: dict | None) -> None:
        self.heads, self.dim, self.group = heads, dim, group
        self.page_bytes = _page_bytes(heads, dim, group)
        self.base, self.capacity = {16: 0, 8: 0, 4: 0}, {16: 0, 8: 0, 4: 0}
        cursor = 0
        if pages:
            for bits in (16, 8, 4):
                n = int(pages.get(bits, 0))
                self.base[bits] = cursor
                self.capacity[bits] = n
                self._free[bits].add_run(cursor, self.page_bytes[bits], n)
                cursor += n * self.page_bytes[bits]
        self.nbytes = max(cursor, 16)

    @cached_property
    def _free(self) -> dict:
        """Free slots by precision (made when asked for: a pool that names a caller's memory has none)."""
        return {bits: _FreeSlots() for bits in (16, 8, 4)}

    @classmethod
    def over(cls, arena: torch.Tensor, heads: int, dim: int, *, group: int = 64, pages: dict | None = None) -> "PagePool":
        """A pool over a caller's arena: a contiguous, 16-byte aligned uint8 CUDA tensor.

        ``pages`` lays its slots out as the constructor does (FP16, then INT8,
        then INT4 slots, all free); without it the pool only names the memory
        that existing tables point into, and has no slots of its own.  The arena
        never grows: a request for more slots raises MemoryError."""
        if dim not in (64, 128) or not group_ok(dim, group):
            raise ValueError(f"supported geometry: head dim 64 or 128, scale groups 32, 64, 128, {BLOCK * dim}")
        if arena.dtype != torch.uint8 or arena.dim() != 1 or not arena.is_contiguous() or arena.data_ptr() % 16 \
                or not arena.is_cuda:
            raise ValueError("the arena must be a contiguous, 16-byte aligned one-dimensional uint8 CUDA tensor")
        pool = cls.__new__(cls)
        pool.device, pool.fixed = arena.device, True
        pool._lay_out(heads, dim, group, pages)
        if pages and pool.nbytes > arena.numel():
            raise ValueError(f"{pool.nbytes} bytes of page slots do not fit an arena of {arena.numel()}")
        pool.nbytes, pool.arena = arena.numel(), arena
        return pool

    def free_slots(self, bits: int) -> int:
        return len(self._free[bits])

    def alloc(self, bits: int) -> int:
        if not len(self._free[bits]):
            raise MemoryError(f"page pool has no free {bits}-bit page slots")
        return int(self._free[bits].take(1)[0])

    def check_free(self, bits: int, n: int) -> None:
        """Raise MemoryError unless ``n`` slots of ``bits`` are free (nothing changes)."""
        if n > len(self._free[bits]):
            raise MemoryError(f"page pool has {len(self._free[bits])} free {bits}-bit slots, {n} requested")

    def alloc_many(self, bits: int, n: int) -> np.ndarray:
        self.check_free(bits, n)
        return self._free[bits].take(n)

    def free(self, bits: int, offset: int) -> None:
        self._free[bits].give(np.array([offset], np.int64))

    def free_many(self, bits: int, offsets) -> None:
        self._free[bits].give(np.asarray(offsets, np.int64).reshape(-1))

    @property
    def untouched(self) -> bool:
        """Whether no slot was ever taken and the pool never grew or was shuffled: its slots are then handed
        out in ascending order from each class's base (the order compact_pages fills them in)."""
        return all(self._free[b].untouched(self.base[b], self.capacity[b]) for b in (4, 8, 16))

    def claim(self, bits: int, n: int) -> None:
        """Take the first ``n`` slots of an untouched pool's class without naming them."""
        self._free[bits].skip(n)

    def reserve(self, bits: int, n: int) -> None:
        """Make at least ``n`` slots of ``bits`` free, growing the arena if needed.

        Growth appends a region of new slots (at least doubling the class) and
        copies the old arena into a larger one on the current stream: byte
        offsets, and so descriptors, stay valid, but tensors viewing the old
        arena (``page_view``) do not follow.  Owners that hand out page views
        (``PagedLayer``) never grow their pool."""
        short = n - len(self._free[bits])
        if short <= 0:
            return
        if self.fixed:
            self.check_free(bits, n)  # raises: the arena is the caller's
        extra = max(short, self.capacity[bits], 64)
        start = self.nbytes
        old = self.arena
        self.nbytes = start + extra * self.page_bytes[bits]
        self.arena = torch.empty(self.nbytes, dtype=torch.uint8, device=self.device)
        self.arena[:start].copy_(old[:start])
        self.arena[start:].zero_()
        self._free[bits].add_run(start, self.page_bytes[bits], extra)  # old free slots are taken first
        self.capacity[bits] += extra

    def page_view(self, offset: int, bits: int) -> torch.Tensor:
        """uint8 view ``[heads, record_bytes]`` of one page."""
        rec = self.page_bytes[bits] // self.heads
        return self.arena[offset:offset + self.page_bytes[bits]].view(self.heads, rec)


class PagedBatch:
    """Page tables of ``batch`` sequences for one layer over a shared pool.

    ``table[b, j]`` is the descriptor of page ``j`` of sequence ``b``;
    ``seq_blocks[b]`` the number of pages sequence ``b`` uses.  Skip entries
    (evicted or invisible pages) are never read by the decode kernel.

    ``tokens`` (an int32 tensor ``[batch]`` on the pool's device, one int for
    all sequences, or None where they are not known) is how many tokens each
    sequence holds, evicted ones included: column ``j`` holds positions ``16 j``
    to ``16 j + 15``.  Attention that goes by position needs it.
    """

    tokens = None

    def __init__(self, pool: PagePool, batch: int, max_blocks: int):
        self.pool = pool
        self.batch, self.max_blocks = batch, max_blocks
        self.table = torch.zeros((batch, max_blocks), dtype=torch.int64, device=pool.device)
        self.seq_blocks = torch.full((batch,), max_blocks, dtype=torch.int32, device=pool.device)

    @classmethod
    def over(cls, pool: PagePool, table: torch.Tensor, *, tokens=None) -> "PagedBatch":
        """A batch over an existing ``[batch, max_blocks]`` descriptor table (a
        view, no allocation); every sequence uses all ``max_blocks`` entries, or
        those of its ``tokens`` where attention goes by position."""
        view = cls.__new__(cls)
        view.pool, view.table, view.seq_blocks, view.tokens = pool, table, None, tokens
        view.batch, view.max_blocks = int(table.shape[0]), int(table.shape[1])
        return view

    heads = property(lambda self: self.pool.heads)
    dim = property(lambda self: self.pool.dim)
    group = property(lambda self: self.pool.group)
    block = BLOCK

    def resident_bytes(self) -> int:
        """Payload + scale bytes of the pages this table references (skips excluded)."""
        d = self.table.cpu().numpy().reshape(-1)
        modes = d & 3
        total = 0
        for bits, mode in BITS_TO_MODE.items():
            total += int((modes == mode).sum()) * self.pool.heads * algorithmic_record_bytes(
                self.pool.dim, self.pool.group, bits)
        return total


def algorithmic_record_bytes(dim: int, group: int, bits: int) -> int:
    """Payload + scale bytes of one (page, head) record, without alignment pad."""
    payload = BLOCK * dim * bits // 8
    scales = 0 if bits == 16 else BLOCK * dim // group
    return 2 * payload + 4 * scales


def pack_dense(pool: PagePool, key: torch.Tensor, value: torch.Tensor, block_bits, *,
               visible=None, semantics: str = "tensor", lengths=None) -> PagedBatch:
    """Pack dense fp16 K/V ``[batch, heads, tokens, head_dim]`` into ``pool``.

    ``block_bits[b][j]`` is the precision of block ``j`` of sequence ``b``:
    16, 8 or 4, or 0 for an evicted block (no storage, skipped by decode).
    ``visible`` (same shape, bool): False hides a resident block (kept in the
    pool, skipped by decode), as focus/local visibility does.  ``lengths[b]`` (tokens,
    default all) lets the last block of a sequence be partial.  ``semantics``
    selects the quantizer: ``"tensor"`` = backend.quantize_tensor with
    ``group`` elements per scale (backend.py:183-226), ``"page"`` =
    packed_decode.pack_page (packed_decode.py:48-67).  Returns the batch's
    page table; physical placement follows the pool's free-list order.
    """
    if key.shape != value.shape or key.ndim != 4:
        raise ValueError("key and value must share [batch, heads, tokens, head_dim]")
    batch, heads, tokens, dim = key.shape
    if (heads, dim) != (pool.heads, pool.dim):
        raise ValueError("key/value geometry does not match the page pool")
    _lib.require_cuda(key, "key")
    nblk = -(-tokens // BLOCK)
    bits = np.asarray(block_bits, dtype=np.int64).reshape(batch, nblk)
    if not np.isin(bits, (0, 4, 8, 16)).all():
        raise ValueError("block precision must be 16, 8, 4 or 0 (evicted)")
    lengths = np.full(batch, tokens, np.int64) if lengths is None else np.asarray(lengths, np.int64)
    if (lengths < 0).any() or (lengths > tokens).any():
        raise ValueError("lengths must lie in [0, tokens]")
    padded = nblk * BLOCK
    if padded != tokens or key.dtype != torch.float16 or not key.is_contiguous():
        pad = lambda t: torch.nn.functional.pad(t.half(), (0, 0, 0, padded - tokens)).contiguous()
        key, value = pad(key), pad(value)
    blocks_used = -(-lengths // BLOCK)
    j = np.arange(nblk)[None, :]
    bits = np.where(j < blocks_used[:, None], bits, 0)
    ntok = np.clip(lengths[:, None] - j * BLOCK, 1, BLOCK)
    offsets = np.zeros((batch, nblk), np.int64)
    codes = np.zeros((batch, nblk), np.int64)
    for b_ in BITS_TO_MODE:  # every class checked before any slot is taken
        pool.check_free(b_, int((bits == b_).sum()))
    dev = pool.device
    status, stream = _lib.status_ptr(dev), _lib.stream_of(dev)  # an earlier kernel's error, before any change
    for b_, mode in BITS_TO_MODE.items():
        where = bits == b_
        offsets[where] = pool.alloc_many(b_, int(where.sum()))
        codes[where] = mode
    desc = encode_array(codes, ntok, offsets)
    dst = torch.from_numpy(desc.reshape(-1)).to(dev)
    sem = _lib.SEM_TENSOR if semantics == "tensor" else _lib.SEM_PAGE
    _lib.call("akv_pack_pages", key.data_ptr(), value.data_ptr(), heads * padded * dim, padded * dim,
              nblk, batch * nblk, dst.data_ptr(), pool.arena.data_ptr(), pool.nbytes, heads, dim,
              pool.group, sem, status, stream)
    out = PagedBatch(pool, batch, nblk)
    if visible is not None:
        desc = np.where(np.asarray(visible, bool).reshape(batch, nblk), desc, 0)
    out.table.copy_(torch.from_numpy(desc))
    out.seq_blocks.copy_(torch.from_numpy(blocks_used.astype(np.int32)))
    out.lengths = lengths
    out.tokens = torch.from_numpy(lengths.astype(np.int32)).to(dev)
    return out

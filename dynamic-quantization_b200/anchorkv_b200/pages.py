"""Forking sequences that share pages, and compacting an arena.

The reference's cache holds one sequence and allocates every page by itself
(packed_decode.py:108-154), so it has neither.  Here sequences of a batch can
name the same pages:

* :func:`fork_pages` gives new sequences (beams, samples of one prompt) their
  parents' page tables in one launch over all layers, and copies only the
  half-filled page that each new sequence goes on writing to;
* :func:`compact_pages` moves the pages that a table names into another arena,
  each once, in table order, and returns the table over it: a fragmented or
  oversized arena shrinks to what is live, and each sequence's pages lie together.

Both run on the device from tables on the device; neither synchronises.  Who
holds which slot stays host bookkeeping of the pool's owner
(:class:`anchorkv_b200.live.PagedKVStore` does it for ``fork``, ``crop`` and
``compact``).
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .decode import _workspace, _workspace_bytes
from .pool import PagePool


_Slots = ctypes.c_int64 * 6  # first byte and count of the INT4, INT8 and FP16 slots


def _check_table(pool: PagePool, table: torch.Tensor, dims) -> None:
    if table.dtype != torch.int64 or table.dim() not in dims or not table.is_cuda:
        raise ValueError("a page table is an int64 CUDA tensor [batch, columns] or [layers, batch, columns]")
    if table.device != pool.arena.device:
        raise ValueError("the page table and the pool's arena must be on one device")


def fork_pages(pool: PagePool, table: torch.Tensor, parents: torch.Tensor, fresh: torch.Tensor | None = None, *,
               tokens=None) -> torch.Tensor:
    """The page table of sequences that continue ``parents``.

    ``table``: ``[layers, batch, columns]`` (or ``[batch, columns]``) int64
    descriptors over ``pool``; ``parents``: int64 CUDA ``[children]``, the
    sequence each child continues (any number of children per parent).
    ``tokens``: tokens each parent holds (int32 CUDA ``[batch]``, or one int).
    ``fresh``: int64 CUDA ``[layers, children]`` descriptors of free slots; where
    it is not 0 and the parent's last page is half filled, that page is copied
    there and the child's entry names the copy (same precision; slots distinct).
    Elsewhere the child shares its parent's pages.  At most one child may go on
    writing to a page, so all but one child of a parent need a fresh slot.

    Returns the children's table, contiguous; ``table`` is left as it is."""
    _check_table(pool, table, (2, 3))
    three = table if table.dim() == 3 else table.unsqueeze(0)
    layers, batch, columns = three.shape
    dev = table.device
    if parents.dtype != torch.int64 or parents.dim() != 1 or parents.device != dev or not parents.is_contiguous():
        raise ValueError("parents must be a contiguous int64 tensor [children] on the table's device")
    children = parents.shape[0]
    counts, uniform = None, 0
    if fresh is not None:
        if fresh.dtype != torch.int64 or fresh.numel() != layers * children or fresh.device != dev \
                or not fresh.is_contiguous():
            raise ValueError("fresh must be a contiguous int64 tensor [layers, children] on the table's device")
        if isinstance(tokens, int):
            uniform = tokens
            if not 0 <= tokens < 1 << 31:
                raise ValueError("token counts must be non-negative 32-bit integers")
        elif tokens is None or tokens.dtype != torch.int32 or tuple(tokens.shape) != (batch,) \
                or tokens.device != dev or not tokens.is_contiguous():
            raise ValueError("fresh slots need tokens: an int, or a contiguous int32 tensor [batch] on the "
                             "table's device")
        else:
            counts = tokens
    if batch == 0 and children:
        raise ValueError("the table has no sequence to fork from")
    if three.stride(-1) != 1 or three.stride(1) < columns or three.stride(0) < 0:
        three = three.contiguous()
    with _lib.on_device(dev):
        status, stream = _lib.status_ptr(dev), _lib.stream_of(dev)
        out = three.new_empty((layers, children, columns))
        if out.numel():
            _lib.call("akv_fork_pages", three.data_ptr(), three.stride(0), three.stride(1), layers, batch, columns,
                      None if counts is None else counts.data_ptr(), uniform, parents.data_ptr(), children,
                      None if fresh is None else fresh.data_ptr(), out.data_ptr(), pool.arena.data_ptr(),
                      pool.nbytes, pool.heads, pool.dim, pool.group, status, stream)
    return out if table.dim() == 3 else out[0]


def compact_pages(pool: PagePool, table: torch.Tensor, into: PagePool, live: dict | None = None) -> torch.Tensor:
    """Copy the pages that ``table`` names from ``pool`` into ``into`` and return
    the table over the copies.

    ``table``: int64 descriptors of any shape whose entries are the pages to
    keep (concatenate the tables of several batches).  Each page moves once,
    however many entries name it, to the next slot of its precision in the order
    in which the table first names it; valid-token counts and skip entries stay.
    ``into``: a pool of the same page geometry over another arena, with no slot
    taken and room for the pages.  ``live``: distinct pages of each precision
    (bits -> count), which ``into`` then counts as taken; by default all of its
    slots.  Pages beyond them stay behind: their entries become skip entries and
    the next call raises KernelError.  ``pool`` and ``table`` are left as they are."""
    _check_table(pool, table, range(1, 9))
    if (into.heads, into.dim, into.group) != (pool.heads, pool.dim, pool.group) or into.arena.device != table.device:
        raise ValueError("the target pool must have the source's page geometry and device")
    if not into.untouched:
        raise ValueError("the target pool must be a new one: no slot taken, not grown, not shuffled")
    taken = into.capacity
    if live is not None:
        taken = {b: int(live.get(b, 0)) for b in (4, 8, 16)}
        for b, n in taken.items():
            if n < 0:
                raise ValueError("page counts must be non-negative")
            into.check_free(b, n)
    flat = table.contiguous()
    dev = table.device
    source, target = pool.arena.data_ptr(), into.arena.data_ptr()
    if source < target + into.nbytes and target < source + pool.nbytes:
        raise ValueError("the target pool must have an arena of its own")
    if flat.numel() == 0:
        return flat.clone()
    with _lib.on_device(dev):
        nbytes = _workspace_bytes(dev, flat.numel(), pool.nbytes, pool.heads, pool.dim, pool.group,
                                  entry="akv_compact_workspace_bytes")
        if nbytes < 0:
            raise ValueError("unsupported page geometry")
        status, stream = _lib.status_ptr(dev), _lib.stream_of(dev)
        out = torch.empty_like(flat)
        ws = _workspace(dev, nbytes, stream)
        base = into.base  # no page goes to a slot that is not counted as taken
        slots = _Slots(base[4], taken[4], base[8], taken[8], base[16], taken[16])
        _lib.call("akv_compact_pages", flat.data_ptr(), flat.numel(), out.data_ptr(), pool.arena.data_ptr(),
                  pool.nbytes, into.arena.data_ptr(), into.nbytes, slots, pool.heads, pool.dim, pool.group,
                  ws.data_ptr(), ws.numel(), status, stream)
    for b, n in taken.items():
        into.claim(b, n)
    return out

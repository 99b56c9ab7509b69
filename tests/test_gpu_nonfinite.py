"""Rows whose scores are not numbers, in every form that attention by position runs in.

A NaN in a query row, or in every key that some warp sees, makes the rows that see
it NaN and leaves the others as they are. Zeros stay what a row that sees nothing gets."""

import numpy as np
import pytest
import torch

import anchorkv_b200 as akv
from anchorkv_b200 import pool as P
from position_reference import assert_rows_close, attention_rows_torch

pytestmark = pytest.mark.gpu

HQ, HKV, DIM, SCALE = 16, 2, 128, .02
# rows, tokens, window: items with a CTA each, equal ranges joined by a CTA a row or by a
# warp a row, and operand tiles
FORMS = pytest.mark.parametrize("rows,lengths,window", [
    (5, [150, 70], None), (1, [150, 70], 90), (1, [33000, 20000], 30000), (12, [5000, 3000], None),
    (2100, [2500, 2150], None)], ids=["own", "own-window", "ranges-wide", "ranges", "tiles"])


def _store(cuda, lengths, bits):
    """Small whole numbers, which INT4 pages of scale 1 hold exactly."""
    gen = torch.Generator().manual_seed(len(lengths) + lengths[0])
    span = -(-max(lengths) // 16) * 16
    k, v = (torch.randint(-7, 8, (len(lengths), HKV, span, DIM), generator=gen).half() for _ in range(2))
    k[..., ::32] = v[..., ::32] = 7  # every group's largest
    k, v = k.to(cuda), v.to(cuda)
    nblk = span // 16
    pool = P.PagePool(HKV, DIM, pages={bits: len(lengths) * nblk}, device=cuda)
    return P.pack_dense(pool, k, v, np.full((len(lengths), nblk), bits), lengths=lengths), k, v


def _call(q, store, rows, window):
    if rows == 1:
        return akv.packed_attention(q, store, SCALE, window=window)
    return akv.chunk_attention(q, store, SCALE, window=window)


def _check(out, nan, q, k, v, lengths, window):
    """NaN where `nan` [batch, heads, rows] says so, the definition elsewhere."""
    assert torch.isnan(out[nan]).all()
    want, tol = [], []
    for b, n in enumerate(lengths):
        held = torch.arange(k.shape[2], device=k.device) < n
        w, t = attention_rows_torch(q[b], k[b], v[b], held, n, SCALE, window)
        want.append(w), tol.append(t)
    want, tol = np.stack(want), np.stack(tol)
    gone = nan.cpu().numpy()
    want[gone] = 0
    assert_rows_close(out.masked_fill(nan[..., None], 0), want, tol)
    assert akv.take_device_status(out.device) == 0


@FORMS
@pytest.mark.parametrize("bits", [4, 16])
def test_a_nan_query_row_is_nan(cuda, rows, lengths, window, bits):
    store, k, v = _store(cuda, lengths, bits)
    q = torch.randn((2, HQ, rows, DIM), generator=torch.Generator().manual_seed(rows)).half().to(cuda)
    bad = q.clone()
    nan = torch.zeros((2, HQ, rows), dtype=torch.bool, device=cuda)
    for b, h, r in ((0, 3, rows - 1), (1, 9, rows // 2), (1, 0, rows - 1)):
        bad[b, h, r, 5] = float("nan")
        nan[b, h, r] = True
    _check(_call(bad, store, rows, window), nan, q, k, v, lengths, window)


@FORMS
@pytest.mark.parametrize("bits", [4, 16])
@pytest.mark.parametrize("share", [1, 4], ids=["whole", "quarter"])
def test_pages_of_nan_keys_make_the_rows_that_see_them_nan(cuda, rows, lengths, window, bits, share):
    """All pages of a head, or its first visible quarter (whole warps' shares): not left out of the sum."""
    store, k, v = _store(cuda, lengths, bits)
    q = torch.randn((2, HQ, rows, DIM), generator=torch.Generator().manual_seed(rows)).half().to(cuda)
    first = 0 if window is None else max(lengths[0] - window, 0) // 16
    pages = -(-lengths[0] // 16)
    rec = store.pool.page_bytes[bits] // HKV
    payload = 16 * DIM * bits // 8
    for j in range(first, first + max(1, (pages - first) // share)):
        off = int(store.table[0, j]) >> 8  # head 0's record
        part = slice(off, off + payload) if bits == 16 else slice(off + 2 * payload, off + 2 * payload + 64)
        store.pool.arena[part].fill_(0xFF)  # its keys, or the 32 fp16 scales of its keys
        assert rec >= 2 * payload
    nan = torch.zeros((2, HQ, rows), dtype=torch.bool, device=cuda)
    nan[0, :HQ // HKV] = True  # their positions are past the first page, and within the window
    _check(_call(q, store, rows, window), nan, q, k, v, lengths, window)

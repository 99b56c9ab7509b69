"""A chunk over sequences whose operand tiles exceed the workspace one call may take.

The workspace stays at 2 GiB, and slices of KV heads give what whole calls give."""

import numpy as np
import pytest
import torch

import anchorkv_b200 as akv
from anchorkv_b200 import _lib
from anchorkv_b200 import pool as P
from position_reference import assert_rows_close, attention_rows_torch

pytestmark = pytest.mark.gpu

HEADS, HQ, ROWS, PAGES = 7, 14, 60, 64


@pytest.mark.parametrize("dim,columns,lengths", [(128, 80000, [16 * 80000 - 5]),
                                                (64, 100000, [16 * 100000 - 3, 16 * 90000 + 1])])
def test_kv_heads_go_in_slices(cuda, dim, columns, lengths):
    batch, span, scale = len(lengths), 16 * columns, dim ** -.5
    gen = torch.Generator().manual_seed(dim)
    k, v = (torch.randn((1, HEADS, 16 * PAGES, dim), generator=gen).half().to(cuda) for _ in range(2))
    pool = P.PagePool(HEADS, dim, pages={16: PAGES}, device=cuda)
    few = P.pack_dense(pool, k, v, np.full((1, PAGES), 16))
    order = torch.randint(0, PAGES, (batch, columns), generator=gen).to(cuda)
    tokens = torch.tensor(lengths, dtype=torch.int32, device=cuda)
    store = P.PagedBatch.over(pool, few.table[0][order], tokens=tokens)
    need = HEADS * span * dim * 4
    assert need > 2 << 30, "a sequence's operand tiles do not fit"
    held = _lib.load().akv_chunk_workspace_bytes(batch, ROWS, HQ, HEADS, dim, columns, 0, 0, 4)
    assert 1 << 30 < held <= 2 << 30
    q = torch.randn((batch, HQ, ROWS, dim), generator=gen).half().to(cuda)
    token_major = q.transpose(1, 2).contiguous().transpose(1, 2)
    out = torch.full((batch, ROWS, HQ, dim), 7., dtype=torch.float16, device=cuda).transpose(1, 2)
    akv.chunk_attention(token_major, store, scale, out=out)
    assert akv.take_device_status(cuda) == 0
    group = HQ // HEADS
    there = torch.ones(span, dtype=torch.bool, device=cuda)
    for b in range(batch):
        at = (16 * order[b][:, None] + torch.arange(16, device=cuda)).reshape(-1)
        for h in (0, 2, 3, 6):  # the slices' first and last heads among them
            heads = slice(group * h, group * h + group)
            want, tol = attention_rows_torch(q[b, heads], k[0, h:h + 1, at], v[0, h:h + 1, at], there, lengths[b], scale)
            # the tolerance's share for subnormal weights, 2^-25 of the largest each, is 2^-32 in these forms
            seen = lengths[b] - ROWS + 1 + np.arange(ROWS)[None, :, None]
            tol -= seen * (2.0 ** -25 - 2.0 ** -32) * float(v[0, h].abs().max())
            assert tol.max() < .02 * np.abs(want).max()
            assert_rows_close(out[b, heads], want, tol)

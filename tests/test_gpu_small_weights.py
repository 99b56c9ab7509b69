"""Many small weights behind one large: a first token that takes most of the attention.

Key 0 has a score of GAP above the others, which are all alike, with value 0 there
and 1 elsewhere; a row that sees n others gives n w / (1 + n w), w = exp(-GAP) =
2^-25.5. The weights are fp16 operands of P.V, scaled by 2^7 beside a largest
of at least 1: below 2^-21 of it they are subnormal, off by 2^-32 each, against
n w the rest is relative: half a step of fp16 for a weight, for the output, and
2^-13 for the fp32 scores."""

import math

import numpy as np
import pytest
import torch

import anchorkv_b200 as akv
from anchorkv_b200 import pool as P

pytestmark = pytest.mark.gpu

GAP = 25.5 * math.log(2)


def _store(cuda, batch, columns, heads, dim):
    """Sequences of one first page and, again and again, one other page."""
    k, v = torch.zeros((1, heads, 32, dim)), torch.ones((1, heads, 32, dim))
    k[:, :, 0, 3], v[:, :, 0] = 8, 0
    pool = P.PagePool(heads, dim, pages={16: 2}, device=cuda)
    two = P.pack_dense(pool, k.half().to(cuda), v.half().to(cuda), np.full((1, 2), 16))
    table = two.table[:, 1:].expand(batch, columns).contiguous()
    table[:, 0] = two.table[0, 0]
    return P.PagedBatch.over(pool, table, tokens=16 * columns)


def _check(out, others):
    """`others` [rows]: tokens beside the first that each row sees."""
    n = torch.as_tensor(others, dtype=torch.float64)[:, None]
    want = n * math.exp(-GAP) / (1 + n * math.exp(-GAP))
    tol = (2 * 2.0 ** -11 + 2.0 ** -13) * want + n * 2.0 ** -32 + 2.0 ** -25
    off = (out.double().cpu() - want).abs()
    assert (off <= tol).all(), f"off by up to {(off / want).max():.3g} of the value"
    assert akv.take_device_status(out.device) == 0


def test_operand_tiles_over_a_long_sequence(cuda):
    """160 units of 256 rows, so that a CTA's share is a whole sequence."""
    columns, rows, dim = 16384, 640, 64
    store = _store(cuda, 1, columns, 8, dim)
    q = torch.zeros((1, 64, rows, dim), dtype=torch.float16, device=cuda)
    q[..., 3] = 8
    out = akv.chunk_attention(q, store, GAP / 64)
    _check(out, 16 * columns - rows + np.arange(rows))


def test_windowed_decode_of_a_large_batch(cuda):
    """2400 items, so that a warp's share is a whole sequence."""
    columns, batch, dim = 2048, 300, 128
    store = _store(cuda, batch, columns, 8, dim)
    q = torch.zeros((batch, 16, 1, dim), dtype=torch.float16, device=cuda)
    q[..., 3] = 8
    out = akv.packed_attention(q, store, GAP / 64, window=20000, sinks=1)
    _check(out, [20000])

"""Windowed decode and chunk attention against the definition in float64.

Lengths, windows, sinks and row counts are chosen around page borders (16
tokens), odd head counts and rows that see nothing; the tolerance is worked out
per output in position_reference."""

import numpy as np
import pytest
import torch

import anchorkv_b200 as akv
import workloads as W
from anchorkv_b200 import pool as P
from paged_reference import block_values
from position_reference import assert_rows_close, attention_rows_f64

pytestmark = pytest.mark.gpu


def _store(cuda, seed, lengths, kv_heads, dim, group, semantics, mix=None, hidden=0.0, dirty=False):
    """A batch of mixed pages, the fp16 values they hold and which tokens are there."""
    batch, tokens = len(lengths), max(max(lengths), 1)
    nblk = -(-tokens // 16)
    k = W.outlier_kv(seed, (batch, kv_heads, tokens, dim))
    v = W.outlier_kv(seed + 1, (batch, kv_heads, tokens, dim))
    bits = np.array(W.draw_modes(seed + 2, batch * nblk, mix or {16: .2, 8: .3, 4: .4, 0: .1})).reshape(batch, nblk)
    visible = np.array(W.draw_modes(seed + 3, batch * nblk, {16: 1 - hidden, 0: hidden})).reshape(batch, nblk) > 0 \
        if hidden else np.ones((batch, nblk), bool)
    pool = P.PagePool(kv_heads, dim, group=group, pages={b: int((bits == b).sum()) for b in (16, 8, 4)}, device=cuda,
                      shuffle_seed=seed)
    store = P.pack_dense(pool, k.to(cuda), v.to(cuda), bits, visible=visible, semantics=semantics, lengths=lengths)
    span = nblk * 16
    kd, vd = np.zeros((batch, kv_heads, span, dim)), np.zeros((batch, kv_heads, span, dim))
    held = np.zeros((batch, span), bool)
    pad = lambda t: np.pad(t.numpy(), ((0, 0), (0, 0), (0, span - tokens), (0, 0)))  # noqa: E731
    kp, vp = pad(k), pad(v)
    for b in range(batch):
        for j in range(nblk):
            if bits[b, j] == 0 or not visible[b, j] or 16 * j >= lengths[b]:
                continue
            sl = slice(16 * j, 16 * j + 16)
            for h in range(kv_heads):
                kd[b, h, sl] = block_values(kp[b, h, sl], int(bits[b, j]), group, semantics)
                vd[b, h, sl] = block_values(vp[b, h, sl], int(bits[b, j]), group, semantics)
            held[b, sl] = True
    held &= np.arange(span)[None] < np.asarray(lengths)[:, None]
    return store, kd, vd, held


WINDOWS = [
    # dim, q_heads, kv_heads, group, semantics, lengths, window, sinks
    (128, 16, 8, 2048, "tensor", [512], 128, 4),
    (128, 16, 8, 2048, "tensor", [1, 2, 15, 16, 17, 33], 1, 0),
    (128, 8, 8, 64, "page", [97, 65, 640], 16, 16),
    (128, 32, 4, 128, "page", [300, 31, 1200], 100, 37),
    (64, 24, 8, 64, "page", [250, 64, 803], 77, 5),
    (64, 9, 3, 1024, "tensor", [333, 20], 17, 1),
    (64, 40, 2, 32, "page", [129, 450], 300, 300),
    (128, 16, 8, 2048, "tensor", [700, 40], 100000, 3),
    (128, 4, 1, 64, "page", [2000], 1000, 2 ** 31 - 1),
]


@pytest.mark.parametrize("case", WINDOWS, ids=lambda c: f"d{c[0]}_q{c[1]}_kv{c[2]}_g{c[3]}_w{c[6]}_s{c[7]}")
def test_window_decode_against_the_definition(cuda, case):
    dim, hq, hkv, group, semantics, lengths, window, sinks = case
    seed = dim + hq + window % 97
    store, k, v, held = _store(cuda, seed, lengths, hkv, dim, group, semantics, hidden=.1)
    q = W.normal(seed + 9, (len(lengths), hq, 1, dim))
    scale = dim ** -0.5
    out = akv.packed_attention(q.to(cuda), store, scale, window=window, sinks=sinks)
    assert out.shape == q.shape and out.dtype == torch.float16
    assert akv.take_device_status(cuda) == 0
    assert_rows_close(out, *attention_rows_f64(q, k, v, held, lengths, scale, window, sinks))


CHUNKS = [
    # dim, q_heads, kv_heads, group, semantics, lengths, rows, window, sinks
    (128, 16, 8, 2048, "tensor", [512, 77], 5, None, 0),
    (128, 16, 8, 64, "page", [100], 100, None, 0),
    (128, 16, 8, 2048, "tensor", [40, 16, 3, 17], 17, None, 0),
    (128, 32, 8, 2048, "tensor", [400, 333], 33, None, 0),
    (64, 24, 8, 64, "page", [300, 90], 130, 64, 4),
    (64, 3, 3, 1024, "tensor", [257, 256], 2, None, 0),
    (64, 16, 2, 32, "page", [129, 700], 48, 17, 1),
    (128, 8, 8, 128, "page", [260, 513], 260, 100, 20),
    (128, 16, 1, 64, "page", [520], 71, 1, 0),
    (128, 4, 4, 2048, "tensor", [900, 60], 200, 5000, 7),
    (128, 72, 8, 2048, "tensor", [150, 33], 19, 40, 16),
    # enough rows and pages for the tcgen05 tiles
    (128, 8, 1, 2048, "tensor", [2500], 300, None, 0),
    (128, 12, 4, 64, "page", [1700, 30, 900], 190, None, 0),
    (64, 24, 8, 64, "page", [1200, 700], 150, 333, 37),
    (64, 16, 4, 1024, "tensor", [1030, 2, 129, 1500], 257, 16, 1),
    (128, 8, 8, 32, "page", [600, 590], 600, 200, 0),
    (64, 6, 2, 128, "tensor", [4100], 700, 3000, 130),
]


@pytest.mark.parametrize("case", CHUNKS, ids=lambda c: f"d{c[0]}_q{c[1]}_kv{c[2]}_g{c[3]}_r{c[6]}_w{c[7]}_s{c[8]}")
def test_chunks_against_the_definition(cuda, case):
    dim, hq, hkv, group, semantics, lengths, rows, window, sinks = case
    seed = 3 * dim + hq + rows
    store, k, v, held = _store(cuda, seed, lengths, hkv, dim, group, semantics)
    q = W.normal(seed + 9, (len(lengths), hq, rows, dim))
    scale = dim ** -0.5
    out = akv.chunk_attention(q.to(cuda), store, scale, window=window, sinks=sinks)
    assert out.shape == q.shape and out.dtype == torch.float16
    assert akv.take_device_status(cuda) == 0
    assert_rows_close(out, *attention_rows_f64(q, k, v, held, lengths, scale, window, sinks))

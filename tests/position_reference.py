"""Expected output of attention by position over paged stores (test infrastructure).

Query rows are the last tokens of every sequence; the answer is the definition
in float64 over the fp16 values that the pages hold, beside the bound on what a
kernel may be off by:

* P is rounded to fp16 before P.V: each term is off by at most half a step,
  2^-11 of it, so the output by 2^-11 of A, the weighted mean of |v|;
* scores are fp32 sums of fp16 products: an error of 2^-13 in a weight
  (relative) covers 128 terms of the sizes used here with room (a sum of n fp32
  terms is off by at most n 2^-24 of the sum of their sizes: 128 x 2^-24 x 100);
* weights below 2^-14 are fp16 subnormals, off by 2^-25 absolutely beside a sum
  of at least 1: n 2^-25 max|v|;
* the output is rounded to fp16 once: 2^-11 of it, or 2^-25 when it is subnormal.
"""

import numpy as np

BLOCK = 16


def attention_rows_f64(q, k, v, held, tokens, scale, window=None, sinks=0):
    """(output, tolerance), both ``[B, Hq, R, D]`` float64.

    ``q``: ``[B, Hq, R, D]``; ``k``, ``v``: ``[B, Hkv, T, D]`` values as stored;
    ``held``: ``[B, T]`` bool, tokens that are resident and visible;
    ``tokens``: ``[B]`` tokens of each sequence."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    batch, hq, rows, dim = q.shape
    hkv, span = k.shape[1], k.shape[2]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    pos = np.arange(span)
    for b in range(batch):
        for i in range(rows):
            at = int(tokens[b]) - rows + i
            seen = np.asarray(held[b]) & (pos <= at) & (pos < tokens[b]) & (at >= 0)
            if window is not None:
                seen &= (pos > at - window) | (pos < sinks)
            if not seen.any():
                tol[b, :, i] = 0.0
                continue
            for h in range(hq):
                kh, vh = k[b, h // (hq // hkv)][seen], v[b, h // (hq // hkv)][seen]
                s = kh @ q[b, h, i] * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                o = w @ vh
                out[b, h, i] = o
                tol[b, h, i] = ((2.0 ** -11 + 2.0 ** -13) * (w @ np.abs(vh)) + 2.0 ** -11 * np.abs(o)
                                + len(w) * 2.0 ** -25 * np.abs(vh).max() + 2.0 ** -25)
    return out, tol


def assert_rows_close(actual, expected, tolerance):
    a = actual.detach().double().cpu().numpy()
    assert a.shape == expected.shape
    over = np.abs(a - expected) - tolerance
    assert np.isfinite(a).all()
    worst = np.unravel_index(np.argmax(over), over.shape)
    assert over.max() <= 0, f"at {worst}: {a[worst]} against {expected[worst]}, tolerance {tolerance[worst]:.3g}"


def attention_rows_torch(q, k, v, held, tokens, scale, window=None, sinks=0):
    """attention_rows_f64 of one sequence as float64 matrix products on the tensors' device, for long ones.

    ``q``: ``[Hq, R, D]``; ``k``, ``v``: ``[Hkv, T, D]``; ``held``: ``[T]`` bool; gives numpy arrays ``[Hq, R, D]``."""
    import torch

    groups = q.shape[0] // k.shape[0]
    q, k, v = q.double(), k.double().repeat_interleave(groups, 0), v.double().repeat_interleave(groups, 0)
    rows, span = q.shape[1], k.shape[1]
    at = torch.arange(tokens - rows, tokens, device=q.device)[:, None]
    pos = torch.arange(span, device=q.device)
    seen = held & (pos <= at) & (pos < tokens) & (at >= 0)
    if window is not None:
        seen = seen & ((pos > at - window) | (pos < sinks))
    s = (q @ k.transpose(1, 2) * scale).masked_fill(~seen, -torch.inf)
    w = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e300)) * seen
    w = w / w.sum(-1, keepdim=True).clamp_min(1e-300)
    o = w @ v
    some = seen.any(-1)[None, :, None]
    largest = v.abs().amax((1, 2))[:, None, None]
    tol = ((2.0 ** -11 + 2.0 ** -13) * (w @ v.abs()) + 2.0 ** -11 * o.abs()
           + seen.sum(-1)[None, :, None] * 2.0 ** -25 * largest + 2.0 ** -25) * some
    return o.cpu().numpy(), tol.cpu().numpy()

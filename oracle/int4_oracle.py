"""CPU oracle (numpy) of the rotary positions and of the 4-bit paged cache.

``quantise`` repeats the FP32 steps that define the cache's contents one by
one (numpy's elementwise float32 operations round to nearest, without fused
multiply-adds), so records can be compared bit for bit; the rotation's and
the attention's expected values are float64.
"""

from __future__ import annotations

import numpy as np

PAGE, DIM, GROUP, RECORD = 16, 128, 32, 2560


def rotate(x, cos, sin, interleaved=False, adjoint=False, dtype=np.float64):
    """x [T, H, D] turned by cos, sin [T, pairs] in ``dtype`` arithmetic."""
    x = np.asarray(x, dtype)
    c = np.asarray(cos, dtype)[:, None]
    s = np.asarray(sin, dtype)[:, None] * dtype(-1 if adjoint else 1)
    pairs = c.shape[-1]
    out = x.copy()
    ia = np.arange(pairs) * (2 if interleaved else 1)
    ib = ia + (1 if interleaved else pairs)
    a, b = x[..., ia], x[..., ib]
    out[..., ia] = a * c - b * s
    out[..., ib] = b * c + a * s
    return out


def quantise(x):
    """float32 rows [..., 128] -> codes uint8 [..., 128] (0..15) and float16
    scales and midpoints [..., 4]."""
    x = np.asarray(x, np.float32)
    x = np.minimum(np.maximum(x, np.float32(-65504)), np.float32(65504))
    x = x.reshape(*x.shape[:-1], 4, GROUP)
    lo, hi = x.min(-1), x.max(-1)
    s16 = ((hi - lo) * np.float32(1.0 / 15.0)).astype(np.float16)
    s = s16.astype(np.float32)
    m16 = (lo + np.float32(8) * s).astype(np.float16)
    m = m16.astype(np.float32)
    with np.errstate(divide="ignore"):
        inv = np.where(s > 0, np.float32(1) / s, np.float32(0)).astype(np.float32)
    z = np.rint((x - m[..., None]) * inv[..., None])
    z = np.clip(z, -8, 7).astype(np.int32) + 8
    return z.astype(np.uint8).reshape(*z.shape[:-2], DIM), s16, m16


def key_byte(tok, d):
    g, r = divmod(d, GROUP)
    return 64 * tok + 16 * (r // 8) + 4 * g + (r % 8) // 2, r % 2


def value_byte(tok, d):
    g, r = divmod(d, GROUP)
    row = (tok & 8) + 4 * (tok & 1) + (tok // 2 & 3)
    return 1024 + 64 * row + 8 * (r // 4) + 2 * g + (r % 4) // 2, r % 2


def _maps():
    out = []
    for fn in (key_byte, value_byte):
        at = np.array([[fn(t, d) for d in range(DIM)] for t in range(PAGE)])
        out.append((at[..., 0], at[..., 1]))
    return out


_BYTES = _maps()


def store_token(records, page, head, tok, key, value):
    """Write one token's quantised key and value ((codes, s, m) each) into
    records [pages, Hkv, 2560] (uint8, in place)."""
    rec = records[page, head]
    for (at, nib), (z, s, m), meta in ((_BYTES[0], key, 2048), (_BYTES[1], value, 2304)):
        rec[np.unique(at[tok])] = 0
        np.bitwise_or.at(rec, at[tok], (z << (4 * nib[tok])).astype(np.uint8))
        rec[meta + 16 * tok:meta + 16 * tok + 16] = np.concatenate((s, m)).view(np.uint8)


def load(records):
    """records [..., 2560] -> float64 (z - 8) s and m of keys and values,
    each [..., 16, 128] (x = their sum)."""
    lead = records.shape[:-1]
    out = []
    for (at, nib), meta in zip(_BYTES, (2048, 2304)):
        z = (records[..., at] >> (4 * nib).astype(np.uint8)) & 15
        sm = np.ascontiguousarray(records[..., meta:meta + 256]).view(np.float16)
        sm = sm.reshape(*lead, PAGE, 2, 4).astype(np.float64)
        s, m = (np.repeat(sm[..., i, :], GROUP, axis=-1) for i in (0, 1))
        with np.errstate(invalid="ignore"):  # slots never written may hold NaN scales
            out.append(((z.astype(np.float64) - 8) * s, m))
    return out


def attention(q, k, v, scale):
    """q [G, 128], k and v [T, 128] float64: output [G, 128], base-2 lse [G]
    and the weights [G, T]."""
    score = (q @ k.T) * scale
    top = score.max(-1, keepdims=True)
    p = np.exp(score - top)
    total = p.sum(-1, keepdims=True)
    p /= total
    return p @ v, (top + np.log(total))[:, 0] / np.log(2), p

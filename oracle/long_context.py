"""The 4-bit cache and decode through a window, in 64 bits and plain loops.

    quantise    values -> (n, s, lo) of every group of 32
    records     (n, s, lo) -> the bytes of a cache's records, and back (values)
    visible     positions that a sequence's new token sees
    decode      attention of one query per sequence over given keys and values

Written from the definitions, on numpy arrays; nothing here shares code with the
kernels.
"""

from __future__ import annotations

import numpy as np

GROUP = 32
F16_MOST = 65504.0


def _f16(x):
    """fp16 of x as float64, rounded from fp32 as the definition has it."""
    return np.asarray(x, np.float64).astype(np.float32).astype(np.float16).astype(np.float64)


def quantise(x):
    """x [..., D] -> n [..., D / 32, 32] int, s and lo float64 [..., D / 32]."""
    x = np.asarray(x, np.float64)
    g = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    none = np.isnan(g).any(-1)
    g = np.clip(np.where(none[..., None], 0.0, g), -F16_MOST, F16_MOST)
    lo = _f16(g.min(-1))
    s = _f16(np.maximum((g.max(-1) - lo) / 15, 0.0))
    step = np.where(s > 0, s, 1.0)[..., None]
    n = np.clip(np.rint((g - lo[..., None]) / step), 0, 15)
    n = np.where((s > 0)[..., None], n, 0).astype(np.int64)
    return n, s, np.where(none, np.nan, lo)


def _element(word, e, groups, keys):
    """The element of a head that nibble e of word `word` of its record holds."""
    return (word % groups * 32 + word // groups * 8 if keys else 8 * word) + e


def records(n, s, lo, keys):
    """Bytes [..., 5 D / 8] of heads [..., D / 32, 32]."""
    head, groups = n.shape[:-2], n.shape[-2]
    flat = n.reshape(int(np.prod(head)), groups * 32)
    out = np.zeros((flat.shape[0], groups * 20), np.uint8)
    for word in range(groups * 4):
        for e in range(8):
            x = flat[:, _element(word, e, groups, keys)]
            out[:, 4 * word + e // 2] |= (x << (4 * (e % 2))).astype(np.uint8)
    for i, par in enumerate((s, lo)):
        half = np.ascontiguousarray(par.reshape(len(flat), groups)).astype(np.float16).view(np.uint8)
        out[:, groups * 16 + 2 * groups * i:groups * 16 + 2 * groups * (i + 1)] = half
    return out.reshape(*head, groups * 20)


def values(rec, keys):
    """float64 [..., D] that records [..., 5 D / 8] stand for."""
    rec = np.asarray(rec)
    groups = rec.shape[-1] // 20
    flat = rec.reshape(int(np.prod(rec.shape[:-1])), rec.shape[-1])
    half = np.ascontiguousarray(flat[:, groups * 16:]).view(np.float16).astype(np.float64)
    out = np.empty((flat.shape[0], groups * 32))
    for word in range(groups * 4):
        for e in range(8):
            x = _element(word, e, groups, keys)
            n = flat[:, 4 * word + e // 2] >> (4 * (e % 2)) & 15
            out[:, x] = n * half[:, x // 32] + half[:, groups + x // 32]
    return out.reshape(*rec.shape[:-1], groups * 32)


def sizes(rec, keys):
    """float64 [..., D]: n s + |lo|, which a value's own rounding errors are relative to."""
    groups = np.asarray(rec).shape[-1] // 20
    flat = np.array(rec)
    at = slice(groups * 18, groups * 20)
    flat[..., at] &= np.tile(np.array([0xff, 0x7f], np.uint8), groups)   # |lo|
    return np.abs(values(flat, keys))


def visible(length, window, sinks):
    """The positions below `length` that the last of them sees."""
    return np.array([j for j in range(max(0, length))
                     if not window or j < sinks or j > length - 1 - window], np.int64)


def decode(q, keys, vals, scale, key_size=None, val_size=None):
    """(out, spread, weight) of q [H, D] over keys and vals [n, Hkv, D], float64: out =
    softmax(scale q . k) v; spread the same with |v| (or val_size); weight [H, D] what an
    error of the scores relative to scale |q| . |k| (or key_size) does to out: the sum of
    p |v - out| |q| . |k| scale."""
    H, D = q.shape
    out, spread, weight = np.zeros((3, H, D))
    g = H // keys.shape[1] if keys.shape[0] else 1
    if not keys.shape[0]:
        return out, spread, weight
    q = np.asarray(q, np.float64)
    with np.errstate(all="ignore"):
        for h in range(H):
            k, v = keys[:, h // g].astype(np.float64), vals[:, h // g].astype(np.float64)
            s = k @ q[h] * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            ks, vs = (np.abs(x) if y is None else y[:, h // g]
                      for x, y in ((k, key_size), (v, val_size)))
            size = ks @ np.abs(q[h]) * abs(scale)
            out[h], spread[h] = p @ v, p @ vs
            weight[h] = (p * size) @ np.abs(v - out[h])
    return out, spread, weight

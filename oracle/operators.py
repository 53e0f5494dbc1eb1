"""What the operators around paged attention compute, in 64 bits and plain loops.

    rotate        rotary positions with several axes
    prompt        causal attention over packed prompts
    find_free, fork, free, compact   the cache's pages and their counts

Written from the definitions, on numpy arrays; nothing here shares code with the
kernels.
"""

from __future__ import annotations

import numpy as np


def rotate(x, positions, inv_freq, axes=None, interleaved=False):
    """x [n, H, D], positions [axes, n], inv_freq [pairs] (as float32 holds it) ->
    float64 [n, H, D]."""
    x = np.asarray(x, np.float64)
    positions = np.atleast_2d(np.asarray(positions))
    freq = np.asarray(inv_freq, np.float64)
    out = x.copy()
    for i, f in enumerate(freq):
        axis = 0 if axes is None else int(axes[i])
        if not 0 <= axis < positions.shape[0]:
            axis = 0
        # the turn's fraction first: cos and sin of a small angle
        t = positions[axis].astype(np.longdouble) * np.longdouble(f) / (2 * np.longdouble(np.pi))
        t = (t - np.rint(t)).astype(np.float64) * 2 * np.pi
        c, s = np.cos(t)[:, None], np.sin(t)[:, None]
        p, q = (2 * i, 2 * i + 1) if interleaved else (i, len(freq) + i)
        out[:, :, p] = x[:, :, p] * c - x[:, :, q] * s
        out[:, :, q] = x[:, :, q] * c + x[:, :, p] * s
    return out


def prompt(q, k, v, cu, scale):
    """(out, spread) float64 [T, H, D]: causal attention of every sequence, and the
    same with |v| in the place of v.  Rows of no sequence are NaN."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    out = np.full(q.shape, np.nan)
    spread = np.full(q.shape, np.nan)
    g = q.shape[1] // k.shape[1]
    for a, b in zip(cu[:-1], cu[1:]):
        for i in range(a, b):
            for h in range(q.shape[1]):
                s = k[a:i + 1, h // g] @ q[i, h] * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                out[i, h] = p @ v[a:i + 1, h // g]
                spread[i, h] = p @ np.abs(v[a:i + 1, h // g])
    return out, spread


def find_free(refs, n):
    ids = [i for i, c in enumerate(refs) if c <= 0][:n]
    return np.array(ids + [-1] * (n - len(ids)), np.int32)


def fork(pool, tables, ctx, refs, parents, children, fresh):
    """In place on copies' arrays [L, 2, NB, BS, ...], [B, MB], [B], [NB]; forked [n]."""
    B, MB = tables.shape
    NB, BS = pool.shape[2:4]
    done = np.zeros(len(parents), np.int32)
    for i, (p, c, f) in enumerate(zip(parents, children, fresh)):
        if not (0 <= p < B and 0 <= c < B) or p == c:
            continue
        n = min(max(int(ctx[p]), 0), MB * BS)
        full, rem = divmod(n, BS)
        tables[c], ctx[c] = -1, 0
        if rem:
            last = tables[p, full]
            if not (0 <= last < NB and 0 <= f < NB) or last == f:
                continue
            tables[c, full] = f
            refs[f] += 1
            pool[:, :, f, :rem] = pool[:, :, last, :rem]
        for j in range(full):
            tables[c, j] = tables[p, j]
            if 0 <= tables[p, j] < NB:
                refs[tables[p, j]] += 1
        ctx[c] = n
        done[i] = 1
    return done


def free(tables, ctx, refs, rows):
    for b in rows:
        if not 0 <= b < len(ctx):
            continue
        for j in tables[b]:
            if 0 <= j < len(refs) and refs[j] > 0:
                refs[j] -= 1
        tables[b], ctx[b] = -1, 0


def compact(pool, tables, refs):
    """In place; (moved_to, live)."""
    live = int((refs > 0).sum())
    moved_to = np.where(refs > 0, np.arange(len(refs)), -1).astype(np.int32)
    holes = [i for i in range(live) if refs[i] <= 0]
    movers = [i for i in range(len(refs) - 1, live - 1, -1) if refs[i] > 0]
    assert len(holes) == len(movers)
    for to, at in zip(holes, movers):
        pool[:, :, to] = pool[:, :, at]
        refs[to], refs[at] = refs[at], 0
        moved_to[at] = to
    for b in range(tables.shape[0]):
        for j in range(tables.shape[1]):
            if 0 <= tables[b, j] < len(refs):
                tables[b, j] = moved_to[tables[b, j]]
    return moved_to, live

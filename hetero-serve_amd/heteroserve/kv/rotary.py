"""Rotary positions with several axes, and their write into the paged cache.

    rotate_qk          queries and keys turned by their positions
    rotate_append_kv   the same, and keys and values into the cache in one launch
    axes_of            the axis of each pair, from the pairs that each axis has

No reference counterpart (its models learn their positions); append_kv
(kv/pack.py) is the write without a rotation.

    q           [n, H, D], k, v [n, Hkv, D], float32, float16 or bfloat16, rows
                as far apart as they like (slices of a fused QKV output)
    positions   int32 [axes, n], or [n] for one axis.  Text counts up on every
                axis; the patches of an image or video have a time, a height and a
                width
    inv_freq    float32 [pairs], pairs <= D / 2: pair i turns by
                positions[axis_i] * inv_freq[i] radians; elements of a head from
                2 * pairs on pass unchanged
    axes        int32 [pairs], the axis of each pair (entries that name no axis
                count as 0), or None: all on the first
    interleaved pairs are elements (2 i, 2 i + 1) instead of (i, pairs + i)
    out_dtype   of the returned q and k (default: the dtype they came in;
                paged_attention takes float32 queries)

Positions, axes, tables and numbers of other integer types are converted, the far ones
to the nearest that 32 bits hold; others are refused (a position of 1.5 is not 1).
"""

from __future__ import annotations

from .. import _hip


def axes_of(sections, interleaved: bool = False):
    """int32 [sum(sections)]: axis a has sections[a] pairs, one behind the other, or
    dealt in turn (0, 1, 2, 0, 1, 2, ..., an axis that has its pairs left out)."""
    import torch

    left = [int(s) for s in sections]
    if any(s < 0 for s in left):
        raise RuntimeError(f"sections must not be negative, got {list(sections)}")
    if not interleaved:
        return torch.tensor([a for a, s in enumerate(left) for _ in range(s)], dtype=torch.int32)
    out = []
    while any(left):
        for a, s in enumerate(left):
            if s:
                out.append(a)
                left[a] -= 1
    return torch.tensor(out, dtype=torch.int32)


def rotate_qk(q, k, positions, inv_freq, axes=None, interleaved: bool = False, out_dtype=None):
    """(q, k) turned, contiguous."""
    return _hip.rotary(q, k, positions, inv_freq, axes, interleaved, out_dtype)


def rotate_append_kv(q, k, v, positions, inv_freq, k_cache, v_cache, block_tables, cache_positions,
                     seq_ids=None, axes=None, interleaved: bool = False, out_dtype=None,
                     keep_k: bool = False):
    """rotate_qk, and append_kv of the turned keys (from fp32, rounded once to the
    cache's dtype) and of the values: row i goes to position cache_positions[i]
    of sequence seq_ids[i] (row i of the tables when None).  The place in the
    cache is the token's number in its sequence, which with several axes is none
    of its positions.  Returns (q, k), k None unless keep_k (prompt_attention
    reads the keys again, paged_attention does not)."""
    return _hip.rotary_append(q, k, v, positions, inv_freq, k_cache, v_cache, block_tables,
                              cache_positions, seq_ids, axes, interleaved, out_dtype, keep_k)

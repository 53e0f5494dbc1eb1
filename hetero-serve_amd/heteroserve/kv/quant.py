"""A paged cache held in 4 bits: rows quantised as they are written, and read back.

    empty_pool_q4   a pool for it
    append_kv_q4    new K/V rows into their slots (append_kv of kv/pack.py for this cache)
    read_kv_q4      what the cache holds of given tokens, in an ordinary type

No reference counterpart: its pools hold fp32, fp16 or bf16.  A pool is uint8
[L, 2, num_blocks, block_size, n_kv_heads, record_bytes(D)], so kv/pages.py's copies, forks,
frees and compactions and kv/pack.py's export_blocks_device and write_blocks_device take
it as it is; paged_attention_q4 (model/paged_attn_q4.py) attends to it.  D is 32, 64, 128
or 256.

Every 32 elements of a head share a step and a lowest value, both fp16: 5 bits an element
instead of 16.

    lo = min x,  s = max(0, (max x - lo) / 15),  n = (x - lo) / s to the nearest of 0 .. 15

and x is held as n s + lo, at most about half a step off.  Values beyond fp16's largest
count as that, infinities too; a group of 32 that holds a NaN reads as NaN as a whole.  A
record of zeros, as an empty pool has them, reads as zeros.  The layout of a record is
given with hs_q4_append in include/hsattn_ops.h.

    k, v            [n, Hkv, D] or [n, Hkv * D], float32, float16 or bfloat16, rows as far
                    apart as they like (slices of a fused QKV output)
    k_cache/v_cache [num_blocks, block_size, Hkv, record_bytes(D)] uint8, contiguous (views
                    pool[layer, 0] / pool[layer, 1])
    block_tables    int32 [B, max_blocks], -1 padded
    positions       [n]: row i is the token at this place of its sequence
    seq_ids         [n], the table row of each; None: row i of the tables

Rows whose sequence is outside [0, B), whose position is past the table or whose table
entry is padding are not written, and read as zeros.  Tables, positions and sequence ids
of other integer types are converted, the far ones to the nearest that 32 bits hold.
"""

from __future__ import annotations

from .. import _hip


def record_bytes(head_dim: int) -> int:
    """Bytes of one token's head in the cache."""
    head_dim = int(head_dim)
    if head_dim not in (32, 64, 128, 256):
        raise RuntimeError(f"head_dim must be 32, 64, 128 or 256, got {head_dim}")
    return head_dim // 2 + head_dim // 8


def empty_pool_q4(num_layers: int, num_blocks: int, block_size: int, n_kv_heads: int, head_dim: int,
                  device="cuda"):
    """uint8 [L, 2, num_blocks, block_size, n_kv_heads, record_bytes(head_dim)] of zeros."""
    import torch

    return torch.zeros((num_layers, 2, num_blocks, block_size, n_kv_heads, record_bytes(head_dim)),
                       dtype=torch.uint8, device=device)


def append_kv_q4(k_cache, v_cache, block_tables, positions, k, v, seq_ids=None) -> None:
    """Row i of k and v, quantised, to position positions[i] of sequence seq_ids[i].  Rows
    must not share a slot."""
    _hip.q4_append(k_cache, v_cache, block_tables, positions, k, v, seq_ids)


def read_kv_q4(k_cache, v_cache, block_tables, positions, seq_ids=None, dtype=None):
    """(k, v) [n, Hkv, D] of dtype (float32, float16 or bfloat16; float16 when None): the
    tokens at positions[i] of sequences seq_ids[i], n s + lo rounded to fp32 and then to
    dtype.  In float16 values beyond its largest count as that (lo + 15 s may be: s is
    rounded)."""
    return _hip.q4_read(k_cache, v_cache, block_tables, positions, seq_ids, dtype)

"""Paged decode attention over a cache held in 4 bits.

No reference counterpart; the call is paged_attn.paged_attention's with a cache of
kv/quant.py and, if wanted, a window (paged_attn_window.py):

    q                   [B, H, D]            float32, D 32, 64, 128 or 256
    k_cache / v_cache   [num_blocks, block_size, n_kv_heads, record_bytes(D)] uint8
                        (views pool[layer, 0] / pool[layer, 1])
    block_tables        [B, max_blocks]      int32, -1 for unused slots
    context_lens        [B]                  int32, the new token counted
    window, sinks       of each context the last `window` tokens and the first `sinks`
                        are seen; window 0: all of them
    ->                  [B, H, D]            float32

The cache's values n s + lo are never written out.  The matrix cores multiply the whole
numbers n - 8 by the query and by probability times step, each in two fp16 terms of 22
bits that are scaled by head (and group), so what is lost is relative to the largest of
them; the keys' steps and the values' middles lo + 8 s are applied in fp32.  The result is as near as
fp32 arithmetic's on the values, relative to the range of their group of 32.
A sequence without tokens gets a row of zeros.
"""

from __future__ import annotations

from typing import Optional

from .. import _hip


def is_available() -> bool:
    return _hip.ready()


def build_error() -> Optional[str]:
    return _hip.error()


def paged_attention_q4(q, k_cache, v_cache, block_tables, context_lens, scale, window: int = 0,
                       sinks: int = 0):
    return _hip.q4_decode(q, k_cache, v_cache, block_tables, context_lens, scale, window, sinks)

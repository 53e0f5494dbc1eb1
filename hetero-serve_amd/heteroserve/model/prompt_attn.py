"""Causal attention over whole prompts, straight from the projection's K and V.

No reference counterpart: its engine prefills through the paged cache, one
sequence's chunk at a time (heteroserve/model/torch_engine.py:292-313).  For a
prompt without a cached prefix that reads back what was just written, so here
q, k and v are the rows of the projection, all sequences packed one behind the
other; the cache is written beside it (kv.rotary.rotate_append_kv, kv.pack.append_kv
or scatter_kv).  Chunks that continue a cached context stay with
paged_attn_prefill.paged_attention_prefill_varlen.

    q            [T, H, D] float32, float16 or bfloat16; D 32, 64, 128 or 256
    k, v         [T, Hkv, D] of q's dtype, H a multiple of Hkv
    cu_seqlens   [B + 1] int32: sequence b owns rows cu_seqlens[b]:cu_seqlens[b+1]
    max_seqlen   the longest sequence's rows (rows from there on are not computed)
    ->           [T, H, D] of q's dtype; row i attends to its sequence's rows <= i

Slices of a fused QKV output are read in place where rows and heads lie
multiples of 16 bytes (at most 2^22 elements) apart; other layouts are copied
first.  Rows behind the last sequence are left as they were in ``out`` (not set
where the call makes it), which must be contiguous and no part of q, k or v.  Products run on the matrix cores, of 16-bit inputs in
their own type, the probabilities rounded to it, of float32 ones in three bf16
terms a number, as accurate as float32; scores, softmax and sums are fp32.
"""

from __future__ import annotations

from typing import Optional

from .. import _hip


def is_available() -> bool:
    return _hip.ready()


def build_error() -> Optional[str]:
    return _hip.error()


def prompt_attention(q, k, v, cu_seqlens, max_seqlen: int, scale: float, out=None):
    return _hip.prompt_attention(q, k, v, cu_seqlens, max_seqlen, scale, out)

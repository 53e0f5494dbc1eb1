"""Paged decode attention through a sliding window, with first tokens that stay visible.

No reference counterpart (its models see their whole context); the call is
paged_attn.paged_attention's, over the same caches, with

    window   the new token sees the last `window` tokens of its context, itself among
             them (a query at position p: p - window + 1 .. p); 0: all of them
    sinks    and the first `sinks` tokens, whatever the window

so a step reads window + sinks tokens however long the context is.  Windows and sinks may
begin and end anywhere in a page; tokens that are not seen are not read, so their pages may
have been given back (their table entries may be -1 or anything).  A sequence without
tokens gets a row of zeros.
"""

from __future__ import annotations

from typing import Optional

from .. import _hip


def is_available() -> bool:
    return _hip.ready()


def build_error() -> Optional[str]:
    return _hip.error()


def paged_attention_window(q, k_cache, v_cache, block_tables, context_lens, scale, window: int,
                           sinks: int = 0):
    return _hip.window_decode(q, k_cache, v_cache, block_tables, context_lens, scale, window, sinks)

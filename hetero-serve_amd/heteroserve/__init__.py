"""hetero-serve's paged-attention hot path, rebuilt for MI355X (gfx950).

The modules on that path are ``model.paged_attn*`` (decode and prefill
attention entry points with the reference's signatures) and ``kv.pack``
(KV-block pack / unpack / gather).  Beside it are ``model.prompt_attn``
(attention over whole prompts), ``kv.rotary`` (rotary positions and their cache
write), ``kv.pages`` (copies, forks, frees and compaction of the cache's
pages), ``kv.quant`` (a cache in 4 bits), ``model.paged_attn_q4`` (decode over
it) and ``model.paged_attn_window`` (decode through a sliding window).  Their
kernels live in libhsattn.so, loaded through ``heteroserve._hip``.
"""

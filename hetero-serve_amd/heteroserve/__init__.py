"""hetero-serve's paged-attention hot path, rebuilt for MI355X (gfx950).

Only the modules on that path exist here: ``model.paged_attn*`` (decode and
prefill attention entry points with the reference's signatures) and
``kv.pack`` (KV-block pack / unpack / gather), and beside it
``model.prompt_attn`` (attention over whole prompts), ``kv.rotary`` (rotary
positions and their cache write) and ``kv.pages`` (copies, forks, frees and
compaction of the cache's pages).  Their kernels live in libhsattn.so, loaded
through ``heteroserve._hip``.
"""

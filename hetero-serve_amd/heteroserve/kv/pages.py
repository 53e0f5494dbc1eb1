"""Pages of the paged cache while its sequences live: copies, forks, frees, compaction.

    copy_blocks        pool[:, :, dst] = pool[:, :, src], all layers, one launch
    find_free_blocks   the lowest blocks that nobody holds
    fork_blocks        children share their parent's full blocks and get a copy of
                       the last, unfinished one (parallel samples, beams)
    free_blocks        finished sequences give their blocks back
    compact_blocks     live blocks move into the lowest ids

The reference keeps counts and tables on the host (heteroserve/kv/blocks.py:62)
and copies pages between pools only.  Here the state is three int32 tensors that
stay on the device beside the pool, and every call runs in stream order without a
copy to the host, so a step that forks or frees can be captured in a graph:

    block_tables   [B, MB], -1 padded, as the attention reads them
    context_lens   [B]
    ref_counts     [num_blocks]: how many table rows (or other holders, such as a
                   prefix cache) keep a block; a block is free at 0

Row indexes and fresh blocks come as device tensors of integers, which are not read back
(one that names no row or block is skipped), or from the host, where they follow torch
indexing (but a fresh block of -1 is none, as from find_free_blocks) and mistakes
raise before anything is launched.  A mask is no list of rows, on either side.  copy_blocks reads its ids back, as the pack calls
do.
"""

from __future__ import annotations

from array import array

from .. import _hip
from .pack import _check_pool, _ids_tensor, _normalise_ids


def _host_ids(block_ids, num_blocks: int):
    """Block ids as an array("q"), wrapped and refused as _normalise_ids does.  A list of
    ids that need no wrapping, the usual case, takes no numpy call (16 ids: 1.5 us
    instead of 13)."""
    if type(block_ids) is list and block_ids:
        try:
            ids = array("q", block_ids)
            if 0 <= min(ids) and max(ids) < num_blocks:
                return ids
        except (TypeError, ValueError, OverflowError):
            pass
    return array("q", _normalise_ids(block_ids, num_blocks).tolist())


def copy_blocks(pool, src_ids, dst_ids) -> None:
    """pool[:, :, dst_ids[i]] = pool[:, :, src_ids[i]], bit for bit.  Ids follow
    torch indexing; a destination may not repeat nor be a source."""
    _hip.lib("KV copy HIP kernel")
    _check_pool(pool)
    src = _host_ids(src_ids, pool.shape[2])
    dst = _host_ids(dst_ids, pool.shape[2])
    n = len(src)
    if len(dst) != n:
        raise RuntimeError(f"{n} source blocks for {len(dst)} destinations")
    if n == 0:
        return
    to = set(dst)
    if len(to) != n:
        raise RuntimeError("a destination block repeats")
    if not to.isdisjoint(src):
        raise RuntimeError("a block is both source and destination")
    if 2 * n <= _hip.HOST_IDS:
        _hip.kv_copy_host_ids(pool, src, dst)
    else:
        both = _ids_tensor(src + dst, pool.device)
        _hip.kv_copy(pool, both[:n], both[n:])


def find_free_blocks(ref_counts, n: int):
    """int32 [n] on the device: the lowest blocks with a count of 0, ascending, -1
    past the last one.  Nothing is reserved until a count goes up."""
    n = int(n)
    if n < 0:
        raise RuntimeError("n must not be negative")
    if n >= 1 << 31:
        raise RuntimeError(f"n must be below 2^31, got {n}")
    return _hip.kv_find_free(ref_counts, n)


def _indexes(values, size: int, what: str, device, none: bool = False):
    """(int32 device tensor, host array or None): host values are checked and
    wrapped as torch indexing does, or, with none, -1 is kept and the only value
    below 0."""
    import torch

    if torch.is_tensor(values) and values.is_cuda:
        return _hip._whole_on(what, values if values.dim() == 1 else values.reshape(-1), device), None
    import numpy as np

    if torch.is_tensor(values):
        values = values.numpy() if values.dtype is torch.uint64 else values.tolist()
    host = np.asarray(values).reshape(-1)
    if host.size and host.dtype.kind not in "iu":
        raise RuntimeError(f"{what} must be integers, got {host.dtype}")
    bad = host >= size        # in the values' own type: past 2^63 is not below 0
    if host.dtype.kind == "i":
        bad |= host < (-1 if none else -size)
    if bad.any():
        i = int(host[int(np.argmax(bad))])
        raise IndexError(f"{what} index {i} is out of bounds for size {size}")
    host = host.astype(np.int64)
    if not none:
        host = np.where(host < 0, host + size, host)
    return torch.from_numpy(host.astype(np.int32)).to(device), host


def _repeats(ids) -> bool:
    return len(set(ids.tolist())) != len(ids)


def fork_blocks(pool, block_tables, context_lens, ref_counts, parents, children, fresh):
    """Row children[i] becomes a fork of row parents[i]: the full blocks are shared
    (counts up by 1), the tokens of the last, unfinished block are copied to block
    fresh[i] (count up by 1; unused where the parent's context ends with a
    block).  Changes block_tables, context_lens and ref_counts in place and returns
    int32 [n]: 1, or 0 where the fork could not be made (fresh[i] is -1 because
    the pool is full, or the parent's table has no last block), which leaves the
    child empty.

    A parent may have several children.  Children must be rows that hold no
    blocks, and must not repeat nor be parents; fresh blocks must not repeat."""
    _hip.lib("KV fork HIP kernel")
    _check_pool(pool)
    if block_tables.dim() != 2:
        raise RuntimeError("block_tables must be [B, max_blocks]")
    B, dev = block_tables.shape[0], pool.device
    parents, host_p = _indexes(parents, B, "parent row", dev)
    children, host_c = _indexes(children, B, "child row", dev)
    fresh, host_f = _indexes(fresh, pool.shape[2], "fresh block", dev, none=True)
    if host_c is not None and _repeats(host_c):
        raise RuntimeError("a child row repeats")
    if host_f is not None and _repeats(host_f[host_f >= 0]):
        raise RuntimeError("a fresh block repeats")
    if host_c is not None and host_p is not None and not set(host_c.tolist()).isdisjoint(host_p.tolist()):
        raise RuntimeError("a row is both parent and child")
    return _hip.kv_fork(pool, block_tables, context_lens, ref_counts, parents, children, fresh)


def free_blocks(block_tables, context_lens, ref_counts, rows) -> None:
    """Table rows `rows` give up their blocks: counts go down by 1 (never below 0),
    the rows become -1 and their context lengths 0, all in place.  A row that
    repeats is freed once."""
    _hip.lib("KV free HIP kernel")
    if block_tables.dim() != 2:
        raise RuntimeError("block_tables must be [B, max_blocks]")
    rows, _ = _indexes(rows, block_tables.shape[0], "row", ref_counts.device)
    _hip.kv_free(block_tables, context_lens, ref_counts, rows)


def compact_blocks(pool, block_tables, ref_counts):
    """The live blocks move into blocks [0, live), the highest into the lowest hole
    and so on, for all layers; block_tables and ref_counts follow in place.  Returns
    (moved_to int32 [num_blocks], live int32 [1]): every live block's new id, -1
    for the free ones, for whoever else keeps ids (a prefix cache's hashes)."""
    _hip.lib("KV compaction HIP kernel")
    _check_pool(pool)
    return _hip.kv_compact(pool, block_tables, ref_counts)

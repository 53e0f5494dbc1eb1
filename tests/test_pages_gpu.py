"""Copies, forks, frees and compaction of a cache's pages, bit for bit against
plain loops over the same arrays."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import operators as ops  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _pool(L, NB, BS, H, D, dtype=torch.bfloat16, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(L, 2, NB, BS, H, D, generator=gen, device=DEV).to(dtype)


def _words(x):
    return x.cpu().view(torch.int32 if x.element_size() == 4 else torch.int16).numpy()


def _dev(a):
    return torch.tensor(np.asarray(a, np.int32), device=DEV)


def _batch(rng, B, lens, MB, NB, BS, share=True):
    """Random tables for `lens` (rows from len(lens) on are empty), counts included."""
    tables = np.full((B, MB), -1, np.int32)
    refs = np.zeros(NB, np.int32)
    ids = rng.permutation(NB)
    at = 0
    for b, n in enumerate(lens):
        k = -(-n // BS)
        tables[b, :k] = ids[at:at + k]
        at += k
        if share and b and k > 1:      # the first block of the row before, if it is full
            if lens[b - 1] >= BS:
                tables[b, 0] = tables[b - 1, 0]
        np.add.at(refs, tables[b, :k], 1)
    ctx = np.zeros(B, np.int32)
    ctx[:len(lens)] = lens
    return tables, ctx, refs


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("L,NB,BS,H,D,n", [(3, 9, 16, 2, 64, 4), (1, 5, 5, 1, 7, 2), (2, 2000, 4, 1, 32, 700),
                                           (1, 4, 16, 12, 64, 1), (4, 40, 16, 8, 128, 20)])
def test_copy(dtype, L, NB, BS, H, D, n):
    from heteroserve.kv import pages

    pool = _pool(L, NB, BS, H, D, dtype)
    rng = np.random.default_rng(n)
    ids = rng.permutation(NB)
    src, dst = ids[:n].tolist(), ids[n:2 * n].tolist()
    src[-1] = src[0]                   # a source may repeat
    want = _words(pool).copy()
    want[:, :, dst] = want[:, :, src]
    pages.copy_blocks(pool, src, [d - NB if i % 2 else d for i, d in enumerate(dst)])
    assert np.array_equal(_words(pool), want)


def test_copy_through_the_allocator_and_refusals():
    from heteroserve.kv import pack, pages

    class Alloc(pack.HipKVMixin):
        pool = _pool(2, 6, 16, 2, 64)

    a = Alloc()
    want = _words(a.pool).copy()
    want[:, :, [4, 5]] = want[:, :, [0, 0]]
    a.copy_blocks([0, 0], torch.tensor([4, -1]))
    assert np.array_equal(_words(a.pool), want)
    pages.copy_blocks(a.pool, [], [])
    for src, dst, match in (([1], [2, 3], "destinations"), ([1, 2], [3, 3], "repeats"),
                            ([1, 2], [2, 3], "both source"), ([1, 2], [3, -3], "repeats")):
        with pytest.raises(RuntimeError, match=match):
            pages.copy_blocks(a.pool, src, dst)
    with pytest.raises(IndexError):
        pages.copy_blocks(a.pool, [0], [6])
    with pytest.raises(RuntimeError, match="contiguous"):
        pages.copy_blocks(a.pool[:, :, ::2], [0], [1])
    assert np.array_equal(_words(a.pool), want)


@pytest.mark.parametrize("NB", [1, 63, 4096, 4097, 9000, 70001])
@pytest.mark.parametrize("density", [0.0, 0.5, 0.999, 1.0])
def test_find_free(NB, density):
    from heteroserve.kv import pages

    rng = np.random.default_rng(NB)
    refs = (rng.random(NB) < density).astype(np.int32) * rng.integers(1, 4, NB).astype(np.int32)
    for n in (1, 7, 1500, NB + 3):
        got = pages.find_free_blocks(_dev(refs), n)
        assert np.array_equal(got.cpu().numpy(), ops.find_free(refs, n)), n
    # counts that start off a 16-byte boundary
    wide = _dev(np.concatenate([[0, 0, 0], refs]))
    assert np.array_equal(pages.find_free_blocks(wide[3:], 9).cpu().numpy(), ops.find_free(refs, 9))
    assert pages.find_free_blocks(_dev(refs), 0).shape == (0,)


def _fork_case(dtype, L, BS, H, D, lens, kids, seed, extra=0, NB=None):
    rng = np.random.default_rng(seed)
    n = len(lens) * kids
    MB = max(1, max(-(-x // BS) for x in lens)) + extra
    NB = NB or sum(-(-x // BS) for x in lens) + n + 5
    tables, ctx, refs = _batch(rng, len(lens) + n + 2, lens, MB, NB, BS)
    pool = _pool(L, NB, BS, H, D, dtype, seed)
    parents = np.repeat(np.arange(len(lens)), kids).astype(np.int32)
    children = (len(lens) + 1 + rng.permutation(n)).astype(np.int32)
    return pool, tables, ctx, refs, parents, children


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("L,BS,H,D,lens,kids", [
    (2, 16, 2, 64, [1, 16, 17, 0, 47], 2), (1, 5, 1, 7, [3, 5, 12], 3), (3, 8, 4, 128, [100, 64], 4),
    (1, 16, 1, 32, [5000], 2), (1, 32, 8, 128, [33], 1)])
def test_fork(dtype, L, BS, H, D, lens, kids):
    """Blocks that end inside a page, whole ones, empty parents, shared blocks,
    several children; host and device indexes."""
    from heteroserve.kv import pages

    for on_device in (False, True):
        pool, tables, ctx, refs, parents, children = _fork_case(dtype, L, BS, H, D, lens, kids, BS)
        want = [_words(pool).copy(), tables.copy(), ctx.copy(), refs.copy()]
        t, c, r = _dev(tables), _dev(ctx), _dev(refs)
        fresh = pages.find_free_blocks(r, len(parents))
        done = ops.fork(*want, parents, children, fresh.cpu().numpy())
        p, k = (_dev(parents), _dev(children)) if on_device else (parents.tolist(), children.tolist())
        got = pages.fork_blocks(pool, t, c, r, p, k, fresh if on_device else fresh.tolist())
        assert np.array_equal(got.cpu().numpy(), done) and done.all()
        for x, w in zip((_words(pool), t.cpu(), c.cpu(), r.cpu()), want):
            assert np.array_equal(np.asarray(x), w)


def test_fork_where_it_cannot_be_made():
    """A full pool, rows and blocks that are none, a last block that is padding, a
    context past the table, a row that is its own parent."""
    from heteroserve.kv import pages

    rng = np.random.default_rng(3)
    tables, ctx, refs = _batch(rng, 12, [20, 33, 40, 16], 3, 16, 16, share=False)
    ctx[2] = 1000                      # past the table: its 48 tokens count
    tables[1, 2] = -1                  # the last block is missing
    pool = _pool(2, 16, 16, 2, 64)
    parents = np.array([0, 0, 1, 2, 3, 99, 0, -7, 5], np.int32)
    children = np.array([5 - 1, 6, 7, 8, 9, 10, 77, 11, 5], np.int32)
    free = ops.find_free(refs, 6)      # 16 blocks, 9 of them held
    fresh = np.array([free[5], -1, free[4], -1, -1, free[3], free[2], free[1], free[0]], np.int32)
    want = [_words(pool).copy(), tables.copy(), ctx.copy(), refs.copy()]
    done = ops.fork(*want, parents, children, fresh)
    assert done.tolist() == [1, 0, 0, 1, 1, 0, 0, 0, 0]
    t, c, r = _dev(tables), _dev(ctx), _dev(refs)
    got = pages.fork_blocks(pool, t, c, r, _dev(parents), _dev(children), _dev(fresh))
    assert got.cpu().tolist() == done.tolist()
    for x, w in zip((_words(pool), t.cpu(), c.cpu(), r.cpu()), want):
        assert np.array_equal(np.asarray(x), w)


@pytest.mark.parametrize("B,MB,NB", [(5, 4, 40), (64, 300, 30000), (1, 1, 1)])
def test_free(B, MB, NB):
    """Shared blocks lose one holder each; rows that repeat, rows that are none,
    entries that are no blocks, counts that are 0 already."""
    from heteroserve.kv import pages

    rng = np.random.default_rng(B)
    tables = np.full((B, MB), -1, np.int32)
    refs = np.zeros(NB, np.int32)
    for b in range(B):
        k = int(rng.integers(0, MB + 1))
        tables[b, :k] = rng.permutation(NB)[:k]
        np.add.at(refs, tables[b, :k], 1)
    refs[rng.integers(0, NB, 3)] = 0
    if MB > 2:
        tables[0, 1], tables[B - 1, 0] = NB, 2 ** 31 - 1
    ctx = rng.integers(1, 99, B).astype(np.int32)
    rows = rng.permutation(B)[:(B + 1) // 2].astype(np.int32)
    t, c, r = _dev(tables), _dev(ctx), _dev(refs)
    ops.free(tables, ctx, refs, rows)
    pages.free_blocks(t, c, r, _dev(np.concatenate([rows, rows[:1], [-1, B, 2 ** 31 - 1]])))
    assert np.array_equal(t.cpu(), tables) and np.array_equal(c.cpu(), ctx)
    assert np.array_equal(r.cpu(), refs)
    pages.free_blocks(t, c, r, [b - B for b in range(B)])      # the rest, from the host
    assert (t.cpu() == -1).all() and (c.cpu() == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("L,NB,BS,H,D,density", [
    (2, 50, 16, 2, 64, 0.4), (1, 33, 5, 1, 7, 0.5), (1, 9000, 2, 1, 16, 0.3), (3, 20, 16, 8, 128, 0.9),
    (1, 64, 16, 1, 32, 0.0), (1, 64, 16, 1, 32, 1.0), (1, 1, 16, 1, 32, 1.0)])
def test_compact(dtype, L, NB, BS, H, D, density):
    from heteroserve.kv import pages

    rng = np.random.default_rng(NB)
    refs = ((rng.random(NB) < density) | (density == 1.0)).astype(np.int32) * rng.integers(1, 5, NB).astype(np.int32)
    tables = rng.integers(-1, NB, (6, 11)).astype(np.int32)     # some name free blocks
    tables[0, 0], tables[1, 1] = NB, -5
    pool = _pool(L, NB, BS, H, D, dtype)
    want = [_words(pool).copy(), tables.copy(), refs.copy()]
    t, r = _dev(tables), _dev(refs)
    moved, live = ops.compact(*want)
    got_moved, got_live = pages.compact_blocks(pool, t, r)
    assert got_live.item() == live
    assert np.array_equal(got_moved.cpu(), moved)
    for x, w in zip((_words(pool), t.cpu(), r.cpu()), want):
        assert np.array_equal(np.asarray(x), w)
    pages.compact_blocks(pool, t, r)                            # nothing left to move
    for x, w in zip((_words(pool), t.cpu(), r.cpu()), want):
        assert np.array_equal(np.asarray(x), w)


def test_replayed_in_a_graph():
    """Fork, free and compaction of one step, captured: every replay does what the
    eager calls do from the same state."""
    from heteroserve.kv import pages

    pool, tables, ctx, refs, parents, children = _fork_case(torch.bfloat16, 2, 16, 2, 64, [20, 50], 2, 1)
    state = [pool, _dev(tables), _dev(ctx), _dev(refs)]
    first = [x.clone() for x in state]
    p, k, done = _dev(parents), _dev(children), _dev([0])

    def step():
        fresh = pages.find_free_blocks(state[3], len(parents))
        forked = pages.fork_blocks(*state, p, k, fresh)
        pages.free_blocks(*state[1:], done)
        moved, live = pages.compact_blocks(state[0], state[1], state[3])
        return fresh, forked, moved, live

    want = [x.clone() for x in step()]
    after = [x.clone() for x in state]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        for x, y in zip(state, first):
            x.copy_(y)
        for x in got:
            x.fill_(-9)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, w in zip((*got, *state), (*want, *after)):
            assert torch.equal(x, w)


def test_refusals():
    from heteroserve.kv import pages

    pool = _pool(1, 8, 16, 1, 32)
    t, c, r = _dev(np.full((4, 2), -1)), _dev(np.zeros(4)), _dev(np.zeros(8))

    def refused(match, call, *args, err=RuntimeError):
        with pytest.raises(err, match=match):
            call(*args)

    fork, free = pages.fork_blocks, pages.free_blocks
    refused("child row repeats", fork, pool, t, c, r, [0, 0], [1, 1], [0, 1])
    refused("fresh block repeats", fork, pool, t, c, r, [0, 0], [1, 2], [3, 3])
    refused("both parent and child", fork, pool, t, c, r, [0, 1], [1, 2], [0, 1])
    refused("same length", fork, pool, t, c, r, [0], [1, 2], [0, 1])
    refused("out of bounds", fork, pool, t, c, r, [4], [1], [0], err=IndexError)
    refused("out of bounds", fork, pool, t, c, r, [0], [1], [8], err=IndexError)
    refused("integers", fork, pool, t, c, r, [0.5], [1], [0])
    refused("written in place", fork, pool, t.long(), c, r, [0], [1], [0])
    refused("written in place", fork, pool, t.t(), c, r, [0], [1], [0])
    refused("one per block", fork, pool, t, c, r[:7], [0], [1], [0])
    refused("per table row", free, t, c[:3], r, [0])
    refused("out of bounds", free, t, c, r, [-5], err=IndexError)
    refused("on CUDA", free, t.cpu(), c, r, [0])
    refused("must not be negative", pages.find_free_blocks, r, -1)
    refused("written in place", pages.find_free_blocks, r.long(), 1)
    refused("one entry per block", pages.compact_blocks, pool, t, r[:7])
    refused("contiguous", pages.compact_blocks, pool[:, :, ::2], t, r)
    assert (t.cpu() == -1).all() and (r.cpu() == 0).all()


def test_no_fresh_block_from_the_host_is_no_block():
    """-1 of find_free_blocks, brought to the host and back, is not the last block."""
    from heteroserve.kv import pages

    rng = np.random.default_rng(3)
    tables, ctx, refs = _batch(rng, 8, [20, 32], 3, 5, 16, share=False)
    refs[:] = np.maximum(refs, (np.arange(5) < 4))          # a full pool but for one block or none
    pool = _pool(1, 5, 16, 2, 64)
    want = [_words(pool).copy(), tables.copy(), ctx.copy(), refs.copy()]
    fresh = [-1, -1, -1]
    done = ops.fork(*want, [0, 0, 1], [4, 5, 6], fresh)
    assert done.tolist() == [0, 0, 1]
    t, c, r = _dev(tables), _dev(ctx), _dev(refs)
    got = pages.fork_blocks(pool, t, c, r, [0, 0, 1], [4, 5, 6], fresh)
    assert got.tolist() == done.tolist()
    for x, w in zip((_words(pool), t.cpu(), c.cpu(), r.cpu()), want):
        assert np.array_equal(np.asarray(x), w)
    with pytest.raises(IndexError, match="fresh block index -2"):
        pages.fork_blocks(pool, t, c, r, [0], [4], [-2])
    with pytest.raises(RuntimeError, match="2\\^31"):
        pages.find_free_blocks(r, 2 ** 31)


def test_copies_replayed_in_a_graph():
    """Block ids of a captured copy are the graph's own: replays copy what the pool then
    holds."""
    from heteroserve.kv import pages

    pool = _pool(2, 9, 16, 2, 64)
    src, dst = [0, 1, 1], [6, 7, 8]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pages.copy_blocks(pool, src, dst)
    src[:], dst[:] = [5, 5, 5], [2, 3, 4]
    for i in range(3):
        pool.copy_(_pool(2, 9, 16, 2, 64, seed=i))
        want = pool.clone()
        want[:, :, 6:] = want[:, :, [0, 1, 1]]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(pool, want)


def test_copies_of_pages_that_are_no_multiples_of_16_bytes_and_of_bytes():
    from heteroserve.kv import pages

    for shape, dtype in (((2, 2, 6, 3, 1, 5), torch.float16), ((1, 2, 6, 16, 1, 8), torch.uint8),
                         ((1, 2, 6, 5, 1, 3), torch.uint8)):
        pool = torch.randint(0, 120, shape, device=DEV).to(dtype)
        want = pool.clone()
        want[:, :, [4, 0]] = want[:, :, [2, 5]]
        pages.copy_blocks(pool, [2, 5], [4, 0])
        assert torch.equal(pool, want)

"""The operators together, as a server uses them: prompts are rotated into the paged
cache and attended to, their sequences are forked into samples, the samples decode a
token each, some finish, and the pool is compacted.

Every attention is compared with 64-bit arithmetic on what the cache holds: 1e-5 for
float32 and float16 caches and 5e-5 for bfloat16 ones, the decode kernels' own
bounds (their two-term operands carry 16 bits of a bf16 cache's products)."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import operators as ops  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DECODE_TOL = {F32: 1e-5, F16: 1e-5, BF16: 5e-5}
H, HKV, D, BS, L, B, MB, NB = 8, 2, 64, 16, 2, 12, 8, 64
SCALE = D ** -0.5


def _dev(a):
    return torch.tensor(np.asarray(a, np.int32), device=DEV)


def _rows(n, dtype, gen):
    """Slices of one fused projection's rows."""
    x = torch.randn(n, (H + 2 * HKV) * D, generator=gen, device=DEV).to(dtype)
    q, k, v = x.split([H * D, HKV * D, HKV * D], 1)
    return q.view(n, H, D), k.view(n, HKV, D), v.view(n, HKV, D)


class _Server:
    """The state on the device; the steps are all the framework's calls."""

    def __init__(self, dtype, interleaved, seed=1):
        from heteroserve.kv import rotary

        self.gen = torch.Generator(device=DEV).manual_seed(seed)
        self.dtype, self.interleaved = dtype, interleaved
        self.pool = torch.zeros(L, 2, NB, BS, HKV, D, dtype=dtype, device=DEV)
        self.tables = torch.full((B, MB), -1, dtype=torch.int32, device=DEV)
        self.ctx = torch.zeros(B, dtype=torch.int32, device=DEV)
        self.refs = torch.zeros(NB, dtype=torch.int32, device=DEV)
        self.freq = (10000.0 ** (-torch.arange(D // 2, device=DEV) / (D // 2))).float()
        self.axes = rotary.axes_of([16, 8, 8], interleaved=True).to(DEV)

    def hold(self, rows, lens):
        """Blocks for contexts of `lens` tokens of table rows that hold none."""
        from heteroserve.kv import pages

        need = [-(-n // BS) for n in lens]
        got = pages.find_free_blocks(self.refs, sum(need))
        at = 0
        for r, k in zip(rows, need):
            self.tables[r, :k] = got[at:at + k]
            at += k
        self.refs[got.long()] += 1

    def write(self, layer, q, k, v, at, seq, out_dtype=None, keep_k=False):
        from heteroserve.kv import rotary

        where = torch.stack([at, at // 2, at % 3])     # a time, a height and a width
        return rotary.rotate_append_kv(q, k, v, where, self.freq, self.pool[layer, 0],
                                       self.pool[layer, 1], self.tables, at, seq, axes=self.axes,
                                       interleaved=self.interleaved, out_dtype=out_dtype, keep_k=keep_k)

    def cached(self, layer, row, n):
        """(k, v) float64 [n, HKV, D]: what the cache holds of a sequence."""
        ids = self.tables[row, :-(-n // BS)].long()
        return [self.pool[layer, c][ids].reshape(-1, HKV, D)[:n].double().cpu().numpy() for c in (0, 1)]

    def decode(self, layer, q):
        from heteroserve.model import paged_attn

        return paged_attn.paged_attention(q, self.pool[layer, 0], self.pool[layer, 1], self.tables,
                                          self.ctx, SCALE)

    def check_decode(self, layer, q, got):
        for b, n in enumerate(self.ctx.tolist()):
            if not n:
                continue
            k, v = self.cached(layer, b, n)
            s = np.einsum("hd,nhd->hn", q[b].double().cpu().numpy(), k.repeat(H // HKV, 1)) * SCALE
            p = np.exp(s - s.max(1, keepdims=True))
            want = np.einsum("hn,nhd->hd", p / p.sum(1, keepdims=True), v.repeat(H // HKV, 1))
            err = np.abs(got[b].double().cpu().numpy() - want).max()
            assert err <= DECODE_TOL[self.dtype], (layer, b, n, err)

    def check_counts(self):
        held = torch.zeros(NB, dtype=torch.int64, device=DEV)
        ids = self.tables[self.tables >= 0].long()
        held.index_add_(0, ids, torch.ones_like(ids))
        assert torch.equal(held, self.refs.long())


def _check_prompts(q, k, v, got, cu, dtype):
    """q, k, v: what the kernel was given.  With u = 2^-24: a score is off by (D + 4) u S
    for S = the largest sum |q k| scale, an exponential by 4 u more, a sum of n <= 64
    terms by 64 u; the output by twice their sum times sum P |v|.  16 bits: the
    probabilities rounded (below fp16's normal range by 2^-25 |v| each), and the output."""
    q, k, v, got = (x.double().cpu().numpy() for x in (q, k, v, got))
    want, spread = ops.prompt(q, k, v, cu, SCALE)
    S = (np.abs(q).max(axis=(0, 1)) * np.abs(k).max(axis=(0, 1))).sum() * SCALE
    rel = 2 * (2 * (D + 4) * 2.0 ** -24 * S + 4 * 2.0 ** -24 + 64 * 2.0 ** -24)
    tol = rel * spread
    if dtype is not F32:
        half = torch.finfo(dtype).eps / 2
        tol = tol + half * spread * (1 + rel) + half * (np.abs(want) + tol) + 2.0 ** -25 * (64 * np.abs(v).max() + 1)
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_prompts_samples_and_compaction(dtype, interleaved):
    from heteroserve.kv import pages
    from heteroserve.model.prompt_attn import prompt_attention

    s = _Server(dtype, interleaved)
    lens = [40, 1, 64, 17]                   # ends inside a page, one token, whole pages
    rows = [5, 2, 7, 0]                      # their table rows, in no order
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    at = _dev(np.concatenate([np.arange(n) for n in lens]))
    seq = _dev(np.repeat(rows, lens))
    s.hold(rows, lens)
    for r, n in zip(rows, lens):
        s.ctx[r] = n
    for layer in range(L):
        q, k, v = _rows(sum(lens), dtype, s.gen)
        qr, kr = s.write(layer, q, k, v, at, seq, keep_k=True)
        where = np.stack([at.cpu().numpy(), at.cpu().numpy() // 2, at.cpu().numpy() % 3])
        eps = torch.finfo(dtype).eps / 2
        for x, y in ((q, qr), (k, kr)):
            x = x.double().cpu().numpy()
            want = ops.rotate(x, where, s.freq.cpu().numpy(), s.axes.cpu().numpy(), interleaved)
            # below 2^-20 (|a| + |b|) in fp32, then rounded once
            assert (np.abs(y.double().cpu().numpy() - want) <= (eps + 2.0 ** -20) * 2 * np.abs(x).max()).all()
        for b, r in enumerate(rows):         # the cache holds what the attention gets
            kc, vc = s.cached(layer, r, lens[b])
            assert np.array_equal(kc, kr[cu[b]:cu[b + 1]].double().cpu().numpy())
            assert np.array_equal(vc, v[cu[b]:cu[b + 1]].double().cpu().numpy())
        got = prompt_attention(qr, kr, v, torch.tensor(cu, device=DEV), max(lens), SCALE)
        _check_prompts(qr, kr, v, got, cu, dtype)

    # two samples of three of them; the parents keep their blocks
    parents, children = [5, 5, 7, 7, 0, 0], [1, 3, 4, 6, 8, 9]
    before = s.pool.clone()
    fresh = pages.find_free_blocks(s.refs, len(parents))
    assert pages.fork_blocks(s.pool, s.tables, s.ctx, s.refs, parents, children, fresh).tolist() == [1] * 6
    s.check_counts()
    for p, c in zip(parents, children):
        n = int(s.ctx[p])
        assert int(s.ctx[c]) == n
        for layer in range(L):
            for x, y in zip(s.cached(layer, p, n), s.cached(layer, c, n)):
                assert np.array_equal(x, y)

    # a token each: a context that ends with a page needs a new one first
    full = [b for b in parents + children + [2] if int(s.ctx[b]) % BS == 0 and int(s.ctx[b])]
    full = sorted(set(full))
    new = pages.find_free_blocks(s.refs, len(full))
    for b, block in zip(full, new):
        s.tables[b, int(s.ctx[b]) // BS] = block
        s.refs[block.long()] += 1
    s.check_counts()
    live = torch.nonzero(s.ctx).flatten().int()
    step = s.ctx[live.long()].clone()
    s.ctx[live.long()] += 1
    queries = []
    for layer in range(L):
        q, k, v = _rows(len(live), dtype, s.gen)
        turned, none = s.write(layer, q, k, v, step, live, out_dtype=F32)
        assert none is None
        queries.append(torch.zeros(B, H, D, device=DEV).index_copy_(0, live.long(), turned))
        s.check_decode(layer, queries[layer], s.decode(layer, queries[layer]))
    # nobody wrote into a page that somebody else reads: the shared full pages are as they were
    shared = (s.refs > 1).nonzero().flatten()
    assert len(shared) and torch.equal(s.pool[:, :, shared], before[:, :, shared])

    # parents and one sample finish; the pool shrinks, and nothing else changes
    pages.free_blocks(s.tables, s.ctx, s.refs, [5, 7, 0, 3])
    s.check_counts()
    want = [s.decode(layer, queries[layer]) for layer in range(L)]
    moved, n_live = pages.compact_blocks(s.pool, s.tables, s.refs)
    s.check_counts()
    assert int((s.refs > 0).sum()) == int(n_live) == int((s.refs[:int(n_live)] > 0).sum())
    assert int((moved >= 0).sum()) == int(n_live) and int(moved.max()) == int(n_live) - 1
    for layer in range(L):
        got = s.decode(layer, queries[layer])
        alive = s.ctx > 0
        assert torch.equal(got[alive], want[layer][alive])
        s.check_decode(layer, queries[layer], got)
    pages.free_blocks(s.tables, s.ctx, s.refs, list(range(B)))
    assert not s.refs.any() and not s.ctx.any()


def test_a_captured_step_beside_eager_work():
    """One decode step (rotate, write, attend) in a graph, replayed from different
    states, with the pages' eager calls between: as the eager steps, bit for bit."""
    from heteroserve.kv import pages

    runs = []
    for captured in (False, True):
        s = _Server(BF16, False, seed=4)
        lens = [33, 50]
        s.hold([0, 1], [n + 12 for n in lens])
        s.ctx[:2] = _dev(lens)
        s.pool.normal_(generator=s.gen)
        x = torch.empty(B, (H + 2 * HKV) * D, dtype=BF16, device=DEV)
        q, k, v = x.split([H * D, HKV * D, HKV * D], 1)
        q, k, v = q.view(B, H, D), k.view(B, HKV, D), v.view(B, HKV, D)

        def step():
            # empty rows have no block at position 0: their tokens are not written
            turned, _ = s.write(1, q, k, v, s.ctx, None, out_dtype=F32)
            s.ctx += (s.ctx > 0).int()
            return s.decode(1, turned)

        x.normal_(generator=s.gen)
        if captured:
            state = [t.clone() for t in (s.pool, s.ctx)]
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step()
            s.pool.copy_(state[0])
            s.ctx.copy_(state[1])
        got = []
        for i in range(4):
            x.normal_(generator=s.gen)
            torch.cuda.synchronize()
            if captured:
                graph.replay()
            else:
                out = step()
            torch.cuda.synchronize()
            got.append(out.clone())
            if i == 0:
                fresh = pages.find_free_blocks(s.refs, 2)
                pages.fork_blocks(s.pool, s.tables, s.ctx, s.refs, [0, 1], [4, 3], fresh)
            if i == 1:
                pages.free_blocks(s.tables, s.ctx, s.refs, [0])
                pages.compact_blocks(s.pool, s.tables, s.refs)
        runs.append([*got, s.pool, s.tables, s.ctx, s.refs])
    for i, (a, b) in enumerate(zip(*runs)):
        assert torch.equal(a, b), i

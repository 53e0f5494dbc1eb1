"""The 4-bit cache and the window together, as a server uses them: prompts are written in 4
bits and decoded over, their prefixes are read back for the next turn's prefill, old pages
behind a window are given back; in graphs, on streams, in threads and far into large
caches.

Tolerances of the attention are those of arithmetic in fp32 on what the caches hold: (D +
64) 2^-23 of the scores' sizes, which move a row by p |v - out|, and (n + 64) 2^-23 of sum
p |v|.  Calls that run the same kernels on the same values in the same order are compared
bit for bit."""

from __future__ import annotations

import threading

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import long_context as lc  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
H, HKV, BS = 8, 2, 16


def _np(x):
    return x.double().cpu().numpy()


def _dev(a):
    return torch.tensor(np.asarray(a, np.int32), device=DEV)


def _check(q, got, k, v, D, sizes=(None, None)):
    """One sequence's rows against 64 bits, of the visible keys and values."""
    want, spread, weight = lc.decode(_np(q), k, v, D ** -0.5, *sizes)
    tol = (D + 64) * 2.0 ** -23 * weight + (len(k) + 64) * 2.0 ** -23 * spread
    assert (np.abs(_np(got) - want) <= tol).all()


class _Chat:
    """Sequences in a pool of L layers: tables, lengths and the steps, in 4 bits or in dtype."""

    def __init__(self, lens, room, D, dtype, q4, L=1, seed=0):
        from heteroserve.kv import quant

        self.gen = torch.Generator(DEV).manual_seed(seed)
        self.D, self.dtype, self.q4, self.L = D, dtype, q4, L
        B = len(lens)
        self.MB = -(-(max(lens) + room) // BS)
        order = np.random.default_rng(seed).permutation(B * self.MB + 2)[:B * self.MB]
        self.tables = _dev(order.reshape(B, self.MB))
        if q4:
            self.pool = quant.empty_pool_q4(L, B * self.MB + 2, BS, HKV, D, device=DEV)
        else:
            self.pool = torch.zeros(L, 2, B * self.MB + 2, BS, HKV, D, dtype=dtype, device=DEV)
        self.ctx = torch.zeros(B, dtype=torch.int32, device=DEV)
        self.fill(lens)

    def rows(self, n):
        """q, k, v as slices of a fused projection's rows."""
        D = self.D
        x = torch.randn(n, (H + 2 * HKV) * D, generator=self.gen, device=DEV).to(self.dtype)
        q, k, v = x.split([H * D, HKV * D, HKV * D], 1)
        return q.view(n, H, D), k.view(n, HKV, D), v.view(n, HKV, D)

    def write(self, layer, at, k, v, seq=None):
        from heteroserve.kv import pack, quant

        call = quant.append_kv_q4 if self.q4 else pack.append_kv
        call(self.pool[layer, 0], self.pool[layer, 1], self.tables, at, k, v, seq_ids=seq)

    def fill(self, lens):
        at, seq = _dev(np.concatenate([np.arange(n) for n in lens])), _dev(np.repeat(np.arange(len(lens)), lens))
        self.written = []
        for layer in range(self.L):
            _, k, v = self.rows(len(at))
            self.write(layer, at, k, v, seq)
            self.written.append((k, v))
        self.ctx.copy_(_dev(lens))

    def attend(self, layer, q, window=0, sinks=0):
        from heteroserve.model.paged_attn_q4 import paged_attention_q4
        from heteroserve.model.paged_attn_window import paged_attention_window

        args = (q.float(), self.pool[layer, 0], self.pool[layer, 1], self.tables, self.ctx, self.D ** -0.5)
        return (paged_attention_q4 if self.q4 else paged_attention_window)(*args, window, sinks)

    def step(self, x, window=0, sinks=0):
        """A token of every sequence through all layers, from one fused projection's rows."""
        D = self.D
        q, k, v = x.split([H * D, HKV * D, HKV * D], 1)
        for layer in range(self.L):
            self.write(layer, self.ctx, k, v)
        self.ctx += 1
        return torch.stack([self.attend(layer, q.view(-1, H, D), window, sinks) for layer in range(self.L)])

    def held(self, layer, b, at):
        """(records or rows) of keys and values at positions `at` of sequence b."""
        page = self.tables[b].long()[torch.tensor(at // BS, device=DEV)]
        return [self.pool[layer, c][page, torch.tensor(at % BS, device=DEV)].cpu() for c in (0, 1)]

    def check(self, layer, q, got, window=0, sinks=0):
        for b, n in enumerate(self.ctx.tolist()):
            k, v = self.held(layer, b, lc.visible(n, window, sinks))
            if self.q4:
                k, v = k.numpy(), v.numpy()
                _check(q[b], got[b], lc.values(k, True), lc.values(v, False), self.D,
                       (lc.sizes(k, True), lc.sizes(v, False)))
            else:
                _check(q[b], got[b], _np(k), _np(v), self.D)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
def test_a_second_turn(dtype, D):
    """Prompts into 4 bits, decode steps with and without a window, then the second turn:
    the cached prefixes are read back as a paged cache of 16 or 32 bits, padded to whole
    pages, the new chunks written behind them, and the chunks prefilled over both."""
    from heteroserve.kv import pack, quant
    from heteroserve.model.paged_attn_prefill import paged_attention_prefill_varlen

    lens = [70, 1, 33, 16]
    s = _Chat(lens, 40, D, dtype, True, L=2, seed=D)
    for layer in range(2):
        k, v = s.written[layer]
        for b in range(4):
            cut = slice(sum(lens[:b]), sum(lens[:b + 1]))
            for i, (got, x) in enumerate(zip(s.held(layer, b, np.arange(lens[b])), (k[cut], v[cut]))):
                assert np.array_equal(got.numpy(), lc.records(*lc.quantise(_np(x)), keys=i == 0))
    for i in range(3):
        window, sinks = ((0, 0), (20, 2), (1, 0))[i]
        x = torch.randn(4, (H + 2 * HKV) * D, generator=s.gen, device=DEV).to(dtype)
        out = s.step(x, window, sinks)
        for layer in range(2):
            s.check(layer, x[:, :H * D].reshape(4, H, D), out[layer], window, sinks)

    had, new = s.ctx.tolist(), [5, 20, 1, 17]
    pages = [-(-(n + m) // BS) for n, m in zip(had, new)]
    tables = torch.full((4, max(pages)), -1, dtype=torch.int32)
    at, seq = [], []
    for b in range(4):
        tables[b, :pages[b]] = torch.arange(pages[b]) + sum(pages[:b])
        here = np.arange(pages[b] * BS)
        at.append(np.where(here < had[b], here, -1))      # zeros behind the prefix
        seq.append(np.full(pages[b] * BS, b))
    at, seq = _dev(np.concatenate(at)), _dev(np.concatenate(seq))
    tables = tables.to(DEV)
    chunk_at = _dev(np.concatenate([n + np.arange(m) for n, m in zip(had, new)]))
    chunk_seq = _dev(np.repeat(np.arange(4), new))
    for layer in range(2):
        k, v = quant.read_kv_q4(s.pool[layer, 0], s.pool[layer, 1], s.tables, at, seq, dtype=dtype)
        k, v = k.view(-1, BS, HKV, D), v.view(-1, BS, HKV, D)
        q, k_new, v_new = s.rows(sum(new))
        pack.append_kv(k, v, tables, chunk_at, k_new, v_new, seq_ids=chunk_seq)
        s.write(layer, chunk_at, k_new, v_new, chunk_seq)
        cu = _dev(np.concatenate([[0], np.cumsum(new)]))
        got = paged_attention_prefill_varlen(q.float().contiguous(), cu, max(new), k, v, tables,
                                             s.ctx + _dev(new), D ** -0.5, use_mfma=dtype is not F32)
        for b in range(4):
            ids = tables[b, :pages[b]].long()
            kk, vv = (_np(x[ids].reshape(-1, HKV, D)) for x in (k, v))
            for i, x in enumerate(s.held(layer, b, np.arange(had[b]))):
                want = torch.tensor(lc.values(x.numpy(), i == 0)).to(F32).to(dtype)
                assert np.array_equal((kk, vv)[i][:had[b]], _np(want))
            for i in range(new[b]):
                n, row = had[b] + i + 1, sum(new[:b]) + i
                want = lc.decode(_np(q[row]), kk[:n], vv[:n], D ** -0.5)[0]
                # the prefill kernels' own bound
                np.testing.assert_allclose(_np(got[row]), want, rtol=1e-3, atol=1e-3)
    s.ctx += _dev(new)
    q = s.rows(4)[0]
    for layer in range(2):
        s.check(layer, q, s.attend(layer, q))


@pytest.mark.parametrize("q4,dtype,D", [(True, F16, 64), (False, F32, 64), (False, BF16, 128), (False, F16, 256)])
def test_pages_behind_the_window_are_given_back(q4, dtype, D):
    """A decode step after step: pages that the window has left (and no sink lies in) lose
    their entry and are filled with what would show."""
    window, sinks = 24, 3
    s = _Chat([60, 5, 0], 24, D, dtype, q4, seed=3)
    s.ctx[2] = 0
    for i in range(20):
        x = torch.randn(3, (H + 2 * HKV) * D, generator=s.gen, device=DEV).to(dtype)
        out = s.step(x, window, sinks)
        s.check(0, x[:, :H * D].reshape(3, H, D), out[0], window, sinks)
        for b, n in enumerate(s.ctx.tolist()):
            for j in range(1, max(0, n - window) // BS):
                block = int(s.tables[b, j])
                if block >= 0:
                    s.pool[:, :, block] = 0xff if q4 else float("nan")
                    s.tables[b, j] = -1
    assert int((s.tables < 0).sum()) >= 2


def _states(s):
    return [s.pool.clone(), s.ctx.clone()]


@pytest.mark.parametrize("q4,dtype,D,window,sinks", [(True, BF16, 128, 0, 0), (True, F32, 64, 900, 4),
                                                     (False, BF16, 64, 900, 4), (False, F32, 32, 700, 1),
                                                     (False, F16, 256, 900, 0)])
def test_a_captured_step_beside_eager_work(q4, dtype, D, window, sinks):
    """A step of two layers in a graph, replayed with eager calls of the same sizes, and
    another graph's replays, between: as the eager steps, bit for bit.  Rows are of several
    parts, so both have workspaces."""
    runs = []
    for captured in (False, True):
        s = _Chat([2000, 3, 911], 20, D, dtype, q4, L=2, seed=7)
        x = torch.zeros(3, (H + 2 * HKV) * D, dtype=dtype, device=DEV)
        start = _states(s)
        graphs = []
        if captured:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                s.step(x, window, sinks)
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            for _ in range(2):
                graphs.append(torch.cuda.CUDAGraph())
                with torch.cuda.graph(graphs[-1]):
                    out = s.step(x, window, sinks)
                graphs.append(out)
            s.pool.copy_(start[0])
            s.ctx.copy_(start[1])
        got = []
        for i in range(5):
            x.normal_(generator=s.gen)
            torch.cuda.synchronize()
            if captured:
                which = i % 2 * 2
                graphs[which].replay()
                out = graphs[which + 1]
            else:
                out = s.step(x, window, sinks)
            got.append(out.clone())
            # eager work on the same sizes, and on others
            q = torch.ones(3, H, D, device=DEV)
            got.append(s.attend(0, q, window, sinks))
            got.append(s.attend(1, q[:, :HKV].contiguous(), 5, 0))
        runs.append(got + _states(s))
    for i, (a, b) in enumerate(zip(*runs)):
        assert torch.equal(a, b), i


@pytest.mark.parametrize("q4", [True, False])
def test_two_streams_and_two_threads(q4):
    """Calls at once share no workspace."""
    chats = [_Chat([1500, 20 + i], 20, 64, BF16, q4, seed=20 + i) for i in range(2)]
    qs = [torch.randn(2, H, 64, generator=s.gen, device=DEV) for s in chats]
    want = [s.attend(0, q, 1200, 2) for s, q in zip(chats, qs)]
    streams = [torch.cuda.Stream() for _ in chats]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (s, q) in enumerate(zip(chats, qs)):
            with torch.cuda.stream(streams[i]):
                got[i].append(s.attend(0, q, 1200, 2))
    torch.cuda.synchronize()

    def run(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(10):
                got[i].append(chats[i].attend(0, qs[i], 1200, 2))
            streams[i].synchronize()

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        assert len(got[i]) == 20
        assert all(torch.equal(x, want[i]) for x in got[i])


@pytest.mark.parametrize("q4,dtype,D", [(True, BF16, 128), (True, F16, 32), (False, BF16, 128), (False, F32, 64),
                                        (False, F16, 256)])
def test_far_into_a_large_cache(q4, dtype, D):
    """Pages past 2^32 bytes give what the same pages near a cache's start give, written, read
    and attended to."""
    from heteroserve.kv import pack, quant

    row = HKV * (D // 2 + D // 8 if q4 else D * torch.finfo(dtype).bits // 8)
    NB = 2 ** 32 // (BS * row) + 40
    shape = (BS, HKV, D // 2 + D // 8) if q4 else (BS, HKV, D)
    kind = torch.uint8 if q4 else dtype
    gen = torch.Generator(DEV).manual_seed(D)
    n = 300
    k, v = (torch.randn(n, HKV, D, generator=gen, device=DEV).to(dtype) for _ in range(2))
    q = torch.randn(1, H, D, generator=gen, device=DEV)
    outs = []
    for blocks, first in ((30, 5), (NB, NB - 25)):
        cache = torch.empty(2, blocks, *shape, dtype=kind, device=DEV)
        bt = torch.arange(first, first + 20, dtype=torch.int32, device=DEV).flip(0)[None]
        cache[:, first:first + 20] = 0
        at, seq = torch.arange(n, device=DEV, dtype=torch.int32), torch.zeros(n, dtype=torch.int32, device=DEV)
        (quant.append_kv_q4 if q4 else pack.append_kv)(cache[0], cache[1], bt, at, k, v, seq_ids=seq)
        out = [cache[:, first:first + 20].clone()]
        if q4:
            from heteroserve.model.paged_attn_q4 import paged_attention_q4 as attend

            out += quant.read_kv_q4(cache[0], cache[1], bt, at, seq_ids=seq, dtype=F32)
        else:
            from heteroserve.model.paged_attn_window import paged_attention_window as attend
        for window in (0, 100):
            out.append(attend(q, cache[0], cache[1], bt, torch.tensor([n]), 0.1, window, 3))
        outs.append(out)
        del cache
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    assert outs[0][0].any() and torch.isfinite(outs[0][-1]).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_window_rounding_errors_average_out(dtype, D):
    """Second and third terms are there: of 300 keys, probabilities are off by up to 2^-20 and
    products by 2^-22, which leaves 2^-24 of the sum of their sizes where errors do not depend
    on one another, and sums of 10 chunks' products rounded to 2^-24 about 2^-23.  A missing
    second fp16 term (2^-12 of each product) leaves 2^-17, a missing third bf16 one
    (2^-18) 2^-23 and is not told apart, a missing second one (2^-9) 2^-14."""
    from heteroserve.model.paged_attn_window import paged_attention_window

    gen = torch.Generator(DEV).manual_seed(D)
    B, n, pages = 24, 300, 19
    cache = torch.randn(2, B * pages, BS, HKV, D, generator=gen, device=DEV).to(dtype)
    q = torch.randn(B, H, D, generator=gen, device=DEV)
    bt = torch.arange(B * pages, device=DEV).view(B, pages)
    got = _np(paged_attention_window(q, cache[0], cache[1], bt, torch.full((B,), n), D ** -0.5, 0))
    err = size = 0.0
    for b in range(B):
        k, v = (_np(cache[c, b * pages:(b + 1) * pages].reshape(-1, HKV, D)[:n]) for c in (0, 1))
        want, spread, _ = lc.decode(_np(q[b]), k, v, D ** -0.5)
        err += ((got[b] - want) ** 2).sum()
        size += (spread ** 2).sum()
    assert np.sqrt(err / size) <= 2.0 ** -22


def test_small_and_odd_arguments():
    """No rows, tables without columns, integers of 64 bits, views that are not contiguous."""
    from heteroserve.kv import quant
    from heteroserve.model.paged_attn_q4 import paged_attention_q4
    from heteroserve.model.paged_attn_window import paged_attention_window

    pool = quant.empty_pool_q4(1, 4, BS, HKV, 64, device=DEV)
    cache = torch.randn(2, 4, BS, HKV, 64, device=DEV)
    kc, vc = pool[0, 0], pool[0, 1]
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    bt = torch.tensor([[2, 1], [3, 0]], device=DEV)
    quant.append_kv_q4(kc, vc, bt, none, cache[0, 0, :0], cache[1, 0, :0], seq_ids=none)
    assert not pool.any()
    k, v = quant.read_kv_q4(kc, vc, bt, none, seq_ids=none)
    assert k.shape == v.shape == (0, HKV, 64) and k.dtype is F16
    at = torch.arange(20, device=DEV)
    quant.append_kv_q4(kc, vc, bt, at, cache[0].view(-1, HKV, 64)[:20], cache[1].view(-1, HKV, 64)[:20],
                       seq_ids=torch.zeros(20, dtype=torch.int64, device=DEV))
    ctx = torch.tensor([20, 0], device=DEV)
    q = torch.randn(2, H, 64, device=DEV)
    wide = torch.randn(2, H, 128, device=DEV)
    wide[..., ::2] = q
    for call, args in ((paged_attention_q4, (kc, vc)), (paged_attention_window, (cache[0], cache[1]))):
        want = call(q, *args, bt, ctx, 0.1, 7, 2)
        assert torch.isfinite(want).all() and want[0].any() and not want[1].any()
        assert torch.equal(call(wide[..., ::2], *args, bt, ctx, 0.1, 7, 2), want)
        turned = q.transpose(0, 1).contiguous().transpose(0, 1)
        assert torch.equal(call(turned, *args, bt.t().contiguous().t(), ctx, 0.1, 7, 2), want)
        both = call(q[:1].expand(2, H, 64), *args, bt[:1].expand(2, 2), ctx[:1].expand(2), 0.1, 7, 2)
        assert torch.equal(both[0], both[1])
        assert call(q[:0], *args, bt[:0], ctx[:0], 0.1, 7, 2).shape == (0, H, 64)
        with pytest.raises(RuntimeError, match="positive"):
            call(q, *args, bt[:, :0], ctx, 0.1, 7, 2)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,D", [(16, 32), (8, 64), (12, 128), (6, 256), (3, 128), (5, 64)])
def test_rows_of_whole_waves_and_others(dtype, heads, D):
    """Rows of 64 and 192 words, whose place is a wave's, and of 48 and 40, to the byte; some
    of them name no slot."""
    from heteroserve.kv import quant

    gen = torch.Generator(DEV).manual_seed(D)
    n, NB, page = 75, 7, 13
    k, v = (torch.randn(n, heads, D, generator=gen, device=DEV).to(dtype) for _ in range(2))
    bt = torch.tensor([[3, 0, 6], [5, 2, -1]], dtype=torch.int32)
    seq, at = np.arange(n) % 2, np.arange(n) // 2
    seq[10], at[20] = 7, 3 * page
    pool = quant.empty_pool_q4(1, NB, page, heads, D, device=DEV).fill_(0x5a)
    want = pool.cpu().numpy()
    quant.append_kv_q4(pool[0, 0], pool[0, 1], bt, torch.tensor(at), k, v, seq_ids=torch.tensor(seq))
    named = np.array([s < 2 and p < 3 * page and bt[s, p // page] >= 0 for s, p in zip(seq, at)])
    assert 2 < (~named).sum() < n // 2
    for i, x in enumerate((k, v)):
        rec = lc.records(*lc.quantise(_np(x)), keys=i == 0)
        want[0, i][bt.numpy()[seq[named], at[named] // page], at[named] % page] = rec[named]
    assert np.array_equal(pool.cpu().numpy(), want)
    got = quant.read_kv_q4(pool[0, 0], pool[0, 1], bt, torch.tensor(at), seq_ids=torch.tensor(seq), dtype=dtype)
    for i, x in enumerate(got):
        held = np.zeros((n, heads, D))
        held[named] = lc.values(want[0, i][bt.numpy()[seq[named], at[named] // page], at[named] % page], i == 0)
        assert torch.equal(x.cpu(), torch.tensor(held).to(F32).to(dtype))


@pytest.mark.parametrize("B", [1, 2, 3, 8, 9, 16, 24, 30])
def test_batches_of_every_count(B):
    """Rows and parts are dealt to the chip in an order that depends on their number."""
    for q4, D in ((True, 128), (False, 64)):
        lens = [int(x) for x in np.linspace(2600, 1, B)]
        s = _Chat(lens, 0, D, BF16, q4, seed=B)
        q = s.rows(B)[0]
        s.check(0, q, s.attend(0, q))
        s.check(0, q, s.attend(0, q, 2100, 1), 2100, 1)


@pytest.mark.parametrize("B", [63, 64, 65, 128, 129, 200, 256, 257])
@pytest.mark.parametrize("q4", [True, False])
def test_large_ragged_batches(q4, B):
    """Whole parts, parts that are not, and empty rows in every order, on both sides of the
    counts where parts are dealt otherwise; pages are shared, so that they stay few."""
    from heteroserve.kv import quant
    from heteroserve.model.paged_attn_q4 import paged_attention_q4
    from heteroserve.model.paged_attn_window import paged_attention_window

    rng = np.random.default_rng(B)
    D, pages, MB = 64, 300, 280
    gen = torch.Generator(DEV).manual_seed(B)
    k, v = (torch.randn(pages * BS, HKV, D, generator=gen, device=DEV) for _ in range(2))
    lens = rng.choice([0, 1, 255, 256, 257, 512, 513, 1024, 2048, 3333, MB * BS], B)
    lens[B // 2] = MB * BS                   # a row of the table's width
    bt = rng.integers(0, pages, (B, MB)).astype(np.int32)
    q = torch.randn(B, H, D, generator=gen, device=DEV)
    args = (_dev(bt), _dev(lens), D ** -0.5)
    if q4:
        pool = quant.empty_pool_q4(1, pages, BS, HKV, D, device=DEV)
        at = torch.arange(pages * BS)
        quant.append_kv_q4(pool[0, 0], pool[0, 1], torch.arange(pages)[None], at, k, v,
                           seq_ids=torch.zeros_like(at))
        got = paged_attention_q4(q, pool[0, 0], pool[0, 1], *args)
        k, v = (lc.values(pool[0, i].cpu().numpy().reshape(-1, HKV, 5 * D // 8), i == 0) for i in (0, 1))
    else:
        got = paged_attention_window(q, k.half().view(pages, BS, HKV, D), v.half().view(pages, BS, HKV, D),
                                     *args, 0)
        k, v = _np(k.half()), _np(v.half())
    for b in range(B):
        pos = np.arange(lens[b])
        rows = bt[b, pos // BS] * BS + pos % BS
        _check(q[b], got[b], k[rows], v[rows], D)


@pytest.mark.parametrize("q4", [True, False])
def test_a_captured_batch_with_other_lengths(q4):
    """More parts than the chip holds at a time, whose length follows the rows': a graph of one
    call, replayed over other lengths and tables with eager calls between, is the eager
    call to the bit."""
    from heteroserve.model.paged_attn_q4 import paged_attention_q4
    from heteroserve.model.paged_attn_window import paged_attention_window

    rng = np.random.default_rng(5)
    B, heads, kv, D, pages, MB = 48, 16, 8, 128, 400, 300
    gen = torch.Generator(DEV).manual_seed(5)
    if q4:
        cache = torch.randint(0, 120, (2, pages, BS, kv, 80), generator=gen, device=DEV, dtype=torch.uint8)
        call = paged_attention_q4                # (bytes below 0x78: finite steps and lowest values)
    else:
        cache = torch.randn(2, pages, BS, kv, D, generator=gen, device=DEV).half()
        call = paged_attention_window
    tables = _dev(rng.integers(0, pages, (B, MB)))
    ctx = _dev(np.full(B, MB * BS))
    q = torch.randn(B, heads, D, generator=gen, device=DEV) * 1e-4

    def run():
        return call(q, cache[0], cache[1], tables, ctx, 0.1, 0, 0)

    lengths = [rng.integers(0, MB * BS + 1, B), np.full(B, 3), np.where(np.arange(B) == 7, MB * BS, 0),
               np.full(B, MB * BS), rng.integers(500, 600, B)]
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for lens in lengths:
        ctx.copy_(_dev(lens))
        tables.copy_(_dev(rng.integers(0, pages, (B, MB))))
        want = run().clone()
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.isfinite(want).all()
        assert not want[torch.tensor(lens == 0, device=DEV)].any()


@pytest.mark.parametrize("q4,dtype,D", [(True, F16, 128), (True, F16, 256), (False, BF16, 64), (False, F16, 128),
                                        (False, F32, 64), (False, BF16, 256)])
@pytest.mark.parametrize("odd", [float("nan"), float("inf"), -float("inf")])
def test_a_query_that_is_no_number(q4, dtype, D, odd):
    """It takes its own head's row, and no other."""
    s = _Chat([70, 300], 0, D, dtype, q4, seed=D)
    q = s.rows(2)[0].float().contiguous()
    want = s.attend(0, q, 100, 2)
    q[1, 3, 17] = odd
    got = s.attend(0, q, 100, 2)
    assert torch.isfinite(want).all() and not torch.isfinite(got[1, 3]).any()
    got[1, 3] = want[1, 3]
    assert torch.equal(got, want)


@pytest.mark.parametrize("q4", [True, False])
@pytest.mark.parametrize("long", [0, 1, 20])
def test_tables_wider_than_most_rows(q4, long):
    """A table of 32768 tokens, of which `long` rows hold all and the others few or none; the
    workgroups are counted for the longest."""
    from heteroserve.kv import quant
    from heteroserve.model.paged_attn_q4 import paged_attention_q4
    from heteroserve.model.paged_attn_window import paged_attention_window

    rng = np.random.default_rng(long)
    B, D, pages, MB = 40, 32, 200, 2048
    gen = torch.Generator(DEV).manual_seed(long)
    k, v = (torch.randn(pages * BS, HKV, D, generator=gen, device=DEV).half() for _ in range(2))
    lens = rng.integers(0, 700, B)
    lens[rng.permutation(B)[:long]] = MB * BS
    lens[:3] = 0
    bt = rng.integers(0, pages, (B, MB)).astype(np.int32)
    q = torch.randn(B, H, D, generator=gen, device=DEV)
    args = (_dev(bt), _dev(lens), D ** -0.5)
    if q4:
        pool = quant.empty_pool_q4(1, pages, BS, HKV, D, device=DEV)
        at = torch.arange(pages * BS)
        quant.append_kv_q4(pool[0, 0], pool[0, 1], torch.arange(pages)[None], at, k, v,
                           seq_ids=torch.zeros_like(at))
        got = paged_attention_q4(q, pool[0, 0], pool[0, 1], *args)
        k, v = (lc.values(pool[0, i].cpu().numpy().reshape(-1, HKV, 5 * D // 8), i == 0) for i in (0, 1))
    else:
        got = paged_attention_window(q, k.view(pages, BS, HKV, D), v.view(pages, BS, HKV, D), *args, 0)
        k, v = _np(k), _np(v)
    seen = 0
    for b in range(B):
        pos = np.arange(lens[b])
        rows = bt[b, pos // BS] * BS + pos % BS
        if lens[b] < MB * BS or seen < 4:
            _check(q[b], got[b], k[rows], v[rows], D)
        seen += lens[b] == MB * BS
    assert torch.isfinite(got).all()

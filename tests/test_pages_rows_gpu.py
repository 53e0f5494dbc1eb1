"""Rows and blocks that are none, given to the page operations on the device: what they
name stays as it was."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import operators as ops  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _dev(a):
    return torch.tensor(np.asarray(a, np.int32), device=DEV)


class _State:
    """Six rows that hold blocks, two that hold none, and blocks that nobody holds."""

    def __init__(self, L=2, NB=40, BS=16, MB=4):
        rng = np.random.default_rng(NB)
        lens = [20, 64, 1, 33, 16, 50]
        self.tables = np.full((8, MB), -1, np.int32)
        self.refs = np.zeros(NB, np.int32)
        self.ctx = np.zeros(8, np.int32)
        ids = rng.permutation(NB)
        for b, n in enumerate(lens):
            k = -(-n // BS)
            self.tables[b, :k], ids = ids[:k], ids[k:]
            self.refs[self.tables[b, :k]] = 1 + b % 2
            self.ctx[b] = n
        gen = torch.Generator(device=DEV).manual_seed(NB)
        self.pool = torch.randn(L, 2, NB, BS, 2, 64, generator=gen, device=DEV).to(torch.bfloat16)

    def on_device(self):
        return self.pool, _dev(self.tables), _dev(self.ctx), _dev(self.refs)

    def host(self):
        return [self.pool.view(torch.int16).cpu().numpy().copy(), self.tables.copy(), self.ctx.copy(),
                self.refs.copy()]

    @staticmethod
    def same(got, want):
        got = [got[0].view(torch.int16).cpu(), *(x.cpu() for x in got[1:])]
        return all(np.array_equal(x.numpy(), w) for x, w in zip(got, want))


@pytest.mark.parametrize("parent", [-1, 8, -2 ** 31, 2 ** 31 - 1])
def test_fork_of_a_row_that_is_none_leaves_the_child(parent):
    """A step of fixed size whose parents alone are padded: the children's rows hold
    sequences, and keep them."""
    from heteroserve.kv import pages

    s = _State()
    state, want = s.on_device(), s.host()
    parents, children = [parent, 0, parent, parent, 4], [1, 6, 5, 2, 4]
    fresh = ops.find_free(s.refs, 5)
    done = ops.fork(*want, parents, children, fresh)
    assert done.tolist() == [0, 1, 0, 0, 0]
    assert want[2].tolist() == [20, 64, 1, 33, 16, 50, 20, 0]
    got = pages.fork_blocks(*state, _dev(parents), _dev(children), _dev(fresh))
    assert got.tolist() == done.tolist()
    assert s.same(state, want)


@pytest.mark.parametrize("bad", [torch.tensor([True, False, True, True, False, False, True, True]),
                                 torch.tensor([1.0, 2.9]), torch.tensor([3.0], dtype=torch.float16)])
def test_rows_on_the_device_must_be_integers_too(bad):
    """As from the host: a mask or a number with a fraction is no list of rows."""
    from heteroserve.kv import pages

    s = _State()
    state, want = s.on_device(), s.host()
    for rows in (bad, bad.to(DEV)):
        with pytest.raises(RuntimeError, match="row must be integers"):
            pages.free_blocks(*state[1:], rows)
        for given in ([rows, [6] * len(rows), [0] * len(rows)], [[0], rows, [1]], [[0], [6], rows]):
            with pytest.raises(RuntimeError, match="must be integers"):
                pages.fork_blocks(*state, *given)
    assert s.same(state, want)


@pytest.mark.parametrize("dtype", [torch.int64, torch.uint32, torch.uint64])
def test_rows_on_the_device_past_32_bits_are_none(dtype):
    """They are skipped, and are not the rows and blocks of their lower 32 bits."""
    from heteroserve.kv import pages

    s = _State()
    state, want = s.on_device(), s.host()
    far = [2 ** 32 - 1] if dtype is torch.uint32 else [2 ** 32, 2 ** 32 + 1, 2 ** 33 + 2, 2 ** 63 - 1]
    if dtype is torch.int64:
        far += [-2 ** 32 + 3, -2 ** 63 + 4]
    if dtype is torch.uint64:
        far += [2 ** 64 - 1, 2 ** 63 + 5]
    wide = torch.tensor(far, dtype=dtype, device=DEV)
    n = len(far)
    pages.free_blocks(*state[1:], wide)
    assert s.same(state, want)
    child, fresh = _dev([6] + [-1] * (n - 1)), _dev(ops.find_free(s.refs, n))
    assert not pages.fork_blocks(*state, wide, child, fresh).any()
    assert not pages.fork_blocks(*state, _dev([0] * n), wide, fresh).any()
    assert s.same(state, want)
    want[1][6], want[2][6] = -1, 0
    assert not pages.fork_blocks(*state, _dev([0] + [-1] * (n - 1)), child, wide).any()
    assert s.same(state, want)


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64,
                                   torch.uint16, torch.uint32, torch.uint64])
def test_rows_of_every_integer_type(dtype):
    from heteroserve.kv import pages

    s = _State()
    state, want = s.on_device(), s.host()
    fresh = ops.find_free(s.refs, 2)
    done = ops.fork(*want, [0, 3], [6, 7], fresh)
    rows = [torch.tensor(x, device=DEV).to(dtype) for x in ([0, 3], [6, 7], fresh)]
    assert pages.fork_blocks(*state, *rows).tolist() == done.tolist() == [1, 1]
    ops.free(*want[1:], [7, 0])
    pages.free_blocks(*state[1:], torch.tensor([7, 0], device=DEV).to(dtype))
    assert s.same(state, want)

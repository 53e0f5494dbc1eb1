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

"""CPU checks of the row and block indexes that the page operations take from the host."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")


def _indexes(values, **kw):
    from heteroserve.kv import pages

    return pages._indexes(values, 8, "row", torch.device("cpu"), **kw)[0].tolist()


def test_wrapped_and_kept():
    assert _indexes([0, -1, 7, -8]) == [0, 7, 7, 0]
    assert _indexes(np.array([3, 7], np.uint64)) == [3, 7]
    assert _indexes(torch.tensor([1, -2])) == [1, 6]
    assert _indexes([2, -1], none=True) == [2, -1]
    assert _indexes([]) == []


@pytest.mark.parametrize("value", [2 ** 64 - 1, 2 ** 64 - 8, 2 ** 63, 8])
@pytest.mark.parametrize("none", [False, True])
def test_unsigned_values_past_64_bits_signed_are_no_negative_ones(value, none):
    for values in (np.array([0, value], np.uint64), torch.tensor([0, value], dtype=torch.uint64)):
        with pytest.raises(IndexError, match=f"row index {value} is out of bounds"):
            _indexes(values, none=none)


@pytest.mark.parametrize("values", [[0.0], [True], np.array([1.5]), torch.tensor([True]), [2 ** 70]])
def test_what_is_no_integer(values):
    with pytest.raises(RuntimeError, match="row must be integers"):
        _indexes(values)


def test_block_ids_past_64_bits_signed_are_no_negative_ones():
    """Of copies, and of the pack calls, which take them the same way."""
    from heteroserve.kv import pack, pages

    for read in (pages._host_ids, pack._normalise_ids):
        assert read(torch.tensor([1, 6], dtype=torch.uint64), 8).tolist() == [1, 6]
        for values in (np.array([2 ** 64 - 1], np.uint64), torch.tensor([0, 2 ** 64 - 1], dtype=torch.uint64)):
            with pytest.raises(IndexError, match=f"index {2 ** 64 - 1} is out of bounds"):
                read(values, 8)

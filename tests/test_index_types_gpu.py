"""Positions, sequence numbers, tables and offsets of other types than int32: whole
numbers count as they are, those past 32 bits name nothing, and no others are taken."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def _rows(n, H, Hkv, D, dtype, seed=3):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(n, h, D, generator=gen, device=DEV).to(dtype) for h in (H, Hkv, Hkv)]


def _freq(pairs):
    return torch.tensor((100.0 ** (-np.arange(pairs) / pairs)).astype(np.float32), device=DEV)


def _append(pos, at, seq, tables, axes=None):
    from heteroserve.kv import rotary

    q, k, v = _rows(6, 2, 1, 64, F32)
    kc, vc = torch.zeros(2, 5, 4, 1, 64, device=DEV)
    q, _ = rotary.rotate_append_kv(q, k, v, pos, _freq(32), kc, vc, tables, at, seq, axes=axes)
    return q, kc, vc


POS, AT, SEQ = [[5, 6, 7, 8, 9, 10], [0, 1, 2, 0, 1, 2]], [0, 1, 2, 3, 4, 5], [0, 0, 1, 1, 0, 1]
TABLES = [[2, 0], [1, 4]]


def _int(values, dtype=torch.int32, device=DEV):
    return torch.tensor(values, device=device).to(dtype)


@pytest.mark.parametrize("dtype", [torch.int64, torch.int16, torch.uint8, torch.uint32])
@pytest.mark.parametrize("device", [DEV, "cpu"])
def test_other_integer_types(dtype, device):
    axes = [i % 2 for i in range(32)]
    want = _append(*(_int(x) for x in (POS, AT, SEQ, TABLES, axes)))
    got = _append(*(_int(x, dtype, device) for x in (POS, AT, SEQ, TABLES, axes)))
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    got = _append(POS, AT, SEQ, TABLES, axes)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("far", [2 ** 32, 2 ** 32 + 1, 2 ** 63 - 1, -2 ** 32, -2 ** 32 + 1])
@pytest.mark.parametrize("device", [DEV, "cpu"])
def test_numbers_past_32_bits_name_nothing(far, device):
    """They are not the slots, sequences, blocks and axes of their lower 32 bits."""
    rows = [_int(x) for x in (POS, AT, SEQ, TABLES)]

    def wide(values, i):
        x = torch.tensor(values, device=device)
        x.view(-1)[i] = far
        return x

    skip = _int(AT)
    skip[1] = -1
    want = _append(rows[0], skip, *rows[2:])
    for given in ([rows[0], wide(AT, 1), *rows[2:]], [*rows[:2], wide(SEQ, 1), rows[3]]):
        got = _append(*given)
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    holed = _int([[2, -1], [1, 4]])
    want = _append(*rows[:3], holed)
    assert all(torch.equal(x, y) for x, y in zip(_append(*rows[:3], wide(TABLES, 1)), want))
    axes = [1] * 32
    first = _int([0] + axes[1:])
    want = _append(*rows, first)
    assert all(torch.equal(x, y) for x, y in zip(_append(*rows, wide(axes, 0)), want))


@pytest.mark.parametrize("device", [DEV, "cpu"])
def test_offsets_of_prompts_past_32_bits_are_past_the_rows(device):
    from heteroserve.model.prompt_attn import prompt_attention

    q, k, v = _rows(50, 2, 1, 64, BF16)
    want = prompt_attention(q, k, v, _int([0, 20, 50]), 30, 0.125)
    for cu in ([0, 20, 2 ** 32], [-2 ** 32 + 7, 20, 2 ** 33 + 30], [-2 ** 63, 20, 2 ** 63 - 1]):
        got = prompt_attention(q, k, v, torch.tensor(cu, device=device), 30, 0.125)
        assert torch.equal(got, want)
    assert torch.equal(prompt_attention(q, k, v, torch.tensor([0, 20, 50], device=device), 30, 0.125), want)


@pytest.mark.parametrize("device", [DEV, "cpu"])
def test_no_whole_numbers_are_refused(device):
    """A position of 1.5 is not 1, nor a mask a list."""
    from heteroserve.kv import rotary
    from heteroserve.model.prompt_attn import prompt_attention

    good = [_int(x) for x in (POS, AT, SEQ, TABLES, [0, 1] * 16)]
    names = ["positions", "cache_positions", "seq_ids", "block_tables", "axes"]
    for i, name in enumerate(names):
        for dtype in (torch.float32, torch.bool, torch.float64):
            given = list(good)
            given[i] = given[i].to(device=device, dtype=dtype)
            with pytest.raises(RuntimeError, match=f"{name} must be integers"):
                _append(*given)
    q, k, v = _rows(6, 2, 1, 64, F32)
    with pytest.raises(RuntimeError, match="positions must be integers"):
        rotary.rotate_qk(q, k, torch.arange(6, device=device) + 0.5, _freq(32))
    with pytest.raises(RuntimeError, match="positions must be"):
        rotary.rotate_qk(q, k, [1, 2, 3], _freq(32))
    with pytest.raises(RuntimeError, match="cu_seqlens must be integers"):
        prompt_attention(q, k, v, torch.tensor([0.0, 6.0], device=device), 6, 0.1)
    # none at all have no type of their own
    q, k, v = (x[:0] for x in (q, k, v))
    assert rotary.rotate_qk(q, k, [], _freq(32))[0].shape == (0, 2, 64)

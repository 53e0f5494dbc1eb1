"""Every form of the whole-prompt kernels at sizes that reach it on a device of any number
of CUs: workgroups of 128 rows for every type and head dim, their tiles taken by number
and searched for in both orders; and offsets that are none, with guards around every
tensor.  Tolerances, in a row's 2-norm, are those of test_prompt_gpu.py's long prompts:
64 u for fp32 sums and half a step each for 16-bit probabilities and outputs.  Those are
for a scale of D^-1/2.  A score's error is that of its products and their sum times the
scale, and a probability's relative error is its score's: with a scale s above D^-1/2 both
are s D^1/2 times as large, and so is the fp32 part of the tolerance."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES, DIMS = [F32, F16, BF16], [32, 64, 128, 256]


def _cus():
    return torch.cuda.get_device_properties(0).multi_processor_count


def _rows(lens, H, Hkv, D, dtype, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    n = sum(lens)
    rows = torch.randn(n, (H + 2 * Hkv) * D, generator=gen, device=DEV).to(dtype)
    q, k, v = rows.split([H * D, Hkv * D, Hkv * D], 1)
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    return q.view(n, H, D), k.view(n, Hkv, D), v.view(n, Hkv, D), cu


def _dense(q, k, v, cu, scale, heads=None):
    """float64 on the GPU, the given heads (all): [T, heads, D]."""
    heads = range(q.shape[1]) if heads is None else heads
    g = q.shape[1] // k.shape[1]
    out = torch.full((q.shape[0], len(heads), q.shape[2]), np.nan, dtype=torch.float64, device=DEV)
    for a, b in zip(cu[:-1], cu[1:]):
        a, b = int(a), int(b)
        later = torch.ones(b - a, b - a, dtype=torch.bool, device=DEV).triu(1)
        for i, h in enumerate(heads):
            s = torch.mm(q[a:b, h].double(), k[a:b, h // g].double().t().contiguous()) * scale
            out[a:b, i] = torch.mm(torch.softmax(s.masked_fill(later, -np.inf), -1), v[a:b, h // g].double())
    return out


def _close(got, want, dtype, scale=0.0):
    tol = 64 * 2.0 ** -24 * max(1.0, abs(scale) * got.shape[-1] ** 0.5)
    tol += 0 if dtype is F32 else torch.finfo(dtype).eps
    rel = ((got.double() - want).norm(dim=-1) / want.norm(dim=-1)).max().item()
    assert rel <= tol, (rel, tol)


def _call(q, k, v, cu, longest, scale, out=None):
    from heteroserve.model.prompt_attn import prompt_attention

    return prompt_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device=DEV), longest, scale, out=out)


def _filled():
    """Prompts of one length, 3 tiles of 128 rows each, 8 heads: three workgroups and more
    a CU, which split no keys, and no rows past an end that smaller workgroups would save."""
    return [300] * (_cus() // 8 + 1), 8, 2


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("scale", [None, 0.0, -0.2])
def test_a_filled_device(dtype, D, scale):
    lens, H, Hkv = _filled()
    q, k, v, cu = _rows(lens, H, Hkv, D, dtype, D)
    scale = D ** -0.5 if scale is None else scale
    _close(_call(q, k, v, cu, 300, scale), _dense(q, k, v, cu, scale), dtype, scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_lies_behind_a_row_of_a_filled_device(dtype, D, where, bad):
    """Rows in front of it, of other sequences and of other heads are as without it."""
    lens, H, Hkv = _filled()
    q, k, v, cu = _rows(lens, H, Hkv, D, dtype, D + 1)
    clean = _call(q, k, v, cu, 300, D ** -0.5)
    dirty = {"k": k, "v": v}[where]
    at = 600 + 137                      # inside a tile of rows and of keys
    dirty[at, 1, 5] = bad
    got = _call(q, k, v, cu, 300, D ** -0.5)
    same = torch.ones(got.shape[:2], dtype=torch.bool, device=DEV)
    same[600:900, 4:] = False
    assert torch.equal(got[same], clean[same])
    assert torch.isfinite(got[:at]).all()
    # rows that share a tile with it are computed again, by another order of sums
    _close(got[600:at, 4:], _dense(q[600:at], k[600:at], v[600:at], [0, at - 600], D ** -0.5, range(4, 8)),
           dtype)
    want = _dense(q[600:900], k[600:900], v[600:900], [0, 300], D ** -0.5, range(4, 8))[137:]
    behind = got[at:900, 4:].double()
    assert torch.equal(torch.isnan(want), torch.isnan(behind))
    assert torch.equal(want == np.inf, behind == np.inf) and torch.equal(want == -np.inf, behind == -np.inf)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("order", ["levels", "sequences", "many"])
def test_tiles_that_are_searched_for(dtype, D, order):
    """Lengths of 0 to 900: longest walks first where the keys and values fit the L2s
    (32 MB), a sequence's tiles together where they do not, sequences as they come where
    there are more than lanes."""
    # tiles of 128 rows: 8 + 1 + 4 + 2 + 1 + 0 + 1 + 3 of 8 sequences, 1785 rows
    lens = [900, 1, 400, 130, 64, 0, 33, 257]
    if order == "many":
        lens, H, Hkv = lens * 9, 8, 2
        assert 180 * H > 3 * _cus()
    else:
        H, Hkv = (16, 2) if order == "levels" else (16, 16)
        lens = lens * 3
        size = 4 if dtype is F32 else 2
        if order == "sequences":
            while sum(lens) * Hkv * D * 2 * size <= 32 << 20:
                H = Hkv = 2 * Hkv
        else:
            assert sum(lens) * Hkv * D * 2 * size <= 32 << 20
        assert len(lens) <= 64 and 60 * H > 3 * _cus()
    q, k, v, cu = _rows(lens, H, Hkv, D, dtype, D + len(lens))
    _close(_call(q, k, v, cu, 900, D ** -0.5), _dense(q, k, v, cu, D ** -0.5), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,T,H,Hkv,longest", [
    (64, 40, 2, 1, 64), (128, 40, 64, 8, 32), (64, 300, 2, 1, 300), (256, 300, 2, 2, 300),
    (64, 700, 32, 8, 700), (64, 900, 64, 8, 900), (128, 900, 64, 64, 900)])
def test_offsets_that_are_none_and_guards(dtype, D, T, H, Hkv, longest):
    """Rows of offsets before 0 and behind the last row count as those; a sequence whose
    end is before its start has none.  NaN around the inputs and a mark around and in the
    output show what is read and written."""
    guard = 33
    bufs = []
    for i, h in enumerate((H, Hkv, Hkv)):
        gen = torch.Generator(device=DEV).manual_seed(T + i)
        b = torch.full((T + 2 * guard, h, D), float("nan"), dtype=dtype, device=DEV)
        b[guard:-guard] = torch.randn(T, h, D, generator=gen, device=DEV).to(dtype)
        bufs.append(b)
    q, k, v = (b[guard:-guard] for b in bufs)
    big = 2 ** 31 - 1
    for cu in ([-5, T // 2, big], [T * 3 // 4, T // 4, T], [T + 10, T + 20, T + 30], [-big - 1, -1, 0],
               [big, -big - 1, T // 3], [0, T // 5, T // 5, T + 7]):
        out = torch.full((T + 2 * guard, H, D), 7.0, dtype=dtype, device=DEV)
        got = _call(q, k, v, cu, longest, D ** -0.5, out=out[guard:-guard])
        assert (out[:guard] == 7.0).all() and (out[-guard:] == 7.0).all()
        left = torch.ones(T, dtype=torch.bool, device=DEV)
        for a, b in zip(cu[:-1], cu[1:]):
            a = min(max(a, 0), T)
            b = min(max(a, min(b, T)), a + longest)
            if a < b:
                assert left[a:b].all()          # no two sequences share a row here
                left[a:b] = False
                _close(got[a:b], _dense(q[a:b], k[a:b], v[a:b], [0, b - a], D ** -0.5), dtype)
        assert (got[left] == 7.0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_sequences_cut_short(dtype):
    """Rows from max_seqlen on, and rows of no sequence, stay; the others are exact."""
    q, k, v, _ = _rows([123], 2, 1, 64, dtype, 3)
    out = torch.full((123, 2, 64), 7.0, dtype=dtype, device=DEV)
    got = _call(q, k, v, [5, 20, 53], 17, 0.125, out=out)
    assert (got[:5] == 7.0).all() and (got[37:] == 7.0).all()
    want = _dense(q, k, v, [5, 20, 37], 0.125)
    _close(got[5:37], want[5:37], dtype)

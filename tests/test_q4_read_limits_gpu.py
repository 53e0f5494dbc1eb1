"""What is read back of groups at fp16's limits: a step is rounded, so lo + 15 s may lie beyond fp16's
largest number although the row did not; values beyond it count as that, as they do when they
are written."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import long_context as lc  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
MOST = 65504.0


def _written(x):
    """A cache of one page with rows x [n, 1, D] as keys and -x as values."""
    from heteroserve.kv import quant

    n, _, D = x.shape
    pool = quant.empty_pool_q4(1, 2, n, 1, D, device=DEV)
    args = (pool[0, 0], pool[0, 1], torch.tensor([[1]]), torch.arange(n))
    quant.append_kv_q4(*args, x, -x, seq_ids=torch.zeros(n, dtype=torch.int32))
    return args


def _rows():
    rng = np.random.default_rng(0)
    ends = [(0, MOST), (-MOST, MOST), (-MOST, 0), (60000, MOST), (-MOST, -60000), (MOST, MOST), (0, 1e30),
            (-np.inf, np.inf), (0, np.inf), (-1e38, 1.0), (65000, 65520), (0, 61000), (-30000, 65500)]
    x = np.stack([rng.uniform(max(a, -2 * MOST), min(b, 2 * MOST), 32) for a, b in ends])
    x[:, 3], x[:, 17] = np.array(ends).T
    return torch.tensor(x.reshape(-1, 1, 32), device=DEV).to(F32)


@pytest.mark.parametrize("out", [F32, F16, BF16])
def test_what_is_written_at_the_limits_is_read_back(out):
    from heteroserve.kv import quant

    x = _rows()
    args = _written(x)
    got = quant.read_kv_q4(*args, seq_ids=torch.zeros(len(x), dtype=torch.int32), dtype=out)
    beyond = 0
    for i, rows in enumerate((x, -x)):
        n, s, lo = lc.quantise(rows.double().cpu().numpy())
        held = torch.tensor((n * s[..., None] + lo[..., None]).reshape(x.shape)).to(F32)
        beyond += int((held.abs() >= 65520).sum())           # what rounds to an infinity
        want = held.clamp(-MOST, MOST) if out is F16 else held
        assert torch.equal(got[i].cpu(), want.to(out))
        assert torch.isfinite(got[i]).all()
    assert beyond > 5
    x[2, 0, 5] = float("nan")
    args = _written(x)
    for rows in quant.read_kv_q4(*args, seq_ids=torch.zeros(len(x), dtype=torch.int32), dtype=out):
        assert torch.isnan(rows[2]).all() and int(torch.isnan(rows).sum()) == 32


def test_a_prefix_at_the_limits_is_prefilled():
    """Read as fp16 and attended to: rows are finite."""
    from heteroserve.kv import quant
    from heteroserve.model.paged_attn_window import paged_attention_window

    x = torch.zeros(13, 1, 32, device=DEV)
    x[:, 0, 7], x[:, 0, 20] = MOST, -MOST
    k, v = quant.read_kv_q4(*_written(x), seq_ids=torch.zeros(13, dtype=torch.int32))
    assert k.dtype is F16
    got = paged_attention_window(torch.ones(1, 1, 32, device=DEV), k[None], v[None], torch.tensor([[0]]),
                                 torch.tensor([13]), 1e-6, window=0)
    assert torch.isfinite(got).all()

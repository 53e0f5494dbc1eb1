"""All terms of the query and of the probabilities reach the matrix cores: numbers whose bits lie in
three bf16 terms of 8, with sums that cancel what the first two hold, so that the third decides.

Scores are sums that fp32 holds exactly.  Then a probability is off by exp2's 2^-22, and sums, a
reciprocal and a product by 2^-24 each: 2^-21 of the row, where values are 1, 0 and -1.  Each test
says what a missing third term would leave, which is more."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from oracle import long_context as lc  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
X = 1 + 2.0 ** -9 + 2.0 ** -18          # 1 | 2^-9 | 2^-18
LIMIT = 2.0 ** -21
LOG2E = np.float32(1.4426950408889634)
# a scale that is 1 in log2 units: fp32's product with log2(e) is
SCALE = next(float(s) for s in np.float32(np.log(2)) + np.arange(-4, 5) * np.float32(2.0 ** -25)
             if np.float32(np.float32(s) * LOG2E) == 1)


def _bf16_terms(x, n):
    """The sum of the first n bf16 terms of x."""
    left, out = torch.as_tensor(x, dtype=torch.float64), 0
    for _ in range(n):
        term = left.float().bfloat16().double()
        left, out = left - term, out + term
    return np.asarray(out)


def _attend(q, k, v, dtype):
    """(got, want) [H, D] of one sequence in one page; the oracle has scores in log2 units."""
    from heteroserve.model.paged_attn_window import paged_attention_window

    n = k.shape[0]
    cache = torch.zeros(2, 1, 32, *k.shape[1:], dtype=dtype, device=DEV)
    cache[0, 0, :n], cache[1, 0, :n] = (torch.tensor(x, device=DEV).to(dtype) for x in (k, v))
    got = paged_attention_window(torch.tensor(q[None], dtype=torch.float32, device=DEV), cache[0], cache[1],
                                 torch.tensor([[0]]), torch.tensor([n]), SCALE, window=0)
    return got[0].double().cpu().numpy(), lc.decode(q, k, v, np.log(2))[0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_the_query(dtype, D):
    """Two keys; one's score is the sum of 2^-9 and 2^-18 that X is more than 1, 2 + 2^-8 in all: a
    third term that is missing moves the row by 2^-8 ln 2 p (1 - p) 2, some 2^-10."""
    q, k, v = np.ones((2, D)), np.zeros((2, 1, D)), np.ones((2, 1, D))
    q[:, ::2] = X
    k[0, 0, ::2], k[0, 0, 1::2] = 2048 / D, -2048 / D
    v[1] = -1
    got, want = _attend(q, k, v, dtype)
    assert np.abs(lc.decode(_bf16_terms(q, 2), k, v, np.log(2))[0] - want).min() > 100 * LIMIT
    assert np.abs(got - want).max() <= LIMIT


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
def test_the_probabilities(dtype, D):
    """Of 9 keys 8 have the probability X / 2 of the other, whose value is 0.  Their third terms
    are 2^-18 of the row.  (Their score is what fp32 has next to log2(X / 2).)"""
    down = float(np.float32(-np.log2(X / 2)))
    q, k, v = np.zeros((3, D)), np.zeros((9, 1, D)), np.ones((9, 1, D))
    q[:, 5] = down
    k[1:, 0, 5] = -1
    v[0] = 0
    got, want = _attend(q, k, v, dtype)
    p = 2.0 ** -down
    lost = 8 * (p - _bf16_terms(p, 2)) / (1 + 8 * p)
    assert abs(lost) > 4 * LIMIT and np.abs(got - want).max() <= LIMIT

"""That the comparison of paged_strict.py sees mistakes, planted in what it is given.  No GPU needed."""
import math

import pytest
import torch

import paged_reference as ref
import paged_strict as strict
from paged_reference import Batch


def answers(batch, **kw):
    return strict.attention(batch.q, batch.k_cache, batch.v_cache, batch.table, batch.lens, batch.cu, **kw)


@pytest.mark.parametrize("dtype,d", [(torch.float16, 64), (torch.bfloat16, 40)])
def test_the_same_as_the_other_reference_where_all_is_finite(dtype, d):
    batch = Batch([3, 0, 90, 1], [100, 20, 80, 0], 4, 2, d, 16, dtype, seed=1, first=2, behind=1)
    for mask in (dict(causal=True), dict(window=(20, 3)), dict(causal=True, window=(0, -1))):
        mine, other = answers(batch, **mask), ref.attention(batch.q, batch.k_cache, batch.v_cache, batch.table, batch.lens, batch.cu, d ** -0.5,
                                                            mask.get("causal", False), mask.get("window", (-1, -1)))
        rows = mine[4]
        assert torch.equal(rows, ~torch.isposinf(other[1][:, 0]))
        assert torch.allclose(mine[0][rows], other[0][rows], rtol=1e-12, atol=1e-14) and torch.allclose(mine[1][rows], other[1][rows], rtol=1e-12, atol=1e-12)
        assert (mine[2][rows] <= other[2][rows] * (1 + 1e-9)).all() and (mine[3][rows] <= other[3][rows] * (1 + 1e-9)).all()


def test_mistakes_are_seen():
    batch = Batch([3], [100], 2, 1, 64, 16, torch.float16, seed=3)
    batch.q[:, :, 0] = 1.0
    batch.k_cache[:, :, 3, 0] = -math.inf
    at, row = int(batch.table[0, 40 // 16]), 40 % 16
    batch.v_cache[at, :, row, 2], batch.v_cache[at, :, row, 5] = math.inf, -math.inf
    want = answers(batch, causal=True)
    O, L = want[0].clone(), want[1].clone()
    assert torch.isposinf(O[..., 2]).all() and torch.isneginf(O[..., 5]).all() and torch.isfinite(L).all()
    strict.check(O, L, want)
    for where, value in (((0, 0, 7), 123.0), ((0, 0, 7), math.nan), ((1, 1, 2), math.nan), ((1, 1, 2), -math.inf), ((1, 1, 5), 0.0), ((2, 0, 0), math.inf)):
        bad = O.clone()
        bad[where] = value
        with pytest.raises(AssertionError):
            strict.check(bad, L, want)
    for value in (-55.0, math.nan, -math.inf):
        bad = L.clone()
        bad[1, 0] = value
        with pytest.raises(AssertionError):
            strict.check(O, bad, want)

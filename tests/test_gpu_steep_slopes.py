"""A bias by distance with steep slopes: what a score's rounding grows by."""
import pytest
import torch

import scored_reference as ref
from paged_reference import Batch
from test_gpu_paged_scores import call, want

pytestmark = pytest.mark.gpu

SHAPES = [("few", [3, 40], [900, 130], 8, 2, 1), ("mid", [600, 333], [1500, 700], 12, 4, 3), ("paired", [400], [1600], 24, 8, 3), ("tall", [520], [2000], 32, 8, 3)]
MASKS = [{"causal": True}, {"window": (-1, 20)}]
DIMS = [40, 64, 128]


@pytest.mark.parametrize("softcap", [0.0, 5.0])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: s[0])
@pytest.mark.parametrize("mask", MASKS, ids=lambda m: next(iter(m)))
@pytest.mark.parametrize("d", DIMS)
def test_rounding_grows_with_the_slope(fa, shape, softcap, d, mask):
    """The bounds of scored_reference.py, whose part of the bias is that of a key's own distance, and what the places of the tiles add to it: scores are summed up from
    slope * (key - first of its tile of up to 64) on, in d products and sums and three parts of the slope; the tile's distance, at most 64 more than the key's, and
    the reference it is taken from are rounded three times.  Below x = (d + 11) 2^-24 * 64 |slope| for any key: LSE moves by x, O by 2 x max |v|."""
    _, news, lens, H, Hk, splits = shape
    batch = Batch(news, lens, H, Hk, d, 16, torch.bfloat16 if d == 64 else torch.float16, seed=d)
    slopes = torch.tensor([2.0 ** (-4 + h % 10) for h in range(H)])  # 1 / 16 ... 32
    slopes[-1] = fa.FLASH_MAX_SLOPE
    how = dict(mask, softcap=softcap)
    O, L, bO, bL, mine = want(batch, how, {"slopes": slopes})
    x = 1.05 * (d + 11) * 2.0 ** -24 * 64 * slopes.double()
    bL, bO = bL + x, bO + 2 * x[:, None] * float(batch.v_cache.abs().max())
    ref.check(*call(fa, batch, how, {"slopes": slopes}, num_splits=splits), (O, L, bO, bL, mine))

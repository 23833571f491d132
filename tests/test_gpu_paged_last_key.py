"""Values that are not finite in V at a sequence's last key, which is not masked for the rows that see it: they get them, whatever part of a tile the
sequence ends in."""
import math

import pytest
import torch

import paged_strict as strict
from paged_reference import Batch

pytestmark = pytest.mark.gpu

# (tokens, keys, heads, K/V heads): ends on and off the tiles of 32 and 64 keys, in one tile, two, three and more
FEW = [([1] * 7, [5, 32, 64, 96, 130, 191, 700], 8, 2), ([7, 20, 3], [200, 77, 128], 4, 4), ([40, 1], [40, 33], 2, 1)]
TALL = [([300, 70, 1], [333, 200, 64], 96, 96), ([300, 80, 90], [700, 80, 128], 80, 40), ([70, 70, 70, 70], [70, 127, 129, 192], 96, 96)]


def spoil(batch):
    """+inf, -inf and NaN in columns of V of each sequence's last key, and an infinity of the other sign at key 0 of one of them"""
    for row, n in zip(batch.table, batch.lens.tolist()):
        at, j = int(row[(n - 1) // batch.page]), (n - 1) % batch.page
        batch.v_cache[at, :, j, 3], batch.v_cache[at, :, j, 5], batch.v_cache[at, :, j, 1], batch.v_cache[at, :, j, 6] = math.inf, -math.inf, math.nan, math.inf
        if n > 1:
            batch.v_cache[int(row[0]), :, 0, 6] = -math.inf


@pytest.mark.parametrize("shape", FEW + TALL, ids=lambda s: f"{len(s[0])}x{max(s[0])}-{s[2]}")
@pytest.mark.parametrize("dtype,d", [(torch.float16, 64), (torch.bfloat16, 128), (torch.float16, 80), (torch.bfloat16, 40), (torch.float16, 8)])
def test_last_key(fa, dtype, d, shape):
    news, lens, H, Hk = shape
    batch = Batch(news, lens, H, Hk, d, 16, dtype, seed=d)
    spoil(batch)
    for kw in (dict(causal=True), dict(), dict(causal=True, window=(45, -1)), dict(window=(100, 3))):
        want = strict.attention(batch.q, batch.k_cache, batch.v_cache, batch.table, batch.lens, batch.cu, **kw)
        for splits in (1, 3):
            got = fa.flash_forward_paged(*batch.cuda(), max_seqlen_q=max(news), num_splits=splits, **kw)
            strict.check(*got, want, f"{kw} {splits}")

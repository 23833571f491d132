"""Scores of -inf among others, and infinite values that rows see, by class and sign, in both forms of flash_forward_paged."""
import math

import pytest
import torch

import paged_strict as strict
from paged_reference import Batch

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
FEW = [([3], [100], 2, 1), ([1, 1, 9], [300, 65, 40], 8, 2)]
TALL = [([300, 70, 1], [333, 200, 64], 96, 96)]


def put(cache, batch, b, j, column, value):
    cache[int(batch.table[b, j // batch.page]), :, j % batch.page, column] = value


@pytest.mark.parametrize("shape", FEW + TALL, ids=lambda s: f"{len(s[0])}x{max(s[0])}-{s[2]}")
@pytest.mark.parametrize("dtype,d", [(F16, 64), (BF16, 128), (BF16, 40)])
def test_keys_that_count_for_nothing(fa, dtype, d, shape):
    """Keys whose score is -inf weigh nothing, whatever their V holds (as long as it is finite)."""
    news, lens, H, Hk = shape
    batch = Batch(news, lens, H, Hk, d, 16, dtype, seed=3)
    batch.q[:, :, 0] = 1.0
    for b, n in enumerate(lens):
        for j in range(2, n, 7):
            put(batch.k_cache, batch, b, j, 0, -math.inf)
            put(batch.v_cache, batch, b, j, 1, 1000.0)
    for mask in (dict(causal=True), dict(window=(60, 2))):
        want = strict.attention(batch.q, batch.k_cache, batch.v_cache, batch.table, batch.lens, batch.cu, **mask)
        assert torch.isfinite(want[0]).all()
        for splits in (1, 2):
            got = fa.flash_forward_paged(*batch.cuda(), max_seqlen_q=max(news), num_splits=splits, **mask)
            strict.check(*got, want, f"{mask} {splits}")


@pytest.mark.parametrize("shape", FEW + TALL, ids=lambda s: f"{len(s[0])}x{max(s[0])}-{s[2]}")
@pytest.mark.parametrize("dtype,d", [(F16, 64), (BF16, 128), (BF16, 40)])
def test_infinite_values_that_rows_see(fa, dtype, d, shape):
    """Either sign, both, and one beside a value that is not a number, in keys all over the sequence: what a row sees it gets."""
    news, lens, H, Hk = shape
    batch = Batch(news, lens, H, Hk, d, 16, dtype, seed=4)
    for b, n in enumerate(lens):
        for j, column, value in ((0, 0, math.inf), (n // 2, 1, -math.inf), (n // 3, 2, math.inf), (n - 1, 2, -math.inf), (n - 2, 3, math.nan), (n // 2, 3, math.inf)):
            put(batch.v_cache, batch, b, j, column, value)
    for mask in (dict(causal=True), dict(), dict(causal=True, window=(30, -1))):
        want = strict.attention(batch.q, batch.k_cache, batch.v_cache, batch.table, batch.lens, batch.cu, **mask)
        for splits in (1, 2):
            got = fa.flash_forward_paged(*batch.cuda(), max_seqlen_q=max(news), num_splits=splits, **mask)
            strict.check(*got, want, f"{mask} {splits}")

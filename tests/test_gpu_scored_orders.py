"""Other scores over a paged cache in launches whose 256-row work-groups are ordered by the end of their keys over all sequences.  test_scored_orders.py holds every
case here to that."""
import pytest
import torch

import scored_reference as ref
from paged_reference import Batch
from test_gpu_paged_scores import call, tree, want
from test_gpu_scored_forms import CAUSAL, SCORES, both, extras, left

pytestmark = pytest.mark.gpu

# (new tokens, keys) per sequence, H, H_kv, d
CHUNKS = [([233, 65, 124, 222, 29, 231, 23], [233, 72, 124, 312, 65, 389, 157], 48, 24, 64),
          ([154, 85, 104, 64, 102, 15, 16, 75, 70, 149, 49, 138, 125], [335, 85, 106, 103, 102, 106, 168, 81, 114, 149, 49, 329, 224], 32, 16, 128)]
AHEAD = [([216, 103, 34, 4, 141, 216, 206, 127, 17, 36, 22], [339, 427, 158, 4, 141, 216, 206, 127, 132, 36, 566], 32, 16, 64),
         ([154, 30, 19, 78, 9, 100, 111, 96, 59, 73, 38, 143, 9, 6, 15], [154, 30, 19, 78, 611, 100, 286, 150, 715, 73, 38, 359, 9, 6, 635], 32, 16, 128)]
BEHIND = [([204, 91, 2, 75, 34, 186, 82], [227, 438, 596, 75, 150, 186, 497], 128, 8, 128)]
TREES = [([82, 38, 81, 53, 63, 18, 23, 36, 55, 52, 18, 73], [82, 114, 81, 53, 63, 18, 23, 36, 55, 653, 18, 73], 80, 16, 64),
         ([84, 1, 5, 24, 49, 59, 61, 4, 42, 72, 61, 83, 31, 44], [84, 1, 5, 302, 49, 59, 61, 4, 42, 186, 113, 83, 31, 640], 64, 16, 128)]
CASES = [(shape, mask, kind) for shapes, mask in ((CHUNKS, CAUSAL), (AHEAD, both(-1, 20)), (BEHIND, left(150))) for shape in shapes for kind in SCORES]
TREE_CASES = [(shape, kind) for shape in TREES for kind in ("", "cap", "slopes", "both")]


@pytest.mark.parametrize("shape,mask,kind", CASES, ids=lambda v: v if isinstance(v, str) else None)
def test_scores(fa, shape, mask, kind):
    news, lens, H, Hk, d = shape
    batch = Batch(news, lens, H, Hk, d, 16, torch.bfloat16, seed=d)
    how, kw = extras(kind, H, lens, mask)
    ref.check(*call(fa, batch, how, kw, num_splits=1), want(batch, how, kw), kind)


@pytest.mark.parametrize("shape,kind", TREE_CASES, ids=lambda v: v if isinstance(v, str) else None)
def test_trees(fa, shape, kind):
    news, lens, H, Hk, d = shape
    batch = Batch(news, lens, H, Hk, d, 16, torch.bfloat16, seed=d)
    how, kw = tree(news, kind, H, d)
    ref.check(*call(fa, batch, how, kw, num_splits=1), want(batch, how, kw), kind)

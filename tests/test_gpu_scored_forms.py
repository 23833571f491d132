"""Other scores over a paged cache, each kind and mask in each form of the kernels: 32 rows, 128 rows, 128 rows in two groups of waves, 256 rows, whole and in
splits.  test_scored_forms.py holds every case here to the form that it is listed under."""
import math

import pytest
import torch

import paged_launches
import scored_reference as ref
from paged_reference import Batch
from test_gpu_paged_scores import call, tree, want

pytestmark = pytest.mark.gpu

CAUSAL, ALL = {"causal": True}, {}


def left(n):
    return {"causal": True, "window": (n, -1)}


def both(n, right):
    return {"window": (n, right)}


SCORES = ["cap", "slopes", "both", "prefix", "cap prefix", "slopes prefix", "both prefix"]
BARE = SCORES[:3]  # (a prefix takes the left end off the estimate of a window, and gets another form)
RAGGED = ([300, 70, 1], [420, 200, 64], 96, 48)
# form, (new tokens, keys) per sequence, H, H_kv, splits, mask, scores, head dimensions in turn
FORMS = [
    ("few", [1, 0, 3, 5], [900, 17, 3, 130], 4, 4, 1, CAUSAL, SCORES, (8, 64, 128)),
    ("few", [1, 0, 3, 5], [900, 17, 3, 130], 4, 4, 3, left(40), SCORES, (64, 80, 128)),
    ("few", [40, 3], [700, 100], 6, 2, 1, both(-1, 20), SCORES, (128, 40, 64)),
    ("few", [40, 3], [700, 100], 6, 2, 3, both(300, 7), SCORES, (64, 128, 96)),
    ("few", [40, 3], [700, 100], 6, 2, 1, ALL, SCORES, (80, 64, 128)),
    ("mid", *RAGGED, 1, CAUSAL, SCORES, (64, 128, 40)),
    ("mid", *RAGGED, 1, left(40), BARE, (64, 128, 80)),
    ("mid", [600, 333], [1500, 700], 12, 4, 3, left(600), SCORES, (64, 128, 80)),
    ("mid", [600, 333], [1500, 700], 12, 4, 3, both(-1, 20), SCORES, (128, 64, 40)),
    ("mid", [600, 333], [1500, 700], 12, 4, 3, both(700, 30), SCORES, (64, 80, 128)),
    ("paired", [400], [1600], 24, 8, 3, CAUSAL, SCORES, (64, 128, 80)),
    ("paired", [400], [1600], 24, 8, 3, left(1023), SCORES, (128, 64, 40)),
    ("paired", [800], [1100], 32, 8, 1, left(600), SCORES, (64, 128, 80)),
    ("paired", [400], [1600], 24, 8, 3, both(-1, 20), SCORES, (40, 128, 64)),
    ("paired", [800], [1100], 32, 8, 1, both(700, 30), SCORES, (128, 64, 80)),
    ("tall", *RAGGED, 1, both(-1, 20), SCORES, (64, 128, 80)),
    ("tall", *RAGGED, 1, both(150, 30), SCORES[3:], (128, 64, 40)),
    ("tall", [300, 250, 77], [340, 310, 140], 64, 16, 1, both(300, 30), BARE, (64, 128, 40)),
    ("tall", [300, 250, 77], [340, 310, 140], 64, 16, 1, left(300), BARE, (64, 64, 64)),
    ("tall", [1500], [1500], 32, 8, 1, left(300), BARE, (128, 80, 128)),
    ("tall", [520], [2000], 32, 8, 3, both(-1, 20), SCORES[3:], (80, 64, 128)),
    ("tall", [520], [2000], 32, 8, 3, left(1023), SCORES[3:], (64, 128, 80)),
]
CASES = [(form, news, lens, H, Hk, splits, mask, kind, dims[i % 3]) for form, news, lens, H, Hk, splits, mask, kinds, dims in FORMS for i, kind in enumerate(kinds)]
TREES = [
    ("few", [100, 256], [777, 256], 1, 1, 1, 300, (64, 128)),
    ("mid", [200, 256, 9], [263, 256, 700], 66, 33, 1, 300, (64, 128)),
    ("paired", [128, 128, 128], [900, 1500, 2000], 24, 24, 2, 700, (128, 64)),
    ("paired", [256, 200], [256, 1500], 64, 1, 1, 300, (64, 80)),
    ("tall", [256, 256, 256, 256], [600, 500, 700, 800], 64, 8, 1, -1, (64, 128)),
    ("tall", [256, 256, 256, 256], [600, 500, 700, 800], 64, 8, 1, 300, (128, 40)),
]
TREE_CASES = [(form, news, lens, H, Hk, splits, window, kind, dims[i % 2]) for form, news, lens, H, Hk, splits, window, dims in TREES
              for i, kind in enumerate(("cap", "slopes", "both", ""))]


def names(v):
    return "-".join(str(x) for x in (v if isinstance(v, (list, tuple)) else v.values())) if isinstance(v, (list, tuple, dict)) else None


def extras(kind, H, lens, mask):
    how, kw = dict(mask), {}
    if kind.startswith(("cap", "both")):
        how["softcap"] = 5.0
    if kind.startswith(("slopes", "both")):
        kw["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) * (-1 if h == 1 else 1) for h in range(H)])  # (one that prefers the distance)
    if kind.endswith("prefix"):
        kw["prefix"] = torch.tensor([[n - 3, 0, n // 2, n + 50][b % 4] for b, n in enumerate(lens)], dtype=torch.int32)
    return how, kw


def arguments(news, lens, H, Hk, d, splits, mask, kind=None, words=0):
    """The call as paged_launches.call has it."""
    how, kw = extras(kind or "", H, lens, mask)
    places = {"slopes": ("alibi_slopes", 0xc00000), "prefix": ("prefix_lens", 0xd00000)}
    more = dict(places[k] for k in kw)
    if words:
        more.update(tree_mask=0xe00000, tree_words=words, tree_stride=words)
    return paged_launches.call(news, lens, H, Hk, d, max_seqlen_q=max(news), num_splits=splits, dtype="bf16" if d % 16 else "fp16", **how, **more)


@pytest.mark.parametrize("form,news,lens,H,Hk,splits,mask,kind,d", CASES, ids=names)
def test_scores(fa, form, news, lens, H, Hk, splits, mask, kind, d):
    batch = Batch(news, lens, H, Hk, d, 16, torch.bfloat16 if d % 16 else torch.float16, seed=d + splits)
    how, kw = extras(kind, H, lens, mask)
    ref.check(*call(fa, batch, how, kw, num_splits=splits), want(batch, how, kw), f"{form} {kind}")


@pytest.mark.parametrize("form,news,lens,H,Hk,splits,window,kind,d", TREE_CASES, ids=names)
def test_trees(fa, form, news, lens, H, Hk, splits, window, kind, d):
    batch = Batch(news, lens, H, Hk, d, 16, torch.bfloat16 if d % 16 else torch.float16, seed=d + splits)
    how, kw = tree(news, kind, H, d)
    if window >= 0:
        how["window"] = (window, -1)
    ref.check(*call(fa, batch, how, kw, num_splits=splits), want(batch, how, kw), f"{form} {kind}")


# the last key's V is not finite: sequences that end on and off a tile, of one tile and of many
LAST = [("few", [1, 7, 3], [300, 64, 7], 4, 4, 1), ("mid", *RAGGED, 1), ("mid", [600, 333], [1500, 700], 12, 4, 3), ("paired", [400], [1590], 24, 8, 3),
        ("tall", [520], [2001], 32, 8, 3)]
LAST_CASES = [(*shape, kind, d) for shape in LAST for kind, d in (("cap", 64), ("slopes", 128), ("both", 80))]


@pytest.mark.parametrize("form,news,lens,H,Hk,splits,kind,d", LAST_CASES, ids=names)
def test_infinite_v_of_the_last_key(fa, form, news, lens, H, Hk, splits, kind, d):
    """It reaches the last token, which alone sees it, and no other row, call after call."""
    batch = Batch(news, lens, H, Hk, d, 16, torch.float16, seed=d)
    how, kw = extras(kind, H, lens, CAUSAL)
    if "slopes" in kw:
        kw["slopes"] = kw["slopes"].abs()
    fine = want(batch, how, kw)
    for row, n in zip(batch.table, lens):
        batch.v_cache[int(row[(n - 1) // 16]), :, (n - 1) % 16, 3] = math.inf
    last = [int(t) - 1 for t, m in zip(batch.cu[1:], news) if m]
    first = call(fa, batch, how, kw, num_splits=splits)
    for _ in range(4):
        o, lse = call(fa, batch, how, kw, num_splits=splits)
        assert torch.equal(o, first[0]) and torch.equal(lse, first[1])
    o = first[0].cpu()
    assert torch.isposinf(o[last, :, 3]).all()
    o[last, :, 3] = fine[0][last, :, 3].to(o.dtype)
    ref.check(o, first[1], fine, f"{form} {kind}")

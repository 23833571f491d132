"""flash_forward_paged with capped scores, a bias by distance, a prefix and trees of drafted tokens, against 64 bits."""
import math

import pytest
import torch

import scored_reference as ref
from paged_reference import Batch

pytestmark = pytest.mark.gpu

# (new tokens, keys) per sequence, H, H_kv: what the forms of 32, 128 and 256 rows get (the last in so many splits)
FEW = [([1, 1, 1, 1], [1, 70, 333, 1000], 8, 2), ([1, 0, 3, 5], [900, 17, 3, 130], 4, 4), ([7, 2], [300, 65], 15, 3)]
MID = [([300, 70, 1], [420, 200, 64], 96, 48), ([290, 0, 150], [280, 9, 700], 80, 40)]
PAIRED = [([256], [2500], 32, 8, 3)]  # 128 rows in two groups of waves
TALL = [([520], [2000], 32, 8, 3), ([1500], [1500], 32, 8, 1)]
DIMS = [8, 40, 64, 80, 128]
KINDS = ["cap", "slopes", "both", "prefix", "prefix window", "cap prefix", "slopes window", "slopes all"]


def extras(kind, H, lens):
    """Arguments of the call and of the reference."""
    how, kw = {"causal": True}, {}
    if "cap" in kind or kind == "both":
        how["softcap"] = 5.0  # (scores of unit normal rows reach 4)
    if "slopes" in kind or kind == "both":
        kw["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) * (-1 if h == 1 else 1) for h in range(H)])  # (one that prefers the distance)
    if "prefix" in kind:
        kw["prefix"] = torch.tensor([[0, n // 2, n, n + 50, -3][b % 5] for b, n in enumerate(lens)], dtype=torch.int32)
    if "window" in kind:
        how["window"] = (40, -1)
    if "all" in kind:
        how["causal"] = False
        how["window"] = (-1, 20)
    return how, kw


def call(fa, batch, how, kw, **more):
    names = {"slopes": "alibi_slopes", "prefix": "prefix_lens", "mask": "tree_mask"}
    return fa.flash_forward_paged(*batch.cuda(), max_seqlen_q=max(batch.news), **how, **{names[k]: v.cuda() for k, v in kw.items()}, **more)


def want(batch, how, kw):
    return ref.attention(batch.q, batch.k_cache, batch.v_cache, batch.table, batch.lens, batch.cu, **how, **kw)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", range(3))
@pytest.mark.parametrize("d,dtype,splits", [(8, torch.bfloat16, 1), (40, torch.float16, 3), (64, torch.bfloat16, 0), (80, torch.float16, 1), (128, torch.bfloat16, 3), (128, torch.float16, 0)])
def test_few_rows(fa, kind, shape, d, dtype, splits):
    news, lens, H, Hk = FEW[shape]
    batch = Batch(news, lens, H, Hk, d, 16 if d < 100 else 48, dtype, seed=d + shape, first=2, behind=1)
    how, kw = extras(kind, H, lens)
    ref.check(*call(fa, batch, how, kw, num_splits=splits), want(batch, how, kw), kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape", range(2))
@pytest.mark.parametrize("d,dtype,splits", [(40, torch.bfloat16, 1), (64, torch.float16, 3), (80, torch.bfloat16, 2), (128, torch.float16, 1), (128, torch.bfloat16, 3)])
def test_rows_between(fa, kind, shape, d, dtype, splits):
    news, lens, H, Hk = MID[shape]
    batch = Batch(news, lens, H, Hk, d, 64, dtype, seed=d + shape, behind=3)
    how, kw = extras(kind, H, lens)
    ref.check(*call(fa, batch, how, kw, num_splits=splits), want(batch, how, kw), kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d,dtype", [(40, torch.bfloat16), (64, torch.float16), (80, torch.float16), (128, torch.bfloat16)])
def test_two_groups_of_waves(fa, kind, d, dtype):
    news, lens, H, Hk, splits = PAIRED[0]
    batch = Batch(news, lens, H, Hk, d, 16, dtype, seed=d, first=1)
    how, kw = extras(kind, H, lens)
    if "window" in kind or "all" in kind:  # (pieces of tiles enough)
        how["window"] = (600, -1) if "window" in kind else (-1, 700)
        splits = 1 if "window" in kind else splits
    ref.check(*call(fa, batch, how, kw, num_splits=splits), want(batch, how, kw), kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("shape,d,dtype", [(0, 40, torch.bfloat16), (0, 64, torch.float16), (0, 80, torch.bfloat16), (0, 128, torch.float16), (1, 80, torch.float16), (1, 128, torch.bfloat16)])
def test_many_rows(fa, kind, shape, d, dtype):
    news, lens, H, Hk, splits = TALL[shape]
    if shape == 1 and kind not in ("cap", "slopes", "prefix"):
        pytest.skip("the smaller one has it")
    batch = Batch(news, lens, H, Hk, d, 64, dtype, seed=d + shape, behind=3)
    how, kw = extras(kind, H, lens)
    ref.check(*call(fa, batch, how, kw, num_splits=splits), want(batch, how, kw), kind)


# ---------------------------------------------------------------------------------------------------- trees

TREES_FEW = [([5, 1, 13, 2], [5, 300, 130, 66], 4, 4), ([25], [1025], 8, 2), ([64, 7], [64, 400], 1, 1), ([100, 256], [777, 256], 1, 1)]
TREES_MID = [([64, 30, 1], [200, 31, 640], 320, 40), ([200, 256, 9], [263, 256, 700], 66, 33)]
TREES_PAIRED = [([128, 128, 128], [900, 1500, 2000], 24, 24, 3)]
TREES_TALL = [([256, 200], [256, 1500], 64, 1, 3), ([128, 256], [3000, 1000], 64, 8, 1)]
TREE_KINDS = ["", "cap", "slopes", "both", "window", "slopes window"]


def tree(news, kind, H, seed, words=None):
    parents = ref.random_parents(news, seed)
    cu = [sum(news[:b]) for b in range(len(news) + 1)]
    mask, _ = ref.tree_mask(parents, cu, [0] * len(news), words or -(-max(news) // 64))
    how, kw = extras(kind.replace("window", ""), H, [])
    how["causal"] = seed % 2 == 1  # (not looked at)
    kw["mask"] = mask
    if "window" in kind:
        how["window"] = (max(max(news) - 1, 100), -1)
    return how, kw


@pytest.mark.parametrize("kind", TREE_KINDS)
@pytest.mark.parametrize("shape", range(4))
@pytest.mark.parametrize("d,dtype,splits", [(24, torch.bfloat16, 1), (64, torch.float16, 3), (96, torch.float16, 1), (128, torch.bfloat16, 0)])
def test_trees_few_rows(fa, kind, shape, d, dtype, splits):
    news, lens, H, Hk = TREES_FEW[shape]
    batch = Batch(news, lens, H, Hk, d, 16, dtype, seed=d + shape)
    how, kw = tree(news, kind, H, d + shape)
    ref.check(*call(fa, batch, how, kw, num_splits=splits), want(batch, how, kw), kind)


@pytest.mark.parametrize("kind", TREE_KINDS)
@pytest.mark.parametrize("shape", range(2))
@pytest.mark.parametrize("d,dtype,splits", [(64, torch.bfloat16, 1), (80, torch.float16, 3), (128, torch.float16, 1), (128, torch.bfloat16, 2)])
def test_trees_rows_between(fa, kind, shape, d, dtype, splits):
    news, lens, H, Hk = TREES_MID[shape]
    batch = Batch(news, lens, H, Hk, d, 32, dtype, seed=d + shape)
    how, kw = tree(news, kind, H, d + shape)
    ref.check(*call(fa, batch, how, kw, num_splits=splits), want(batch, how, kw), kind)


@pytest.mark.parametrize("kind", TREE_KINDS)
@pytest.mark.parametrize("d,dtype", [(40, torch.float16), (64, torch.bfloat16), (80, torch.bfloat16), (128, torch.float16)])
def test_trees_two_groups_of_waves(fa, kind, d, dtype):
    news, lens, H, Hk, splits = TREES_PAIRED[0]
    batch = Batch(news, lens, H, Hk, d, 48, dtype, seed=d)
    how, kw = tree(news, kind, H, d)
    ref.check(*call(fa, batch, how, kw, num_splits=splits), want(batch, how, kw), kind)


@pytest.mark.parametrize("kind", TREE_KINDS)
@pytest.mark.parametrize("shape,d,dtype", [(0, 40, torch.float16), (0, 64, torch.bfloat16), (0, 80, torch.float16), (0, 128, torch.bfloat16), (1, 80, torch.bfloat16), (1, 128, torch.float16)])
def test_trees_many_rows(fa, kind, shape, d, dtype):
    news, lens, H, Hk, splits = TREES_TALL[shape]
    if shape == 1 and kind not in ("", "both"):
        pytest.skip("the smaller one has it")
    batch = Batch(news, lens, H, Hk, d, 32, dtype, seed=d + shape)
    how, kw = tree(news, kind, H, d + shape)
    ref.check(*call(fa, batch, how, kw, num_splits=splits), want(batch, how, kw), kind)


@pytest.mark.parametrize("H,Hk", [(2, 1), (192, 48)])
def test_masks_of_any_shape(fa, H, Hk):
    """Rows without a bit, with bits past the chunk, with more words than the chunk needs, not of a tree; a chunk without keys in front of it."""
    news, lens = [70, 3, 1], [70, 40, 1]
    batch = Batch(news, lens, H, Hk, 64, 16, torch.float16, seed=9)
    g = torch.Generator().manual_seed(4)
    mask = torch.randint(-2 ** 62, 2 ** 62, (74, 4), generator=g)
    mask[5] = mask[71] = mask[73] = 0
    mask[6] = -1
    wide = torch.full((74, 7), -1, dtype=torch.int64)
    wide[:, 1:5] = mask
    for m in (mask, wide[:, 1:5]):
        for how in ({}, {"softcap": 4.0}):
            o, lse = fa.flash_forward_paged(*batch.cuda(), max_seqlen_q=70, tree_mask=m.cuda() if m is mask else wide.cuda()[:, 1:5], **how)
            ref.check(o, lse, want(batch, how, {"mask": mask}))
            assert torch.isneginf(lse[5]).all() and torch.isneginf(lse[73]).all() and torch.isfinite(lse[71]).all()


def all_but(bit):
    """64 bits but one, as a signed number"""
    return 2 ** 63 - 1 if bit == 63 else ~(1 << bit)


@pytest.mark.parametrize("news,lens,H,Hk", [([5, 1], [40, 77], 2, 1), ([120, 40], [300, 44], 192, 48), ([128, 128, 128], [900, 1500, 2000], 24, 24), ([256, 200], [256, 1500], 64, 1)])
def test_what_is_not_seen_does_not_matter(fa, news, lens, H, Hk):
    """Infinities and NaN in pages behind the sequences, in keys that the mask hides from all, and in V of keys that some rows see."""
    for dtype in (torch.float16, torch.bfloat16):
        batch = Batch(news, lens, H, Hk, 64, 16, dtype, seed=1, stale=math.nan)
        how, kw = tree(news, "slopes", H, 2)
        hidden = lens[0] - news[0] + news[0] // 2  # a drafted token that nobody sees, of V a row that is not a number
        kw["mask"][:news[0], (news[0] // 2) // 64] &= all_but((news[0] // 2) % 64)
        at, row = int(batch.table[0, hidden // 16]), hidden % 16
        batch.v_cache[at, :, row] = math.inf
        batch.k_cache[at, :, row] = math.nan
        for softcap in (0.0, 5.0):
            how["softcap"] = softcap
            for splits in (1, 3):
                o, lse = call(fa, batch, how, kw, num_splits=splits)
                ref.check(o, lse, want(batch, how, kw))
        # one that its own row alone sees
        last = lens[0] - 1
        kw["mask"][:news[0] - 1, (news[0] - 1) // 64] &= all_but((news[0] - 1) % 64)
        at, row = int(batch.table[0, last // 16]), last % 16
        fine = want(batch, how, kw)
        batch.v_cache[at, :, row, 3] = math.inf
        o, lse = call(fa, batch, how, kw)
        # (the head whose slope prefers the distance gives it a weight of e^-100 and less, down to 0 in 32 bits: no number, or nothing of it where it is
        # alone with such keys in a split, which the merge does not read)
        assert torch.isposinf(o[news[0] - 1, kw["slopes"].cuda() > 0, 3]).all()
        o[news[0] - 1, :, 3] = fine[0][news[0] - 1, :, 3].to(o.dtype)
        ref.check(o, lse, fine)


def test_infinite_scores_are_capped(fa):
    """A product of infinity counts as the cap, of minus infinity as its negative."""
    batch = Batch([2], [40], 1, 1, 64, 16, torch.bfloat16, seed=3)
    batch.q[:, :, 0] = 1.0
    batch.k_cache[..., 0] = 0.0
    for j, x in ((3, math.inf), (30, -math.inf)):
        batch.k_cache[int(batch.table[0, j // 16]), 0, j % 16, 0] = x
    o, lse = call(fa, batch, {"softcap": 6.0}, {})
    for j, x in ((3, 1e30), (30, -1e30)):  # (far beyond the cap, and finite)
        batch.k_cache[int(batch.table[0, j // 16]), 0, j % 16, 0] = x
    o2, lse2 = call(fa, batch, {"softcap": 6.0}, {})
    assert torch.isfinite(o).all() and torch.equal(o, o2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("cap", [1e-3, 0.5, 30.0, 1000.0])
def test_small_and_large_caps(fa, cap):
    for news, lens, H, Hk in (FEW[0], MID[1], TALL[0][:4]):
        batch = Batch(news, lens, H, Hk, 64, 16, torch.bfloat16, seed=5)
        batch.q *= 4
        how = {"causal": True, "softcap": cap}
        ref.check(*call(fa, batch, how, {}), want(batch, how, {}))


def test_a_cap_alone_changes_what_it_should(fa):
    """Without a cap, slopes of 0, an empty prefix, and a mask that is the causal one: the same as the call without them, within the bounds of both."""
    news, lens, H, Hk = [40, 1], [100, 64], 4, 2
    batch = Batch(news, lens, H, Hk, 64, 16, torch.float16, seed=6)
    plain = fa.flash_forward_paged(*batch.cuda(), causal=True, max_seqlen_q=40)
    ordered = torch.cat([torch.tensor([[(1 << (i + 1)) - 1] for i in range(n)]) for n in news])
    bound = want(batch, {"causal": True}, {})
    for kw in ({"slopes": torch.zeros(H)}, {"prefix": torch.zeros(2, dtype=torch.int32)}, {"mask": ordered}):
        o, lse = call(fa, batch, {"causal": True}, kw)
        ref.check(o, lse, bound)
        assert ((o - plain[0]).abs().cpu().double() <= 2 * bound[2]).all() and ((lse - plain[1]).abs().cpu().double() <= 2 * bound[3]).all()


def test_rows_of_no_sequence_stay(fa):
    for shape in (FEW[2], MID[0], PAIRED[0][:4], TALL[0][:4]):
        news, lens, H, Hk = shape
        batch = Batch(news, lens, H, Hk, 64, 16, torch.bfloat16, seed=7, first=3, behind=4)
        T = batch.q.shape[0]
        for splits in (1, 3):
            out, lse = torch.full((T, H, 64), 7.0, dtype=torch.bfloat16, device="cuda"), torch.full((T, H), 7.0, device="cuda")
            how, kw = extras("both", H, lens)
            call(fa, batch, how, kw, out=out, lse=lse, num_splits=splits)
            ref.check(out, lse, want(batch, how, kw))
            for t in (out, lse):
                assert (t[:3] == 7).all() and (t[-4:] == 7).all()


@pytest.mark.parametrize("shape", [FEW[2], MID[0], PAIRED[0][:4], TALL[0][:4]])
def test_strides_streams_and_both_ways_in(fa, shape):
    """Heads before or behind rows in a page, strided queries and results, a stream of the caller's, workspace of the caller's: always the same result."""
    news, lens, H, Hk = shape
    batch = Batch(news, lens, H, Hk, 64, 16, torch.float16, seed=8)
    how, kw = extras("both", H, lens)
    first = call(fa, batch, how, kw, num_splits=3)
    q, kc, vc, table, ln, cu = batch.cuda()
    T = q.shape[0]
    wide = torch.randn((T, H, 128), device="cuda").half()
    wide[..., :64] = q
    rows_first = kc.transpose(1, 2).contiguous().transpose(1, 2)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    workspace = (torch.empty(T * H * 3 * 64, device="cuda"), torch.empty(T * H * 3, device="cuda"))
    out = torch.empty((T, H, 96), dtype=torch.float16, device="cuda")[..., :64]
    o, lse = fa.flash_forward_paged(wide[..., :64], rows_first, vc, table, ln, cu, max_seqlen_q=max(news), num_splits=3, workspace=workspace, out=out, stream=stream,
                                    alibi_slopes=kw["slopes"].cuda(), **how)
    stream.synchronize()
    assert torch.equal(o, first[0]) and torch.equal(lse, first[1])


def test_captured_and_replayed(fa):
    """A graph of trees and of capped scores follows lengths, masks and prefixes."""
    news, H, Hk, d = [9, 1, 30], 8, 2, 64
    batches = [Batch(news, lens, H, Hk, d, 16, torch.bfloat16, seed=s, spare=60 - sum(-(-n // 16) for n in lens)) for s, lens in enumerate(([9, 200, 100], [300, 1, 31], [10, 17, 480]))]
    width = 40
    parents = [ref.random_parents(news, s) for s in range(3)]
    masks = [ref.tree_mask(p, [0, 9, 10, 40], [0] * 3, 1)[0] for p in parents]
    prefixes = [torch.tensor([s, 100 * s, 5], dtype=torch.int32) for s in range(3)]
    tables = []
    for b in batches:
        t = torch.zeros((3, width), dtype=torch.int32)
        t[:, :b.table.shape[1]] = b.table
        tables.append(t)
    q, kc, vc, _, lens, cu = batches[0].cuda()
    table, mask, prefix = tables[0].cuda(), masks[0].cuda(), prefixes[0].cuda()
    slopes = torch.tensor([2.0 ** -h for h in range(H)], device="cuda")

    def both():
        return (fa.flash_forward_paged(q, kc, vc, table, lens, cu, 30, 500, tree_mask=mask, alibi_slopes=slopes),
                fa.flash_forward_paged(q, kc, vc, table, lens, cu, 30, 500, causal=True, softcap=8.0, prefix_lens=prefix))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        both()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = both()
    for s in (0, 1, 2, 0):
        b = batches[s]
        for dst, src in ((q, b.q), (kc, b.k_cache), (vc, b.v_cache), (table, tables[s]), (lens, b.lens), (mask, masks[s]), (prefix, prefixes[s])):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        eager = both()
        for r, e in zip(res, eager):
            assert torch.equal(r[0], e[0]) and torch.equal(r[1], e[1])
        ref.check(*res[0], ref.attention(b.q, b.k_cache, b.v_cache, tables[s], b.lens, b.cu, slopes=slopes.cpu(), mask=masks[s]), f"tree {s}")
        ref.check(*res[1], ref.attention(b.q, b.k_cache, b.v_cache, tables[s], b.lens, b.cu, causal=True, softcap=8.0, prefix=prefixes[s]), f"prefix {s}")


def test_long_chunks_in_order_and_in_pieces(fa):
    """Launches of many sequences with a prefix: row blocks ordered by the end of their keys, and the pieces that they have."""
    g = torch.Generator().manual_seed(0)
    news = [int(x) for x in torch.randint(1, 500, (9,), generator=g)]
    lens = [n + int(x) for n, x in zip(news, torch.randint(0, 300, (9,), generator=g))]
    batch = Batch(news, lens, 32, 8, 64, 16, torch.bfloat16, seed=11)
    how, kw = extras("prefix", 32, lens)
    ref.check(*call(fa, batch, how, kw, num_splits=1), want(batch, how, kw))
    news, lens = [700, 300], [700, 820]
    batch = Batch(news, lens, 8, 2, 64, 16, torch.bfloat16, seed=12)
    for prefix in ([0, 700], [333, 10], [700, 820]):
        how, kw = {"causal": True}, {"prefix": torch.tensor(prefix, dtype=torch.int32)}
        for splits in (2, 5):
            ref.check(*call(fa, batch, how, kw, num_splits=splits), want(batch, how, kw))

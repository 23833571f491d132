"""Other scores and masks over a paged cache, and drafted tokens, at the ends of their ranges: many sequences, pages far apart, the smallest cap, windows that
end inside a tile in front of a tree, calls side by side."""
import pytest
import torch

import scored_reference as ref
from paged_reference import Batch
from test_gpu_paged_scores import call, extras, tree, want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["both", "slopes", "prefix", "tree", "tree both"])
@pytest.mark.parametrize("longest,H,Hk,d,splits", [(4, 4, 2, 64, 0), (4, 8, 1, 128, 2), (60, 8, 2, 64, 1)])
def test_many_sequences(fa, kind, longest, H, Hk, d, splits):
    """More than a wave has lanes, some without new tokens, some without keys."""
    g = torch.Generator().manual_seed(longest + d)
    news = [int(x) for x in torch.randint(0, longest + 1, (71,), generator=g)]
    lens = [n + int(x) for n, x in zip(news, torch.randint(0, 150, (71,), generator=g))]
    lens[3] = lens[70] = 0
    batch = Batch(news, lens, H, Hk, d, 16, torch.bfloat16, seed=d)
    how, kw = tree(news, kind[5:], H, longest + d) if kind.startswith("tree") else extras(kind, H, lens)
    ref.check(*call(fa, batch, how, kw, num_splits=splits), want(batch, how, kw), kind)


@pytest.mark.parametrize("news,H,Hk", [([20, 3], 4, 2), ([40, 64], 48, 16), ([256, 250], 16, 1)])
@pytest.mark.parametrize("d,splits", [(64, 1), (128, 3)])
def test_windows_that_end_in_front_of_a_tree(fa, news, H, Hk, d, splits):
    """... inside the tile that the tree begins in, or a little in front of it."""
    for behind in (0, 5, 62, 63, 130):
        lens = [n + 64 * 9 + 30 for n in news]
        batch = Batch(news, lens, H, Hk, d, 16, torch.float16, seed=d + behind)
        for kind in ("", "slopes"):
            how, kw = tree(news, kind, H, 2)
            how["window"] = (max(news) - 1 + behind, -1)
            ref.check(*call(fa, batch, how, kw, num_splits=splits), want(batch, how, kw), f"{kind} {behind}")


def test_the_smallest_cap(fa):
    batch = Batch([3, 100], [40, 333], 8, 2, 64, 16, torch.float16, seed=1)
    slopes = torch.tensor([2.0 ** -h for h in range(8)])
    for kw in ({}, {"slopes": slopes}):
        how = {"causal": True, "softcap": fa.FLASH_MIN_SOFTCAP}
        ref.check(*call(fa, batch, how, kw), want(batch, how, kw))


def far_pages(cache, stride):
    """The cache's pages so many elements apart."""
    pages, Hk, page, d = cache.shape
    room = torch.empty((pages - 1) * stride + Hk * page * d, dtype=cache.dtype, device="cuda")
    far = torch.as_strided(room, cache.shape, (stride, page * d, d, 1))
    far.copy_(cache)
    return far


def test_pages_far_apart(fa):
    """Offsets past 32 bits, in bytes and in elements."""
    news, lens = [30, 2], [60, 20]
    batch = Batch(news, lens, 4, 2, 64, 16, torch.bfloat16, seed=3)
    stride = 2 ** 32 // (batch.k_cache.shape[0] - 2) // 8 * 8
    kc, vc = far_pages(batch.k_cache, stride), far_pages(batch.v_cache, stride)
    index = [t.cuda() for t in (batch.table, batch.lens, batch.cu)]
    parents = ref.random_parents(news, 1)
    mask, _ = ref.tree_mask(parents, batch.cu, batch.lens, 1)
    o, lse = fa.flash_forward_paged(batch.q.cuda(), kc, vc, *index, 30, 60, softcap=5.0, tree_mask=mask.cuda())
    ref.check(o, lse, want(batch, {"softcap": 5.0}, {"mask": mask}))
    path, accepted = torch.tensor([[2, 7, 11, 29], [1, 5, 5, 5]], dtype=torch.int32), torch.tensor([4, 1], dtype=torch.int32)
    k, v, after = ref.keep(batch.k_cache, batch.v_cache, batch.table, batch.lens, batch.cu, path, accepted)
    got = fa.flash_keep_paged(kc, vc, *index, path.cuda(), accepted.cuda())
    assert torch.equal(got.cpu(), after) and torch.equal(kc.cpu(), k) and torch.equal(vc.cpu(), v)


def test_calls_side_by_side(fa):
    """Two streams, each a step of its own: the results are those of one after the other."""
    parts = []
    for s in range(2):
        news, lens = [25 + 30 * s, 3], [700, 64 + s]
        batch = Batch(news, lens, 32, 8, 64 << s, 16, torch.bfloat16, seed=s)
        kw = {"parents": ref.random_parents(news, s).cuda()}
        path = torch.tensor([[1, 3, 8, 9], [0, 1, 2, 9]], dtype=torch.int32).cuda()
        parts.append((batch, batch.cuda(), kw["parents"], path, torch.tensor([4, 4], dtype=torch.int32).cuda(), torch.cuda.Stream()))

    def run(part, stream):
        batch, (q, kc, vc, table, lens, cu), parents, path, accepted, _ = part
        mask, _ = fa.flash_tree_mask(parents, cu, lens, max(batch.news), stream=stream)
        o, lse = fa.flash_forward_paged(q, kc, vc, table, lens, cu, max(batch.news), 700, num_splits=3, softcap=20.0, tree_mask=mask, stream=stream)
        caches = kc.clone(), vc.clone()
        stream.synchronize()
        torch.cuda.synchronize()
        return [mask, o, lse, fa.flash_keep_paged(*caches, table, lens, cu, path, accepted, stream=stream), *caches]

    torch.cuda.synchronize()
    alone = [run(p, p[-1]) for p in parts]
    torch.cuda.synchronize()
    for _ in range(3):
        masks, answers = [], []
        for batch, (q, kc, vc, table, lens, cu), parents, _, _, stream in parts:
            masks.append(fa.flash_tree_mask(parents, cu, lens, max(batch.news), stream=stream)[0])
        for _ in range(4):
            for (batch, (q, kc, vc, table, lens, cu), _, _, _, stream), mask in zip(parts, masks):
                answers.append(fa.flash_forward_paged(q, kc, vc, table, lens, cu, max(batch.news), 700, num_splits=3, softcap=20.0, tree_mask=mask, stream=stream))
        torch.cuda.synchronize()
        for i, (o, lse) in enumerate(answers):
            assert torch.equal(o, alone[i % 2][1]) and torch.equal(lse, alone[i % 2][2])
    for a, (batch, index, _, path, accepted, _) in zip(alone, parts):
        k, v, after = ref.keep(batch.k_cache, batch.v_cache, batch.table, batch.lens, batch.cu, path.cpu(), accepted.cpu())
        assert torch.equal(a[3].cpu(), after) and torch.equal(a[4].cpu(), k) and torch.equal(a[5].cpu(), v)

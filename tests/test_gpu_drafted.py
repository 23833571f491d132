"""flash_tree_mask, flash_keep_paged, and a whole step of checking drafted tokens."""
import pytest
import torch

import scored_reference as ref
from paged_reference import Batch

pytestmark = pytest.mark.gpu


def offsets(news, first=0):
    return torch.tensor([first + sum(news[:b]) for b in range(len(news) + 1)], dtype=torch.int32)


@pytest.mark.parametrize("news", [[1], [25], [64], [65, 3, 0, 1], [256, 1, 130], [200] * 70])
@pytest.mark.parametrize("shape", ["random", "chain", "star", "odd"])
def test_masks_and_positions(fa, news, shape):
    T, B = sum(news), len(news)
    within = torch.cat([torch.arange(n) for n in news])
    parents = {"random": lambda: ref.random_parents(news, T), "chain": lambda: within - 1, "star": lambda: torch.where(within == 0, -1, 0),
               "odd": lambda: torch.where(within % 5 == 0, within + 3, torch.where(within % 7 == 0, -9, within // 2 - 1))}[shape]().to(torch.int32)
    cu, lens = offsets(news), torch.tensor([n + 37 * b for b, n in enumerate(news)], dtype=torch.int32)
    words = max(1, -(-max(news) // 64))
    want = ref.tree_mask(parents, cu, lens, words)
    mask, positions = fa.flash_tree_mask(parents.cuda(), cu.cuda(), lens.cuda(), max(news))
    assert mask.shape == (T, words) and mask.dtype == torch.int64 and positions.dtype == torch.int32
    assert torch.equal(mask.cpu(), want[0]) and torch.equal(positions.cpu(), want[1])
    # without lengths, into rows of the caller's, on a stream of the caller's
    rows, at = torch.zeros((T, words + 3), dtype=torch.int64, device="cuda"), torch.zeros(T, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = fa.flash_tree_mask(parents.cuda(), cu.cuda(), None, max(news), mask=rows[:, 1:words + 1], positions=at, stream=s)
    s.synchronize()
    assert got[0].data_ptr() == rows[:, 1:].data_ptr() and torch.equal(rows[:, 1:words + 1].cpu(), want[0]) and torch.equal(at.cpu(), ref.tree_mask(parents, cu, None, words)[1])
    assert (rows[:, 0] == 0).all() and (rows[:, words + 1:] == 0).all()


def test_rows_of_no_sequence_and_chunks_longer_than_said(fa):
    news = [70, 5]
    cu = offsets(news, first=2)
    parents = torch.cat((torch.tensor([0, 0]), ref.random_parents(news, 1), torch.tensor([0])))
    mask, positions = torch.full((78, 1), 5, dtype=torch.int64, device="cuda"), torch.full((78,), 5, dtype=torch.int32, device="cuda")
    lens = torch.tensor([100, 5], dtype=torch.int32)
    fa.flash_tree_mask(parents.int().cuda(), cu.cuda(), lens.cuda(), 64, mask=mask, positions=positions)
    want = ref.tree_mask(parents[2:-1], offsets(news), lens, 1)
    for got, w in ((mask, want[0]), (positions, want[1])):
        assert torch.equal(got[2:-1].cpu(), w) and (got[:2] == 5).all() and got[-1] == 5
    # offsets that make no sense lead nowhere
    for bad in ([0, 100, 7], [-5, 3, 78], [9, 2, 1]):
        fa.flash_tree_mask(parents.int().cuda(), torch.tensor(bad, dtype=torch.int32, device="cuda"), lens.cuda(), 256)
    torch.cuda.synchronize()


def accepted_paths(news, seed):
    """Growing numbers below n, of all lengths; entries behind a path's end are not set."""
    g = torch.Generator().manual_seed(seed)
    L = max(max(news), 1)
    path, count = torch.full((len(news), L), -7, dtype=torch.int32), []
    for b, n in enumerate(news):
        k = int(torch.randint(0, n + 1, (1,), generator=g)) if b % 3 else min(n, 5)
        path[b, :k] = torch.randperm(n, generator=g)[:k].sort().values.int()
        count.append(k)
    return path, torch.tensor(count, dtype=torch.int32)


@pytest.mark.parametrize("news,lens", [([1], [1]), ([9, 1, 0, 30], [25, 64, 16, 30]), ([256, 100], [300, 107]), ([20] * 40, [20 + 3 * b for b in range(40)])])
@pytest.mark.parametrize("layers,Hk,d,page,dtype", [(0, 2, 64, 16, torch.float16), (3, 1, 8, 16, torch.bfloat16), (2, 8, 128, 48, torch.bfloat16), (1, 20, 80, 16, torch.float16)])
def test_keeps_the_path(fa, news, lens, layers, Hk, d, page, dtype):
    batch = Batch(news, lens, Hk, Hk, d, page, dtype, seed=len(news) + d)
    caches = [c if layers == 0 else torch.stack([c * (i + 1) for i in range(layers)]) for c in (batch.k_cache, batch.v_cache)]
    path, accepted = accepted_paths(news, d)
    want = ref.keep(*caches, batch.table, batch.lens, batch.cu, path, accepted)
    index = [t.cuda() for t in (batch.table, batch.lens, batch.cu, path, accepted)]
    got = [c.cuda() for c in caches]
    after = fa.flash_keep_paged(*got, *index)
    assert after.dtype == torch.int32 and torch.equal(after.cpu(), want[2]) and torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    # rows before heads in a page, results into a tensor of the caller's, on a stream of the caller's
    got = [c.cuda().transpose(-3, -2).contiguous().transpose(-3, -2) for c in caches]
    out, s = torch.zeros(len(news), dtype=torch.int32, device="cuda"), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    assert fa.flash_keep_paged(*got, *index, out=out, stream=s) is out
    s.synchronize()
    assert torch.equal(out.cpu(), want[2]) and torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_keep_of_what_makes_no_sense(fa):
    """Paths that do not grow, name no token or claim more than there is end where they do; places and pages that are not there are not touched."""
    news, lens = [6, 6, 6, 6, 6, 6], [30, 30, 30, 30, 30, 3]
    batch = Batch(news, lens, 2, 2, 64, 16, torch.float16, seed=2)
    path = torch.tensor([[1, 1, 2, 3], [0, 2, 6, 7], [3, 2, 4, 5], [2, 3, 4, 5], [-1, 2, 3, 4], [1, 2, 4, 5]], dtype=torch.int32)
    accepted = torch.tensor([4, 4, 4, 100, 4, 4], dtype=torch.int32)
    table = batch.table.clone()
    table[3, 1] = 10 ** 6
    want = ref.keep(batch.k_cache, batch.v_cache, table, batch.lens, batch.cu, path, accepted)
    assert want[2].tolist() == [25, 26, 25, 28, 24, 1]
    got = [c.cuda() for c in (batch.k_cache, batch.v_cache)]
    after = fa.flash_keep_paged(*got, table.cuda(), batch.lens.cuda(), batch.cu.cuda(), path.cuda(), accepted.cuda())
    assert torch.equal(after.cpu(), want[2]) and torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])
    for lens in ([-5] * 6, [2 ** 31 - 1] * 6):
        fa.flash_keep_paged(*got, table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"), batch.cu.cuda(), path.cuda(), (-accepted).cuda())
    torch.cuda.synchronize()
    assert torch.equal(got[0].cpu(), want[0])


def step(fa, q, k, v, kc, vc, table, lens, cu, parents, path, accepted, inv_freq, most):
    """One step of checking drafted trees: (answers, their LSE, mask, positions, lengths afterwards)"""
    mask, positions = fa.flash_tree_mask(parents, cu, lens, most)
    turned = fa.flash_append_paged(k, v, kc, vc, table, lens, cu, q=q, inv_freq=inv_freq, positions=positions)
    o, lse = fa.flash_forward_paged(turned, kc, vc, table, lens, cu, most, 600, tree_mask=mask)
    return o, lse, turned, positions, fa.flash_keep_paged(kc, vc, table, lens, cu, path, accepted)


@pytest.mark.parametrize("captured", [False, True])
def test_a_step_of_drafted_tokens(fa, captured):
    """The answers are those of each path by itself, and the cache afterwards is that of the accepted tokens alone."""
    news, lens, H, Hk, d, page = [12, 1, 40], [100, 30, 512], 4, 2, 64, 16
    dtype = torch.float16
    batch = Batch(news, lens, H, Hk, d, page, dtype, seed=5)
    g = torch.Generator().manual_seed(6)
    k, v = torch.randn((53, Hk, d), generator=g).to(dtype), torch.randn((53, Hk, d), generator=g).to(dtype)
    parents = ref.random_parents(news, 3)
    f = fa.rotary_frequencies(d)[0]
    # accepted: the whole path to a token in the middle of each tree
    path, count = torch.full((3, 40), -1, dtype=torch.int32), []
    for b, n in enumerate(news):
        on = ref.tree_paths(parents[int(batch.cu[b]):], n)[n * 3 // 4].nonzero()[:, 0]
        path[b, :len(on)] = on.int()
        count.append(len(on))
    accepted = torch.tensor(count, dtype=torch.int32)
    q, kc, vc, table, ln, cu = batch.cuda()
    args = [q, k.cuda(), v.cuda(), kc, vc, table, ln, cu, parents.cuda(), path.cuda(), accepted.cuda(), f.cuda(), 40]
    if captured:
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step(fa, *args)
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step(fa, *args)
        for _ in range(3):
            kc.copy_(batch.k_cache), vc.copy_(batch.v_cache)
            graph.replay()
            torch.cuda.synchronize()
    else:
        res = step(fa, *args)
    o, lse, turned, positions, after = (t.cpu() for t in res)
    mask, at = ref.tree_mask(parents, batch.cu, batch.lens, 1)
    assert torch.equal(positions, at) and after.tolist() == [n - m + c for n, m, c in zip(lens, news, count)]
    # the cache as the append leaves it, and what the path's rows make of it
    full = [c.cuda() for c in (batch.k_cache, batch.v_cache)]
    again = fa.flash_append_paged(args[1], args[2], *full, table, ln, cu, q=q, inv_freq=args[11], positions=at.cuda())
    assert torch.equal(again.cpu(), turned)
    full = [c.cpu() for c in full]
    ref.check(o, lse, ref.attention(turned, *full, batch.table, batch.lens, batch.cu, mask=mask))
    want = ref.keep(*full, batch.table, batch.lens, batch.cu, path, accepted)
    assert torch.equal(kc.cpu(), want[0]) and torch.equal(vc.cpu(), want[1])
    # a chain of the accepted tokens alone, appended and attended to in order, has the same keys in the same places, and the same answers within their bounds
    for b, n in enumerate(news):
        rows = batch.cu[b] + path[b, :count[b]].long()
        chain = [c.cuda() for c in (batch.k_cache, batch.v_cache)]
        own = (table[b:b + 1], after[b:b + 1].cuda(), torch.tensor([0, count[b]], dtype=torch.int32, device="cuda"))
        qs = fa.flash_append_paged(args[1][rows.cuda()], args[2][rows.cuda()], *chain, *own, q=q[rows.cuda()], inv_freq=args[11])
        assert torch.equal(qs.cpu(), turned[rows])
        o2, lse2 = fa.flash_forward_paged(qs, *chain, *own, causal=True)
        bound = ref.attention(qs.cpu(), *(c.cpu() for c in chain), batch.table[b:b + 1], after[b:b + 1], own[2].cpu(), causal=True)
        assert ((o[rows] - o2.cpu()).abs().double() <= 2 * bound[2]).all() and ((lse[rows] - lse2.cpu()).abs().double() <= 2 * bound[3]).all()
        for c, k in zip(chain, (kc, vc)):
            for j in range(int(after[b])):
                at_page = int(batch.table[b, j // page])
                assert torch.equal(c[at_page, :, j % page], k[at_page, :, j % page])


def test_front_end_and_own_path_agree(fa, monkeypatch):
    from flash_attn_amd import paged

    served = []
    real = paged._native or paged._front_end()

    class Spy:
        def __getattr__(self, name):
            def f(*a):
                r = getattr(real, name)(*a)
                served.append(r is not NotImplemented)
                return r
            return f

    monkeypatch.setattr(paged, "_native", Spy())
    here = torch.cuda.current_stream()
    news, lens = [9, 30], [50, 64]
    batch = Batch(news, lens, 4, 2, 64, 16, torch.bfloat16, seed=1)
    args = batch.cuda()
    parents = ref.random_parents(news, 1).cuda()
    a = fa.flash_tree_mask(parents, args[5], args[4], 30)
    assert served == [True]
    b = fa.flash_tree_mask(parents, args[5], args[4], 30, stream=here)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and served == [True]
    slopes = torch.rand(4, device="cuda")
    for kw in ({"tree_mask": a[0]}, {"softcap": 3.0, "alibi_slopes": slopes}, {"softcap": 3, "tree_mask": a[0]}, {"causal": True, "prefix_lens": torch.tensor([3, 9], dtype=torch.int32, device="cuda")}):
        before = len(served)
        x = fa.flash_forward_paged(*args, max_seqlen_q=30, **kw)
        assert served[before:] == [True]
        y = fa.flash_forward_paged(*args, max_seqlen_q=30, **kw, stream=here)
        assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])
    path, accepted = (t.cuda() for t in accepted_paths(news, 1))
    mine, other = [c.clone() for c in args[1:3]], [c.clone() for c in args[1:3]]
    versions = [c._version for c in mine]
    before = len(served)
    x = fa.flash_keep_paged(*mine, *args[3:], path, accepted)
    assert served[before:] == [True] and all(c._version > n for c, n in zip(mine, versions))
    y = fa.flash_keep_paged(*other, *args[3:], path, accepted, stream=here)
    assert torch.equal(x, y) and all(torch.equal(p, q) for p, q in zip(mine, other))
    with pytest.raises(fa.FlashError):
        fa.flash_keep_paged(*mine, *args[3:], path, accepted, out=args[4])


def test_nothing_to_do(fa):
    batch = Batch([0, 0], [5, 0], 2, 2, 64, 16, torch.float16)
    q, kc, vc, table, lens, cu = batch.cuda()
    mask, positions = fa.flash_tree_mask(torch.zeros(0, dtype=torch.int32, device="cuda"), cu, lens)
    assert mask.shape == (0, 1) and positions.shape == (0,)
    o, lse = fa.flash_forward_paged(q, kc, vc, table, lens, cu, tree_mask=mask, softcap=1.0)
    assert o.shape == (0, 2, 64) and lse.shape == (0, 2)
    for L in (0, 3):
        after = fa.flash_keep_paged(kc, vc, table, lens, cu, torch.zeros((2, L), dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"))
        assert after.tolist() == [5, 0]
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    assert fa.flash_keep_paged(kc, vc, table[:0], none, torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros((0, 3), dtype=torch.int32, device="cuda"), none).shape == (0,)

"""flash_append_paged and flash_forward_paged on the GPU against the 64-bit forms."""
import math

import pytest
import torch

import paged_reference as ref
from paged_reference import Batch

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def run(fa, batch, **kw):
    return fa.flash_forward_paged(*batch.cuda(), **kw)


def check(fa, batch, what="", **kw):
    masks = {k: kw[k] for k in ("causal", "window") if k in kw}
    o, lse = run(fa, batch, **kw)
    ref.check_attention(o, lse, batch.reference(scale=kw.get("softmax_scale"), **masks), what)
    return o, lse


# ---- one token per sequence, and a few


@pytest.mark.parametrize("d", [8, 40, 64, 72, 128])
@pytest.mark.parametrize("H,Hk", [(1, 1), (8, 1), (12, 4), (10, 2), (32, 1)])
def test_single_tokens(fa, H, Hk, d):
    lens = [1, 16, 63, 64, 65, 257, 700]
    dtype = F16 if d in (40, 128) else BF16
    check(fa, Batch([1] * len(lens), lens, H, Hk, d, 16, dtype, seed=d), max_seqlen_q=1, causal=True)


@pytest.mark.parametrize("splits", [1, 2, 5, 9, 128])
@pytest.mark.parametrize("dtype,d", [(F16, 64), (BF16, 128)])
def test_splits_of_single_tokens(fa, splits, dtype, d):
    lens = [3, 1000, 64, 0, 4099]
    check(fa, Batch([1] * 5, lens, 8, 2, d, 32, dtype, seed=splits), max_seqlen_q=1, causal=True, num_splits=splits)


@pytest.mark.parametrize("page", [16, 48, 64, 128, 256, 1008])
def test_page_sizes(fa, page):
    for news, H in (([1, 1, 1], 8), ([70, 3, 129], 8)):
        check(fa, Batch(news, [130, 500, 1300], H, 2, 128, page, F16, seed=page), causal=True)


@pytest.mark.parametrize("news,G", [([2, 1, 4], 8), ([32, 17, 31], 1), ([5, 6, 3], 5), ([16, 1, 0], 2)])
def test_few_tokens(fa, news, G):
    for causal in (False, True):
        check(fa, Batch(news, [40, 17, 333], 2 * G, 2, 64, 16, BF16, seed=G), causal=causal, max_seqlen_q=max(news))


# ---- chunks


@pytest.mark.parametrize("d", [8, 64, 80, 96, 120, 128])
@pytest.mark.parametrize("news,lens,H,Hk", [([33], [33], 1, 1), ([256, 1, 300], [256, 700, 301], 2, 2), ([513, 64], [900, 64], 4, 1), ([40, 0, 95], [1000, 77, 200], 6, 2)])
def test_chunks(fa, news, lens, H, Hk, d):
    dtype = BF16 if d in (64, 96, 128) else F16
    batch = Batch(news, lens, H, Hk, d, 16, dtype, seed=d + H)
    for causal in (False, True):
        check(fa, batch, causal=causal, max_seqlen_q=max(news))


@pytest.mark.parametrize("window", [(0, -1), (1, 0), (63, -1), (64, 5), (100, 100), (5000, -1), (-1, 0), (-1, 70), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("causal", [False, True])
def test_windows(fa, causal, window):
    for news, lens in (([1, 1, 1], [1, 400, 129]), ([200, 37], [600, 37])):
        batch = Batch(news, lens, 4, 2, 64, 16, F16, seed=window[0] % 1000 + 7)
        for splits in (0, 3):
            check(fa, batch, what=f"{news} {splits}", causal=causal, window=window, num_splits=splits)


@pytest.mark.parametrize("splits", [2, 3, 7, 40])
@pytest.mark.parametrize("dtype,d", [(BF16, 64), (F16, 128), (BF16, 72)])
def test_splits_of_chunks(fa, splits, dtype, d):
    check(fa, Batch([100, 3, 290], [1500, 100, 290], 4, 2, d, 16, dtype, seed=splits), causal=True, num_splits=splits)


def test_bounds_past_a_c_int(fa):
    batch = Batch([40], [300], 2, 1, 64, 16, F16, seed=24)
    want = run(fa, batch, causal=True, window=(-1, -1))
    for kw in (dict(window=(2 ** 32 + 5, -1)), dict(window=(-2 ** 32 + 5, 2 ** 40)), dict(max_seqlen_q=2 ** 40, max_seqlen_k=2 ** 33)):
        got = run(fa, batch, causal=True, **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_lengths_of_nothing(fa):
    """Sequences without keys, without new tokens, with more new tokens than keys: rows in front of key 0 see nothing."""
    for news, lens in (([1, 1, 1], [0, 5, 0]), ([40, 0, 3, 290], [10, 9, 0, 280]), ([2, 3], [1, 0])):
        for splits in (0, 2):
            for window in ((-1, -1), (3, -1)):
                check(fa, Batch(news, lens, 4, 2, 64, 16, F16), what=f"{news} {splits} {window}", causal=True, window=window, num_splits=splits)
    check(fa, Batch([40], [10], 4, 2, 64, 16, F16), causal=False)


def test_many_sequences(fa):
    """More sequences than a wave has lanes, with chunks of all kinds."""
    news = [(7 * b) % 90 for b in range(150)]
    lens = [n + (13 * b) % 200 for b, n in enumerate(news)]
    check(fa, Batch(news, lens, 2, 1, 64, 16, BF16, seed=5), causal=True)
    check(fa, Batch([1] * 150, [1 + (31 * b) % 500 for b in range(150)], 2, 1, 64, 16, F16, seed=6), causal=True, max_seqlen_q=1)


@pytest.mark.parametrize("H", [33, 64, 96, 128])
def test_one_head_for_many(fa, H):
    """More query heads per K/V head than a work-group of few rows has rows."""
    for news, lens in (([1, 1], [300, 90]), ([3, 2], [200, 65])):
        for splits in (0, 2):
            check(fa, Batch(news, lens, H, 1, 64, 16, BF16, seed=H), causal=True, max_seqlen_q=max(news), num_splits=splits)


def test_long_chunks_of_short_launches(fa):
    """Chunks of more than 64 rows that work-groups of 32 rows take, and the same sequences in a launch that they do not."""
    for d, dtype in ((64, F16), (128, BF16)):
        few = Batch([90, 500, 1], [200, 700, 64], 2, 2, d, 16, dtype, seed=21)
        check(fa, few, causal=True)
        check(fa, few, causal=True, window=(33, -1))
        check(fa, few)
        many = Batch([90] * 40, [200] * 40, 32, 32, d, 16, dtype, seed=22)
        o, lse = run(fa, many, causal=True)
        for b in (0, 17, 39):
            one = Batch([90], [200], 32, 32, d, 16, dtype)
            one.q, one.k_cache, one.v_cache, one.table = many.q[90 * b:90 * b + 90], many.k_cache, many.v_cache, many.table[b:b + 1]
            ref.check_attention(o[90 * b:90 * b + 90], lse[90 * b:90 * b + 90], one.reference(causal=True), f"{d} {b}")


@pytest.mark.parametrize("B,G,most", [(2, 4, 700), (3, 8, 400), (17, 2, 300), (64, 2, 80), (65, 2, 80)])
def test_row_blocks_of_all_sequences_by_length(fa, B, G, most):
    """Launches whose row blocks are ordered across sequences, and one of too many sequences for that: each block has its place, also where
    sequences are empty, rows stand in front of key 0, or the promised lengths are too short."""
    news = [most] + [(37 * b * most // 64 + b) % most for b in range(1, B)]
    lens = [max(0, n + (29 * b) % 150 - 40) for b, n in enumerate(news)]
    if B > 2:
        news[2], lens[2] = 0, 0
    batch = Batch(news, lens, 8 * G, 8, 64, 16, BF16, seed=B)
    for kw in (dict(causal=True), dict(causal=True, window=(50, -1)), dict(), dict(window=(-1, 33)), dict(window=(70, 0))):
        check(fa, batch, what=f"{kw}", num_splits=1, max_seqlen_q=max(news), **kw)
    want, got = run(fa, batch, causal=True, num_splits=1), run(fa, batch, causal=True, num_splits=1, max_seqlen_k=20)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("B,G,most,splits", [(1, 4, 1500, 7), (1, 4, 1500, 24), (2, 4, 700, 5), (3, 8, 400, 2), (17, 2, 300, 3), (17, 2, 300, 4), (16, 2, 300, 4), (3, 1, 300, 4),
                                             (1, 1, 333, 6), (32, 1, 70, 2)])
def test_pieces_that_row_blocks_have(fa, B, G, most, splits):
    """Splits of chunks whose first row blocks have fewer pieces than the last, in work-groups of 256 and of 32 rows, also where sequences are
    empty, rows stand in front of key 0, or the promised lengths are too short; two of too many sequences and splits for that order."""
    news = [most] + [(37 * b * most // 64 + b) % most for b in range(1, B)]
    lens = [max(0, n + (29 * b) % 250 - 60 * (b > 0)) for b, n in enumerate(news)]
    if B > 2:
        news[2], lens[2] = 0, 0
    Hk = 8 if B * G > 3 else 2
    batch = Batch(news, lens, Hk * G, Hk, 128, 16, F16, seed=B + splits)
    for kw in (dict(causal=True), dict(causal=True, window=(50, -1)), dict(), dict(window=(-1, 33)), dict(causal=True, max_seqlen_k=max(lens)),
               dict(causal=True, max_seqlen_k=40)):
        check(fa, batch, what=f"{kw}", num_splits=splits, max_seqlen_q=max(news), **kw)
    check(fa, batch, causal=True)


def test_no_pages(fa):
    """An empty pool, and a table without columns: rows see nothing, tokens go nowhere."""
    q, k = torch.randn((3, 4, 64), device="cuda").half(), torch.randn((3, 2, 64), device="cuda").half()
    lens, cu = torch.tensor([7, 2], dtype=torch.int32, device="cuda"), torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda")
    for pages, width in ((0, 4), (5, 0), (0, 0)):
        kc, vc = (torch.full((pages, 2, 16, 64), 3.0, dtype=F16, device="cuda") for _ in range(2))
        table = torch.zeros((2, width), dtype=torch.int32, device="cuda")
        for splits in (0, 4):
            o, lse = fa.flash_forward_paged(q, kc, vc, table, lens, cu, causal=True, num_splits=splits)
            assert (o == 0).all() and torch.isneginf(lse).all()
        f = fa.rotary_frequencies(64, device="cuda")[0]
        turned = fa.flash_append_paged(k, k, kc, vc, table, lens, cu, q=q, inv_freq=f)
        assert torch.isfinite(turned).all() and (kc == 3).all() and (vc == 3).all()
    assert fa.flash_forward_paged(q[:0], kc, vc, table[:0], lens[:0], cu[:1])[0].shape == (0, 4, 64)
    assert fa.flash_append_paged(k[:0], k[:0], kc, vc, table, lens, cu) is None


def test_shared_pages(fa):
    """Two sequences whose tables begin with the same pages, and one table for all."""
    batch = Batch([1, 40], [200, 300], 4, 2, 64, 16, F16, seed=23)
    batch.table[1, :10] = batch.table[0, :10]
    check(fa, batch, causal=True)
    q, k, v, table, lens, cu = batch.cuda()
    lens[:] = 200
    o, lse = fa.flash_forward_paged(q, k, v, table[:1].expand(2, -1), lens, cu, causal=True)
    batch.table[1] = batch.table[0]
    batch.lens[:] = 200
    ref.check_attention(o, lse, batch.reference(causal=True))


def test_promises_of_lengths_are_about_speed(fa):
    """max_seqlen_k below the truth, max_seqlen_q above it."""
    batch = Batch([1, 1], [3000, 2000], 8, 2, 128, 16, F16)
    for most in (1, 64, 500, 100000):
        check(fa, batch, causal=True, max_seqlen_q=1, max_seqlen_k=most)
        check(fa, batch, causal=True, max_seqlen_q=1, max_seqlen_k=most, num_splits=4)
    batch = Batch([50, 1], [3000, 2000], 8, 2, 64, 16, F16)
    for most in (50, 51, 1000):
        check(fa, batch, causal=True, max_seqlen_q=most, max_seqlen_k=64, num_splits=3)


def test_scale_and_large_scores(fa):
    batch = Batch([1, 60], [300, 400], 4, 2, 128, 16, BF16, seed=3)
    for scale in (1.0, 1e-3, 0.7):
        check(fa, batch, causal=True, softmax_scale=scale)


def test_rising_scores(fa):
    """Each tile's scores far above the last one's: the running maximum is raised again and again."""
    batch = Batch([1, 40], [900, 900], 2, 1, 64, 16, F16, seed=4)
    for b in range(2):
        j = torch.arange(900)
        batch.k_cache[batch.table[b].long()[j // 16], :, j % 16] *= (0.2 + j / 200.0)[:, None, None].half()
    check(fa, batch, causal=True)


# ---- what is not in the sequence


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("news,lens", [([1, 1, 1], [5, 130, 700]), ([40, 300], [70, 333])])
@pytest.mark.parametrize("dtype,d", [(F16, 64), (BF16, 128), (BF16, 80)])
def test_stale_rows(fa, dtype, d, news, lens, value):
    batch = Batch(news, lens, 4, 2, d, 32, dtype, seed=1, stale=value)
    for splits in (1, 3):
        check(fa, batch, causal=True, num_splits=splits)


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("dtype,d,H", [(F16, 64, 2), (BF16, 128, 4), (F16, 72, 2)])
def test_values_that_a_row_does_not_see(fa, dtype, d, H, value):
    """Not finite in K and V of keys right of the causal diagonal and left of the window: rows that see them have them, others do not."""
    for news, lens, window in (([300], [420], (-1, -1)), ([300], [420], (50, -1)), ([7], [200], (20, 3)), ([1], [200], (20, -1))):
        for which in ("k", "v", "kv"):
            batch = Batch(news, lens, H, 2, d, 16, dtype, seed=2)
            for j in (lens[0] - news[0] + 5, lens[0] - 2, 130):
                at, row = batch.table[0].long()[j // 16], j % 16
                if "k" in which:
                    batch.k_cache[at, :, row] = value if value != value else 0  # (an infinite K makes scores that have no maximum)
                if "v" in which:
                    batch.v_cache[at, :, row, 3] = value
            for splits in (1, 2):
                check(fa, batch, what=f"{news} {window} {which} {splits}", causal=True, window=window, num_splits=splits)


def test_keys_that_count_for_nothing(fa):
    """Keys with a score of -inf among others."""
    batch = Batch([3], [100], 2, 1, 64, 16, F16, seed=3)
    batch.q[:, :, 0] = 1.0
    batch.k_cache[:, :, 3, 0] = -math.inf
    check(fa, batch, causal=True)


def test_rows_of_nobody_stay(fa):
    """Rows in front of the first sequence and behind the last one."""
    for news, H in (([1, 1], 8), ([40, 70], 2)):
        batch = Batch(news, [900, 800], H, 2, 64, 16, F16, first=3, behind=5)
        for splits in (1, 4):
            T = batch.q.shape[0]
            o, lse = torch.full((T, H, 64), 7.0, dtype=F16, device="cuda"), torch.full((T, H), 7.0, device="cuda")
            fa.flash_forward_paged(*batch.cuda(), causal=True, num_splits=splits, out=o, lse=lse)
            ref.check_attention(o, lse, batch.reference(causal=True))
            for t in (o, lse):
                assert (t[:3] == 7).all() and (t[-5:] == 7).all()


# ---- layouts


@pytest.mark.parametrize("news", [[1, 1], [60, 200]])
def test_strides(fa, news):
    """Caches with heads behind the rows of a page, Q and O inside wider rows, a table inside a wider one."""
    batch = Batch(news, [333, 444], 4, 2, 128, 16, BF16, seed=9)
    q, k, v, table, lens, cu = batch.cuda()
    want = fa.flash_forward_paged(q, k, v, table, lens, cu, causal=True)
    kv = torch.stack((k, v), 2).transpose(1, 3).contiguous()  # [pages, page, 2, Hk, d]
    k2, v2 = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
    T = q.shape[0]
    wide_q, wide_o = torch.full((T, 8, 136), 3.0, dtype=BF16, device="cuda"), torch.full((T, 9, 160), 3.0, dtype=BF16, device="cuda")
    wide_q[:, 2:6, :128] = q
    wide_table = torch.full((2, table.shape[1] + 9), -1, dtype=torch.int32, device="cuda")
    wide_table[:, 2:2 + table.shape[1]] = table
    out = wide_o[:, 3:7, 16:144]
    o, lse = fa.flash_forward_paged(wide_q[:, 2:6, :128], k2, v2, wide_table[:, 2:2 + table.shape[1]], lens, cu, causal=True, out=out)
    assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
    wide_o[:, 3:7, 16:144] = 3.0
    assert (wide_o == 3).all()


def test_pages_past_32_bits(fa):
    """A cache of more than 4 GiB, the sequences in its last pages, old ones among them."""
    pages, page, Hk, d = 140000, 128, 2, 64
    k, v = (torch.empty((pages, Hk, page, d), dtype=F16, device="cuda") for _ in range(2))
    assert k.numel() * 2 > 2 ** 32
    for news in ([1, 1], [50, 1]):
        batch = Batch(news, [700, 300], 4, Hk, d, page, F16, seed=11)
        move = torch.randint(139000, 140000, (batch.k_cache.shape[0],), generator=torch.Generator().manual_seed(3)).unique()[:batch.k_cache.shape[0]]
        assert move.numel() == batch.k_cache.shape[0]
        k[move.cuda()], v[move.cuda()] = batch.k_cache.cuda(), batch.v_cache.cuda()
        table = torch.where(batch.table >= 0, move[batch.table.clamp(min=0).long()].int(), -1).cuda()
        q, _, _, _, lens, cu = batch.cuda()
        o, lse = fa.flash_forward_paged(q, k, v, table, lens, cu, causal=True)
        ref.check_attention(o, lse, batch.reference(causal=True))
        # and what is appended there
        new = torch.randn((q.shape[0], Hk, d), device="cuda").half()
        fa.flash_append_paged(new, -new, k, v, table, lens, cu)
        j = (lens.cpu() - 1).long()
        for b in range(2):
            at = int(table[b, int(j[b]) // page])
            assert torch.equal(k[at, :, int(j[b]) % page], new[int(cu[b + 1]) - 1]) and torch.equal(v[at, :, int(j[b]) % page], -new[int(cu[b + 1]) - 1])


def test_tables_with_pages_that_are_not_there(fa):
    """Entries outside the cache, lengths that the table cannot name: nothing outside the tensors is touched, other sequences are right."""
    batch = Batch([1, 1, 1], [300, 300, 300], 4, 2, 64, 16, F16, seed=12)
    good = batch.reference(causal=True)
    for entry in (-1, 10 ** 9, -2 ** 31):
        for length in (300, 10 ** 6, -5, 2 ** 31 - 1):
            q, k, v, table, lens, cu = batch.cuda()
            table[1, 3:] = entry
            lens[1] = length
            for splits in (1, 3):
                o, lse = fa.flash_forward_paged(q, k, v, table, lens, cu, causal=True, max_seqlen_q=1, num_splits=splits)
                for b in (0, 2):
                    ref.check_attention(o[b:b + 1], lse[b:b + 1], tuple(x[b:b + 1] for x in good))
            new = torch.ones((3, 2, 64), dtype=F16, device="cuda")
            k0, v0 = k.clone(), v.clone()
            fa.flash_append_paged(new, new, k, v, table, lens, cu)
            for b in (0, 2):
                k0[int(batch.table[b, 18]), :, 299 % 16] = 1
                v0[int(batch.table[b, 18]), :, 299 % 16] = 1
            assert torch.equal(k, k0) and torch.equal(v, v0)  # nothing of sequence 1
    # offsets of sequences that make no sense
    q, k, v, table, lens, cu = batch.cuda()
    for bad in ([0, 2, 1, 3], [-4, 1, 2, 3], [0, 1, 2, 10 ** 9], [5, 5, 5, 5], [3, 2, 1, 0]):
        cu.copy_(torch.tensor(bad, dtype=torch.int32))
        for most in (1, 0):
            o, lse = fa.flash_forward_paged(q, k, v, table, lens, cu, causal=True, max_seqlen_q=most)
            fa.flash_append_paged(q[:, :2], q[:, 2:], k, v, table, lens, cu)
    torch.cuda.synchronize()


@pytest.mark.parametrize("G,splits", [(8, 1), (8, 3), (1, 1), (1, 4)])
def test_offsets_that_make_no_sense(fa, G, splits):
    """In launches whose row blocks are ordered across sequences or come in pieces: rows in front of O and behind it stay as they are."""
    batch = Batch([300, 20, 80], [400, 20, 200], 8 * G, 8, 64, 16, F16, seed=G)
    q, k, v, table, lens, cu = batch.cuda()
    T, H = q.shape[0], q.shape[1]
    for bad in ([0, 300, 20, 400], [-4, 100, 200, 400], [0, 1, 399, 10 ** 9], [500, 500, 500, 500], [400, 300, 20, 0], [0, 2 ** 31 - 1, -2 ** 31, 400], [0, 400, 0, 400]):
        cu.copy_(torch.tensor(bad, dtype=torch.int32))
        for length in (None, -3, 2 ** 31 - 1):
            own = lens.clone()
            if length is not None:
                own[1] = length
            out, lse = torch.full((T + 64, H, 64), 7.0, dtype=F16, device="cuda"), torch.full((T + 64, H), 7.0, device="cuda")
            for most in (300, 0):
                fa.flash_forward_paged(q, k, v, table, own, cu, causal=True, max_seqlen_q=most, max_seqlen_k=400, num_splits=splits, out=out[32:32 + T], lse=lse[32:32 + T])
            for x in (out, lse):
                assert (x[:32] == 7).all() and (x[32 + T:] == 7).all()


# ---- calls


def test_same_bits_again(fa):
    for news, lens in (([1] * 6, [4000, 10, 2000, 777, 1, 64]), ([200, 3, 100], [900, 800, 100])):
        batch = Batch(news, lens, 8, 2, 128, 16, BF16, seed=13)
        o, lse = run(fa, batch, causal=True)
        for _ in range(3):
            o2, lse2 = run(fa, batch, causal=True)
            assert torch.equal(o, o2) and torch.equal(lse, lse2)


def test_workspace_and_streams(fa):
    batch = Batch([1, 1], [2000, 1000], 8, 2, 64, 16, F16, seed=14)
    args = batch.cuda()
    S = fa.paged_resolve_splits(2, 8, 2, 64, 2, 16, args[3].shape[1], max_seqlen_q=1, causal=True)
    assert S > 1
    ob, lb = fa.paged_workspace_bytes(2, 8, 2, 64, 2, 16, args[3].shape[1], max_seqlen_q=1, causal=True)
    assert (ob, lb) == (2 * 8 * S * 64 * 4, 2 * 8 * S * 4)
    o, lse = fa.flash_forward_paged(*args, causal=True, max_seqlen_q=1)
    own = torch.full((ob // 4,), math.nan, device="cuda"), torch.full((lb // 4,), math.nan, device="cuda")
    o2, lse2 = fa.flash_forward_paged(*args, causal=True, max_seqlen_q=1, workspace=own)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    with pytest.raises(ValueError):
        fa.flash_forward_paged(*args, causal=True, max_seqlen_q=1, workspace=(own[0][1:], own[1]))
    # two streams at once, each with results and workspace of its own
    sides = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s in sides:
            got.append(fa.flash_forward_paged(*args, causal=True, max_seqlen_q=1, stream=s))
        for s in sides:
            with torch.cuda.stream(s):
                got.append(fa.flash_forward_paged(*args, causal=True, max_seqlen_q=1))
    torch.cuda.synchronize()
    for o2, lse2 in got:
        assert torch.equal(o, o2) and torch.equal(lse, lse2)


def test_captured_steps_follow_lengths_and_pages(fa):
    """A captured step of append and attention, replayed as the sequences grow, beside a second graph and eager calls."""
    B, H, Hk, d, page, width = 3, 8, 2, 128, 16, 40
    g = torch.Generator().manual_seed(15)
    pool = torch.randperm(B * width, generator=g, dtype=torch.int32).view(B, width).cuda()
    k, v = (torch.randn((B * width, Hk, page, d), generator=g).half().cuda() for _ in range(2))
    lens, cu = torch.tensor([400, 15, 1], dtype=torch.int32, device="cuda"), torch.arange(B + 1, dtype=torch.int32, device="cuda")
    q, kn, vn = (torch.randn((B, h, d), generator=g).half().cuda() for h in (H, Hk, Hk))
    f = fa.rotary_frequencies(d, device="cuda")[0]

    def step(k, v):
        turned = fa.flash_append_paged(kn, vn, k, v, pool, lens, cu, q=q, inv_freq=f)
        return fa.flash_forward_paged(turned, k, v, pool, lens, cu, max_seqlen_q=1, causal=True)

    mine = k.clone(), v.clone()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step(k, v)
        graphs.append((graph, res))
    for n in range(6):
        lens.add_(1 if n else 0)
        q.normal_(), kn.normal_(), vn.normal_()
        want = step(*mine)
        torch.cuda.synchronize()
        for graph, res in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(res[0], want[0]) and torch.equal(res[1], want[1]), n
        assert torch.equal(k, mine[0]) and torch.equal(v, mine[1])


@pytest.mark.parametrize("G,splits", [(8, 1), (8, 3), (1, 4)])
def test_captured_chunks_follow_lengths_and_offsets(fa, G, splits):
    """A captured call of ragged chunks, in order of lengths or in pieces, replayed with other chunks of the same tokens."""
    Hk, d, T = 4, 64, 600
    batch = Batch([300, 100, 200], [700, 700, 700], Hk * G, Hk, d, 16, BF16, seed=31)
    q, k, v, table, lens, cu = batch.cuda()
    kw = dict(causal=True, num_splits=splits, max_seqlen_q=600, max_seqlen_k=700)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = fa.flash_forward_paged(q, k, v, table, lens, cu, **kw)
    for news, keys in (([300, 100, 200], [700, 100, 333]), ([600, 0, 0], [600, 20, 0]), ([0, 1, 599], [5, 700, 650]), ([200, 200, 200], [200, 100, 700]), ([7, 590, 3], [7, 700, 3])):
        cu.copy_(torch.tensor([0, news[0], news[0] + news[1], T], dtype=torch.int32))
        lens.copy_(torch.tensor(keys, dtype=torch.int32))
        want = fa.flash_forward_paged(q, k, v, table, lens, cu, **kw)
        torch.cuda.synchronize()
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, want[0]) and torch.equal(lse, want[1]), (news, keys)
        batch.cu, batch.lens = cu.cpu(), lens.cpu()
        ref.check_attention(o, lse, batch.reference(causal=True), f"{news} {keys}")


# ---- append


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(128, 128), (64, 32), (80, 40), (40, 6), (8, 8), (96, 0)])
def test_append(fa, dtype, interleaved, d, rot):
    """Ragged chunks into shuffled pages: turned K, V as it is, turned Q, everything else untouched."""
    news, lens, H, Hk = [1, 45, 0, 17], [33, 45, 12, 100], 6, 2
    batch = Batch(news, lens, H, Hk, d, 16, dtype, seed=d + rot, first=2, behind=3)
    q, k_cache, v_cache, table, lens_g, cu = batch.cuda()
    T = q.shape[0]
    g = torch.Generator().manual_seed(1)
    k, v = torch.randn((T, Hk, d), generator=g).to(dtype), torch.randn((T, Hk, d), generator=g).to(dtype)
    f, factor = (fa.rotary_frequencies(rot)[0], 1.2) if rot else (None, 1.0)
    place = torch.cat([torch.zeros(2, dtype=torch.long)] + [torch.arange(n - m, n) for m, n in zip(news, lens)] + [torch.zeros(3, dtype=torch.long)])
    owner = torch.cat([torch.full((m,), b) for b, m in enumerate(news)])
    for positions in (None, place * 7 + 1000000) if rot else (None,):
        kc, vc = k_cache.clone(), v_cache.clone()
        out = torch.full_like(q, 5.0)
        if rot:
            got = fa.flash_append_paged(k.cuda(), v.cuda(), kc, vc, table, lens_g, cu, q=q, inv_freq=f.cuda(), interleaved=interleaved, factor=factor,
                                        positions=None if positions is None else positions.cuda(), out=out)
            assert got is out
        else:
            assert fa.flash_append_paged(k.cuda(), v.cuda(), kc, vc, table, lens_g, cu) is None
        at = (batch.table[owner].long().gather(1, (place[2:-3] // 16)[:, None])[:, 0], place[2:-3] % 16)
        # V and everything that is not a new row, bit by bit
        want_v = batch.v_cache.clone()
        want_v[at[0], :, at[1]] = v[2:-3]
        assert torch.equal(vc.cpu(), want_v)
        rest = kc.cpu().clone()
        rest[at[0], :, at[1]] = batch.k_cache[at[0], :, at[1]]
        assert torch.equal(rest, batch.k_cache)
        new = kc.cpu()[at[0], :, at[1]]
        if not rot:
            assert torch.equal(new, k[2:-3])
            continue
        cos, sin = ref.angles((place if positions is None else positions).numpy()[2:-3], f.numpy())
        for x, y in ((k, new), (batch.q, out.cpu()[2:-3])):
            want = ref.rotate(x[2:-3], cos[:, None], sin[:, None], interleaved, factor)
            assert ((y.double() - want).abs() <= ref.rotate_bound(x[2:-3], cos[:, None], interleaved, factor, dtype, want)).all()
        assert (out[:2] == 5).all() and (out[-3:] == 5).all()


def test_append_in_place_and_strides(fa):
    """K, V and Q as slices of one projection, Q turned where it is; heads behind the rows of a page."""
    B, H, Hk, d = 5, 8, 2, 64
    lens, cu = torch.tensor([3, 17, 40, 1, 64], dtype=torch.int32, device="cuda"), torch.arange(B + 1, dtype=torch.int32, device="cuda")
    table = torch.randperm(B * 4, generator=torch.Generator().manual_seed(2), dtype=torch.int32).view(B, 4).cuda()
    f = fa.rotary_frequencies(d, device="cuda")[0]
    qkv = torch.randn((B, H + 2 * Hk, d), device="cuda").bfloat16()
    q, k, v = qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:]
    plain = [torch.zeros((20, Hk, 16, d), dtype=BF16, device="cuda") for _ in range(2)]
    want = fa.flash_append_paged(k.contiguous(), v.contiguous(), *plain, table, lens, cu, q=q.contiguous(), inv_freq=f)
    other = [torch.zeros((20, 16, Hk, d), dtype=BF16, device="cuda").transpose(1, 2) for _ in range(2)]
    kv = qkv[:, H:].clone()
    got = fa.flash_append_paged(k, v, *other, table, lens, cu, q=q, inv_freq=f, out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got, want) and torch.equal(qkv[:, H:], kv)
    assert torch.equal(other[0], plain[0]) and torch.equal(other[1], plain[1])


# ---- together


@pytest.mark.parametrize("chunks", [[1] * 9, [64, 100, 1, 1, 37], [300]])
@pytest.mark.parametrize("H,Hk,d", [(8, 2, 128), (4, 4, 64)])
def test_prompt_in_pieces(fa, chunks, H, Hk, d):
    """A sequence that grows chunk by chunk, two of them side by side, against flash_forward over the whole of it with turned Q and K."""
    B, N, page = 2, sum(chunks), 16
    g = torch.Generator().manual_seed(16)
    q, k, v = (torch.randn((B, N, h, d), generator=g).half().cuda() for h in (H, Hk, Hk))
    f = fa.rotary_frequencies(d, device="cuda")[0]
    pages = -(-N // page)
    table = torch.randperm(B * pages, generator=g, dtype=torch.int32).view(B, pages).cuda()
    kc, vc = (torch.full((B * pages, Hk, page, d), math.nan, dtype=F16, device="cuda") for _ in range(2))
    os, ls, done = [], [], 0
    for n in chunks:
        lens = torch.full((B,), done + n, dtype=torch.int32, device="cuda")
        cu = torch.arange(0, (B + 1) * n, n, dtype=torch.int32, device="cuda")
        new = [x[:, done:done + n].reshape(B * n, -1, d) for x in (q, k, v)]
        turned = fa.flash_append_paged(new[1], new[2], kc, vc, table, lens, cu, q=new[0], inv_freq=f)
        o, lse = fa.flash_forward_paged(turned, kc, vc, table, lens, cu, n, done + n, causal=True)
        os.append(o.view(B, n, H, d)), ls.append(lse.view(B, n, H))
        done += n
    turn = lambda x: fa.flash_rotary(x.transpose(1, 2), torch.arange(N, device="cuda"), f, out=torch.empty_like(x.transpose(1, 2).contiguous()))  # noqa: E731
    want, wl = fa.flash_forward(turn(q), turn(k), v.transpose(1, 2).contiguous(), causal=True)
    o, lse = torch.cat(os, 1).transpose(1, 2), torch.cat(ls, 1).transpose(1, 2)
    # both round P and O to fp16: twice (2 * 2^-11 |v| and 2^-11 |O|), |v| at most 6 here, and sum p |v| mostly below 1
    assert (o.float() - want.float()).abs().max() <= 4 * 2.0 ** -11 * v.abs().max()
    assert (lse - wl).abs().max() <= 1e-4  # the bound that flash_forward's own LSE is held to
    # the heads of a K/V head that were appended are those that flash_forward read
    j = torch.arange(N, device="cuda")
    assert torch.equal(kc[table[0].long()[j // page], :, j % page], turn(k)[0].transpose(0, 1))

"""The 256-row form of flash_forward_paged: every number of columns that it works on, pages and strides, masks, splits, values that are not finite, and launches
whose row blocks are ordered across sequences.  test_paged_forms.py sees to it that the calls below get that form."""
import math

import pytest
import torch

import paged_strict as strict
from paged_reference import Batch

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
DIMS = {8: 32, 32: 32, 40: 48, 48: 48, 56: 64, 64: 64, 72: 80, 80: 80, 88: 96, 96: 96, 104: 112, 112: 112, 120: 128, 128: 128}  # d -> columns worked on
# (tokens, keys, heads, K/V heads)
SHAPES = [([300, 70, 1], [333, 200, 64], 96, 96), ([300, 80, 90], [700, 80, 128], 80, 40), ([130, 0, 260], [1000, 50, 260], 90, 18)]
MASKS = [dict(causal=True), dict(), dict(causal=True, window=(45, -1)), dict(window=(100, 3))]


def dtype_of(d):
    """(of the two dimensions of each number of columns one has either type)"""
    return BF16 if d % 16 else F16


def reference(batch, **kw):
    return strict.attention(batch.q, batch.k_cache, batch.v_cache, batch.table, batch.lens, batch.cu, **kw)


def check(fa, batch, want, what="", **kw):
    got = fa.flash_forward_paged(*batch.cuda(), max_seqlen_q=max(batch.news), **kw)
    strict.check(*got, want, f"{what} {kw}")
    return got


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[2]}-{s[3]}")
@pytest.mark.parametrize("d", DIMS)
def test_columns(fa, d, shape):
    """Each number of columns in either type, whole and in splits, under each kind of mask."""
    news, lens, H, Hk = shape
    batch = Batch(news, lens, H, Hk, d, 16, dtype_of(d), seed=d)
    for mask in MASKS if shape is SHAPES[0] else MASKS[::2]:
        want = reference(batch, **mask)
        for splits in (1, 3):
            check(fa, batch, want, num_splits=splits, **mask)


@pytest.mark.parametrize("page", [48, 64, 144, 1008])
@pytest.mark.parametrize("d", [64, 80, 128])
def test_page_sizes(fa, d, page):
    news, lens, H, Hk = SHAPES[1]
    batch = Batch(news, lens, H, Hk, d, page, BF16, seed=page)
    want = reference(batch, causal=True)
    for splits in (1, 4):
        check(fa, batch, want, causal=True, num_splits=splits)


@pytest.mark.parametrize("d", [40, 72, 128])
def test_strides(fa, d):
    """Caches with heads behind the rows of a page, Q and O inside wider rows, a table inside a wider one."""
    news, lens, H, Hk = SHAPES[1]
    batch = Batch(news, lens, H, Hk, d, 32, F16, seed=9)
    q, k, v, table, lens, cu = batch.cuda()
    want = check(fa, batch, reference(batch, causal=True), causal=True)
    kv = torch.stack((k, v), 2).transpose(1, 3).contiguous()  # [pages, page, 2, Hk, d]
    T = q.shape[0]
    wide_q, wide_o = (torch.full((T, H + 5, d + 24), 3.0, dtype=F16, device="cuda") for _ in range(2))
    wide_q[:, 2:2 + H, :d] = q
    wide_table = torch.full((3, table.shape[1] + 9), -1, dtype=torch.int32, device="cuda")
    wide_table[:, 2:2 + table.shape[1]] = table
    out = wide_o[:, 3:3 + H, 16:16 + d]
    o, lse = fa.flash_forward_paged(wide_q[:, 2:2 + H, :d], kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2), wide_table[:, 2:2 + table.shape[1]], lens, cu,
                                    max(news), causal=True, out=out)
    assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
    wide_o[:, 3:3 + H, 16:16 + d] = 3.0
    assert (wide_o == 3).all()


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("d", [8, 48, 80, 112, 128])
def test_rows_of_nobody_stay(fa, d, splits):
    news, lens, H, Hk = SHAPES[0]
    batch = Batch(news, lens, H, Hk, d, 16, BF16, seed=d, first=3, behind=5)
    T = batch.q.shape[0]
    o, lse = torch.full((T, H, d), 7.0, dtype=BF16, device="cuda"), torch.full((T, H), 7.0, device="cuda")
    check(fa, batch, reference(batch, causal=True), causal=True, num_splits=splits, out=o, lse=lse)
    for t in (o, lse):
        assert (t[:3] == 7).all() and (t[-5:] == 7).all()


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("d", [40, 64, 80, 128])
def test_stale_rows(fa, d, value):
    """Rows of the cache that no sequence has."""
    news, lens, H, Hk = SHAPES[0]
    batch = Batch(news, lens, H, Hk, d, 48, dtype_of(d), seed=1, stale=value)
    want = reference(batch, causal=True)
    assert torch.isfinite(want[0]).all()
    for splits in (1, 3):
        check(fa, batch, want, causal=True, num_splits=splits)


@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("d", [8, 64, 72, 120])
def test_values_that_a_row_does_not_see(fa, d, value):
    """Not finite in K and V of keys right of the causal diagonal and left of the window: rows that see them have them, others do not."""
    news, lens, H, Hk = [300, 70, 1], [420, 200, 64], 96, 48
    for mask in (dict(causal=True), dict(causal=True, window=(50, -1)), dict(window=(20, 3))):
        for which in ("k", "v", "kv"):
            batch = Batch(news, lens, H, Hk, d, 16, dtype_of(d), seed=2)
            for b in (0, 1):
                for j in (lens[b] - news[b] + 5, lens[b] - 2, 130):
                    at, row = batch.table[b].long()[j // 16], j % 16
                    if "k" in which:
                        batch.k_cache[at, :, row] = value if value != value else 0  # (an infinite K makes scores that have no maximum)
                    if "v" in which:
                        batch.v_cache[at, :, row, 3] = value
            want = reference(batch, **mask)
            for splits in (1, 2):
                check(fa, batch, want, which, num_splits=splits, **mask)


@pytest.mark.parametrize("d", [32, 64, 80, 128])
def test_scales_and_rising_scores(fa, d):
    """Large and small scales, and tiles whose scores are each far above the last one's: the running maximum is raised again and again."""
    news, lens, H, Hk = SHAPES[1]
    batch = Batch(news, lens, H, Hk, d, 16, dtype_of(d), seed=3)
    for scale in (1.0, 1e-3):
        check(fa, batch, reference(batch, scale=scale, causal=True), softmax_scale=scale, causal=True)
    for b, n in enumerate(lens):
        j = torch.arange(n)
        batch.k_cache[batch.table[b].long()[j // 16], :, j % 16] *= (0.2 + j / 150.0)[:, None, None].to(dtype_of(d))
    want = reference(batch, causal=True)
    for splits in (1, 3):
        check(fa, batch, want, causal=True, num_splits=splits)


def test_lengths_of_nothing(fa):
    """Sequences without keys, without new tokens, with more new tokens than keys: rows in front of key 0 see nothing."""
    for d in (64, 96):
        batch = Batch([290, 0, 150, 40], [280, 9, 0, 10], 80, 40, d, 16, F16, seed=d)
        for mask in (dict(causal=True), dict(causal=True, window=(3, -1)), dict()):
            want = reference(batch, **mask)
            for splits in (1, 2):
                check(fa, batch, want, num_splits=splits, **mask)


@pytest.mark.parametrize("d", [48, 80, 128])
def test_same_bits_again(fa, d):
    news, lens, H, Hk = SHAPES[2]
    args = Batch(news, lens, H, Hk, d, 16, BF16, seed=13).cuda()
    for splits in (1, 3):
        kw = dict(max_seqlen_q=max(news), causal=True, num_splits=splits)
        o, lse = fa.flash_forward_paged(*args, **kw)
        for _ in range(3):
            o2, lse2 = fa.flash_forward_paged(*args, **kw)
            assert torch.equal(o, o2) and torch.equal(lse, lse2)


# ---- row blocks of all sequences, ordered by the end of their keys


def ordered_batch(B, d, Hk, G, most, seed=0):
    news = [most] + [(37 * b * most // 64 + b) % most for b in range(1, B)]
    lens = [max(0, n + (29 * b) % 150 - 40) for b, n in enumerate(news)]
    if B > 2:
        news[2], lens[2] = 0, 0
    return Batch(news, lens, Hk * G, Hk, d, 16, BF16, seed=seed)


ORDERED = [(2, 64, 16, 4, 700), (3, 128, 16, 8, 400), (9, 80, 8, 4, 500), (64, 64, 4, 2, 300)]  # B, d, K/V heads, group, longest chunk


@pytest.mark.parametrize("shape", ORDERED, ids=str)
def test_ordered(fa, shape):
    """Each block has its place, also where sequences are empty, rows stand in front of key 0, or the promised lengths are too short."""
    batch = ordered_batch(*shape, seed=shape[0])
    for mask in (dict(causal=True), dict(causal=True, window=(50, -1)), dict(), dict(window=(-1, 33))):
        check(fa, batch, reference(batch, **mask), num_splits=1, **mask)
    args, kw = batch.cuda(), dict(causal=True, num_splits=1, max_seqlen_q=max(batch.news))
    want, got = fa.flash_forward_paged(*args, **kw), fa.flash_forward_paged(*args, max_seqlen_k=20, **kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


SENSELESS = dict(news=[300, 20, 80], lens=[400, 20, 200], d=64, Hk=32, G=8)


def test_offsets_that_make_no_sense_in_ordered_launches(fa):
    """Rows in front of O and behind it stay as they are."""
    c = SENSELESS
    batch = Batch(c["news"], c["lens"], c["Hk"] * c["G"], c["Hk"], c["d"], 16, F16, seed=8)
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
                fa.flash_forward_paged(q, k, v, table, own, cu, causal=True, max_seqlen_q=most, max_seqlen_k=400, num_splits=1, out=out[32:32 + T], lse=lse[32:32 + T])
            for x in (out, lse):
                assert (x[:32] == 7).all() and (x[32 + T:] == 7).all()


CAPTURED = dict(news=[300, 100, 200], lens=[700, 700, 700], d=64, Hk=16, G=8)


@pytest.mark.parametrize("splits", [1, 3])
def test_captured_chunks_follow_lengths_and_offsets(fa, splits):
    """A captured call, ordered (one split) or in pieces, replayed with other chunks of the same tokens."""
    c, T = CAPTURED, 600
    batch = Batch(c["news"], c["lens"], c["Hk"] * c["G"], c["Hk"], c["d"], 16, BF16, seed=31)
    q, k, v, table, lens, cu = batch.cuda()
    kw = dict(causal=True, num_splits=splits, max_seqlen_q=T, max_seqlen_k=700)
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
        strict.check(o, lse, reference(batch, causal=True), f"{news} {keys}")

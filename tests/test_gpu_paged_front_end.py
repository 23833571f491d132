"""The native front end's rotary, append and paged against paged.py's own path, which calls on a given stream take."""
import pytest
import torch

from paged_reference import Batch

pytestmark = pytest.mark.gpu


class Spy:
    """Counts what the front end served."""

    def __init__(self, real):
        self.real, self.served = real, 0

    def __getattr__(self, name):
        f = getattr(self.real, name)

        def call(*args):
            res = f(*args)
            self.served += res is not NotImplemented
            return res

        return call


@pytest.fixture
def spy(fa, monkeypatch):
    from flash_attn_amd import paged

    s = Spy(paged._native or paged._front_end())
    assert hasattr(s.real, "bind_paged"), "the native front end has not been built"
    monkeypatch.setattr(paged, "_native", s)
    return s


def same(a, b):
    a, b = (x if isinstance(x, tuple) else (x,) for x in (a, b))
    return len(a) == len(b) and all(x is y is None or (torch.equal(x, y) and x.stride() == y.stride()) for x, y in zip(a, b))


@pytest.mark.parametrize("kw", [{}, {"causal": True, "max_seqlen_q": 1}, {"window": (30, -1), "causal": True}, {"softmax_scale": 1}, {"num_splits": 3, "max_seqlen_k": 500}])
def test_forward(fa, spy, kw):
    args = Batch([1, 1], [700, 65], 8, 2, 64, 16, torch.bfloat16).cuda()
    got = fa.flash_forward_paged(*args, **kw)
    assert spy.served == 1
    assert same(got, fa.flash_forward_paged(*args, **kw, stream=torch.cuda.current_stream()))
    out, lse = torch.empty_like(got[0]), torch.empty_like(got[1])
    mine = fa.flash_forward_paged(*args, **kw, out=out, lse=lse, workspace=(torch.empty(100000, device="cuda"), torch.empty(2000, device="cuda")))
    assert spy.served == 2 and mine[0] is not None and mine[0].data_ptr() == out.data_ptr() and same(mine, got)


def test_append_and_rotary(fa, spy):
    batch = Batch([3, 1], [70, 65], 8, 2, 64, 16, torch.float16)
    q, kc, vc, table, lens, cu = batch.cuda()
    k, f = torch.randn((4, 2, 64), device="cuda").half(), fa.rotary_frequencies(32, device="cuda")[0]
    pos = torch.tensor([5, 6, 7, 8], device="cuda")
    for kw in ({}, {"inv_freq": f}, {"inv_freq": f, "q": q, "interleaved": True, "factor": 1.5}, {"inv_freq": f, "q": q, "positions": pos}):
        caches = [c.clone() for c in (kc, vc, kc, vc)]
        before = spy.served
        a = fa.flash_append_paged(k, -k, *caches[:2], table, lens, cu, **kw)
        assert spy.served == before + 1
        b = fa.flash_append_paged(k, -k, *caches[2:], table, lens, cu, **kw, stream=torch.cuda.current_stream())
        assert (a is None) == ("q" not in kw) and same(a, b) and torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])
    for x, p in ((q, pos), (torch.randn((2, 3, 4, 40), device="cuda"), pos.int()), (torch.randn((2, 4, 3, 40), device="cuda").transpose(1, 2), torch.arange(8, device="cuda").view(2, 4))):
        for kw in ({}, {"interleaved": True, "inverse": True, "factor": 2}):
            before = spy.served
            a = fa.flash_rotary(x, p, f[:16], **kw)
            assert spy.served == before + 1
            assert same(a, fa.flash_rotary(x, p, f[:16], **kw, stream=torch.cuda.current_stream()))


def test_leaves_what_it_cannot_serve(fa, spy):
    q, kc, vc, table, lens, cu = Batch([1, 1], [70, 65], 8, 2, 64, 16, torch.float16).cuda()
    f, pos = fa.rotary_frequencies(32, device="cuda")[0], torch.arange(2, device="cuda")
    for bad in (lambda: fa.flash_forward_paged(q[:, :3], kc, vc, table, lens, cu), lambda: fa.flash_forward_paged(q, kc, vc, table.long(), lens, cu),
                lambda: fa.flash_forward_paged(q, kc, vc[:1], table, lens, cu), lambda: fa.flash_forward_paged(q.cpu(), kc, vc, table, lens, cu),
                lambda: fa.flash_append_paged(q, q, kc, vc, table, lens, cu), lambda: fa.flash_append_paged(q[:, :2], q[:, :2], kc, vc, table, lens, cu, q=q),
                lambda: fa.flash_rotary(q, pos.float(), f), lambda: fa.flash_rotary(q, pos[:1], f), lambda: fa.flash_rotary(q, pos, f.cpu())):
        with pytest.raises(ValueError):
            bad()
    assert spy.served == 0
    with pytest.raises(fa.FlashError):  # the library's own refusal
        fa.flash_forward_paged(q, kc, vc, table, lens, cu, softmax_scale=0.0)
    x = torch.randn((2, 8, 64), device="cuda", requires_grad=True)
    y = fa.flash_rotary(x, pos, f)
    assert y.requires_grad and spy.served == 1  # (the call inside, where no gradient is asked for)
    assert fa.flash_rotary(x.detach(), pos, f).requires_grad is False and spy.served == 2

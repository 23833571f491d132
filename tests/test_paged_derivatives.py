"""What flash_append_paged, flash_forward_paged and flash_rotary do with tensors that derivatives are asked of: no result may be detached from one of them without a
word.  No GPU needed: every call here ends before anything is launched."""
import pytest
import torch


def tensors():
    f16 = torch.float16
    return dict(k=torch.zeros((3, 2, 64), dtype=f16), v=torch.zeros((3, 2, 64), dtype=f16), k_cache=torch.zeros((8, 2, 16, 64), dtype=f16),
                v_cache=torch.zeros((8, 2, 16, 64), dtype=f16), block_table=torch.zeros((2, 4), dtype=torch.int32), seqlens_k=torch.zeros(2, dtype=torch.int32),
                cu_seqlens_q=torch.zeros(3, dtype=torch.int32), q=torch.zeros((3, 4, 64), dtype=f16), inv_freq=torch.ones(32), out=torch.zeros((3, 4, 64), dtype=f16),
                lse=torch.zeros((3, 4)))


APPEND = ("k", "v", "k_cache", "v_cache", "block_table", "seqlens_k", "cu_seqlens_q", "q", "inv_freq", "out")
FORWARD = ("q", "k_cache", "v_cache", "block_table", "seqlens_k", "cu_seqlens_q", "out", "lse")


def calls(fa, name):
    """The calls that take an argument of that name."""
    t = tensors()
    t[name].requires_grad_()
    if name in APPEND:
        yield lambda: fa.flash_append_paged(**{x: t[x] for x in APPEND})
    if name in FORWARD:
        yield lambda: fa.flash_forward_paged(**{x: t[x] for x in FORWARD})


@pytest.mark.parametrize("name", [x for x in tensors() if x not in ("block_table", "seqlens_k", "cu_seqlens_q")])
def test_tensors_that_require_a_gradient(fa, name):
    for call in calls(fa, name):
        with pytest.raises(ValueError, match="has no gradients"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="must be on the GPU"):  # (gets past that)
            call()


@pytest.mark.parametrize("name", [x for x, t in tensors().items() if t.is_floating_point()])
def test_forward_mode(fa, name):
    from torch.autograd import forward_ad

    def give_tangent(t):
        t[name] = forward_ad.make_dual(t[name], torch.ones_like(t[name]))
        return t

    with forward_ad.dual_level():
        for names, f in ((APPEND, fa.flash_append_paged), (FORWARD, fa.flash_forward_paged)):
            if name in names:
                t = give_tangent(tensors())
                with pytest.raises(ValueError, match="has no forward-mode derivatives"):
                    f(**{x: t[x] for x in names})
        if name in ("q", "inv_freq", "out"):  # (rotary's x, inv_freq and out)
            t = give_tangent(tensors())
            for x in (t["q"], t["q"].detach().requires_grad_()) if name != "q" else (t["q"],):
                with pytest.raises(ValueError, match="has no forward-mode derivatives"):
                    fa.flash_rotary(x, torch.arange(3), t["inv_freq"], out=t["out"])

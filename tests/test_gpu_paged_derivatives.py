"""flash_rotary, flash_append_paged and flash_forward_paged beside autograd: derivatives that a call would drop are refused, on the native front end's way
and on paged.py's own."""
import pytest
import torch

from paged_reference import Batch

pytestmark = pytest.mark.gpu


def setup(fa):
    """Arguments of a step by name, [append, forward]"""
    q, k_cache, v_cache, table, lens, cu = Batch([1, 2], [70, 65], 4, 2, 64, 16, torch.float16).cuda()
    k, v = torch.randn((3, 2, 64), device="cuda").half(), torch.randn((3, 2, 64), device="cuda").half()
    cache = dict(k_cache=k_cache, v_cache=v_cache, block_table=table, seqlens_k=lens, cu_seqlens_q=cu)
    return (dict(k=k, v=v, q=q, inv_freq=fa.rotary_frequencies(64, device="cuda")[0], out=torch.empty_like(q), **cache),
            dict(q=q, out=torch.empty_like(q), lse=torch.empty((3, 4), device="cuda"), **cache))


@pytest.mark.parametrize("own_stream", [False, True])
def test_tensors_that_require_a_gradient(fa, own_stream):
    stream = torch.cuda.current_stream() if own_stream else None
    for which, f in enumerate((fa.flash_append_paged, fa.flash_forward_paged)):
        names = [n for n, t in setup(fa)[which].items() if t.is_floating_point()]
        assert len(names) == (7, 5)[which]
        for name in names:
            args = setup(fa)[which]
            want = f(**{n: t.clone() for n, t in args.items()}, stream=stream)
            args[name].requires_grad_()
            with pytest.raises(ValueError, match="has no gradients"):
                f(**args, stream=stream)
            with torch.no_grad():
                got = f(**args, stream=stream)
            for a, b in zip(got, want):
                assert torch.equal(a, b)


@pytest.mark.parametrize("own_stream", [False, True])
def test_forward_mode(fa, own_stream):
    from torch.autograd import forward_ad

    stream = torch.cuda.current_stream() if own_stream else None
    step = setup(fa)
    rotary = dict(x=step[0]["q"], positions=torch.arange(3, device="cuda"), inv_freq=step[0]["inv_freq"])
    with forward_ad.dual_level(), torch.no_grad():
        for f, args in ((fa.flash_append_paged, step[0]), (fa.flash_forward_paged, step[1]), (fa.flash_rotary, rotary)):
            for name, t in args.items():
                if t.is_floating_point():
                    with pytest.raises(ValueError, match="has no forward-mode derivatives"):
                        f(**dict(args, **{name: forward_ad.make_dual(t, torch.ones_like(t))}), stream=stream)
            f(**args, stream=stream)


@pytest.mark.parametrize("own_stream", [False, True])
def test_tensors_that_are_written(fa, own_stream):
    """A backward pass that has saved a tensor which a call then writes must not go on with what it finds there; what a call reads alone stays as it was,
    and tensors of inference mode, which count nothing, are written too."""
    stream = torch.cuda.current_stream() if own_stream else None
    append, forward = setup(fa)
    rotary = dict(x=append["q"], positions=torch.arange(3, device="cuda"), inv_freq=append["inv_freq"], out=append["out"])
    forward.update(num_splits=2, workspace=(torch.empty(100000, device="cuda"), torch.empty(1000, device="cuda")))
    in_place = dict(rotary, x=rotary["out"])
    for f, args, writes in ((fa.flash_rotary, rotary, ("out",)), (fa.flash_rotary, in_place, ("x",)), (fa.flash_append_paged, append, ("k_cache", "v_cache", "out")),
                            (fa.flash_forward_paged, forward, ("out", "lse"))):
        given = {n: t for n, t in args.items() if isinstance(t, torch.Tensor)}
        for name in writes:
            w = torch.ones((), device="cuda", dtype=given[name].dtype, requires_grad=True)
            loss = (w * given[name]).sum()
            f(**args, stream=stream)
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                loss.backward()
        before = {n: t._version for n, t in given.items()}
        f(**args, stream=stream)
        written = {n for n, t in given.items() if t._version != before[n]}
        assert written - {"x", "out"} == set(writes) - {"x", "out"} and set(writes) <= written, f
    assert all(t._version > 0 for t in forward["workspace"])
    with torch.inference_mode():
        append, forward = setup(fa)
        fa.flash_append_paged(**append, stream=stream)
        fa.flash_forward_paged(**forward, stream=stream)
        fa.flash_rotary(append["q"], rotary["positions"], rotary["inv_freq"], out=append["q"], stream=stream)

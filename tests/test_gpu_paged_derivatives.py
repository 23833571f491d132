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

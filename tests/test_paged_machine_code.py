"""Waits in the built code of the paged attention that no result shows to be there: whether a read of LDS comes before the request that fills it has
landed depends on the moment.  No GPU needed."""
import functools

import machine_code
from flash_attn_amd import binding


@functools.lru_cache(maxsize=None)
def tall_kernels():
    return [(name, code) for name, code in machine_code.kernels(binding.library_path()) if "paged_tall_kernel" in name]


def test_barriers_in_front_of_the_loop_wait_for_tiles():
    """The 256-row form passes four barriers in front of its loop: columns cleared; K(0) there; V(0) and K(1) there; and, the second group of waves alone, which
    runs half an iteration behind, V(1) there, since the first group reads that in front of the barrier that ends the second one's
    first iteration.  Each of the last three has a wait for requests since the barrier before it."""
    assert len(tall_kernels()) == 14  # 32, 48, 64, 80, 96, 112 and 128 columns, fp16 and bf16
    for name, code in tall_kernels():
        barriers = [i for i, (op, _) in enumerate(code) if op == "s_barrier"][:4]
        for before, at in zip(barriers, barriers[1:]):
            assert any(op == "s_waitcnt" and "vmcnt" in args for op, args in code[before:at]), (name, barriers.index(at))

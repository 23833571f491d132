"""Which form of the paged attention the calls of the GPU tests get, so that a change of the rules cannot leave a form without its tests.  No GPU needed."""
from paged_launches import call, record

import test_gpu_paged_last_key as last_key


def test_last_key_reaches_both_forms():
    for shapes, form in ((last_key.FEW, "few"), (last_key.TALL, "tall")):
        calls = [call(*shape, d, causal=causal, max_seqlen_q=max(shape[0]), num_splits=splits)
                 for shape in shapes for d in (8, 40, 64, 80, 128) for causal in (0, 1) for splits in (1, 3)]
        launches = record(calls)
        assert {x["form"] for x in launches} == {form}
        assert max(x["splits"] for x in launches) > 1

"""Every case of test_gpu_scored_orders.py is an ordered launch of 256-row work-groups.  No GPU needed."""
import test_gpu_scored_forms as forms
import test_gpu_scored_orders as orders
from scored_launches import record


def test_orders():
    calls = [forms.arguments(*shape, 1, mask, kind) for shape, mask, kind in orders.CASES]
    calls += [forms.arguments(*shape, 1, {}, kind, -(-max(shape[0]) // 64)) for shape, kind in orders.TREE_CASES]
    for c, x in zip(calls, record(calls)):
        assert x["form"] == "tall" and x["ordered"] > 0 and not x["direct"] and x["splits"] == 1, (c, x)

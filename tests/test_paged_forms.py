"""Which form of the paged attention the calls of the GPU tests get, so that a change of the rules cannot leave a form without its tests.  No GPU needed."""
from paged_launches import call, record

import test_gpu_paged_last_key as last_key
import test_gpu_paged_odd_scores as odd_scores
import test_gpu_paged_tall as tall


def test_last_key_reaches_both_forms():
    for shapes, form in ((last_key.FEW, "few"), (last_key.TALL, "tall")):
        calls = [call(*shape, d, causal=causal, max_seqlen_q=max(shape[0]), num_splits=splits)
                 for shape in shapes for d in (8, 40, 64, 80, 128) for causal in (0, 1) for splits in (1, 3)]
        launches = record(calls)
        assert {x["form"] for x in launches} == {form}
        assert max(x["splits"] for x in launches) > 1


def test_tall_tests_reach_the_tall_form_and_all_its_columns():
    calls, columns = [], []
    for news, lens, H, Hk in tall.SHAPES + [([300, 70, 1], [420, 200, 64], 96, 48), ([290, 0, 150, 40], [280, 9, 0, 10], 80, 40)]:
        for d in tall.DIMS:
            for mask in tall.MASKS:
                for splits in (1, 3):
                    calls.append(call(news, lens, H, Hk, d, max_seqlen_q=max(news), num_splits=splits, dtype="bf16" if d % 16 else "fp16", **mask))
                    columns.append(tall.DIMS[d])
    for page in (48, 64, 144, 1008):
        news, lens, H, Hk = tall.SHAPES[1]
        for d in (64, 80, 128):
            calls.append(call(news, lens, H, Hk, d, page, max_seqlen_q=max(news), num_splits=4, causal=True))
            columns.append(tall.DIMS[d])
    launches = record(calls)
    assert {x["form"] for x in launches} == {"tall"} and [x["columns"] for x in launches] == columns
    assert {x["splits"] for x in launches} >= {1, 2, 3} and any(x["pieces"] for x in launches)


def test_ordered_tests_reach_ordered_launches():
    calls = []
    for B, d, Hk, G, most in tall.ORDERED:
        batch = tall.ordered_batch(B, d, Hk, G, most)
        for mask in (dict(causal=True), dict(causal=True, window=(50, -1)), dict(), dict(window=(-1, 33)), dict(causal=True, max_seqlen_k=20)):
            calls.append(call(batch.news, batch.lens.tolist(), Hk * G, Hk, d, max_seqlen_q=most, num_splits=1, **mask))
    for c, most, width in ((tall.SENSELESS, 300, 0), (tall.SENSELESS, 0, 400), (tall.CAPTURED, 600, 700)):
        calls.append(call(c["news"], c["lens"], c["Hk"] * c["G"], c["Hk"], c["d"], max_seqlen_q=most, max_seqlen_k=width, num_splits=1, causal=True))
    for c, x in zip(calls, record(calls)):
        assert x["form"] == "tall" and x["ordered"] > 0 and not x["direct"], (c, x)
    c = tall.CAPTURED
    x, = record([call(c["news"], c["lens"], c["Hk"] * c["G"], c["Hk"], c["d"], max_seqlen_q=600, max_seqlen_k=700, num_splits=3, causal=True)])
    assert x["form"] == "tall" and x["pieces"]


def test_odd_scores_reach_both_forms():
    for shapes, form in ((odd_scores.FEW, "few"), (odd_scores.TALL, "tall")):
        calls = [call(*shape, d, max_seqlen_q=max(shape[0]), num_splits=splits, **mask) for shape in shapes for d in (40, 64, 128) for splits in (1, 2)
                 for mask in (dict(), dict(causal=True), dict(causal=True, window=(30, -1)), dict(window=(60, 2)))]
        assert {x["form"] for x in record(calls)} == {form}

"""Every case of test_gpu_scored_forms.py and test_gpu_steep_slopes.py gets the form that it is there for, and the kernel of its scores.  No GPU needed."""
import test_gpu_scored_forms as forms
import test_gpu_steep_slopes as steep
from test_scored_arguments import launched

KINDS = {"": 1, "prefix": 1, "cap": 2, "cap prefix": 2, "slopes": 3, "slopes prefix": 3, "both": 4, "both prefix": 4}


def test_forms():
    calls, want, cases = [], [], forms.CASES + forms.TREE_CASES + forms.LAST_CASES
    for form, news, lens, H, Hk, splits, mask, kind, d in forms.CASES:
        calls.append(forms.arguments(news, lens, H, Hk, d, splits, mask, kind))
        want.append([form, KINDS[kind]])
    for form, news, lens, H, Hk, splits, window, kind, d in forms.TREE_CASES:
        calls.append(forms.arguments(news, lens, H, Hk, d, splits, {"window": (window, -1)}, kind, -(-max(news) // 64)))
        want.append([form, KINDS[kind]])
    for form, news, lens, H, Hk, splits, kind, d in forms.LAST_CASES:
        calls.append(forms.arguments(news, lens, H, Hk, d, splits, forms.CAUSAL, kind))
        want.append([form, KINDS[kind]])
    wrong = [(case, got) for case, got, w in zip(cases, launched(calls), want) if got != w]
    assert not wrong, "\n".join(str(x) for x in wrong)


def test_every_form_has_every_kind():
    masks = {"causal": lambda m: m == forms.CAUSAL, "left": lambda m: m.get("window", (-1, -1))[0] >= 0, "right": lambda m: not m.get("causal") and m.get("window", (-1, -1))[1] >= 0}
    for form in ("few", "mid", "paired", "tall"):
        mine = [c for c in forms.CASES if c[0] == form]
        assert {c[7] for c in mine} == set(forms.SCORES)
        for name, is_one in masks.items():
            if (form, name) != ("tall", "causal"):  # (test_gpu_paged_scores.py: unsplit and in splits)
                assert {c[7] for c in mine if is_one(c[6])} == set(forms.SCORES), (form, name)
        assert {c[5] > 1 for c in mine} == {False, True}


def test_forms_of_steep_slopes():
    calls, want = [], []
    for form, news, lens, H, Hk, splits in steep.SHAPES:
        for mask in steep.MASKS:
            for d in steep.DIMS:
                for kind in ("slopes", "both"):
                    calls.append(forms.arguments(news, lens, H, Hk, d, splits, mask, kind))
                    want.append([form, KINDS[kind]])
    assert launched(calls) == want

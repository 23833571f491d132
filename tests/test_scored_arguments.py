"""What the paged attention's other scores and masks, flash_tree_mask and flash_keep_paged refuse, and which kernels the calls of the GPU tests get.  No GPU needed:
every call here ends before anything is launched, or in a process in which nothing can be."""
import ctypes as C
import math
import os
import re
import subprocess
import sys
import tempfile

import pytest
import torch

import paged_launches
import test_gpu_paged_scores as scores
from test_paged_arguments import E_ALIGN, E_HEADDIM, E_INVAL, E_NODEVICE, ROOT, paged_params, tensors


@pytest.fixture(scope="module")
def paged(fa):
    from flash_attn_amd import paged

    paged._lib()
    return paged


def test_structs_match_the_header(paged):
    structs = {"flash_tree_params": paged.TreeParams, "flash_keep_params": paged.KeepParams}
    prog = '#include <stdio.h>\n#include <stddef.h>\n#include "flash_attn_mi355.h"\nint main(){printf("%d %d\\n", (int)FLASH_MAX_SOFTCAP, FLASH_MAX_TREE_TOKENS);'
    for name, s in structs.items():
        prog += f'printf("%zu\\n", sizeof({name}));' + "".join(f'printf("%zu\\n", offsetof({name}, {f[0]}));' for f in s._fields_)
    with tempfile.TemporaryDirectory() as td:
        src, exe = os.path.join(td, "t.c"), os.path.join(td, "t")
        open(src, "w").write(prog + "return 0;}\n")
        subprocess.check_call(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), src, "-o", exe])
        out = [int(x) for x in subprocess.check_output([exe]).split()]
    assert out[:2] == [paged.FLASH_MAX_SOFTCAP, paged.FLASH_MAX_TREE_TOKENS]
    out = out[2:]
    for s in structs.values():
        assert out.pop(0) == C.sizeof(s)
        for f in s._fields_:
            assert out.pop(0) == getattr(s, f[0]).offset, f
    assert not out


TREE = {"tree_mask": 0x110000, "tree_words": 1, "tree_stride": 1}


@pytest.mark.parametrize("code,kw", [
    (E_INVAL, {"softcap": -1.0}), (E_INVAL, {"softcap": math.nan}), (E_INVAL, {"softcap": math.inf}), (E_INVAL, {"softcap": 1001.0}), (E_ALIGN, {"alibi_slopes": 0x110002}),
    (E_ALIGN, {"prefix_lens": 0x110001}), (E_ALIGN, {**TREE, "tree_mask": 0x110004}), (E_INVAL, {**TREE, "tree_words": 0}), (E_INVAL, {**TREE, "tree_words": 5}),
    (E_INVAL, {**TREE, "tree_stride": -1}), (E_INVAL, {**TREE, "prefix_lens": 0x120000}), (E_INVAL, {**TREE, "window_right": 3}), (E_INVAL, {**TREE, "total_q": 65}),
    (E_INVAL, {**TREE, "total_q": 100, "max_seqlen_q": 65}), (E_INVAL, {**TREE, "window_left": 3}), (E_INVAL, {**TREE, "total_q": 40, "max_seqlen_q": 30, "window_left": 28})])
def test_forward_refuses(paged, code, kw):
    p = paged_params(paged, **kw)
    assert paged._lib().flash_forward_paged(C.byref(p), None) == code
    assert paged._lib().flash_forward_paged_resolve_splits(C.byref(p)) == code
    assert paged._lib().flash_forward_paged_workspace_bytes(C.byref(p), None, None) == code


def tree_params(paged, **kw):
    p = paged.TreeParams()
    paged._lib().flash_tree_params_init(C.byref(p))
    p.parents, p.cu_seqlens_q, p.seqlens_k, p.mask, p.positions, p.B, p.total_q, p.words, p.mask_stride = 0x1000, 0x2000, 0x3000, 0x4000, 0x5000, 2, 10, 2, 2
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("code,kw", [
    (E_INVAL, {"B": -1}), (E_INVAL, {"B": 2 ** 24}), (E_INVAL, {"total_q": -1}), (E_INVAL, {"total_q": 2 ** 25 + 1}), (E_INVAL, {"words": 0}), (E_INVAL, {"words": 5, "mask_stride": 5}),
    (E_INVAL, {"mask_stride": 1}), (E_INVAL, {"parents": None}), (E_INVAL, {"cu_seqlens_q": None}), (E_INVAL, {"mask": None}), (E_ALIGN, {"parents": 0x1002}),
    (E_ALIGN, {"cu_seqlens_q": 0x2001}), (E_ALIGN, {"seqlens_k": 0x3002}), (E_ALIGN, {"mask": 0x4004}), (E_ALIGN, {"positions": 0x5002}), (0, {"B": 0}), (0, {"total_q": 0, "mask": None})])
def test_tree_mask_refuses(paged, code, kw):
    assert paged._lib().flash_tree_mask(C.byref(tree_params(paged, **kw)), None) == code
    assert paged._lib().flash_tree_mask(None, None) == E_INVAL


def keep_params(paged, **kw):
    p = paged.KeepParams()
    paged._lib().flash_keep_params_init(C.byref(p))
    p.K_cache, p.V_cache, p.block_table, p.seqlens_k, p.cu_seqlens_q, p.path, p.accepted, p.seqlens_out = (0x100000 * i for i in range(1, 9))
    p.B, p.H_kv, p.d, p.layers, p.num_pages, p.page_size, p.max_pages, p.max_path = 2, 2, 64, 3, 100, 16, 50, 7
    p.kc_page, p.kc_head, p.kc_row = p.vc_page, p.vc_head, p.vc_row = 2048, 1024, 64
    p.kc_layer = p.vc_layer = 204800
    p.block_table_stride, p.path_stride = 50, 7
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("code,kw", [
    (E_INVAL, {"B": -1}), (E_INVAL, {"H_kv": 0}), (E_INVAL, {"d": 0}), (E_INVAL, {"d": 60}), (E_HEADDIM, {"d": 136}), (E_INVAL, {"layers": -1}), (E_INVAL, {"num_pages": -1}),
    (E_INVAL, {"page_size": 0}), (E_INVAL, {"page_size": 24}), (E_INVAL, {"max_pages": -1}), (E_INVAL, {"page_size": 2 ** 16, "max_pages": 2 ** 16}), (E_INVAL, {"max_path": -1}),
    (E_INVAL, {"kc_row": 68}), (E_INVAL, {"vc_page": -64}), (E_INVAL, {"kc_layer": 4}), (E_INVAL, {"vc_head": 2 ** 62}), (E_INVAL, {"block_table_stride": -1}), (E_INVAL, {"path_stride": -1}),
    (E_INVAL, {"K_cache": None}), (E_INVAL, {"V_cache": None}), (E_INVAL, {"V_cache": 0x100000}), (E_INVAL, {"block_table": None}), (E_INVAL, {"seqlens_k": None}),
    (E_INVAL, {"cu_seqlens_q": None}), (E_INVAL, {"path": None}), (E_INVAL, {"accepted": None}), (E_INVAL, {"seqlens_out": None}), (E_INVAL, {"seqlens_out": 0x400004}),
    (E_INVAL, {"seqlens_out": 0x500008}), (E_INVAL, {"seqlens_out": 0x6ffffc}), (E_INVAL, {"kc_page": 0}), (E_INVAL, {"kc_row": 0}), (E_INVAL, {"vc_head": 0}), (E_INVAL, {"vc_layer": 0}),
    (E_INVAL, {"B": 2 ** 20, "layers": 16}), (E_INVAL, {"H_kv": 2 ** 20, "B": 500, "layers": 1}), (E_ALIGN, {"K_cache": 0x100008}), (E_ALIGN, {"V_cache": 0x200002}),
    (E_ALIGN, {"block_table": 0x300002}), (E_ALIGN, {"seqlens_k": 0x400001}), (E_ALIGN, {"cu_seqlens_q": 0x500002}), (E_ALIGN, {"path": 0x600002}), (E_ALIGN, {"accepted": 0x700002}),
    (E_ALIGN, {"seqlens_out": 0x800002}), (0, {"B": 0}), (0, {"layers": 0, "K_cache": None})])
def test_keep_refuses(paged, code, kw):
    assert paged._lib().flash_keep_paged(C.byref(keep_params(paged, **kw)), None) == code
    assert paged._lib().flash_keep_paged(None, None) == E_INVAL


@pytest.mark.skipif(torch.cuda.is_available(), reason="would launch with these pointers")
def test_good_arguments_get_as_far_as_the_device(paged):
    L = paged._lib()
    for kw in ({"softcap": 1000.0}, {"alibi_slopes": 0x110000}, {"prefix_lens": 0x110000}, TREE, {**TREE, "window_left": 4, "softcap": 1e-3, "is_causal": 1}):
        assert L.flash_forward_paged(C.byref(paged_params(paged, **kw)), None) == E_NODEVICE
    for kw in ({}, {"seqlens_k": None, "positions": None}):
        assert L.flash_tree_mask(C.byref(tree_params(paged, **kw)), None) == E_NODEVICE
    for kw in ({}, {"layers": 1, "kc_layer": 0, "vc_layer": 0}, {"max_path": 0, "path": None}, {"num_pages": 0, "K_cache": None}):
        assert L.flash_keep_paged(C.byref(keep_params(paged, **kw)), None) == E_NODEVICE


def test_python_refuses(fa):
    """What the GPU is not needed for; the last of each: tensors that are not there."""
    q, kc, vc, table, lens, cu = args = tensors()
    for kw in ({"alibi_slopes": torch.ones(3)}, {"alibi_slopes": torch.ones(4, dtype=torch.float64)}, {"alibi_slopes": torch.ones(8)[::2]}, {"prefix_lens": torch.zeros(2)},
               {"prefix_lens": torch.zeros(3, dtype=torch.int32)}, {"tree_mask": torch.zeros((3, 1), dtype=torch.int32)}, {"tree_mask": torch.zeros((2, 1), dtype=torch.int64)},
               {"tree_mask": torch.zeros((3, 5), dtype=torch.int64)}, {"tree_mask": torch.zeros((3, 0), dtype=torch.int64)}, {"tree_mask": torch.zeros(3, dtype=torch.int64)},
               {"tree_mask": torch.zeros((3, 4), dtype=torch.int64)[:, ::2]}, {"alibi_slopes": torch.ones(4, requires_grad=True)}, {"softcap": 1.0}):
        with pytest.raises(ValueError):
            fa.flash_forward_paged(*args, **kw)
    parents = torch.zeros(3, dtype=torch.int32)
    for a, kw in (((parents.long(), cu, lens), {}), ((parents, cu.long(), lens), {}), ((parents, cu, lens[:1]), {}), ((parents[None], cu, lens), {}), ((torch.zeros(6, dtype=torch.int32)[::2], cu, lens), {}),
                  ((torch.zeros(300, dtype=torch.int32), cu, lens), {}), ((torch.zeros(300, dtype=torch.int32), cu, lens, 257), {}), ((parents, torch.zeros(0, dtype=torch.int32)), {}),
                  ((parents, cu, lens), {})):
        with pytest.raises(ValueError):
            fa.flash_tree_mask(*a, **kw)
    path, count = torch.zeros((2, 3), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    good = [kc, vc, table, lens, cu, path, count]
    for at, bad in ((0, kc[0]), (0, kc.float()), (0, kc[:7]), (1, vc.bfloat16()), (1, vc.repeat(1, 1, 1, 2)[..., ::2]), (2, table.long()), (2, table[:1]), (3, lens[:1]), (4, cu[:2]), (5, path[0]),
                    (5, path.long()), (5, path[:1]), (5, path.t().contiguous().t()), (6, count[:1]), (6, count.long()), (0, kc.clone().requires_grad_()), (0, kc)):
        mine = list(good)
        mine[at] = bad
        with pytest.raises(ValueError):
            fa.flash_keep_paged(*mine)
    with pytest.raises(ValueError):
        fa.flash_keep_paged(*good, out=torch.zeros(3, dtype=torch.int32))


def test_split_counts(fa):
    """A tree has no diagonal, a prefix takes the end off a window; the workspace goes by the same counts."""
    size = dict(max_seqlen_q=64, max_seqlen_k=4000)
    assert fa.paged_resolve_splits(1, 8, 8, 64, 64, 16, 300, causal=True, window=(63, -1), num_splits=128, **size) <= 3
    for kw in (dict(prefix=True), dict(tree_words=1)):
        S = fa.paged_resolve_splits(1, 8, 8, 64, 64, 16, 300, causal=True, window=(63, -1), num_splits=128, **size, **kw)
        assert S > 3 if "prefix" in kw else S <= 5
        assert fa.paged_workspace_bytes(1, 8, 8, 64, 64, 16, 300, causal=True, window=(63, -1), num_splits=128, **size, **kw) == (4 * 64 * 8 * S * 64, 4 * 64 * 8 * S)
    with pytest.raises(fa.FlashError):
        fa.paged_resolve_splits(1, 8, 8, 64, 65, 16, 300, tree_words=1)


_CHILD = """
import ctypes as C, json, re, sys
sys.path.insert(0, %r)
sys.modules["torch"] = None
rec = C.CDLL(%r, mode=C.RTLD_GLOBAL)
rec.recorder_name.restype = C.c_char_p
from flash_attn_amd import paged
L = paged._lib()
res = []
for call in json.load(sys.stdin):
    p = paged.PagedParams()
    L.flash_paged_params_init(C.byref(p))
    for name, value in call.items():
        setattr(p, name, value)
    for i, name in enumerate(("Q", "O", "K_cache", "V_cache", "LSE", "O_partial", "LSE_partial", "block_table", "seqlens_k", "cu_seqlens_q")):
        setattr(p, name, 0x100000 * (i + 1))
    p.q_head = p.o_head = p.kc_row = p.vc_row = p.d
    p.q_token = p.o_token = p.H * p.d
    p.kc_head = p.vc_head = p.page_size * p.d
    p.kc_page = p.vc_page = p.H_kv * p.page_size * p.d
    p.block_table_stride, p.softmax_scale = p.max_pages, 0.125
    rec.recorder_clear()
    assert L.flash_forward_paged(C.byref(p), None) == 0, call
    name = rec.recorder_name(0).decode()
    paired = "Li2ELb" in name and "mid" in name  # (template arguments: D, columns, stages, groups of waves, bf16, kind)
    res.append(["paired" if paired else re.search("scored_(few|mid|tall)_kernel", name).group(1), int(re.search("ELi(.)EEEv", name).group(1))])
json.dump(res, sys.stdout)
"""


def launched(calls):
    import json

    out = subprocess.run([sys.executable, "-c", _CHILD % (ROOT, paged_launches._recorder())], input=json.dumps(calls), capture_output=True, text=True, timeout=600)
    assert out.returncode == 0, out.stderr[-3000:]
    return json.loads(out.stdout)


def test_forms_of_the_gpu_tests():
    """The shapes of test_gpu_paged_scores.py reach the form that they are there for, and the calls the kernel of their kind."""
    calls, want = [], []
    for shapes, form, dims in ((scores.FEW, "few", (8, 40, 64, 80, 128)), (scores.MID, "mid", (40, 64, 80, 128)), (scores.PAIRED, "paired", (40, 64, 80, 128)), (scores.TALL[:1], "tall", (40, 64, 80, 128)), (scores.TALL[1:], "tall", (80, 128))):
        for news, lens, H, Hk, *splits in shapes:
            for d in dims:
                for kind, number in (("cap", 2), ("slopes", 3), ("both", 4), ("prefix", 1), ("cap prefix", 2)):
                    how, kw = scores.extras(kind, H, lens)
                    extra = {"softcap": how.get("softcap", 0.0)}
                    if "slopes" in kw:
                        extra["alibi_slopes"] = 0xc00000
                    if "prefix" in kw:
                        extra["prefix_lens"] = 0xd00000
                    calls.append(paged_launches.call(news, lens, H, Hk, d, max_seqlen_q=max(news), causal=True, num_splits=splits[0] if splits else 1, **extra))
                    want.append([form, number])
    for shapes, form, dims in ((scores.TREES_FEW, "few", (24, 64, 96, 128)), (scores.TREES_MID, "mid", (64, 80, 128)), (scores.TREES_PAIRED, "paired", (40, 64, 80, 128)), (scores.TREES_TALL[:1], "tall", (40, 64, 80, 128)),
                               (scores.TREES_TALL[1:], "tall", (80, 128))):
        for news, lens, H, Hk, *splits in shapes:
            for d in dims:
                words = -(-max(news) // 64)
                calls.append(paged_launches.call(news, lens, H, Hk, d, max_seqlen_q=max(news), num_splits=splits[0] if splits else 1, tree_mask=0xe00000, tree_words=words, tree_stride=words))
                want.append([form, 1])
    assert launched(calls) == want


@pytest.mark.parametrize("code,kw", [
    (E_INVAL, {"softcap": 0.9e-6}), (E_INVAL, {"softcap": 1e-40}), (E_INVAL, {"softcap": 1e-6, "softmax_scale": 1e33}), (E_INVAL, {"alibi_slopes": 0x110000, "softmax_scale": 1e-39}),
    (E_NODEVICE, {"softcap": 1e-6}), (E_NODEVICE, {"softcap": 1e-6, "alibi_slopes": 0x110000, "softmax_scale": 1e-39}), (E_NODEVICE, {"alibi_slopes": 0x110000, "softmax_scale": 1e-38}),
    (E_NODEVICE, {"softmax_scale": 1e-39})])
@pytest.mark.skipif(torch.cuda.is_available(), reason="would launch with these pointers")
def test_units_of_scores_are_finite(paged, code, kw):
    """A cap below FLASH_MIN_SOFTCAP, and units in which a product or a distance of 0 would be 0 times infinity, are refused."""
    assert paged.FLASH_MIN_SOFTCAP == 1e-6
    assert paged._lib().flash_forward_paged(C.byref(paged_params(paged, **kw)), None) == code

"""What flash_rotary, flash_append_paged and flash_forward_paged refuse, their split counts and workspace sizes, and the frequencies of rotary
positions.  No GPU needed: every call here ends before anything is launched."""
import ctypes as C
import math
import os
import subprocess
import sys
import tempfile

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
E_INVAL, E_HEADDIM, E_ALIGN, E_WORKSPACE, E_SPLITS, E_NODEVICE = -1, -2, -3, -4, -5, -7


@pytest.fixture(scope="module")
def paged(fa):
    from flash_attn_amd import paged

    paged._lib()
    return paged


def test_structs_match_the_header(paged):
    structs = {"flash_rotary_params": paged.RotaryParams, "flash_paged_params": paged.PagedParams}
    prog = '#include <stdio.h>\n#include <stddef.h>\n#include "flash_attn_mi355.h"\nint main(){'
    for name, s in structs.items():
        prog += f'printf("%zu\\n", sizeof({name}));' + "".join(f'printf("%zu\\n", offsetof({name}, {f[0]}));' for f in s._fields_)
    with tempfile.TemporaryDirectory() as td:
        src, exe = os.path.join(td, "t.c"), os.path.join(td, "t")
        open(src, "w").write(prog + "return 0;}\n")
        subprocess.check_call(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), src, "-o", exe])
        out = [int(x) for x in subprocess.check_output([exe]).split()]
    for s in structs.values():
        assert out.pop(0) == C.sizeof(s)
        for f in s._fields_:
            assert out.pop(0) == getattr(s, f[0]).offset, f
    assert not out


def rotary_params(paged, **kw):
    p = paged.RotaryParams()
    paged._lib().flash_rotary_params_init(C.byref(p))
    assert p.factor == 1.0
    p.X, p.Y, p.positions, p.inv_freq = 0x10000, 0x20000, 0x30000, 0x40000
    p.B, p.H, p.N, p.d, p.rot = 1, 2, 3, 64, 64
    p.x_batch, p.x_head, p.x_row = p.y_batch, p.y_head, p.y_row = 384, 192, 64
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("code,kw", [
    (E_INVAL, {"dtype": 3}), (E_INVAL, {"dtype": -1}), (E_INVAL, {"B": -1}), (E_INVAL, {"H": -1}), (E_INVAL, {"N": -1}), (E_INVAL, {"d": 0}),
    (E_INVAL, {"rot": 0}), (E_INVAL, {"rot": 3}), (E_INVAL, {"rot": 66}), (E_INVAL, {"d": 1000, "rot": 514}), (E_INVAL, {"factor": math.nan}),
    (E_INVAL, {"factor": math.inf}), (E_INVAL, {"X": None}), (E_INVAL, {"Y": None}), (E_INVAL, {"positions": None}), (E_INVAL, {"inv_freq": None}),
    (E_INVAL, {"x_row": -64}), (E_INVAL, {"y_head": -1}), (E_INVAL, {"positions_batch": -1}), (E_INVAL, {"B": 2 ** 30, "N": 2 ** 30}), (E_INVAL, {"B": 2, "N": 2 ** 24 + 1}), (E_INVAL, {"H": 2 ** 24 + 1}), (E_INVAL, {"H": 2 ** 30, "d": 2, "rot": 2}),
    (E_INVAL, {"Y": 0x10000, "y_row": 128}), (E_INVAL, {"y_row": 0}), (E_INVAL, {"y_head": 0}), (E_INVAL, {"B": 2, "y_batch": 0}),
    (E_INVAL, {"Y": 0x10000, "x_row": 0, "y_row": 0}), (E_INVAL, {"Y": 0x10000, "y_head": 64}),
    (E_ALIGN, {"X": 0x10001}), (E_ALIGN, {"Y": 0x20001}), (E_ALIGN, {"dtype": 2, "X": 0x10002}), (E_ALIGN, {"positions": 0x30002}),
    (E_ALIGN, {"positions": 0x30004, "positions_64": 1}), (E_ALIGN, {"inv_freq": 0x40002}), (0, {"B": 0}), (0, {"H": 0}), (0, {"N": 0, "X": None})])
def test_rotary_refuses(paged, code, kw):
    assert paged._lib().flash_rotary(C.byref(rotary_params(paged, **kw)), None) == code
    assert paged._lib().flash_rotary(None, None) == E_INVAL


def paged_params(paged, **kw):
    p = paged.PagedParams()
    paged._lib().flash_paged_params_init(C.byref(p))
    assert (p.window_left, p.window_right, p.factor) == (-1, -1, 1.0)
    p.dtype, p.B, p.H, p.H_kv, p.d, p.total_q, p.num_pages, p.page_size, p.max_pages = 0, 2, 8, 2, 64, 5, 100, 16, 50
    p.Q, p.O, p.K, p.V, p.K_cache, p.V_cache, p.LSE = 0x10000, 0x20000, 0x30000, 0x40000, 0x50000, 0x60000, 0x70000
    p.block_table, p.seqlens_k, p.cu_seqlens_q = 0x80000, 0x90000, 0xa0000
    p.q_token = p.o_token = 512
    p.k_token = p.v_token = 128
    p.q_head = p.o_head = p.k_head = p.v_head = 64
    p.kc_page, p.kc_head, p.kc_row = p.vc_page, p.vc_head, p.vc_row = 2048, 1024, 64
    p.block_table_stride, p.softmax_scale, p.num_splits = 50, 0.125, 1
    p.inv_freq, p.rot = 0xb0000, 64
    for k, v in kw.items():
        setattr(p, k, v)
    return p


BOTH = [
    (E_INVAL, {"dtype": 2}), (E_INVAL, {"dtype": -1}), (E_INVAL, {"B": -1}), (E_INVAL, {"H": 0}), (E_INVAL, {"H_kv": 0}), (E_INVAL, {"H": 7}),
    (E_INVAL, {"d": 0}), (E_INVAL, {"d": 60, "rot": 4}), (E_HEADDIM, {"d": 136}), (E_INVAL, {"total_q": -1}), (E_INVAL, {"num_pages": -1}),
    (E_INVAL, {"page_size": 0}), (E_INVAL, {"page_size": 24}), (E_INVAL, {"page_size": -16}), (E_INVAL, {"max_pages": -1}),
    (E_INVAL, {"page_size": 2 ** 16, "max_pages": 2 ** 16}), (E_INVAL, {"total_q": 2 ** 25, "H": 1024, "H_kv": 1024}), (E_INVAL, {"total_q": 2 ** 25 + 1}), (E_INVAL, {"B": 2 ** 25}), (E_INVAL, {"total_q": 1, "H": 2 ** 24 + 2}),
    (E_INVAL, {"block_table": None}), (E_INVAL, {"seqlens_k": None}), (E_INVAL, {"cu_seqlens_q": None}), (E_INVAL, {"K_cache": None}),
    (E_INVAL, {"V_cache": None}), (E_INVAL, {"block_table_stride": -1}), (E_INVAL, {"kc_row": 68}), (E_INVAL, {"vc_page": 2052}), (E_INVAL, {"vc_head": -64}),
    (E_INVAL, {"kc_row": 2 ** 27}), (E_INVAL, {"kc_page": 2 ** 31}), (E_INVAL, {"vc_page": 2 ** 33}), (E_INVAL, {"q_token": 516}), (E_INVAL, {"q_head": 4}), (E_INVAL, {"o_head": -64}), (E_INVAL, {"Q": None, "O": None, "K": None}),
    (E_INVAL, {"O": None}), (E_ALIGN, {"Q": 0x10008}), (E_ALIGN, {"O": 0x20002}), (E_ALIGN, {"K_cache": 0x50008}), (E_ALIGN, {"V_cache": 0x60004}),
    (E_ALIGN, {"block_table": 0x80002}), (E_ALIGN, {"seqlens_k": 0x90001}), (E_ALIGN, {"cu_seqlens_q": 0xa0002}), (0, {"B": 0}), (0, {"total_q": 0, "Q": None})]


@pytest.mark.parametrize("code,kw", BOTH)
def test_paged_calls_refuse(paged, code, kw):
    p = paged_params(paged, **kw)
    assert paged._lib().flash_forward_paged(C.byref(p), None) == code
    assert paged._lib().flash_append_paged(C.byref(p), None) == code


@pytest.mark.parametrize("code,kw", [
    (E_INVAL, {"softmax_scale": 0.0}), (E_INVAL, {"softmax_scale": -1.0}), (E_INVAL, {"softmax_scale": math.nan}), (E_INVAL, {"softmax_scale": math.inf}),
    (E_INVAL, {"LSE": None}), (E_INVAL, {"o_token": 0}), (E_INVAL, {"o_head": 0}), (E_ALIGN, {"LSE": 0x70002}), (E_SPLITS, {"num_splits": 129}), (E_WORKSPACE, {"num_splits": 4}),
    (E_WORKSPACE, {"num_splits": 4, "O_partial": 0x100000}), (E_ALIGN, {"num_splits": 4, "O_partial": 0x100008, "LSE_partial": 0x200000}),
    (E_ALIGN, {"num_splits": 4, "O_partial": 0x100000, "LSE_partial": 0x200002}), (E_INVAL, {"max_seqlen_q": -1}), (E_INVAL, {"max_seqlen_k": -1}),
    (E_INVAL, {"B": 2 ** 24, "total_q": 2 ** 24, "H": 100, "H_kv": 100})])
def test_forward_refuses(paged, code, kw):
    assert paged._lib().flash_forward_paged(C.byref(paged_params(paged, **kw)), None) == code
    assert paged._lib().flash_forward_paged(None, None) == E_INVAL


@pytest.mark.parametrize("code,kw", [
    (E_INVAL, {"rot": 0}), (E_INVAL, {"rot": 66}), (E_INVAL, {"rot": 7}), (E_INVAL, {"factor": math.nan}), (E_ALIGN, {"inv_freq": 0xb0002}),
    (E_ALIGN, {"positions": 0x11002}), (E_ALIGN, {"positions": 0x11004, "positions_64": 1}), (E_INVAL, {"K": None}), (E_INVAL, {"V": None}),
    (E_INVAL, {"k_token": 132}), (E_INVAL, {"kc_page": 0}), (E_INVAL, {"kc_row": 0}), (E_INVAL, {"vc_head": 0}), (E_INVAL, {"o_token": 0}), (E_INVAL, {"v_head": 4}), (E_ALIGN, {"K": 0x30008}), (E_ALIGN, {"V": 0x40008}), (E_INVAL, {"O": 0x10000, "o_token": 1024})])
def test_append_refuses(paged, code, kw):
    assert paged._lib().flash_append_paged(C.byref(paged_params(paged, **kw)), None) == code
    assert paged._lib().flash_append_paged(None, None) == E_INVAL


@pytest.mark.skipif(torch.cuda.is_available(), reason="would launch with these pointers")
def test_good_arguments_get_as_far_as_the_device(paged):
    L = paged._lib()
    assert L.flash_rotary(C.byref(rotary_params(paged)), None) == E_NODEVICE
    for p in (paged_params(paged), paged_params(paged, Q=0x10000, O=0x10000), paged_params(paged, inv_freq=None, rot=0, Q=None, O=None)):
        assert L.flash_append_paged(C.byref(p), None) == E_NODEVICE
    assert L.flash_forward_paged(C.byref(paged_params(paged)), None) == E_NODEVICE


def test_split_counts_and_workspace(fa):
    """Counts are within the limits, give every split a tile, and the workspace is theirs; without keys or tokens there is one."""
    for B, H, Hk, d, T, page, pages, mq, mk in ((1, 32, 8, 128, 1, 16, 400, 1, 5003), (64, 32, 8, 128, 64, 64, 300, 1, 16385), (1, 8, 8, 64, 1, 16, 8, 1, 100),
                                                (1, 32, 8, 128, 512, 16, 1100, 512, 16896), (4, 32, 4, 128, 9000, 32, 128, 4096, 4096), (2, 4, 2, 64, 0, 16, 10, 0, 0),
                                                (1, 1, 1, 8, 1, 16, 0, 1, 0), (1, 1, 1, 8, 1, 16, 2 ** 26, 1, 0)):
        for window in ((-1, -1), (100, -1), (2 ** 31 - 1, 2 ** 31 - 1)):
            for asked in (0, 1, 2, 7, 128):
                kw = dict(max_seqlen_q=mq, max_seqlen_k=mk, causal=True, window=window, num_splits=asked)
                S = fa.paged_resolve_splits(B, H, Hk, d, T, page, pages, **kw)
                keys = min(mk or page * pages, page * pages)
                assert 1 <= S <= 128 and (S == 1 or S <= -(-keys // 64)) and (asked == 0 or S <= asked)
                assert fa.paged_workspace_bytes(B, H, Hk, d, T, page, pages, **kw) == ((0, 0) if S == 1 else (4 * T * H * S * d, 4 * T * H * S))
                if T == 0 or pages == 0:
                    assert S == 1
    with pytest.raises(fa.FlashError):
        fa.paged_resolve_splits(1, 8, 3, 64, 1, 16, 4)
    with pytest.raises(fa.FlashError):
        fa.paged_workspace_bytes(1, 8, 2, 64, 1, 16, 4, num_splits=129)
    # what does not fit a C int is as good as what does
    huge = dict(max_seqlen_q=2 ** 40, max_seqlen_k=2 ** 40, window=(2 ** 32 + 5, -2 ** 32 + 5))
    assert fa.paged_resolve_splits(1, 8, 1, 64, 1, 16, 100, num_splits=7, **huge) == fa.paged_resolve_splits(1, 8, 1, 64, 1, 16, 100, num_splits=7)
    with pytest.raises(fa.FlashError):
        fa.paged_resolve_splits(1, 8, 1, 64, 1, 16, 100, num_splits=2 ** 32 + 1)
    # a window bounds the keys that there are to cut
    assert fa.paged_resolve_splits(1, 8, 1, 64, 1, 16, 10000, max_seqlen_q=1, causal=True, window=(63, -1), num_splits=128) <= 3


def tensors(T=3, H=4, Hk=2, d=64, page=16, B=2, dtype=torch.float16):
    return [torch.zeros((T, H, d), dtype=dtype), torch.zeros((8, Hk, page, d), dtype=dtype), torch.zeros((8, Hk, page, d), dtype=dtype),
            torch.zeros((B, 4), dtype=torch.int32), torch.zeros(B, dtype=torch.int32), torch.zeros(B + 1, dtype=torch.int32)]


@pytest.mark.parametrize("at,change", [
    (0, lambda t: t[0]), (0, lambda t: t.float()), (0, lambda t: t.bfloat16()), (0, lambda t: t[:, :3]), (0, lambda t: t[..., :32]),
    (0, lambda t: t.repeat(1, 1, 2)[..., ::2]), (1, lambda t: t[0]), (1, lambda t: t.float()), (1, lambda t: t[:7]), (2, lambda t: t.bfloat16()),
    (2, lambda t: t.repeat(1, 1, 1, 2)[..., ::2]), (3, lambda t: t.long()), (3, lambda t: t[0]), (3, lambda t: t[:1]), (3, lambda t: t.t().contiguous().t()),
    (4, lambda t: t.long()), (4, lambda t: t[:1]), (5, lambda t: t[:2]), (5, lambda t: t.float()), (5, lambda t: t.repeat(2)[::2]), (0, lambda t: t)])
def test_python_refuses(fa, at, change):
    """The last one: tensors that are not on the GPU."""
    args = tensors()
    args[at] = change(args[at])
    with pytest.raises(ValueError):
        fa.flash_forward_paged(*args)
    if at:
        with pytest.raises(ValueError):
            fa.flash_append_paged(torch.zeros((3, 2, 64), dtype=torch.float16), torch.zeros((3, 2, 64), dtype=torch.float16), *args[1:])


def test_python_append_refuses(fa):
    q, kc, vc, table, lens, cu = tensors()
    k, f = torch.zeros((3, 2, 64), dtype=torch.float16), torch.ones(32)
    cache = (kc, vc, table, lens, cu)
    for args, kw in (((k, k[:2]), {}), ((k[:, :1], k), {}), ((k, k.float()), {}), ((k, k), {"q": q}), ((k, k), {"out": q, "inv_freq": f}), ((k, k), {"positions": lens}),
                     ((k, k), {"q": q, "inv_freq": f.double()}), ((k, k), {"q": q, "inv_freq": torch.ones(33)}), ((k, k), {"q": q, "inv_freq": torch.ones(0)}),
                     ((k, k), {"inv_freq": f, "positions": torch.zeros(3)}), ((k, k), {"inv_freq": f, "positions": torch.zeros(2, dtype=torch.int64)}), ((k[0], k), {})):
        with pytest.raises(ValueError):
            fa.flash_append_paged(*args, *cache, **kw)


def test_python_rotary_refuses(fa):
    x, n, f = torch.zeros((1, 2, 3, 16)), torch.arange(3), torch.ones(8)
    for args in ((x[0, 0], n, f), (x.double(), n, f), (x.transpose(2, 3), n, f), (x, n.float(), f), (x, n[:2], f), (x, torch.arange(6)[::2], f), (x, n, f.double()),
                 (x, n, torch.ones(9)), (x, n, torch.ones(0)), (x, n, f[None]), (x, n, f)):
        with pytest.raises(ValueError):
            fa.flash_rotary(*args)
    with pytest.raises(ValueError):
        fa.flash_rotary(x.requires_grad_(), n, f, out=torch.zeros((1, 2, 3, 16)))


def test_gradients_that_nobody_works_out(fa):
    x, n, f = torch.zeros((1, 2, 3, 16)), torch.arange(3), torch.ones(8, requires_grad=True)
    for y in (x, x.clone().requires_grad_()):
        with pytest.raises(ValueError, match="inv_freq gets no gradient"):
            fa.flash_rotary(y, n, f)
    with pytest.raises(ValueError, match="out must not"):
        fa.flash_rotary(x, n, f.detach(), out=torch.zeros((1, 2, 3, 16), requires_grad=True))


def test_sizes_past_a_c_int(fa):
    good = [1, 8, 8, 64, 1, 16, 100]
    fa.paged_resolve_splits(*good)
    for i in range(len(good)):
        with pytest.raises(ValueError, match="too large"):
            fa.paged_resolve_splits(*[2 ** 32 + v if k == i else v for k, v in enumerate(good)])
        with pytest.raises(ValueError, match="too large"):
            fa.paged_workspace_bytes(*[2 ** 32 + v if k == i else v for k, v in enumerate(good)])


def test_frequencies(fa):
    """Each scaling against its formula, in 64 bits."""
    L, s = 4096, 8.0
    plain = [10000.0 ** (-2 * i / 64) for i in range(32)]
    ntk = [(10000.0 * s ** (64 / 62)) ** (-2 * i / 64) for i in range(32)]
    yarn = []
    for w in plain:
        r = L * w / (2 * math.pi)
        keep = min(1.0, max(0.0, (r - 1) / 31))
        yarn.append(w * keep + w / s * (1 - keep))
    for kw, want, factor in (({}, plain, 1.0), ({"scaling": "linear", "stretch": s}, [w / s for w in plain], 1.0), ({"scaling": "ntk", "stretch": s}, ntk, 1.0),
                             ({"scaling": "yarn", "stretch": s, "original_length": L}, yarn, 0.1 * math.log(s) + 1)):
        f, m = fa.rotary_frequencies(64, **kw)
        assert f.dtype == torch.float32 and f.shape == (32,) and abs(m - factor) < 1e-12
        assert all(abs(float(a) - b) <= 2.0 ** -24 * b * 1.01 for a, b in zip(f, want))
    assert abs(ntk[-1] * s - plain[-1]) < 1e-12 and ntk[0] == plain[0]
    for kw in ({"scaling": "yarn"}, {"scaling": "other"}, {"stretch": 0.0}, {"base": -1.0}, {"scaling": "yarn", "original_length": 10, "beta_fast": 1.0}):
        with pytest.raises(ValueError):
            fa.rotary_frequencies(64, **kw)
    for rot in (0, 3, -2):
        with pytest.raises(ValueError):
            fa.rotary_frequencies(rot)


def test_host_side_under_asan_and_ubsan():
    """This file against a build of the library whose host code is instrumented, in a child process."""
    if "FLASH_PAGED_UNDER_ASAN" in os.environ:
        pytest.skip("this is the child")
    subprocess.check_call(["make", "-s", "-C", os.path.join(ROOT, "flash_attn_amd", "csrc"), "asan"])
    clang = "/opt/rocm/lib/llvm/bin/clang"
    if not os.path.exists(clang):
        pytest.skip("no clang to ask for its sanitizer runtime")
    rt = subprocess.check_output([clang, "-print-file-name=libclang_rt.asan-x86_64.so"], text=True).strip()
    if not os.path.isabs(rt) or not os.path.exists(rt):
        pytest.skip("clang has no shared AddressSanitizer runtime here")
    env = dict(os.environ, FLASH_PAGED_UNDER_ASAN="1")
    env["LD_PRELOAD"] = rt + (":" + env["LD_PRELOAD"] if env.get("LD_PRELOAD") else "")
    env["ASAN_OPTIONS"] = "detect_leaks=0:exitcode=99"
    env["UBSAN_OPTIONS"] = "print_stacktrace=1:halt_on_error=1"
    runner = ("import sys; sys.path.insert(0, %r); sys.path.insert(0, %r)\n"
              "from flash_attn_amd import binding\n"
              "binding._LIB_PATH = %r\n"
              "binding.lib(); maps = open('/proc/self/maps').read()\n"
              "assert 'libflash_attn_mi355_asan.so' in maps and 'libclang_rt.asan' in maps, 'sanitizer build not loaded'\n"
              "import pytest\n"
              "sys.exit(pytest.main(['-x', '-q', '-p', 'no:cacheprovider', %r]))\n"
              % (ROOT, os.path.join(ROOT, "tests"), os.path.join(ROOT, "flash_attn_amd", "lib", "libflash_attn_mi355_asan.so"), os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", runner], env=env, capture_output=True, text=True, timeout=900, cwd=ROOT)
    assert r.returncode == 0, (r.stdout[-3000:], r.stderr[-3000:])
    assert "passed" in r.stdout and "ERROR: AddressSanitizer" not in r.stderr and "runtime error" not in r.stderr

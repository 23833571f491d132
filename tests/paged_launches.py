"""What flash_forward_paged would launch, seen without a GPU: record() runs calls of the C ABI in a child process in which tests/paged_recorder.cpp
stands in for the HIP runtime's launch entry points."""
import ctypes as C
import functools
import json
import os
import re
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


@functools.lru_cache(maxsize=None)
def _recorder():
    so = os.path.join(tempfile.mkdtemp(prefix="paged_recorder_"), "recorder.so")
    subprocess.check_call(["/opt/rocm/bin/hipcc", "-x", "hip", "--offload-host-only", "--offload-arch=gfx950", "-std=c++17", "-O1", "-shared", "-fPIC",
                           "-fvisibility=hidden", "-I", os.path.join(ROOT, "flash_attn_amd", "csrc"), os.path.join(HERE, "paged_recorder.cpp"), "-o", so])
    return so


def call(news, lens, H, Hk, d, page=16, dtype="fp16", first=0, behind=0, width=None, **kw):
    """The call that flash_forward_paged makes of a paged_reference.Batch of these arguments, for record()."""
    need = [-(-n // page) for n in lens]
    c = dict(dtype=int(dtype == "bf16"), B=len(news), H=H, H_kv=Hk, d=d, total_q=first + sum(news) + behind, num_pages=sum(need) + 2, page_size=page,
             max_pages=width or max(need + [1]), is_causal=int(kw.pop("causal", False)), num_splits=kw.pop("num_splits", 0))
    c["window_left"], c["window_right"] = kw.pop("window", (-1, -1))
    return dict(c, **kw)


def record(calls):
    """Per call a dict: form ("tall" or "few"), columns (that the tall form works on), groups, direct, ordered, pieces, splits."""
    out = subprocess.run([sys.executable, os.path.abspath(__file__), _recorder()], input=json.dumps(calls), capture_output=True, text=True, timeout=600)
    assert out.returncode == 0, out.stderr[-3000:]
    return json.loads(out.stdout)


def _child(so):
    sys.path.insert(0, ROOT)
    sys.modules["torch"] = None  # (the binding loads torch's HIP runtime first where there is one)
    rec = C.CDLL(so, mode=C.RTLD_GLOBAL)
    rec.recorder_name.restype, rec.recorder_groups.restype = C.c_char_p, C.c_longlong
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
        rc = L.flash_forward_paged(C.byref(p), None)
        assert rc == 0 and rec.recorder_count() >= 1, (rc, call)
        name = rec.recorder_name(0).decode()
        m = re.search(r"paged_(few|tall)_kernelILi\d+E(?:Li(\d+)E)?", name)
        order = [rec.recorder_order(0, i) for i in range(4)]
        res.append(dict(form=m.group(1), columns=int(m.group(2) or 0), groups=rec.recorder_groups(0), direct=order[0], ordered=order[1], pieces=order[2],
                        splits=order[3]))
    json.dump(res, sys.stdout)


if __name__ == "__main__":
    _child(sys.argv[1])

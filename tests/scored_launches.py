"""What flash_forward_paged with other scores would launch, seen without a GPU: record() runs calls of the C ABI (paged_launches.call) in a child process in which
tests/scored_recorder.cpp stands in for the HIP runtime's launch entry points."""
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
    so = os.path.join(tempfile.mkdtemp(prefix="scored_recorder_"), "recorder.so")
    subprocess.check_call(["/opt/rocm/bin/hipcc", "-x", "hip", "--offload-host-only", "--offload-arch=gfx950", "-std=c++17", "-O1", "-shared", "-fPIC",
                           "-fvisibility=hidden", "-I", os.path.join(ROOT, "flash_attn_amd", "csrc"), os.path.join(HERE, "scored_recorder.cpp"), "-o", so])
    return so


def record(calls):
    """Per call a dict: form ("few", "mid", "paired" or "tall"), groups, direct, ordered, pieces, splits."""
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
        name = rec.recorder_name().decode()
        assert rc == 0 and name, (rc, call)
        form = re.search("scored_(few|mid|tall)_kernel", name).group(1)
        if form == "mid" and re.search("Li2ELb[01]", name):  # (template arguments: D, columns, stages, groups of waves, bf16, kind)
            form = "paired"
        res.append(dict(zip(("direct", "ordered", "pieces", "splits"), (rec.recorder_order(i) for i in range(4))), form=form, groups=rec.recorder_groups()))
    json.dump(res, sys.stdout)


if __name__ == "__main__":
    _child(sys.argv[1])

"""What a wave of the paged attention goes by when it clears rows of V past a sequence's end, checked on the host (tests/clear_past_test.cpp): no result is
sure to show that two waves got in each other's way.  No GPU needed."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "flash_attn_amd", "csrc")


def test_rows_past_the_end_are_seen_while_another_wave_clears_them(tmp_path):
    exe = str(tmp_path / "clear_past_test")
    subprocess.check_call(["/opt/rocm/bin/hipcc", "-x", "hip", "--offload-host-only", "--offload-arch=gfx950", "-std=c++17", "-O1",
                           "-I", CSRC, os.path.join(HERE, "clear_past_test.cpp"), "-o", exe])
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr

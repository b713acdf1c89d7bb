"""The compiled 256 x 256 GEMM kernels leave the registers of their LDS reads in flight alone (tools/check_async_frags.py over hipcc's listing)."""
import concurrent.futures
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"


def run(path):
    return subprocess.run([sys.executable, os.path.join(ROOT, "tools", "check_async_frags.py"), str(path), "kern"], capture_output=True, text=True)


def test_reads_are_followed_along_the_branches(tmp_path):
    head, tail = "kern: ; @kern\n", "\ts_endpgm\n\t.end_amdhsa_kernel\n"
    #  a loop laid out behind the code that follows it: the wait is on the way there, though not in front of it in the text
    far = "\ts_branch .LBB0_2\n.LBB0_1:\n\tv_mov_b32 v2, v0\n%s.LBB0_2:\n\tds_read_b128 v[2:5], v9\n%s\ts_cbranch_scc0 .LBB0_2\n\ts_branch .LBB0_1\n\t.end_amdhsa_kernel\n"
    for text, bad in ((head + "\tds_read_b128 v[2:5], v9\n\ts_waitcnt lgkmcnt(0)\n\tv_mov_b32 v2, v0\n" + tail, False),
                      (head + "\tds_read_b128 v[2:5], v9\n\tv_mov_b32 v2, v0\n\ts_waitcnt lgkmcnt(0)\n" + tail, True),
                      (head + far % ("\ts_endpgm\n", "\ts_waitcnt lgkmcnt(0)\n"), False), (head + far % ("\ts_endpgm\n", ""), True)):
        f = tmp_path / "x.s"
        f.write_text(text)
        r = run(f)
        assert r.returncode == int(bad), r.stdout


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no compiler")
def test_wide_gemm_kernels(tmp_path):
    from more4d_amd.build import CSRC, FLAGS

    def listing(name):
        out = tmp_path / (name + ".s")
        subprocess.run([HIPCC, *FLAGS, "-S", "--cuda-device-only", "-c", os.path.join(CSRC, name + ".hip"), "-o", str(out)], check=True, capture_output=True)
        r = subprocess.run([sys.executable, os.path.join(ROOT, "tools", "check_async_frags.py"), str(out), "gemm_bt256w"], capture_output=True, text=True)
        return name, r.returncode, r.stdout[-2000:]

    with concurrent.futures.ThreadPoolExecutor(5) as ex:
        for name, rc, text in ex.map(listing, ("gemm_wide_store", "gemm_wide_resid", "gemm_wide_gelu", "gemm_wide_f32", "gemm_wide_adapters")):
            assert rc == 0 and "fragment reads checked" in text, (name, text)

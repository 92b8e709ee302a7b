"""packed_wave_kernel waits for its sequences' lengths, which come by LDS-DMA, by the number of
loads asked for behind them: the wait must allow no more than there are. On the gfx950 assembly,
CPU only."""
import os
import re
import shutil
import subprocess
import tempfile

import pytest

from tests.test_asm_waits import CSRC, ROOT


def lengths_waits(text):
    """(loads behind the lengths, loads that the wait allows) of each wait up to their first read."""
    found = []
    for body in re.split(r"^_ZN", text, flags=re.M):
        if "packed_wave_kernel" not in body.split(":", 1)[0] or not re.search(r"ELb1EEEv", body.split(":", 1)[0]):
            continue
        behind = None
        for line in body.splitlines():
            op = line.strip().split(" ")[0].split("\t")[0]
            if op == "global_load_lds_dword":
                behind = 0
            elif behind is not None and op.startswith(("global_load", "global_store", "buffer_")):
                behind += 1
            elif behind is not None and op == "ds_read_b32":
                break
            elif behind is not None and op == "s_waitcnt" and "vmcnt" in line:
                found.append((behind, int(re.search(r"vmcnt\((\d+)\)", line).group(1))))
    return found


@pytest.mark.skipif(shutil.which("hipcc") is None, reason="hipcc not installed")
def test_lengths_have_landed():
    with tempfile.TemporaryDirectory() as tmp:
        out = os.path.join(tmp, "t.s")
        subprocess.run(["hipcc", "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature",
                        "-Xclang", "-packed-fp32-ops", f"-I{os.path.join(ROOT, 'include')}", "--cuda-device-only",
                        "-S", os.path.join(CSRC, "packed_attention.hip"), "-o", out], check=True,
                       stderr=subprocess.DEVNULL, timeout=600)
        found = lengths_waits(open(out).read())
    assert len(found) >= 8, found  # two types, two head sizes, keys shared or not: one or two each
    assert all(allowed <= behind for behind, allowed in found), found


def test_the_check_finds_a_wait_that_allows_too_much():
    name = "_ZN3tpp18packed_wave_kernelIDF16bLi64ELi1ELb1EEEvNS_10PackedArgsEi:\n"
    body = "\tglobal_load_lds_dword v[6:7], off\n\tglobal_load_lds_dword v[6:7], off\n\tglobal_load_dwordx4 v[66:69], v[6:7], off\n"
    assert lengths_waits(name + body + "\ts_waitcnt vmcnt(1)\n\tds_read_b32 v8, v7\n") == [(1, 1)]
    assert lengths_waits(name + body + "\ts_waitcnt vmcnt(2)\n\tds_read_b32 v8, v7\n") == [(1, 2)]

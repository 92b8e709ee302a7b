"""The waits of the inline-asm LDS reads in tree_attention.hip, checked on its
gfx950 assembly as test_asm_waits.py does for the other sources. CPU only."""
import os
import shutil
import subprocess
import tempfile

import pytest

from tests.test_asm_waits import CSRC, ROOT, scan


@pytest.mark.skipif(shutil.which("hipcc") is None, reason="hipcc not installed")
def test_no_access_to_asm_loaded_registers_before_their_wait():
    src = os.path.join(CSRC, "tree_attention.hip")
    with tempfile.TemporaryDirectory() as tmp:
        out = os.path.join(tmp, "t.s")
        subprocess.run(["hipcc", "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature",
                        "-Xclang", "-packed-fp32-ops", f"-I{os.path.join(ROOT, 'include')}",
                        "--cuda-device-only", "-S", src, "-o", out], check=True, stderr=subprocess.DEVNULL,
                       timeout=600)
        text = open(out).read()
    loads, bad = scan(text)
    assert loads > 0 and not bad, "registers touched before their wait:\n" + "\n".join(bad[:10])

"""The attention kernels compiled for gfx950 (here, without a GPU): waits for memory are the compiler's own, and none needs scratch memory."""
import os
import re
import subprocess

import pytest

from fusedkernellibrary_amd import build

pytestmark = pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="no hipcc")


@pytest.mark.parametrize("name", ["tree_attention_64", "merge", "rows"])
def test_no_wait_counts_on_what_the_compiler_makes_of_the_loads(tmp_path, name):
    """No load and no wait is written by hand: one that counted the loads behind it would be short if two of them were merged."""
    out = tmp_path / "kernels.s"
    r = subprocess.run([build.HIPCC, *[f for f in build.HIP_FLAGS if f != "-fPIC"], "--offload-device-only", "-I", build.INCLUDE, "-Rpass-analysis=kernel-resource-usage", "-S",
                        os.path.join(build.CSRC, "attention", name + ".hip"), "-o", str(out)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    assert not [line for line in r.stderr.splitlines() if "warning" in line and ("asm" in line or "reserved" in line)]
    scratch = re.findall(r"ScratchSize \[bytes/lane\]: (\d+)", r.stderr)
    assert scratch and set(scratch) == {"0"}
    by_hand = re.findall(r";#?APP\n(.*?);#?NO_APP", out.read_text(), re.S) + re.findall(r"#ASMSTART\n(.*?)#ASMEND", out.read_text(), re.S)
    assert not [text for text in by_hand if re.search(r"s_waitcnt|load|store|ds_|m0", text)]

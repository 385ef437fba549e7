"""The kernels of a step around attention, and of shaped attention, compiled for gfx950 (here, without a GPU)."""
import os
import re
import subprocess

import pytest

from fusedkernellibrary_amd import build

pytestmark = pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="no hipcc")


@pytest.mark.parametrize("name", ["step_tables", "verify", "keep", "rows_axes", "shaped_attention_64", "shaped_attention_256"])
def test_what_the_kernels_are_compiled_to(tmp_path, name):
    """No scratch memory, no load and no wait by hand, and no vector shift of 64 bits whose amount is in the last register that a wave has
    (registers are dealt out by eights): such shifts have gone wrong now and then."""
    out = tmp_path / "kernels.s"
    r = subprocess.run([build.HIPCC, *[f for f in build.HIP_FLAGS if f != "-fPIC"], "--offload-device-only", "-I", build.INCLUDE, "-Rpass-analysis=kernel-resource-usage", "-S",
                        os.path.join(build.CSRC, "attention", name + ".hip"), "-o", str(out)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    scratch = re.findall(r"ScratchSize \[bytes/lane\]: (\d+)", r.stderr)
    assert scratch and set(scratch) == {"0"}
    text = out.read_text()
    by_hand = re.findall(r";#?APP\n(.*?);#?NO_APP", text, re.S) + re.findall(r"#ASMSTART\n(.*?)#ASMEND", text, re.S)
    assert not [t for t in by_hand if re.search(r"s_waitcnt|load|store|ds_|m0", t)]
    kernels = text.split(".amdhsa_next_free_vgpr ")
    assert len(kernels) > 1
    for body, behind in zip(kernels, kernels[1:]):
        last = (int(behind.split()[0]) + 7) // 8 * 8 - 1
        amounts = re.findall(r"v_(?:lshlrev_b64|lshrrev_b64|ashrrev_i64)\S* v\[\d+:\d+\], v(\d+),", body)
        assert str(last) not in amounts

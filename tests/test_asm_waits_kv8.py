"""The waits round inline asm in the 8-bit cache's kernels, on the CPU."""
import shutil
import subprocess

import pytest

import build as B
from test_asm_waits import short_waits


@pytest.mark.parametrize("source", ["dip_kv8", "dip_kv8_attn"])
def test_asm_results_wait_for_their_readers(source, tmp_path):
    if shutil.which(B.HIPCC) is None:
        pytest.skip("hipcc not available")
    out = tmp_path / "kernels.s"
    subprocess.run([B.HIPCC, *B.COMMON, *B.EXTRA.get(source, []), "--cuda-device-only", "-S",
                    str(B.CSRC / f"{source}.hip"), "-o", str(out)],
                   check=True, capture_output=True, text=True, timeout=600)
    lines = out.read_text().splitlines()
    assert any("v_permlane16_swap" in l for l in lines)
    assert not short_waits(lines)

"""What the 4-bit cache's kernels decide from a position, on the CPU."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
CSRC = ROOT / "dynamic-input-pruning_amd" / "csrc"


def test_rows_outside_the_cache(tmp_path):
    import build as B
    if shutil.which(B.HIPCC) is None:
        pytest.skip("hipcc not available")
    exe = tmp_path / "rows"
    subprocess.run([B.HIPCC, "-x", "hip", "--offload-host-only", "-O2", "-std=c++17", f"-I{CSRC}",
                    str(Path(__file__).resolve().parent / "kv4_rows_in_cache.cpp"), "-o", str(exe)],
                   check=True, capture_output=True, text=True, timeout=240)
    p = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert p.returncode == 0, p.stdout

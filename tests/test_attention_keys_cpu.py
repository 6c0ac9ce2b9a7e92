"""What the attention kernels are given, on the host: the tiles of keys that a block of rows goes through
(csrc/attention_keys.h) and the launches of a call (csrc/attention_groups.h)."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
@pytest.mark.parametrize("name", ["keys", "groups"])
def test_ranges(name, tmp_path):
    exe = tmp_path / f"attention_{name}_check"
    cmd = ["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
           "-I", str(ROOT / "strata-rs_b200" / "csrc"), str(ROOT / "tests" / f"attention_{name}_check.cpp"), "-o", str(exe)]
    subprocess.run(cmd, check=True, capture_output=True, text=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr

"""Host code of the key/value cache (csrc/kv_index.hpp), compiled for the CPU and run."""
import os
import subprocess

import pytest

from conftest import ROOT


@pytest.mark.parametrize("program", ["kv_overlap", "kv_parts"])
def test_host_program(tmp_path, program):
    exe = str(tmp_path / program)
    r = subprocess.run(["/opt/rocm/bin/hipcc", "-std=c++17", "-O1", "-x", "hip", "--cuda-host-only", "-I", os.path.join(ROOT, "qwen3-tts-rs_amd", "csrc"),
                        os.path.join(ROOT, "tests", program + ".cpp"), "-o", exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr

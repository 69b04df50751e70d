"""Key/value cache handle (KVCache): refusals that need no GPU, and the reference the GPU tests compare with."""
import ctypes as C
import math
import os
import re
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
from conftest import ROOT  # noqa: E402
from kv_reference import TOP, held  # noqa: E402
from qwen3_tts_rs_amd import KVBatch, KVCache, QttsError, _lib  # noqa: E402


def test_structs_match_the_header():
    """ctypes and Rust structs: the header's fields in its order."""
    hdr = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "qtts.h")).read(), flags=re.S)
    rs = open(os.path.join(ROOT, "qwen-tts-hip-sys", "src", "lib.rs")).read()
    for cname, py in (("qtts_kv_config", _lib.KvConfig), ("qtts_kv_batch", _lib.KvBatch), ("qtts_kv_rows", _lib.KvRows),
                      ("qtts_kv_attend_args", _lib.KvAttendArgs)):
        body = re.search(r"typedef struct \{([^}]*)\}\s*" + cname + ";", hdr).group(1)
        fields = []
        for d in body.split(";"):
            d = d.strip()
            if d:
                fields += [x.strip(" *\n") for x in re.sub(r"^(const\s+)?\w+\b", "", d).split(",")]
        assert [f for f, _ in py._fields_] == fields, cname
        assert re.findall(r"pub (\w+):", re.search(r"pub struct " + cname + r" \{(.*?)\n\}", rs, flags=re.S).group(1)) == fields, cname


def test_open_refuses_without_a_context_or_format():
    lib = _lib.load()
    out = C.c_void_p()
    assert lib.qtts_kv_open(None, C.byref(_lib.KvConfig(1, 1, 64, 1, 64, 0)), C.byref(out)) == -1
    for fn in (lib.qtts_kv_write, lib.qtts_kv_read, lib.qtts_kv_attend):
        assert fn(None, 0, None, None, None) == -1
    assert lib.qtts_kv_bytes(None) == 0
    lib.qtts_kv_close(None)
    with pytest.raises(QttsError, match="unknown format"):
        KVCache(pages=1, kv_heads=1, head_dim=64, format="fp4")


def test_batch_refusals():
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    table = torch.zeros(2, 3, dtype=torch.int32)
    KVBatch(i32(0, 1, 2), i32(4, 5), table, 2, 1, 5)
    with pytest.raises(QttsError, match="int32"):
        KVBatch(i32(0, 1, 2).long(), i32(4, 5), table, 2, 1, 5)
    with pytest.raises(QttsError, match="contiguous"):
        KVBatch(i32(0, 1, 2), i32(4, 5), table.t(), 2, 1, 5)
    with pytest.raises(QttsError, match="same number"):
        KVBatch(i32(0, 1), i32(4, 5), table, 2, 1, 5)
    with pytest.raises(QttsError, match="out of range"):
        KVBatch(i32(0, 1, 2), i32(4, 5), table, -1, 1, 5)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_the_held_values(fmt):
    """The reference itself: held values are within half a step of the block's grid, the largest element is never cut, and holding
    them again changes nothing."""
    rng = np.random.default_rng(5)
    x = torch.from_numpy(rng.standard_normal((50, 4, 64)) * np.exp(rng.standard_normal((50, 4, 1)) * 6)).float()
    x[0] = 0
    x[1, 0, :32] = TOP[fmt] * 2.0 ** -3  # exactly at the top
    x[2, 0, 3], x[2, 1, 40] = math.inf, math.nan
    y = held(x, fmt)
    assert torch.equal(held(y.float(), fmt)[3:], y[3:])
    assert torch.equal(y[0], torch.zeros(4, 64, dtype=torch.float64)) and torch.equal(y[1, 0, :32], x[1, 0, :32].double())
    assert y[2, 0, :32].isnan().all() and not y[2, 0, 32:].isnan().any() and y[2, 1, 32:].isnan().all() and not y[2, 1, :32].isnan().any()
    a = x.double().unflatten(-1, (2, 32)).abs().amax(-1, keepdim=True)[3:]
    err = (y - x.double()).unflatten(-1, (2, 32)).abs()[3:]
    # scale <= 2 a / top, half a step: 1/2 unit (int8), 2^-4 of the value or 2^-10 units (e4m3)
    step = a * 2 / TOP[fmt]
    bound = step / 2 if fmt == "int8" else torch.maximum(x.double().unflatten(-1, (2, 32)).abs()[3:] * 2.0 ** -4, step * 2.0 ** -10)
    assert (err <= bound).all()


def test_index_functions_stay_inside_their_buffers(tmp_path):
    """tests/kv_bounds.cpp: the kernels' own index functions on arrays that hold anything, run on the CPU."""
    import subprocess
    exe = str(tmp_path / "kv_bounds")
    r = subprocess.run(["/opt/rocm/bin/hipcc", "-std=c++17", "-O1", "-x", "hip", "--cuda-host-only", "-I", os.path.join(ROOT, "qwen3-tts-rs_amd", "csrc"),
                        os.path.join(ROOT, "tests", "kv_bounds.cpp"), "-o", exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr

"""Attention and rotary positions, what needs no GPU: index arithmetic of the masks, frequencies, refusals without a handle."""
import ctypes as C
import math
import os
import shutil
import subprocess

import numpy as np
import pytest

from sddmm_gpu_b200 import api

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_mask_arithmetic(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no compiler")
    exe = str(tmp_path / "attention_mask")
    build = subprocess.run([cxx, "-std=c++17", "-Wall", "-O1", "-I", os.path.join(ROOT, "sddmm_gpu_b200", "csrc"),
                            os.path.join(ROOT, "tests", "c_abi", "attention_mask.cpp"), "-o", exe], capture_output=True, text=True)
    assert build.returncode == 0, build.stderr
    run = subprocess.run([exe], capture_output=True, text=True)
    assert run.returncode == 0 and "FAILED" not in run.stdout, run.stdout + run.stderr


@pytest.mark.parametrize("rot", [2, 6, 64, 128])
def test_frequencies(rot):
    f = 10000.0 ** (-np.arange(0, rot, 2) / rot)
    close = lambda a, b: np.testing.assert_allclose(a, b, rtol=1e-14)  # noqa: E731
    close(api.rotary_frequencies(rot), f)
    close(api.rotary_frequencies(rot, base=5e5), 5e5 ** (-np.arange(0, rot, 2) / rot))
    close(api.rotary_frequencies(rot, factor=4.0), f / 4)
    got = api.rotary_frequencies(rot, factor=8.0, original_len=4096, low_turns=1, high_turns=32)
    turns = 4096 * f / (2 * math.pi)
    close(got[turns >= 32], f[turns >= 32])
    close(got[turns <= 1], f[turns <= 1] / 8)
    kept = np.clip((turns - 1) / 31, 0, 1)
    close(got, f * kept + f * (1 - kept) / 8)


@pytest.mark.parametrize("bad", [dict(rot_dim=0), dict(rot_dim=3), dict(rot_dim=-2), dict(rot_dim=514), dict(base=0.0), dict(base=math.inf),
                                 dict(factor=0.0), dict(factor=math.nan), dict(original_len=-1.0), dict(original_len=10.0, low_turns=2.0, high_turns=2.0),
                                 dict(original_len=10.0, high_turns=math.inf)])
def test_frequencies_refused(bad):
    args = dict(rot_dim=8)
    args.update(bad)
    with pytest.raises(api.SddmmError) as e:
        api.rotary_frequencies(**args)
    assert e.value.status == api.INVALID_ARG


def test_null_handles_are_refused():
    L = api.lib()
    out, n = C.c_void_p(), C.c_int64()
    none = None
    assert L.sddmm_attention_plan(None, None, C.byref(out)) == api.INVALID_ARG
    assert L.sddmm_attention_workspace(None, 0, C.byref(n)) == api.INVALID_ARG
    assert L.sddmm_attention_forward(None, none, none, none, none, None, None, 0, 0) == api.INVALID_ARG
    assert L.sddmm_attention_backward(None, none, none, none, none, None, none, none, none, none, None, 0, 0) == api.INVALID_ARG
    assert L.sddmm_attention_destroy(None) == api.OK
    assert L.sddmm_attention_last_kernel(None) == b"none"
    assert L.sddmm_rotary(None, None, None, 1, 0) == api.INVALID_ARG
    assert L.sddmm_rotary_frequencies(8, 1e4, 1.0, 0.0, 1.0, 32.0, None) == api.INVALID_ARG

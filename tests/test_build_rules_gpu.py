"""The kernels around user-defined ops are compiled with the library's own switches."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

PROGRAM = """
import torch
from spla_amd import _lib
from spla_amd.kernels import _ptr, current_stream_ptr
x = torch.arange(1000, dtype=torch.float32, device="cuda")
out = torch.empty_like(x)
_lib.call("splahip_map_jit", 2, 1000, _ptr(x), _ptr(out), b"(T a) { return (a + 3.0f) * (a + 5.0f); }", current_stream_ptr())
assert torch.equal(out, (x + 3) * (x + 5))
print("map ok")
"""


def test_user_ops_are_compiled_without_packed_fp32_arithmetic(tmp_path):
    """the compiler library's own log of the run-time compilation names the switch"""
    log = tmp_path / "compiler.log"
    run = subprocess.run([sys.executable, "-c", PROGRAM], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=100,
                         env={**os.environ, "AMD_COMGR_EMIT_VERBOSE_LOGS": "1", "AMD_COMGR_REDIRECT_LOGS": str(log)})
    assert run.returncode == 0 and "map ok" in run.stdout, run.stdout + run.stderr
    compiled = [line for line in log.read_text().splitlines() if '"-ffp-contract=off"' in line]
    assert compiled and all('"-packed-fp32-ops"' in line for line in compiled), compiled

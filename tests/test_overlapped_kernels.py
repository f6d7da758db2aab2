"""Kernels that may start before the one in front of them in the stream has ended read nothing through
the read-only path, which is defined for data that nobody writes during the kernel's life."""

from __future__ import annotations

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "custom-3dgs-cuda_b200" / "csrc"


def code_of(path):
    return re.sub(r"//[^\n]*", "", path.read_text())


def test_no_read_only_loads_in_overlapped_kernels():
    files = [f for f in sorted(CSRC.glob("*.cu")) if "launch_overlapped" in code_of(f)]
    assert {"attention_single.cu", "rotary.cu", "rms_norm.cu"} <= {f.name for f in files}
    headers = ["attention.cuh", "overlap.cuh", "tensor_core.cuh", "token_types.cuh", "tma.cuh"]
    for f in files + [CSRC / h for h in headers]:
        for bad in (r"ld\.global\.nc", r"__ldg\(", r"__restrict__"):
            assert not re.search(bad, code_of(f)), (f.name, bad)


def test_overlapped_kernels_wait():
    """Each of them waits for the kernel in front."""
    for f in sorted(CSRC.glob("*.cu")):
        if "launch_overlapped" in code_of(f) and "__global__" in code_of(f):
            assert "wait_for_previous();" in code_of(f), f.name

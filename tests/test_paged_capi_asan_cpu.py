"""Host sanitizer builds of the C ABI of the paged cache and of grouped heads
(CPU only), as test_capi_asan_cpu.py builds csrc/capi.cpp: sources compiled for
the host alone with AddressSanitizer and UndefinedBehaviorSanitizer, linked with a
driver of tests/asan whose recorders stand in for the kernel launchers."""

import os
import shutil
import subprocess
from pathlib import Path

import pytest

from test_capi_asan_cpu import CSRC, ROOT, SAN


def _run(tmp_path, *sources):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    common = ["-x", "hip", "--cuda-host-only", "-std=c++17", "-O1", "-g", *SAN, f"-I{CSRC}", f"-I{ROOT / 'include'}"]
    objs = []
    for src in sources:
        obj = tmp_path / (src.stem + ".o")
        # (A file with kernels: its device code's symbol keeps its plain name, which the driver defines.)
        plain = ["-fuse-cuid=none"] if src.suffix == ".hip" else []
        subprocess.run([hipcc, *common, *plain, "-c", str(src), "-o", str(obj)], check=True, capture_output=True)
        objs.append(str(obj))
    exe = tmp_path / "driver"
    subprocess.run([hipcc, *SAN, *objs, "-o", str(exe)], check=True, capture_output=True)
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:halt_on_error=1",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    res = subprocess.run([str(exe)], capture_output=True, text=True, env=env, timeout=300)
    assert res.returncode == 0, res.stdout + res.stderr[-4000:]
    assert "all checks passed" in res.stdout


needs_hipcc = pytest.mark.skipif(shutil.which("hipcc") is None and not Path("/opt/rocm/bin/hipcc").exists(),
                                 reason="hipcc not available")


@needs_hipcc
def test_paged_capi_under_address_and_ub_sanitizers(tmp_path):
    _run(tmp_path, CSRC / "paged_capi.cpp", CSRC / "paged.hip", ROOT / "tests" / "asan" / "paged_driver.cpp")


@needs_hipcc
def test_grouped_dispatch_under_address_and_ub_sanitizers(tmp_path):
    _run(tmp_path, CSRC / "capi.cpp", ROOT / "tests" / "asan" / "grouped_driver.cpp")

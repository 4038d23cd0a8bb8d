"""Host sanitizer build of the learned bias by relative position and of rotary
embedding (CPU only): sources compiled for the host alone with AddressSanitizer and
UndefinedBehaviorSanitizer, as test_capi_asan_cpu.py builds csrc/capi.cpp, linked with
tests/asan/rel_driver.cpp, whose hipLaunchKernel sees what every kernel is given."""

import concurrent.futures
import os
import shutil
import subprocess

from test_capi_asan_cpu import CSRC, ROOT, SAN
from test_paged_capi_asan_cpu import needs_hipcc

SOURCES = ("capi.cpp", "paged_capi.cpp", "paged.hip", "rel_capi.cpp", "rel.hip", "rel_fwd.hip", "rel_bwd.hip",
           "rel_f32.hip", "rel_paged.hip", "bias.hip", "generic.hip", "rotary.hip")


@needs_hipcc
def test_position_capi_under_address_and_ub_sanitizers(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"

    def compiled(src):
        obj = tmp_path / (src.stem + ".o")
        # (A file with kernels: its device code's symbol keeps its plain name, which the driver defines.)
        subprocess.run([hipcc, "-x", "hip", "--cuda-host-only", "-std=c++17", "-O1", "-g", *SAN, "-fuse-cuid=none",
                        f"-I{CSRC}", f"-I{ROOT / 'include'}", "-c", str(src), "-o", str(obj)], check=True,
                       capture_output=True)
        return str(obj)

    with concurrent.futures.ThreadPoolExecutor(4) as pool:
        objs = list(pool.map(compiled, [*(CSRC / s for s in SOURCES), ROOT / "tests" / "asan" / "rel_driver.cpp"]))
    exe = tmp_path / "driver"
    # (Every such file defines the same empty id.)
    subprocess.run([hipcc, *SAN, *objs, "-Wl,-z,muldefs", "-o", str(exe)], check=True, capture_output=True)
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:halt_on_error=1",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    res = subprocess.run([str(exe)], capture_output=True, text=True, env=env, timeout=300)
    assert res.returncode == 0, res.stdout + res.stderr[-4000:]
    assert "all checks passed" in res.stdout

"""The host code of the gated recurrence, the RMS norm and the 8-bit product under
AddressSanitizer and UndefinedBehaviorSanitizer (the host side only), driven by
tests/operator_host_checks.cpp.  CPU only: no call reaches a launch."""
import concurrent.futures as cf
import os
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "gdn2-jax-kernel_amd" / "csrc"
SOURCES = ["gdn2_gscan.hip", "gdn2_norm.hip", "gdn2_int8.hip"]
SAN = ["-Xarch_host", "-fsanitize=address", "-Xarch_host", "-fsanitize=undefined",
       "-Xarch_host", "-fno-sanitize-recover=all"]


def test_host_code_under_asan_and_ubsan(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    clangxx = "/opt/rocm/llvm/bin/clang++"
    if not Path(hipcc).exists() or not Path(clangxx).exists():
        pytest.skip("ROCm toolchain not available")

    def compile_one(src):
        obj = tmp_path / (Path(src).stem + ".o")
        cmd = [hipcc, "-x", "hip", "--offload-arch=gfx950", "-O1", "-g", "-std=c++17", "-fPIC",
               "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops", *SAN, f"-I{CSRC}",
               f"-I{ROOT / 'include'}", "-c", str(CSRC / src), "-o", str(obj)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        assert res.returncode == 0, res.stderr[-2000:]
        return obj

    with cf.ThreadPoolExecutor(max_workers=3) as ex:
        objs = list(ex.map(compile_one, SOURCES))
    checks = tmp_path / "checks.o"
    subprocess.run([clangxx, "-O1", "-g", "-std=c++17", "-fsanitize=address,undefined",
                    f"-I{ROOT / 'include'}", "-c", str(ROOT / "tests" / "operator_host_checks.cpp"),
                    "-o", str(checks)], check=True)
    exe = tmp_path / "checks"
    subprocess.run([hipcc, "--offload-arch=gfx950", *SAN, str(checks), *map(str, objs), "-o",
                    str(exe)], check=True)
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0",
               UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1")
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=600, env=env)
    assert res.returncode == 0 and " 0 failures" in res.stdout, res.stdout + res.stderr[-4000:]

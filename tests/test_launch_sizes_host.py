"""Every size that the entry points take can be launched: the host code of the kernels, compiled
alone, against a runtime that only looks at the grids (tests/launch_sizes_checks.cpp).  CPU only."""
import concurrent.futures as cf
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
CSRC = ROOT / "gdn2-jax-kernel_amd" / "csrc"
SOURCES = ["gdn2_conv.hip", "gdn2_ssm.hip", "gdn2_fp8.hip"]


def test_every_size_that_is_taken_can_be_launched(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not Path(hipcc).exists():
        pytest.skip("ROCm toolchain not available")

    def compile_one(src):
        obj = tmp_path / (Path(src).stem + ".o")
        cmd = [hipcc, "-x", "hip", "--offload-arch=gfx950", "--offload-host-only", "-O2",
               "-std=c++17", "-fPIC", f"-I{CSRC}", f"-I{ROOT / 'include'}", "-c", str(src), "-o", str(obj)]
        res = subprocess.run(cmd, capture_output=True, text=True)
        assert res.returncode == 0, res.stderr[-2000:]
        return obj

    checks = ROOT / "tests" / "launch_sizes_checks.cpp"
    with cf.ThreadPoolExecutor(max_workers=4) as ex:
        objs = list(ex.map(compile_one, [checks, *(CSRC / s for s in SOURCES)]))
    exe = tmp_path / "checks"
    # the plain linker: the runtime's functions are the test's own; the kernels' device code, which
    # each object names, is nowhere
    subprocess.run(["g++", "-Wl,--unresolved-symbols=ignore-in-object-files", *map(str, objs), "-o",
                    str(exe)], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and " 0 failures" in res.stdout, res.stdout + res.stderr[-4000:]

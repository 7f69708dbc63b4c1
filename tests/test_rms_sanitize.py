"""The root-mean-square norm's entry points of the C ABI under the host
sanitizers (CPU only): tests/sanitize/rms_validate.c makes each of them refuse
bad arguments (null pointers, types, sizes and strides that overflow, groups,
small workspaces) and asks the size queries over their whole range; any
sanitizer report fails the run."""

import os
import subprocess
from pathlib import Path

import pytest

HERE = Path(__file__).resolve().parent / "sanitize"
OBJECTS = HERE.parents[1] / "gfx1010-kernels_amd" / "_build"


def test_rms_validation_paths_run_clean_under_host_sanitizers():
    if not list(OBJECTS.glob("rms_float_*.o")):
        pytest.skip("library objects not built (gfx1010-kernels_amd/build.py)")
    build = subprocess.run(["make", "-s", "-C", str(HERE), "rms_validate"], capture_output=True,
                           text=True, timeout=900)
    assert build.returncode == 0, build.stdout + build.stderr
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=0:abort_on_error=1",
               UBSAN_OPTIONS="halt_on_error=1:print_stacktrace=1", HIP_VISIBLE_DEVICES="")
    run = subprocess.run([str(HERE / "rms_validate")], capture_output=True, text=True,
                         timeout=300, env=env)
    assert run.returncode == 0, run.stdout + run.stderr
    assert run.stdout.strip().splitlines()[-1] == "ok", run.stdout + run.stderr

"""The checks and launch geometries of the operators around a fold under AddressSanitizer and UndefinedBehaviorSanitizer:
tests/san/driver_ops.c calls every entry point with random and boundary arguments, stand-ins in place of the launches."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "hcomm_amd", "csrc")
SAN = os.path.join(ROOT, "tests", "san")


@pytest.mark.skipif(shutil.which("gcc") is None, reason="no gcc")
def test_operators_host_code_is_clean_under_asan_and_ubsan(tmp_path):
    exe = str(tmp_path / "ops_driver")
    cmd = ["gcc", "-O1", "-g", "-std=c11", "-fsanitize=address,undefined", "-fno-sanitize-recover=undefined", "-fno-omit-frame-pointer",
           "-DHG_STUB_GPU_PRESENT", "-I" + os.path.join(ROOT, "include"), "-I" + CSRC]
    cmd += [os.path.join(CSRC, f) for f in ("hg_api.c", "hg_batch.c", "hg_sched.c", "hg_plan.c", "hg_check.c", "hg_ops.c")]
    cmd += [os.path.join(SAN, "stubs.c"), os.path.join(SAN, "driver_ops.c"), "-o", exe, "-lpthread", "-lm"]
    build = subprocess.run(cmd, capture_output=True, text=True)
    if build.returncode != 0 and "sanitize" in build.stderr + build.stdout and "cannot find" in build.stderr:
        pytest.skip("the sanitizer runtimes are not installed")
    assert build.returncode == 0, build.stderr[-2000:]
    run = subprocess.run([exe], capture_output=True, text=True, timeout=300, env=dict(os.environ, UBSAN_OPTIONS="print_stacktrace=1"))
    assert run.returncode == 0, (run.stdout[-1000:], run.stderr[-3000:])
    assert " bad 0" in run.stdout and "runtime error" not in run.stderr
    assert int(run.stdout.split()[1]) > 10000 and int(run.stdout.split()[3]) > 10000  # both kinds of call were met

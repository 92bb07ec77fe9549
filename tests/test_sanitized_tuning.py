"""The first phases of the operators for tuning the router and the norms under AddressSanitizer + UndefinedBehaviorSanitizer (host code, CPU only).

Their refusals and plans run in a child python process against the build of the library whose host code is instrumented; any report ends the child.
"""
import os
import subprocess
import sys

from test_sanitized_host import ROOT, _build_module


def test_refusals_and_plans_are_clean_under_asan_and_ubsan():
    build = _build_module()
    env = dict(os.environ)
    env["OPAPI_LIBRARY_PATH"] = build.build_sanitized()
    runtime = build.sanitizer_runtime()
    env["LD_PRELOAD"] = runtime + (":" + env["LD_PRELOAD"] if env.get("LD_PRELOAD") else "")  # the runtime has to come first
    env["ASAN_OPTIONS"] = "detect_leaks=0:halt_on_error=1:abort_on_error=1:detect_odr_violation=0"
    env["UBSAN_OPTIONS"] = "halt_on_error=1:print_stacktrace=1"
    res = subprocess.run([sys.executable, "-m", "pytest", "-x", "-q", "-m", "not gpu", "-p", "no:cacheprovider", "tests/test_moe_tuning.py"], cwd=ROOT, env=env,
                         stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=900)
    tail = res.stdout[-4000:]
    assert "AddressSanitizer" not in res.stdout and "runtime error:" not in res.stdout, tail
    assert res.returncode == 0 and " passed" in res.stdout, tail

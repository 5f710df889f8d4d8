"""The C entries of packed batches, tables on the GPU and shared prefixes under AddressSanitizer (CPU only): the refusals of
tests/test_packed_shared_host.py, none of which reaches a HIP call, against the sanitized build of the library's host code."""

import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "triton-llm_amd"))

from triton_llm import _build  # noqa: E402


def test_refusals_under_asan(tmp_path):
    if not (shutil.which("hipcc") or os.path.exists("/opt/rocm/bin/hipcc")):
        pytest.skip("hipcc not available")
    rt = _build.asan_runtime()
    if rt is None:
        pytest.skip("no shared ASan runtime in this toolchain")
    env = dict(os.environ)
    env["TRITON_LLM_HIP_LIB"] = _build.build_host_asan(str(tmp_path))
    env["LD_PRELOAD"] = rt + (":" + env["LD_PRELOAD"] if env.get("LD_PRELOAD") else "")
    env["ASAN_OPTIONS"] = "detect_leaks=0:exitcode=23"
    run = subprocess.run([sys.executable, "-m", "pytest", "-q", "-p", "no:cacheprovider", os.path.join(ROOT, "tests", "test_packed_shared_host.py")],
                         env=env, cwd=ROOT, capture_output=True, text=True, timeout=600)
    assert "AddressSanitizer" not in run.stdout + run.stderr, (run.stdout + run.stderr)[-4000:]
    assert run.returncode == 0, run.stdout[-4000:]
    assert " passed" in run.stdout and "failed" not in run.stdout

"""Host-side code of the sparse MLP half under AddressSanitizer and UBSan, on the CPU:
the experts' packed arrays, calls in passes and the executor's halves
(``tests/host/moe_test.cpp``), against launches that touch what the kernels touch
(``tests/host/fake_moe.cpp``). Any sanitizer report aborts the run.
"""
import os
import shutil
import subprocess

import pytest

HOST = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host")


@pytest.mark.skipif(shutil.which("make") is None or not os.path.exists("/opt/rocm/bin/hipcc"),
                    reason="needs make and hipcc")
def test_host_code_of_the_mlp_half_clean_under_asan_ubsan():
    r = subprocess.run(["make", "-C", HOST, "-j8", "run_moe"], capture_output=True, text=True,
                       timeout=600)
    out = r.stdout + r.stderr
    assert r.returncode == 0, out[-6000:]
    assert "ALL OK" in out, out[-3000:]
    assert "runtime error" not in out and "AddressSanitizer" not in out, out[-6000:]

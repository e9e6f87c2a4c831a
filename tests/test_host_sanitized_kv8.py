"""Host-side code of the 8-bit cache and the rotary positions under AddressSanitizer and UBSan, on
the CPU (``tests/host/kv8_test.cpp``): how attention cuts a row's pages, over head layouts,
lengths, windows and prefixes; the entries, against launches that touch what the kernels touch
(``tests/host/fake_kv8.cpp``). Any sanitizer report aborts the run.
"""
import os
import shutil
import subprocess

import pytest

HOST = os.path.join(os.path.dirname(os.path.abspath(__file__)), "host")


@pytest.mark.skipif(shutil.which("make") is None or not os.path.exists("/opt/rocm/bin/hipcc"),
                    reason="needs make and hipcc")
def test_host_code_of_the_8_bit_cache_clean_under_asan_ubsan():
    r = subprocess.run(["make", "-C", HOST, "-j8", "run_kv8"], capture_output=True, text=True,
                       timeout=600)
    out = r.stdout + r.stderr
    assert r.returncode == 0, out[-6000:]
    assert "ALL OK" in out, out[-3000:]
    assert "runtime error" not in out and "AddressSanitizer" not in out, out[-6000:]

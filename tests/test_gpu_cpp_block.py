"""GPU run of tests/cpp/block_tests.cpp: the grouped-query block's operators and
Graph nodes through include/evk_ai.h."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_cpp_block_suite():
    exe = os.path.join(ROOT, "evk_amd", "bin", "block_tests")
    assert os.path.exists(exe), "evk_amd/bin/block_tests is not built: run `python -m evk_amd.build`"
    print("running", exe, flush=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=110)
    sys.stdout.write(r.stdout[-4000:])
    assert r.returncode == 0 and "ALL PASSED" in r.stdout, r.stdout[-3000:] + r.stderr[-2000:]

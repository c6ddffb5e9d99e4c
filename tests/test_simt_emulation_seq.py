"""The sequence operators' device tests on the emulated device (tests/simt: the kernels' own sources, a fibre per lane), where there is no GPU."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SIMT = os.path.join(ROOT, "tests", "simt")
CLANG = os.environ.get("SIMT_CXX", "/opt/rocm/lib/llvm/bin/clang++")

pytestmark = [pytest.mark.cpu_only,
              pytest.mark.skipif(not os.path.exists(CLANG) or os.uname().machine != "x86_64", reason="the SIMT emulation build needs the ROCm clang++ on an x86-64 host")]


def test_the_device_tests_of_the_sequence_operators_pass_on_the_emulated_device():
    subprocess.run(["bash", os.path.join(SIMT, "build.sh")], check=True, timeout=1500)
    env = dict(os.environ, CRNN_HIP_LIB=os.path.join(SIMT, "libcrnn_simt.so"), SIMT_THREADS=os.environ.get("SIMT_THREADS", "4"))
    out = subprocess.run([sys.executable, "-m", "pytest", "tests/test_seq.py", "-m", "gpu", "-q", "-p", "no:cacheprovider"], cwd=ROOT, env=env,
                         capture_output=True, text=True, timeout=800)
    assert out.returncode == 0 and " passed" in out.stdout, out.stdout[-3000:] + out.stderr[-1000:]

"""One HIP runtime per process: libcrnn_hip.so and PyTorch must resolve to the same libamdhip64, whichever is loaded first."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ORDERS = {"library_first": "import crnn_amd, torch", "torch_first": "import torch, crnn_amd"}


def _run(code):
    out = subprocess.run([sys.executable, "-c", f"import sys; sys.path.insert(0, {ROOT!r})\n" + code], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]
    return out.stdout


@pytest.mark.parametrize("order", sorted(ORDERS))
def test_one_hip_runtime_is_mapped(order):
    out = _run(ORDERS[order] + """
maps = {l.split()[-1] for l in open("/proc/self/maps") if "libamdhip64" in l}
print(len({__import__("os").path.realpath(m) for m in maps}))
""")
    assert out.split()[-1] == "1", out


@pytest.mark.gpu
@pytest.mark.parametrize("order", sorted(ORDERS))
def test_library_and_torch_see_the_device_in_one_process(order):
    out = _run(ORDERS[order] + """
import numpy as np
from crnn_amd.cathode import svgd_update
rng = np.random.default_rng(0)
h = svgd_update(1 + 0.05 * rng.standard_normal((6, 17)), rng.standard_normal((6, 17)), 0.01)[3]
print(h > 0 and torch.cuda.is_available() and float(torch.ones(3, device="cuda").sum()) == 3.0)
""")
    assert out.split()[-1] == "True", out

"""Page plans, adapters and sampling on torch tensors: see step_torch_check.py."""
import importlib.util
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu


def test_torch_tensors_on_side_streams_and_captured(gpu):
    if importlib.util.find_spec("torch") is None:  # not imported here: it would bring its HIP runtime with it
        pytest.skip("needs torch")
    script = os.path.join(os.path.dirname(os.path.abspath(__file__)), "step_torch_check.py")
    # the first import of torch on a machine can take minutes
    out = subprocess.run([sys.executable, "-u", script], capture_output=True, text=True, timeout=300)
    print(out.stdout)
    assert out.returncode == 0 and out.stdout.strip().endswith("ok"), out.stdout + out.stderr

"""calm_amd/paged.py on torch tensors: streams, captured graphs, strides, refusals -- one child process, because torch and this library share a
HIP runtime only where torch is imported first."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT


@pytest.mark.gpu
def test_paged_operators_on_torch_tensors():
    r = subprocess.run([sys.executable, "-u", os.path.join(ROOT, "tests", "paged_torch_child.py")], capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and r.stdout.rstrip().endswith("ALL OK"), r.stdout[-2000:] + r.stderr[-3000:]

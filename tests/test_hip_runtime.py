"""The library and torch in one process.  No GPU is needed."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("first", ["from fhemamba_amd import core", "import torch",
                                   "from fhemamba_amd import _lib; _lib.device_free_bytes()"])
def test_one_hip_runtime_in_either_order_of_imports(first):
    """They share streams and memory, so they have to share the runtime."""
    pytest.importorskip("torch")
    code = (f"{first}\nimport torch\nfrom fhemamba_amd import clear, _lib\n_lib.device_free_bytes()\n"
            "print(len({line.split()[-1] for line in open('/proc/self/maps') if 'libamdhip64' in line}))")
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                         env={**os.environ, "PYTHONPATH": os.path.join(ROOT, "fhe-mamba_amd")})
    assert run.returncode == 0, run.stderr
    assert run.stdout.split()[-1] == "1"

"""The library without a usable torch beside it.  No GPU is needed."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def imports(code, *paths):
    path = os.pathsep.join([*paths, os.path.join(ROOT, "fhe-mamba_amd")])
    code += "\nfrom fhemamba_amd import _lib\nprint(_lib.lib.fhe_abi_version())\n"
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                         env={**os.environ, "PYTHONPATH": path})
    assert run.returncode == 0, run.stderr
    assert run.stdout.split()[-1] == "1"


def test_a_runtime_that_does_not_load(tmp_path):
    """A damaged or foreign HIP runtime in torch's folder leaves the system's."""
    lib = tmp_path / "torch" / "lib"
    lib.mkdir(parents=True)
    (tmp_path / "torch" / "__init__.py").write_text("")
    (lib / "libamdhip64.so").write_text("not a library")
    imports("", str(tmp_path))


@pytest.mark.parametrize("stand_in", ["None", "types.ModuleType('torch')"])
def test_a_stand_in_for_torch(stand_in):
    imports(f"import sys, types\nsys.modules['torch'] = {stand_in}")

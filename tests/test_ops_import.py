"""ops imports on a torch without CUDA bindings (its host-only parts are used there)."""
import subprocess
import sys

import pytest

from conftest import ROOT


@pytest.mark.parametrize("missing", ["_cuda_getDevice", "_cuda_getCurrentRawStream"])
def test_without_a_private_name_of_torch(missing):
    code = (f"import torch\nif hasattr(torch._C, {missing!r}): del torch._C.{missing}\n"
            "from qweninferenceengine_b200 import ops\nassert callable(ops._current_device)\nassert callable(ops._raw_stream)\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]

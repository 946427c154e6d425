"""The module's shortcuts to torch's current device and stream: used where this torch has them, replaced by
the public calls where not."""

import subprocess
import sys
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent


@pytest.mark.parametrize("gone", [["_cuda_getDevice"], ["_cuda_getCurrentRawStream"], ["_cuda_getDevice", "_cuda_getCurrentRawStream"]])
def test_import_without_the_private_names(gone):
    code = "import torch\n" + "".join(f"del torch._C.{n}\n" for n in gone if hasattr(torch._C, n)) + \
        "from opac1ty_b200 import kv, score\nassert callable(kv._get_device) and callable(score._raw_stream)\n"
    subprocess.run([sys.executable, "-c", code], cwd=ROOT, check=True, timeout=300)


@pytest.mark.gpu
def test_the_shortcuts_name_the_current_device_and_stream(cuda_device):
    from opac1ty_b200 import kv

    assert kv._get_device() == torch.cuda.current_device()
    with torch.cuda.stream(torch.cuda.Stream()) as _:
        assert kv._raw_stream(cuda_device.index) == torch.cuda.current_stream(cuda_device).cuda_stream
        assert kv._public_stream(cuda_device.index) == torch.cuda.current_stream(cuda_device).cuda_stream

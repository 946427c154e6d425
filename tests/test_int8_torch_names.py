"""int8's shortcut to torch's allocation: used where this torch has it, replaced by the public call where not."""

import subprocess
import sys
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent
GONE = "import torch\ng = getattr(getattr(torch._C, '_dynamo', None), 'guards', None)\nif hasattr(g, '_empty_strided_cuda'): del g._empty_strided_cuda\n"


def test_import_without_the_private_name():
    code = GONE + "from opac1ty_b200 import int8\nassert int8._empty_strided is None\n"
    subprocess.run([sys.executable, "-c", code], cwd=ROOT, check=True, timeout=300)


@pytest.mark.gpu
def test_results_without_it(cuda_device):
    code = GONE + """
from opac1ty_b200 import int8
x = torch.randn(7, 300, device='cuda:0')
h, r = int8.add_rmsnorm(x, x, values=torch.float16)
y = int8.linear(r, int8.Int8Weight.quantize(x))
assert h.shape == (7, 300) and r.codes.shape == (7, 300) and r.values.dtype == torch.float16 and y.shape == (7, 7)
assert torch.equal(h, x + x) and (y.diagonal() > 0).all()
"""
    subprocess.run([sys.executable, "-c", code], cwd=ROOT, check=True, timeout=300)


@pytest.mark.gpu
def test_the_shortcut_gives_what_is_asked_for(cuda_device):
    from opac1ty_b200 import int8

    like = torch.zeros(1, device=cuda_device)
    for shape, strides in (((3, 5), (5, 1)), ((0, 64), (64, 1)), ((17,), (1,)), ((0,), (1,))):
        for dtype in (torch.float16, torch.bfloat16, torch.float32):
            t = int8._empty(like, cuda_device.index, shape, strides, dtype)
            assert tuple(t.shape) == shape and t.dtype == dtype and t.device == cuda_device and t.is_contiguous()
            assert t.data_ptr() % 128 == 0

"""Every way in which the 8-bit product deals its work, bit for bit against its definition: products whose plan is the
same for any likely number of clusters on the device (test_int8_plan.py holds them to it)."""

import pytest
import torch

import int8_ref
from int8_plan import SHAPES
from opac1ty_b200 import int8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dealt", list(SHAPES), ids=lambda d: f"tokens{d[0]}-pairs{d[1]}-rounds{d[2]}")
def test_results(cuda_device, dealt):
    rows, m, k = SHAPES[dealt]
    x = int8.Int8Rows(int8_ref.codes(rows, k, 1, cuda_device), int8_ref.scales(rows, 1, cuda_device))
    w = int8.Int8Weight(int8_ref.codes(m, k, 2, cuda_device), int8_ref.scales(m, 2, cuda_device))
    b = torch.randn(m, generator=torch.Generator().manual_seed(3)).to(cuda_device)
    held = torch.full((rows + 1, m + 1), 5.0, device=cuda_device)
    int8.linear(x, w, bias=b, out=held[:rows, :m])
    # the sums by fp64 products on the device, exact in any order; then the stated fp32 operations
    s = (x.codes.double() @ w.codes.double().T).float()
    want = s * x.scales[:, None] * w.scales[None, :] + b[None, :]
    assert torch.equal(held[:rows, :m], want)
    assert (held[rows] == 5).all() and (held[:, m] == 5).all()

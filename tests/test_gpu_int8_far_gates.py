"""Gates far below 0 beside values of `up` that bring their products back into range, against the definition in 64
bits: 1 / (1 + exp(-g)) is below fp32's normal range from -87.4 on, and exp(-g) above its range from -88.8 on."""

import numpy as np
import pytest
import torch

from int8_ref import BF16, E, F16, F32, check_rows, f64
from opac1ty_b200 import int8

pytestmark = pytest.mark.gpu


def e_far(least):
    """Of v, relative: the exponent g log2 e by half a step and a constant off by less than half of one (|g| 1.5 E of the
    power); twice (the root of the power, squared) a power of two by 2 steps of fp32 (a step is 2 E), 1 + it by a
    rounding and its reciprocal by a step; three products."""
    return (-least * 1.5 + 2 * (4 + 1 + 2) + 3) * E


def check(gate, up, least):
    g, u = f64(gate), f64(up)
    with np.errstate(all="ignore"):
        v = g / (1 + np.exp(-g)) * u
    check_rows(int8.silu_mul(gate, up, values=F32), v, e_far(least), 0.0)
    return v


def draw(rows, n, lo, hi, dtype, device, seed):
    g = torch.Generator(device=device).manual_seed(seed)
    gate = (lo + (hi - lo) * torch.rand(rows, n, generator=g, device=device)).to(dtype)
    up = (torch.randn(rows, n, generator=g, device=device).clamp(-3, 3) * 1e38).to(dtype)
    return gate, up


@pytest.mark.parametrize("n", [1, 9, 1000, 2047, 4096, 14336, 20000, 40000])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lo,hi", [(-88.7, -87.4), (-44.5, -43.5), (-150, -60), (-110, -89)])
def test_large_up(cuda_device, n, dtype, lo, hi):
    gate, up = draw(4, n, lo, hi, dtype, cuda_device, n)
    up[:, 0] = 2e38  # (no row may be all small: those near 2^-100 may go either way)
    v = check(gate, up, lo - 1)
    assert (np.abs(v).max(-1) > 2.0 ** -99).all()


@pytest.mark.parametrize("n", [300, 5000])
def test_one_far_gate_in_a_row(cuda_device, n):
    """It has the row's largest value, or one beside an ordinary row's."""
    gate, up = draw(6, n, -5, 5, F32, cuda_device, 1)
    up *= 1e-38
    at = torch.arange(6, device=cuda_device) * 40 + 3
    rows = torch.arange(6, device=cuda_device)
    gate[rows, at] = torch.tensor([-88.0, -89.0, -95.0, -60.0, -87.4, -100.0], device=cuda_device)
    up[rows, at] = torch.tensor([3e38, -3e38, 3e38, 1e27, 3e38, 3e38], device=cuda_device)
    check(gate, up, -100)


def test_halves(cuda_device):
    """fp16's largest `up`: beside a row whose largest value is just above 2^-100."""
    gate = torch.tensor([[-84.0, -87.5, -88.0, -86.0]], dtype=F16, device=cuda_device).repeat(2, 500)
    up = torch.tensor([[65504.0, -65504.0, 65504.0, 1000.0]], dtype=F16, device=cuda_device).repeat(2, 500)
    v = check(gate, up, -88)
    assert np.abs(v).max() > 2.0 ** -99 and np.abs(v[0, 1]) * 127 / np.abs(v).max() > 1


def test_beyond(cuda_device):
    """From -174 on nothing is left, whatever `up` is; an infinite gate below 0 stays -inf * 0, a NaN."""
    gate = torch.full((4, 3000), -180.0, device=cuda_device)
    up = torch.full((4, 3000), 3e38, device=cuda_device)
    gate[1] = -3e38
    gate[2, 7] = float("-inf")
    gate[3, 11] = 1.0
    r = int8.silu_mul(gate, up, values=F32)
    assert not r.scales[:2].any() and not r.codes[:3].any() and torch.isnan(r.scales[2])
    assert r.codes[3, 11] == 127 and r.codes[3].count_nonzero() == 1

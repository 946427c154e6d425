"""Codes of rows as they are: round(q) with q the fp32 nearest to v * 127 / a, for values whose quotient lies
beside a half, where a quotient one step off would round to another code.

v * 127 has 31 bits at the most, so a double holds it; the quotient of that and a (24 bits) is a midpoint of two fp32
values or at least 2^-49 of itself away from one, so rounding it to a double first changes nothing.  The kernel forms
it as q + r / a with q off by two steps at most, the remainder r and 1 / a to 2^-23 of themselves: before its last
rounding it is within 2^-21 steps, 2^-44 of itself, of the quotient.  Where that reaches across a midpoint both neighbours
are right."""

import numpy as np
import pytest
import torch

from opac1ty_b200 import int8

pytestmark = pytest.mark.gpu


def check(codes, v):
    u = v * 127 / np.abs(v).max(-1, keepdims=True)
    lo, hi = (np.rint((u * (1 + s * 2.0 ** -44)).astype(np.float32)) for s in (-1, 1))
    got = codes.cpu().numpy()
    assert (lo != hi).mean() < 1e-4
    wrong = (got != lo) & (got != hi)
    assert not wrong.any(), f"{wrong.sum()} of {wrong.size}, first at {np.argwhere(wrong)[0]}"


def beside_halves(rows, n, seed, power=0):
    """Rows with their largest value first and then values within 4 steps of (k + 1/2) a / 127."""
    rng = np.random.default_rng(seed)
    a = (1 + rng.random((rows, 1))).astype(np.float32)
    k = rng.integers(0, 127, size=(rows, n))
    v = ((k + 0.5) * a.astype(np.float64) / 127).astype(np.float32)
    v = (v.view(np.int32) + rng.integers(-4, 5, size=v.shape, dtype=np.int32)).view(np.float32)
    v *= rng.choice([-1, 1], size=v.shape).astype(np.float32)
    v[:, :1] = a
    return v * np.float32(2.0 ** power)


@pytest.mark.parametrize("power", [-99, -20, 0, 60, 126])
@pytest.mark.parametrize("rows,n", [(200, 1000), (100, 1011), (40, 4096), (20, 20000), (3, 40000)])
def test_quantize(cuda_device, rows, n, power):
    v = beside_halves(rows, n, n + power + 200, power)
    check(int8.quantize(torch.from_numpy(v).to(cuda_device)).codes, v.astype(np.float64))

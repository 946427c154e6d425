"""Rows into 8 bits on the GPU (quantize, silu_mul, add_rmsnorm) against their definitions in 64 bits."""

import ctypes

import numpy as np
import pytest
import torch

from int8_ref import BF16, E, F16, F32, check_rows, f64
from opac1ty_b200 import _lib, int8

pytestmark = pytest.mark.gpu

WIDTHS = [1, 7, 8, 9, 255, 256, 257, 600, 1000, 1024, 1025, 2047, 4096, 5003, 8192, 14336, 16384, 16385, 28672, 32768,
          32769, 131071]
# relative errors of v, from the roundings that make it.  silu(g): the exponent g log2 e by a rounding and
# half of one of the constant, so its power by |g| 1.5 E, the power of two by 2 steps of fp32 (a step is
# 2 E), 1 + it by a rounding, the reciprocal by a step, two products.  Gates in the tests stay below 20
# (or are so far out that the power is 0 or infinite)
E_SILU = (20 * 1.5 + 4 + 1 + 2 + 2) * E
E_SUM = E           # h + y
E_NORM = E_SUM + E  # times the weight


def values(rows, n, seed, dtype, device, spread=True):
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(rows, n, generator=g, device=device)
    if spread:  # rows of very different sizes, a few large values
        x *= 10.0 ** torch.linspace(-2, 2, rows, device=device)[:, None]
        x[:, ::97] *= 9
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_halves_go_to_even(cuda_device, dtype):
    """Codes of 16-bit inputs are exact: v * 127 / a of 8- and 11-bit mantissas is a half, or lies 2^-12 of a
    step beside one at the least, so 64-bit arithmetic (v * 127 is exact, the quotient nearest) decides it."""
    x = values(600, 1000, 5, dtype, cuda_device)
    x[:, :8] = x.abs().amax(-1, keepdim=True) * torch.tensor([127 / 128, 0.5, 0.25, 1 / 8, -0.5, -0.25, 1.0, -1.0], device=cuda_device)
    x[::3] = (x[::3].float() / x[::3].float().abs().amax() * 254).round().to(dtype)  # small whole numbers
    r = int8.quantize(x)
    v = f64(x)
    u = v * 127 / np.maximum(np.abs(v).max(-1, keepdims=True), 1e-30)
    assert ((np.abs(u) % 1) == 0.5).sum() > 1000
    assert np.array_equal(r.codes.cpu().numpy(), np.rint(u).astype(np.int8))


def e_ss(n):
    """Of the root of a sum of n squares: the longest chain of fp32 additions (32 values of a thread, or a
    1024th of the row, then twice 5 steps of a warp), the squares' rounding, the division by n (two roundings)
    and the addition; and of its reciprocal, by two steps of fp32."""
    return (max(32, -(-n // 1024)) + 10 + 1 + 3) * E / 2 + 4 * E


@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_quantize(cuda_device, n, dtype):
    x = values(5, n, n, dtype, cuda_device)
    for held in (None, F16, BF16, F32):
        r = int8.quantize(x, values=held)
        assert (r.values is None) == (held is None) and r.codes.shape == (5, n)
        check_rows(r, f64(x), 0.0, 0.0)


@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_silu_mul(cuda_device, n, dtype):
    gu = (values(3, 2 * n, n, dtype, cuda_device, spread=False) * 3).clamp(-20, 20)
    g, u = f64(gu[:, :n]), f64(gu[:, n:])
    v = g / (1 + np.exp(-g)) * u
    check_rows(int8.silu_mul(gu, values=F16), v, E_SILU, 0.0)
    gate, up = gu[:, :n].contiguous(), gu[:, n:].contiguous()
    a, b = int8.silu_mul(gate, up), int8.silu_mul(gu)
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)


@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("h_type,y_type,w_type", [(F32, F16, F16), (F32, BF16, None), (F32, F32, F32), (F16, F16, BF16),
                                                  (BF16, BF16, BF16), (F16, None, F16), (BF16, None, None), (F32, None, F32)])
def test_add_rmsnorm(cuda_device, n, h_type, y_type, w_type):
    rows = 4
    h = values(rows, n, n, h_type, cuda_device)
    y = None if y_type is None else values(rows, n, n + 1, y_type, cuda_device, spread=False)
    w = None if w_type is None else (1 + 0.3 * values(1, n, n + 2, F32, cuda_device, spread=False)[0]).to(w_type)
    before = h.clone()
    h_new, r = int8.add_rmsnorm(h, y, w, eps=1e-5, values=F16)
    assert torch.equal(h, before)
    t = f64(h) + (0 if y is None else f64(y))
    if y is None:
        assert h_new is h
    else:
        assert torch.equal(h_new, (h.float() + y.float()).to(h_type))
    rms = np.sqrt((t * t).mean(-1) + 1e-5)
    # h + y may cancel: what the fp32 sum is off by is relative to itself, so every t is off by E at most
    check_rows(r, t if w is None else t * f64(w), (0 if y is None else E_SUM) + (0 if w is None else E), e_ss(n) + 2 * E, rms)
    again = h.clone()
    h_in, r2 = int8.add_rmsnorm(again, y, w, eps=1e-5, h_out=again)
    assert h_in is again and torch.equal(again, h_new if y is not None else before)
    assert torch.equal(r.codes, r2.codes) and torch.equal(r.scales, r2.scales)


def test_many_rows(cuda_device):
    """More rows than a grid dimension other than the first takes, and every row by itself."""
    x = values(70001, 40, 3, F16, cuda_device)
    check_rows(int8.quantize(x, values=F16), f64(x), 0.0, 0.0)
    for rows, n in ((3001, 1300), (3001, 8192), (700, 16000), (200, 2000)):
        x = values(rows, n, 4, BF16, cuda_device)
        check_rows(int8.quantize(x), f64(x), 0.0, 0.0)


@pytest.mark.parametrize("n", [40, 2000, 40000])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_rows_of_zeros_infinities_and_nan(cuda_device, n, dtype):
    x = values(9, n, 1, dtype, cuda_device, spread=False)
    x[1] = 0
    x[2, n - 1] = float("inf")
    x[3, 0] = float("nan")
    x[4, n // 2] = float("-inf")
    x[5] = 0
    x[5, 3] = torch.finfo(dtype).tiny if dtype == F16 else 1e-38  # fp16: a live row; others: below 2^-100
    x[6] = 0
    x[6, 5] = -torch.finfo(dtype).max
    x[7] = float("nan")
    x[8, 1:3] = torch.tensor([float("inf"), float("nan")], dtype=dtype)
    check_rows(int8.quantize(x, values=F32), f64(x), 0.0, 0.0)
    w = torch.ones(n, dtype=F32, device=cuda_device)
    h, r = int8.add_rmsnorm(x, None, w, h_out=torch.empty_like(x), values=F32)
    assert torch.equal(h.nan_to_num(3.0), x.nan_to_num(3.0))
    t = f64(x)
    with np.errstate(all="ignore"):
        rms = np.sqrt((t * t).mean(-1) + 1e-5)
    check_rows(r, t, 0.0, e_ss(n) + 2 * E, rms)
    gu = torch.cat([x, torch.ones_like(x)], -1)
    g = f64(x)
    with np.errstate(all="ignore"):
        v = g / (1 + np.exp(-g))
    # silu(-inf) is -inf * 0, a NaN; a gate this far below 0 that the quotient's denominator leaves fp32
    # is 0 instead of about 1e-36: both below every code of these rows
    check_rows(int8.silu_mul(gu), v, E_SILU, 0.0)


def test_squares_beyond_fp32(cuda_device):
    for big in (1e19, 1e30, 3e38):
        h = torch.full((2, 5000), big, device=cuda_device)
        h[0, 1::2] *= -0.5
        _, r = int8.add_rmsnorm(h, eps=1e-5)
        t = f64(h)
        check_rows(r, t, 0.0, e_ss(5000) + 4 * E, np.sqrt((t * t).mean(-1)))
    _, r = int8.add_rmsnorm(h, None, torch.full((5000,), 10.0, device=cuda_device))  # 3e39 is no fp32
    assert torch.isnan(r.scales).all() and not r.codes.any()


@pytest.mark.parametrize("shift", [1, 3, 4])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_strides_and_alignment(cuda_device, shift, dtype):
    n, rows = 1011, 6
    wide = values(rows, 2 * n + 40, 8, dtype, cuda_device)
    x = wide[:, shift:shift + n]
    a, b = int8.quantize(x, values=F16), int8.quantize(x.contiguous(), values=F16)
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales) and torch.equal(a.values, b.values)
    u = wide[:, shift + n + 1:shift + 2 * n + 1]
    a, b = int8.silu_mul(x, u), int8.silu_mul(x.contiguous(), u.contiguous())
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    out = torch.full((rows, n + 9), 5, dtype=dtype, device=cuda_device)
    w = values(1, n + 1, 9, dtype, cuda_device, spread=False)[0]
    ha, a = int8.add_rmsnorm(x, u, w[1:], h_out=out[:, 1:n + 1])
    hb, b = int8.add_rmsnorm(x.contiguous(), u.contiguous(), w[1:].clone())
    assert torch.equal(ha, hb) and torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    assert (out[:, 0] == 5).all() and (out[:, n + 1:] == 5).all()


@pytest.mark.parametrize("n", [9, 1011, 2005])
def test_nothing_is_written_beside_the_rows(cuda_device, n):
    ld = -(-n // 16) * 16 + 16
    x = values(3, n, 2, F16, cuda_device)
    codes = torch.full((5, ld), 99, dtype=torch.int8, device=cuda_device)
    scales = torch.full((5,), -1.0, device=cuda_device)
    vals = torch.full((5, n + 3), -2.0, dtype=BF16, device=cuda_device)
    c = _lib.I8Rows(3, n, ld, codes[1:].data_ptr(), scales[1:].data_ptr())
    stream = torch.cuda.current_stream(cuda_device).cuda_stream
    _lib.check(_lib.load().opc_i8_quantize(x.data_ptr(), n, _lib.OPC_F16, ctypes.byref(c), vals[1:].data_ptr(), n + 3,
                                           _lib.OPC_BF16, stream))
    want = int8.quantize(x, values=BF16)
    assert torch.equal(codes[1:4, :n], want.codes) and torch.equal(scales[1:4], want.scales)
    assert torch.equal(vals[1:4, :n], want.values)
    codes[1:4, :n], scales[1:4], vals[1:4, :n] = 99, -1.0, -2.0
    assert (codes == 99).all() and (scales == -1).all() and (vals == -2).all()


@pytest.mark.parametrize("n", [1000, 60000])
def test_rows_past_32_bits(cuda_device, n):
    """Places in x, the codes and the values beyond 2^31: the rows there are those of a call by themselves."""
    rows = 2**31 // n + 70
    x = torch.randint(-30000, 30000, (rows, n), dtype=torch.int16, device=cuda_device,
                      generator=torch.Generator(device=cuda_device).manual_seed(1)).view(BF16)
    x = x.nan_to_num_(1.0, 2.0, 3.0)
    r = int8.quantize(x, values=BF16)
    for a in (0, rows - 75, rows - 5):
        want = int8.quantize(x[a:a + 5].clone(), values=BF16)
        assert torch.equal(r.codes[a:a + 5], want.codes) and torch.equal(r.scales[a:a + 5], want.scales)
        assert torch.equal(r.values[a:a + 5], want.values)


def test_no_rows(cuda_device):
    x = torch.empty(0, 64, dtype=F16, device=cuda_device)
    assert int8.quantize(x, values=F16).values.shape == (0, 64)
    assert int8.silu_mul(x).codes.shape == (0, 32)
    h, r = int8.add_rmsnorm(x, x)
    assert h.shape == (0, 64) and r.scales.shape == (0,)


def test_captured_and_on_another_stream(cuda_device):
    h, y = values(7, 4096, 1, F32, cuda_device), values(7, 4096, 2, F16, cuda_device)
    w = torch.ones(4096, dtype=F16, device=cuda_device)
    side = torch.cuda.Stream(cuda_device)
    side.wait_stream(torch.cuda.current_stream(cuda_device))
    with torch.cuda.stream(side):
        int8.add_rmsnorm(h, y, w)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            h2, r = int8.add_rmsnorm(h, y, w, values=F16)
        for seed in (3, 4):
            h.copy_(values(7, 4096, seed, F32, cuda_device))
            g.replay()
            h3, r3 = int8.add_rmsnorm(h, y, w, values=F16)
            assert torch.equal(h2, h3) and torch.equal(r.codes, r3.codes) and torch.equal(r.values, r3.values)
    torch.cuda.synchronize(cuda_device)


def test_refusals(cuda_device):
    x = values(2, 64, 1, F16, cuda_device)
    with pytest.raises(ValueError, match="x must be"):
        int8.quantize(x.cpu())
    with pytest.raises(ValueError, match="x must be"):
        int8.quantize(x.T)
    with pytest.raises(ValueError, match="x must be"):
        int8.quantize(x.to(torch.int8))
    with pytest.raises(ValueError, match="values must be"):
        int8.quantize(x, values=torch.float64)
    with pytest.raises(ValueError, match="rows of 131072"):
        int8.quantize(torch.zeros(1, 131072, device=cuda_device))
    with pytest.raises(ValueError, match="rows of 0"):
        int8.quantize(x[:, :0])
    with pytest.raises(_lib.OpcError, match="leading dimension"):
        int8.quantize(x[:1].expand(2, 64))
    with pytest.raises(ValueError, match="even width"):
        int8.silu_mul(x[:, :63])
    with pytest.raises(ValueError, match="up must be"):
        int8.silu_mul(x, x[:, :32])
    with pytest.raises(ValueError, match="gate is"):
        int8.silu_mul(x, x.float())
    with pytest.raises(ValueError, match="y must be"):
        int8.add_rmsnorm(x, x[:1])
    with pytest.raises(ValueError, match="beside an h"):
        int8.add_rmsnorm(x, x.float())
    with pytest.raises(ValueError, match="weight must be"):
        int8.add_rmsnorm(x, x, x[0, :32])
    with pytest.raises(ValueError, match="h_out is"):
        int8.add_rmsnorm(x, x, h_out=x.float())
    with pytest.raises(ValueError, match="overlap"):
        int8.add_rmsnorm(x, x, h_out=x[:1].expand(2, 64))
    for eps in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(_lib.OpcError, match="eps"):
            int8.add_rmsnorm(x, x, eps=eps)

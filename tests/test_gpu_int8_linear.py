"""The product of 8-bit tokens and weights on the GPU: bit for bit against its definition (the sum of
products is exact, the operations after it are named in the header)."""

import ctypes
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import int8_ref
from int8_ref import BF16, F16, F32
from opac1ty_b200 import _lib, int8

pytestmark = pytest.mark.gpu


def operands(rows, m, k, device, seed=0, extreme=False, ldx=None, ldw=None):
    x = int8.Int8Rows(int8_ref.codes(rows, k, seed, device, extreme, ldx), int8_ref.scales(rows, seed, device))
    w = int8.Int8Weight(int8_ref.codes(m, k, seed + 1, device, extreme, ldw), int8_ref.scales(m, seed + 1, device))
    return x, w


def same(y, x, w, bias=None):
    want = int8_ref.linear(x.codes, x.scales, w.codes, w.scales, bias, y.dtype)
    got = y.cpu()
    assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0)), \
        f"{(got != want).sum().item()} of {got.numel()} differ, first at {(got != want).nonzero()[0].tolist()}"


ROWS = [1, 2, 3, 5, 7, 8, 9, 15, 16, 17, 24, 31, 32, 33, 63, 64, 65, 100, 128, 129, 200, 255, 256, 257, 300, 511, 513]


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("m,k", [(1, 1), (100, 100), (1011, 1000), (4096, 1024), (513, 4099)])
def test_rows(cuda_device, rows, m, k):
    x, w = operands(rows, m, k, cuda_device, seed=rows)
    same(int8.linear(x, w), x, w)


@pytest.mark.parametrize("k", [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1000, 2048, 14336, 28675])
@pytest.mark.parametrize("rows", [1, 4, 8, 20, 130])
def test_widths(cuda_device, rows, k):
    x, w = operands(rows, 333, k, cuda_device, seed=k)
    same(int8.linear(x, w, dtype=BF16), x, w)


@pytest.mark.parametrize("m", [1, 15, 16, 17, 127, 128, 129, 255, 256, 257, 511, 1030, 32000])
@pytest.mark.parametrize("rows", [1, 6, 40, 270])
def test_channels(cuda_device, rows, m):
    x, w = operands(rows, m, 512, cuda_device, seed=m)
    same(int8.linear(x, w, dtype=F32), x, w)


@pytest.mark.parametrize("rows,m,k", [(1, 28672, 4096), (8, 6144, 4096), (24, 4096, 14336), (512, 6144, 4096),
                                      (777, 28672, 4096), (2049, 4096, 2048), (5000, 520, 640), (130, 20000, 256)])
def test_layers(cuda_device, rows, m, k):
    x, w = operands(rows, m, k, cuda_device, seed=5)
    same(int8.linear(x, w), x, w)


@pytest.mark.parametrize("rows", [1, 8, 30, 300])
@pytest.mark.parametrize("bias", [F16, BF16, F32])
@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_bias_and_types(cuda_device, rows, bias, dtype):
    x, w = operands(rows, 700, 900, cuda_device, seed=2)
    b = torch.randn(700, generator=torch.Generator().manual_seed(1)).to(bias).to(cuda_device)
    same(int8.linear(x, w, bias=b, dtype=dtype), x, w, b)


@pytest.mark.parametrize("rows", [1, 9, 140])
def test_the_largest_sums(cuda_device, rows):
    """131071 products of -128 and -128 are 2^31 - 16384."""
    x, w = operands(rows, 40, 131071, cuda_device, extreme=True)
    y = int8.linear(x, w, dtype=F32)
    same(y, x, w)
    assert (y > 0).all()


@pytest.mark.parametrize("rows", [1, 5, 40, 300])
def test_strides_and_what_lies_beside_the_result(cuda_device, rows):
    m, k = 515, 777
    x, w = operands(rows, m, k, cuda_device, seed=3, ldx=1024, ldw=800)
    for dtype in (F16, F32):
        for shift in (0, 1, 3):
            held = torch.full((rows + 2, m + 7), 5.0, dtype=dtype, device=cuda_device)
            out = held[1:rows + 1, shift:shift + m]
            assert int8.linear(x, w, out=out) is out
            same(out, x, w)
            out.fill_(5.0)
            assert (held == 5).all()


@pytest.mark.parametrize("rows", [2, 50, 300])
def test_nan_zero_and_infinite_scales(cuda_device, rows):
    x, w = operands(rows, 300, 200, cuda_device)
    x.scales[1] = float("nan")
    x.codes[1] = 0
    w.scales[7] = float("nan")
    x.scales[0] = 0.0
    w.scales[9] = float("inf")
    y = int8.linear(x, w, dtype=F32)
    assert torch.isnan(y[1]).all() and torch.isnan(y[:, 7]).all()
    same(y, x, w)


@pytest.mark.parametrize("rows", [1, 5, 12, 40, 300])
@pytest.mark.parametrize("k,ldx,ldw", [(777, 784, 800), (777, 1024, 784), (40, 48, 400), (4100, 4112, 4128)])
def test_rows_that_start_on_16_bytes_only(cuda_device, rows, k, ldx, ldw):
    """Weights as they are given (Int8Weight would lay them out anew)."""
    m = 515
    x = int8.Int8Rows(int8_ref.codes(rows, k, 1, cuda_device, ld=ldx), int8_ref.scales(rows, 1, cuda_device))
    held = int8_ref.codes(m + 1, k, 2, cuda_device, ld=ldw)
    w = int8.Int8Rows(held[1:], int8_ref.scales(m, 2, cuda_device))
    assert w.c.ld == ldw and w.c.codes % 128
    same(int8.linear(x, w), x, w)


def _random_codes(rows, ld, device, seed):
    return torch.randint(-128, 128, (rows, ld), dtype=torch.int8, device=device, generator=torch.Generator(device=device).manual_seed(seed))


def test_results_past_32_bits(cuda_device):
    """70001 x 32800 results (their places pass 2^31): those at the end, and at the 2^31st place."""
    rows, m, k = 70001, 32800, 48
    x = int8.Int8Rows(_random_codes(rows, k, cuda_device, 1), int8_ref.scales(rows, 1, cuda_device))
    w = int8.Int8Weight(_random_codes(m, k, cuda_device, 2), int8_ref.scales(m, 2, cuda_device))
    y = int8.linear(x, w)
    for a in (0, 2**31 // m - 2, rows - 5):
        want = int8_ref.linear(x.codes[a:a + 5], x.scales[a:a + 5], w.codes, w.scales, None, F16)
        assert torch.equal(y[a:a + 5].cpu(), want)


@pytest.mark.parametrize("rows", [1, 40])
def test_weights_past_32_bits(cuda_device, rows):
    m, k = 70001, 65536
    x = int8.Int8Rows(_random_codes(rows, k, cuda_device, 1), int8_ref.scales(rows, 1, cuda_device))
    w = int8.Int8Weight(_random_codes(m, k, cuda_device, 2), int8_ref.scales(m, 2, cuda_device))
    y = int8.linear(x, w, dtype=F32)
    for a in (0, 2**32 // k - 3, m - 6):
        want = int8_ref.linear(x.codes, x.scales, w.codes[a:a + 6], w.scales[a:a + 6], None, F32)
        assert torch.equal(y[:, a:a + 6].cpu(), want)


FIRST_CALL = """
import torch
from opac1ty_b200 import int8
dev = torch.device("cuda", 0)
x = int8.Int8Rows(torch.ones(40, 256, dtype=torch.int8, device=dev), torch.ones(40, device=dev))
w = int8.Int8Weight(torch.ones(300, 256, dtype=torch.int8, device=dev), torch.ones(300, device=dev))
t = torch.ones(40, 256, device=dev)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = int8.linear(x, w)
    h, r = int8.add_rmsnorm(t, t)
    z = int8.linear(r, w)
g.replay()
torch.cuda.synchronize()
assert (y == 256).all() and (h == 2).all() and (r.codes == 127).all() and ((z - 256).abs() < 0.25).all()
print("as it should")
"""


def test_a_process_whose_first_calls_are_captured(cuda_device):
    r = subprocess.run([sys.executable, "-c", FIRST_CALL], capture_output=True, text=True, timeout=300,
                       cwd=Path(__file__).resolve().parent.parent)
    assert r.returncode == 0 and "as it should" in r.stdout, r.stderr[-2000:]


def test_no_rows(cuda_device):
    x, w = operands(1, 64, 64, cuda_device)
    none = int8.Int8Rows(x.codes[:0], x.scales[:0])
    assert int8.linear(none, w).shape == (0, 64)


def test_streams_side_by_side(cuda_device):
    x, w = operands(40, 4096, 8192, cuda_device)
    want = int8.linear(x, w)
    torch.cuda.synchronize(cuda_device)
    streams = [torch.cuda.Stream(cuda_device) for _ in range(3)]
    outs = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(int8.linear(x, w))
    torch.cuda.synchronize(cuda_device)
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("rows", [1, 8, 24, 200])
def test_captured(cuda_device, rows):
    """A block's calls in a graph, replayed with new inputs; two graphs captured on one stream side by side."""
    hidden, inter = 512, 1376
    _, up = operands(1, 2 * inter, hidden, cuda_device, seed=1)
    _, down = operands(1, hidden, inter, cuda_device, seed=2)
    w = torch.ones(hidden, dtype=F16, device=cuda_device)

    def block(h, y):
        h2, a = int8.add_rmsnorm(h, y, w)
        return h2, int8.linear(int8.silu_mul(int8.linear(a, up)), down)

    graphs = []
    for i in range(2):
        h, y = torch.zeros(rows, hidden, device=cuda_device), torch.zeros(rows, hidden, dtype=F16, device=cuda_device)
        block(h, y)
        torch.cuda.synchronize(cuda_device)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = block(h, y)
        graphs.append((g, h, y, out))
    side = torch.cuda.Stream(cuda_device)
    for seed in range(3):
        gen = torch.Generator(device=cuda_device).manual_seed(seed)
        for _, h, y, _ in graphs:
            h.normal_(generator=gen)
            y.normal_(generator=gen)
        torch.cuda.synchronize(cuda_device)
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
        torch.cuda.synchronize(cuda_device)
        for _, h, y, out in graphs:
            want = block(h, y)
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@pytest.mark.parametrize("rows", [1, 70])
def test_weights_of_a_layer(cuda_device, rows):
    """A 2-bit layer's weights in 8 bits: within half an 8-bit step of the dequantized ones, and a product
    within what those steps and the tokens' own can add up to."""
    from opac1ty_b200 import synthetic
    from opac1ty_b200.layer import dequantize, prepare_layer

    dl = prepare_layer(synthetic.random_layer(520, 384, 6, 3), device=cuda_device)
    w = int8.Int8Weight.from_layer(dl)
    full = dequantize(dl).double()
    step = w.scales.double()[:, None]
    assert ((w.codes.double() * step - full).abs() <= step * (0.5 + 127 * 2.0 ** -22)).all()
    x16 = torch.randn(rows, 384, generator=torch.Generator().manual_seed(5)).half().to(cuda_device)
    x = int8.quantize(x16)
    y = int8.linear(x, w, dtype=F32).double()
    want = x16.double() @ full.T
    # |x w - x' w'| <= sum |x| |w - w'| + |x - x'| |w'|, with half a step each (and fp32's roundings after the sum)
    hx = 0.501 * x.scales.double()[:, None]
    bound = x16.double().abs() @ (0.501 * step).expand(-1, 384).T + hx @ (w.codes.double() * step).abs().sum(-1)[None, :]
    assert ((y - want).abs() <= bound + want.abs() * 2.0 ** -21).all()


def test_refusals(cuda_device):
    x, w = operands(4, 64, 48, cuda_device)
    _, other = operands(1, 64, 64, cuda_device)
    with pytest.raises(ValueError, match="x has rows of 48"):
        int8.linear(x, other)
    with pytest.raises(ValueError, match="results are"):
        int8.linear(x, w, dtype=torch.int32)
    with pytest.raises(ValueError, match="out must be"):
        int8.linear(x, w, out=torch.empty(4, 63, dtype=F16, device=cuda_device))
    with pytest.raises(ValueError, match="overlap"):
        int8.linear(x, w, out=torch.empty(1, 64, dtype=F16, device=cuda_device).expand(4, 64))
    with pytest.raises(ValueError, match="bias must be"):
        int8.linear(x, w, bias=torch.zeros(63, device=cuda_device))
    with pytest.raises(ValueError, match="start on 16 bytes"):
        int8.Int8Rows(torch.zeros(4, 50, dtype=torch.int8, device=cuda_device), torch.ones(4, device=cuda_device))
    with pytest.raises(ValueError, match="start on 16 bytes"):
        int8.Int8Rows(torch.zeros(4, 64, dtype=torch.int8, device=cuda_device)[:, 1:49], torch.ones(4, device=cuda_device))
    with pytest.raises(ValueError, match="codes must be"):
        int8.Int8Rows(torch.zeros(4, 48, dtype=torch.uint8, device=cuda_device), torch.ones(4, device=cuda_device))
    with pytest.raises(ValueError, match="scales must be"):
        int8.Int8Rows(torch.zeros(4, 48, dtype=torch.int8, device=cuda_device), torch.ones(3, device=cuda_device))
    with pytest.raises(ValueError, match="no channels"):
        int8.Int8Weight(torch.zeros(0, 48, dtype=torch.int8, device=cuda_device), torch.ones(0, device=cuda_device))
    # weights are laid out once, whatever they come as
    codes = int8_ref.codes(64, 48, 1, cuda_device)
    odd = torch.zeros(64, 50, dtype=torch.int8, device=cuda_device)
    odd[:, 1:49] = codes
    for given in (odd[:, 1:49], codes.T.contiguous().T):
        held = int8.Int8Weight(given, w.scales)
        assert torch.equal(int8.linear(x, held), int8.linear(x, w))
    assert torch.equal(held.codes, w.codes)


def test_results_carry_no_gradient(cuda_device):
    """Results carry no gradient, whatever their inputs ask for."""
    t = torch.randn(3, 64, device=cuda_device, requires_grad=True)
    r = int8.quantize(t, values=F32)
    assert not r.values.requires_grad
    h, r = int8.add_rmsnorm(t, t)
    assert not h.requires_grad


def test_device_error_word_is_clear(cuda_device):
    code = ctypes.c_int32(0)
    _lib.check(_lib.load().opc_take_device_error(cuda_device.index, ctypes.byref(code)))
    assert code.value == 0

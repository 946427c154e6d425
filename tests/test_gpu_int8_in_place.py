"""Tensors that the 8-bit calls write in place of a new one count as changed: what autograd or the framework's own caches
keep of them is stale."""

import pytest
import torch

import int8_ref
from opac1ty_b200 import _lib, int8

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


def calls(device):
    x = int8.Int8Rows(int8_ref.codes(4, 64, 1, device), int8_ref.scales(4, 1, device))
    w = int8.Int8Weight(int8_ref.codes(64, 64, 2, device), int8_ref.scales(64, 2, device))
    y = torch.ones(4, 64, device=device)
    return [lambda t: int8.linear(x, w, out=t), lambda t: int8.add_rmsnorm(t, y, h_out=t), lambda t: int8.add_rmsnorm(y, y, h_out=t),
            lambda t: int8.add_rmsnorm(y, h_out=t)]


@pytest.mark.parametrize("which", range(4))
def test_a_backward_pass_notices(cuda_device, which):
    leaf = torch.randn(4, 64, device=cuda_device, requires_grad=True)
    t = leaf * 2
    loss = (t * t).sum()  # keeps t
    calls(cuda_device)[which](t.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("which", range(4))
def test_versions(cuda_device, which):
    call = calls(cuda_device)[which]
    t = torch.zeros(4, 64, device=cuda_device)
    before = t._version
    call(t)
    assert t._version > before
    with torch.inference_mode():  # (no versions there)
        s = torch.zeros(4, 64, device=cuda_device)
        call(s)
    assert torch.equal(s, t) or which == 1  # (t + y of what t held)


def test_inputs_are_not_changed(cuda_device):
    h, y = torch.ones(4, 64, device=cuda_device), torch.ones(4, 64, device=cuda_device)
    versions = h._version, y._version
    new, r = int8.add_rmsnorm(h, y, values=F16)
    same, _ = int8.add_rmsnorm(h)
    int8.quantize(h)
    int8.linear(r, int8.Int8Weight.quantize(h), dtype=F32)
    assert same is h and (h._version, y._version) == versions and new._version == 0


@pytest.mark.parametrize("n", [60, 1011, 4096, 14336, 28672, 40000])
def test_the_sum_over_either_of_its_parts(cuda_device, n):
    g = torch.Generator(device=cuda_device).manual_seed(n)
    wide = torch.randn(50, 2 * n + 8, generator=g, device=cuda_device)
    for h, y in ((wide[:, :n], wide[:, n:2 * n]), (wide[:, :n].half(), wide[:, n:2 * n].half())):
        want, r = int8.add_rmsnorm(h, y)
        for first in (True, False):
            hh, yy = (h.clone(), y.clone()) if h.dtype == F16 else (lambda c: (c[:, :n], c[:, n:2 * n]))(wide.clone())
            out = hh if first else yy
            got, s = int8.add_rmsnorm(hh, yy, h_out=out)
            assert got is out and torch.equal(out, want) and torch.equal(yy if first else hh, y if first else h)
            assert torch.equal(s.codes, r.codes) and torch.equal(s.scales, r.scales)


def test_other_overlaps_are_refused(cuda_device):
    t = torch.randn(8, 64, device=cuda_device)
    before = t.clone()
    for h, y, w, h_out in ((t[:4], None, None, t[1:5]), (t[:4], t[4:], t[0], t[:4]), (t[:2], t[2:4].half(), None, t[1:3])):
        with pytest.raises(_lib.OpcError, match="overlaps"):
            int8.add_rmsnorm(h, y, w, h_out=h_out)
    assert torch.equal(t, before)

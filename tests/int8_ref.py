"""The 8-bit forms' definitions in numpy, for the tests: float64 where a value is checked within bounds, the
stated fp32 operations where it is checked bit for bit."""

import numpy as np
import torch

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
LEAST = 2.0 ** -100
E = 2.0 ** -24  # half a step of fp32, relative


def f64(t):
    return t.detach().double().cpu().numpy()


def check_rows(r, v, e_v, e_scale, rms=None):
    """r (Int8Rows) against rows v (float64, before their scale).  e_v: how far the kernel's own v may be
    off, relative (a few roundings to fp32); e_scale: likewise for the scale beyond that; rms: what the
    scale is divided by."""
    codes, scales = r.codes.cpu().numpy().astype(np.float64), f64(r.scales)
    bad = ~np.isfinite(v).all(-1)
    a = np.abs(np.where(np.isfinite(v), v, 0)).max(-1)
    zero = ~bad & (a < LEAST)
    live = ~bad & ~zero
    assert np.isnan(scales[bad]).all() and not codes[bad].any()
    assert not scales[zero].any() and not codes[zero].any()
    # code = round(v * 127 / a): v and a off by e_v each; the quotient the nearest fp32, or (e_v > 0) v times
        # 127 times a reciprocal that is off by a step at most: two more roundings and a step of 2 E
    u = v[live] * (127.0 / a[live])[:, None]
    off = np.abs(codes[live] - u)
    assert (off <= 0.5 + np.abs(u) * (2 * e_v + (E if e_v == 0 else 4 * E)) * 1.01).all(), off.max() - 0.5
    want = a[live] / 127.0 / (1.0 if rms is None else rms[live])
    assert (np.abs(scales[live] - want) <= want * (e_v + e_scale + 2 * E) * 1.01).all()
    if r.values is not None:
        got = (r.codes.float() * r.scales[:, None]).to(r.values.dtype)
        assert torch.equal(got.nan_to_num(7.0), r.values.nan_to_num(7.0))


def linear(xc, xs, wc, ws, bias, dtype):
    """The product as it is defined, operation by operation: the sum exact, then fp32."""
    s = xc.cpu().double() @ wc.cpu().double().T  # (below 2^53: exact in any order)
    y = s.float() * xs.cpu()[:, None] * ws.cpu()[None, :]
    if bias is not None:
        y = y + bias.cpu().float()[None, :]
    return y.to(dtype)


def codes(rows, n, seed, device, extreme=False, ld=None):
    """Codes in rows that start on 16 bytes (`ld` bytes apart), the bytes between them filled with 99."""
    g = torch.Generator().manual_seed(seed)
    ld = -(-n // 16) * 16 if ld is None else ld
    held = torch.full((rows, ld), 99, dtype=torch.int8)
    held[:, :n] = -128 if extreme else torch.randint(-128, 128, (rows, n), generator=g, dtype=torch.int8)
    return held.to(device)[:, :n]


def scales(rows, seed, device):
    g = torch.Generator().manual_seed(seed + 77)
    return (0.01 * (0.5 + torch.rand(rows, generator=g))).to(device)

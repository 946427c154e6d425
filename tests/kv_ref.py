"""The 4-bit paged cache in 64 bits, row by row from the definitions in include/opc_b200.h: what the
kernels of ``opac1ty_b200.kv`` are checked against."""

from __future__ import annotations

import numpy as np
import torch


class Setup:
    """A batch of sequences over shuffled pages, with tensors on `device`."""

    def __init__(self, device, q_lens, kv_lens, kv_heads, hd, page, seed=0, pad_rows=0, spare_pages=2, extra_cols=1):
        from opac1ty_b200 import kv

        rng = np.random.default_rng(seed)
        self.q_lens, self.kv_lens = list(q_lens), list(kv_lens)
        self.kv_heads, self.hd, self.page = kv_heads, hd, page
        self.rounded = False  # the batch's bounds send sequences of few rows to the form for many
        used = [-(-max(n, 0) // page) for n in kv_lens]
        self.n_pages = sum(used) + spare_pages
        order = rng.permutation(self.n_pages)
        width = max(used + [0]) + extra_cols
        table = np.full((len(kv_lens), width), -1, dtype=np.int32)  # entries past the end are never read
        at = 0
        for s, u in enumerate(used):
            table[s, :u] = order[at:at + u]
            at += u
        self.table = table
        self.rows = sum(q_lens) + pad_rows
        starts = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
        self.starts = starts
        self.cache = kv.KVCache(kv_heads, hd, self.n_pages, page, device=device)
        self.batch = kv.KVBatch(torch.from_numpy(starts).to(device),
                                torch.tensor(kv_lens, dtype=torch.int32, device=device),
                                torch.from_numpy(table).to(device), n_tokens=self.rows,
                                max_q=max(q_lens + [0]) if isinstance(q_lens, list) else max(q_lens),
                                max_kv=max(list(kv_lens) + [0]))

    def place(self, r):
        """(sequence, position) of row r; None for a row of no sequence."""
        for s in range(len(self.q_lens)):
            if self.starts[s] <= r < self.starts[s + 1]:
                return s, self.kv_lens[s] - (int(self.starts[s + 1]) - r)
        return None

    def block(self, s, pos):
        """(index of the page, place in it) of a position."""
        return int(self.table[s, pos // self.page]), pos % self.page


def parts(pages, page, hd):
    """Views (key codes [.., page, hd/2], value codes, key pairs [.., page, 2] fp16, value pairs) of pages."""
    half = page * hd // 2
    lead = pages.shape[:-1]
    kc = pages[..., :half].reshape(*lead, page, hd // 2)
    vc = pages[..., half:2 * half].reshape(*lead, page, hd // 2)
    pairs = np.ascontiguousarray(pages[..., 2 * half:]).view(np.float16).reshape(*lead, 2, page, 2)
    return kc, vc, pairs[..., 0, :, :], pairs[..., 1, :, :]


def nibbles(codes):
    return np.stack([codes & 15, codes >> 4], axis=-1).reshape(*codes.shape[:-1], -1)


def values(pages, page, hd):
    """(k, v) float64 [n_pages][kv_heads][page][hd] that the bytes stand for."""
    kc, vc, kp, vp = parts(pages, page, hd)
    f = lambda c, p: p[..., :1].astype(np.float64) * (nibbles(c).astype(np.float64) + p[..., 1:].astype(np.float64))
    with np.errstate(invalid="ignore"):
        return f(kc, kp), f(vc, vp)


def rotate64(x, pos, inv_freq, interleaved):
    """x [heads][hd] float64 turned at `pos`; the first 2 * len(inv_freq) dimensions are."""
    x = x.copy()
    n = len(inv_freq)
    ang = float(pos) * np.asarray(inv_freq, dtype=np.float64)
    c, s = np.cos(ang), np.sin(ang)
    a, b = (x[:, 0:2 * n:2].copy(), x[:, 1:2 * n:2].copy()) if interleaved else (x[:, :n].copy(), x[:, n:2 * n].copy())
    u, w = a * c - b * s, b * c + a * s
    if interleaved:
        x[:, 0:2 * n:2], x[:, 1:2 * n:2] = u, w
    else:
        x[:, :n], x[:, n:2 * n] = u, w
    return x


def quantize32(x):
    """(codes, scale, zero) of heads x [..., hd] by the definition's fp32 operations, one at a time."""
    x = x.astype(np.float32)
    lo, hi = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
    big = np.maximum(np.abs(lo), np.abs(hi))
    want = np.maximum((hi - lo) * np.float32(1.0 / 15.0), big * np.float32(2.0 ** -10))
    scale = np.maximum(want.astype(np.float16).astype(np.float32), np.float32(2.0 ** -24))
    zero = (lo / scale).astype(np.float16)
    n = np.rint(x * (np.float32(1.0) / scale) - zero.astype(np.float32))
    return np.clip(n, 0, 15).astype(np.uint8), scale, zero


def attention64(su: Setup, pages_np, q, scale, table_ok=None):
    """(out, lse, weighted |v|, bound of the scores' error, bound of the values' error) per row in
    float64; rows of no sequence are NaN.  The last three feed the tolerances."""
    k, v = values(pages_np, su.page, su.hd)
    with np.errstate(invalid="ignore"):
        off_k, off_v = (np.abs(s * (np.float64(1) * cz.astype(np.float16) - cz))
                        for s, cz in _codes_plus_zero(pages_np, su.page, su.hd))
    _, _, kp, _ = parts(pages_np, su.page, su.hd)
    R, H, hd = q.shape
    G = H // su.kv_heads
    out = np.full((R, H, hd), np.nan)
    lse = np.full((R, H), np.nan)
    mag = np.zeros((R, H, hd))
    dlt = np.zeros((R, H))
    dv = np.zeros((R, H, hd))
    for r in range(R):
        p = su.place(r)
        if p is None:
            continue
        s, pos = p
        if pos < 0:
            out[r], lse[r] = 0.0, -np.inf
            continue
        # many rows per kv head (more than the 16, or with large heads 8, of the form for steps): code +
        # zero goes to the tensor cores rounded to fp16, which moves the scores and values by this
        rounded = su.q_lens[s] * G > (16 if hd <= 128 else 8) or su.rounded
        idx = np.arange(pos + 1)
        pg, off = su.table[s, idx // su.page], idx % su.page
        for h in range(H):
            kk, vv = k[pg, h // G, off], v[pg, h // G, off]
            pr = kp[pg, h // G, off].astype(np.float64)
            qq = q[r, h].astype(np.float64)
            sc = scale * (kk @ qq)
            m = sc.max()
            if not np.isfinite(m):
                out[r, h], lse[r, h] = np.nan, np.nan
                continue
            e = np.exp(sc - m)
            w = e / e.sum()
            out[r, h] = w @ vv
            lse[r, h] = m + np.log(e.sum())
            mag[r, h] = w @ np.abs(vv)
            # fp32 sums of up to hd products q * code (at most 15) and q * zero, a few roundings each
            dlt[r, h] = abs(scale) * np.max(np.abs(pr[:, 0]) * (15.0 + np.abs(pr[:, 1]))) * np.abs(qq).sum() * 2.0 ** -21
            if rounded:
                dlt[r, h] += abs(scale) * np.max(off_k[pg, h // G, off] @ np.abs(qq))
                dv[r, h] = w @ off_v[pg, h // G, off]
    return out, lse, mag, dlt, dv


def _codes_plus_zero(pages, page, hd):
    """(scale, code + zero) of keys and of values, float64."""
    kc, vc, kp, vp = parts(pages, page, hd)
    for c, p in ((kc, kp), (vc, vp)):
        yield p[..., :1].astype(np.float64), nibbles(c).astype(np.float64) + p[..., 1:].astype(np.float64)


def check_attention(got, got_lse, ref, eps, live=None):
    """Tolerance: the output's rounding (eps/2 of it); each weight rounded once to fp16 (2^-11, plus
    what the fp32 exponential and sums add, 2^-18) and off by twice the scores' error, which moves
    the result by at most that times sum w |v|; the values' own error."""
    out, lse, mag, d, dv = ref
    live = np.isfinite(lse) if live is None else live
    tol = eps / 2 * np.abs(out) + ((2.0 ** -11 + 2.0 ** -18 + 2 * d[..., None]) * mag + dv) * (1 + eps) + 2.0 ** -24
    err = np.abs(got.astype(np.float64) - out)
    bad = ~(err <= tol) & live[..., None]
    assert not bad.any(), (np.argwhere(bad)[:4], err[bad][:4], tol[bad][:4])
    if got_lse is not None:
        tl = d + 2.0 ** -20 + 2.0 ** -21 * np.abs(np.where(live, lse, 0))
        el = np.abs(np.where(live, got_lse, 0) - np.where(live, lse, 0))
        assert (el <= tl).all(), (el.max(), tl[el > tl][:4])


def filled_pages(rng, n_pages, kv_heads, page, hd, mean=0.0):
    """Pages of quantized random heads: uint8 [n_pages][kv_heads][page * (hd + 8)]."""
    out = []
    pairs = []
    for which in range(2):
        x = rng.standard_normal((n_pages, kv_heads, page, hd)).astype(np.float32) + (mean if which == 0 else 0.0)
        c, s, z = quantize32(x)
        c = c.reshape(*c.shape[:-1], hd // 2, 2)
        out.append((c[..., 0] | (c[..., 1] << 4)).reshape(n_pages, kv_heads, -1))
        pr = np.concatenate([s.astype(np.float16), z], -1)
        pairs.append(np.ascontiguousarray(pr).view(np.uint8).reshape(n_pages, kv_heads, -1))
    return np.concatenate(out + pairs, -1)

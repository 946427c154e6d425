"""Attention over the 4-bit paged cache in 64 bits, with a bound of what the kernels' documented
roundings (include/opc_b200.h) may move each result and log sum by.  Keys of pages that the table
does not name take no part."""

from __future__ import annotations

import numpy as np

from kv_ref import nibbles, parts

LIFT = 5  # the reference of a row's weights: the largest is 2^LIFT in fp16 when it is set


def heads_of(pages, page, hd):
    """(scale, zero, codes) of keys and of values, float64, [pages][kv heads][page][...]."""
    kc, vc, kp, vp = parts(pages, page, hd)
    for c, p in ((kc, kp), (vc, vp)):
        yield p[..., :1].astype(np.float64), p[..., 1:].astype(np.float64), nibbles(c).astype(np.float64)


class Exact:
    """``out`` [rows][heads][hd], ``lse`` [rows][heads], and the bounds ``tol`` and ``tol_lse`` of what the
    kernels may be off by; rows of no sequence are NaN in all."""

    def __init__(self, su, pages, q, scale, eps, many=None):
        (ks, kz, kc), (vs, vz, vc) = heads_of(pages, su.page, su.hd)
        R, H, hd = q.shape
        G = H // su.kv_heads
        self.out, self.tol = np.full((R, H, hd), np.nan), np.full((R, H, hd), np.nan)
        self.lse, self.tol_lse = np.full((R, H), np.nan), np.full((R, H), np.nan)
        for r in range(R):
            p = su.place(r)
            if p is None:
                continue
            s, pos = p
            form_many = many if many is not None else su.q_lens[s] * G > (16 if hd <= 128 else 8)
            idx = np.arange(max(pos + 1, 0))
            pg, off = su.table[s, idx // su.page], idx % su.page
            there = (pg >= 0) & (pg < su.n_pages)
            idx, pg, off = idx[there], pg[there], off[there]
            # per kv head and tile of 128 keys: the largest scale of a value up to its end
            far = np.arange(max(min(su.kv_lens[s], (pos // 128 + 1) * 128), 0))
            tiles = su.table[s, far // su.page]
            held = (tiles >= 0) & (tiles < su.n_pages)
            for h in range(H):
                if pg.size == 0:
                    self.out[r, h], self.tol[r, h] = 0.0, 0.0
                    self.lse[r, h], self.tol_lse[r, h] = -np.inf, 0.0
                    continue
                at = (pg, h // G, off)
                largest = np.abs(vs[tiles[held], h // G, far[held] % su.page]).max()
                k = ks[at] * (kc[at] + kz[at])
                cz = vc[at] + vz[at]
                v = vs[at] * cz
                qq = q[r, h]
                if not np.isfinite(qq).all():
                    continue  # NaN
                sc = scale * (k @ qq)
                top = sc.max()
                e = np.exp(sc - top)
                T = e.sum()
                w = e / T
                out = w @ v
                # A score: hd / 16 + 1 accumulations in fp32, each cutting at most 2^-23 of sums that stay below
                # sum |q| (16 + |zero|) scale_k, and four roundings of 2^-24 of factors and products.
                big = np.max(ks[at][:, 0] * (16 + np.abs(kz[at][:, 0])))
                d = abs(scale) * big * np.abs(qq).sum() * (hd / 16 + 2) * 2.0 ** -23 + np.abs(sc).max() * 2.0 ** -22
                # Weights off by a factor of e^(+-2d); where one score leads by more than that, by what the others can be.
                mag = w @ np.abs(v)
                gap = top - np.partition(sc, -2)[-2] if sc.size > 1 else np.inf
                moved = np.minimum(np.expm1(min(2 * d, 700.0)) * mag,
                                   2 * sc.size * np.exp(np.clip(2 * d - gap, -700.0, 700.0)) * np.abs(v).max(0))
                # A weight rounded to fp16: 2^-11 of it and 2^-18 from the exponential and the sums, or half a step of
                # fp16's smallest, 2^-25, at a reference that is 2^LIFT and at most twice the largest scale of the keys
                # so far, whole tiles of 128 (what a row does not see of them included).
                small = sc.size * 2.0 ** (-25 - LIFT) * 2 * largest * np.abs(cz).max(0) / T
                # Products of 16 keys at a time: codes enter as code * 2^-24, fp16 numbers of exponent 2^-14, and what
                # lies 2^-24 below the largest exponent of a product is cut, for 16 products and the sum: 17 * 2^-24 *
                # 2^-14, in code steps 2^-10, of the largest weight (times its scale) among them.
                ws = np.zeros(-(-(pos + 1) // 16) * 16)
                ws[idx] = w * np.abs(vs[at][:, 0])
                cut = 17 * 2.0 ** -14 * ws.reshape(-1, 16).max(1).sum()
                sums = 2.0 ** -23 * (sc.size / 16 + 8) * (w @ (np.abs(vs[at]) * (16 + np.abs(vz[at]))))
                tol = moved + (2.0 ** -11 + 2.0 ** -18) * mag + small + cut + sums
                if form_many:  # code + zero rounded to fp16
                    tol += w @ np.abs(vs[at] * (cz.astype(np.float16) - cz))
                self.out[r, h] = out
                self.tol[r, h] = tol * (1 + eps) + eps / 2 * np.abs(out) + 2.0 ** -24
                self.lse[r, h] = top + np.log(T)
                self.tol_lse[r, h] = d + 2.0 ** -20 + 2.0 ** -21 * abs(self.lse[r, h])

    def check(self, out, lse):
        live = ~np.isnan(self.lse)
        err = np.abs(out - self.out)
        bad = ~(err <= self.tol) & live[..., None]
        assert not bad.any(), (np.argwhere(bad)[:4], err[bad][:4], self.tol[bad][:4])
        with np.errstate(invalid="ignore"):
            off = np.where(np.isneginf(self.lse), np.where(np.isneginf(lse), 0.0, np.inf), np.abs(lse - self.lse))
        bad = ~(off <= self.tol_lse) & live
        assert not bad.any(), (np.argwhere(bad)[:4], off[bad][:4], self.tol_lse[bad][:4])

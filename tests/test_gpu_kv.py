"""The paged 4-bit cache on the GPU: append, read and attention against 64-bit evaluations of the
definitions (kv_ref), at the sizes, strides, masks and lengths where they can go wrong."""

import ctypes

import numpy as np
import pytest
import torch

from kv_ref import Setup, attention64, check_attention, filled_pages, parts, quantize32, rotate64, values
from opac1ty_b200 import _lib, kv

pytestmark = pytest.mark.gpu

EPS = {torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}  # torch.finfo(t).eps
F16, BF16 = torch.float16, torch.bfloat16


def device_error(dev):
    code = ctypes.c_int32(0)
    _lib.check(_lib.load().opc_take_device_error(dev.index, ctypes.byref(code)))
    return code.value


def rows(rng, n, heads, hd, dtype, dev, mean=0.0):
    return torch.from_numpy((rng.standard_normal((n, heads, hd)) + mean).astype(np.float32)).to(dtype).to(dev)


def f64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def check_append(su, k, v, q, q_out, inv_freq, interleaved, pages_before):
    """Stored heads, turned q, and every byte that no row owns."""
    kn, vn = f64(k), f64(v)
    pages = su.cache.pages.cpu().numpy()
    kc, vc, kp, vp = (a.copy() for a in parts(pages, su.page, su.hd))
    kx, vx = values(pages, su.page, su.hd)
    want = pages_before.copy()
    wkc, wvc, wkp, wvp = parts(want, su.page, su.hd)
    owned = np.zeros((su.n_pages, su.page), dtype=bool)
    eps = EPS[k.dtype]
    for r in range(su.rows):
        p = su.place(r)
        if p is None or p[1] < 0:
            if q is not None:
                assert torch.equal(q_out[r], torch.full_like(q_out[r], 7.0))  # left as it was
            continue
        s, pos = p
        pg, off = su.block(s, pos)
        assert not owned[pg, off]
        owned[pg, off] = True
        # v: no rotation, so the fp32 definition gives the very bytes
        c, sc, z = quantize32(vn[r])
        got = np.stack([vc[pg, :, off] & 15, vc[pg, :, off] >> 4], -1).reshape(su.kv_heads, su.hd)
        assert np.array_equal(got, c)
        assert np.array_equal(vp[pg, :, off, 0], sc[:, 0].astype(np.float16)) and np.array_equal(vp[pg, :, off, 1], z[:, 0])
        # k: within half a step of the turned value, and what clamping to codes 0..15 adds: the
        # rounding of the scale moves the top by at most 15 * 2^-11 steps, that of the zero either
        # end by |zero| * 2^-11; the fp32 products add a few 2^-24 of the values
        t = rotate64(kn[r], pos, inv_freq, interleaved) if inv_freq is not None else kn[r]
        scale, zero = kp[pg, :, off, :1].astype(np.float64), kp[pg, :, off, 1:].astype(np.float64)
        tol = scale * (0.5 + (15 + np.abs(zero)) * 2.0 ** -11) + 2.0 ** -21 * np.abs(t).max(-1, keepdims=True)
        assert (np.abs(kx[pg, :, off] - t) <= tol).all()
        # the scale itself, to one rounding
        lo, hi = t.min(-1), t.max(-1)
        ref = np.maximum(np.maximum((hi - lo) / 15, np.maximum(abs(lo), abs(hi)) / 1024), 2.0 ** -24)
        assert (np.abs(scale[:, 0] - ref) <= 2.0 ** -11 * ref + 2.0 ** -22 * np.abs(t).max(-1) / 15 + 2.0 ** -25).all()
        if q is not None:
            qq = f64(q[r])
            tq = rotate64(qq, pos, inv_freq, interleaved) if inv_freq is not None else qq
            big = np.abs(qq).max(-1, keepdims=True)
            assert (np.abs(f64(q_out[r]) - tq) <= eps / 2 * np.abs(tq) + 2.0 ** -22 * big + 2.0 ** -25).all()
    keep = ~owned
    assert np.array_equal(kc[keep.nonzero()[0], :, keep.nonzero()[1]], wkc[keep.nonzero()[0], :, keep.nonzero()[1]])
    assert np.array_equal(vc[keep.nonzero()[0], :, keep.nonzero()[1]], wvc[keep.nonzero()[0], :, keep.nonzero()[1]])
    for g, w in ((kp, wkp), (vp, wvp)):
        assert np.array_equal(g[keep.nonzero()[0], :, keep.nonzero()[1]].view(np.uint16),
                              w[keep.nonzero()[0], :, keep.nonzero()[1]].view(np.uint16))


def freq(rot, theta=10000.0):
    return theta ** (-np.arange(0, rot, 2, dtype=np.float64) / rot)


@pytest.mark.parametrize("hd,page,heads,kv_heads,dtype,interleaved,rot", [
    (128, 64, 8, 2, F16, False, 128), (64, 16, 4, 4, BF16, True, 64), (32, 16, 3, 1, F16, False, 32),
    (96, 32, 6, 2, BF16, False, 96), (192, 128, 2, 2, F16, True, 192), (256, 256, 4, 1, F16, False, 256),
    (128, 16, 7, 1, F16, False, 64), (96, 16, 2, 2, F16, True, 32), (256, 16, 2, 2, BF16, False, 16),
    (64, 32, 2, 1, F16, False, 0)])
@pytest.mark.parametrize("lens", [
    ([1], [1]), ([1, 0, 3, 1], [17, 5, 3, 64]), ([5, 70, 2], [5, 133, 1])])  # the last: kv_len < q_len
def test_append_and_q(cuda_device, hd, page, heads, kv_heads, dtype, interleaved, rot, lens):
    rng = np.random.default_rng(hd + page + len(lens[0]))
    su = Setup(cuda_device, lens[0], lens[1], kv_heads, hd, page, seed=3, pad_rows=3)
    su.cache.pages.copy_(torch.from_numpy(rng.integers(0, 256, tuple(su.cache.pages.shape), dtype=np.uint8)))
    before = su.cache.pages.cpu().numpy()
    k, v, q = (rows(rng, su.rows, n, hd, dtype, cuda_device, 0.5) for n in (kv_heads, kv_heads, heads))
    rope = kv.Rope(rot, interleaved=interleaved, device=cuda_device) if rot else None
    q_out = torch.full_like(q, 7.0)
    assert kv.append(su.cache, su.batch, k, v, q=q, rope=rope, q_out=q_out) is q_out
    check_append(su, k, v, q, q_out, freq(rot) if rot else None, interleaved, before)
    assert device_error(cuda_device) == 0


def test_append_many_rows_takes_the_four_row_form(cuda_device):
    rng = np.random.default_rng(1)
    su = Setup(cuda_device, [601, 1, 333], [700, 9, 333], 2, 64, 32, seed=4, pad_rows=2)
    before = su.cache.pages.cpu().numpy()
    k, v, q = (rows(rng, su.rows, n, 64, F16, cuda_device) for n in (2, 2, 4))
    q_out = torch.full_like(q, 7.0)
    kv.append(su.cache, su.batch, k, v, q=q, rope=kv.Rope(64, device=cuda_device), q_out=q_out)
    check_append(su, k, v, q, q_out, freq(64), False, before)


@pytest.mark.parametrize("ld,off", [(6 * 64, 0), (6 * 64 + 8, 0), (6 * 64 + 3, 0), (6 * 64 + 8, 1)])
def test_append_parts_of_a_fused_row_in_place(cuda_device, ld, off):
    # q|k|v of one product: leading dimensions that are and are not multiples of 8, an odd start
    rng = np.random.default_rng(5)
    hd, su = 64, Setup(cuda_device, [2, 9], [2, 40], 1, 64, 16)
    buf = torch.from_numpy(rng.standard_normal((su.rows, ld + off)).astype(np.float32)).half().to(cuda_device)
    q, k, v = buf[:, off:off + 4 * hd], buf[:, off + 4 * hd:off + 5 * hd], buf[:, off + 5 * hd:off + 6 * hd]
    before, q0 = su.cache.pages.cpu().numpy(), q.clone()
    tail = buf[:, off + 6 * hd:].clone()
    kv.append(su.cache, su.batch, k, v, q=q, rope=kv.Rope(hd, device=cuda_device), q_out=q)
    check_append(su, k.reshape(-1, 1, hd), v.reshape(-1, 1, hd), q0.reshape(-1, 4, hd), q.reshape(-1, 4, hd), freq(hd), False, before)
    assert torch.equal(buf[:, off + 6 * hd:], tail)


def test_append_far_positions(cuda_device):
    # the angle at position 2e9 is formed without rounding; float64 gives it to 2e9 * 2^-53 radians
    rng = np.random.default_rng(6)
    page, hd, pos = 256, 64, 1_999_999_990
    cache = kv.KVCache(1, hd, 2, page, device=cuda_device)
    table = torch.full((1, (pos + 20) // page + 1), -1, dtype=torch.int32, device=cuda_device)
    table[0, pos // page:] = 1
    batch = kv.KVBatch(torch.tensor([0, 3], dtype=torch.int32, device=cuda_device),
                       torch.tensor([pos + 3], dtype=torch.int32, device=cuda_device), table, 3, 3, pos + 3)
    k, v, q = (rows(rng, 3, 1, hd, F16, cuda_device) for _ in range(3))
    out = kv.append(cache, batch, k, v, q=q, rope=kv.Rope(hd, theta=500000.0, device=cuda_device))
    for r in range(3):
        t = rotate64(f64(q[r]), pos + r, freq(hd, 500000.0), False)
        tol = 2.0 ** -11 * np.abs(t) + (2.0 ** -22 + 2e9 * 2.0 ** -52) * np.abs(f64(q[r])).max()
        assert (np.abs(f64(out[r]) - t) <= tol).all()
    assert device_error(cuda_device) == 0


def test_append_heads_of_special_values(cuda_device):
    hd, su = 32, Setup(cuda_device, [9], [9], 1, 32, 16)
    x = np.zeros((9, 1, hd), dtype=np.float32)
    x[1] = 3.25                       # constant
    x[2] = -1000.0
    x[2, 0, 5] = -1000.5              # a small spread far from 0
    x[3, 0, 0] = np.inf
    x[4, 0, 7] = np.nan
    x[5, 0, 31] = -np.inf
    x[6] = 6e-8                       # the smallest fp16 subnormal, everywhere
    x[7, 0, ::2], x[7, 0, 1::2] = 65504.0, -65504.0
    x[8, 0, 3] = 1.0                  # one value, the rest 0
    t = torch.from_numpy(x).half().to(cuda_device)
    kv.append(su.cache, su.batch, t, t)
    k, v = kv.read(su.cache, su.batch)
    assert torch.equal(k.isnan(), v.isnan())
    kn = f64(k)[:, 0]
    assert np.array_equal(np.isnan(kn).all(-1), [False, False, False, True, True, True, False, False, False])
    assert np.array_equal(kn[0], np.zeros(hd))
    xn = f64(t)[:, 0]
    pages = su.cache.pages.cpu().numpy()
    _, _, kp, _ = parts(pages, 16, hd)
    for i in (1, 2, 6, 7, 8):
        pg, off = su.block(0, i)
        s, z = (abs(float(a)) for a in kp[pg, 0, off])
        # a step, what clamping adds (see check_append), and the rounding of the read value
        tol = s * (0.5 + (15 + z) * 2.0 ** -11) + 2.0 ** -11 * np.abs(xn[i]).max() + 2.0 ** -24
        assert (np.abs(kn[i] - xn[i]) <= tol).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,page", [(32, 16), (96, 64), (128, 128), (256, 32)])
def test_read_gives_the_values(cuda_device, hd, page, dtype):
    rng = np.random.default_rng(hd)
    su = Setup(cuda_device, [1, 0, 20], [33, 0, 20], 3, hd, page, pad_rows=2)
    su.cache.pages.copy_(torch.from_numpy(filled_pages(rng, su.n_pages, 3, page, hd)))
    kx, vx = values(su.cache.pages.cpu().numpy(), page, hd)
    k = torch.full((su.rows, 3, hd), 5.0, dtype=dtype, device=cuda_device)
    v = k.clone()
    kv.read(su.cache, su.batch, k=k, v=v)
    for r in range(su.rows):
        p = su.place(r)
        for got, ref in ((k, kx), (v, vx)):
            if p is None:
                assert torch.equal(got[r], torch.full_like(got[r], 5.0))
                continue
            pg, off = su.block(*p)
            assert (np.abs(f64(got[r]) - ref[pg, :, off]) <= (EPS[dtype] / 2 + 2.0 ** -23) * np.abs(ref[pg, :, off]) + 2.0 ** -25).all()


def run_attention(su, rng, heads, dtype, dev, scale=None, mean=0.0, q_scale=1.0, pages=None):
    su.cache.pages.copy_(torch.from_numpy(filled_pages(rng, su.n_pages, su.kv_heads, su.page, su.hd, mean) if pages is None else pages))
    q = (rows(rng, su.rows, heads, su.hd, dtype, dev).float() * q_scale).to(dtype)
    out = torch.full_like(q, 9.0)
    res, lse = kv.attention(su.cache, su.batch, q, scale=scale, out=out, return_lse=True)
    ref = attention64(su, su.cache.pages.cpu().numpy(), f64(q), su.hd ** -0.5 if scale is None else scale)
    live = np.isfinite(ref[1])
    check_attention(f64(out), lse.cpu().numpy().astype(np.float64), ref, EPS[dtype], live)
    for r in range(su.rows):
        p = su.place(r)
        if p is None:
            assert torch.equal(out[r], torch.full_like(out[r], 9.0))
        elif p[1] < 0:
            assert torch.equal(out[r], torch.zeros_like(out[r])) and torch.isneginf(lse[r]).all()
    return q, out, lse


SHAPES = [  # hd, page, heads, kv_heads, type
    (128, 64, 8, 2, F16), (128, 16, 16, 2, BF16), (64, 32, 4, 4, F16), (32, 16, 3, 1, F16), (96, 16, 6, 3, BF16),
    (192, 64, 4, 2, F16), (256, 128, 8, 1, BF16), (128, 256, 7, 1, F16), (64, 16, 24, 1, F16), (256, 16, 2, 2, F16)]


@pytest.mark.parametrize("hd,page,heads,kv_heads,dtype", SHAPES)
@pytest.mark.parametrize("lens", [
    ([1], [1]), ([1, 1, 1, 1, 1], [1, 15, 16, 17, 129]), ([1, 0, 1], [0, 30, 400]), ([2, 3, 1], [2, 65, 513]),
    ([1, 1], [2000, 640])])
def test_attention_steps(cuda_device, hd, page, heads, kv_heads, dtype, lens):
    rng = np.random.default_rng(hd * 7 + page + sum(lens[1]))
    run_attention(Setup(cuda_device, lens[0], lens[1], kv_heads, hd, page, pad_rows=2), rng, heads, dtype, cuda_device)
    assert device_error(cuda_device) == 0


@pytest.mark.parametrize("hd,page,heads,kv_heads,dtype", SHAPES)
@pytest.mark.parametrize("lens", [
    ([17], [17]), ([64, 1, 0, 33], [64, 200, 7, 150]), ([130], [259]), ([9, 40], [3, 40]), ([128, 127], [128, 383])])
def test_attention_prompts(cuda_device, hd, page, heads, kv_heads, dtype, lens):
    rng = np.random.default_rng(hd * 3 + page + sum(lens[1]))
    run_attention(Setup(cuda_device, lens[0], lens[1], kv_heads, hd, page, pad_rows=1), rng, heads, dtype, cuda_device)
    assert device_error(cuda_device) == 0


@pytest.mark.parametrize("lens", [([1], [300]), ([90], [300])])
@pytest.mark.parametrize("scale,q_scale", [(0.0, 1.0), (-0.1, 1.0), (1.0, 3.0), (1e-3, 300.0), (0.088, 1e-6)])
def test_attention_scales(cuda_device, lens, scale, q_scale):
    # weights from uniform to a single one; a negative and a zero scale; large and tiny queries
    rng = np.random.default_rng(8)
    run_attention(Setup(cuda_device, lens[0], lens[1], 2, 128, 64), rng, 8, F16, cuda_device, scale=scale, q_scale=q_scale)


@pytest.mark.parametrize("lens", [([1], [700]), ([100], [700])])
@pytest.mark.parametrize("vscale", [2.0 ** -12, 300.0])
def test_attention_values_of_other_magnitudes(cuda_device, lens, vscale):
    # the weights' fp16 form must neither underflow nor overflow with the values' scales
    rng = np.random.default_rng(9)
    su = Setup(cuda_device, lens[0], lens[1], 2, 128, 64)
    pages = filled_pages(rng, su.n_pages, 2, 64, 128)
    _, _, _, vp = parts(pages, 64, 128)
    vp = vp.copy()
    ramp = np.where(np.arange(64) % 5 == 0, vscale, 1.0 if vscale > 1 else vscale / 4)
    vp[..., 0] = (vp[..., 0].astype(np.float32) * ramp).astype(np.float16)
    pages[..., 64 * 128 + 256:] = np.ascontiguousarray(vp).view(np.uint8).reshape(*pages.shape[:-1], -1)
    run_attention(su, rng, 8, F16, cuda_device, pages=pages)


@pytest.mark.parametrize("lens", [([1, 2], [37, 100]), ([20, 70], [37, 100])])
def test_attention_ignores_what_lies_past_the_end(cuda_device, lens):
    # NaN scales and zeros in unused places of the last pages, and in pages of no sequence
    rng = np.random.default_rng(10)
    su = Setup(cuda_device, lens[0], lens[1], 2, 64, 32)
    pages = filled_pages(rng, su.n_pages, 2, 32, 64)
    used = np.zeros((su.n_pages, 32), dtype=bool)
    for s, n in enumerate(su.kv_lens):
        for p in range(n):
            used[su.block(s, p)] = True
    pairs = np.ascontiguousarray(pages[..., 32 * 64:]).view(np.float16).reshape(su.n_pages, 2, 2, 32, 2)
    pairs[np.broadcast_to(~used[:, None, None, :], pairs.shape[:-1])] = np.nan
    pages[..., 32 * 64:] = pairs.view(np.uint8).reshape(su.n_pages, 2, -1)
    run_attention(su, rng, 4, F16, cuda_device, pages=pages)


@pytest.mark.parametrize("q_len,kv_len,at", [(1, 100, 40), (40, 100, 80), (130, 300, 200)])
def test_a_nan_head_reaches_only_the_rows_that_see_it(cuda_device, q_len, kv_len, at):
    rng = np.random.default_rng(11)
    su = Setup(cuda_device, [q_len], [kv_len], 2, 128, 16)
    full = kv.KVBatch(torch.tensor([0, kv_len], dtype=torch.int32, device=cuda_device), su.batch.kv_len, su.batch.page_table)
    k, v = (rows(rng, kv_len, 2, 128, F16, cuda_device) for _ in range(2))
    k[at, 0, 3] = float("nan")
    v[at, 1, 5] = float("inf")
    kv.append(su.cache, full, k, v)
    q = rows(rng, q_len, 4, 128, F16, cuda_device)
    out, lse = kv.attention(su.cache, su.batch, q, return_lse=True)
    first = max(0, at - (kv_len - q_len))  # the first row that sees it
    sees = torch.arange(q_len) >= first
    nan = out.isnan().all(-1).cpu()
    assert torch.equal(out.isnan().any(-1).cpu(), nan)
    assert torch.equal(nan, sees[:, None].expand(-1, 4))
    assert torch.equal(lse.isnan().cpu(), sees[:, None] & torch.tensor([True, True, False, False]))


def test_attention_is_deterministic_and_indifferent_to_other_sequences(cuda_device):
    rng = np.random.default_rng(12)
    su = Setup(cuda_device, [1, 1, 1], [5000, 33, 5000], 2, 128, 64)
    q, out, lse = run_attention(su, rng, 8, F16, cuda_device)
    for _ in range(3):
        again, l2 = kv.attention(su.cache, su.batch, q, return_lse=True)
        assert torch.equal(again, out) and torch.equal(l2, lse)


def test_rows_of_prompts_and_steps_agree(cuda_device):
    # a prompt appended and attended whole, in ragged chunks, and token by token
    rng = np.random.default_rng(13)
    n, hd, page = 150, 64, 16
    su = Setup(cuda_device, [n], [n], 2, hd, page)
    rope = kv.Rope(hd, device=cuda_device)
    q, k, v = (rows(rng, n, h, hd, F16, cuda_device) for h in (4, 2, 2))
    qr = kv.append(su.cache, su.batch, k, v, q=q, rope=rope)
    whole = kv.attention(su.cache, su.batch, qr)
    pages = su.cache.pages.clone()
    for cuts in ([0, 1, 2, 50, 149, 150], list(range(0, n + 1, 5)), list(range(n + 1))):
        su.cache.pages.zero_()
        for a, b in zip(cuts, cuts[1:]):
            part = kv.KVBatch(torch.tensor([0, b - a], dtype=torch.int32, device=cuda_device),
                              torch.tensor([b], dtype=torch.int32, device=cuda_device), su.batch.page_table, b - a, b - a, b)
            qp = kv.append(su.cache, part, k[a:b], v[a:b], q=q[a:b], rope=rope)
            assert torch.equal(qp, qr[a:b])
            out = kv.attention(su.cache, part, qp)
            # two results, each within its own tolerance of the exact one (check_attention)
            d = (out.float() - whole[a:b].float()).abs().max().item()
            assert d <= 2 * (2.0 ** -11 * 4 + 2.0 ** -10 * 4)
        assert torch.equal(su.cache.pages, pages)


def test_offsets_past_32_bits(cuda_device):
    # the pages in use lie beyond 4 GiB of a large cache
    rng = np.random.default_rng(14)
    hd, page, kvh = 128, 256, 8
    n_pages = (5 << 30) // (page * (hd + 8) * kvh)
    cache = kv.KVCache(kvh, hd, n_pages, page, device=cuda_device)
    n = 700
    table = torch.tensor([[n_pages - 1, n_pages - 3, n_pages - 2]], dtype=torch.int32, device=cuda_device)
    su = Setup(cuda_device, [n], [n], kvh, hd, page)
    su.table = su.table[:, :3]
    small = kv.KVBatch(su.batch.q_start, su.batch.kv_len, torch.from_numpy(np.ascontiguousarray(su.table)).to(cuda_device))
    big = kv.KVBatch(su.batch.q_start, su.batch.kv_len, table)
    k, v, q = (rows(rng, n, h, hd, F16, cuda_device) for h in (kvh, kvh, 8))
    kv.append(cache, big, k, v)
    kv.append(su.cache, small, k, v)
    for a, b in zip(kv.read(cache, big), kv.read(su.cache, small)):
        assert torch.equal(a, b)
    assert torch.equal(kv.attention(cache, big, q), kv.attention(su.cache, small, q))
    step = kv.KVBatch(torch.tensor([0, 1], dtype=torch.int32, device=cuda_device), su.batch.kv_len, table)
    step_small = kv.KVBatch(step.q_start, su.batch.kv_len, small.page_table)
    assert torch.equal(kv.attention(cache, step, q[:1]), kv.attention(su.cache, step_small, q[:1]))


def test_bad_pages_and_lengths_are_recorded_and_skipped(cuda_device):
    rng = np.random.default_rng(15)
    for bad in (-1, 99, -2**31, 2**31 - 1):
        su = Setup(cuda_device, [1, 2], [40, 50], 1, 64, 16)
        su.table[0, 2] = bad  # the page of sequence 0's new row
        batch = kv.KVBatch(su.batch.q_start, su.batch.kv_len, torch.from_numpy(su.table).to(cuda_device))
        k, v, q = (rows(rng, 3, h, 64, F16, cuda_device) for h in (1, 1, 2))
        kv.append(su.cache, batch, k, v, q=q)
        assert device_error(cuda_device) == 2
        out = kv.attention(su.cache, batch, q)
        assert device_error(cuda_device) == 2 and torch.isfinite(out).all()
    # lengths beyond the bound and beyond the table
    su = Setup(cuda_device, [1], [40], 1, 64, 16)
    k, v, q = (rows(rng, 1, h, 64, F16, cuda_device) for h in (1, 1, 2))
    for kv_len, max_kv in ((41, 40), (40 + 64, 10**6)):
        b = kv.KVBatch(su.batch.q_start, torch.tensor([kv_len], dtype=torch.int32, device=cuda_device), su.batch.page_table, 1, 1, max_kv)
        before = su.cache.pages.clone()
        kv.append(su.cache, b, k, v)
        assert device_error(cuda_device) == 2 and torch.equal(su.cache.pages, before)
    # a sequence with more rows than max_q: the others are right, the error is recorded
    su = Setup(cuda_device, [40, 1], [40, 60], 1, 64, 16)
    b = kv.KVBatch(su.batch.q_start, su.batch.kv_len, su.batch.page_table, 41, 1, 60)
    su.cache.pages.copy_(torch.from_numpy(filled_pages(rng, su.n_pages, 1, 16, 64)))
    q = rows(rng, 41, 2, 64, F16, cuda_device)
    good = kv.attention(su.cache, su.batch, q)
    assert device_error(cuda_device) == 0
    out = kv.attention(su.cache, b, q)
    assert device_error(cuda_device) == 2
    assert (out[40].float() - good[40].float()).abs().max() <= 2.0 ** -8


def test_captured_graphs_replay_with_new_lengths(cuda_device):
    rng = np.random.default_rng(16)
    n = 900
    su = Setup(cuda_device, [1, 1], [n, n], 2, 128, 64)
    su.cache.pages.copy_(torch.from_numpy(filled_pages(rng, su.n_pages, 2, 64, 128)))
    q = rows(rng, 2, 8, 128, F16, cuda_device)
    out = torch.zeros_like(q)
    lens = torch.tensor([n, n], dtype=torch.int32, device=cuda_device)
    batch = kv.KVBatch(su.batch.q_start, lens, su.batch.page_table, 2, 1, n)
    kv.attention(su.cache, batch, q, out=out)  # loads the kernels
    graphs, outs = [], []
    side = torch.cuda.Stream()
    for i in range(2):  # two graphs captured on one stream
        o = torch.zeros_like(q)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            kv.attention(su.cache, batch, q, out=o)
        graphs.append(g)
        outs.append(o)
    for a, b in ((n, 1), (64, 65), (513, n - 1)):
        lens.copy_(torch.tensor([a, b], dtype=torch.int32))
        want = kv.attention(su.cache, batch, q)
        torch.cuda.synchronize()
        s0, s1 = torch.cuda.Stream(), torch.cuda.Stream()
        for _ in range(3):  # replayed side by side: each has a workspace of its own
            with torch.cuda.stream(s0):
                graphs[0].replay()
            with torch.cuda.stream(s1):
                graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_calls_on_two_streams_at_once(cuda_device):
    rng = np.random.default_rng(17)
    su = Setup(cuda_device, [1], [4000], 4, 128, 64)
    su.cache.pages.copy_(torch.from_numpy(filled_pages(rng, su.n_pages, 4, 64, 128)))
    qs = [rows(rng, 1, 16, 128, F16, cuda_device) for _ in range(2)]
    want = [kv.attention(su.cache, su.batch, q) for q in qs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(kv.attention(su.cache, su.batch, qs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_python_refusals(cuda_device):
    su = Setup(cuda_device, [2], [10], 2, 64, 16)
    z = lambda *s, t=F16: torch.zeros(*s, dtype=t, device=cuda_device)
    k, q = z(2, 2, 64), z(2, 4, 64)
    for bad in (z(3, 2, 64), z(2, 1, 64), z(2, 2, 32), z(2, 2, 64, t=torch.float32), z(2, 2, 64, t=BF16), k.cpu(), z(2, 64, 2).transpose(1, 2)):
        with pytest.raises(ValueError):
            kv.append(su.cache, su.batch, k, bad)
    with pytest.raises(ValueError):
        kv.append(su.cache, su.batch, k, k, q_out=q)
    with pytest.raises(ValueError):
        kv.attention(su.cache, su.batch, z(1, 4, 64))
    with pytest.raises(_lib.OpcError):
        kv.attention(su.cache, su.batch, z(2, 3, 64))
    with pytest.raises(_lib.OpcError) as e:
        kv.attention(su.cache, su.batch, q, workspace=z(16, t=torch.uint8))
    assert e.value.code == _lib.OPC_ERR_WORKSPACE
    with pytest.raises(ValueError):
        kv.KVBatch(su.batch.q_start, su.batch.kv_len.long(), su.batch.page_table)
    with pytest.raises(ValueError):
        kv.KVBatch(su.batch.q_start[:1], su.batch.kv_len, su.batch.page_table)
    with pytest.raises(ValueError):
        kv.KVCache(2, 64, 3, 16, pages=z(10, t=torch.uint8))
    with pytest.raises(ValueError):
        kv.Rope(24, device=cuda_device)
    with pytest.raises(_lib.OpcError):
        kv.KVCache(2, 80, 3, 16, device=cuda_device)

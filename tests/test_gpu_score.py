"""Token log probabilities on the GPU against 64-bit evaluations of the definitions."""

import ctypes

import numpy as np
import pytest
import torch

from opac1ty_b200 import _lib
from opac1ty_b200.score import token_logprobs

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def device_error(dev):
    code = ctypes.c_int32(0)
    _lib.check(_lib.load().opc_take_device_error(dev.index, ctypes.byref(code)))
    return code.value


def reference(x, targets, k):
    """logits x float64 [rows][vocab] -> (logprob, entropy, ids, top) by the definitions."""
    rows, vocab = x.shape
    with np.errstate(all="ignore"):
        m = np.max(np.where(np.isnan(x), -np.inf, x), -1, keepdims=True)
        base = np.where(np.isneginf(m), 0.0, m)
        log_z = np.log(np.exp(x - base).sum(-1, keepdims=True))
        broken = (np.isnan(x) | np.isposinf(x)).any(-1, keepdims=True)
        lp = np.where(np.isneginf(x), -np.inf, (x - base) - log_z)  # (base alone may dwarf log_z)
        lp = np.where(broken, np.nan, lp)
        p = np.exp(lp)
        ent = -np.where(p > 0, p * lp, 0.0).sum(-1)
        ent = np.where(broken[:, 0], np.nan, ent)
    order = np.argsort(np.where(np.isnan(x), np.inf, -x), axis=-1, kind="stable")  # NaN last, ties by index
    ids = order[:, :k]
    given = np.array([0.0 if t < 0 else np.nan if t >= vocab else lp[r, t] for r, t in enumerate(targets)])
    return given, ent, ids, np.take_along_axis(lp, ids, -1)


def check(x, targets, k, res):
    xd = x.double().cpu().numpy()
    rows, vocab = xd.shape
    given, ent, ids, top = reference(xd, targets, k)
    assert np.array_equal(res.top_ids.cpu().numpy(), ids)
    # x - max and its exponential to a few 2^-24 of |x - max| (terms beyond 90 vanish: 90 * 2^-23
    # of the sum at most), sums in a tree or a short chain of fp32 additions (64 * 2^-24), the
    # logarithm to 2^-22 of its value
    span = np.minimum(np.nanmax(np.where(np.isfinite(xd), np.abs(xd), 0), -1) * 2, 90)
    d = (span * 2.0 ** -23 + 64 * 2.0 ** -24 + 2.0 ** -21 * (1 + np.log(vocab)))

    def close(got, want, tol):
        got = got.cpu().numpy().astype(np.float64)
        fin = np.isfinite(want)
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isneginf(got), np.isneginf(want))
        err = np.abs(np.where(fin, got, 0) - np.where(fin, want, 0))
        assert (err <= tol + 2.0 ** -22 * np.abs(np.where(fin, want, 0))).all(), err.max()

    if res.logprob is not None:
        close(res.logprob, given, d)
    close(res.top_logprobs, top, d[:, None])
    # entropy = log Z - sum(e * y) / Z: the second term has the size of the entropy plus log Z
    close(res.entropy, ent, 4 * d * (1 + np.log(vocab)))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (1, 5, 5), (3, 31, 7), (2, 1000, 32), (5, 4099, 20), (1, 32000, 5),
                                          (1, 128256, 20), (40, 50257, 1), (700, 260, 3), (1, 7, 0), (9, 2048, 32)])
def test_random_rows(cuda_device, dtype, rows, vocab, k):
    g = torch.Generator().manual_seed(rows * vocab + k)
    x = (torch.randn(rows, vocab, generator=g) * 3).to(dtype).to(cuda_device)
    t = torch.randint(-1, vocab, (rows,), generator=g, dtype=torch.int32)
    res = token_logprobs(x, t.to(cuda_device), top_k=k)
    check(x, t.tolist(), k, res)
    again = token_logprobs(x, t.to(cuda_device), top_k=k)
    for a, b in zip(res, again):
        assert torch.equal(a.view(torch.int32), b.view(torch.int32))
    assert device_error(cuda_device) == 0


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("rows,vocab", [(1, 9000), (3, 40000), (300, 3000)])
@pytest.mark.parametrize("kind", ["equal", "few values", "ascending", "descending", "one peak", "mostly masked", "blocks"])
def test_orders_and_ties(cuda_device, dtype, rows, vocab, kind):
    rng = np.random.default_rng(vocab)
    i = np.arange(vocab, dtype=np.float64)
    x = {"equal": np.full(vocab, 2.5), "few values": rng.integers(0, 3, vocab) * 1.0, "ascending": i / vocab * 60 - 30,
         "descending": 30 - i / vocab * 60, "one peak": np.where(i == vocab // 2, 40.0, -3.0),
         "mostly masked": np.where(rng.random(vocab) < 20 / vocab, 1.0, -np.inf),
         "blocks": np.where((i.astype(int) // 64) % 7 == 3, 5.0 + (i % 64) / 16, rng.standard_normal(vocab))}[kind]
    x = torch.from_numpy(np.stack([np.roll(x, 17 * r) for r in range(rows)])).to(dtype).to(cuda_device)
    t = list(rng.integers(0, vocab, rows))
    res = token_logprobs(x, torch.tensor(t, device=cuda_device), top_k=32)
    check(x, t, 32, res)


def test_special_rows(cuda_device):
    vocab = 777
    x = torch.randn(8, vocab, generator=torch.Generator().manual_seed(1))
    x[0] = float("-inf")
    x[1, 5:] = float("-inf")
    x[2, 100] = float("nan")
    x[3, 7] = float("inf")
    x[4] = float("nan")
    x[5] = torch.finfo(F32).min           # a mask of the type's lowest value
    x[5, 600] = 1.0
    x[6, :] = torch.where(torch.arange(vocab) % 2 == 0, 0.0, -0.0)   # signed zeros are equal
    x[7] = torch.finfo(F32).max / 4
    x = x.to(cuda_device)
    t = [3, 6, 0, 7, 1, 600, 776, 0]
    check(x, t, 12, token_logprobs(x, torch.tensor(t, device=cuda_device), top_k=12))
    h = x.half()                           # the lowest value becomes -infinity
    check(h, t, 12, token_logprobs(h, torch.tensor(t, device=cuda_device), top_k=12))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_rows_near_the_lowest_value(cuda_device, dtype):
    # masks of the lowest value beside -infinity: rows of nothing else, and few ordinary logits among them
    low, vocab = torch.finfo(dtype).min, 5000
    x = torch.full((5, vocab), low, dtype=dtype)
    x[0, ::2] = float("-inf")
    x[1, 3:4990] = float("-inf")
    x[2, 17] = -5.0
    x[3, 1000:] = float("-inf")
    x[3, 5] = low * 0.75
    x[4, ::3] = float("-inf")
    x[4, 4999] = float("nan")
    x = x.to(cuda_device)
    t = [1, 0, 17, 5, 1]
    check(x, t, 6, token_logprobs(x, torch.tensor(t, device=cuda_device), top_k=6))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows", [1, 400])
def test_one_nan_or_infinity_anywhere(cuda_device, dtype, rows):
    # in the first group of a thread, a later one, the tail, a masked region
    vocab = 20011
    base = torch.randn(rows, vocab, generator=torch.Generator().manual_seed(rows)) * 2
    base[:, 9000:12000] = float("-inf")
    for bad in (float("nan"), float("inf")):
        for at in (0, 7, 5000, 9500, 11999, 15000, 20010):
            x = base.clone().to(dtype)
            x[0, at] = bad
            x = x.to(cuda_device)
            r = token_logprobs(x, torch.full((rows,), 3, device=cuda_device), top_k=2)
            for v in (r.logprob, r.entropy, r.top_logprobs[:, 0]):
                assert v[0].isnan() and v[1:].isfinite().all()


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("ld,off", [(1003, 0), (1008, 0), (1024, 3), (1001, 1)])
def test_strides_and_alignment(cuda_device, dtype, ld, off):
    rows, vocab = 6, 1000
    buf = torch.full((rows * ld + off + 8,), 99.0, dtype=dtype, device=cuda_device)  # what lies between rows is never taken
    x = torch.as_strided(buf, (rows, vocab), (ld, 1), off)
    x.copy_(torch.randn(rows, vocab, device=cuda_device) * 2)
    t = [0, 999, 500, 1, 2, 3]
    check(x, t, 9, token_logprobs(x, torch.tensor(t, device=cuda_device), top_k=9))


def test_targets_outside_the_vocabulary(cuda_device):
    x = torch.randn(4, 100, device=cuda_device)
    r = token_logprobs(x, torch.tensor([-1, 100, 5, 2**40], device=cuda_device))
    lp = r.logprob.cpu()
    assert lp[0] == 0 and lp[1].isnan() and lp[2].isfinite() and lp[3].isnan()
    assert device_error(cuda_device) == 2


def test_parts_can_be_left_out_and_refusals(cuda_device):
    x = torch.randn(4, 100, device=cuda_device)
    r = token_logprobs(x, entropy=False)
    assert r.logprob is None and r.entropy is None and r.top_ids.shape == (4, 0)
    assert token_logprobs(x[:0], top_k=3).top_ids.shape == (0, 3)
    t = torch.zeros(4, dtype=torch.int32, device=cuda_device)
    for bad in (x.double(), x.cpu(), x[0], x.t()):
        with pytest.raises(ValueError):
            token_logprobs(bad)
    for bad in (t[:3], t.float(), t.cpu()):
        with pytest.raises(ValueError):
            token_logprobs(x, bad)
    with pytest.raises(_lib.OpcError):
        token_logprobs(x, top_k=33)
    with pytest.raises(_lib.OpcError):
        token_logprobs(x[:, :3], top_k=4)


def test_offsets_past_32_bits(cuda_device):
    # rows whose first element lies beyond 2^32 elements
    ld, rows, vocab = 1 << 31, 3, 5000
    buf = torch.empty(2 * ld + vocab, dtype=F16, device=cuda_device)
    x = torch.as_strided(buf, (rows, vocab), (ld, 1))
    x.copy_(torch.randn(rows, vocab, device=cuda_device))
    t = [1, 2, 3]
    check(x, t, 4, token_logprobs(x, torch.tensor(t, device=cuda_device), top_k=4))


def test_captured_graph_replays_on_new_logits(cuda_device):
    x = torch.randn(2, 9000, device=cuda_device).half()
    t = torch.tensor([5, 6], dtype=torch.int32, device=cuda_device)
    token_logprobs(x, t, top_k=4)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = token_logprobs(x, t, top_k=4)
    for seed in range(3):
        x.copy_(torch.randn(2, 9000, generator=torch.Generator().manual_seed(seed)))
        g.replay()
        torch.cuda.synchronize()
        check(x, t.tolist(), 4, r)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("ld,off", [(50003, 0), (50001, 1), (50008, 3)])
def test_few_long_rows_in_strided_logits(cuda_device, dtype, ld, off):
    """Rows of 50001 with odd strides and starts, few enough to be divided over CTAs."""
    flat = torch.randn(3 * ld + 8, generator=torch.Generator().manual_seed(ld)).mul(3).to(dtype).to(cuda_device)
    x = flat.as_strided((3, 50001), (ld, 1), off)
    t = [0, 50000, 777]
    check(x, t, 32, token_logprobs(x, torch.tensor(t, dtype=torch.int32, device=cuda_device), top_k=32))


def test_calls_on_two_streams_at_once(cuda_device):
    xs = [torch.randn(2, 60000, generator=torch.Generator().manual_seed(i)).half().to(cuda_device) for i in range(2)]
    t = torch.tensor([3, 4], dtype=torch.int32, device=cuda_device)
    want = [token_logprobs(x, t, top_k=9) for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(token_logprobs(xs[i], t, top_k=9))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert torch.equal(r.logprob, want[i].logprob) and torch.equal(r.top_ids, want[i].top_ids)
            assert torch.equal(r.entropy, want[i].entropy) and torch.equal(r.top_logprobs, want[i].top_logprobs)

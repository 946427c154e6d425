"""Attention over keys far from 0, whose zeros are hundreds of steps: the scores carry every bit of the keys
(in the form for prompts as code - 8 and a product of the zeros with the sum of q, in parts).  Rows that
see one key, or few, show a score as their log sum.  Without a GPU: that the bound notices rounded keys
and dropped parts."""

import numpy as np
import pytest
import torch

from kv_exact import Exact, heads_of
from kv_ref import Setup, filled_pages
from opac1ty_b200 import kv
from test_gpu_kv import BF16, EPS, F16, device_error, f64

HD, HEADS, KVH, PAGE, MEANS = 128, 8, 2, 32, [0.0, 20.0, 60.0, -300.0]


class Host(Setup):
    """What the 64-bit evaluation needs of a batch, without a device."""

    def __init__(self, q_len, kv_len, kv_heads, hd, page):
        self.q_lens, self.kv_lens, self.kv_heads, self.hd, self.page = [q_len], [kv_len], kv_heads, hd, page
        self.starts = np.array([0, q_len])
        self.n_pages = -(-kv_len // page)
        self.table = np.arange(self.n_pages, dtype=np.int32)[None]


def queries(rng, n, dtype):
    # (a mean gives sum q its largest size)
    return torch.from_numpy((rng.standard_normal((n, HEADS, HD)) + 0.5).astype(np.float32)).to(dtype)


def high11(x):
    return (x.astype(np.float32).view(np.uint32) & np.uint32(0xffffe000)).view(np.float32).astype(np.float64)


@pytest.mark.parametrize("mean", [20.0, 60.0])  # (below 0 code + zero and zero + 8 fit fp16 and 11 bits: nothing is lost)
@pytest.mark.parametrize("wrong", ["rounded keys", "one part of sum q", "one part of the zeros"])
def test_the_bound_notices_lost_bits(mean, wrong):
    rng = np.random.default_rng(int(abs(mean)))
    n = 40
    su = Host(n, n, KVH, HD, PAGE)
    pages = filled_pages(rng, su.n_pages, KVH, PAGE, HD, mean)
    q = f64(queries(rng, n, F16))
    ref = Exact(su, pages, q, HD ** -0.5, EPS[F16])
    (s, z, c), _ = heads_of(pages, PAGE, HD)
    over = 0
    for h in range(HEADS):  # row 0 sees key 0 alone, row 1 keys 0 and 1, ...
        for r in range(n):
            idx = np.arange(r + 1)
            at = (su.table[0, idx // PAGE], h // (HEADS // KVH), idx % PAGE)
            if wrong == "rounded keys":
                sc = s[at][:, 0] * ((c[at] + z[at]).astype(np.float16).astype(np.float64) @ q[r, h])
            else:
                total, zero = q[r, h].sum(), z[at][:, 0] + 8
                if wrong == "one part of sum q":
                    total = high11(np.array([total]))[0]
                else:
                    zero = high11(zero)
                sc = s[at][:, 0] * ((c[at] - 8) @ q[r, h] + zero * total)
            sc = sc * HD ** -0.5
            lse = sc.max() + np.log(np.exp(sc - sc.max()).sum())
            over += abs(lse - ref.lse[r, h]) > ref.tol_lse[r, h]
    assert over > 5, over


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("mean", MEANS)
@pytest.mark.parametrize("q_lens,kv_lens", [([40], [40]), ([300], [300]), ([40], [1500]), ([1, 1, 2, 1], [1, 2, 3, 700])])
def test_keys_far_from_zero(cuda_device, q_lens, kv_lens, mean, dtype):
    rng = np.random.default_rng(int(abs(mean)) + sum(kv_lens))
    su = Setup(cuda_device, q_lens, kv_lens, KVH, HD, PAGE)
    pages = filled_pages(rng, su.n_pages, KVH, PAGE, HD, mean)
    su.cache.pages.copy_(torch.from_numpy(pages))
    q = queries(rng, su.rows, dtype).to(cuda_device)
    out, lse = kv.attention(su.cache, su.batch, q, return_lse=True)
    Exact(su, pages, f64(q), HD ** -0.5, EPS[dtype]).check(f64(out), f64(lse))
    assert device_error(cuda_device) == 0

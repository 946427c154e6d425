"""Attention of queries of very different sizes in one call: every row's result is its own, whatever
the rows beside it hold."""

import numpy as np
import pytest
import torch

from kv_exact import Exact
from kv_ref import Setup, filled_pages
from opac1ty_b200 import kv
from test_gpu_kv import BF16, EPS, F16, device_error, f64, rows

pytestmark = pytest.mark.gpu

LENS = [([1, 3], [300, 200]), ([40], [70]), ([150, 60], [300, 60]), ([40], [1500])]


def run(su, dev, q, pages, scale=None, many=None):
    scale = su.hd ** -0.5 if scale is None else scale
    su.cache.pages.copy_(torch.from_numpy(pages))
    out, lse = kv.attention(su.cache, su.batch, q, scale=scale, return_lse=True)
    ref = Exact(su, pages, f64(q), scale, EPS[q.dtype], many)
    ref.check(f64(out), f64(lse))
    odd = ~torch.isfinite(q.float()).all(-1)
    assert torch.equal(out.isnan().all(-1), odd) and torch.equal(out.isnan().any(-1), odd)
    assert torch.equal(lse.isnan(), odd)
    assert device_error(dev) == 0
    return out, lse


@pytest.mark.parametrize("hd,page,heads,kv_heads", [(128, 64, 8, 2), (64, 32, 4, 1), (96, 16, 3, 1), (256, 64, 2, 1)])
@pytest.mark.parametrize("q_lens,kv_lens", LENS)
@pytest.mark.parametrize("kind", ["inf", "nan", "large", "small", "all"])
def test_rows_beside_odd_bf16_queries(cuda_device, hd, page, heads, kv_heads, q_lens, kv_lens, kind):
    rng = np.random.default_rng(hd + sum(kv_lens))
    su = Setup(cuda_device, q_lens, kv_lens, kv_heads, hd, page)
    pages = filled_pages(rng, su.n_pages, kv_heads, page, hd)
    q = rows(rng, su.rows, heads, hd, BF16, cuda_device)
    last = su.rows - 1
    if kind in ("inf", "all"):
        q[0, 0, 3] = float("inf")
        q[last, 1, hd - 1] = float("-inf")
    if kind in ("nan", "all"):
        q[last // 2, 0, 7] = float("nan")
    if kind in ("large", "all"):
        q[1, 1] *= 1e30
        q[last, 0] *= 2.0 ** 20
    if kind in ("small", "all"):
        q[2, 0] *= 1e-30
        q[2, 1] = 0.0
        q[last, heads - 1] *= 2.0 ** -20
    run(su, cuda_device, q, pages)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,heads,kv_heads", [(128, 8, 2), (64, 3, 1), (256, 4, 1)])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 2, 1], [1, 2, 3, 300]), ([40], [40])])
@pytest.mark.parametrize("small", [2.0 ** -12, 2.0 ** -14, 2.0 ** -18])
def test_tiny_queries_and_a_large_scale(cuda_device, hd, heads, kv_heads, q_lens, kv_lens, dtype, small):
    # Scores of ordinary size from queries near fp16's smallest; rows that see one key show a score as
    # their log sum.
    rng = np.random.default_rng(hd + int(1 / small))
    su = Setup(cuda_device, q_lens, kv_lens, kv_heads, hd, 32)
    q = (rows(rng, su.rows, heads, hd, torch.float32, cuda_device) * small).to(dtype)
    run(su, cuda_device, q, filled_pages(rng, su.n_pages, kv_heads, 32, hd), scale=hd ** -0.5 / small)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,heads,kv_heads", [(128, 8, 2), (64, 3, 1), (256, 4, 1)])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 2, 1], [1, 2, 300, 4000]), ([40], [40]), ([40], [1500])])
@pytest.mark.parametrize("scale", [1e6, 1e31])
def test_scores_far_below_zero(cuda_device, hd, heads, kv_heads, q_lens, kv_lens, dtype, scale):
    # every score of a row is hugely negative, and the largest of them takes all of the weight
    rng = np.random.default_rng(hd + sum(kv_lens))
    su = Setup(cuda_device, q_lens, kv_lens, kv_heads, hd, 32)
    q = rows(rng, su.rows, heads, hd, dtype, cuda_device, mean=-0.5)
    run(su, cuda_device, q, filled_pages(rng, su.n_pages, kv_heads, 32, hd, mean=1.0), scale=scale)

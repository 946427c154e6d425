"""Attention over tables that do not name every page: the keys of such a page take no part, in the
form for steps and in the one for prompts."""

import numpy as np
import pytest
import torch

from kv_exact import Exact
from kv_ref import Setup, filled_pages
from opac1ty_b200 import kv
from test_gpu_kv import BF16, EPS, F16, device_error, f64, rows

pytestmark = pytest.mark.gpu

BAD = [-1, 2**31 - 1, -2**31, 100000]


@pytest.mark.parametrize("hd,page,heads,kv_heads,dtype", [
    (128, 64, 8, 2, F16), (64, 16, 4, 1, BF16), (128, 256, 4, 1, BF16), (256, 32, 2, 1, F16), (96, 128, 3, 3, F16)])
@pytest.mark.parametrize("q_lens,kv_lens,holes", [
    ([1, 2], [700, 300], [(0, 0), (1, 50)]),             # steps, the first page among them
    ([40], [40], [(0, 0)]),                              # a prompt whose first rows see nothing
    ([70, 33], [700, 500], [(0, 0), (0, 130), (0, 699), (1, 300)]),  # prompts, keys split over CTAs
    ([300, 1], [600, 90], [(0, 10), (0, 320), (0, 599), (1, 89)]),   # both forms; pages in masked tiles
    ([64], [1500], [(0, p) for p in range(256, 1500)])])  # whole splits without a key
def test_keys_of_missing_pages_take_no_part(cuda_device, hd, page, heads, kv_heads, dtype, q_lens, kv_lens, holes):
    rng = np.random.default_rng(hd + page + sum(kv_lens))
    su = Setup(cuda_device, q_lens, kv_lens, kv_heads, hd, page, pad_rows=1)
    for i, (s, pos) in enumerate(holes):
        su.table[s, pos // page] = BAD[i % len(BAD)]
    batch = kv.KVBatch(su.batch.q_start, su.batch.kv_len, torch.from_numpy(su.table).to(cuda_device),
                       n_tokens=su.rows, max_q=max(q_lens), max_kv=max(kv_lens))
    # keys around 1 and queries around -0.5: scores far below 0, which a key of score 0 would dominate
    pages = filled_pages(rng, su.n_pages, kv_heads, page, hd, mean=1.0)
    su.cache.pages.copy_(torch.from_numpy(pages))
    q = rows(rng, su.rows, heads, hd, dtype, cuda_device, mean=-0.5)
    out, lse = kv.attention(su.cache, batch, q, return_lse=True)
    assert device_error(cuda_device) == 2
    Exact(su, pages, f64(q), hd ** -0.5, EPS[dtype]).check(f64(out), f64(lse))

"""Attention rows in which one key with a value of 0 has nearly all of the weight: the result is what the
many others give, each with a weight below the half step of fp16's smallest number."""

import numpy as np
import pytest
import torch

from opac1ty_b200 import kv
from test_gpu_kv import BF16, EPS, F16, device_error, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hd,group", [(128, 4), (64, 1), (256, 2)])
@pytest.mark.parametrize("q_len", [1, 40])
@pytest.mark.parametrize("at", [0, 4500])
def test_many_small_weights_beside_one_large(cuda_device, hd, group, q_len, at, dtype):
    # 20 sequences over the same pages, 40 kv heads: as many items as leave none split into many
    rng = np.random.default_rng(hd + q_len)
    n, bits, seqs, kvh, page = 8192, 26, 20, 40, 64
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda_device)
    cache = kv.KVCache(kvh, hd, n // page, page, device=cuda_device)
    table = torch.arange(n // page, dtype=torch.int32, device=cuda_device)[None]
    one = kv.KVBatch(i32([0, n]), i32([n]), table, n, n, n)
    # keys of 0, one whose score lies 2^26 above them; values around 1
    k = torch.zeros(n, kvh, hd, dtype=F16, device=cuda_device)
    k[at] = bits * np.log(2.0) / hd ** 0.5
    v = (rows(rng, n, kvh, hd, torch.float32, cuda_device) * 0.01 + 1).to(F16)
    v[at] = 0
    kv.append(cache, one, k, v)
    kx, vx = kv.read(cache, one, torch.bfloat16, k=k.clone(), v=v.clone())
    batch = kv.KVBatch(i32([q_len * s for s in range(seqs + 1)]), i32([n] * seqs), table.repeat(seqs, 1), q_len * seqs, q_len, n)
    q = torch.ones(q_len * seqs, kvh * group, hd, dtype=dtype, device=cuda_device)
    out = kv.attention(cache, batch, q).double()
    # the weights in 64 bits, from the keys as stored: p beside 1
    p = torch.exp(-kx[at].double().sum(-1) * hd ** -0.5)[:, None]
    first = n - q_len  # the rows' own positions differ by less than the tolerance: q_len / n of the sum
    want = (p * vx.double().sum(0) / (1 + (n - 1) * p)).repeat_interleave(group, 0)
    # The reference puts the largest weight at 2^5, times at least half of the scales' power of two: p is 2^-22
    # there at least, rounded by 2^-25 at most.  And the result's rounding.
    tol = 2.0 ** -3 + q_len / first + EPS[dtype] + 2.0 ** -7
    assert ((out / want - 1).abs() <= tol).all(), (out / want).aminmax()
    assert device_error(cuda_device) == 0

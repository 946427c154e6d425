"""The workspace of attention between calls: its counts are zero whatever ran, in both forms."""

import numpy as np
import pytest
import torch

from kv_ref import Setup, filled_pages
from opac1ty_b200 import kv
from test_gpu_kv import F16, device_error, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q_lens,kv_lens", [([1], [9000]), ([1] * 7, [5000, 1, 0, 300, 2000, 129, 777]), ([60], [3000]), ([1, 200, 3], [2000, 900, 40])])
def test_counts_are_zero_between_calls(cuda_device, q_lens, kv_lens):
    rng = np.random.default_rng(len(q_lens))
    su = Setup(cuda_device, q_lens, kv_lens, 2, 128, 64)
    su.cache.pages.copy_(torch.from_numpy(filled_pages(rng, su.n_pages, 2, 64, 128)))
    q = rows(rng, su.rows, 8, 128, F16, cuda_device)
    ws = torch.zeros(kv.attention_workspace_bytes(su.cache, su.batch, 8), dtype=torch.uint8, device=cuda_device)
    want = kv.attention(su.cache, su.batch, q, workspace=ws)
    for _ in range(3):
        assert not ws[:4096].any()
        assert torch.equal(kv.attention(su.cache, su.batch, q, workspace=ws), want)
    assert device_error(cuda_device) == 0

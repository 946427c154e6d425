"""Batches of many sequences and long ones, in both of the attention's forms at once, and the paged
cache's calls and the token log probabilities in one captured run."""

import numpy as np
import pytest
import torch

from kv_ref import Setup, attention64, check_attention, filled_pages
from opac1ty_b200 import kv
from opac1ty_b200.score import token_logprobs
from test_gpu_kv import BF16, F16, device_error, f64, rows, run_attention
from test_gpu_score import check as check_logprobs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [32, 33, 64, 65, 300])
@pytest.mark.parametrize("hd,page,heads,kv_heads,dtype", [(64, 16, 4, 2, F16), (128, 32, 8, 1, BF16), (256, 64, 2, 2, F16)])
def test_many_sequences_of_one_row(cuda_device, n, hd, page, heads, kv_heads, dtype):
    """Lengths from 0 to 300, some sequences without rows: the table of lengths takes several passes of a warp."""
    rng = np.random.default_rng(n + hd)
    q_lens = [int(i % 7 != 3) for i in range(n)]
    kv_lens = [int(v) for v in rng.integers(0, 300, size=n)]
    run_attention(Setup(cuda_device, q_lens, kv_lens, kv_heads, hd, page, pad_rows=3), rng, heads, dtype, cuda_device)
    assert device_error(cuda_device) == 0


@pytest.mark.parametrize("hd,page,heads,kv_heads,dtype", [(64, 16, 4, 2, F16), (128, 64, 8, 2, BF16), (128, 16, 16, 1, F16), (256, 32, 4, 2, F16)])
def test_steps_and_prompts_in_one_batch(cuda_device, hd, page, heads, kv_heads, dtype):
    """Sequences on both sides of the bound between the forms, interleaved; the lengths are unknown to the host."""
    rng = np.random.default_rng(hd + page)
    q_lens = [1, 40, 2, 0, 3, 70, 4, 1, 5, 8, 9, 16, 17, 1]
    kv_lens = [500, 40, 130, 20, 3, 333, 4, 0, 700, 8, 1000, 16, 100, 1]
    run_attention(Setup(cuda_device, q_lens, kv_lens, kv_heads, hd, page, pad_rows=2), rng, heads, dtype, cuda_device)
    assert device_error(cuda_device) == 0


def test_many_sequences_of_both_forms(cuda_device):
    rng = np.random.default_rng(3)
    q_lens = [int(v) for v in rng.choice([0, 1, 1, 1, 2, 5, 30], size=150)]
    kv_lens = [max(int(v), q) if i % 9 else int(v) % 20 for i, (v, q) in enumerate(zip(rng.integers(0, 200, size=150), q_lens))]
    run_attention(Setup(cuda_device, q_lens, kv_lens, 1, 64, 32, pad_rows=1), rng, 4, F16, cuda_device)
    assert device_error(cuda_device) == 0


@pytest.mark.parametrize("hd,heads,n,q_len", [(32, 4, 60001, 1), (64, 8, 60000, 1), (128, 8, 60033, 1), (128, 8, 33000, 2),
                                              (192, 8, 30000, 1), (256, 7, 30001, 1)])
def test_one_long_sequence_over_every_multiprocessor(cuda_device, hd, heads, n, q_len):
    """One kv head: its keys are cut over all CTAs, whose records are merged in several rounds."""
    rng = np.random.default_rng(n)
    page = 256
    one = filled_pages(rng, 8, 1, page, hd)
    su = Setup(cuda_device, [q_len], [n], 1, hd, page)
    pages = one[rng.integers(0, 8, size=su.n_pages)]
    run_attention(su, rng, heads, F16, cuda_device, q_scale=2.0, pages=pages)


@pytest.mark.parametrize("hd,heads,dtype", [(32, 1, F16), (64, 4, BF16), (96, 2, F16), (128, 8, F16), (192, 3, F16), (256, 2, BF16)])
@pytest.mark.parametrize("q_len,n", [(40, 1500), (18, 5003), (129, 2049), (257, 900)])
def test_prompts_split_over_their_keys(cuda_device, hd, heads, dtype, q_len, n):
    """Few tiles of rows: several CTAs share a tile's keys, and rows end inside different ones."""
    rng = np.random.default_rng(hd + n)
    run_attention(Setup(cuda_device, [q_len], [n], 1, hd, 64, pad_rows=1), rng, heads, dtype, cuda_device)


@pytest.mark.parametrize("q_lens", [[1, 1, 1], [30, 40, 20]])
def test_lengths_below_zero_and_below_the_rows(cuda_device, q_lens):
    """Nothing is stored or attended at negative positions, and nothing is recorded as an error."""
    rng = np.random.default_rng(6)
    su = Setup(cuda_device, q_lens, [-5, 25, 0], 2, 64, 16)
    run_attention(su, rng, 4, F16, cuda_device)
    before = su.cache.pages.clone()
    k, v = (rows(rng, su.rows, 2, 64, F16, cuda_device) for _ in range(2))
    kv.append(su.cache, su.batch, k, v)
    changed = {(p, i) for p, i in zip(*np.nonzero((su.cache.pages != before).any(-1).cpu().numpy()))}
    assert {p for p, _ in changed} <= set(su.table[1, :2].tolist())  # only the middle sequence stores anything
    assert device_error(cuda_device) == 0


def test_a_step_captured_from_append_to_log_probabilities(cuda_device):
    """Append, attend, a head and the log probabilities as one graph, replayed over growing lengths."""
    rng = np.random.default_rng(21)
    hd, heads, kvh, vocab, page = 64, 8, 2, 5003, 16
    start = [5, 200, 31]
    steps = 20
    su = Setup(cuda_device, [1, 1, 1], [s + steps for s in start], kvh, hd, page)
    su.cache.pages.copy_(torch.from_numpy(filled_pages(rng, su.n_pages, kvh, page, hd)))
    pages0 = su.cache.pages.clone()
    rope = kv.Rope(hd, device=cuda_device)
    head = (torch.randn(heads * hd, vocab, generator=torch.Generator().manual_seed(1)) * 0.2).half().to(cuda_device)
    qkv = torch.zeros(3, (heads + 2 * kvh) * hd, dtype=F16, device=cuda_device)
    target = torch.zeros(3, dtype=torch.int32, device=cuda_device)
    lens = torch.tensor(start, dtype=torch.int32, device=cuda_device)
    batch = kv.KVBatch(su.batch.q_start, lens, su.batch.page_table, 3, 1, max(start) + steps)

    def step():
        q, k, v = qkv.split([heads * hd, kvh * hd, kvh * hd], 1)
        qr = kv.append(su.cache, batch, k.unflatten(1, (kvh, hd)), v.unflatten(1, (kvh, hd)), q=q.unflatten(1, (heads, hd)), rope=rope)
        out = kv.attention(su.cache, batch, qr)
        logits = out.flatten(1) @ head
        return qr, out, logits, token_logprobs(logits, target, top_k=6)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    su.cache.pages.copy_(pages0)
    for i in range(steps):
        qkv.copy_(torch.from_numpy(rng.standard_normal(qkv.shape).astype(np.float16)))
        target.copy_(torch.from_numpy(rng.integers(0, vocab, size=3).astype(np.int32)))
        lens.copy_(torch.tensor([s + i + 1 for s in start], dtype=torch.int32))
        graph.replay()
        qr, out, logits, res = [t.clone() if torch.is_tensor(t) else t for t in got]
        check_logprobs(logits, target.tolist(), 6, res)
        if i in (0, 7, steps - 1):
            now = Setup(cuda_device, [1, 1, 1], [s + i + 1 for s in start], kvh, hd, page)
            now.table = su.table
            ref = attention64(now, su.cache.pages.cpu().numpy(), f64(qr), hd ** -0.5)
            check_attention(f64(out), None, ref, torch.finfo(F16).eps)
        pages = su.cache.pages.clone()
        again = step()  # the same step, eagerly: the same bits, and the cache as the replay left it
        assert torch.equal(again[1], out) and torch.equal(su.cache.pages, pages)
        assert torch.equal(again[3].logprob, res.logprob) and torch.equal(again[3].top_ids, res.top_ids)
    assert device_error(cuda_device) == 0


@pytest.mark.parametrize("hd,heads", [(64, 4), (128, 16), (256, 2)])
@pytest.mark.parametrize("q_len", [0, 1, 2, 20])
def test_a_padded_batch_of_one_sequence(cuda_device, hd, heads, q_len):
    """Bounds for 40 rows, as a captured graph has them, and fewer in use: the form is chosen by the bounds."""
    rng = np.random.default_rng(hd + q_len)
    su = Setup(cuda_device, [q_len], [700], 1, hd, 32, pad_rows=40 - q_len)
    su.batch = kv.KVBatch(su.batch.q_start, su.batch.kv_len, su.batch.page_table, n_tokens=40, max_q=40, max_kv=1000)
    su.rounded = True
    q, out, lse = run_attention(su, rng, heads, F16, cuda_device)
    assert device_error(cuda_device) == 0


def test_refusals_of_workspaces_and_tables(cuda_device):
    """A workspace elsewhere and a table whose rows overlap are refused before anything is launched."""
    su = Setup(cuda_device, [1, 1], [10, 20], 1, 64, 16)
    q = torch.zeros(2, 2, 64, dtype=F16, device=cuda_device)
    need = kv.attention_workspace_bytes(su.cache, su.batch, 2)
    for ws in (torch.zeros(need, dtype=torch.uint8), torch.zeros(need, dtype=torch.float32, device=cuda_device),
               torch.zeros(2 * need, dtype=torch.uint8, device=cuda_device)[::2]):
        with pytest.raises(ValueError, match="workspace"):
            kv.attention(su.cache, su.batch, q, workspace=ws)
        with pytest.raises(ValueError, match="workspace"):
            token_logprobs(q[:, 0], workspace=ws)
    with pytest.raises(ValueError, match="overlap"):
        kv.KVBatch(su.batch.q_start, su.batch.kv_len, su.batch.page_table[:1].expand(2, -1))


def test_attention_in_place_of_its_queries(cuda_device):
    """out may be q: every CTA of an item has read its rows before the item's result is written."""
    rng = np.random.default_rng(31)
    su = Setup(cuda_device, [1, 60, 2], [4000, 2000, 300], 2, 128, 64)
    q, out, lse = run_attention(su, rng, 8, F16, cuda_device)
    for _ in range(3):
        x = q.clone()
        kv.attention(su.cache, su.batch, x, out=x)
        assert torch.equal(x, out)

"""The host side of the paged 4-bit cache and the log probabilities, without a GPU: sizes, the
rotation's fixed-point frequencies, and every refusal of the C entry points (checked before any
device is touched)."""

import ctypes
import math
from fractions import Fraction

import numpy as np
import pytest

from opac1ty_b200 import _lib


def plan(kv_heads=2, head_dim=64, page_size=16, n_pages=3):
    c = _lib.KvCache()
    rc = _lib.load().opc_kv_plan(kv_heads, head_dim, page_size, n_pages, ctypes.byref(c))
    return rc, c


@pytest.mark.parametrize("hd", [32, 64, 96, 128, 192, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_plan_sizes(hd, page):
    rc, c = plan(5, hd, page, 7)
    assert rc == _lib.OPC_OK
    assert c.head_bytes == page * (hd + 8) and c.head_bytes % 16 == 0
    assert c.total_bytes == 7 * 5 * c.head_bytes


def test_plan_of_a_cache_past_32_bits():
    rc, c = plan(64, 256, 256, 1 << 20)
    assert rc == _lib.OPC_OK and c.total_bytes == (1 << 20) * 64 * 256 * 264


@pytest.mark.parametrize("kw,code", [
    (dict(head_dim=80), _lib.OPC_ERR_UNSUPPORTED), (dict(head_dim=0), _lib.OPC_ERR_UNSUPPORTED),
    (dict(head_dim=512), _lib.OPC_ERR_UNSUPPORTED), (dict(page_size=8), _lib.OPC_ERR_UNSUPPORTED),
    (dict(page_size=48), _lib.OPC_ERR_UNSUPPORTED), (dict(page_size=512), _lib.OPC_ERR_UNSUPPORTED),
    (dict(kv_heads=0), _lib.OPC_ERR_INVALID), (dict(n_pages=0), _lib.OPC_ERR_INVALID),
    (dict(kv_heads=70000), _lib.OPC_ERR_INVALID)])
def test_plan_refuses(kw, code):
    assert plan(**kw)[0] == code
    assert "opc_kv_plan" in _lib.last_error()


def test_rope_turns_are_exact_fractions_of_a_turn():
    f = np.concatenate([500000.0 ** (-np.arange(0, 128, 2) / 128), [0.0, 1.0, 2 * math.pi, 7.5, -1.0]])
    out = np.zeros(f.size, dtype=np.uint64)
    assert _lib.load().opc_rope_turns(f.ctypes.data, f.size, out.ctypes.data) == _lib.OPC_OK
    # 2 pi to 60 digits
    two_pi = Fraction("6.283185307179586476925286766559005768394338798750211641949889")
    for x, u in zip(f, out):
        t = Fraction(float(x)) / two_pi
        t -= math.floor(t)
        d = abs(Fraction(int(u), 1 << 64) - t)
        d = min(d, 1 - d)
        # the quotient's rounding in a 64-bit mantissa, at most 2^-64 of the turns before the modulo
        assert d <= (1 + abs(Fraction(float(x)))) * Fraction(1, 1 << 63)


def test_rope_turns_refuses():
    lib = _lib.load()
    f, u = np.array([np.inf]), np.zeros(1, dtype=np.uint64)
    assert lib.opc_rope_turns(f.ctypes.data, 1, u.ctypes.data) == _lib.OPC_ERR_INVALID
    assert lib.opc_rope_turns(None, 1, u.ctypes.data) == _lib.OPC_ERR_INVALID
    assert lib.opc_rope_turns(f.ctypes.data, -1, u.ctypes.data) == _lib.OPC_ERR_INVALID


P = 1 << 20  # an aligned stand-in for a device address: nothing below reads it


def batch(**kw):
    d = dict(n_seqs=2, n_tokens=4, max_q=2, max_kv=40, q_start=P, kv_len=P, page_table=P, table_stride=3, max_pages=3)
    d.update(kw)
    return _lib.KvBatch(**d)


def cache(**kw):
    _, c = plan()
    c.pages = P
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def call_append(c=None, b=None, heads=4, dtype=_lib.OPC_F16, rope=None, k=P, ldk=128, v=P, ldv=128, q=P, ldq=256, qo=P,
                ldo=256):
    c, b = cache() if c is None else c, batch() if b is None else b
    r = ctypes.byref(rope) if rope is not None else None
    return _lib.load().opc_kv_append(ctypes.byref(c), ctypes.byref(b), heads, dtype, r, k, ldk, v, ldv, q, ldq, qo, ldo, None)


INVALID, UNSUPPORTED = _lib.OPC_ERR_INVALID, _lib.OPC_ERR_UNSUPPORTED


@pytest.mark.parametrize("kw,code", [
    (dict(c=cache(pages=None)), INVALID), (dict(c=cache(pages=P + 4)), INVALID), (dict(c=cache(head_dim=80)), INVALID),
    (dict(c=cache(head_bytes=17)), INVALID), (dict(c=cache(total_bytes=1)), INVALID),
    (dict(b=batch(n_seqs=-1)), INVALID), (dict(b=batch(n_tokens=-1)), INVALID), (dict(b=batch(max_kv=-1)), INVALID),
    (dict(b=batch(n_seqs=70000)), INVALID), (dict(b=batch(table_stride=2)), INVALID), (dict(b=batch(q_start=None)), INVALID),
    (dict(b=batch(kv_len=None)), INVALID), (dict(b=batch(page_table=None)), INVALID),
    (dict(dtype=_lib.OPC_F32), UNSUPPORTED), (dict(dtype=7), UNSUPPORTED), (dict(heads=-1), INVALID), (dict(heads=0), INVALID),
    (dict(q=None), INVALID), (dict(qo=None), INVALID), (dict(k=None), INVALID), (dict(v=None), INVALID),
    (dict(k=P + 1), INVALID), (dict(ldk=127), INVALID), (dict(ldv=1), INVALID), (dict(ldq=255), INVALID), (dict(ldo=0), INVALID),
    (dict(rope=_lib.Rope(rot_dim=24, turns=P)), UNSUPPORTED), (dict(rope=_lib.Rope(rot_dim=128, turns=P)), UNSUPPORTED),
    (dict(rope=_lib.Rope(rot_dim=64, turns=None)), INVALID), (dict(rope=_lib.Rope(rot_dim=64, turns=P + 4)), INVALID)])
def test_append_refuses(kw, code):
    assert call_append(**kw) == code
    assert "opc_kv_append" in _lib.last_error()


def test_empty_batches_are_done_without_a_device():
    assert call_append(b=batch(n_tokens=0, q_start=None, kv_len=None, page_table=None)) == _lib.OPC_OK
    assert call_append(b=batch(n_seqs=0, q_start=None, kv_len=None, page_table=None)) == _lib.OPC_OK
    lib = _lib.load()
    assert lib.opc_kv_read(ctypes.byref(cache()), ctypes.byref(batch(n_tokens=0)), 0, None, 0, None, 0, None) == _lib.OPC_OK
    assert lib.opc_kv_attention(ctypes.byref(cache()), ctypes.byref(batch(n_seqs=0)), 4, 0, 1.0, None, 0, None, 0, None, None,
                                0, None) == _lib.OPC_OK
    assert lib.opc_token_logprobs(None, 0, 0, 0, 5, None, None, None, 0, None, None, None, 0, None) == _lib.OPC_OK


@pytest.mark.parametrize("kw,code", [
    (dict(k=None), INVALID), (dict(v=None), INVALID), (dict(ldk=10), INVALID), (dict(dtype=2), UNSUPPORTED)])
def test_read_refuses(kw, code):
    d = dict(k=P, v=P, ldk=128, ldv=128, dtype=0)
    d.update(kw)
    rc = _lib.load().opc_kv_read(ctypes.byref(cache()), ctypes.byref(batch()), d["dtype"], d["k"], d["ldk"], d["v"], d["ldv"], None)
    assert rc == code and "opc_kv_read" in _lib.last_error()


@pytest.mark.parametrize("kw,code", [
    (dict(heads=3), INVALID), (dict(heads=0), INVALID), (dict(dtype=2), UNSUPPORTED), (dict(scale=math.nan), INVALID),
    (dict(scale=math.inf), INVALID), (dict(q=None), INVALID), (dict(out=None), INVALID), (dict(ldq=255), INVALID),
    (dict(ldo=255), INVALID)])
def test_attention_refuses(kw, code):
    d = dict(heads=4, dtype=0, scale=0.1, q=P, ldq=256, out=P, ldo=256)
    d.update(kw)
    rc = _lib.load().opc_kv_attention(ctypes.byref(cache()), ctypes.byref(batch()), d["heads"], d["dtype"], d["scale"], d["q"],
                                      d["ldq"], d["out"], d["ldo"], None, P, 1 << 20, None)
    assert rc == code and "opc_kv_attention" in _lib.last_error()


@pytest.mark.parametrize("kw,code", [
    (dict(rows=-1), INVALID), (dict(vocab=0), INVALID), (dict(top_k=-1), INVALID), (dict(top_k=33), INVALID),
    (dict(vocab=4, top_k=5), INVALID), (dict(dtype=3), UNSUPPORTED), (dict(targets=None), INVALID),
    (dict(logprob=None), INVALID), (dict(top_k=2, ids=None), INVALID), (dict(top_k=2, top=None), INVALID),
    (dict(logits=None), INVALID), (dict(logits=P + 1), INVALID), (dict(dtype=2, logits=P + 2), INVALID), (dict(ld=99), INVALID)])
def test_logprobs_refuse(kw, code):
    d = dict(logits=P, ld=100, dtype=0, rows=3, vocab=100, targets=P, logprob=P, entropy=P, top_k=0, ids=P, top=P)
    d.update(kw)
    rc = _lib.load().opc_token_logprobs(d["logits"], d["ld"], d["dtype"], d["rows"], d["vocab"], d["targets"], d["logprob"],
                                        d["entropy"], d["top_k"], d["ids"], d["top"], P, 1 << 20, None)
    assert rc == code and "opc_token_logprobs" in _lib.last_error()


def test_workspace_sizes_of_refused_requests_are_zero():
    lib = _lib.load()
    assert lib.opc_kv_attention_workspace_bytes(None, None, 4, 0) == 0
    assert lib.opc_kv_attention_workspace_bytes(ctypes.byref(cache()), ctypes.byref(batch()), 3, 0) == 0
    assert lib.opc_token_logprobs_workspace_bytes(3, 100, 33, 0) == 0


def call_attention_of(kv_heads, head_dim=64, heads=None, max_kv=100, **kw):
    _, c = plan(kv_heads, head_dim, 16, 3)
    c.pages = P
    heads = kv_heads if heads is None else heads
    ld = heads * head_dim
    return _lib.load().opc_kv_attention(ctypes.byref(c), ctypes.byref(batch(max_kv=max_kv, max_pages=1 << 20, table_stride=1 << 20, **kw)),
                                        heads, 0, 1.0, P, ld, P, ld, None, P, 1 << 20, None)


@pytest.mark.parametrize("n_seqs,kv_heads,max_kv", [(65535, 20000, 100), (65535, 16385, 1), (1, 65535, 128 * 65535), (65535, 1, 2**31 - 1)])
def test_attention_refuses_more_work_than_it_counts(n_seqs, kv_heads, max_kv):
    # places of the line of work: (stages of 128 keys, one at least, + 3) for every sequence and kv head
    assert n_seqs * kv_heads * (max(1, -(-min(max_kv, 1 << 24) // 128)) + 3) > 2**32 - 1
    assert call_attention_of(kv_heads, max_kv=max_kv, n_seqs=n_seqs, n_tokens=n_seqs, max_q=1) == INVALID
    assert "too many for one call" in _lib.last_error()


@pytest.mark.parametrize("n_seqs,kv_heads,n_tokens,max_q", [(1, 65535, 1 << 24, 1 << 24), (2, 65535, 1 << 24, (1 << 24) - 1)])
def test_attention_refuses_more_tiles_than_a_grid_has(n_seqs, kv_heads, n_tokens, max_q):
    # tiles of 256 rows, for every kv head: before anything is launched, for the sequences of few rows too
    assert call_attention_of(kv_heads, n_seqs=n_seqs, n_tokens=n_tokens, max_q=max_q) == INVALID
    assert "too many for one call" in _lib.last_error()


def test_plan_refuses_sizes_past_64_bits():
    assert plan(65535, 256, 256, 2**31 - 1)[0] == INVALID
    assert "opc_kv_plan" in _lib.last_error()
    rc, c = plan(63000, 256, 256, 2**31 - 1)  # below 2^63 bytes
    assert rc == _lib.OPC_OK and c.total_bytes == (2**31 - 1) * 63000 * 256 * 264
    # a cache of such sizes that was filled by hand
    big = cache(kv_heads=65535, head_dim=256, page_size=256, n_pages=2**31 - 1, head_bytes=256 * 264)
    big.total_bytes = ((2**31 - 1) * 65535 * 256 * 264 + 2**63) % 2**64 - 2**63  # what 64 bits make of it
    assert call_append(c=big) == INVALID and "opc_kv_append" in _lib.last_error()


def test_tensor_memory_is_allocated_before_dependents_may_start():
    """A dependent kernel may take tensor memory before it waits; a CTA that asked for its own only then could
    wait for a kernel that waits for it.  Such a hang is not for a GPU: the order is read in the source."""
    from opac1ty_b200.build import CSRC

    for name in ("opc_kv_prompt.cuh", "opc_gemm.cuh"):
        text = (CSRC / name).read_text()
        alloc, at = text.index('"tcgen05.alloc'), text.find("griddep_launch_dependents();")
        assert at < 0 or alloc < at, name

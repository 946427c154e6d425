"""The norm's rows beside their codes (OPC_I8_UNROUNDED), and the engine's layers with element-wise outliers, whose
tokens take no rounding to 8 bits."""

import ctypes

import numpy as np
import pytest
import torch

import engine_model
from int8_ref import BF16, E, F16, F32, f64
from opac1ty_b200 import _lib, int8
from opac1ty_b200.engine import Engine
from test_gpu_engine_int8 import MODELS, SEEN, SPARSE, _off, _tokens, forward64_int8, in_8_bits, make, q8
from test_gpu_int8_rows import WIDTHS, e_ss, values

pytestmark = pytest.mark.gpu
UNROUNDED = 0x100
TYPES = {F16: _lib.OPC_F16, BF16: _lib.OPC_BF16, F32: _lib.OPC_F32}


def norm(h, y, w, held, h_out=None, eps=1e-5, ldv=None, flag=UNROUNDED):
    """(normalized rows, codes, scales) through the C call."""
    rows, n = h.shape
    ld = -(-n // 16) * 16
    ldv = n if ldv is None else ldv
    codes = torch.full((rows, ld), 99, dtype=torch.int8, device=h.device)
    scales = torch.empty(rows, device=h.device)
    out = torch.full((rows, ldv), 5.0, dtype=held, device=h.device)
    c = _lib.I8Rows(rows, n, ld, codes.data_ptr(), scales.data_ptr())

    def place(t):
        return (None, 0, 0) if t is None else (t.data_ptr(), t.stride(0), TYPES[t.dtype])

    _lib.check(_lib.load().opc_i8_add_rmsnorm(*place(h), *place(y), None if w is None else w.data_ptr(), 0 if w is None else TYPES[w.dtype],
                                              eps, *place(h_out)[:2], ctypes.byref(c), out.data_ptr(), ldv, TYPES[held] | flag,
                                              torch.cuda.current_stream(h.device).cuda_stream))
    assert (codes[:, n:] == 99).all() and (out[:, n:] == 5).all()
    return out[:, :n], codes[:, :n], scales


@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("h_type,y_type,w_type", [(F32, F16, F16), (F32, BF16, None), (F32, F32, F32), (F16, F16, BF16),
                                                  (BF16, BF16, BF16), (F16, None, F16), (BF16, None, None), (F32, None, F32)])
def test_rows_as_formed(cuda_device, n, h_type, y_type, w_type):
    h = values(4, n, n, h_type, cuda_device)
    y = None if y_type is None else values(4, n, n + 1, y_type, cuda_device, spread=False)
    w = None if w_type is None else (1 + 0.3 * values(1, n, n + 2, F32, cuda_device, spread=False)[0]).to(w_type)
    t = f64(h) + (0 if y is None else f64(y))
    want = t * (1 if w is None else f64(w)) / np.sqrt((t * t).mean(-1, keepdims=True) + 1e-5)
    # the sum's and the weight's roundings, the factor's (the root's E_ss and two steps of fp32), the product's
    e = 2 * E + e_ss(n) + 4 * E + E
    h_out = torch.empty_like(h)
    _, codes, scales = norm(h, y, w, F16, flag=0, h_out=h_out)
    for held, half in ((F16, 2.0 ** -11), (BF16, 2.0 ** -8), (F32, 0.0)):
        again = h.clone()
        got, c, s = norm(again, y, w, held, h_out=again, ldv=n + 3)
        off = np.abs(f64(got) - want)
        assert (off <= np.abs(want) * (e + half) * 1.01 + (2.0 ** -25 if held == F16 else 0)).all()  # (half a step of fp16's smallest)
        assert torch.equal(again, h_out)
        # a call without them sums the squares in another order; its codes do not depend on them
        assert (np.abs(f64(s) - f64(scales)) <= f64(scales) * 2 * (e_ss(n) + 4 * E)).all()
        assert torch.equal(c, codes)


@pytest.mark.parametrize("n", [40, 2000, 40000])
def test_rows_of_zeros_infinities_and_nan(cuda_device, n):
    h = values(5, n, 1, F32, cuda_device, spread=False)
    h[1] = 0
    h[2, n - 1] = float("inf")
    h[3, 0] = float("nan")
    h[4] = 1e30
    got, codes, scales = norm(h, None, None, F32)
    assert torch.isfinite(got[0]).all() and not got[1].any() and not codes[1:4].any()
    assert torch.isnan(got[2, n - 1]) and torch.isnan(got[3]).all() and torch.isnan(scales[2:4]).all()
    assert ((got[4] - 1).abs() < 1e-5).all() and (codes[4] == 127).all()


def test_refusals(cuda_device):
    h = values(2, 64, 1, F32, cuda_device)
    for bad in (0x203, 0x200, 0x103, -1):
        with pytest.raises(_lib.OpcError, match="element type"):
            norm(h, None, None, F16, flag=bad)
    c = _lib.I8Rows(2, 64, 64, h.data_ptr(), h.data_ptr())
    rc = _lib.load().opc_i8_quantize(h.data_ptr(), 64, _lib.OPC_F32, ctypes.byref(c), h.data_ptr(), 64, UNROUNDED, None)
    assert rc == _lib.OPC_ERR_UNSUPPORTED


def forward64_unrounded(m, tokens, disturb=0.0, seed=0):
    """forward64_int8 in which layers with element-wise outliers take their tokens as they are."""
    held = {k: v["type"] for k, v in m["layers"].items()}
    some = in_8_bits(len(tokens))[:, None]
    rng = np.random.default_rng(seed)
    L, hd, H, KV = m["layers"], m["hd"], m["heads"], m["kv_heads"]
    W = {k: engine_model.dequantize_np(v).astype(np.float64) for k, v in L.items() if v["type"] in ("quantized", "sparse_outlier")}
    vec = {k: np.asarray(v["data"], dtype=np.float64).reshape(-1) for k, v in L.items() if v["type"] == "fp16_passthrough"}
    T, pos = len(tokens), np.arange(len(tokens), dtype=np.float64)

    def mul(x, name):
        x = x * (1 + disturb * rng.uniform(-1, 1, x.shape))
        w = W[name]
        return x @ w.T if held[name] == "sparse_outlier" else np.where(some, q8(x) @ q8(w).T, x @ w.T)

    h = W["model.embed_tokens.weight"][np.asarray(tokens)].copy()
    for i in range(m["n_layers"]):
        p = f"model.layers.{i}."
        xn = engine_model._rms(h, vec.get(p + "input_layernorm.weight"), m["eps"])
        q = engine_model._rope(mul(xn, p + "self_attn.q_proj.weight"), pos, hd, m["theta"]).reshape(T, H, hd)
        k = engine_model._rope(mul(xn, p + "self_attn.k_proj.weight"), pos, hd, m["theta"]).reshape(T, KV, hd)
        v = mul(xn, p + "self_attn.v_proj.weight").reshape(T, KV, hd)
        att = np.zeros((T, H, hd))
        for hh in range(H):
            kh = hh // (H // KV)
            sc = np.where(np.tril(np.ones((T, T), dtype=bool)), q[:, hh] @ k[:, kh].T / np.sqrt(hd), -np.inf)
            sc = np.exp(sc - sc.max(axis=1, keepdims=True))
            att[:, hh] = (sc / sc.sum(axis=1, keepdims=True)) @ v[:, kh]
        h = h + mul(att.reshape(T, H * hd), p + "self_attn.o_proj.weight")
        xn = engine_model._rms(h, vec.get(p + "post_attention_layernorm.weight"), m["eps"])
        g, u = mul(xn, p + "mlp.gate_proj.weight"), mul(xn, p + "mlp.up_proj.weight")
        h = h + mul(g / (1.0 + np.exp(-g)) * u, p + "mlp.down_proj.weight")
    return engine_model._rms(h, vec.get("model.norm.weight"), m["eps"]) @ W["lm_head.weight"].T


@pytest.mark.parametrize("n", [65, 150, 300, 600])
def test_a_model_of_such_layers_keeps_its_logits(tmp_path, cuda_device, n):
    """Disturbing every product's tokens by 2^-11 of themselves moves the logits by at most 0.0006 of their norm (in the
    float64 pass, three seeds for each of these lengths); bringing the norms' tokens into 8 bits moved them by 0.008 to 0.022.
    The two engines differ in the order of the norms' sums alone."""
    p = tmp_path / "sparse.bf2"
    m = engine_model.build(p, element=True)
    toks = _tokens(n, m["vocab"], n)
    with Engine(p, prompt_bits=8) as a, Engine(p) as b:
        x, y = a.forward(toks).astype(np.float64), b.forward(toks).astype(np.float64)
    assert _off(x, y) <= 2 * 0.0006


def test_a_model_of_both_kinds(tmp_path, cuda_device):
    """Nearer to the float64 pass that leaves such layers' tokens as they are than to the one that brings them into 8 bits."""
    m = make(tmp_path / "mixed.bf2", "mixed")
    assert set(SPARSE) == {k for k, v in m["layers"].items() if v["type"] == "sparse_outlier"} and "mixed" in MODELS
    got, want, old = [], [], []
    with Engine(m["path"], prompt_bits=8) as eng:
        for n, seed in ((65, 21), (100, 22), (200, 23), (300, 24), (400, 25), (512, 26)):
            toks = _tokens(n, m["vocab"], seed)
            got.append(eng.forward(toks).astype(np.float64))
            want.append(forward64_unrounded(m, toks)[-1])
            old.append(forward64_int8(m, toks)[-1])
    got, want, old = np.stack(got), np.stack(want), np.stack(old)
    assert _off(got, want) <= 3 * SEEN["mixed"]
    assert np.linalg.norm(got - want) < np.linalg.norm(got - old)

"""bf_engine_create_kv4 and bf_engine_score on the GPU: the engine on a 4-bit paged cache, and what a
model thinks of given tokens, against the float64 forward pass of engine_model.

The 4-bit cache's float64 pass quantizes every rotated key and value head by the cache's definition
(kv_ref.quantize32) and rounds nothing else.  The engine's own keys and values carry fp16 rounding, so
a share of the codes lands on the other side of a rounding boundary, each by a whole step.  How much
that moves the logits was found in the float64 pass alone, by disturbing keys and values by 2^-10
before they are quantized (three seeds, Frobenius norm over all positions of the differences against
that of the logits): 0.036 for 4 heads of 64, 0.034 for 8 of 32, 0.054 for 2 of 128.  The tolerance is
three times that, because the engine rounds a dozen intermediate results and not one; leaving out the
quantization would miss it (0.13, 0.09, 0.18), and so would another rotary base (0.23 and more)."""

import json

import numpy as np
import pytest
from click.testing import CliRunner

import engine_model
from engine_model import build, forward64, rel_err
from kv_ref import quantize32
from opac1ty_b200.engine import Engine, EngineError

pytestmark = pytest.mark.gpu
TOL16 = 2e-2  # of max |logit|: fp16 cache, as in test_gpu_engine


def _tokens(n, vocab, seed=1):
    return np.random.default_rng(seed).integers(1, vocab, size=n).tolist()


def _rounded(x):
    codes, scale, zero = quantize32(x)
    return scale.astype(np.float64) * (codes.astype(np.float64) + zero.astype(np.float64))


def forward64_kv4(m, tokens):
    """forward64 with every key and value head replaced by what 4 bits hold of it."""
    L = m["layers"]
    W = {k: engine_model.dequantize_np(v).astype(np.float64) for k, v in L.items() if v["type"] == "quantized"}
    vec = {k: np.asarray(v["data"], dtype=np.float64).reshape(-1) for k, v in L.items() if v["type"] == "fp16_passthrough"}
    hd, H, KV, eps, theta = m["hd"], m["heads"], m["kv_heads"], m["eps"], m["theta"]
    T = len(tokens)
    pos = np.arange(T, dtype=np.float64)
    h = W["model.embed_tokens.weight"][np.asarray(tokens)].copy()
    for i in range(m["n_layers"]):
        p = f"model.layers.{i}."
        xn = engine_model._rms(h, vec.get(p + "input_layernorm.weight"), eps)
        q = engine_model._rope(xn @ W[p + "self_attn.q_proj.weight"].T, pos, hd, theta).reshape(T, H, hd)
        k = _rounded(engine_model._rope(xn @ W[p + "self_attn.k_proj.weight"].T, pos, hd, theta).reshape(T, KV, hd))
        v = _rounded((xn @ W[p + "self_attn.v_proj.weight"].T).reshape(T, KV, hd))
        att = np.zeros((T, H, hd))
        for hh in range(H):
            kh = hh // (H // KV)
            sc = q[:, hh] @ k[:, kh].T / np.sqrt(hd)
            sc = np.where(np.tril(np.ones((T, T), dtype=bool)), sc, -np.inf)
            sc = np.exp(sc - sc.max(axis=1, keepdims=True))
            att[:, hh] = (sc / sc.sum(axis=1, keepdims=True)) @ v[:, kh]
        h = h + att.reshape(T, H * hd) @ W[p + "self_attn.o_proj.weight"].T
        xn = engine_model._rms(h, vec.get(p + "post_attention_layernorm.weight"), eps)
        g = xn @ W[p + "mlp.gate_proj.weight"].T
        h = h + (g / (1.0 + np.exp(-g)) * (xn @ W[p + "mlp.up_proj.weight"].T)) @ W[p + "mlp.down_proj.weight"].T
    return engine_model._rms(h, vec.get("model.norm.weight"), eps) @ W["lm_head.weight"].T


def _log_softmax(x):
    m = x.max(-1, keepdims=True)
    return x - m - np.log(np.exp(x - m).sum(-1, keepdims=True))


@pytest.fixture(scope="module")
def models(tmp_path_factory, cuda_device):
    d = tmp_path_factory.mktemp("kv4")
    out = {}
    for hd, kw in ((64, dict()), (32, dict(heads=8, kv_heads=2)), (128, dict(heads=2, kv_heads=1))):
        out[hd] = build(d / f"hd{hd}.bf2", **kw)
        out[hd]["path"] = d / f"hd{hd}.bf2"
    return out


TOL4 = {64: 3 * 0.036, 32: 3 * 0.034, 128: 3 * 0.054}


@pytest.mark.parametrize("hd", [64, 32, 128])
@pytest.mark.parametrize("n,steps", [(100, 100), (100, 20), (600, 8)])
def test_kv4_matches_float64(models, hd, n, steps):
    """Single tokens alone, a prompt and then tokens, a prompt over two chunks and then tokens."""
    m = models[hd]
    toks = _tokens(n, m["vocab"], seed=3)
    ref = forward64_kv4(m, toks)
    with Engine(m["path"], kv_bits=4) as eng:
        if n > steps:
            eng.prefill(toks[:-steps])
        got = np.stack([eng.forward_step(t) for t in toks[-steps:]]).astype(np.float64)
        assert eng.position == n
    want = ref[-steps:]
    assert np.linalg.norm(got - want) <= TOL4[hd] * np.linalg.norm(want)


def test_kv4_cache_size_reset_and_generation(models):
    m = models[64]
    with Engine(m["path"], max_context=100, kv_bits=4) as eng:  # 2 pages of 64 positions
        assert eng.kv_cache_size == m["n_layers"] * m["kv_heads"] * 128 * (m["hd"] + 8)
        prompt = _tokens(40, m["vocab"], seed=5)
        a = eng.forward(prompt)
        eng.forward(_tokens(90, m["vocab"], seed=6))
        assert np.array_equal(eng.forward(prompt), a)  # forward() starts over: nothing of the longer text is left
        one = eng.generate_tokens(prompt, 12, temperature=0.0)
        assert eng.generate_tokens(prompt, 12, temperature=0.0) == one and len(one) >= 1
        with pytest.raises(EngineError, match="context full"):
            eng.prefill([1] * 101)


@pytest.mark.parametrize("hidden,heads,fp16", [(192, 4, False), (320, 2, True)])
def test_kv4_refuses_a_head_dimension(tmp_path, cuda_device, hidden, heads, fp16):
    """Heads of 48 fit neither cache (the engine takes multiples of 32), heads of 160 the fp16 cache only."""
    p = tmp_path / "heads.bf2"
    m = build(p, hidden=hidden, heads=heads, kv_heads=heads // 2)
    with pytest.raises(EngineError, match="head_dim"):
        Engine(p, kv_bits=4)
    if fp16:
        with Engine(p) as eng:
            toks = _tokens(5, m["vocab"])
            assert rel_err(eng.forward(toks), forward64(m, toks)[-1]) < TOL16


def _check_score(s, toks, ref, delta):
    """Every number of a score against the logits `ref`, which the engine's are within delta of."""
    n = len(toks) - 1
    lp = _log_softmax(ref[:n])
    p = np.exp(lp)
    assert s.logprob.shape == (n,) and s.entropy.shape == (n,)
    eps = 2 * delta  # of every log probability
    assert np.all(np.abs(s.logprob - lp[np.arange(n), toks[1:]]) <= eps)
    entropy = -(p * lp).sum(-1)
    # |H(q) - H(p)| <= sum |q - p| |log p| + sum q |log p - log q|, with q <= e^eps p
    assert np.all(np.abs(s.entropy - entropy) <= (np.exp(eps) - 1) * entropy + eps)
    k = s.top_ids.shape[1]
    if k:
        best = -np.sort(-lp, axis=-1)[:, :k]
        assert np.all(np.abs(s.top_logprobs - best) <= eps)  # order statistics move by no more than the values
        assert np.all(np.diff(s.top_logprobs, axis=1) <= 0)
        assert np.all(np.abs(s.top_logprobs - np.take_along_axis(lp, s.top_ids, 1)) <= eps)
        hit = s.top_ids == np.asarray(toks[1:])[:, None]
        rows = hit.any(1)
        assert np.array_equal(s.top_logprobs[hit], s.logprob[rows])  # the same logit gives the same number


@pytest.mark.parametrize("n,top_k", [(2, 5), (3, 0), (100, 32), (513, 4), (600, 1)])
def test_score_matches_float64(models, n, top_k):
    """fp16 cache.  513: the second chunk has one token and no successor; 600 takes several groups of rows."""
    m = models[64]
    toks = _tokens(n, m["vocab"], seed=9)
    ref = forward64(m, toks)
    with Engine(m["path"]) as eng:
        s = eng.score(toks, top_k=top_k)
        assert eng.position == n
        _check_score(s, toks, ref, TOL16 * np.abs(ref).max())
        assert s.perplexity == pytest.approx(np.exp(-s.logprob.astype(np.float64).mean()))
        again = eng.score(toks, top_k=top_k)
        for a, b in zip(s, again):
            assert np.array_equal(a, b)
        # the cache holds the text: the next step continues it
        t = _tokens(1, m["vocab"], seed=10)[0]
        assert rel_err(eng.forward_step(t), forward64(m, toks + [t])[-1]) < TOL16


def test_score_on_the_4_bit_cache(models):
    """Norm-wise, as for the logits: the log probabilities of the text, the cache's three calls together."""
    m = models[64]
    toks = _tokens(300, m["vocab"], seed=11)
    ref = forward64_kv4(m, toks)
    with Engine(m["path"], kv_bits=4) as eng:
        s = eng.score(toks, top_k=3)
        with Engine(m["path"]) as full:
            s16 = full.score(toks)
    lp = _log_softmax(ref)[np.arange(299), toks[1:]]
    # a log probability moves with one logit and with the log of the sum: twice the logits' error, whose
    # root mean square is TOL4 of the logits'
    rms = np.sqrt(np.mean(ref * ref))
    assert np.sqrt(np.mean((s.logprob - lp) ** 2)) <= 2 * TOL4[64] * rms
    assert np.sqrt(np.mean((s.logprob - s16.logprob) ** 2)) > 0  # another cache, other numbers
    assert np.all(s.top_logprobs[:, 0] >= s.logprob)


def test_score_of_one_token_and_refusals(models):
    m = models[64]
    with Engine(m["path"], max_context=8) as eng:
        s = eng.score([5])
        assert s.logprob.size == 0 and eng.position == 1 and np.isnan(s.perplexity)
        for toks, k, msg in (([], 0, "no tokens"), ([1, 2], 33, "top_k"), ([1, 2], -1, "top_k"),
                             ([1, m["vocab"]], 0, "outside"), ([1] * 9, 0, "context full")):
            with pytest.raises(EngineError, match=msg):
                eng.score(toks, top_k=k)
        assert eng.score([1, 2, 3]).logprob.shape == (2,)  # usable after them


def test_command_line(models):
    from opac1ty_b200.cli import cli

    m = models[64]
    for bits in ("16", "4"):
        res = CliRunner().invoke(cli, ["score", str(m["path"]), "--tokens", "5, 9 17", "--top", "2", "--kv-bits", bits])
        assert res.exit_code == 0, res.output
        out = json.loads(res.output)
        assert out["tokens"] == 3 and len(out["logprobs"]) == 2 and len(out["top"][0]) == 2
        with Engine(m["path"], kv_bits=int(bits), max_context=3) as eng:
            s = eng.score([5, 9, 17], top_k=2)
        assert out["perplexity"] == pytest.approx(s.perplexity, rel=1e-6)
    res = CliRunner().invoke(cli, ["score", str(m["path"]), "--text", "hello"])
    assert res.exit_code == 0 and json.loads(res.output)["tokens"] == 5

"""The serving operators around the 4-bit paged cache, as cases to measure: appending rotated keys
and values, attention over the cache, and the log probabilities of given tokens.

The cache holds, for every page and kv head, one block of ``page_size * (head_dim + 8)`` bytes: the
keys' 4-bit codes [page_size][head_dim / 2], the values' codes, then a (scale, zero) pair of fp16 per
token for the keys and one for the values.  Dimension d of a token is nibble d % 2 of byte d // 2; a
value stands for ``scale * (code + zero)``.  Stored heads follow from x (after the rotation) as

    scale = max(fp16(max((max x - min x) / 15, max |x| / 1024)), 2**-24)
    zero  = fp16(min x / scale)
    code  = clamp(round(x / scale - zero), 0, 15)

A batch is packed: rows q_start[s] .. q_start[s+1] are the last rows of sequence s, which holds
kv_len[s] tokens once they are in; row i of it sits at position kv_len - q_len + i, in page
page_table[s][position // page_size].
"""

import math

import torch

own = False

SCALE_MIN = 2.0 ** -24
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# --------------------------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------------------------
def listed():
    return [
        # One sequence's next token in a chat at 4000 tokens: the whole call is latency.
        {"name": "append_one", "op": "append", "seqs": 1, "q_min": 1, "q_max": 1, "kv_min": 4000, "kv_max": 4000,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "type": "fp16", "pairs": "half"},
        # A step of a busy server: 96 sequences of very different ages, one token each.
        {"name": "append_96", "op": "append", "seqs": 96, "q_min": 1, "q_max": 1, "kv_min": 1, "kv_max": 8191,
         "heads": 64, "kv_heads": 8, "head_dim": 128, "page": 16, "type": "bf16", "pairs": "adjacent"},
        # Prompts of odd lengths arriving together, some behind a long shared history.
        {"name": "append_prompts", "op": "append", "seqs": 5, "q_min": 1, "q_max": 2047, "kv_min": 2047,
         "kv_max": 40001, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "type": "fp16", "pairs": "half"},
        # The next token's attention at 4000 tokens: latency again.
        {"name": "attend_one", "op": "attend", "seqs": 1, "q_min": 1, "q_max": 1, "kv_min": 4000, "kv_max": 4000,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "type": "fp16"},
        # One long document: the cache is larger than L2 and has to be split over the whole GPU.
        {"name": "attend_long", "op": "attend", "seqs": 1, "q_min": 1, "q_max": 1, "kv_min": 131071, "kv_max": 131071,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "type": "fp16"},
        # A step of a busy server over sequences of very different lengths, small pages.
        {"name": "attend_64", "op": "attend", "seqs": 64, "q_min": 1, "q_max": 1, "kv_min": 1, "kv_max": 8192,
         "heads": 64, "kv_heads": 8, "head_dim": 128, "page": 16, "type": "bf16"},
        # Draft tokens checked three at a time, heads of 64, as many kv heads as query heads.
        {"name": "attend_draft", "op": "attend", "seqs": 16, "q_min": 1, "q_max": 3, "kv_min": 33, "kv_max": 2049,
         "heads": 16, "kv_heads": 16, "head_dim": 64, "page": 32, "type": "fp16"},
        # One 512-token chunk of a prompt against what is cached already.
        {"name": "attend_chunk", "op": "attend", "seqs": 1, "q_min": 512, "q_max": 512, "kv_min": 4096, "kv_max": 4096,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "type": "fp16"},
        # Whole prompts of odd lengths: compute bound.
        {"name": "attend_prompts", "op": "attend", "seqs": 3, "q_min": 1500, "q_max": 4097, "kv_min": 1500,
         "kv_max": 4097, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "type": "fp16"},
        # One generated token with its 20 alternatives.
        {"name": "logprob_one", "op": "logprob", "rows": 1, "vocab": 128256, "top": 20, "masked": 0, "type": "fp16"},
        # A few sequences of a small vocabulary, part of it forbidden, logits in 32 bits.
        {"name": "logprob_17", "op": "logprob", "rows": 17, "vocab": 32000, "top": 5, "masked": 413, "type": "fp32"},
        # Scoring documents: the logits of 2048 positions.
        {"name": "logprob_2048", "op": "logprob", "rows": 2048, "vocab": 128256, "top": 8, "masked": 0, "type": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "logprob"])
    kind = rng.choice(["fp16", "bf16"])
    if op == "logprob":
        vocab = _log_int(rng, 256, 128256)
        kind = rng.choice(["fp16", "bf16", "fp32"])
        return {"op": op, "rows": _log_int(rng, 1, 1024 if kind == "fp32" else 2048), "vocab": vocab,
                "top": rng.randint(0, 32), "masked": rng.choice([0, rng.randint(1, vocab // 4)]), "type": kind}
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    heads = min(64, kv_heads * rng.choice([1, 2, 4, 7, 8]))
    heads -= heads % kv_heads
    c = {"op": op, "heads": heads, "kv_heads": kv_heads, "head_dim": rng.choice([32, 64, 96, 128, 128, 192, 256]),
         "page": rng.choice([16, 32, 64, 128, 256]), "type": kind}
    if op == "append":
        c["pairs"] = rng.choice(["half", "adjacent"])
    if rng.random() < 0.6:  # a step: one or a few tokens of each sequence
        c["seqs"] = _log_int(rng, 1, 64)
        c["kv_max"] = _log_int(rng, 16, min(131071, 250000 // (c["seqs"] * max(1, c["kv_heads"] // 4))))
        c["kv_min"] = rng.randint(1, c["kv_max"])
        c["q_min"], c["q_max"] = 1, rng.choice([1, 1, 1, 2, 5])
    else:  # prompts, or chunks of them
        c["seqs"] = rng.randint(1, 2)
        c["heads"] = max(kv_heads, min(heads, 4096 // c["head_dim"]))
        c["heads"] -= c["heads"] % kv_heads
        c["q_max"] = _log_int(rng, 16, 2048)
        c["q_min"] = rng.randint(1, c["q_max"])
        c["kv_max"] = c["q_max"] + rng.choice([0, _log_int(rng, 1, 2000)])
        c["kv_min"] = rng.randint(c["q_max"], c["kv_max"])
    return c


def _lengths(case):
    """(q_len, kv_len) of every sequence, spread over their ranges; the first has the longest."""
    def spread(lo, hi, step):
        return [hi if s == 0 else lo + int((hi - lo) * ((s * step) % 1.0)) for s in range(case["seqs"])]

    kv = spread(case["kv_min"], case["kv_max"], 0.6180339887498949)
    q = spread(case["q_min"], case["q_max"], 0.7548776662466927)
    return [min(a, b) for a, b in zip(q, kv)], kv


def work(case):
    size = {"fp16": 2, "bf16": 2, "fp32": 4}[case["type"]]
    if case["op"] == "logprob":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (12 + 8 * case["top"]), "flops": 5 * n}
    q, kv = _lengths(case)
    hd, heads, kvh, rows = case["head_dim"], case["heads"], case["kv_heads"], sum(q)
    if case["op"] == "append":
        # k, v and q in, q out, the stored heads written, and read back as k and v
        held = rows * kvh * (hd + 8)
        return {"bytes": rows * size * hd * (2 * kvh + 2 * heads) + 2 * held + 2 * rows * kvh * hd * size,
                "flops": rows * hd * (4 * heads + 16 * kvh)}
    pairs = sum(b * (b + 1) // 2 - (b - a) * (b - a + 1) // 2 for a, b in zip(q, kv))
    return {"bytes": sum(kv) * kvh * (hd + 8) + 2 * rows * heads * hd * size + 4 * rows * heads,
            "flops": 4 * pairs * heads * hd}


# --------------------------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------------------------
def _quantize(x):
    """Codes (in fp32), scale and zero (fp32, of fp16 precision) of heads x [..., head_dim] fp32."""
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    big = torch.maximum(lo.abs(), hi.abs())
    scale = torch.maximum((hi - lo) / 15.0, big / 1024.0).half().float().clamp_min(SCALE_MIN)
    zero = (lo / scale).half().float()
    return (x * (1.0 / scale) - zero).round().clamp(0, 15), scale, zero


def _block(codes, scale, zero):
    """(bytes of the codes [..., head_dim/2], bytes of the (scale, zero) pairs [..., 4])."""
    c = codes.to(torch.uint8).unflatten(-1, (-1, 2))
    pair = torch.cat([scale, zero], -1).half().contiguous()
    return c[..., 0] | (c[..., 1] << 4), pair.view(torch.uint8)


def _pages(case, n_pages, g, device):
    """A cache of random keys (with channel means, as keys have) and values."""
    kvh, hd, page = case["kv_heads"], case["head_dim"], case["page"]
    pages = torch.empty(n_pages, kvh, page * (hd + 8), dtype=torch.uint8, device=device)
    mean = 1.2 * torch.randint(0, 2, (kvh, 1, hd), generator=g, device=device).mul(2).sub(1).float()
    step = max(1, (1 << 26) // (kvh * page * hd))
    for a in range(0, n_pages, step):
        n = min(step, n_pages - a)
        k = torch.randn(n, kvh, page, hd, generator=g, device=device) + mean
        v = torch.randn(n, kvh, page, hd, generator=g, device=device)
        (kc, kp), (vc, vp) = _block(*_quantize(k)), _block(*_quantize(v))
        pages[a:a + n] = torch.cat([t.reshape(n, kvh, -1) for t in (kc, vc, kp, vp)], -1)
    return pages


def prepare(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=device)
    g.manual_seed(int(seed))
    kind = TYPES[case["type"]]
    s = {"case": case, "device": device}
    if case["op"] == "logprob":
        rows, vocab = case["rows"], case["vocab"]
        # a language model's logits: a broad bulk, and for most rows a few tokens far above it
        x = torch.randn(rows, vocab, generator=g, device=device, dtype=torch.float32).mul_(2.0)
        at = torch.randint(0, vocab, (rows, 6), generator=g, device=device)
        x.scatter_add_(1, at, 14.0 * torch.rand(rows, 6, generator=g, device=device))
        if case["masked"]:
            x[:, vocab - case["masked"]:] = -math.inf
        s["logits"] = x.to(kind)
        s["targets"] = torch.randint(0, vocab - case["masked"], (rows,), generator=g, device=device,
                                     dtype=torch.int32)
        return s
    q, kv = _lengths(case)
    page, hd, heads, kvh, rows = case["page"], case["head_dim"], case["heads"], case["kv_heads"], sum(q)
    used = [-(-n // page) for n in kv]
    width, n_pages = max(used), sum(used)
    order = torch.randperm(n_pages, generator=g, device=device, dtype=torch.int32)
    at = torch.tensor([sum(used[:i]) for i in range(len(used))], device=device, dtype=torch.int32)
    col = torch.arange(width, device=device, dtype=torch.int32)
    have = torch.tensor(used, device=device, dtype=torch.int32)
    index = (at[:, None] + col[None, :]).clamp(max=n_pages - 1).long()
    table = torch.where(col[None, :] < have[:, None], order[index], torch.full_like(order[index], -1))
    s["page_table"] = table.contiguous()
    s["q_start"] = torch.tensor([0] + [sum(q[:i + 1]) for i in range(len(q))], device=device, dtype=torch.int32)
    s["kv_len"] = torch.tensor(kv, device=device, dtype=torch.int32)
    s["max_q"], s["max_kv"] = max(q), max(kv)
    # the projections of one fused q|k|v product, row by row
    s["q"] = torch.randn(rows, heads, hd, generator=g, device=device).to(kind)
    if case["op"] == "append":
        mean = 1.2 * torch.randint(0, 2, (kvh, hd), generator=g, device=device).mul(2).sub(1).float()
        s["k"] = (torch.randn(rows, kvh, hd, generator=g, device=device) + mean).to(kind)
        s["v"] = torch.randn(rows, kvh, hd, generator=g, device=device).to(kind)
        s["pages"] = torch.zeros(n_pages, kvh, page * (hd + 8), dtype=torch.uint8, device=device)
    else:
        s["pages"] = _pages(case, n_pages, g, device)
    # what a server keeps from step to step: the rotation's frequencies and the batch's description
    s["inv_freq"] = 500000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device=device) / hd)
    if own:
        from opac1ty_b200 import kv as K

        s["cache"] = K.KVCache(kvh, hd, n_pages, page, pages=s["pages"])
        s["batch"] = K.KVBatch(s["q_start"], s["kv_len"], s["page_table"], n_tokens=rows, max_q=s["max_q"],
                               max_kv=s["max_kv"])
        s["rope"] = K.Rope(hd, inv_freq=s["inv_freq"].cpu(), interleaved=case.get("pairs") == "adjacent",
                           device=device)
    return s


# --------------------------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        if op == "append":
            from opac1ty_b200 import kv as K

            q = K.append(s["cache"], s["batch"], s["k"], s["v"], q=s["q"], rope=s["rope"])
            k, v = K.read(s["cache"], s["batch"], dtype=s["k"].dtype)
            return {"q": q, "k": k, "v": v}
        if op == "attend":
            from opac1ty_b200 import kv as K

            out, lse = K.attention(s["cache"], s["batch"], s["q"], return_lse=True)
            return {"out": out, "lse": lse}
        from opac1ty_b200 import score

        r = score.token_logprobs(s["logits"], s["targets"], top_k=s["case"]["top"])
        return {"logprob": r.logprob, "entropy": r.entropy, "ids": r.top_ids, "top": r.top_logprobs}
    return {"append": _append, "attend": _attend, "logprob": _logprob}[op](s)


def _places(s):
    """Of every row: its position, page and place in that page."""
    n = s["q"].shape[0]
    row = torch.arange(n, device=s["device"])
    start, kv = s["q_start"].long(), s["kv_len"].long()
    seq = torch.searchsorted(start, row, right=True) - 1
    pos = kv[seq] - (start[seq + 1] - row)
    page = s["case"]["page"]
    return pos, s["page_table"].long()[seq, pos // page], pos % page


def _rotate(x, angle, pairs):
    x = x.float()
    c, n = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if pairs == "half":
        a, b = x.chunk(2, -1)
        return torch.cat([a * c - b * n, b * c + a * n], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)


def _append(s):
    case, kind = s["case"], s["q"].dtype
    page, hd, kvh = case["page"], case["head_dim"], case["kv_heads"]
    pos, at, off = _places(s)
    angle = pos.double()[:, None] * s["inv_freq"][None, :]
    q = _rotate(s["q"], angle, case["pairs"]).to(kind)
    half = page * hd // 2
    kc, vc = s["pages"][..., :half].unflatten(-1, (page, -1)), s["pages"][..., half:2 * half].unflatten(-1, (page, -1))
    kp = s["pages"][..., 2 * half:2 * half + 4 * page].unflatten(-1, (page, 4))
    vp = s["pages"][..., 2 * half + 4 * page:].unflatten(-1, (page, 4))
    head = torch.arange(kvh, device=s["device"])[None, :]
    where = (at[:, None], head, off[:, None])
    kc[where], kp[where] = _block(*_quantize(_rotate(s["k"], angle, case["pairs"])))
    vc[where], vp[where] = _block(*_quantize(s["v"].float()))
    return {"q": q, "k": _values(kc[where], kp[where]).to(kind), "v": _values(vc[where], vp[where]).to(kind)}


def _values(codes, pairs):
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float()
    p = pairs.contiguous().view(torch.float16).float()
    return p[..., :1] * (c + p[..., 1:])


def _attend(s):
    case = s["case"]
    page, hd, heads, kvh = case["page"], case["head_dim"], case["heads"], case["kv_heads"]
    half = page * hd // 2
    b = s["pages"][s["page_table"].long().clamp_min(0)].transpose(1, 2)  # [seq][kv head][page][bytes]
    k = _values(b[..., :half].unflatten(-1, (page, -1)), b[..., 2 * half:2 * half + 4 * page].unflatten(-1, (page, 4)))
    v = _values(b[..., half:2 * half].unflatten(-1, (page, -1)), b[..., 2 * half + 4 * page:].unflatten(-1, (page, 4)))
    k, v = k.flatten(2, 3), v.flatten(2, 3)  # [seq][kv head][key][dim]
    start, kv = s["q_start"].long(), s["kv_len"].long()
    n = start[1:] - start[:-1]
    i = torch.arange(s["max_q"], device=s["device"])
    j = torch.arange(k.shape[2], device=s["device"])
    row = (start[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][row].float().unflatten(2, (kvh, -1)).permute(0, 2, 3, 1, 4)  # [seq][kv head][head of it][query][dim]
    x = torch.matmul(q.flatten(2, 3), k.transpose(-1, -2)).unflatten(2, (-1, s["max_q"])) * hd ** -0.5
    seen = j <= (kv - n)[:, None, None] + i[None, :, None]
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    big = x.amax(-1, keepdim=True).clamp_min(-3e38)
    p = (x - big).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), v).unflatten(2, (-1, s["max_q"])) / total.clamp_min(1e-38)
    lse = (total.log() + big).squeeze(-1)
    real = (i[None, :] < n[:, None]).flatten()
    out = o.permute(0, 3, 1, 2, 4).flatten(2, 3).flatten(0, 1)[real]
    return {"out": out.to(s["q"].dtype), "lse": lse.permute(0, 3, 1, 2).flatten(2, 3).flatten(0, 1)[real]}


def _logprob(s):
    x, top = s["logits"].float(), s["case"]["top"]
    big = x.amax(-1, keepdim=True)
    y = x - big
    e = y.exp()
    total = e.sum(-1, keepdim=True)
    lse = total.log()
    entropy = lse.squeeze(-1) - (e * y.clamp_min(-1e30)).sum(-1) / total.squeeze(-1)
    given = y.gather(1, s["targets"].long()[:, None]) - lse
    ids = y.sort(dim=-1, descending=True, stable=True).indices[:, :top]
    return {"logprob": given.squeeze(-1), "entropy": entropy, "ids": ids.int(), "top": y.gather(1, ids) - lse}


# --------------------------------------------------------------------------------------------
# The same from the definitions, in 64 bits
# --------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprob":
        return _exact_logprob(s)
    q, kv = _lengths(case)
    return _exact_append(s, q, kv) if case["op"] == "append" else _exact_attend(s, q, kv)


def _exact_logprob(s):
    parts = []
    for x in s["logits"].split(64):
        x = x.double()
        lse = torch.logsumexp(x, -1, keepdim=True)
        lp = x - lse
        h = -torch.where(x > -math.inf, lp.exp() * lp, torch.zeros_like(lp)).sum(-1)
        parts.append((lp, h))
    ids = s["logits"].double().sort(dim=-1, descending=True, stable=True).indices[:, :s["case"]["top"]]
    lp = torch.cat([p[0] for p in parts])
    return {"logprob": lp[torch.arange(lp.shape[0], device=lp.device), s["targets"].long()],
            "entropy": torch.cat([p[1] for p in parts]), "ids": ids.int(), "top": lp.gather(1, ids)}


def _turned(x, pos, inv_freq, pairs):
    """x [rows][heads][dim] turned as complex numbers by exp(i * position * frequency)."""
    x = x.double()
    d = x.shape[-1] // 2
    z = torch.complex(x[..., :d], x[..., d:]) if pairs == "half" else torch.view_as_complex(x.unflatten(-1, (d, 2)))
    angle = pos.double()[:, None] * inv_freq
    z = z * torch.polar(torch.ones_like(angle), angle)[:, None]
    return torch.cat([z.real, z.imag], -1) if pairs == "half" else torch.view_as_real(z).flatten(-2)


def _held(x):
    """What the cache holds for heads x: the definition's scale, zero and codes, as values."""
    lo, hi = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    scale = torch.maximum(torch.maximum((hi - lo) / 15, torch.maximum(-lo, hi).abs() / 1024).half().double(),
                          torch.tensor(SCALE_MIN, dtype=torch.float64, device=x.device))
    zero = (lo / scale).half().double()
    return scale * (torch.clamp(torch.round(x / scale - zero), 0, 15) + zero)


def _exact_append(s, q, kv):
    pairs = s["case"]["pairs"]
    pos = torch.cat([torch.arange(b - a, b, device=s["device"]) for a, b in zip(q, kv)])
    return {"q": _turned(s["q"], pos, s["inv_freq"], pairs),
            "k": _held(_turned(s["k"], pos, s["inv_freq"], pairs)), "v": _held(s["v"].double())}


def _exact_attend(s, q, kv):
    case = s["case"]
    page, hd, heads, kvh = case["page"], case["head_dim"], case["heads"], case["kv_heads"]
    half, group = page * hd // 2, heads // kvh
    outs, lses, row = [], [], 0
    for i, (a, b) in enumerate(zip(q, kv)):
        block = s["pages"][s["page_table"][i, :-(-b // page)].long()]  # [page][kv head][bytes]
        n = block.shape[0] * page

        def held(first, second, count=n):
            c = block[..., first:first + half].reshape(-1, kvh, page, hd // 2, 1)
            c = (c >> torch.tensor([0, 4], dtype=torch.uint8, device=c.device)) % 16
            p = block[..., second:second + 4 * page].contiguous().view(torch.float16).reshape(-1, kvh, page, 1, 2).double()
            x = (c.reshape(-1, kvh, page, hd).double() + p[..., 1]) * p[..., 0]
            return x.transpose(0, 1).reshape(kvh, count, hd)[:, :b]

        k, v = held(0, 2 * half), held(half, 2 * half + 4 * page)
        hidden = torch.arange(b, device=k.device)[None, :] > torch.arange(b - a, b, device=k.device)[:, None]
        out = torch.empty(a, heads, hd, dtype=torch.float64, device=k.device)
        lse = torch.empty(a, heads, dtype=torch.float64, device=k.device)
        for h in range(heads):
            x = s["q"][row:row + a, h].double() @ k[h // group].T / math.sqrt(hd)
            x.masked_fill_(hidden, -math.inf)
            lse[:, h] = torch.logsumexp(x, -1)
            out[:, h] = (x - lse[:, h, None]).exp_() @ v[h // group]
        outs.append(out)
        lses.append(lse)
        row += a
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}

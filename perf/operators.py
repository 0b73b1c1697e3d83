"""Operators of the text side of the pipeline, as cases that can be timed and checked.

Two operators, each in its plain form (elementary torch operations in 32 bits) and as a user calls the kernels:

  attention  softmax over the keys that a query may see: causal, prefix and document masks, padded batches, mask
             tensors, scores capped by a tanh, a bias by distance, grouped key/value heads; whole prompts and single
             tokens against a long cache.
  linear     y = act(x W^T + bias) + residual in one kernel.
"""
import math

import torch

own = False

GELU_TANH = math.sqrt(2.0 / math.pi)


def _attention(name, b, h, hk, sq, skv, d, **more):
    case = {"name": name, "op": "attention", "b": b, "h": h, "hk": hk, "sq": sq, "skv": skv, "d": d, "causal": False,
            "prefix": 0, "docs": 0, "ragged": False, "at_end": False, "cap": 0.0, "bias": "", "head_major": False}
    return {**case, **more}


def _linear(name, m, k, n, act, bias="bf16", residual=False):
    return {"name": name, "op": "linear", "m": m, "k": k, "n": n, "act": act, "bias": bias, "residual": residual}


def listed():
    return [
        # The text context in front of the UNet: a pair of 77-token prompts, 768 wide. The smallest call.
        _attention("prompt_77", 2, 12, 12, 77, 77, 64, causal=True),
        # A long prompt through a causal decoder with four query heads to each key/value head. The largest call.
        _attention("prompt_4096_grouped", 1, 32, 8, 4096, 4096, 128, causal=True),
        # Prompts of ragged lengths packed into one row of tokens, with some padding behind the last.
        _attention("documents_4097", 1, 8, 8, 4097, 4097, 80, causal=True, docs=13),
        # A prefix that sees itself whole and a causal rest, scores capped.
        _attention("prefix_capped_1000", 2, 8, 4, 1000, 1000, 160, causal=True, prefix=300, cap=30.0),
        # A bidirectional text encoder with a learned bias by distance over a right-padded batch.
        _attention("encoder_distance_1024", 4, 8, 8, 1024, 1024, 64, ragged=True, bias="table", head_major=True),
        # The UNet's cross-attention to text whose padding is masked by an additive mask tensor.
        _attention("cross_masked_77", 2, 8, 8, 4096, 77, 40, bias="mask_pad"),
        # A region mask: every query row has keys of its own that it may see.
        _attention("region_masked_1024", 2, 8, 8, 1024, 1024, 80, bias="mask_full"),
        # A few tokens at the end of each cache of a ragged batch, linear bias by distance.
        _attention("tokens_5_slopes", 4, 8, 2, 5, 5001, 128, causal=True, ragged=True, at_end=True, bias="slopes"),
        # One token against a long cache, a full batch: the whole cache is read once.
        _attention("token_cache_16384", 16, 32, 8, 1, 16384, 128, ragged=True),
        # One token against a short cache: latency.
        _attention("token_cache_777", 1, 8, 2, 1, 777, 64),
        # The feed-forward projection of a pair of 77-token prompts, with the residual.
        _linear("linear_prompt", 154, 768, 1280, "quick_gelu", bias="f32", residual=True),
        # The widest feed-forward projection of the batch-16 UNet's top level.
        _linear("linear_65536", 65536, 320, 1280, "gelu", residual=True),
    ]


ACTS = ("gelu", "gelu_tanh", "quick_gelu", "silu", "relu")


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("prompt", "prompt", "cross", "token", "token", "linear", "linear"))
    if kind == "linear":
        m, k, n = _log(rng, 1, 65536), _log(rng, 64, 5120), _log(rng, 64, 5120)
        k = k if rng.random() < 0.25 else -(-k // 8) * 8  # most weights have rows of whole 16-byte words
        while m * k * n > 65536 * 320 * 1280:
            m = m // 2 + 1
        case = _linear("", m, k, n, rng.choice(ACTS), rng.choice(("bf16", "f32", "none")), rng.random() < 0.5)
    else:
        hk = rng.choice((1, 2, 4, 5, 8))
        h = hk * rng.choice((1, 1, 2, 3, 4, 8))
        d = rng.choice((40, 64, 64, 72, 80, 96, 128, 128, 160, 256))
        bias = rng.choice(("", "", "slopes", "table", "mask_full" if kind != "token" else "slopes"))
        more = {"cap": rng.choice((0.0, 0.0, 20.0, 50.0)), "bias": bias, "head_major": rng.random() < 0.3}
        if kind == "prompt":
            b, sq = rng.choice((1, 2, 3, 8)), _log(rng, 1, 4096)
            skv = sq
            more |= rng.choice(({"causal": True}, {"causal": True, "prefix": rng.randint(1, sq)}, {"ragged": True},
                                {"causal": True, "docs": rng.randint(1, 16)}, {"docs": rng.randint(1, 16)},
                                {"causal": True, "ragged": True}))
        elif kind == "cross":
            b, sq, skv = rng.choice((1, 2, 3, 8)), _log(rng, 16, 4096), _log(rng, 1, 1024)
            more |= {"ragged": rng.random() < 0.5, "bias": rng.choice(("mask_pad", "mask_full"))}
        else:
            b, sq, skv = _log(rng, 1, 16), rng.choice((1, 1, 1, 2, 5, 16)), _log(rng, 64, 16384)
            more |= {"ragged": True, "causal": sq > 1, "at_end": True}
        while b * h * sq * skv * d > 16 * 4096 * 4096 * 128 and b > 1:
            b -= 1
        while b * h * sq * skv * d > 16 * 4096 * 4096 * 128:
            sq, skv = (sq + 1) // 2, (skv + 1) // 2
            more["prefix"] = min(more.get("prefix", 0), sq)
        while b * hk * skv * d > 16 * 8 * 16384 * 128:
            b -= 1
        case = _attention("", b, h, hk, sq, skv, d, **more)
    del case["name"]
    return case


# --- what a case holds besides its random values --------------------------------------------------------------------


def _lens(c):
    """Valid keys of each sequence of a padded batch: from nearly full down to half."""
    return [max(1, c["sq"] if c["at_end"] else 1, c["skv"] - i * c["skv"] // (2 * c["b"]) - c["skv"] % 7)
            for i in range(c["b"])] if c["ragged"] else [c["skv"]] * c["b"]


def _offsets(c):
    """Borders of the documents of each sequence: uneven lengths, about a thirtieth left as padding behind them."""
    rows = []
    for i in range(c["b"]):
        share = [1 + (7 * (j + i)) % 5 for j in range(c["docs"])]
        end = c["sq"] - c["sq"] // 30
        rows.append([0] + [end * sum(share[:j + 1]) // sum(share) for j in range(c["docs"])])
    return rows


def _window(c):
    """(lo, hi) of the keys that each query row of each sequence may see, mask tensors apart: two [b][sq] lists."""
    lens, lo, hi = _lens(c), [], []
    for i in range(c["b"]):
        first = lens[i] - c["sq"] if c["at_end"] else c["skv"] - c["sq"]
        off = _offsets(c)[i] if c["docs"] else None
        los, his = [], []
        for r in range(c["sq"]):
            a, z = 0, lens[i]
            if c["causal"]:
                z = min(z, max(first + r + 1, c["prefix"]))
            if off is not None:
                mine = [(s, e) for s, e in zip(off, off[1:]) if s <= r < e]
                a, z = (max(a, mine[0][0]), min(z, mine[0][1])) if mine else (0, 0)
            los.append(a)
            his.append(max(a, z))
        lo.append(los)
        hi.append(his)
    return lo, hi


def work(c):
    if c["op"] == "linear":
        m, k, n = c["m"], c["k"], c["n"]
        extra = {"bf16": 2 * n, "f32": 4 * n, "none": 0}[c["bias"]] + (2 * m * n if c["residual"] else 0)
        return {"bytes": 2 * (m * k + n * k + m * n) + extra, "flops": 2 * m * k * n}
    lo, hi = _window(c)
    pairs = sum(z - a for rows in zip(lo, hi) for a, z in zip(*rows))
    keys = sum(max(his) - min(los) for los, his in zip(lo, hi))
    extra = {"": 0, "slopes": 4 * c["h"], "table": 4 * c["h"] * 257, "mask_pad": 2 * c["b"] * c["skv"],
             "mask_full": c["sq"] * c["skv"]}[c["bias"]]
    return {"bytes": 2 * (2 * c["b"] * c["sq"] * c["h"] * c["d"] + 2 * keys * c["hk"] * c["d"]) + extra,
            "flops": 4 * pairs * c["h"] * c["d"]}


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, scale=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    if c["op"] == "linear":
        m, k, n = c["m"], c["k"], c["n"]
        return {"case": c, "x": normal(m, k), "w": normal(n, k, scale=1.5 * k ** -0.5),
                "bias": None if c["bias"] == "none" else
                normal(n, scale=0.3, dtype=torch.float32 if c["bias"] == "f32" else torch.bfloat16),
                "residual": normal(m, n) if c["residual"] else None}
    b, h, hk, sq, skv, d = (c[x] for x in ("b", "h", "hk", "sq", "skv", "d"))

    def heads(s, n, scale=1.0):
        return normal(b, n, s, d, scale=scale) if c["head_major"] else normal(b, s, n * d, scale=scale)

    s = {"case": c, "q": heads(sq, h, 4.0 if c["cap"] else 1.5), "k": heads(skv, hk), "v": heads(skv, hk),
         "lens": None, "q_start": None, "offsets": None, "slopes": None, "table": None, "mask": None}
    if c["ragged"]:
        s["lens"] = torch.tensor(_lens(c), dtype=torch.int32, device="cuda")
        if c["at_end"]:
            s["q_start"] = s["lens"] - sq
    if c["docs"]:
        s["offsets"] = torch.tensor(_offsets(c), dtype=torch.int32, device="cuda")
    if c["bias"] == "slopes":
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, h + 1, device="cuda") / h) * \
            (0.5 + torch.rand(h, generator=g, device="cuda"))
    elif c["bias"] == "table":
        s["table"] = torch.randn(h, 257, generator=g, device="cuda")
    elif c["bias"] == "mask_pad":  # each text is padded from its own length on; the padding's mask is -inf
        n = torch.randint(1, skv + 1, (b, 1, 1, 1), generator=g, device="cuda")
        at = torch.arange(skv, device="cuda")
        s["mask"] = torch.where(at < n, 0.0, -math.inf).to(torch.bfloat16)
    elif c["bias"] == "mask_full":  # regions: a query sees a key when they share one of eight regions
        mine, theirs = (torch.randint(1, 256, (x,), generator=g, device="cuda") for x in (sq, skv))
        s["mask"] = (mine[:, None] & theirs[None, :] & 0x55) != 0
    return s


# --- one pass --------------------------------------------------------------------------------------------------------


def run(s):
    return _run_linear(s) if s["case"]["op"] == "linear" else _run_attention(s)


def _run_linear(s):
    c = s["case"]
    if own:
        from npu_ai_b200 import kernels
        return kernels.gemm(s["x"], s["w"], s["bias"], out_dtype=torch.bfloat16, residual=s["residual"],
                            activation=c["act"])
    y = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if c["act"] == "gelu":
        y = 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    elif c["act"] == "gelu_tanh":
        y = 0.5 * y * (1.0 + torch.tanh(GELU_TANH * (y + 0.044715 * y * y * y)))
    elif c["act"] == "quick_gelu":
        y = y / (1.0 + torch.exp(-1.702 * y))
    elif c["act"] == "silu":
        y = y / (1.0 + torch.exp(-y))
    else:
        y = torch.clamp(y, min=0.0)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(torch.bfloat16)


def _run_attention(s):
    c = s["case"]
    b, h, hk, sq, skv, d = (c[x] for x in ("b", "h", "hk", "sq", "skv", "d"))
    if own:
        from npu_ai_b200 import kernels
        return kernels.attention(s["q"], s["k"], s["v"], h, head_major_in=c["head_major"],
                                 head_major_out=c["head_major"], out_dtype=torch.bfloat16, kv_heads=hk,
                                 causal=c["causal"], q_start=s["q_start"], prefix_len=c["prefix"] or None,
                                 kv_lens=s["lens"], doc_offsets=s["offsets"], softcap=c["cap"] or None,
                                 slopes=s["slopes"], distance_bias=s["table"], mask=s["mask"])
    split = (lambda t, n: t) if c["head_major"] else (lambda t, n: t.unflatten(-1, (n, d)).transpose(1, 2))
    q = split(s["q"], h).float().unflatten(1, (hk, h // hk))
    k, v = (split(s[x], hk).float().unsqueeze(2) for x in ("k", "v"))
    scores = (q @ k.transpose(-1, -2) * d ** -0.5).flatten(1, 2)  # [b, h, sq, skv]
    if c["cap"]:
        scores = c["cap"] * torch.tanh(scores / c["cap"])
    key = torch.arange(skv, device=q.device)
    first = s["q_start"][:, None] if s["q_start"] is not None else skv - sq
    at = (torch.arange(sq, device=q.device) + first).expand(b, sq)[:, None, :, None]  # each query's place among the keys
    if c["bias"] == "slopes":
        scores = scores - s["slopes"][None, :, None, None] * (key - at).abs().float()
    elif c["bias"] == "table":
        scores = scores + s["table"][:, (key - at).clamp(-128, 128)[:, 0] + 128].movedim(0, 1)
    seen = torch.ones(b, 1, sq, skv, dtype=torch.bool, device=q.device)
    if s["lens"] is not None:
        seen = seen & (key < s["lens"][:, None, None, None])
    if c["causal"]:
        seen = seen & ((key <= at) | (key < c["prefix"]))
    if s["offsets"] is not None:
        which = (key[None, :, None] >= s["offsets"][:, None, :]).sum(-1)  # 0: before the first, docs + 1: behind the last
        inside = (which >= 1) & (which <= c["docs"])
        seen = seen & ((which[:, :, None] == which[:, None, :]) & inside[:, :, None])[:, None]
    if s["mask"] is not None:
        if s["mask"].dtype == torch.bool:
            seen = seen & s["mask"]
        else:
            scores = scores + s["mask"].float()
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total == 0.0, 1.0, total)).unflatten(1, (hk, h // hk))
    o = (p @ v).flatten(1, 2)  # [b, h, sq, d]
    return (o if c["head_major"] else o.transpose(1, 2).flatten(2)).to(torch.bfloat16)


# --- the definitions in 64 bits --------------------------------------------------------------------------------------


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "linear":
        w = s["w"].double().t().contiguous()
        return torch.cat([_exact_rows(c, s, w, at, min(c["m"], at + 8192)) for at in range(0, c["m"], 8192)])
    b, h, hk, sq, skv, d = (c[x] for x in ("b", "h", "hk", "sq", "skv", "d"))
    lo, hi = (torch.tensor(x, device="cuda")[:, :, None] for x in _window(c))
    j = torch.arange(skv, device="cuda")
    out = torch.empty(b, h, sq, d, dtype=torch.float64, device="cuda")
    for i in range(b):
        delta = j - ((int(s["q_start"][i]) if s["q_start"] is not None else skv - sq) +
                     torch.arange(sq, device="cuda")[:, None])
        for n in range(h):
            def head(t, at):
                return (t[i, at] if c["head_major"] else t[i, :, at * d:(at + 1) * d]).double()
            z = torch.einsum("qd,kd->qk", head(s["q"], n), head(s["k"], n // (h // hk))) / math.sqrt(d)
            if c["cap"]:
                z = torch.tanh(z / c["cap"]).mul(c["cap"])
            if s["slopes"] is not None:
                z -= s["slopes"][n].double() * delta.abs()
            if s["table"] is not None:
                z += s["table"][n].double()[delta.clip(-128, 128).add(128)]
            if c["bias"] == "mask_pad":
                z += s["mask"][i, 0].double()
            hidden = (j < lo[i]) | (j >= hi[i])
            if c["bias"] == "mask_full":
                hidden = hidden | ~s["mask"]
            z.masked_fill_(hidden, -math.inf)
            # a row that sees nothing is zero
            out[i, n] = torch.softmax(z, -1).nan_to_num(0.0) @ head(s["v"], n // (h // hk))
    return out if c["head_major"] else out.permute(0, 2, 1, 3).reshape(b, sq, h * d)


def _exact_rows(c, s, w, start, stop):
    y = s["x"][start:stop].double() @ w
    y = y if s["bias"] is None else y + s["bias"].double()
    normal = torch.distributions.Normal(torch.zeros((), dtype=torch.float64, device="cuda"), 1.0)
    act = {"gelu": lambda: y * normal.cdf(y), "quick_gelu": lambda: y * torch.sigmoid(1.702 * y),
           "gelu_tanh": lambda: y * torch.sigmoid(2.0 * GELU_TANH * (y + 0.044715 * y ** 3)),
           "silu": lambda: y * torch.sigmoid(y), "relu": lambda: torch.relu(y)}[c["act"]]()
    return act if s["residual"] is None else act + s["residual"][start:stop].double()

"""Operators of a text model's cached steps, as cases that can be timed and checked.

Three operators, each in its plain form (elementary torch operations) and as a user calls the kernels:

  rope       rotary positions: half and interleaved layouts, part of the head, frequencies scaled for long contexts, and
             the rotation back.
  append     new keys and values into the pages of a cache, the keys (and the queries) rotated on the way.
  attention  a few new tokens of each sequence against its pages: one token of a batch, one long sequence, ragged lengths.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _rope(name, b, s, h, d, **more):
    case = {"name": name, "op": "rope", "b": b, "s": s, "h": h, "d": d, "rot": d, "interleaved": False, "scaling": "",
            "start": 0, "positions": False, "inverse": False, "head_major": False, "src": "bf16", "dst": "bf16"}
    return {**case, **more}


def _append(name, b, s, h, hk, d, page, cached, **more):
    case = {"name": name, "op": "append", "b": b, "s": s, "h": h, "hk": hk, "d": d, "page": page, "cached": cached,
            "rot": d, "interleaved": False, "scaling": "", "ragged": False, "head_major": False, "src": "bf16"}
    return {**case, **more}


def _attention(name, b, h, hk, sq, d, page, cached, **more):
    case = {"name": name, "op": "attention", "b": b, "h": h, "hk": hk, "s": sq, "d": d, "page": page, "cached": cached,
            "ragged": False, "cap": 0.0, "slopes": False, "head_major": False}
    return {**case, **more}


def listed():
    return [
        # The query heads of one token, far into a long context. The smallest call.
        _rope("rope_token", 1, 1, 32, 128, start=100000, scaling="yarn"),
        # A pair of 77-token prompts of a text encoder, pairs next to each other, a quarter of each head rotated.
        _rope("rope_prompt_77", 2, 77, 12, 64, rot=16, interleaved=True, src="f32"),
        # Keys of a ragged batch rotated back to position 0, every token with a position of its own.
        _rope("rope_back_1001", 3, 1001, 8, 80, rot=40, positions=True, inverse=True, src="f32", dst="f32",
              head_major=True),
        # The query and key heads of a long prompt's fused projection. The largest rotation.
        _rope("rope_prompt_16384", 1, 16384, 40, 128, scaling="yarn"),
        # One token of each of 16 sequences: what every layer of a decoding step does before its attention.
        _append("append_tokens_16", 16, 1, 32, 8, 128, 16, 4000, ragged=True),
        # A ragged batch of prompts straight from a projection in f32, into pages that its lengths do not fill.
        _append("append_prompts_1000", 4, 1000, 8, 2, 160, 48, 100, rot=64, interleaved=True, ragged=True, src="f32"),
        # Two long prompts. The largest append.
        _append("append_prompt_8192", 2, 8192, 32, 8, 128, 64, 0, head_major=True, scaling="linear"),
        # One token against a short cache: latency.
        _attention("token_777", 1, 8, 2, 1, 64, 16, 777),
        # One token of each sequence of a full ragged batch against long caches: the largest call.
        _attention("token_16384", 16, 32, 8, 1, 128, 64, 16384, ragged=True),
        # One token of a single sequence with a very long cache: all of the GPU on eight key/value heads.
        _attention("token_131072", 1, 32, 8, 1, 128, 16, 131071),
        # Many short caches, a key/value head for every query head, capped scores.
        _attention("tokens_short_64", 64, 16, 16, 1, 80, 24, 700, ragged=True, cap=30.0),
        # A few tokens at the end of each cache of a ragged batch, linear bias by distance.
        _attention("tokens_5_slopes", 4, 8, 2, 5, 128, 32, 5001, ragged=True, slopes=True, head_major=True),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("rope", "append", "attention", "attention"))
    hk = rng.choice((1, 2, 4, 5, 8))
    h = hk * rng.choice((1, 1, 2, 3, 4, 8))
    d = rng.choice((40, 64, 64, 72, 80, 96, 128, 128, 160, 256))
    turn = {"rot": rng.choice((d, d, d // 2, d // 4 // 2 * 2)), "interleaved": rng.random() < 0.5,
            "scaling": rng.choice(("", "linear", "yarn")), "src": rng.choice(("bf16", "bf16", "f32"))}
    if op == "rope":
        b, s = _log(rng, 1, 64), _log(rng, 1, 16384)
        while b * s * h * d > 16384 * 40 * 128 // (2 if turn["src"] == "f32" else 1):
            b, s = (b + 1) // 2, s if b > 1 else s // 2
        case = _rope("", b, s, h, d, **turn, start=_log(rng, 1, 1000000), positions=rng.random() < 0.3,
                     inverse=rng.random() < 0.3, head_major=rng.random() < 0.3, dst=rng.choice(("bf16", "f32")))
        while b * s * h * d * (4 if case["dst"] == "f32" else 2) > 16384 * 40 * 128 * 2:
            b, s = (b + 1) // 2, s if b > 1 else s // 2
        case |= {"b": b, "s": s}
    elif op == "append":
        b, s = _log(rng, 1, 64), rng.choice((1, 1, 2, _log(rng, 1, 8192)))
        while b * s * (h + 2 * hk) * d * (2 if turn["src"] == "f32" else 1) > 16384 * 48 * 128:
            b, s = (b + 1) // 2, s if b > 1 else s // 2
        cached = _log(rng, 1, 8192)
        while b * (cached + s) * hk * d > 16384 * 32 * 128:
            cached = cached // 2
            b, s = (b + 1) // 2, s if b > 1 else s // 2
        case = _append("", b, s, h, hk, d, rng.choice((1, 7, 16, 16, 24, 32, 64, 256)), cached, **turn,
                       ragged=rng.random() < 0.7, head_major=rng.random() < 0.5)
    else:
        b, sq, cached = _log(rng, 1, 128), rng.choice((1, 1, 1, 2, 5, 16)), _log(rng, 16, 131072)
        while b * hk * cached * d > 12 * 8 * 16384 * 128 or b * h * sq * cached * d > 8 * 16 * 32 * 16384 * 128:
            b, cached = (b + 1) // 2, cached if b > 1 else cached // 2
        case = _attention("", b, h, hk, sq, d, rng.choice((1, 7, 16, 16, 24, 32, 64, 256)), cached,
                          ragged=rng.random() < 0.7, cap=rng.choice((0.0, 0.0, 20.0, 50.0)), slopes=rng.random() < 0.25,
                          head_major=rng.random() < 0.5)
    del case["name"]
    return case


# --- what a case holds besides its random values --------------------------------------------------------------------


def _frequencies(c):
    """Radians a position of each pair, in 64 bits, and the factor of the rotated values."""
    r, base = c["rot"], 10000.0
    f = base ** (torch.arange(0, r, 2, dtype=torch.float64) / -r)
    if c["scaling"] == "linear":
        return f / 4.0, 1.0
    if c["scaling"] == "yarn":  # a context of 4096 stretched 32 times; pairs that turn often keep their speed
        turns = 4096 * f / (2.0 * math.pi)
        keep = torch.clamp((torch.log(turns) - math.log(1.0)) / (math.log(32.0) - math.log(1.0)), 0.0, 1.0)
        return f * keep + f / 32.0 * (1.0 - keep), 0.1 * math.log(32.0) + 1.0
    return f, 1.0


def _starts(c):
    """Tokens that each sequence's cache holds before the call (append), uneven in a ragged batch."""
    return [c["cached"] - (i * c["cached"] // (2 * c["b"]) + i % 3 if c["ragged"] else 0) if c["cached"] > 3 else
            c["cached"] for i in range(c["b"])]


def _counts(c):
    """New tokens of each sequence of a padded batch: from all down to half."""
    return [max(1, c["s"] - i * c["s"] // (2 * c["b"])) if c["ragged"] else c["s"] for i in range(c["b"])]


def _lens(c):
    """Keys of each sequence, its new tokens among them: from all down to half."""
    return [max(c["s"], c["cached"] - i * c["cached"] // (2 * c["b"]) - c["cached"] % 7 * (i % 2)) if c["ragged"] else
            max(c["s"], c["cached"]) for i in range(c["b"])]


def work(c):
    size = {"bf16": 2, "f32": 4}
    if c["op"] == "rope":
        n = c["b"] * c["s"] * c["h"]
        return {"bytes": n * c["d"] * (size[c["src"]] + size[c["dst"]]) + 4 * c["rot"] +
                4 * c["b"] * (c["s"] if c["positions"] else 1), "flops": 3 * n * c["rot"]}
    if c["op"] == "append":
        n = sum(_counts(c))
        q = c["b"] * c["s"] * c["h"]
        return {"bytes": (q + 2 * n * c["hk"]) * c["d"] * (size[c["src"]] + 2) + 4 * c["rot"] + 8 * c["b"] +
                4 * sum(k // c["page"] + 1 for k in _counts(c)), "flops": 3 * (q + n * c["hk"]) * c["rot"]}
    lens = _lens(c)
    seen = sum(k * c["s"] - c["s"] * (c["s"] - 1) // 2 for k in lens)
    return {"bytes": 4 * sum(lens) * c["hk"] * c["d"] + 4 * c["b"] * c["s"] * c["h"] * c["d"] + 4 * c["b"] +
            4 * sum(-(-k // c["page"]) for k in lens) + (4 * c["h"] if c["slopes"] else 0),
            "flops": 4 * seen * c["h"] * c["d"]}


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, scale=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    b, h, d, n = c["b"], c["h"], c["d"], c["s"]
    s = {"case": c}
    if c["op"] != "attention":
        f, s["magnitude"] = _frequencies(c)
        s["freqs"] = f.cuda()
    if c["op"] == "rope":
        s["x"] = normal(*((b, h, n, d) if c["head_major"] else (b, n, h * d)), dtype=DTYPES[c["src"]])
        s["at"] = torch.randint(0, c["start"] + 1, (b, n) if c["positions"] else (b,), generator=g, device="cuda",
                                dtype=torch.int32)
        return s
    hk, page = c["hk"], c["page"]
    most = max(x + y for x, y in zip(_starts(c), _counts(c))) if c["op"] == "append" else max(_lens(c))
    width = -(-most // page)
    pages = b * width + 3
    shape = (pages, hk, page, d) if c["head_major"] else (pages, page, hk, d)
    s["k_pages"], s["v_pages"] = (normal(*shape) for _ in range(2))
    if c["head_major"]:  # the pages hold one head after the other
        s["k_pages"], s["v_pages"] = s["k_pages"].transpose(1, 2), s["v_pages"].transpose(1, 2)
    s["table"] = torch.randperm(pages, generator=g, device="cuda")[:b * width].view(b, width).to(torch.int32)
    if c["op"] == "append":
        qkv = normal(b, n, (h + 2 * hk) * d, dtype=DTYPES[c["src"]])  # one fused projection
        s["q"], s["k"], s["v"] = qkv.split((h * d, hk * d, hk * d), -1)
        s["starts"], s["counts"] = ints(_starts(c)), ints(_counts(c)) if c["ragged"] else None
        return s
    s["q"] = normal(b, n, h * d, scale=4.0 if c["cap"] else 1.5)
    s["lens"] = ints(_lens(c))
    s["slopes"] = None
    if c["slopes"]:
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, h + 1, device="cuda") / h) * \
            (0.5 + torch.rand(h, generator=g, device="cuda"))
    return s


# --- one pass --------------------------------------------------------------------------------------------------------


def run(s):
    return {"rope": _run_rope, "append": _run_append, "attention": _run_attention}[s["case"]["op"]](s)


def _run_rope(s):
    c = s["case"]
    if own:
        from npu_ai_b200 import kernels
        return kernels.rope(s["x"], s["freqs"], c["h"], s["at"], interleaved=c["interleaved"], magnitude=s["magnitude"],
                            inverse=c["inverse"], head_major=c["head_major"], out_dtype=DTYPES[c["dst"]])
    x = s["x"] if c["head_major"] else s["x"].unflatten(-1, (c["h"], c["d"])).transpose(1, 2)
    at = s["at"] if c["positions"] else s["at"][:, None] + torch.arange(c["s"], device=x.device)
    y = _turn(c, x.float(), at, s["freqs"], s["magnitude"], c["inverse"]).to(DTYPES[c["dst"]])
    return y if c["head_major"] else y.transpose(1, 2).flatten(2)


def _turn(c, x, at, freqs, magnitude, inverse=False):
    """x [b, heads, s, d] in 32 bits, rotated by the angles at[b, s] * freqs, which are worked out in 64."""
    angle = (at.double()[..., None] * freqs)[:, None]
    cos, sin = (torch.cos(angle) * magnitude).float(), (torch.sin(angle) * magnitude).float()
    if inverse:
        sin = -sin
    r = c["rot"]
    first, second = (x[..., :r:2], x[..., 1:r:2]) if c["interleaved"] else (x[..., :r // 2], x[..., r // 2:r])
    one, two = first * cos - second * sin, second * cos + first * sin
    turned = torch.stack((one, two), -1).flatten(-2) if c["interleaved"] else torch.cat((one, two), -1)
    return torch.cat((turned, x[..., r:]), -1)


def _run_append(s):
    c = s["case"]
    if own:
        from npu_ai_b200 import kernels
        q = kernels.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["starts"], counts=s["counts"],
                                 q=s["q"], heads=c["h"], freqs=s["freqs"], interleaved=c["interleaved"],
                                 magnitude=s["magnitude"])
        return q, s["k_pages"], s["v_pages"]
    at = s["starts"][:, None] + torch.arange(c["s"], device=s["q"].device)
    split = (lambda t, n: t.unflatten(-1, (n, c["d"])).transpose(1, 2).float())
    q, k = (_turn(c, split(s[x], n), at, s["freqs"], s["magnitude"]) for x, n in (("q", c["h"]), ("k", c["hk"])))
    k, v = (t.transpose(1, 2).to(torch.bfloat16) for t in (k, split(s["v"], c["hk"])))  # [b, s, hk, d]
    for i, n in enumerate(_counts(c)):
        where = at[i, :n]
        page = s["table"][i][(where // c["page"]).long()].long()
        s["k_pages"][page, (where % c["page"]).long()] = k[i, :n]
        s["v_pages"][page, (where % c["page"]).long()] = v[i, :n]
    return q.transpose(1, 2).flatten(2).to(torch.bfloat16), s["k_pages"], s["v_pages"]


def _run_attention(s):
    c = s["case"]
    b, h, hk, sq, d = (c[x] for x in ("b", "h", "hk", "s", "d"))
    if own:
        from npu_ai_b200 import kernels
        return kernels.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], h,
                                       out_dtype=torch.bfloat16, softcap=c["cap"] or None, slopes=s["slopes"])
    k, v = (s[x][s["table"].long()].flatten(1, 2).transpose(1, 2).float().unsqueeze(2) for x in ("k_pages", "v_pages"))
    q = s["q"].unflatten(-1, (h, d)).transpose(1, 2).float().unflatten(1, (hk, h // hk))
    scores = (q @ k.transpose(-1, -2) * d ** -0.5).flatten(1, 2)  # [b, h, sq, width * page]
    if c["cap"]:
        scores = c["cap"] * torch.tanh(scores / c["cap"])
    key = torch.arange(scores.shape[-1], device=q.device)
    at = (s["lens"][:, None] - sq + torch.arange(sq, device=q.device))[:, None, :, None]
    if s["slopes"] is not None:
        scores = scores - s["slopes"][:, None, None] * (at - key).abs().float()
    scores = torch.where(key <= at, scores, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    v = torch.where((key < s["lens"][:, None])[:, None, None, :, None], v, 0.0)  # what lies behind the last key is not read
    o = (p.unflatten(1, (hk, h // hk)) @ v).flatten(1, 2)
    return o.transpose(1, 2).flatten(2).to(torch.bfloat16)


# --- the definitions in 64 bits --------------------------------------------------------------------------------------


def _exact_turn(c, x, at, freqs, magnitude, inverse=False):
    """x [s, heads, d] at the positions at[s], each pair a complex number times magnitude e^{i angle}."""
    r, half = c["rot"], c["rot"] // 2
    i = torch.arange(half, device=x.device)
    re, im = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half)
    angle = torch.outer(at.double(), freqs if not inverse else -freqs)[:, None, :]
    z = torch.complex(x[..., re], x[..., im]) * torch.polar(torch.full_like(angle, magnitude), angle)
    y = x.clone()
    y[..., re], y[..., im] = z.real, z.imag
    return y


def exact(c, seed):
    s = prepare(c, seed)
    b, n, h, d = c["b"], c["s"], c["h"], c["d"]
    if c["op"] == "rope":
        rows = []
        for i in range(b):
            x = (s["x"][i].transpose(0, 1) if c["head_major"] else s["x"][i].view(n, h, d)).double()
            at = s["at"][i] if c["positions"] else int(s["at"][i]) + torch.arange(n, device="cuda")
            y = _exact_turn(c, x, at, s["freqs"], s["magnitude"], c["inverse"])
            rows.append(y.transpose(0, 1) if c["head_major"] else y.reshape(n, h * d))
        return torch.stack(rows)
    hk, page = c["hk"], c["page"]
    if c["op"] == "append":
        kp, vp = s["k_pages"].double(), s["v_pages"].double()
        qs = []
        for i, (first, m) in enumerate(zip(_starts(c), _counts(c))):
            at = torch.arange(first, first + n, device="cuda")
            turned = [_exact_turn(c, s[x][i].reshape(n, -1, d).double(), at, s["freqs"], s["magnitude"]) for x in ("q", "k")]
            qs.append(turned[0].reshape(n, h * d))
            slot = s["table"][i].long().repeat_interleave(page) * page + torch.arange(page, device="cuda").repeat(
                s["table"].shape[1])  # of every position of the sequence
            slot = slot[first:first + m]
            for pool, new in ((kp, turned[1]), (vp, s["v"][i].reshape(n, hk, d).double())):
                pool[slot // page, slot % page] = new[:m]
        return torch.stack(qs), kp, vp
    out = torch.empty(b, n, h, d, dtype=torch.float64, device="cuda")
    for i, m in enumerate(_lens(c)):
        mine = s["table"][i, :-(-m // page)].long()
        for j in range(hk):
            k, v = (s[x][mine, :, j].reshape(-1, d)[:m].double() for x in ("k_pages", "v_pages"))
            heads = slice(j * (h // hk), (j + 1) * (h // hk))
            q = s["q"][i].view(n, h, d)[:, heads].double()
            z = torch.einsum("tad,kd->tak", q, k) / math.sqrt(d)
            if c["cap"]:
                z = torch.tanh(z / c["cap"]).mul(c["cap"])
            ahead = torch.arange(m, device="cuda") - torch.arange(m - n, m, device="cuda")[:, None]  # of the query, [n, m]
            if s["slopes"] is not None:
                z += s["slopes"][heads].double()[:, None] * ahead[:, None]
            z.masked_fill_((ahead > 0)[:, None], -math.inf)
            out[i, :, heads] = torch.einsum("tak,kd->tad", torch.softmax(z, -1), v)
    return out.view(b, n, h * d)

"""Masked attention on the B200 (npub200_attention_masked through kernels.attention) against the formula in 64 bits.

Tolerance, per element, from the arithmetic and not from a run. P is rounded to bf16 (relative 2^-8 at most), so o is off
by at most 2^-8 A with A = sum_j p_j |v_j|. The scores are f32: a dot product of D bf16 products is off by D 2^-23
sum|q k|, the cap by a few 2^-22 of the cap, each bias and the base change by half a step of the largest score; an error
e in a score moves p by 2e relative (numerator and denominator). The output rounds once more.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
INF = float("inf")


def _qkv(B, H, Hk, Sq, Skv, D, seed, dev, q_scale=1.0, head_major=False):
    g = torch.Generator(device=dev).manual_seed(seed)

    def make(S, n, s=1.0):
        shape = (B, n, S, D) if head_major else (B, S, n * D)
        return (torch.randn(*shape, generator=g, device=dev) * s).to(BF16)
    return make(Sq, H, q_scale), make(Skv, Hk), make(Skv, Hk)


def _heads(t, n, head_major):
    t = t.double()
    return t if head_major else t.unflatten(-1, (n, -1)).transpose(1, 2)


def oracle(q, k, v, H, Hk, head_major=False, scale=None, causal=False, q_start=None, prefix_len=None, kv_lens=None,
           doc_offsets=None, softcap=None, slopes=None, distance_bias=None, mask=None):
    """(o, tolerance before the output's rounding), both [B, H, Sq, D] in 64 bits."""
    dev = q.device
    q, k, v = _heads(q, H, head_major), _heads(k, Hk, head_major), _heads(v, Hk, head_major)
    B, _, Sq, D = q.shape
    Skv = k.shape[2]
    k, v = (t.repeat_interleave(H // Hk, 1) for t in (k, v))
    scale = D ** -0.5 if scale is None else scale
    i, j = torch.arange(Sq, device=dev)[:, None], torch.arange(Skv, device=dev)[None]
    start = torch.as_tensor(Skv - Sq if q_start is None else q_start, device=dev).reshape(-1, 1, 1, 1)
    p = (i + start).expand(B, 1, Sq, 1)
    seen = torch.ones(B, H, Sq, Skv, dtype=torch.bool, device=dev)
    if kv_lens is not None:
        seen &= j < kv_lens.view(B, 1, 1, 1)
    if causal:
        prefix = torch.as_tensor(0 if prefix_len is None else prefix_len, device=dev).reshape(-1, 1, 1, 1)
        seen &= (j <= p) | (j < prefix)
    if doc_offsets is not None:
        off = doc_offsets.reshape(-1, doc_offsets.shape[-1]).expand(B, -1)
        for b in range(B):
            same = torch.zeros(Sq, Skv, dtype=torch.bool, device=dev)
            for s, e in zip(off[b].tolist(), off[b].tolist()[1:]):
                same[max(s, 0):max(e, 0), max(s, 0):max(e, 0)] = True
            seen[b] &= same
    seen = seen.clone()
    # keys that the lengths, causal and document rules hide from every row may hold anything
    used = seen.any(2)
    v = torch.where(used[..., None], v, 0.0)
    k = torch.where(used[..., None], k, 0.0)
    s = q @ k.transpose(-1, -2) * scale
    e = D * 2.0 ** -23 * scale * (q.abs() @ k.abs().transpose(-1, -2)).amax(-1, keepdim=True)
    big = s.abs()
    if softcap is not None:
        s = softcap * torch.tanh(s / softcap)
        e = e + 16 * 2.0 ** -23 * softcap
    if slopes is not None:
        bias = -slopes.double().view(1, H, 1, 1) * (j - p).abs()
        s, big = s + bias, big + bias.abs()
    if distance_bias is not None:
        R = distance_bias.shape[1] // 2
        bias = distance_bias.double()[:, (j - p).clamp(-R, R)[:, 0] + R].transpose(0, 1)
        s, big = s + bias, big + bias.abs()
    if mask is not None:
        m4 = mask if mask.dim() == 4 else mask[None, None]
        if mask.dtype == torch.bool:
            seen &= m4
        else:
            s = s + m4.double()
            seen &= m4 > -INF
            big = big + torch.where(m4.double().abs() < 1e30, m4.double().abs(), 0.0)
    e = e + 8 * 2.0 ** -24 * torch.where(seen, big, 0.0).amax(-1, keepdim=True)
    s = torch.where(seen, s, -INF)
    top = s.amax(-1, keepdim=True)
    w = torch.where(seen, torch.exp(s - torch.where(top == -INF, 0.0, top)), 0.0)
    w = w / w.sum(-1, keepdim=True).clamp_min(1e-300)
    return w @ v, (2.0 ** -8 + 2.0 ** -18 + 2.5 * e) * (w @ v.abs()) + 1e-30


def check(out, ref, tol, H, head_major):
    o = _heads(out, H, head_major)
    tol = tol + (2.0 ** -8 if out.dtype == BF16 else 2.0 ** -23) * (ref.abs() + tol)
    err = (o - ref).abs()
    assert bool(torch.isfinite(o).all()), "non-finite output"
    assert bool((err <= tol).all()), f"{float((err / tol).max())} of the tolerance"
    assert bool((o[(ref == 0).all(-1)] == 0).all()), "a row that sees nothing is not zero"


def run(dev, B, H, Hk, Sq, Skv, D, seed=0, q_scale=1.0, head_major=False, out_dtype=torch.float32, variant=0, **kw):
    from npu_ai_b200 import kernels
    q, k, v = _qkv(B, H, Hk, Sq, Skv, D, seed, dev, q_scale, head_major)
    out = kernels.attention(q, k, v, H, head_major_in=head_major, head_major_out=head_major, out_dtype=out_dtype,
                            variant=variant, kv_heads=Hk, **kw)
    kernels.check_status(dev)
    check(out, *oracle(q, k, v, H, Hk, head_major, **kw), H, head_major)
    return q, k, v, out


def ints(dev, *x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("D", [8, 24, 40, 64, 72, 80, 96, 104, 128, 136, 160, 192, 200, 256])
@pytest.mark.parametrize("S", [1, 77, 128, 300])
def test_causal_every_head_dim(cuda_device, D, S):
    run(cuda_device, 2, 4, 2, S, S, D, seed=S + D, causal=True)
    run(cuda_device, 1, 3, 3, S, S, D, seed=S + D, causal=True, out_dtype=BF16, head_major=True)


@pytest.mark.parametrize("heads", [(1, 1), (8, 8), (8, 1), (12, 4), (14, 2), (130, 1), (6, 3)])
@pytest.mark.parametrize("sizes", [(1, 500), (5, 77), (33, 64), (129, 129), (200, 1000)])
@pytest.mark.parametrize("head_major", [False, True])
def test_grouped_heads(cuda_device, heads, sizes, head_major):
    """Groups of every kind of size (few queries share a tile, many do not; 130 heads do not fit one tile)."""
    H, Hk = heads
    run(cuda_device, 2, H, Hk, *sizes, 64, seed=H + sizes[0], head_major=head_major, causal=sizes[0] > 1)
    run(cuda_device, 2, H, Hk, *sizes, 40, seed=H + sizes[1], head_major=head_major, softcap=5.0, q_scale=3.0)


@pytest.mark.parametrize("splits", [0, 1, 2, 3, 7, 32, 33, 64])
def test_split_keys(cuda_device, splits):
    """Parts of a row's keys joined: more parts than tiles (empty parts), more than 32, ragged lengths, both types."""
    lens = ints(cuda_device, 1000, 1, 0, 64)
    for kw in (dict(), dict(causal=True, q_start=lens - 3), dict(softcap=20.0, q_scale=4.0)):
        run(cuda_device, 4, 8, 2, 3, 1000, 128, variant=splits, kv_lens=lens, **kw)
        run(cuda_device, 4, 8, 2, 3, 1000, 256, variant=splits, kv_lens=lens, out_dtype=BF16, head_major=True, **kw)
    run(cuda_device, 1, 2, 2, 200, 513, 40, variant=splits, causal=True)


def test_one_token_long_cache(cuda_device):
    lens = ints(cuda_device, 20000, 12345, 7)
    run(cuda_device, 3, 16, 4, 1, 20000, 128, kv_lens=lens)
    run(cuda_device, 3, 4, 4, 1, 20000, 64, kv_lens=lens, q_start=lens - 1, causal=True,
        slopes=torch.tensor([0.5, 0.1, 0.01, 0.0], device=cuda_device))


def test_lengths_zero_one_full_and_out_of_range(cuda_device):
    """Lengths below 0 and above the tensor are clamped."""
    from npu_ai_b200 import kernels
    lens = ints(cuda_device, 0, 1, 63, 64, 65, 300)
    run(cuda_device, 6, 4, 2, 100, 300, 80, kv_lens=lens)
    q, k, v = _qkv(2, 4, 2, 10, 300, 80, 3, cuda_device)
    a = kernels.attention(q, k, v, 4, kv_lens=ints(cuda_device, -5, 2 ** 31 - 1))
    b = kernels.attention(q, k, v, 4, kv_lens=ints(cuda_device, 0, 300))
    assert torch.equal(a, b) and bool((a[0] == 0).all())


@pytest.mark.parametrize("splits", [1, 5])
def test_stale_cache_memory_is_never_used(cuda_device, splits):
    """NaN and infinities behind a sequence's length, past the causal end of every row and outside every document."""
    from npu_ai_b200 import kernels
    for D in (40, 128, 160):
        q, k, v = _qkv(3, 4, 2, 5, 700, D, D, cuda_device)
        lens = ints(cuda_device, 130, 0, 699)
        for t, bad in ((k, float("nan")), (v, INF)):
            for b, n in enumerate(lens.tolist()):
                t[b, n:] = bad
        kw = dict(kv_lens=lens)
        out = kernels.attention(q, k, v, 4, variant=splits, **kw)
        check(out, *oracle(q, k, v, 4, 2, **kw), 4, False)
        q, k, v = _qkv(1, 2, 2, 200, 200, D, D, cuda_device)
        k[:, :33], v[:, :33], k[:, 150:], v[:, 150:] = INF, float("nan"), float("nan"), float("nan")
        kw = dict(doc_offsets=ints(cuda_device, 33, 100, 150), causal=True)
        out = kernels.attention(q, k, v, 2, variant=splits, **kw)
        check(out, *oracle(q, k, v, 2, 2, **kw), 2, False)
        q, k, v = _qkv(1, 2, 2, 20, 200, D, D, cuda_device)
        k[:, 100:], v[:, 100:] = float("nan"), float("nan")
        kw = dict(causal=True, q_start=80)
        out = kernels.attention(q, k, v, 2, variant=splits, **kw)
        check(out, *oracle(q, k, v, 2, 2, **kw), 2, False)
    kernels.check_status(cuda_device)


@pytest.mark.parametrize("Sq,Skv,start", [(100, 300, None), (100, 300, 0), (100, 300, 250), (100, 300, -50), (64, 64, 1),
                                          (300, 100, None), (100, 100, -100), (3, 200, 10 ** 12), (3, 200, -10 ** 12)])
def test_causal_positions(cuda_device, Sq, Skv, start):
    """Positions before the first key (rows that see nothing), past the last, and far out of range."""
    run(cuda_device, 2, 4, 2, Sq, Skv, 64, causal=True, q_start=start)
    if start is not None and abs(start) < 2 ** 31:
        run(cuda_device, 2, 4, 2, Sq, Skv, 64, causal=True, q_start=ints(cuda_device, start, start + 7))


@pytest.mark.parametrize("prefix", [0, 1, 64, 100, 299, 300, 5000])
def test_prefix(cuda_device, prefix):
    run(cuda_device, 2, 4, 2, 300, 300, 64, causal=True, prefix_len=prefix)
    run(cuda_device, 2, 4, 2, 300, 300, 80, causal=True, prefix_len=ints(cuda_device, prefix, 17),
        kv_lens=ints(cuda_device, 250, 300))


@pytest.mark.parametrize("causal", [False, True])
def test_documents(cuda_device, causal):
    """Uneven, empty and single-token documents, tokens before the first and behind the last, borders per sequence."""
    S = 400
    for off in ((0, 400), (0, 1, 2, 2, 2, 65, 300, 390), (10, 10), (100, 228, 228, 400), (5,), (0, 0, 0, 400),
                tuple(range(0, 401, 5))):
        run(cuda_device, 2, 2, 2, S, S, 64, causal=causal, doc_offsets=ints(cuda_device, *off))
    off = torch.stack([ints(cuda_device, 0, 7, 300, 400), ints(cuda_device, 3, 4, 4, 350)])
    run(cuda_device, 2, 4, 1, S, S, 128, causal=causal, doc_offsets=off, out_dtype=BF16,
        distance_bias=torch.randn(4, 33, device=cuda_device))


def test_documents_with_borders_out_of_range(cuda_device):
    """Borders outside the sequence or out of order read and write nothing they should not."""
    from npu_ai_b200 import kernels
    q, k, v = _qkv(1, 2, 2, 200, 200, 64, 5, cuda_device)
    a = kernels.attention(q, k, v, 2, doc_offsets=ints(cuda_device, -50, 100, 100000))
    check(a, *oracle(q, k, v, 2, 2, doc_offsets=ints(cuda_device, 0, 100, 200)), 2, False)
    b = kernels.attention(q, k, v, 2, doc_offsets=ints(cuda_device, 150, 20, 90, -4, 180))
    kernels.check_status(cuda_device)
    assert bool(torch.isfinite(b).all())


@pytest.mark.parametrize("cap", [0.5, 5.0, 30.0, 1e6])
def test_softcap(cuda_device, cap):
    run(cuda_device, 2, 4, 2, 130, 257, 64, q_scale=6.0, softcap=cap)
    run(cuda_device, 2, 4, 2, 130, 130, 128, q_scale=6.0, softcap=cap, causal=True, scale=0.3)


@pytest.mark.parametrize("R", [0, 1, 16, 128, 1000])
def test_distance_bias(cuda_device, R):
    g = torch.Generator(device=cuda_device).manual_seed(R)
    table = torch.randn(4, 2 * R + 1, generator=g, device=cuda_device) * 3
    run(cuda_device, 2, 4, 2, 300, 300, 64, distance_bias=table)
    run(cuda_device, 2, 4, 2, 5, 700, 64, distance_bias=table, q_start=ints(cuda_device, 100, 650), causal=True)
    run(cuda_device, 2, 4, 4, 200, 90, 160, distance_bias=table, softcap=8.0, q_scale=3.0)


def test_slopes(cuda_device):
    slopes = torch.tensor([0.5, 0.0, 0.01, -0.02], device=cuda_device)
    run(cuda_device, 2, 4, 2, 300, 300, 64, slopes=slopes)
    run(cuda_device, 2, 4, 1, 4, 900, 128, slopes=slopes, causal=True, kv_lens=ints(cuda_device, 900, 500),
        q_start=ints(cuda_device, 896, 496))


def _masks(B, H, Sq, Skv, dev, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    keep = torch.rand(B, H, Sq, Skv, generator=g, device=dev) < 0.6
    keep[:, :, Sq // 2] = False          # a row that the mask leaves nothing
    keep[:, :, 0, 1:] = False            # and one with a single key
    add = torch.where(keep, torch.randn(B, H, Sq, Skv, generator=g, device=dev), -INF)
    return keep, add


@pytest.mark.parametrize("Skv", [1, 77, 128, 200])
@pytest.mark.parametrize("shape", ["bhqk", "b11k", "11qk", "1hqk", "qk", "b1qk"])
def test_mask_tensors(cuda_device, Skv, shape):
    """Every broadcast of a bool, bf16 and f32 mask, with rows that have none, one and some of the keys."""
    B, H, Sq = 2, 4, 70
    for seed, (t, dtype) in enumerate(((0, torch.bool), (1, BF16), (1, torch.float32))):
        m = _masks(B, H, Sq, Skv, cuda_device, seed)[t].to(dtype)
        cut = {"bhqk": m, "b11k": m[:, :1, 3:4], "11qk": m[:1, :1], "1hqk": m[:1], "qk": m[1, 1], "b1qk": m[:, 2:3]}
        run(cuda_device, B, H, 2, Sq, Skv, 64, mask=cut[shape])
        run(cuda_device, B, H, 4, Sq, Skv, 40, mask=cut[shape], softcap=10.0, q_scale=3.0, out_dtype=BF16)
    run(cuda_device, B, H, 2, Skv, Skv, 64, causal=True, mask=_masks(B, H, Skv, Skv, cuda_device, 9)[0])


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
def test_mask_of_the_lowest_value(cuda_device, dtype):
    """The type's lowest finite value is a score: next to others it hides a key, alone it gives the average."""
    low = torch.finfo(dtype).min
    m = torch.zeros(1, 1, 40, 150, dtype=dtype, device=cuda_device)
    m[..., 10:] = low
    m[:, :, 7] = low
    m[:, :, 8, 100:] = -INF
    m[:, :, 8, :100] = low
    m[:, :, 9] = -INF
    q, k, v, out = run(cuda_device, 1, 2, 2, 40, 150, 64, mask=m)
    mean = v.double().mean(1)
    assert float((out[:, 7].double() - mean).abs().max()) <= 2.0 ** -8 * float(v.double().abs().mean(1).max())


def test_running_max_moves_over_masked_tiles(cuda_device):
    """Rows whose first tiles are hidden, with much larger scores in later tiles (the O correction path)."""
    from npu_ai_b200 import kernels
    g = torch.Generator(device=cuda_device).manual_seed(7)
    q, k, v = _qkv(1, 2, 2, 256, 1024, 64, 1, cuda_device, 2.0)
    k = (k.float() * torch.linspace(0.2, 6.0, 1024, device=cuda_device).view(1, -1, 1)).to(BF16)
    keep = torch.rand(256, 1024, generator=g, device=cuda_device) < 0.3
    keep[::3, :500] = False
    for variant in (1, 4):
        out = kernels.attention(q, k, v, 2, mask=keep, variant=variant)
        kernels.check_status(cuda_device)
        check(out, *oracle(q, k, v, 2, 2, mask=keep), 2, False)


def test_everything_together(cuda_device):
    """All modifiers at once, as one call of a decoder: grouped heads, lengths, prefix, cap, both biases and a mask."""
    dev = cuda_device
    for Sq, Skv, D in ((200, 333, 80), (4, 2000, 128)):
        kw = dict(causal=True, q_start=ints(dev, Skv - Sq, 50, 0), prefix_len=ints(dev, 20, 0, 100),
                  kv_lens=ints(dev, Skv, Skv // 2, 0), softcap=15.0, slopes=torch.rand(8, device=dev) * 0.1,
                  distance_bias=torch.randn(8, 65, device=dev), mask=_masks(3, 8, Sq, Skv, dev, 3)[1][:, :1].to(BF16))
        run(dev, 3, 8, 2, Sq, Skv, D, q_scale=3.0, **kw)
        run(dev, 3, 8, 8, Sq, Skv, D, q_scale=3.0, head_major=True, out_dtype=BF16, **kw)


def test_strided_views_and_untouched_memory(cuda_device):
    """Padded rows for every operand, an output view whose surroundings stay, a cache larger than the call."""
    from npu_ai_b200 import kernels
    B, H, Hk, Sq, Skv, D = 2, 6, 2, 50, 90, 40
    q, k, v = _qkv(B, H, Hk, Sq, Skv, D, 4, cuda_device)

    def padded(t, extra_rows):
        buf = torch.full((B, t.shape[1] + extra_rows, t.shape[2] + 16), float("nan"), dtype=BF16, device=cuda_device)
        buf[:, :t.shape[1], :t.shape[2]] = t
        return buf[:, :t.shape[1], :t.shape[2]]
    for variant in (1, 3):
        buf = torch.full((B, Sq + 3, H * D + 12), 5.0, device=cuda_device)
        kernels.attention(padded(q, 5), padded(k, 100), padded(v, 100), H, out=buf[:, :Sq, :H * D], causal=True,
                          variant=variant)
        kernels.check_status(cuda_device)
        check(buf[:, :Sq, :H * D], *oracle(q, k, v, H, Hk, causal=True), H, False)
        assert bool((buf[:, Sq:] == 5.0).all()) and bool((buf[..., H * D:] == 5.0).all())


def test_graph_streams_and_repeats(cuda_device):
    """Captured and replayed with new lengths, two graphs and an eager call at once on several streams, same bits."""
    from npu_ai_b200 import kernels
    q, k, v = _qkv(2, 8, 2, 1, 4000, 128, 3, cuda_device)
    lens = ints(cuda_device, 4000, 100)
    eager = kernels.attention(q, k, v, 8, kv_lens=lens)
    outs, graphs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(kernels.attention(q, k, v, 8, kv_lens=lens))
        graphs.append(g)
    streams = [torch.cuda.Stream(cuda_device) for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[2]):
            other = kernels.attention(q, k, v, 8, kv_lens=lens)
    torch.cuda.synchronize()
    assert all(torch.equal(o, eager) for o in (*outs, other))
    lens.copy_(ints(cuda_device, 77, 4000))
    graphs[0].replay()
    torch.cuda.synchronize()
    check(outs[0], *oracle(q, k, v, 8, 2, kv_lens=lens), 8, False)


def test_lengths_written_by_the_previous_kernel(cuda_device):
    """Lengths, positions and masks produced on the stream right before the call (programmatic launch must wait)."""
    from npu_ai_b200 import kernels
    q, k, v = _qkv(4, 8, 8, 64, 512, 64, 3, cuda_device)
    x = torch.randn(512, 512, device=cuda_device).to(BF16)
    for n in (1, 100, 512, 3):
        kernels.gemm(x, x)
        lens = torch.full((4,), n, dtype=torch.int32, device=cuda_device)
        out = kernels.attention(q, k, v, 8, kv_lens=lens)
        out2 = kernels.attention(out.to(BF16), k, v, 8, kv_lens=lens)
        check(out, *oracle(q, k, v, 8, 8, kv_lens=lens), 8, False)
        check(out2, *oracle(out.to(BF16), k, v, 8, 8, kv_lens=lens), 8, False)


def test_forced_timeout_reports_status_and_recovers(cuda_device):
    from npu_ai_b200 import kernels
    q, k, v = _qkv(1, 2, 2, 256, 512, 40, 2, cuda_device)
    kernels.status(cuda_device)
    kernels.set_wait_timeout_ns(2_000_000)
    kernels.set_debug_flags(1)
    try:
        kernels.attention(q, k, v, 2, causal=True)
        with pytest.raises(RuntimeError, match="failure status"):
            kernels.check_status(cuda_device)
    finally:
        kernels.set_debug_flags(0)
        kernels.set_wait_timeout_ns(0)
    run(cuda_device, 1, 2, 2, 256, 512, 40, causal=True)


@pytest.mark.parametrize("variant", [1, 2])
def test_forced_timeout_with_two_streams(cuda_device, variant):
    """The same with two streams of key tiles in a CTA (eight tiles, whole and in two parts)."""
    from npu_ai_b200 import kernels
    q, k, v = _qkv(1, 2, 2, 256, 512, 64, 2, cuda_device)
    mask = torch.ones(256, 512, dtype=torch.bool, device=cuda_device)
    kernels.status(cuda_device)
    kernels.set_wait_timeout_ns(2_000_000)
    kernels.set_debug_flags(1)
    try:
        kernels.attention(q, k, v, 2, mask=mask, variant=variant)
        with pytest.raises(RuntimeError, match="failure status"):
            kernels.check_status(cuda_device)
    finally:
        kernels.set_debug_flags(0)
        kernels.set_wait_timeout_ns(0)
    run(cuda_device, 1, 2, 2, 256, 512, 64, mask=mask, variant=variant)


def test_ctypes_binding_gives_the_same(cuda_device, monkeypatch):
    """Without the torch operators the same call goes through ctypes."""
    from npu_ai_b200 import _lib, kernels
    q, k, v = _qkv(2, 8, 2, 7, 900, 80, 5, cuda_device)
    kw = dict(causal=True, kv_lens=ints(cuda_device, 900, 333), q_start=ints(cuda_device, 893, 326), softcap=9.0,
              slopes=torch.rand(8, device=cuda_device), distance_bias=torch.randn(8, 9, device=cuda_device),
              prefix_len=ints(cuda_device, 4, 5), mask=_masks(2, 1, 7, 900, cuda_device, 2)[1].to(BF16))
    a = kernels.attention(q, k, v, 8, **kw)
    s = torch.randn(1, 100, 80, device=cuda_device).to(BF16)
    kd = dict(doc_offsets=ints(cuda_device, 0, 30, 90))
    c = kernels.attention(s, s, s, 2, **kd)
    monkeypatch.setattr(_lib, "torch_ops", lambda: None)
    assert torch.equal(a, kernels.attention(q, k, v, 8, **kw))
    assert torch.equal(c, kernels.attention(s, s, s, 2, **kd))


@pytest.mark.parametrize("B,H,Hk,Sq,Skv,D", [
    (1, 2, 1, 1, 777, 64), (1, 4, 4, 300, 1100, 64), (1, 2, 2, 1000, 2000, 40), (1, 3, 3, 128, 600, 136), (2, 6, 2, 9, 450, 72),
    (1, 1, 1, 40, 1000, 256), (1, 2, 2, 1, 800, 8), (3, 8, 1, 3, 300, 200)])
@pytest.mark.parametrize("variant", [0, 2, 3, 4, 7, 13, 16])
def test_parts_joined_by_a_cluster(cuda_device, B, H, Hk, Sq, Skv, D, variant):
    """Few parts of few CTAs are joined through the shared memory of a cluster: parts without a tile, rows that a part
    does not see, output rows of every alignment."""
    from npu_ai_b200 import kernels
    lens = ints(cuda_device, *[max(Skv - 200 * b, 1) for b in range(B)])
    run(cuda_device, B, H, Hk, Sq, Skv, D, causal=True, kv_lens=lens, variant=variant, seed=Skv)
    run(cuda_device, B, H, Hk, Sq, Skv, D, softcap=6.0, q_scale=4.0, head_major=True, out_dtype=BF16, variant=variant, seed=1)
    q, k, v = _qkv(B, H, Hk, Sq, Skv, D, 2, cuda_device)
    buf = torch.full((B, Sq, H * D + 3), 7.0, dtype=BF16, device=cuda_device)
    view = buf[..., 1:H * D + 1]
    kernels.attention(q, k, v, H, kv_heads=Hk, kv_lens=lens, out=view, variant=variant)
    kernels.check_status(cuda_device)
    check(view.contiguous(), *oracle(q, k, v, H, Hk, kv_lens=lens), H, False)
    view.fill_(7.0)
    assert bool((buf == 7.0).all())


@pytest.mark.parametrize("cap", [1e-30, 1e-6, 1e6, 1e30])
def test_extreme_caps(cuda_device, cap):
    """Caps that flatten every score and caps that change none, at the ends of the range."""
    run(cuda_device, 2, 4, 2, 70, 300, 64, q_scale=3.0, softcap=cap, causal=True)


@pytest.mark.parametrize("B,H,Hk,Sq,Skv,D", [
    (1, 2, 2, 128, 256, 64), (1, 2, 2, 128, 255, 64), (1, 2, 2, 128, 320, 64), (3, 4, 2, 300, 321, 80), (2, 2, 1, 200, 449, 96),
    (2, 4, 4, 130, 1000, 128), (2, 8, 4, 500, 500, 160), (2, 8, 8, 2100, 300, 136), (1, 4, 4, 777, 777, 40)])
def test_two_streams_of_key_tiles(cuda_device, B, H, Hk, Sq, Skv, D):
    """Few CTAs, or head dims of which an SM holds one CTA, over at least four key tiles: even and odd numbers of tiles,
    rows that see a tile of one stream only, rows that see nothing."""
    lens = ints(cuda_device, *[max(Skv - 130 * b, 1) for b in range(B)])
    run(cuda_device, B, H, Hk, Sq, Skv, D, causal=True, kv_lens=lens, seed=Skv)
    run(cuda_device, B, H, Hk, Sq, Skv, D, causal=True, q_start=-70, head_major=True, out_dtype=BF16, seed=Skv + 1)
    run(cuda_device, B, H, Hk, Sq, Skv, D, softcap=3.0, q_scale=8.0, seed=Skv + 2)
    one = torch.zeros(Sq, Skv, dtype=torch.bool, device=cuda_device)
    one[torch.arange(Sq), torch.arange(Sq) * 7 % Skv] = True  # a single key a row
    one[3] = False
    run(cuda_device, B, H, Hk, Sq, Skv, D, mask=one, seed=Skv + 3)
    slopes = torch.rand(H, device=cuda_device)
    table = torch.randn(H, 41, device=cuda_device)
    run(cuda_device, B, H, Hk, Sq, Skv, D, slopes=slopes, distance_bias=table, kv_lens=lens, seed=Skv + 4)


@pytest.mark.parametrize("Skv", [320, 333])
def test_bool_masks_of_any_byte(cuda_device, Skv):
    """Any nonzero byte shows a key, in rows that 16-byte words divide and in others, for many rows and for one."""
    from npu_ai_b200 import kernels
    g = torch.Generator(device=cuda_device).manual_seed(Skv)
    raw = torch.randint(0, 256, (200, Skv), generator=g, device=cuda_device, dtype=torch.uint8)
    raw *= torch.randint(0, 2, (200, Skv), generator=g, device=cuda_device, dtype=torch.uint8)
    raw[:, 7] = 2
    q, k, v = _qkv(2, 4, 4, 200, Skv, 64, 1, cuda_device)
    for bytes_ in (raw, raw[:1]):
        out = kernels.attention(q, k, v, 4, mask=bytes_.view(torch.bool))
        kernels.check_status(cuda_device)
        check(out, *oracle(q, k, v, 4, 4, mask=(bytes_ != 0).expand(200, Skv)), 4, False)


def test_positions_at_the_ends_of_64_bits(cuda_device):
    from npu_ai_b200 import kernels
    q, k, v = _qkv(1, 2, 2, 130, 100, 64, 1, cuda_device)
    last = kernels.attention(q, k, v, 2, causal=True, q_start=2 ** 63 - 1)
    first = kernels.attention(q, k, v, 2, causal=True, q_start=-2 ** 63)
    far = kernels.attention(q, k, v, 2, causal=True, prefix_len=2 ** 63 - 1, q_start=-2 ** 63)
    kernels.check_status(cuda_device)
    ref = oracle(q, k, v, 2, 2)
    check(last, *ref, 2, False)
    check(far, *ref, 2, False)
    assert bool((first == 0).all())


def test_broadcast_and_odd_strides(cuda_device):
    """A cache shared by the whole batch (stride 0) is refused; single-row dimensions may have any stride."""
    from npu_ai_b200 import kernels
    q, k, v = _qkv(3, 4, 2, 5, 300, 64, 1, cuda_device)
    with pytest.raises(ValueError, match="strides"):
        kernels.attention(q, k[:1].expand(3, -1, -1), v[:1].expand(3, -1, -1), 4, kv_heads=2, causal=True)
    one = q[:1, :1].as_strided((1, 1, 256), (3, 5, 1))
    out = kernels.attention(one, k[:1], v[:1], 4, kv_heads=2, causal=True)
    kernels.check_status(cuda_device)
    check(out, *oracle(q[:1, :1], k[:1], v[:1], 4, 2, causal=True), 4, False)


@pytest.mark.parametrize("Sq", [1, 5, 130])
def test_stale_memory_has_no_say(cuda_device, Sq):
    """Bit for bit the same whatever the cache holds behind the lengths and the kernel before left in shared memory."""
    from npu_ai_b200 import kernels
    q, k, v = _qkv(2, 8, 2, Sq, 700, 64, Sq, cuda_device)
    lens = ints(cuda_device, 700, 333)
    wild = [t * 300.0 for t in _qkv(4, 16, 4, 512, 512, 64, 3, cuda_device)]
    calm = [t * 1e-3 for t in wild]
    both = dict(kv_heads=2, causal=True, q_start=lens - Sq, kv_lens=lens, softcap=5.0,
                slopes=torch.rand(8, device=cuda_device))
    for drop in ("", "slopes", "softcap"):
        kw = {n: a for n, a in both.items() if n != drop}
        ref = None
        for fill in (0.0, 1e4, -1e30, float("nan"), float("inf")):
            k[1, 333:], v[1, 333:] = fill, fill
            for before in (wild, calm):
                kernels.attention(*before, 16, kv_heads=4, softcap=1.0)
                out = kernels.attention(q, k, v, 8, **kw)
                kernels.check_status(cuda_device)
                ref = out if ref is None else ref
                assert torch.equal(out, ref), (drop, fill)


@pytest.mark.parametrize("Sq,variant", [(70, 0), (1, 0), (1, 40), (70, 2)])
def test_offsets_past_32_bits(cuda_device, Sq, variant):
    """Sequences more than 2^31 elements (and 2^32 bytes) apart: queries, cache, mask and output in one large buffer."""
    from npu_ai_b200 import kernels
    H, Hk, Skv, D, far = 4, 2, 300, 64, 2 ** 31 + 4096
    if torch.cuda.mem_get_info(cuda_device)[0] < 16 << 30:
        pytest.skip("needs 16 GB")
    big = torch.empty(far + (1 << 20), dtype=BF16, device=cuda_device)
    src = _qkv(2, H, Hk, Sq, Skv, D, 5, cuda_device)
    bias = torch.randn(2, 1, Sq, Skv, device=cuda_device).to(BF16)
    views, at = [], 0
    for t in (*src, bias, torch.zeros_like(src[0])):
        n = t[0].numel()
        v = big.as_strided(t.shape, (far, *t[0].stride()), at)
        v.copy_(t)
        views.append(v)
        at += (n + 63) // 64 * 64
    q, k, v, mask, out = views
    kernels.attention(q, k, v, H, kv_heads=Hk, causal=True, mask=mask, out=out, variant=variant)
    kernels.check_status(cuda_device)
    check(out, *oracle(*src, H, Hk, causal=True, mask=bias), H, False)


def test_refusals(cuda_device):
    from npu_ai_b200 import kernels
    dev = cuda_device
    q, k, v = _qkv(2, 8, 2, 16, 32, 64, 1, dev)

    def bad(match, *a, **kw):
        with pytest.raises(ValueError, match=match):
            kernels.attention(*(a or (q, k, v, 8)), **kw)
    bad("kv_heads", kv_heads=4)
    bad("kv_heads", q, k[..., :64 * 1].repeat(1, 1, 3), v[..., :64].repeat(1, 1, 3), 8, causal=True)
    bad("prefix_len needs", kv_lens=ints(dev, 1, 2), prefix_len=3)
    bad("kv_lens", kv_lens=ints(dev, 1, 2, 3))
    bad("kv_lens", kv_lens=torch.tensor([1, 2], device=dev))
    bad("kv_lens", kv_lens=torch.tensor([1, 2], dtype=torch.int32))
    bad("q_start", causal=True, q_start=ints(dev, 1))
    bad("as many queries", doc_offsets=ints(dev, 0, 3))
    bad("doc_offsets must", q, k[:, :16], v[:, :16], 8, doc_offsets=torch.tensor([0.0, 3.0], device=dev))
    bad("softcap", softcap=0.0)
    bad("softcap", softcap=float("nan"))
    bad("slopes", slopes=torch.zeros(2, device=dev))
    bad("distance_bias", distance_bias=torch.zeros(8, 4, device=dev))
    bad("mask", mask=torch.zeros(2, 16, 32, device=dev))
    bad("mask", mask=torch.zeros(16, 31, device=dev))
    bad("mask", mask=torch.zeros(16, 32, dtype=torch.float16, device=dev))
    bad("mask", mask=torch.zeros(32, 16, device=dev).t())
    bad("mask", mask=torch.zeros(16, 32))
    bad("output", causal=True, out=torch.zeros(2, 16, 100, device=dev))
    bad("scale", causal=True, scale=0.0)
    bad("bf16", q.float(), k, v, 8, causal=True)
    bad("do not match", q, k, v[:, :5], 8, causal=True)
    bad("16-byte", q, torch.zeros(2 * 32 * 128 + 1, dtype=BF16, device=dev)[1:].view(2, 32, 128), v, 8, causal=True)
    with pytest.raises(RuntimeError, match="variant"):
        kernels.attention(q, k, v, 8, causal=True, variant=65)

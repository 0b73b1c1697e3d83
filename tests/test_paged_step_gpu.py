"""A decoder's cached steps as a user runs them: the fused q/k/v projection, the append with the rotation, the attention over
the pages, the output projection. A ragged prompt and its continuation, token by token, eagerly and as a replayed graph, give
what a contiguous cache gives with rope and kernels.attention on the same tensors, within the attention's tolerance."""
import pytest
import torch

from test_attention_masked_gpu import BF16, check, oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads,page,interleaved", [(8, 2, 16, False), (4, 4, 7, True), (8, 1, 64, False)])
def test_prompt_and_continuation(cuda_device, heads, kv_heads, page, interleaved):
    from npu_ai_b200 import kernels
    dev, d, B, T, steps = cuda_device, 64, 3, 77, 6
    C, most = heads * d, 77 + 6
    g = torch.Generator(device=dev).manual_seed(heads)
    w_qkv, w_out = ((torch.randn(n, C, generator=g, device=dev) * C ** -0.5).to(BF16) for n in ((heads + 2 * kv_heads) * d, C))
    freqs, magnitude = kernels.rope_frequencies(d, scaling="yarn", factor=4.0, device=dev)
    turn = dict(interleaved=interleaved, magnitude=magnitude)
    width = -(-most // page)
    k_pages, v_pages = (torch.full((B * width, page, kv_heads, d), float("nan"), dtype=BF16, device=dev) for _ in range(2))
    table = torch.randperm(B * width, generator=g, device=dev).view(B, width).to(torch.int32)
    flat = [torch.zeros(B, most, kv_heads * d, dtype=BF16, device=dev) for _ in range(2)]  # the same cache in one piece

    def layer(x, starts, lens, counts=None):
        n = x.shape[1]
        y = kernels.gemm(x.view(-1, C), w_qkv, out_dtype=BF16).view(B, n, -1)
        q, k, v = y.split((heads * d, kv_heads * d, kv_heads * d), -1)
        q = kernels.paged_append(k, v, k_pages, v_pages, table, starts, counts=counts, q=q, heads=heads, freqs=freqs, **turn)
        o = kernels.paged_attention(q, k_pages, v_pages, table, lens, heads, q_start=starts, out_dtype=BF16)
        return y, q, o, kernels.gemm(o.view(-1, C), w_out, out_dtype=BF16, residual=x.reshape(-1, C)).view(B, n, C)

    def verify(y, q, o, starts, lens):
        n = y.shape[1]
        nq, nk = heads * d, kv_heads * d
        assert torch.equal(q, kernels.rope(y[..., :nq], freqs, heads, starts, **turn))
        new = kernels.rope(y[..., nq:nq + nk], freqs, kv_heads, starts, **turn), y[..., nq + nk:]
        for f, t in zip(flat, new):
            for b in range(B):
                s, e = int(starts[b]), int(lens[b])
                f[b, s:e] = t[b, :e - s]
        own = torch.arange(n, device=dev) < (lens - starts)[:, None]  # a sequence's own tokens, not its padding
        ref, tol = oracle(q, *flat, heads, kv_heads, causal=True, q_start=starts, kv_lens=lens)
        check(o, ref, tol, heads, False)
        base = kernels.attention(q, *flat, heads, kv_heads=kv_heads, causal=True, q_start=starts, kv_lens=lens, out_dtype=BF16)
        check(base, ref, tol, heads, False)
        assert bool(torch.isfinite(o[own]).all())

    lens = torch.tensor([77, 40, 1], dtype=torch.int32, device=dev)
    zero = torch.zeros_like(lens)
    x = torch.randn(B, T, C, generator=g, device=dev).to(BF16)
    y, q, o, _ = layer(x, zero, lens, counts=lens)
    kernels.check_status(dev)
    verify(y, q, o, zero, lens)
    pages = [t.clone() for t in (k_pages, v_pages)]
    tokens = torch.randn(steps, B, 1, C, generator=g, device=dev).to(BF16)

    starts = lens.clone()
    eager = []
    for tok in tokens:
        y, q, o, out = layer(tok, starts, starts + 1)
        verify(y, q, o, starts, starts + 1)
        eager.append(out)
        starts.add_(1)
    kernels.check_status(dev)

    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        tok = tokens[0].clone()
        starts.copy_(lens)
        layer(tok, starts, starts + 1)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = layer(tok, starts, starts + 1)[3]
            starts.add_(1)
        for t, p in zip((k_pages, v_pages), pages):
            t.copy_(p)
        starts.copy_(lens)
        for t, want in zip(tokens, eager):
            tok.copy_(t)
            graph.replay()
            assert torch.equal(out, want)


def test_runner_methods(cuda_device):
    """NpuGemm's methods take tensors of any device and float type; the same results as the functions they wrap."""
    from npu_ai_b200 import kernels
    from npu_ai_b200.runner import NpuGemm
    g = NpuGemm()
    dev, H, hk, D, page = g.device, 4, 2, 64, 16
    f, m = kernels.rope_frequencies(D)
    x = torch.randn(2, 3, H * D, dtype=torch.float64)
    y = g.rope(x, f, H, torch.tensor([5, 9]), magnitude=1.5)
    assert y.is_cuda and y.dtype == torch.float32
    assert torch.equal(y, kernels.rope(x.float().to(dev), f.to(dev), H, torch.tensor([5, 9], dtype=torch.int32, device=dev),
                                       magnitude=1.5))
    table = torch.arange(4).view(2, 2)
    starts = torch.tensor([0, 20])
    q, k, v = (torch.randn(2, 3, n * D) for n in (H, hk, hk))
    pools = [torch.zeros(4, page, hk, D, dtype=BF16, device=dev) for _ in range(4)]
    turned = g.paged_append(k, v.to(BF16), pools[0], pools[1], table, starts, q=q, heads=H, freqs=f)
    i32 = [t.to(dev, torch.int32) for t in (table, starts)]
    want = kernels.paged_append(k.to(dev), v.to(BF16).float().to(dev), pools[2], pools[3], *i32, q=q.to(dev), heads=H,
                                freqs=f.to(dev))
    assert torch.equal(turned, want) and torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])
    o = g.paged_attention(turned.cpu(), pools[0], pools[1], table, starts + 3, H, softcap=20.0)
    assert o.dtype == torch.float32
    assert torch.equal(o, kernels.paged_attention(want, pools[2], pools[3], i32[0], i32[1] + 3, H, softcap=20.0))
    assert torch.equal(g.paged_attention(turned, pools[0], pools[1], table, starts + 3, H, q_start=starts, out_dtype=BF16),
                       kernels.paged_attention(want, pools[2], pools[3], i32[0], i32[1] + 3, H, q_start=i32[1], out_dtype=BF16))
    kernels.check_status(dev)


def test_written_tensors_have_new_versions(cuda_device):
    """What a call writes counts as written for autograd (a tensor saved before it may not be used after it); what it only
    reads, and inference tensors, are left alone. Gradients are not tracked through the calls."""
    from npu_ai_b200 import kernels
    dev, H, hk, D = cuda_device, 4, 2, 64
    f, _ = kernels.rope_frequencies(D, device=dev)

    def operands():
        return dict(q=torch.randn(2, 3, H * D, device=dev).to(BF16), k=torch.randn(2, 3, hk * D, device=dev).to(BF16),
                    v=torch.randn(2, 3, hk * D, device=dev).to(BF16), kp=torch.zeros(4, 16, hk, D, dtype=BF16, device=dev),
                    vp=torch.zeros(4, 16, hk, D, dtype=BF16, device=dev), o=torch.empty(2, 3, H * D, dtype=BF16, device=dev),
                    table=torch.arange(4, dtype=torch.int32, device=dev).view(2, 2),
                    starts=torch.zeros(2, dtype=torch.int32, device=dev))

    def steps(t):
        yield ["o"], kernels.rope(t["q"], f, H, out=t["o"])
        yield [], kernels.rope(t["q"], f, H)
        yield ["kp", "vp"], kernels.paged_append(t["k"], t["v"], t["kp"], t["vp"], t["table"], t["starts"], q=t["q"], heads=H,
                                                 freqs=f)
        yield ["kp", "vp", "q"], kernels.paged_append(t["k"], t["v"], t["kp"], t["vp"], t["table"], t["starts"], q=t["q"],
                                                      heads=H, q_out=t["q"], freqs=f)
        yield ["o"], kernels.paged_attention(t["q"], t["kp"], t["vp"], t["table"], t["starts"] + 3, H, out=t["o"])
        yield [], kernels.paged_attention(t["q"], t["kp"], t["vp"], t["table"], t["starts"] + 3, H)
    t = operands()
    before = {n: x._version for n, x in t.items()}
    for names, y in steps(t):
        assert y._version == (0 if not names or names == ["kp", "vp"] else before[names[-1]] + 1)
        for n in names:
            before[n] += 1
        assert {n: x._version for n, x in t.items()} == before
    with torch.inference_mode():
        for _ in steps(operands()):
            pass
    w = torch.ones(2, 3, H * D, device=dev, requires_grad=True)
    x = torch.zeros(2, 3, H * D, device=dev)
    loss = (w * x).sum()  # keeps x for w's gradient
    kernels.rope(torch.ones_like(x), f, H, out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    kernels.check_status(dev)


def test_runner_numbers_past_32_bits(cuda_device):
    """64-bit tables, lengths and positions of the runner's methods: a page id past 32 bits is a page that is not there, and
    positions that do not fit are refused."""
    from npu_ai_b200 import kernels
    from npu_ai_b200.runner import NpuGemm
    g = NpuGemm()
    dev, H, hk, D, page = g.device, 4, 2, 64, 16
    f, _ = kernels.rope_frequencies(D, device=dev)
    pools = [torch.full((4, page, hk, D), 9.0, dtype=BF16, device=dev) for _ in range(4)]
    k, v = (torch.randn(2, 3, hk * D, device=dev).to(BF16) for _ in range(2))
    q = torch.randn(2, 3, H * D, device=dev).to(BF16)
    starts = torch.zeros(2, dtype=torch.int64)
    for place in ("cpu", dev):
        table = torch.tensor([[1, -2 ** 63], [2 ** 32, 2 ** 32 + 5]], device=place)
        near = torch.tensor([[1, -1], [-1, 99]], dtype=torch.int32, device=dev)
        counts = torch.tensor([2 ** 40, -2 ** 40 + 3], device=place)
        g.paged_append(k, v, pools[0], pools[1], table, starts, counts=counts, freqs=f)
        kernels.paged_append(k, v, pools[2], pools[3], near, starts.to(dev, torch.int32),
                             counts=torch.tensor([3, 0], dtype=torch.int32, device=dev), freqs=f)
        assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3]) and bool((pools[0][[0, 2, 3]] == 9).all())
        lens = torch.tensor([2 ** 33 + 1, 2 ** 32 + 7], device=place)
        o = g.paged_attention(q, pools[0], pools[1], table, lens, H, q_start=torch.tensor([2 ** 40, 0], device=place))
        want = kernels.paged_attention(q, pools[0], pools[1], near, torch.tensor([32, 32], dtype=torch.int32, device=dev), H,
                                       q_start=torch.tensor([100, 0], dtype=torch.int32, device=dev))
        assert torch.equal(o, want) and bool((o[1] == 0).all())
    far = torch.tensor([0, 2 ** 31])
    for bad in (lambda: g.rope(q, f, H, far), lambda: g.paged_append(k, v, pools[0], pools[1], table, far, freqs=f),
                lambda: g.rope(q, f, H, far.float()), lambda: g.paged_attention(q, pools[0], pools[1], table.float(), lens, H),
                lambda: g.rope(q, f, H, 2 ** 31)):
        with pytest.raises(ValueError):
            bad()
    kernels.check_status(dev)


def test_written_windows_that_overlap_are_refused(cuda_device):
    """Outputs and pools whose rows, pages or heads reach into the next ones, as strides alone can make them."""
    from npu_ai_b200 import kernels
    dev, H, hk, D = cuda_device, 4, 2, 64
    f, _ = kernels.rope_frequencies(D, device=dev)
    q, (k, v) = torch.randn(2, 3, H * D, device=dev).to(BF16), (torch.randn(2, 3, hk * D, device=dev).to(BF16) for _ in range(2))
    kp, vp = (torch.zeros(4, 16, hk, D, dtype=BF16, device=dev) for _ in range(2))
    table, zero = torch.arange(4, dtype=torch.int32, device=dev).view(2, 2), torch.zeros(2, dtype=torch.int32, device=dev)
    buf = torch.full((4, 20, 2 * H, D), 3.0, dtype=BF16, device=dev).view(-1)
    for st in ((3 * H * D, H * D - 8, 1), (2 * H * D, H * D, 1), (8, 2048, 1)):
        o = buf.as_strided((2, 3, H * D), st)
        for call in (lambda: kernels.rope(q, f, H, out=o), lambda: kernels.paged_attention(q, kp, vp, table, zero + 3, H, out=o),
                     lambda: kernels.paged_append(k, v, kp, vp, table, zero, q=q, heads=H, freqs=f, q_out=o)):
            with pytest.raises(ValueError, match="twice"):
                call()
    for st in ((16 * hk * D - 64, hk * D, D, 1), (16 * hk * D, hk * D, D - 8, 1), (16 * hk * D, 64, D, 1)):
        pages = buf.as_strided((4, 16, hk, D), st)
        for pools in ((pages, vp), (kp, pages)):
            with pytest.raises(ValueError, match="twice"):
                kernels.paged_append(k, v, *pools, table, zero)
    assert bool((buf == 3).all()) and bool((kp == 0).all())
    kernels.check_status(dev)

"""The operators of a text transformer's block in a row, as a prompt and its continuation use them: LayerNorm, the q/k/v
projection, masked attention over a key/value cache with grouped heads, the output projection with its residual, LayerNorm,
the feed-forward projection with its activation, and the closing projection with its residual.

Every operator is checked against the formula in 64 bits on the very tensors that it was given, with its own test's
tolerance; the continuation runs one token at a time, eagerly and as a replayed graph, and the two agree bit for bit."""
import pytest
import torch

from test_attention_masked_gpu import check as check_attention, oracle as attention_oracle
from test_gemm_act_gpu import _check as check_gemm_act

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _check_gemm(out, x, w, b, r):
    """The plain product with bias and residual: sums of K products (K 2^-23), one f32 and one bf16 rounding."""
    xd, wd = x.double(), w.double()
    ref = xd @ wd.t() + (0.0 if b is None else b.double()) + (0.0 if r is None else r.double())
    tol = x.shape[-1] * 2.0 ** -23 * (xd.abs() @ wd.abs().t()) + 2.0 ** -22 * ref.abs() + 1e-30
    tol = tol + 2.0 ** -8 * (ref.abs() + tol)
    assert bool(((out.double() - ref).abs() <= tol).all())


def _check_norm(out, x, g, b):
    """f32 statistics over C values and an f32 row in and out: (C + 8) 2^-23 of the normalised value and its parts,
    then one bf16 rounding."""
    xd = x.double()
    mean = xd.mean(-1, keepdim=True)
    rstd = (xd.var(-1, unbiased=False, keepdim=True) + 1e-5).rsqrt()
    ref = (xd - mean) * rstd * g.double() + b.double()
    tol = (x.shape[-1] + 8) * 2.0 ** -23 * ((xd.abs() + mean.abs()) * rstd * g.double().abs() + b.double().abs())
    tol = tol + 2.0 ** -8 * (ref.abs() + tol)
    assert bool(((out.double() - ref).abs() <= tol).all())


class Block:
    def __init__(self, dev, C, heads, kv_heads, hidden, act, rows, batch, seed):
        g = torch.Generator(device=dev).manual_seed(seed)
        d = C // heads

        def w(n, k):
            return (torch.randn(n, k, generator=g, device=dev) * k ** -0.5).to(BF16)
        self.C, self.heads, self.kv_heads, self.d, self.act = C, heads, kv_heads, d, act
        self.qkv, self.out, self.up, self.down = (w((heads + 2 * kv_heads) * d, C), w(C, C), w(hidden, C), w(C, hidden))
        self.b_qkv, self.b_up = (torch.randn(t.shape[0], generator=g, device=dev) for t in (self.qkv, self.up))
        self.norms = [(torch.randn(C, generator=g, device=dev) * 0.1 + 1.0, torch.randn(C, generator=g, device=dev) * 0.1)
                      for _ in range(2)]
        # the cache: garbage wherever nothing has been written
        self.k, self.v = (torch.full((batch, rows, kv_heads * d), float("nan"), dtype=BF16, device=dev) for _ in range(2))

    def __call__(self, x, start, lens, verify, **modifiers):
        """x [B, T, C] at the positions start[b] ..., of which the first lens[b] - start[b] are a sequence's own."""
        from npu_ai_b200 import kernels
        B, T, C = x.shape
        h1 = kernels.layer_norm(x, *self.norms[0])
        y = kernels.gemm(h1.view(B * T, C), self.qkv, self.b_qkv, out_dtype=BF16).view(B, T, -1)
        nq, nk = self.heads * self.d, self.kv_heads * self.d
        q, k, v = y[..., :nq], y[..., nq:nq + nk], y[..., nq + nk:]
        at = (start[:, None] + torch.arange(T, device=x.device)).long().clamp(max=self.k.shape[1] - 1)
        batch = torch.arange(B, device=x.device)[:, None].expand(B, T)
        self.k[batch, at] = k
        self.v[batch, at] = v
        o = kernels.attention(q, self.k, self.v, self.heads, kv_heads=self.kv_heads, causal=True, q_start=start, kv_lens=lens,
                              out_dtype=BF16, **modifiers)
        x2 = kernels.gemm(o.view(B * T, C), self.out, residual=x.reshape(B * T, C), out_dtype=BF16)
        h2 = kernels.layer_norm(x2, *self.norms[1])
        u = kernels.gemm(h2, self.up, self.b_up, out_dtype=BF16, activation=self.act)
        x3 = kernels.gemm(u, self.down, residual=x2, out_dtype=BF16)
        if verify:
            kernels.check_status(x.device)
            _check_norm(h1, x, *self.norms[0])
            _check_gemm(y.view(B * T, -1), h1.view(B * T, C), self.qkv, self.b_qkv, None)
            ref = attention_oracle(q, self.k, self.v, self.heads, self.kv_heads, causal=True, q_start=start,
                                   kv_lens=lens, **modifiers)
            check_attention(o, *ref, self.heads, False)
            _check_gemm(x2, o.view(B * T, C), self.out, None, x.reshape(B * T, C))
            _check_norm(h2, x2, *self.norms[1])
            check_gemm_act(u, h2.cpu(), self.up.cpu(), self.b_up.cpu(), None, self.act)
            _check_gemm(x3, u, self.down, None, x2)
        return x3.view(B, T, C)


@pytest.mark.parametrize("heads,kv_heads,act,modifiers", [
    (8, 8, "quick_gelu", ()), (8, 2, "silu", ("softcap",)), (8, 1, "gelu_tanh", ("slopes",)), (5, 5, "gelu", ())])
def test_prompt_and_continuation(cuda_device, heads, kv_heads, act, modifiers):
    dev = cuda_device
    d = 64
    C, B, T, rows = heads * d, 3, 77, 130
    block = Block(dev, C, heads, kv_heads, 4 * C, act, rows, B, seed=heads + kv_heads)
    mods = {}
    if "softcap" in modifiers:
        mods["softcap"] = 4.0
    if "slopes" in modifiers:
        mods["slopes"] = torch.tensor([2.0 ** -(h + 1) for h in range(heads)], device=dev)
    g = torch.Generator(device=dev).manual_seed(1)
    # A ragged prompt of 77, 40 and 1 tokens.
    lens = torch.tensor([77, 40, 1], dtype=torch.int32, device=dev)
    start = torch.zeros(B, dtype=torch.int32, device=dev)
    x = torch.randn(B, T, C, generator=g, device=dev).to(BF16)
    block(x, start, lens, True, **mods)
    for b, n in enumerate(lens.tolist()):  # padding went into the cache, too: the continuation overwrites it
        assert bool(torch.isfinite(block.k[b, :n]).all())
    cache = [t.clone() for t in (block.k, block.v)]
    tokens = torch.randn(6, B, 1, C, generator=g, device=dev).to(BF16)

    def continuation(step):
        for t, c in zip((block.k, block.v), cache):
            t.copy_(c)
        start.copy_(torch.tensor([77, 40, 1], dtype=torch.int32))
        return [step(tok) for tok in tokens]

    def eager(tok):
        y = block(tok, start, start + 1, True, **mods)
        start.add_(1)
        return y

    first = continuation(eager)
    tok = tokens[0].clone()
    side = torch.cuda.Stream(dev)  # the captured step and its replays run on another stream than the tensors' own
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        block(tok, start, start + 1, False, **mods)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = block(tok, start, start + 1, False, **mods)
            start.add_(1)

        def replayed(t):
            tok.copy_(t)
            graph.replay()
            return y.clone()
        second = continuation(replayed)
    torch.cuda.current_stream(dev).wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a, b)

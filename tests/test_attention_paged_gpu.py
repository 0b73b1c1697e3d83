"""Attention over a cache in pages on the B200 (npub200_attention_paged through kernels.paged_attention) against the formula
in 64 bits, with the oracle and the tolerance of tests/test_attention_masked_gpu.py: the operator is the same, the keys lie
elsewhere. P rounds to bf16 (2^-8 relative), scores are f32 sums, tanh and the biases add a few f32 roundings."""
import ctypes

import pytest
import torch

from test_attention_masked_gpu import BF16, check, ints, oracle

pytestmark = pytest.mark.gpu
NAN = float("nan")


class Cache:
    """Pages that hold NaN wherever no sequence has a key."""

    def __init__(self, dev, lens, hk, D, page, seed=0, width=None, pool_head_major=False, extra=3, scale=1.0):
        g = torch.Generator(device=dev).manual_seed(seed)
        B, most = len(lens), max([0] + [n for n in lens])
        self.width = -(-most // page) if width is None else width
        pages = B * self.width + extra
        shape = (pages, hk, page, D) if pool_head_major else (pages, page, hk, D)
        self.k, self.v = (torch.full(shape, NAN, dtype=BF16, device=dev) for _ in range(2))
        if pool_head_major:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        self.table = torch.randperm(pages, generator=g, device=dev)[:B * self.width].view(B, self.width).to(torch.int32)
        cap = self.width * page
        self.k_flat, self.v_flat = (torch.zeros(B, cap, hk * D, dtype=BF16, device=dev) for _ in range(2))
        for b, n in enumerate(lens):
            n = max(0, min(n, cap))
            for flat, pool in ((self.k_flat, self.k), (self.v_flat, self.v)):
                flat[b, :n] = (torch.randn(n, hk * D, generator=g, device=dev) * scale).to(BF16)
                at = torch.arange(n, device=dev)
                pool[self.table[b].long()[at // page], at % page] = flat[b, :n].unflatten(-1, (hk, D))
        self.lens = ints(dev, *lens)
        self.hk, self.D, self.page, self.B, self.cap = hk, D, page, B, cap


def run(dev, lens, H, hk, D, page, Sq=1, seed=0, q_scale=1.5, head_major=False, head_major_out=False, out_dtype=BF16, variant=0,
        causal=True, q_start=None, softcap=None, slopes=None, width=None, pool_head_major=False, scale=None, cache=None, hide=None,
        repeat=True):
    from npu_ai_b200 import kernels
    c = cache or Cache(dev, lens, hk, D, page, seed, width, pool_head_major)
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    q = (torch.randn(*((c.B, H, Sq, D) if head_major else (c.B, Sq, H * D)), generator=g, device=dev) * q_scale).to(BF16)

    def call():
        return kernels.paged_attention(q, c.k, c.v, c.table, c.lens, H, scale, causal=causal, q_start=q_start, softcap=softcap,
                                       slopes=slopes, head_major_in=head_major, head_major_out=head_major_out,
                                       out_dtype=out_dtype, variant=variant)
    out = call()
    kernels.check_status(dev)
    valid = c.lens.clamp(0, c.cap)
    pad = max(1, c.cap)  # (the oracle wants a key)
    k, v = (torch.nn.functional.pad(t, (0, 0, 0, pad - c.cap)) for t in (c.k_flat, c.v_flat))
    qq = q.transpose(1, 2).flatten(2) if head_major else q
    ref, tol = oracle(qq, k, v, H, hk, scale=scale, causal=causal, kv_lens=valid, softcap=softcap, slopes=slopes,
                      q_start=valid - Sq if q_start is None else q_start, mask=hide)
    check(out, ref, tol, H, head_major_out)
    if repeat:
        assert torch.equal(out, call())
    return out


@pytest.mark.parametrize("D", [8, 24, 40, 64, 72, 80, 96, 104, 128, 136, 160, 192, 200, 256])
@pytest.mark.parametrize("page", [1, 7, 16, 64])
def test_head_dims_and_pages(cuda_device, D, page):
    run(cuda_device, [77, 1, 300], 4, 2, D, page, seed=D)
    run(cuda_device, [50, 129], 3, 3, D, page, Sq=3, seed=D, pool_head_major=True, out_dtype=torch.float32, head_major=True)


@pytest.mark.parametrize("n", [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 255, 1000])
@pytest.mark.parametrize("variant", [0, 1, 2, 3, 1000])
def test_lengths_and_splits(cuda_device, n, variant):
    run(cuda_device, [n], 8, 2, 64, 16, variant=variant, seed=n)
    run(cuda_device, [n, 0, n // 2, 5], 4, 4, 128, 24, Sq=2, variant=variant, seed=n, head_major_out=True)


@pytest.mark.parametrize("H,hk,Sq", [(1, 1, 1), (8, 1, 1), (16, 1, 1), (17, 1, 1), (32, 1, 1), (33, 1, 1), (64, 1, 1), (65, 1, 1),
                                     (128, 2, 1), (4, 2, 8), (4, 2, 9), (8, 2, 5), (8, 2, 16), (5, 5, 33), (2, 1, 100),
                                     (6, 2, 11), (1, 1, 300)])
@pytest.mark.parametrize("variant", [0, 1, 7])
def test_rows(cuda_device, H, hk, Sq, variant):
    """One, two and four warps of rows, several tiles of them, rows whose causal border lies far before the last key."""
    run(cuda_device, [400, Sq, 333, Sq + 1], H, hk, 64, 16, Sq=Sq, variant=variant, seed=H + Sq)


@pytest.mark.parametrize("D", [64, 96, 128, 160, 192, 256])
@pytest.mark.parametrize("H,Sq", [(4, 1), (4, 12), (4, 40)])
def test_modifiers(cuda_device, D, H, Sq):
    g = torch.Generator(device=cuda_device).manual_seed(D)
    slopes = torch.rand(H, generator=g, device=cuda_device)
    lens = [200, 57, 1, 130]
    run(cuda_device, lens, H, 2, D, 16, Sq=Sq, softcap=9.0, q_scale=4.0)
    run(cuda_device, lens, H, 2, D, 16, Sq=Sq, slopes=slopes)
    run(cuda_device, lens, H, 2, D, 16, Sq=Sq, slopes=slopes, softcap=20.0, q_scale=4.0, causal=False, out_dtype=torch.float32)


def test_positions(cuda_device):
    """Queries before the first key, in the middle, behind the last; not causal at all."""
    d = cuda_device
    for start in ([0, 0, 0], [-3, 5, 59], [100, -100, 2 ** 31 - 1], [-2 ** 31, 1, 30]):
        run(d, [60, 33, 100], 4, 2, 64, 16, Sq=6, q_start=ints(d, *start))
        run(d, [60, 33, 100], 4, 2, 64, 16, Sq=6, q_start=ints(d, *start), causal=False)
    run(d, [3, 2, 1], 4, 2, 64, 16, Sq=6)  # more queries than keys: the first see none
    run(d, [3, 0, 1], 4, 2, 64, 16, Sq=6, causal=False)


def test_lengths_outside_the_table(cuda_device):
    run(cuda_device, [-5, 1000, 2 ** 31 - 1, -2 ** 31, 33], 4, 2, 64, 16, width=3)
    run(cuda_device, [5, 0], 4, 2, 64, 16, width=0)


def test_pages_that_are_not_there(cuda_device):
    d = cuda_device
    for Sq in (1, 3):
        lens = [100, 100, 60, 33]
        c = Cache(d, lens, 2, 64, 8)
        hide = torch.ones(4, 1, 1, c.cap, dtype=torch.bool, device=d)
        for b, at, value in ((0, 0, -1), (0, 5, 10 ** 6), (1, 3, c.k.shape[0]), (1, 4, -2 ** 31), (1, 12, 2 ** 31 - 1), (3, 4, -7)):
            c.table[b, at] = value
            hide[b, ..., at * 8:at * 8 + 8] = False
        c.table[2] = -1  # nothing of this one is there
        hide[2] = False
        out = run(d, lens, 4, 2, 64, 8, Sq=Sq, cache=c, hide=hide)
        assert bool((out[2] == 0).all())
        run(d, lens, 4, 2, 64, 8, Sq=Sq, cache=c, hide=hide, variant=1)
    empty = torch.empty(0, 8, 2, 64, dtype=BF16, device=d)
    from npu_ai_b200 import kernels
    o = kernels.paged_attention(torch.ones(2, 1, 256, dtype=BF16, device=d), empty, empty,
                                torch.zeros(2, 4, dtype=torch.int32, device=d), ints(d, 20, 3), 4)
    assert bool((o == 0).all())


def test_nan_and_infinite_scores(cuda_device):
    """A row that sees a NaN score, or an infinite one, is NaN; the others are not touched, whatever part holds the key."""
    from npu_ai_b200 import kernels
    d = cuda_device
    for bad in (NAN, float("inf")):
        for variant in (0, 1, 1000):
            lens = [200, 200, 200]
            c = Cache(d, lens, 2, 64, 16)
            for t in (c.k_flat, c.k):
                pass
            c.k_flat[1, 150, :64] = bad  # key/value head 0 of sequence 1
            c.k[c.table[1, 150 // 16].long(), 150 % 16, 0] = bad
            q = torch.ones(3, 2, 256, dtype=BF16, device=d)
            o = kernels.paged_attention(q, c.k, c.v, c.table, c.lens, 4, variant=variant).view(3, 2, 4, 64)
            kernels.check_status(d)
            assert bool(torch.isnan(o[1, :, :2]).all())
            assert bool(torch.isfinite(o[1, :, 2:]).all()) and bool(torch.isfinite(o[[0, 2]]).all())
    c = Cache(d, [40], 1, 64, 16)
    c.k[...] = NAN
    assert bool(torch.isnan(kernels.paged_attention(torch.ones(1, 1, 64, dtype=BF16, device=d), c.k, c.v, c.table, c.lens,
                                                    1, variant=1)).all())


def test_minus_infinite_scores_weigh_nothing(cuda_device):
    from npu_ai_b200 import kernels
    d = cuda_device
    c = Cache(d, [100], 1, 64, 16)
    at = torch.tensor([3, 17, 18, 50, 99], device=d)
    c.k[c.table[0].long()[at // 16], at % 16] = float("-inf")
    q = torch.ones(1, 1, 64, dtype=BF16, device=d)
    o = kernels.paged_attention(q, c.k, c.v, c.table, c.lens, 1, variant=1)
    seen = torch.ones(1, 1, 1, c.cap, dtype=torch.bool, device=d)
    seen[..., at] = False
    ref, tol = oracle(q, c.k_flat, c.v_flat, 1, 1, kv_lens=c.lens, mask=seen)
    check(o, ref, tol, 1, False)


def test_large_scores(cuda_device):
    """Scores far apart, and rising along the keys so that the maximum moves again and again."""
    from npu_ai_b200 import kernels
    d = cuda_device
    for variant in (0, 1, 1000):
        run(d, [500, 90], 4, 2, 64, 16, q_scale=60.0, variant=variant)
        c = Cache(d, [500], 1, 64, 16)
        ramp = torch.linspace(-30, 30, 500, device=d)[:, None].expand(500, 64).to(BF16)
        at = torch.arange(500, device=d)
        c.k[c.table[0].long()[at // 16], at % 16] = ramp[:, None]
        c.k_flat[0, :500] = ramp
        q = torch.ones(1, 1, 64, dtype=BF16, device=d)
        o = kernels.paged_attention(q, c.k, c.v, c.table, c.lens, 1, variant=variant)
        check(o, *oracle(q, c.k_flat, c.v_flat, 1, 1, kv_lens=c.lens), 1, False)


def test_strides(cuda_device):
    """Queries inside a fused projection, both pools inside one, a table inside a wider one, an output inside a larger one
    at an odd offset whose other elements stay."""
    from npu_ai_b200 import kernels
    d = cuda_device
    lens, H, hk, D, page = [90, 41], 4, 2, 64, 16
    c = Cache(d, lens, hk, D, page)
    q = torch.randn(2, 3, H * D, device=d).to(BF16)
    want = kernels.paged_attention(q, c.k, c.v, c.table, c.lens, H, out_dtype=BF16)
    qkv = torch.randn(2, 3, (H + 2 * hk) * D, device=d).to(BF16)
    qkv[..., :H * D] = q
    both = torch.full((c.k.shape[0], 2, page, hk, D), NAN, dtype=BF16, device=d)
    both[:, 0], both[:, 1] = c.k, c.v
    wide = torch.full((2, c.width + 5), -1, dtype=torch.int32, device=d)
    wide[:, 2:2 + c.width] = c.table
    for off in (0, 1, 2, 8):
        for dtype in (BF16, torch.float32):
            buf = torch.full((2, 3, H * D + 9), 3.0, dtype=dtype, device=d)
            o = kernels.paged_attention(qkv[..., :H * D], both[:, 0], both[:, 1], wide[:, 2:2 + c.width], c.lens, H,
                                        out=buf[..., off:off + H * D])
            assert o.data_ptr() == buf[..., off:].data_ptr()
            assert torch.equal(o.to(BF16), want)
            assert bool((buf[..., :off] == 3).all()) and bool((buf[..., off + H * D:] == 3).all())
    one = q[:1, :1].expand(2, 3, H * D)
    o = kernels.paged_attention(one, c.k, c.v, c.table, c.lens, H, out_dtype=BF16)
    assert torch.equal(o, kernels.paged_attention(one.contiguous(), c.k, c.v, c.table, c.lens, H, out_dtype=BF16))


@pytest.mark.parametrize("D", [64, 80, 128, 256])
def test_both_kinds_of_loads(cuda_device, D):
    """Pools whose heads are one head expanded (no tensor map takes a stride of 0) give what a copy of them gives, and a wide
    table (which decides between the kinds of loads below 128 columns) what a narrow one gives."""
    from npu_ai_b200 import kernels
    d = cuda_device
    for Sq in (1, 4, 12):
        c = Cache(d, [333, 40, 0], 1, D, 32)
        q = torch.randn(3, Sq, 4 * D, device=d).to(BF16)
        one = [t.expand(-1, -1, 2, -1) for t in (c.k, c.v)]
        want = kernels.paged_attention(q, *(t.contiguous() for t in one), c.table, c.lens, 4)
        assert torch.equal(kernels.paged_attention(q, *one, c.table, c.lens, 4), want)
        wide = torch.full((3, 5000), -1, dtype=torch.int32, device=d)
        wide[:, :c.width] = c.table
        assert torch.equal(kernels.paged_attention(q, *(t.contiguous() for t in one), wide, c.lens, 4), want)
    kernels.check_status(d)


def test_shared_pages(cuda_device):
    """Two sequences with the same first pages, and one page many times in one table."""
    d = cuda_device
    c = Cache(d, [64, 64], 2, 64, 16)
    c.table[1, :2] = c.table[0, :2]
    c.table[1, 3] = c.table[1, 2]
    for flat in (c.k_flat, c.v_flat):
        flat[1, :32] = flat[0, :32]
        flat[1, 48:64] = flat[1, 32:48]
    run(d, None, 4, 2, 64, 16, Sq=2, cache=c)


@pytest.mark.parametrize("B", [1, 31, 33, 100, 1500])
def test_batches(cuda_device, B):
    lens = [(37 * i) % 90 for i in range(B)]
    run(cuda_device, lens, 4, 2, 64, 16, seed=B)


def test_long_caches(cuda_device):
    run(cuda_device, [70001], 8, 2, 128, 64, out_dtype=torch.float32)
    run(cuda_device, [40000, 3, 9000], 32, 1, 64, 16, out_dtype=torch.float32, Sq=2)
    run(cuda_device, [30000], 2, 2, 256, 32, out_dtype=torch.float32)


def test_offsets_past_32_bits(cuda_device):
    """Pages behind 2^31 elements of a pool."""
    from npu_ai_b200 import kernels
    d = cuda_device
    page, hk, D = 16, 8, 128
    pages = 2 ** 31 // (page * hk * D) + 9
    c = Cache(d, [100], hk, D, page)
    big = [torch.empty(pages, page, hk, D, dtype=BF16, device=d) for _ in range(2)]
    assert big[0].numel() > 2 ** 31
    far = torch.arange(pages - c.width, pages, device=d)
    for t, small in zip(big, (c.k, c.v)):
        t[far] = small[c.table[0].long()]
    q = torch.randn(1, 1, 8 * D, device=d).to(BF16)
    o = kernels.paged_attention(q, *big, far.to(torch.int32)[None], c.lens, 8)
    assert torch.equal(o, kernels.paged_attention(q, c.k, c.v, c.table, c.lens, 8))


def test_graphs_follow_the_lengths(cuda_device):
    """Two captured graphs on two streams at once, replayed while the lengths grow; equal to eager calls bit for bit."""
    from npu_ai_b200 import kernels
    d = cuda_device
    caches = [Cache(d, [300, 77, 500], 2, 64, 16, seed=i) for i in range(2)]
    qs = [torch.randn(3, 1, 512, device=d).to(BF16) for _ in range(2)]
    lens = [ints(d, 100, 1, 300) for _ in range(2)]
    streams, graphs, outs = [torch.cuda.Stream(d) for _ in range(2)], [], []
    torch.cuda.synchronize()
    for c, q, n, s in zip(caches, qs, lens, streams):
        with torch.cuda.stream(s):
            kernels.paged_attention(q, c.k, c.v, c.table, n, 8)
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                outs.append(kernels.paged_attention(q, c.k, c.v, c.table, n, 8))
            graphs.append(g)
    for step in range(4):
        for g, s, n in zip(graphs, streams, lens):
            with torch.cuda.stream(s):
                n.add_(ints(d, 50, 19, 50))
                for _ in range(3):
                    g.replay()
        torch.cuda.synchronize()
        for c, q, n, o in zip(caches, qs, lens, outs):
            assert torch.equal(o, kernels.paged_attention(q, c.k, c.v, c.table, n, 8))
    kernels.check_status(d)


@pytest.mark.parametrize("page", [16, 7])
@pytest.mark.parametrize("H,Sq", [(4, 1), (4, 8), (4, 16), (4, 40)])
def test_forced_timeout_reports_and_recovers(cuda_device, H, Sq, page):
    from npu_ai_b200 import kernels
    c = Cache(cuda_device, [500, 40], 2, 64, page)
    q = torch.zeros(2, Sq, H * 64, dtype=BF16, device=cuda_device)
    kernels.status(cuda_device)
    kernels.set_wait_timeout_ns(2_000_000)
    kernels.set_debug_flags(1)
    try:
        kernels.paged_attention(q, c.k, c.v, c.table, c.lens, H)
        with pytest.raises(RuntimeError, match="failure status"):
            kernels.check_status(cuda_device)
    finally:
        kernels.set_debug_flags(0)
        kernels.set_wait_timeout_ns(0)
    run(cuda_device, None, H, 2, 64, page, Sq=Sq, cache=c)


def test_c_entry_and_its_workspace(cuda_device):
    """Straight through the C ABI, with a workspace of garbage; one that is too small, missing or misaligned is refused."""
    from npu_ai_b200 import _lib, kernels
    d = cuda_device
    H, hk, D, Sq = 8, 2, 64, 2
    c = Cache(d, [300, 40], hk, D, 16)
    q = torch.randn(2, Sq, H * D, device=d).to(BF16)
    want = kernels.paged_attention(q, c.k, c.v, c.table, c.lens, H)
    p = ctypes.c_void_p
    n = ctypes.c_size_t(0)
    _lib.call("npub200_attention_paged_workspace_size", H, hk, Sq, D, ctypes.byref(n))
    cache = _lib.PagedCache(k=c.k.data_ptr(), v=c.v.data_ptr(), pages=c.k.shape[0], page_size=16, kv_heads=hk, head_dim=D,
                            table=c.table.data_ptr(), table_stride=c.table.stride(0), table_width=c.width,
                            **{f"{x}_{s}": c.k.stride(i) for x in "kv" for i, s in enumerate(("sp", "ss", "sh"))})
    st = (q.stride(0), q.stride(1), D)

    def call(ws, size):
        out = torch.full(q.shape, 5.0, device=d)
        _lib.call("npub200_attention_paged", p(q.data_ptr()), *st, ctypes.byref(cache), p(c.lens.data_ptr()),
                  p(out.data_ptr()), *st, _lib.DTYPE_F32, 2, H, Sq, ctypes.c_float(D ** -0.5), 1, None, ctypes.c_float(0.0),
                  None, p(ws), size, 0, p(torch.cuda.current_stream(d).cuda_stream))
        return out
    ws = torch.full((n.value + 16,), 255, dtype=torch.uint8, device=d)
    assert torch.equal(call(ws.data_ptr(), n.value), want)
    for bad in ((None, n.value), (ws.data_ptr(), n.value - 1), (ws.data_ptr() + 8, n.value)):
        with pytest.raises(ValueError, match="workspace"):
            call(*bad)


def test_empty_calls_and_refusals(cuda_device):
    from npu_ai_b200 import kernels
    d = cuda_device
    c = Cache(d, [20, 9], 2, 64, 8)
    q = torch.randn(2, 1, 256, device=d).to(BF16)
    assert kernels.paged_attention(q[:0], c.k, c.v, c.table[:0], c.lens[:0], 4).shape == (0, 1, 256)
    assert kernels.paged_attention(q[:, :0], c.k, c.v, c.table, c.lens, 4).shape == (2, 0, 256)

    def call(q=q, k=c.k, v=c.v, table=c.table, lens=c.lens, heads=4, **kw):
        return kernels.paged_attention(q, k, v, table, lens, heads, **kw)
    for bad in (dict(q=q.float()), dict(q=q[0]), dict(q=q, head_major_in=True), dict(heads=3), dict(heads=0), dict(k=c.k.float()),
                dict(v=c.v[:2]), dict(table=c.table.long()), dict(table=c.table[:1]), dict(lens=c.lens.long()),
                dict(lens=c.lens[:1]), dict(lens=c.lens.cpu()), dict(q_start=c.lens.float()), dict(slopes=torch.ones(3, device=d)),
                dict(scale=0.0), dict(scale=-1.0), dict(softcap=0.0), dict(softcap=-2.0), dict(out_dtype=torch.float16),
                dict(out=q.float()[:1]), dict(out=torch.zeros(2, 1, 1, device=d).expand(2, 1, 256)), dict(q=q.cpu()),
                dict(q=torch.zeros(2, 1, 257, dtype=BF16, device=d)[..., 1:]), dict(k=c.k[..., :56], v=c.v[..., :56]),
                dict(k=c.k.mT, v=c.v.mT)):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(RuntimeError, match="variant"):
        call(variant=-1)


def test_outputs_that_overlap_are_refused(cuda_device):
    """An output that holds some of the queries elsewhere, or lies in a pool, is refused; one that is the queries is taken."""
    from npu_ai_b200 import kernels
    d = cuda_device
    H, hk, D, page, Sq = 4, 2, 64, 16, 3
    c = Cache(d, [700, 40], hk, D, page)
    buf = torch.randn(2, Sq, 3 * H * D, device=d).to(BF16)
    q, keep = buf[..., :H * D], buf.clone()
    call = lambda q=q, **kw: kernels.paged_attention(q, c.k, c.v, c.table, c.lens, H, **kw)
    pool = torch.empty(50, page, 2 * hk + 1, D, dtype=BF16, device=d)
    dense = torch.randn(2, H, Sq, D, device=d).to(BF16)
    for bad in (dict(out=buf[..., D:D + H * D]), dict(out=buf[..., H * D - 2:2 * H * D - 2]),
                dict(out=buf.view(torch.float32)[..., :H * D]),
                dict(q=dense, head_major_in=True, out=dense.view(2, Sq, H * D)),
                dict(out=c.k.flatten()[:2 * Sq * H * D].view(2, Sq, H * D)),
                dict(out=c.v.view(torch.float32).flatten()[-2 * Sq * H * D:].view(2, Sq, H * D))):
        with pytest.raises(ValueError, match="overlap"):
            call(**bad)
    with pytest.raises(ValueError, match="overlap"):
        kernels.paged_attention(q, pool[:, :, :hk], pool[:, :, hk:2 * hk], c.table, c.lens, H, out=pool[:2, :Sq].flatten(2)[..., 64:])
    assert torch.equal(buf, keep)
    want = call(out_dtype=BF16)
    assert torch.equal(call(out=buf[..., H * D:2 * H * D]), want)


@pytest.mark.parametrize("H,hk,Sq", [(4, 4, 1), (8, 2, 3), (8, 2, 5), (4, 2, 40)])
def test_outputs_in_place_of_the_queries(cuda_device, H, hk, Sq):
    """`out` may be q itself: bit for bit what a fresh output holds, over splits of one block and of many."""
    from npu_ai_b200 import kernels
    d = cuda_device
    for lens, page, variant in (([9000, 77, 0], 16, 0), ([300, 20, 1], 7, 0), ([9000, 500, 40], 16, 1), ([300, 20, 0], 16, 1000)):
        c = Cache(d, lens, hk, 64, page)
        q = torch.randn(3, Sq, H * 64, device=d).to(BF16)
        for _ in range(3):
            x = q.clone()
            want = kernels.paged_attention(q, c.k, c.v, c.table, c.lens, H, out_dtype=BF16, variant=variant)
            assert torch.equal(kernels.paged_attention(x, c.k, c.v, c.table, c.lens, H, out=x, variant=variant), want)
            assert torch.equal(x, want)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("variant", [0, 1])
def test_slopes_of_far_queries(cuda_device, causal, variant):
    """Queries far from every key: the distances differ by less than a step of f32 there, and the softmax depends on their
    differences. The part of a bias that all keys share drops out, so the tolerance is the one of a query next to them."""
    from npu_ai_b200 import kernels
    d = cuda_device
    lens, H, hk, Sq = [200, 33, 1, 500], 4, 2, 3
    slopes = torch.tensor([0.5, 0.011, 2.0 ** -8, 0.3], device=d)
    g = torch.Generator(device=d).manual_seed(5)
    c = Cache(d, lens, hk, 64, 16)
    q = torch.randn(4, Sq, H * 64, generator=g, device=d).to(BF16)
    for start in (2 ** 31 - 1, 2 ** 30 + 7, 2 ** 25 + 1) + (() if causal else (-2 ** 31, -2 ** 25 - 3)):
        starts = ints(d, *(start,) * 4)
        out = kernels.paged_attention(q, c.k, c.v, c.table, c.lens, H, causal=causal, q_start=starts, slopes=slopes,
                                      variant=variant)
        kernels.check_status(d)
        near = c.lens - 1 if start > 0 else torch.zeros_like(c.lens)
        for i in range(Sq):
            row = (q[:, i:i + 1], c.k_flat, c.v_flat, H, hk)
            ref, _ = oracle(*row, causal=causal, kv_lens=c.lens, slopes=slopes, q_start=starts.long() + i)
            tol = oracle(*row, kv_lens=c.lens, slopes=slopes, q_start=near)[1]
            check(out[:, i:i + 1], ref, tol, H, False)


def test_numbers_that_a_narrower_type_does_not_hold(cuda_device):
    """A variant past 32 bits and a cap that is zero in f32 must not pass for the default."""
    from npu_ai_b200 import _lib, kernels
    d = cuda_device
    c = Cache(d, [20], 2, 64, 8)
    q = torch.randn(1, 1, 256, device=d).to(BF16)
    for variant in (2 ** 32, -2 ** 32, 2 ** 63 - 1, -2 ** 63, 2 ** 32 + 1):
        with pytest.raises(RuntimeError, match="variant"):
            kernels.paged_attention(q, c.k, c.v, c.table, c.lens, 4, variant=variant)
    for kw in (dict(softcap=1e-60), dict(softcap=-1e-60), dict(scale=1e-60), dict(scale=1e60), dict(softcap=1e60)):
        with pytest.raises(ValueError, match="softcap|scale"):
            _lib.torch_ops().attention_paged(q, c.k, c.v, c.table, c.lens, None, None, 4, **kw)


@pytest.mark.parametrize("variant", [0, 1, 1000])
def test_rows_with_nothing_but_minus_infinity_are_zeros(cuda_device, variant):
    """As rows that see no key; the sequence's other heads and the batch's other rows are what they are without it."""
    from npu_ai_b200 import kernels
    d = cuda_device
    lens = [200, 200, 33]
    c = Cache(d, lens, 2, 64, 16)
    q = torch.randn(3, 2, 256, device=d).abs().to(BF16)
    want = kernels.paged_attention(q, c.k, c.v, c.table, c.lens, 4, variant=variant).view(3, 2, 4, 64)
    at = torch.arange(200, device=d)
    c.k[c.table[1].long()[at // 16], at % 16, 0] = float("-inf")  # key/value head 0 of sequence 1
    o = kernels.paged_attention(q, c.k, c.v, c.table, c.lens, 4, variant=variant).view(3, 2, 4, 64)
    kernels.check_status(d)
    want[1, :, :2] = 0.0
    assert torch.equal(o, want)

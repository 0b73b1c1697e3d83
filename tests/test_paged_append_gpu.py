"""The paged append on the B200 (npub200_paged_append through kernels.paged_append): what it writes against the rotation's
formula in 64 bits (tests/test_rope_gpu.py, whose tolerance it shares), and that it writes nothing else."""
import pytest
import torch

from test_rope_gpu import BF16, F32, HALF, frequencies, heads_of, make, turned

pytestmark = pytest.mark.gpu


def pool(dev, pages, page, hk, D, head_major=False, fill=None):
    shape = (pages, hk, page, D) if head_major else (pages, page, hk, D)
    p = [torch.full(shape, float("nan"), dtype=BF16, device=dev) if fill is None else
         torch.full(shape, fill, dtype=BF16, device=dev) for _ in range(2)]
    return [t.transpose(1, 2) for t in p] if head_major else p


def run(dev, B, S, H, hk, D, page, width, starts, counts=None, r=None, src=BF16, interleaved=False, head_major=False,
        pool_head_major=False, seed=0, table=None, pages=None, magnitude=1.0):
    from npu_ai_b200 import kernels
    pages = B * width + 2 if pages is None else pages
    kp, vp = pool(dev, pages, page, hk, D, pool_head_major, 7.0)
    g = torch.Generator().manual_seed(seed)
    if table is None:
        table = torch.randperm(B * width + 2, generator=g)[:B * width].view(B, width)
    table = table.to(torch.int32)
    q, k, v = (make(dev, B, S, n, D, src, head_major, seed + i) for i, n in enumerate((max(H, 1), hk, hk)))
    f = frequencies(D if r is None else r, dev)
    st = torch.tensor(starts, dtype=torch.int32)
    n = torch.tensor(counts, dtype=torch.int32) if counts is not None else None
    out = kernels.paged_append(k, v, kp, vp, table.to(dev), st.to(dev), counts=None if n is None else n.to(dev),
                               q=q if H else None, heads=H or None, freqs=f if r != 0 or H else None, interleaved=interleaved,
                               head_major=head_major, magnitude=magnitude)
    at = st.long()[:, None] + torch.arange(S)
    m = magnitude if r != 0 else 1.0
    if H:
        ref, tol = turned(heads_of(q, H, head_major), at.to(dev), f, m, interleaved)
        assert out.dtype == BF16 and out.shape == q.shape
        err = (heads_of(out, H, head_major).double() - ref).abs()
        assert bool((err <= tol + HALF[BF16] * (ref.abs() + tol) + 1e-37).all())
    else:
        assert out is None
    kr, kt = (t.cpu() for t in turned(heads_of(k, hk, head_major), at.to(dev), f, m, interleaved))
    vr = heads_of(v, hk, head_major).double().cpu()
    want = [torch.full((pages, page, hk, D), 7.0, dtype=torch.float64) for _ in range(2)]
    tols = [torch.zeros_like(w) for w in want]
    for b in range(B):
        for s in range(S if n is None else max(0, min(S, int(n[b])))):
            p = int(at[b, s])
            if not 0 <= p < width * page:
                continue
            at_page = int(table[b, p // page])
            if not 0 <= at_page < pages:
                continue
            for w, t, ref, tol in ((want[0], tols[0], kr, kt), (want[1], tols[1], vr, torch.zeros_like(vr))):
                w[at_page, p % page] = ref[b, :, s]
                t[at_page, p % page] = tol[b, :, s] + HALF[BF16] * (ref[b, :, s].abs() + tol[b, :, s])
    for got, w, t in ((kp, want[0], tols[0]), (vp, want[1], tols[1])):
        err = (got.double().cpu() - w).abs()
        assert bool((err <= t).all()), f"{int((err > t).sum())} values of the pages are off"


@pytest.mark.parametrize("page", [1, 7, 16, 48])
@pytest.mark.parametrize("D,r", [(64, None), (80, 20), (160, 64), (66, 66), (64, 0), (2, None)])
@pytest.mark.parametrize("src", [BF16, F32])
def test_pages_widths_and_types(cuda_device, page, D, r, src):
    width = -(-50 // page)
    run(cuda_device, 3, 17, 4, 2, D, page, width, [0, 13, 33], r=r, src=src, seed=page)
    run(cuda_device, 2, 1, 0, 3, D, page, width, [0, 49], r=r, src=src, interleaved=True, head_major=True,
        pool_head_major=True, seed=page, magnitude=1.25)


@pytest.mark.parametrize("H", [0, 6])
def test_counts_and_ends(cuda_device, H):
    """Ragged counts (none, one, all, more than there are, a negative number), tokens before and behind the table."""
    run(cuda_device, 6, 9, H, 2, 64, 8, 4, [0, 5, 5, 3, 1, 2], [0, 1, 9, 100, -3, 4])
    run(cuda_device, 5, 9, H, 2, 64, 8, 2, [-4, 12, 16, -2 ** 31, 2 ** 31 - 5])


def test_pages_that_are_not_there(cuda_device):
    table = torch.tensor([[0, -1, 2], [3, 99, 4], [2 ** 31 - 1, -2 ** 31, 5]])
    run(cuda_device, 3, 24, 2, 2, 64, 8, 3, [0, 0, 0], table=table, pages=6)
    run(cuda_device, 3, 24, 0, 2, 64, 8, 3, [0, 0, 0], table=torch.zeros(3, 3), pages=0)
    run(cuda_device, 3, 4, 2, 2, 64, 8, 0, [0, 0, 0], table=torch.zeros(3, 0), pages=2)


def test_slices_of_a_projection_and_of_a_pool(cuda_device):
    """q, k and v inside one projection, q rotated in place; pages inside one pool of both, a table inside a wider one."""
    from npu_ai_b200 import kernels
    dev = cuda_device
    B, S, H, hk, D, page = 2, 5, 4, 2, 64, 16
    qkv = make(dev, B, S, H + 2 * hk, D, BF16, False, 3)
    keep = qkv.clone()
    q, k, v = qkv.split((H * D, hk * D, hk * D), -1)
    both = torch.zeros(9, 2, page, hk, D, dtype=BF16, device=dev)
    tables = torch.arange(8, dtype=torch.int32, device=dev).view(2, 4)
    starts = torch.tensor([3, 14], dtype=torch.int32, device=dev)
    f = frequencies(D, dev)
    out = kernels.paged_append(k, v, both[:, 0], both[:, 1], tables[:, 1:3], starts, q=q, heads=H, q_out=q, freqs=f)
    assert out.data_ptr() == qkv.data_ptr()
    kp, vp = (torch.zeros(9, page, hk, D, dtype=BF16, device=dev) for _ in range(2))
    other = kernels.paged_append(*(t.contiguous() for t in keep.split((H * D, hk * D, hk * D), -1)[1:]), kp, vp,
                                 tables[:, 1:3].contiguous(), starts, q=keep[..., :H * D].contiguous(), heads=H, freqs=f)
    assert torch.equal(q, other) and torch.equal(both[:, 0], kp) and torch.equal(both[:, 1], vp)
    assert torch.equal(qkv[..., H * D:], keep[..., H * D:])
    # off a 16-byte boundary
    odd = torch.empty(B, S, hk * D + 1, dtype=BF16, device=dev)[..., 1:].copy_(k)
    kp2, vp2 = torch.zeros_like(kp), torch.zeros_like(vp)
    kernels.paged_append(odd, v, kp2, vp2, tables[:, 1:3], starts, freqs=f)
    assert torch.equal(kp2, kp) and torch.equal(vp2, vp)


def test_equals_the_rotation(cuda_device):
    """The keys that it stores are those of rope at the same positions, bit for bit."""
    from npu_ai_b200 import kernels
    dev = cuda_device
    B, S, hk, D, page = 3, 700, 4, 128, 32
    k, v = (make(dev, B, S, hk, D, BF16, False, i) for i in range(2))
    f, m = kernels.rope_frequencies(D, scaling="yarn", factor=8.0, device=dev)
    table = torch.randperm(3 * 40)[:90].view(3, 30).to(torch.int32).to(dev)
    starts = torch.tensor([0, 100, 260], dtype=torch.int32, device=dev)
    kp, vp = pool(dev, 120, page, hk, D)
    kernels.paged_append(k, v, kp, vp, table, starts, freqs=f, magnitude=m)
    want = kernels.rope(k, f, hk, starts, magnitude=m)
    for b in range(B):
        at = torch.arange(S, device=dev) + starts[b]
        assert torch.equal(kp[table[b].long()].flatten(0, 1)[at].flatten(1), want[b])
        assert torch.equal(vp[table[b].long()].flatten(0, 1)[at].flatten(1), v[b])


def test_offsets_past_32_bits(cuda_device):
    """Pages behind 2^31 elements of a pool."""
    from npu_ai_b200 import kernels
    dev = cuda_device
    page, hk, D = 16, 8, 128
    pages = 2 ** 31 // (page * hk * D) + 5
    kp, vp = (torch.empty(pages, page, hk, D, dtype=BF16, device=dev) for _ in range(2))
    assert kp.numel() > 2 ** 31
    table = torch.tensor([[pages - 1, 0], [1, pages - 2]], dtype=torch.int32, device=dev)
    for t in (kp, vp):
        t[table.long().flatten()] = 0.0
    k, v = (make(dev, 2, 20, hk, D, BF16, False, i) for i in range(2))
    kernels.paged_append(k, v, kp, vp, table, torch.zeros(2, dtype=torch.int32, device=dev))
    for b in range(2):
        for t, x in ((kp, k), (vp, v)):
            assert torch.equal(t[table[b].long()].flatten(0, 1)[:20].flatten(1), x[b])


def test_empty_calls_and_refusals(cuda_device):
    from npu_ai_b200 import kernels
    dev = cuda_device
    B, S, H, hk, D = 2, 3, 4, 2, 64
    kp, vp = pool(dev, 4, 8, hk, D, fill=0.0)
    q, k, v = (make(dev, B, S, n, D, BF16, False) for n in (H, hk, hk))
    table = torch.zeros(B, 2, dtype=torch.int32, device=dev)
    ints = torch.zeros(B, dtype=torch.int32, device=dev)
    f = frequencies(D, dev)
    assert kernels.paged_append(k[:0], v[:0], kp, vp, table[:0], ints[:0]) is None
    assert kernels.paged_append(k[:, :0], v[:, :0], kp, vp, table, ints, q=q[:, :0], heads=H, freqs=f).shape == (B, 0, H * D)
    assert bool((kp == 0).all())

    def call(k=k, v=v, kp=kp, vp=vp, table=table, starts=ints, **kw):
        return kernels.paged_append(k, v, kp, vp, table, starts, **kw)
    for bad in (dict(k=k.half()), dict(v=v.float()), dict(v=v[:, :2]), dict(kp=kp.float()), dict(vp=vp[:2]), dict(kp=kp[0]),
                dict(table=table.long()), dict(table=table[:1]), dict(table=table[0]), dict(starts=ints.long()),
                dict(starts=ints[:1]), dict(counts=ints.float()), dict(q=q, heads=H), dict(q=q, freqs=f),
                dict(q=q, heads=3, freqs=f), dict(q=q.float(), heads=H, freqs=f), dict(q=q[:1], heads=H, freqs=f),
                dict(q_out=q, freqs=f), dict(q=q, heads=H, freqs=f, q_out=q.float()), dict(freqs=f.float()),
                dict(freqs=torch.cat((f, f))), dict(k=torch.cat((k, k), -1)), dict(kp=kp[:1].expand(4, 8, hk, D)),
                dict(k=k.cpu()), dict(vp=vp.cpu()), dict(kp=kp.mT), dict(freqs=f, magnitude=float("inf")), dict(vp=kp)):
        with pytest.raises(ValueError):
            call(**bad)
    assert bool((kp == 0).all()) and bool((vp == 0).all())
    mha = make(dev, B, S, H, D, BF16, False)
    kp4, vp4 = pool(dev, 4, 8, H, D, fill=0.0)
    with pytest.raises(ValueError, match="overlap"):
        kernels.paged_append(mha, mha.clone(), kp4, vp4, table, ints, q=mha.clone(), heads=H, freqs=f, q_out=mha)


def test_operands_that_overlap_are_refused(cuda_device):
    """Sources inside the pools, queries written into them, pools moved inside one buffer: refused, whatever the strides;
    neighbours in one buffer are taken."""
    from npu_ai_b200 import kernels
    dev = cuda_device
    B, S, H, hk, D, page = 2, 8, 4, 2, 64, 8
    kp, vp = pool(dev, 6, page, hk, D, fill=1.0)
    k, v = (make(dev, B, S, hk, D, BF16, False, i) for i in range(2))
    q = make(dev, B, S, H, D, BF16, False, 2)
    table = torch.tensor([[0], [1]], dtype=torch.int32, device=dev)
    zero = torch.zeros(B, dtype=torch.int32, device=dev)
    f = frequencies(D, dev)

    def call(k=k, v=v, kp=kp, vp=vp, **kw):
        return kernels.paged_append(k, v, kp, vp, table, zero, **kw)
    tokens, wide = (t[2:4].flatten(2) for t in (kp, vp))  # whole pages of a pool as new tokens
    inside = kp.flatten(0, 1).flatten(1).view(6, page, hk * D)
    long = torch.zeros(6 * page * hk * D + 64, dtype=BF16, device=dev)
    moved = [long[i:i + kp.numel()].view_as(kp) for i in (0, 64)]
    rows = torch.zeros(6, page, 2 * hk, D, dtype=BF16, device=dev)  # views that are not dense
    both = torch.zeros(B, S, (H + 2 * hk) * D, dtype=BF16, device=dev)
    turned = dict(q=q, heads=H, freqs=f)
    for bad in (dict(k=tokens), dict(v=tokens), dict(k=wide), dict(v=wide), dict(k=inside[:2], v=inside[3:5]),
                dict(kp=moved[0], vp=moved[1]), dict(kp=rows[:, :, :hk], vp=rows[:, :, 1:1 + hk]),
                dict(kp=rows[:, :, :hk], k=rows[2:4].flatten(2)[..., 64:192]),
                dict(turned, q=torch.cat((kp, vp), 2)[:2].flatten(2), q_out=kp.view(3, page, 2 * hk, D)[:2].flatten(2)),
                dict(turned, q=rows[:2].flatten(2), kp=rows[:, :, :hk]),
                dict(turned, k=both[..., 64:64 + hk * D], q_out=both[..., :H * D]),
                dict(turned, v=both[..., H * D - 8:(H + hk) * D - 8], q_out=both[..., :H * D])):
        with pytest.raises(ValueError, match="overlap"):
            call(**bad)
    assert bool((kp == 1).all()) and bool((vp == 1).all())
    kp2, vp2 = pool(dev, 6, page, hk, D, fill=0.0)
    want = call(kp=kp2, vp=vp2, **turned)
    both[..., H * D:(H + hk) * D], both[..., (H + hk) * D:] = k, v
    got = call(kp=rows[:, :, :hk], vp=rows[:, :, hk:], k=both[..., H * D:(H + hk) * D], v=both[..., (H + hk) * D:],
               q_out=both[..., :H * D], **turned)
    assert torch.equal(got, want) and torch.equal(rows[:, :, :hk], kp2) and torch.equal(rows[:, :, hk:], vp2)

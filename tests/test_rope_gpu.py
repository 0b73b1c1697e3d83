"""Rotary positions on the B200 (npub200_rope through kernels.rope) against the formula in 64 bits.

Tolerance, per element, from the arithmetic. The angle in turns is rounded to f32 after its reduction to [-1, 1] half turns
(2^-25 of a half turn, pi 2^-25 rad) and p f / (2 pi) carries two roundings of 64 bits (2 pi |turns| 2^-52); sincospif is
good to 2 ulp (2^-22 at most, values up to 1), the magnitude rounds twice (2 x 2^-24 with its own conversion) and two products and a sum round
three times. With W = m (|u| + |v|) that is below W (2^-23 + 2^-22 + 2^-23 + 3 2^-24 + |p f| 2^-51) <= W (2^-21 + |p f| 2^-51).
The output rounds once more: half a step, 2^-8 (bf16) or 2^-24 (f32) of the value."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}


def turned(x, at, freqs, magnitude=1.0, interleaved=False, inverse=False):
    """(value, tolerance before the output's rounding) of x [B, H, S, D] at the positions at [B, S], in 64 bits."""
    x = x.double()
    r = 2 * freqs.numel()
    angle = (at.double()[..., None] * freqs)[:, None]
    c, s = angle.cos() * magnitude, angle.sin() * magnitude
    s = -s if inverse else s
    if interleaved:
        u, v = x[..., 0:r:2], x[..., 1:r:2]
    else:
        u, v = x[..., :r // 2], x[..., r // 2:r]
    w = abs(magnitude) * (u.abs() + v.abs()) * (2.0 ** -21 + angle.abs() * 2.0 ** -51)

    def join(a, b):
        return torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    rest = x[..., r:]
    return (torch.cat((join(u * c - v * s, v * c + u * s), rest), -1), torch.cat((join(w, w), torch.zeros_like(rest)), -1))


def check(y, ref, tol):
    tol = tol + HALF[y.dtype] * (ref.abs() + tol) + 1e-37
    err = (y.double() - ref).abs()
    assert bool((err <= tol).all()), f"{float((err / tol).max())} of the tolerance"


def heads_of(t, H, head_major):
    return t if head_major else t.unflatten(-1, (H, -1)).transpose(1, 2)


def frequencies(r, dev, base=10000.0):
    from npu_ai_b200 import kernels
    return kernels.rope_frequencies(r, base, device=dev)[0] if r else torch.empty(0, dtype=torch.float64, device=dev)


def make(dev, B, S, H, D, dtype, head_major, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return torch.randn(*((B, H, S, D) if head_major else (B, S, H * D)), generator=g, device=dev).to(dtype)


@pytest.mark.parametrize("D,r", [(2, 2), (6, 4), (40, 40), (64, 32), (66, 66), (72, 72), (80, 20), (96, 24), (128, 128),
                                 (160, 64), (256, 250), (64, 0), (1024, 1024)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("src,dst", [(BF16, BF16), (F32, BF16), (BF16, F32), (F32, F32)])
def test_widths_types_and_layouts(cuda_device, D, r, interleaved, src, dst):
    from npu_ai_b200 import kernels
    dev = cuda_device
    f = frequencies(r, dev)
    for B, S, H, head_major in ((1, 1, 1, False), (2, 5, 3, False), (3, 33, 2, True)):
        x = make(dev, B, S, H, D, src, head_major, seed=D + r)
        at = torch.arange(S, device=dev).expand(B, S) + 7
        y = kernels.rope(x, f, H, 7, interleaved=interleaved, head_major=head_major, out_dtype=dst, magnitude=1.25)
        assert y.dtype == dst and y.shape == x.shape
        check(heads_of(y, H, head_major), *turned(heads_of(x, H, head_major), at, f, 1.25, interleaved))


@pytest.mark.parametrize("top", [0, 1, 100000, 2 ** 31 - 1])
def test_positions(cuda_device, top):
    """Starts of each sequence and positions of each token, negative and far ones; expanded and strided tables of them."""
    from npu_ai_b200 import kernels
    dev = cuda_device
    B, S, H, D = 3, 9, 2, 64
    f = frequencies(D, dev)
    x = make(dev, B, S, H, D, F32, False, 1)
    starts = torch.tensor([top, -top, top // 2], dtype=torch.int32, device=dev)
    each = torch.randint(-top, top + 1, (S, B), device=dev).to(torch.int32).t()  # strided
    seq = torch.arange(S, device=dev)
    for given, at in ((starts, starts.long()[:, None] + seq), (each, each), (each[:, :1].expand(B, S), each[:, :1].expand(B, S)),
                      (each[:1].expand(B, S), each[:1].expand(B, S))):
        y = kernels.rope(x, f, H, given)
        check(heads_of(y, H, False), *turned(heads_of(x, H, False), at, f))
    y = kernels.rope(x, f, H, -5)
    check(heads_of(y, H, False), *turned(heads_of(x, H, False), (seq - 5).expand(B, S), f))


def test_strides_and_alignment(cuda_device):
    """Slices of a fused projection, of buffers that start off a 16-byte boundary, expanded inputs and outputs in place."""
    from npu_ai_b200 import kernels
    dev = cuda_device
    B, S, H, D = 2, 13, 4, 64
    f = frequencies(32, dev)
    at = torch.arange(S, device=dev).expand(B, S) + 100
    for off in (0, 1, 2, 4, 8, 3):
        for dtype in (BF16, F32):
            buf = make(dev, B, S, 1, 3 * H * D + 8, dtype, False, off)
            x = buf[..., off:off + H * D]
            ref = turned(heads_of(x, H, False), at, f)
            for interleaved in (False, True):
                ref = turned(heads_of(x, H, False), at, f, interleaved=interleaved)
                check(heads_of(kernels.rope(x, f, H, 100, interleaved=interleaved), H, False), *ref)
                out = torch.full_like(buf, 3.0)
                y = kernels.rope(x, f, H, 100, interleaved=interleaved, out=out[..., off + 1:off + 1 + H * D])
                check(heads_of(y, H, False), *ref)
                assert bool((out[..., :off + 1] == 3).all()) and bool((out[..., off + 1 + H * D:] == 3).all())
            keep = buf.clone()
            ref = turned(heads_of(keep[..., off:off + H * D], H, False), at, f)
            y = kernels.rope(x, f, H, 100, out=x)
            assert y.data_ptr() == x.data_ptr()
            check(heads_of(x, H, False), *ref)
            assert torch.equal(buf[..., off + H * D:], keep[..., off + H * D:])
    one = make(dev, 1, 1, H, D, BF16, False, 3).expand(B, S, H * D)
    check(heads_of(kernels.rope(one, f, H, 100), H, False), *turned(heads_of(one, H, False), at, f))
    x = make(dev, B, S, H, D, BF16, True, 4)  # (B, H, S, D) as a view of (B, S, H, D) and back
    y = kernels.rope(x.transpose(1, 2).contiguous().transpose(1, 2), f, H, 100, head_major=True)
    assert torch.equal(y, kernels.rope(x, f, H, 100, head_major=True))


def test_inverse_and_gradient(cuda_device):
    """The inverse undoes the rotation; with the same magnitude it is the gradient, against the formula's by autograd and
    against differences."""
    from npu_ai_b200 import kernels
    dev = cuda_device
    B, S, H, D, m = 2, 21, 3, 80, 1.3
    for interleaved in (False, True):
        f = frequencies(48, dev)
        x = make(dev, B, S, H, D, F32, True, 5)
        at = torch.arange(S, device=dev).expand(B, S) + 50
        kw = dict(interleaved=interleaved, head_major=True)
        y = kernels.rope(x, f, H, 50, **kw)
        back = kernels.rope(y, f, H, 50, inverse=True, **kw)
        _, tol = turned(x, at, f, interleaved=interleaved)
        u = x.double().abs() + y.double().abs()
        assert bool(((back.double() - x.double()).abs() <= 8 * tol + 8 * 2.0 ** -24 * (u + u.amax(-1, keepdim=True))).all())
        dy = make(dev, B, S, H, D, F32, True, 6)
        dx = kernels.rope(dy, f, H, 50, inverse=True, magnitude=m, **kw)
        xd = x.double().requires_grad_()
        turned(xd, at, f, m, interleaved)[0].backward(dy.double())
        _, tol = turned(dy, at, f, m, interleaved, True)
        check(dx, xd.grad, tol)
        # the operator is linear: a difference over any step is the derivative
        step = make(dev, B, S, H, D, F32, True, 7)
        a, b = (kernels.rope(t, f, H, 50, magnitude=m, **kw).double() for t in (x, x + step))
        exact = (x + step).double() - x.double()
        lhs, rhs = ((b - a) * dy.double()).sum(-1), (exact * dx.double()).sum(-1)
        size = ((a.abs() + b.abs() + 2.6 * (x.abs() + step.abs())) * (dy.abs() + dx.abs())).double().sum(-1) * 4
        assert bool(((lhs - rhs).abs() <= 2.0 ** -20 * size).all())


def test_empty_calls(cuda_device):
    from npu_ai_b200 import kernels
    f = frequencies(64, cuda_device)
    for shape in ((0, 5, 128), (2, 0, 128)):
        x = torch.empty(*shape, dtype=BF16, device=cuda_device)
        assert kernels.rope(x, f, 2).shape == x.shape


def test_refusals(cuda_device):
    from npu_ai_b200 import kernels
    dev = cuda_device
    x = make(dev, 2, 4, 2, 64, BF16, False)
    f = frequencies(64, dev)
    ints = torch.zeros(2, dtype=torch.int32, device=dev)
    for bad in (lambda: kernels.rope(x, f.float(), 2), lambda: kernels.rope(x, f.cpu(), 2), lambda: kernels.rope(x, f, 3),
                lambda: kernels.rope(x, f, 4), lambda: kernels.rope(x, f, 0), lambda: kernels.rope(x.half(), f, 2),
                lambda: kernels.rope(x[0], f, 2), lambda: kernels.rope(x, f, 2, head_major=True),
                lambda: kernels.rope(x, f, 2, ints.long()), lambda: kernels.rope(x, f, 2, ints[:1]),
                lambda: kernels.rope(x, f, 2, ints.cpu()), lambda: kernels.rope(x, f, 2, torch.stack((ints, ints))),
                lambda: kernels.rope(x, f, 2, out=x[:1]), lambda: kernels.rope(x, f, 2, out_dtype=torch.float16),
                lambda: kernels.rope(x.mT, f, 2), lambda: kernels.rope(x, f, 2, magnitude=float("nan")),
                lambda: kernels.rope(x, f, 2, out=x[:, :1].expand(2, 4, 128)),
                lambda: kernels.rope(x.view(-1)[:512].view(1, 4, 128), f, 2, out=x.view(-1)[128:640].view(1, 4, 128)),
                lambda: kernels.rope(x, f.repeat_interleave(2)[::2], 2), lambda: kernels.rope(x, f, 2, 2 ** 31)):
        with pytest.raises(ValueError):
            bad()


def test_graph_and_other_stream(cuda_device):
    """A captured call follows the positions; on another stream than the tensors' own."""
    from npu_ai_b200 import kernels
    dev = cuda_device
    x = make(dev, 2, 3, 4, 64, BF16, False, 9)
    f = frequencies(64, dev)
    starts = torch.tensor([5, 6], dtype=torch.int32, device=dev)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        kernels.rope(x, f, 4, starts)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = kernels.rope(x, f, 4, starts)
        for k in range(3):
            starts.add_(1000 * k)
            graph.replay()
            side.synchronize()
            at = starts.long()[:, None] + torch.arange(3, device=dev)
            check(heads_of(y, 4, False), *turned(heads_of(x, 4, False), at, f))


def test_offsets_past_32_bits(cuda_device):
    """A tensor of more than 2^32 bytes and 2^31 elements, turned in place; its ends and what lies in between."""
    from npu_ai_b200 import kernels
    dev = cuda_device
    S, H, D = 2 ** 18 + 3, 64, 130
    x = torch.empty(1, S, H * D, dtype=BF16, device=dev)
    assert x.numel() > 2 ** 31
    x.copy_(torch.randn(1, 1, H * D, device=dev))
    keep = x[:, :1].clone()
    f = frequencies(130, dev)
    kernels.rope(x, f, H, out=x)
    for s in (0, 1, 2 ** 17, S - 2, S - 1):
        at = torch.full((1, 1), s, device=dev)
        check(heads_of(x[:, s:s + 1], H, False), *turned(heads_of(keep, H, False), at, f))


def test_many_tokens_and_heads(cuda_device):
    """Blocks of several tokens, their last one ragged, and heads split over blocks."""
    from npu_ai_b200 import kernels
    dev = cuda_device
    for B, S, H, D, head_major in ((3, 1001, 5, 72, False), (1, 4099, 8, 64, True), (1, 2, 96, 128, False), (7, 1, 257, 8, False)):
        x = make(dev, B, S, H, D, BF16, head_major, S)
        f = frequencies(D // 2, dev)
        starts = torch.arange(B, dtype=torch.int32, device=dev) * 1000
        y = kernels.rope(x, f, H, starts, head_major=head_major)
        at = starts.long()[:, None] + torch.arange(S, device=dev)
        check(heads_of(y, H, head_major), *turned(heads_of(x, H, head_major), at, f))


def test_outputs_that_overlap_are_refused(cuda_device):
    """Columns of one buffer, which are no dense tensors: an output moved inside its input is refused, one next to it taken."""
    from npu_ai_b200 import kernels
    dev = cuda_device
    B, S, H, D = 2, 5, 4, 64
    f = frequencies(D, dev)
    buf = make(dev, B, S, 3 * H, D, BF16, False, 4)
    x, keep = buf[..., :H * D], buf.clone()
    for out in (buf[..., D // 2:D // 2 + H * D], buf[..., H * D - 2:2 * H * D - 2], buf.view(torch.float32)[..., :H * D],
                torch.as_strided(buf, x.shape, (x.stride(0), x.stride(1) - 8, 1))):
        with pytest.raises(ValueError, match="overlap"):
            kernels.rope(x, f, H, 7, out=out)
    assert torch.equal(buf, keep)
    want = kernels.rope(x, f, H, 7)
    assert torch.equal(kernels.rope(x, f, H, 7, out=buf[..., H * D:2 * H * D]), want)
    assert torch.equal(buf[..., :H * D], keep[..., :H * D]) and torch.equal(buf[..., 2 * H * D:], keep[..., 2 * H * D:])
    assert torch.equal(kernels.rope(x, f, H, 7, out=x), want) and torch.equal(x, want)

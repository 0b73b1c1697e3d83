"""Packed documents whose last keys no row sees, on the B200: such V rows are not read into the result."""
import pytest

from test_attention_masked_gpu import INF, _qkv, check, ints, oracle

pytestmark = pytest.mark.gpu

NAN = float("nan")


@pytest.mark.parametrize("D", [40, 128, 160])
@pytest.mark.parametrize("variant", [1, 2, 5])
@pytest.mark.parametrize("per_batch", [False, True])
def test_documents_whose_ends_no_row_sees(cuda_device, D, variant, per_batch):
    """Documents, causal, and positions that start below 0: a document's last keys come after every row's position. They
    lie between the keys of one Q tile, and may hold anything."""
    from npu_ai_b200 import kernels
    dev, S = cuda_device, 400
    for start, off in ((-50, (0, 130, 150, 240, 400)), (-1, (7, 60, 61, 62, 200, 390)), (-2, tuple(range(0, 401, 5))),
                       (-70, (0, 400))):
        for prefix in (None, 3):
            q, k, v = _qkv(2, 4, 2, S, S, D, D - start, dev)
            kw = dict(causal=True, doc_offsets=ints(dev, *off), prefix_len=prefix,
                      q_start=ints(dev, start, start) if per_batch else start)
            ref = oracle(q, k, v, 4, 2, **kw)
            for s, e in zip(off, off[1:]):
                dead = slice(max(s, e + start, min(prefix or 0, e)), e)
                k[:, dead], v[:, dead] = NAN, INF
            out = kernels.attention(q, k, v, 4, variant=variant, **kw)
            kernels.check_status(dev)
            check(out, *ref, 4, False)

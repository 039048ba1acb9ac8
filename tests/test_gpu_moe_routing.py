"""Which experts are chosen is decided on logits that fp32 sums would order otherwise (gpu).

The expected order is that of 64-bit logits, whose gaps here are at least 2^-31 and whose
own error, D 2^-53 of the sum of magnitudes, is below 2^-38."""
import pytest
import torch

from deepx_op_gpukernelcompiler_b200 import moe_ffn
from test_gpu_moe import DEV, make

pytestmark = pytest.mark.gpu


def _routing(t, k, **kw):
    y, w, ids = moe_ffn(**t, top_k=k, return_routing=True, **kw)
    return w.cpu().double(), ids.cpu().long()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,rows", [(24, (0, 1, 2)), (4096, (0, 1, 2)), (4096, (7, 1500, 4000))])
def test_small_terms_between_large_ones(D, rows, dtype):
    """2^14 + s - 2^14 for small s: an fp32 sum keeps steps of 2^-10 at best."""
    t = make(3, D, 8, 4, dtype)
    t["X"].zero_()
    t["Wr"].zero_()
    t["X"][:, list(rows)] = 128.0
    t["Wr"][rows[0]], t["Wr"][rows[2]] = 128.0, -128.0
    small = torch.tensor([1.0, 3.0, 2.0, 4.0], device=DEV) * 2.0 ** -22
    t["Wr"][rows[1]] = small.to(dtype)
    w, ids = _routing(t, 4)
    assert (ids == torch.tensor([3, 1, 2, 0])).all()
    want = torch.softmax(small.cpu().double() * 128, 0)[[3, 1, 2, 0]]
    # expf and the sum of 4 values, rounded: 8 steps of 2^-24 of a weight of 1/4
    assert (w - want).abs().max() <= 2.0 ** -23


@pytest.mark.parametrize("T,D,E,k", [(1, 512, 8, 3), (2, 1032, 16, 5), (9, 2048, 64, 8),
                                     (64, 1024, 200, 8), (33, 264, 256, 32)])
def test_near_ties(T, D, E, k):
    """Pairs of experts whose columns differ in one small value by its last bit."""
    t = make(T, D, 8, E, torch.bfloat16)
    half = E // 2
    t["X"][:, 5] = 1.0
    t["X"][T // 2:, 5] = -1.0
    t["Wr"][:, half:2 * half] = t["Wr"][:, :half]
    t["Wr"][5, :half] = 2.0 ** -20
    t["Wr"][5, half:2 * half] = 2.0 ** -20 * (1 + 2.0 ** -7)
    logits = t["X"].cpu().double() @ t["Wr"].cpu().double()
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
    gaps = logits.sort(1).values.diff(dim=1)
    assert gaps.min() >= 2.0 ** -31
    for renorm in (True, False):
        w, ids = _routing(t, k, renormalize=renorm)
        assert torch.equal(ids, order)
        want = torch.gather(torch.softmax(logits, 1), 1, order)
        if renorm:
            want = want / want.sum(1, keepdim=True)
        assert (w - want).abs().max() <= 2.0 ** -19

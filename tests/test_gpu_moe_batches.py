"""The mixture-of-experts layer at the sizes it serves, and a token alone against the
same token in a batch (gpu).

Alone or in a batch a token's sums are split over other CTAs, so the bits may differ;
either is within the tolerance of the definition (moe_oracle.py)."""
import pytest
import torch

import moe_oracle as ref
from deepx_op_gpukernelcompiler_b200 import _native as nat
from deepx_op_gpukernelcompiler_b200 import moe_ffn
from test_gpu_moe import DEV, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_token_alone_and_in_a_batch(dtype):
    t = make(24, 512, 640, 8, dtype, bias=True, residual=True)
    Y, W, ids = moe_ffn(**t, top_k=3, return_routing=True)
    for i in (0, 7, 8, 23):
        one = t | {"X": t["X"][i:i + 1], "residual": t["residual"][i:i + 1]}
        want = ref.moe(**one, top_k=3)
        got = moe_ffn(**one, top_k=3, return_routing=True)
        ref.check(got, want, f"token {i} alone")
        ref.check((Y[i:i + 1], W[i:i + 1], ids[i:i + 1]), want, f"token {i} in the batch")
        # the routing does not depend on the batch
        assert torch.equal(got[2], ids[i:i + 1]) and torch.equal(got[1], W[i:i + 1])


@pytest.mark.parametrize("T,D,H,E,k,dtype", [
    (1, 4096, 14336, 3, 2, torch.bfloat16), (8, 2048, 1024, 64, 8, torch.bfloat16),
    (33, 1032, 2824, 16, 4, torch.float16), (64, 2048, 1024, 64, 8, torch.float16),
])
def test_layers_of_the_sizes_that_are_served(T, D, H, E, k, dtype):
    t = make(T, D, H, E, dtype, bias=T == 33, residual=T != 1)
    got = moe_ffn(**t, top_k=k, return_routing=True)
    ref.check(got, ref.moe(**t, top_k=k))
    for _ in range(10):
        again = moe_ffn(**t, top_k=k, return_routing=True)
        assert all(torch.equal(a, b) for a, b in zip(again, got))
    assert nat.device_status(torch.cuda.current_stream().cuda_stream) == 0


def test_experts_that_are_switched_off():
    """Logits of -inf.  One expert left: the second choice is the lowest number of the
    others, with weight 0.  None left: the softmax over nothing, NaN."""
    t = make(5, 64, 72, 4, torch.bfloat16)
    t["br"] = torch.full((4,), float("-inf"), dtype=torch.bfloat16, device=DEV)
    t["br"][2] = 0.0
    got = moe_ffn(**t, top_k=2, return_routing=True)
    assert (got[2] == torch.tensor([2, 0], device=DEV, dtype=torch.int32)).all()
    assert (got[1] == torch.tensor([1.0, 0.0], device=DEV)).all()
    ref.check(got, ref.moe(**t, top_k=2))
    t["br"][2] = float("-inf")
    Y, w, ids = moe_ffn(**t, top_k=2, return_routing=True)
    assert (ids == torch.tensor([0, 1], device=DEV, dtype=torch.int32)).all()
    assert torch.isnan(w).all() and torch.isnan(Y).all()

"""The mixture-of-experts layer where hidden values are small and Wo large (gpu).

Outputs are of ordinary size, so their relative error in the 2-norm is that of the
rounding, at most eps / 2 / sqrt 3 = 0.289 eps if every output had the mantissa 1, plus
that of the hidden values.  Those pass as hi + lo; a relative error of 2^-17 (bf16) or an
absolute one of 2^-37 where they are some 2^-21 (fp16, X of scale 0.001) adds less than
0.002 or 0.02 eps, and its square to the square."""
import pytest
import torch

import moe_oracle as ref
from deepx_op_gpukernelcompiler_b200 import _native as nat
from deepx_op_gpukernelcompiler_b200 import moe_ffn
from test_gpu_moe import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,D,H,E,k", [(1, 1024, 1024, 2, 1), (9, 256, 1000, 5, 2),
                                       (20, 1024, 512, 4, 2), (64, 512, 264, 3, 1)])
@pytest.mark.parametrize("scale", [1.0, 0.1, 0.01, 0.003, 0.001])
def test_small_hidden_values(scale, T, D, H, E, k, dtype):
    t = make(T, D, H, E, dtype)
    t["X"] = (t["X"].float() * scale).to(dtype)
    # SiLU(g) u is some scale^2 / 2 there; Wo brings the output back to ordinary sizes.
    t["Wo"] = (t["Wo"].float() * min(scale ** -2, 4000.0)).to(dtype)
    assert torch.isfinite(t["Wo"]).all()
    Y, _, ids = moe_ffn(**t, top_k=k, return_routing=True)
    y, _, _, _, order = ref.moe(**t, top_k=k)
    assert torch.equal(ids.cpu().long(), order)
    assert y.abs().mean() > 2.0 ** -12  # (few outputs among the subnormals)
    off = ((Y.cpu().double() - y).norm() / y.norm()).item()
    assert off <= 0.3 * torch.finfo(dtype).eps, off / torch.finfo(dtype).eps
    assert nat.device_status(torch.cuda.current_stream().cuda_stream) == 0

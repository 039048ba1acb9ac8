"""The mixture-of-experts layer where a phase has whole waves of tiles behind shared
ones (gpu): very wide layers, and layers on a part of the SMs.

tests/test_moe_plan_cpu.py checks the partition of these sizes."""
import pytest
import torch

import moe_oracle as ref
from deepx_op_gpukernelcompiler_b200 import _native as nat
from deepx_op_gpukernelcompiler_b200 import moe_ffn
from test_gpu_moe import DEV, make

pytestmark = pytest.mark.gpu


def _grid():
    return int(nat.last_launch_plan().split("grid=")[1].split()[0])


@pytest.mark.parametrize("T,D,H,E,k", [(64, 65536, 192, 1, 1), (20, 40072, 1448, 3, 2)])
def test_shared_tiles_then_whole_ones(T, D, H, E, k):
    t = make(T, D, H, E, torch.bfloat16, residual=True)
    got = moe_ffn(**t, top_k=k, return_routing=True)
    assert len(set(got[2].flatten().tolist())) == E
    ref.check(got, ref.moe(**t, top_k=k))
    for _ in range(20):
        assert torch.equal(moe_ffn(**t, top_k=k), got[0])
    assert nat.device_status(torch.cuda.current_stream().cuda_stream) == 0


@pytest.mark.parametrize("sms,T,D,H,E,k", [(24, 33, 7168, 2048, 8, 4), (8, 64, 2880, 2880, 1, 1)])
def test_on_a_part_of_the_sms(sms, T, D, H, E, k):
    t = make(T, D, H, E, torch.bfloat16)
    part = torch.cuda.GreenContext.create(num_sms=sms, device_id=0)
    raw = part.Stream()
    stream = torch.cuda.Stream(stream_id=raw.stream_id, device_index=raw.device_index,
                               device_type=raw.device_type)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        got = moe_ffn(**t, top_k=k, return_routing=True)
        assert _grid() == sms
        again = [moe_ffn(**t, top_k=k) for _ in range(10)]
    stream.synchronize()
    ref.check(got, ref.moe(**t, top_k=k))
    assert all(torch.equal(y, got[0]) for y in again)
    assert nat.device_status(torch.cuda.current_stream().cuda_stream) == 0

"""Layers on a part of the SMs: grids follow the partition of the launching stream (gpu).

Partitions come and go in one process; a new one may have the handle of one that is
gone, with another size."""
import gc

import pytest
import torch

import int8_oracle
import moe_oracle
from deepx_op_gpukernelcompiler_b200 import _native as nat
from deepx_op_gpukernelcompiler_b200 import fused_linear, int8_linear, int8_rows, moe_ffn
from test_gpu_moe import DEV, make

pytestmark = pytest.mark.gpu


def _stream(part):
    raw = part.Stream()
    return torch.cuda.Stream(stream_id=raw.stream_id, device_index=raw.device_index,
                             device_type=raw.device_type)


def _grid():
    return int(nat.last_launch_plan().split("grid=")[1].split()[0])


def test_partitions_that_come_and_go():
    t = make(9, 1024, 264, 4, torch.bfloat16)
    want = moe_oracle.moe(**t, top_k=2)
    g = torch.Generator(device=DEV).manual_seed(3)
    X = torch.randn(300, 512, generator=g, device=DEV).to(torch.bfloat16)
    q = torch.randint(-127, 128, (6000, 512), generator=g, device=DEV, dtype=torch.int8)
    W = int8_rows(q, torch.full((6000,), 1e-3, device=DEV))
    product = int8_oracle.linear(X, W)
    W16 = torch.randn(512, 6000, generator=g, device=DEV).to(torch.bfloat16) / 512 ** 0.5
    whole = fused_linear(X, W16)
    torch.cuda.synchronize()
    for sms in (24, 8, 40, 16, 8, 24):
        part = torch.cuda.GreenContext.create(num_sms=sms, device_id=0)
        stream = _stream(part)
        with torch.cuda.stream(stream):
            got = moe_ffn(**t, top_k=2, return_routing=True)
            assert _grid() == sms
            Y = int8_linear(X, W)
            assert _grid() == sms  # CTA pairs, more tiles than fit
            Y16 = fused_linear(X, W16)
            assert _grid() <= sms
        stream.synchronize()
        moe_oracle.check(got, want, f"{sms} SMs")
        int8_oracle.check(Y, product, f"{sms} SMs")
        assert torch.equal(Y16, whole)
        del stream, part
        gc.collect()
    assert nat.device_status(torch.cuda.current_stream().cuda_stream) == 0

"""The activations of the 8-bit products over their whole range, tails included (gpu).

One 8-bit value 1 with scale 1 times weights 1 with scales v gives act(v) for any fp32
v.  Tolerance of a value y = act(v): the output's rounding, half a step (u |y|, 2^-25
among fp16's subnormals), and before it

    (z 2^-21 + 2^-20) |y|

where e^-z is the exponential that y is made of.  z reaches the exponential by at most
8 roundings (GELU-tanh: x x, 0.0447 x, their multiply-add, two products by constants and
three constants), 8 ln 2 2^-24 < 2^-21 of it; the exponential, the reciprocal, the
products and the erfc polynomial (6.3e-7) make up at most 2^-20 more."""
import math

import pytest
import torch

import int8_oracle as ref
from deepx_op_gpukernelcompiler_b200 import _native as nat
from deepx_op_gpukernelcompiler_b200 import int8_linear

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
RANGE = {"silu": 80.0, "gelu_tanh": 9.0, "gelu_erf": 12.9, "relu": 100.0}


def _tanh_arg(v):
    return 2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)


def _act(v, act):
    # (0.5 (1 + tanh u) = sigmoid(2 u); 1 + tanh u itself cancels, in 64 bits too)
    return v * torch.sigmoid(_tanh_arg(v)) if act == "gelu_tanh" else ref.act64(v, act)


def _exponent(v, act):
    if act == "silu":
        return v.abs()
    if act == "gelu_tanh":
        return _tanh_arg(v).abs()
    return v * v / 2 if act == "gelu_erf" else torch.zeros_like(v)


@pytest.mark.parametrize("kernel", ["decode", "umma"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", list(RANGE))
def test_whole_range(act, dtype, kernel):
    top = RANGE[act]
    v = torch.cat([torch.linspace(-top, top, 20001), torch.logspace(-6, 0, 2000),
                   -torch.logspace(-6, 0, 2000)]).to(DEV)
    one = torch.ones(1, 1, dtype=torch.int8, device=DEV)
    W = torch.zeros(v.numel(), 16, dtype=torch.int8, device=DEV)
    W[:, 0] = 1
    got = int8_linear((one, torch.ones(1, device=DEV)), (W[:, :1], v), activation=act, dtype=dtype,
                      kernel=kernel)[0]
    assert nat.last_launch_plan().startswith("int8_pair" if kernel == "umma" else "int8_tile")
    x = v.cpu().double()
    y = _act(x, act)
    tol = (torch.finfo(dtype).eps / 2 + _exponent(x, act) * 2.0 ** -21 + 2.0 ** -20) * y.abs()
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25
    off = (got.cpu().double() - y).abs() - tol
    i = int(off.argmax())
    assert off[i] <= 0, f"act({x[i].item()}): got {got[i].item()}, want {y[i].item()} +- {tol[i].item()}"


@pytest.mark.parametrize("kernel", ["decode", "umma"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", list(RANGE))
def test_infinite_and_nan_biases(act, dtype, kernel):
    """Each in its column alone; where the definition gives NaN, NaN."""
    inf, nan = float("inf"), float("nan")
    b = torch.tensor([inf, -inf, nan, 1.0, torch.finfo(dtype).max, -torch.finfo(dtype).max, -1.0,
                      0.0], dtype=dtype, device=DEV)
    zero = torch.zeros(3, 16, dtype=torch.int8, device=DEV), torch.ones(3, device=DEV)
    W = torch.zeros(8, 16, dtype=torch.int8, device=DEV), torch.ones(8, device=DEV)
    got = int8_linear(zero, W, b, act, dtype=dtype, kernel=kernel).cpu().double()
    y = _act(b.cpu().double(), act)
    assert torch.equal(torch.isnan(got), torch.isnan(y).expand(3, 8)), (got, y)
    keep = ~torch.isnan(y)
    want = y[keep].to(dtype).double().expand(3, -1)
    assert torch.allclose(got[:, keep], want, rtol=2 * torch.finfo(dtype).eps, atol=0), (got, y)

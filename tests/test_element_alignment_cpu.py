"""Pointers off their elements' alignment are refused before anything is launched (CPU):
a kernel that read through one would fault."""
import ctypes

import pytest

from deepx_op_gpukernelcompiler_b200 import _build, _native as nat

FAKE = 0x1000  # never dereferenced: validation fails first


@pytest.fixture(scope="module")
def lib():
    _build.build()
    return nat.load()


@pytest.mark.parametrize("x,scale,dtype", [(1, 0, nat.DX_DTYPE_BF16), (1, 0, nat.DX_DTYPE_F16),
                                           (2, 0, nat.DX_DTYPE_F32), (0, 2, nat.DX_DTYPE_BF16)])
def test_quantize_rows(lib, x, scale, dtype):
    rc = lib.dx_quantize_rows(FAKE + x, FAKE, FAKE + scale, 2, 8, 8, 8, dtype, None)
    assert rc == nat.DX_ERR_INVALID_ARGUMENT and "aligned to its elements" in nat.last_error()


@pytest.mark.parametrize("dtype,kw", [
    (nat.DX_DTYPE_BF16, dict(sx=2)), (nat.DX_DTYPE_BF16, dict(sw=1)),
    (nat.DX_DTYPE_BF16, dict(bias=1)), (nat.DX_DTYPE_F32, dict(bias=2)),
    (nat.DX_DTYPE_F16, dict(R=1)), (nat.DX_DTYPE_F32, dict(Y=2)), (nat.DX_DTYPE_F16, dict(Y=1)),
])
def test_int8_linear(lib, dtype, kw):
    p = {k: FAKE + kw.get(k, 0) for k in ("sx", "sw", "bias", "R", "Y")}
    rc = lib.dx_int8_linear(FAKE, nat.DX_DTYPE_I8, p["sx"], FAKE, p["sw"], p["bias"], p["R"],
                            p["Y"], 4, 32, 32, 32, 32, 32, 32, dtype, 0, 0, None, 0, None)
    assert rc == nat.DX_ERR_INVALID_ARGUMENT and "aligned to its elements" in nat.last_error()


def test_int8_linear_floating_point_x(lib):
    rc = lib.dx_int8_linear(FAKE + 2, nat.DX_DTYPE_F32, None, FAKE, FAKE, None, None, FAKE, 4, 32,
                            32, 32, 32, 32, 32, nat.DX_DTYPE_BF16, 0, 0, FAKE, 1 << 20, None)
    assert rc == nat.DX_ERR_INVALID_ARGUMENT and "aligned to its elements" in nat.last_error()


@pytest.mark.parametrize("kw", [dict(wu_scale=2), dict(bias_u=1)])
def test_int8_gated_linear(lib, kw):
    p = {k: FAKE + kw.get(k, 0) for k in ("wu_scale", "bias_u")}
    rc = lib.dx_int8_gated_linear(FAKE, nat.DX_DTYPE_I8, FAKE, FAKE, FAKE, FAKE, p["wu_scale"],
                                  None, p["bias_u"], FAKE, 4, 32, 32, 32, 32, 32, 32,
                                  nat.DX_DTYPE_F16, 0, 0, None, 0, None)
    assert rc == nat.DX_ERR_INVALID_ARGUMENT and "aligned to its elements" in nat.last_error()


@pytest.mark.parametrize("kw", [dict(Wr=1), dict(br=1), dict(bg=1), dict(bu=1), dict(bo=1),
                                dict(R=1), dict(Y=1), dict(ids=2), dict(weights=2)])
def test_moe(lib, kw):
    names = ("X", "Wr", "Wg", "Wu", "Wo", "Y", "ids", "weights", "br", "bg", "bu", "bo", "R")
    a = nat.MoeArgs(**{k: FAKE + kw.get(k, 0) for k in names}, T=4, D=64, H=32, E=8, top_k=2,
                    ldx=64, ldwr=8, ldg=32, ldg_expert=2048, ldu=32, ldu_expert=2048, ldo=64,
                    ldo_expert=2048, ldr=64, ldy=64, dtype=nat.DX_DTYPE_BF16, act=0, renormalize=1)
    assert lib.dx_moe(ctypes.addressof(a), None) == nat.DX_ERR_INVALID_ARGUMENT
    assert "aligned to its elements" in nat.last_error()

"""The mixture-of-experts layer's argument checks (CPU; nothing is launched)."""
import ctypes

import pytest
import torch

from deepx_op_gpukernelcompiler_b200 import _build, _native as nat, moe_ffn

FAKE = 0x1000  # never dereferenced: validation fails first


@pytest.fixture(scope="module")
def lib():
    _build.build()
    return nat.load()


def _args(**kw):
    a = dict(X=FAKE, Wr=FAKE, Wg=FAKE, Wu=FAKE, Wo=FAKE, Y=FAKE, ids=FAKE, weights=FAKE, T=4, D=64,
             H=32, E=8, top_k=2, ldx=64, ldwr=8, ldg=32, ldg_expert=2048, ldu=32, ldu_expert=2048,
             ldo=64, ldo_expert=2048, ldr=64, ldy=64, dtype=nat.DX_DTYPE_BF16, act=0, renormalize=1)
    a.update(kw)
    return nat.MoeArgs(**a)


@pytest.mark.parametrize("kw,code,needle", [
    (dict(dtype=nat.DX_DTYPE_F32), nat.DX_ERR_UNSUPPORTED, "fp16"),
    (dict(dtype=9), nat.DX_ERR_INVALID_ARGUMENT, "dtype"),
    (dict(act=7), nat.DX_ERR_INVALID_ARGUMENT, "activation"),
    (dict(T=-1), nat.DX_ERR_INVALID_ARGUMENT, "T >= 0"),
    (dict(T=65), nat.DX_ERR_UNSUPPORTED, "64 tokens"),
    (dict(E=257, ldwr=257), nat.DX_ERR_UNSUPPORTED, "256 experts"),
    (dict(top_k=9), nat.DX_ERR_INVALID_ARGUMENT, "top_k"),
    (dict(top_k=0), nat.DX_ERR_INVALID_ARGUMENT, "top_k"),
    (dict(D=60), nat.DX_ERR_UNSUPPORTED, "multiples of 8"),
    (dict(H=65544), nat.DX_ERR_UNSUPPORTED, "65536"),
    (dict(Wo=None), nat.DX_ERR_INVALID_ARGUMENT, "NULL"),
    (dict(ids=None), nat.DX_ERR_INVALID_ARGUMENT, "NULL"),
    (dict(ldy=63), nat.DX_ERR_INVALID_ARGUMENT, "pitch"),
    (dict(ldwr=7), nat.DX_ERR_INVALID_ARGUMENT, "pitch"),
    (dict(R=FAKE, ldr=8), nat.DX_ERR_INVALID_ARGUMENT, "pitch"),
    (dict(X=FAKE + 2), nat.DX_ERR_UNSUPPORTED, "16-byte"),
    (dict(ldg=36, ldg_expert=4096), nat.DX_ERR_UNSUPPORTED, "16-byte"),
    (dict(ldu_expert=1024), nat.DX_ERR_INVALID_ARGUMENT, "expert's pitch"),
])
def test_host_validation(lib, kw, code, needle):
    a = _args(**kw)
    assert lib.dx_moe(ctypes.addressof(a), None) == code
    assert needle in nat.last_error()


def test_null_and_empty(lib):
    assert lib.dx_moe(None, None) == nat.DX_ERR_INVALID_ARGUMENT
    a = _args(T=0, X=None, Y=None)
    assert lib.dx_moe(ctypes.addressof(a), None) == nat.DX_OK
    assert lib.dx_moe_workspace_size(65, 32, 8, 2) == 0
    assert lib.dx_moe_workspace_size(4, 32, 8, 9) == 0


def test_python_refusals():
    dt = torch.bfloat16
    X, Wr = torch.zeros(4, 64, dtype=dt), torch.zeros(64, 8, dtype=dt)
    Wg, Wo = torch.zeros(8, 64, 32, dtype=dt), torch.zeros(8, 32, 64, dtype=dt)

    def call(X=X, Wr=Wr, Wg=Wg, Wu=Wg, Wo=Wo, top_k=2, **kw):
        return moe_ffn(X, Wr, Wg, Wu, Wo, top_k, **kw)

    with pytest.raises(ValueError, match="CUDA"):
        call()
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        call(X=X.float())
    with pytest.raises(ValueError, match="at most 64 tokens"):
        call(X=torch.zeros(65, 64, dtype=dt))
    with pytest.raises(ValueError, match="top_k"):
        call(top_k=9)
    with pytest.raises(ValueError, match="multiples of 8"):
        call(X=X[:, :60], Wr=Wr[:60])
    with pytest.raises(ValueError, match="Wu must have shape"):
        call(Wu=Wg[:, :, :24])
    with pytest.raises(ValueError, match="Wo must have shape"):
        call(Wo=Wg)
    with pytest.raises(ValueError, match="contiguous rows"):
        call(Wg=Wo.transpose(1, 2))
    with pytest.raises(ValueError, match="dtype"):
        call(Wo=Wo.half())
    with pytest.raises(ValueError, match="bg must be"):
        call(bg=torch.zeros(8, dtype=dt))
    with pytest.raises(ValueError, match="residual"):
        call(residual=torch.zeros(3, 64, dtype=dt))
    with pytest.raises(ValueError, match="activation"):
        call(activation="tanh")

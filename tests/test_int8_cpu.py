"""The 8-bit linear layers' argument checks (CPU; nothing is launched)."""
import ctypes

import pytest
import torch

from deepx_op_gpukernelcompiler_b200 import (Int8Rows, _build, _native as nat, int8_gated_ffn,
                                             int8_gated_linear, int8_linear, int8_rows,
                                             quantize_rows, quantize_weight)

import int8_oracle

FAKE = 0x1000  # never dereferenced: validation fails first


@pytest.fixture(scope="module")
def lib():
    _build.build()
    return nat.load()


def _linear(lib, **kw):
    a = dict(X=FAKE, x_dtype=nat.DX_DTYPE_I8, sx=FAKE, W=FAKE, sw=FAKE, bias=None, R=None, Y=FAKE,
             M=4, N=32, K=32, ldx=32, ldw=32, ldr=32, ldy=32, dtype=nat.DX_DTYPE_BF16, act=0,
             kernel=0, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    return lib.dx_int8_linear(*a.values())


@pytest.mark.parametrize("kw,code,needle", [
    (dict(dtype=nat.DX_DTYPE_I8), nat.DX_ERR_INVALID_ARGUMENT, "dtype"),
    (dict(x_dtype=7), nat.DX_ERR_INVALID_ARGUMENT, "x_dtype"),
    (dict(act=9), nat.DX_ERR_INVALID_ARGUMENT, "activation"),
    (dict(kernel=nat.DX_KERNEL_SIMT), nat.DX_ERR_INVALID_ARGUMENT, "kernel"),
    (dict(M=-1), nat.DX_ERR_INVALID_ARGUMENT, "M=-1"),
    (dict(K=0), nat.DX_ERR_INVALID_ARGUMENT, "K=0"),
    (dict(K=131072, ldx=131072, ldw=131072), nat.DX_ERR_UNSUPPORTED, "overflow"),
    (dict(M=1 << 40), nat.DX_ERR_UNSUPPORTED, "2^22"),
    (dict(Y=None), nat.DX_ERR_INVALID_ARGUMENT, "Y is NULL"),
    (dict(sx=None), nat.DX_ERR_INVALID_ARGUMENT, "scale"),
    (dict(W=None), nat.DX_ERR_INVALID_ARGUMENT, "NULL"),
    (dict(ldx=31), nat.DX_ERR_INVALID_ARGUMENT, "ldx"),
    (dict(ldw=16), nat.DX_ERR_INVALID_ARGUMENT, "pitch"),
    (dict(ldy=31), nat.DX_ERR_INVALID_ARGUMENT, "ldy"),
    (dict(R=FAKE, ldr=2), nat.DX_ERR_INVALID_ARGUMENT, "ldr"),
    (dict(ldw=40), nat.DX_ERR_UNSUPPORTED, "16-byte"),
    (dict(X=FAKE + 8), nat.DX_ERR_UNSUPPORTED, "16-byte"),
    (dict(x_dtype=nat.DX_DTYPE_BF16), nat.DX_ERR_WORKSPACE, "workspace"),
])
def test_linear_host_validation(lib, kw, code, needle):
    assert _linear(lib, **kw) == code
    assert needle in nat.last_error()


def test_empty_products_and_workspace(lib):
    assert _linear(lib, M=0, Y=None) == nat.DX_OK
    assert _linear(lib, N=0, Y=None) == nat.DX_OK
    assert lib.dx_int8_workspace_size(0, 64) == 0
    assert lib.dx_int8_workspace_size(1, 17) >= 32 + 4
    assert lib.dx_int8_workspace_size(5, 1 << 20) == 0


def test_gated_and_quantize_host_validation(lib):
    rc = lib.dx_int8_gated_linear(FAKE, nat.DX_DTYPE_I8, FAKE, FAKE, FAKE, None, FAKE, None, None,
                                  FAKE, 4, 32, 32, 32, 32, 32, 32, nat.DX_DTYPE_F16, 0, 0, None, 0,
                                  None)
    assert rc == nat.DX_ERR_INVALID_ARGUMENT and "Wu" in nat.last_error()
    assert lib.dx_quantize_rows(FAKE, FAKE, FAKE, 2, 8, 8, 8, 5, None) == nat.DX_ERR_INVALID_ARGUMENT
    assert lib.dx_quantize_rows(FAKE, None, FAKE, 2, 8, 8, 8, 1, None) == nat.DX_ERR_INVALID_ARGUMENT
    assert lib.dx_quantize_rows(FAKE, FAKE, FAKE, 2, 8, 7, 8, 1, None) == nat.DX_ERR_INVALID_ARGUMENT
    assert lib.dx_quantize_rows(None, None, None, 0, 8, 8, 8, 1, None) == nat.DX_OK


def _rows(n, k, **kw):
    return Int8Rows(torch.zeros(n, k, dtype=torch.int8), torch.ones(n), **kw)


def test_python_refusals():
    X = torch.zeros(4, 32, dtype=torch.bfloat16)
    W = _rows(16, 32)
    with pytest.raises(ValueError, match="CUDA"):
        quantize_rows(X)
    with pytest.raises(ValueError, match="CUDA"):
        int8_linear(X, W)
    with pytest.raises(ValueError, match="CUDA"):
        int8_gated_linear(X, W, W)
    with pytest.raises(ValueError, match="dtype"):
        int8_linear(X.to(torch.float64), W)
    with pytest.raises(ValueError, match="output dtype"):
        int8_linear(X, W, dtype=torch.int8)
    with pytest.raises(ValueError, match="activation"):
        int8_linear(X, W, activation="tanh")
    with pytest.raises(ValueError, match="kernel"):
        int8_linear(X, W, kernel="simt")
    with pytest.raises(TypeError, match="pair"):
        int8_linear(_rows(4, 32), W.q)
    with pytest.raises(ValueError, match="16 bytes"):
        int8_linear(_rows(4, 24), _rows(16, 24))
    with pytest.raises(ValueError, match="scale per row"):
        int8_linear((torch.zeros(4, 32, dtype=torch.int8), torch.ones(3)), W)
    with pytest.raises(ValueError, match="int8 rows"):
        int8_linear((torch.zeros(4, 32, dtype=torch.uint8), torch.ones(4)), W)
    with pytest.raises(ValueError, match="hidden width"):
        int8_gated_ffn(X, W, None, W, None, _rows(32, 32), None)
    with pytest.raises(ValueError, match="2-D"):
        quantize_weight(torch.zeros(3))


def test_int8_rows_pads_only_where_needed():
    q, s = torch.arange(48, dtype=torch.int8).reshape(3, 16), torch.ones(3)
    assert int8_rows(q, s).q.data_ptr() == q.data_ptr() or q.data_ptr() % 16
    odd = torch.arange(21, dtype=torch.int8).reshape(3, 7)
    r = int8_rows(odd, s)
    assert r.q.stride(0) == 16 and torch.equal(r.q, odd)
    t = int8_rows(odd.t(), torch.ones(7))
    assert torch.equal(t.q, odd.t()) and t.q.stride(1) == 1
    assert torch.equal(t.dequantize(), odd.t().float())
    with pytest.raises(ValueError, match="int8"):
        int8_rows(odd.float(), s)
    with pytest.raises(ValueError, match="scale per row"):
        int8_rows(odd, torch.ones(2))


def test_oracle_rounds_halves_to_even():
    # 127 x / 127 = x: halves stay halves.
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 126.5]])
    q, s = int8_oracle.quantize(x)
    assert q.tolist() == [[127, 0, 2, 2, 0, -2, 126]] and s.item() == 1.0
    q, s = int8_oracle.quantize(torch.tensor([[1.0, float("inf")], [0.0, 0.0]]))
    assert torch.isnan(s[0]) and q[0].tolist() == [0, 0] and s[1] > 0
    assert ctypes.c_float(s[1].item()).value == s[1].item()

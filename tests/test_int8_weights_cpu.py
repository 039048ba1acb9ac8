"""8-bit weights of any pitch and alignment: what is refused, and what is not (CPU)."""
import pytest
import torch

from deepx_op_gpukernelcompiler_b200 import (_build, _native as nat, int8_gated_ffn,
                                             int8_gated_linear, int8_linear)

FAKE = 0x1000  # never dereferenced: validation fails first


@pytest.fixture(scope="module")
def lib():
    _build.build()
    return nat.load()


def _weight(n, k):
    return torch.zeros(n, k, dtype=torch.int8), torch.ones(n)


@pytest.mark.parametrize("K", [24, 1000, 2056, 7])
def test_contiguous_weights_are_taken(K):
    """Only the device is refused here, not the rows' layout."""
    X = torch.zeros(4, K, dtype=torch.bfloat16)
    w, wo = _weight(16, K), _weight(K, 16)
    with pytest.raises(ValueError, match="CUDA"):
        int8_linear(X, w)
    with pytest.raises(ValueError, match="CUDA"):
        int8_gated_linear(X, w, w)
    with pytest.raises(ValueError, match="CUDA"):
        int8_gated_ffn(X, w, None, w, None, wo, None)
    with pytest.raises(ValueError, match="CUDA"):
        int8_linear(X, (w[0][3:, :], w[1][3:]))


def test_weights_that_are_still_refused():
    X = torch.zeros(4, 24, dtype=torch.bfloat16)
    q, s = _weight(24, 16)
    with pytest.raises(ValueError, match="unit stride"):
        int8_linear(X, (q.t(), torch.ones(16)))
    with pytest.raises(ValueError, match="overlap"):
        int8_linear(X, (q[:1, :1].as_strided((16, 24), (4, 1)), torch.ones(16)))
    with pytest.raises(ValueError, match="columns"):
        int8_linear(X, (q, s))
    with pytest.raises(ValueError, match="16 bytes"):  # activations are laid out beforehand
        int8_linear((torch.zeros(4, 24, dtype=torch.int8), torch.ones(4)), _weight(16, 24))


@pytest.mark.parametrize("args,code,needle", [
    ((FAKE, FAKE, -1, 8, 8, 16), nat.DX_ERR_INVALID_ARGUMENT, "negative"),
    ((FAKE, FAKE, 2, 1 << 30, 1 << 30, 1 << 30), nat.DX_ERR_UNSUPPORTED, "2^30"),
    ((None, FAKE, 2, 8, 8, 16), nat.DX_ERR_INVALID_ARGUMENT, "NULL"),
    ((FAKE, None, 2, 8, 8, 16), nat.DX_ERR_INVALID_ARGUMENT, "NULL"),
    ((FAKE, FAKE, 2, 8, 7, 16), nat.DX_ERR_INVALID_ARGUMENT, "ld_src"),
    ((FAKE, FAKE, 2, 17, 17, 16), nat.DX_ERR_INVALID_ARGUMENT, "ld_dst"),
    ((FAKE, FAKE + 8, 2, 8, 8, 16), nat.DX_ERR_INVALID_ARGUMENT, "16-byte"),
    ((FAKE, FAKE, 2, 8, 8, 24), nat.DX_ERR_INVALID_ARGUMENT, "16-byte"),
])
def test_pack_rows_host_validation(lib, args, code, needle):
    assert lib.dx_pack_int8_rows(*args, None) == code
    assert needle in nat.last_error()


def test_pack_nothing(lib):
    assert lib.dx_pack_int8_rows(None, None, 0, 8, 8, 16, None) == nat.DX_OK
    assert lib.dx_pack_int8_rows(None, None, 8, 0, 0, 16, None) == nat.DX_OK

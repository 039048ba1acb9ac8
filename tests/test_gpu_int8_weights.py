"""8-bit weights whose rows do not start on 16 bytes (gpu).

The products of such a weight are those of its padded copy, bit for bit: the sums
are integers."""
import pytest
import torch

import int8_oracle as ref
from deepx_op_gpukernelcompiler_b200 import _native as nat
from deepx_op_gpukernelcompiler_b200 import (int8_gated_ffn, int8_gated_linear, int8_linear,
                                             int8_rows, quantize_rows)

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _weight(N, K, seed):
    g = _gen(seed)
    q = torch.randint(-128, 128, (N, K), generator=g, device=DEV, dtype=torch.int8)
    return q, (torch.rand(N, generator=g, device=DEV) + 0.5) / (73 * K ** 0.5)


def _x(M, K, seed, dtype=torch.bfloat16):
    return torch.randn(M, K, generator=_gen(seed), device=DEV).to(dtype)


def _pack(src, ld, rows, K, dst):
    rc = nat.load().dx_pack_int8_rows(src.data_ptr(), dst.data_ptr(), rows, K, ld, dst.stride(0),
                                      torch.cuda.current_stream().cuda_stream)
    nat.check("dx_pack_int8_rows", rc)


@pytest.mark.parametrize("rows,K", [(1, 1), (1, 16), (3, 15), (1, 100), (5, 17), (200, 33),
                                    (30001, 31), (7, 16384), (3, 20001), (2, 131071)])
def test_pack_rows(rows, K):
    pieces = -(-K // 16) * 16
    for skew, gap in ((0, 0), (1, 0), (7, 5), (12, 4), (15, 17)):
        ld = K + gap
        buf = torch.randint(-128, 128, (skew + rows * ld,), generator=_gen(K), device=DEV,
                            dtype=torch.int8)
        src = buf[skew:]  # ends where its buffer does, when there is no gap
        dst = torch.full((rows + 1, pieces + 16), 99, dtype=torch.int8, device=DEV)
        _pack(src, ld, rows, K, dst)
        assert torch.equal(dst[:rows, :K], src.as_strided((rows, K), (ld, 1)))
        assert (dst[:rows, pieces:] == 99).all() and (dst[rows] == 99).all()


@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 7, 40), (2, 4099, 130), (16, 1000, 777),
                                   (77, 2056, 264), (129, 33, 5001), (333, 1000, 2049)])
def test_products_of_contiguous_weights(M, K, N):
    X, b = _x(M, K, M), _x(1, N, 5)[0]
    R = _x(M, N, 6)
    w, w2 = _weight(N, K, 1), _weight(N, K, 2)
    p, p2 = int8_rows(*w), int8_rows(*w2)
    assert w[0].is_contiguous() and (N == 1 or p.q.stride(0) % 16 == 0)
    for kern in ("auto", "decode", "umma"):
        Y = int8_linear(X, w, b, "silu", residual=R, kernel=kern)
        assert torch.equal(Y, int8_linear(X, p, b, "silu", residual=R, kernel=kern)), kern
        ref.check(Y, ref.linear(X, w, b, "silu", R), kern)
        Y = int8_gated_linear(X, w, w2, b, kernel=kern)
        assert torch.equal(Y, int8_gated_linear(X, p, p2, b, kernel=kern)), kern
        ref.check(Y, ref.gated(X, w, w2, b), kern)
    rows = quantize_rows(X)  # an 8-bit X beside such a weight
    assert torch.equal(int8_linear(rows, w, b), int8_linear(rows, p, b))
    assert nat.device_status(torch.cuda.current_stream().cuda_stream) == 0


def test_views_of_weights():
    """Rows of a larger matrix: from any row and column on, each at its own pitch."""
    X = _x(9, 96, 1)
    q, s = _weight(301, 131, 2)
    for r0, c0 in ((0, 0), (1, 0), (0, 16), (3, 5), (100, 35)):
        w = (q[r0:r0 + 200, c0:c0 + 96], s[r0:r0 + 200].contiguous())
        assert torch.equal(int8_linear(X, w), int8_linear(X, int8_rows(*w))), (r0, c0)
    w = (q.reshape(-1)[1:1 + 64 * 96].reshape(64, 96), s[:64].contiguous())
    assert w[0].data_ptr() % 16 and w[0].stride(0) % 16 == 0
    assert torch.equal(int8_linear(X, w), int8_linear(X, int8_rows(*w)))
    one = (q[7:8, 3:99], s[7:8].contiguous())
    assert torch.equal(int8_linear(X, one), int8_linear(X, int8_rows(*one)))
    none = (q[:0, :96], s[:0])
    assert int8_linear(X, none).shape == (9, 0)


def test_chain_graphs_and_weights_written_before_the_call():
    """The gated FFN on contiguous weights of odd width, captured twice on one stream
    and replayed at once on two, with weights that change between replays."""
    D, H = 200, 519
    wg, wu, wo = _weight(H, D, 1), _weight(H, D, 2), _weight(D, H, 3)
    xs = [_x(4, D, 7), _x(150, D, 8)]
    graphs, outs = [], []
    int8_gated_ffn(xs[0], wg, None, wu, None, wo, None)
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(int8_gated_ffn(x, wg, None, wu, None, wo, None, residual=x))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for step in range(4):
        for w in (wg, wu, wo):
            w[0].copy_(w[0].roll(step, 0))
        want = [int8_gated_ffn(x, int8_rows(*wg), None, int8_rows(*wu), None, int8_rows(*wo), None,
                               residual=x) for x in xs]
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), step
        # and eagerly, right behind the launch that writes a weight
        wg[0].copy_(wg[0].flip(1))
        got = int8_gated_linear(xs[0], wg, wu)
        assert torch.equal(got, int8_gated_linear(xs[0], int8_rows(*wg), int8_rows(*wu)))

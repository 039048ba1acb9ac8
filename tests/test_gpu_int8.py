"""8-bit linear layers on the GPU against their definition in 64 bits (gpu).

The quantised integers and scales have to be equal; the products keep the
tolerance derived in int8_oracle.py."""
import pytest
import torch

import int8_oracle as ref
from deepx_op_gpukernelcompiler_b200 import _native as nat
from deepx_op_gpukernelcompiler_b200 import (Int8Rows, int8_gated_ffn, int8_gated_linear,
                                             int8_linear, int8_rows, quantize_rows,
                                             quantize_weight)

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _x(M, K, dtype, seed, pitch=None):
    g = _gen(seed)
    x = torch.randn(M, K, generator=g, device=DEV) * torch.exp(
        0.7 * torch.randn(K, generator=g, device=DEV))
    if pitch is None:
        return x.to(dtype)
    buf = torch.full((M, pitch), 7.0, dtype=dtype, device=DEV)
    buf[:, :K] = x.to(dtype)
    return buf[:, :K]


def _w(N, K, seed):
    g = _gen(seed)
    q = torch.randint(-127, 128, (N, K), generator=g, device=DEV, dtype=torch.int8)
    s = (torch.rand(N, generator=g, device=DEV) + 0.5) / (73 * K ** 0.5)
    return int8_rows(q, s)


def _vec(N, dtype, seed):
    return torch.randn(N, generator=_gen(seed), device=DEV).to(dtype)


# ------------------------------------------------------------ quantisation
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 4096), (3, 7), (5, 1000), (33, 1029), (700, 513),
                                 (2, 40000), (0, 64)])
def test_quantize_rows(M, K, dtype):
    X = _x(M, K, DT[dtype], 100 * M + K)
    if M > 2:
        X[1] = 0  # a row of zeros
        X[2] *= 2.0 ** -12
    r = quantize_rows(X)
    q, s = ref.quantize(X)
    assert torch.equal(r.q.cpu(), q) and torch.equal(r.scale.cpu(), s)
    assert r.q.stride(0) % 16 == 0 or M <= 1


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_quantize_halves_extremes_and_nonfinite(dtype):
    dt = DT[dtype]
    big = torch.finfo(dt).max
    tiny = torch.finfo(dt).smallest_normal
    rows = [[127.0] + [k / 2 for k in range(-200, 200)],       # halves, both signs
            [63.5] + [k / 4 for k in range(-200, 200)],        # the same halves at another scale
            [big, -big] + [big / 3] * 399,
            [tiny, -tiny / 2, tiny / 4] + [0.0] * 398,
            [0.0] * 401,
            [1.0, float("inf")] + [2.0] * 399,
            [float("nan")] + [1.0] * 400,
            [-float("inf")] * 401]
    X = torch.tensor(rows, dtype=torch.float64).to(dt).to(DEV)
    r = quantize_rows(X)
    q, s = ref.quantize(X)
    assert torch.equal(r.q.cpu(), q)
    assert torch.equal(torch.nan_to_num(r.scale.cpu(), nan=-1.0), torch.nan_to_num(s, nan=-1.0))


def test_quantize_strided_and_misaligned_rows():
    for dtype in DT.values():
        for off, pitch in ((0, 520), (1, 517), (3, 600)):
            base = _x(9, pitch, dtype, off)
            X = base[:, off:off + 500]
            r = quantize_rows(X)
            q, s = ref.quantize(X)
            assert torch.equal(r.q.cpu(), q) and torch.equal(r.scale.cpu(), s)


def test_quantize_weight_is_per_channel():
    W = _x(200, 72, torch.bfloat16, 5)
    r = quantize_weight(W)
    q, s = ref.quantize(W.t())
    assert torch.equal(r.q.cpu(), q) and torch.equal(r.scale.cpu(), s)
    assert (r.dequantize().cpu().t() - W.float().cpu()).abs().max() <= s.max() * 0.5001


def _plan(key):
    return int(nat.last_launch_plan().split(key + "=")[1].split()[0])


# ---------------------------------------------------------------- products
SHAPES = [  # M, K, N
    (1, 1, 1), (1, 128, 128), (1, 4096, 512), (2, 130, 77), (7, 1000, 300), (16, 4096, 1024),
    (17, 33, 129), (32, 2048, 256), (33, 700, 1001), (64, 512, 640), (65, 1024, 384),
    (128, 300, 515), (200, 1029, 260), (333, 1000, 521), (513, 256, 1048),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_linear(M, K, N, dtype):
    dt = DT[dtype]
    X, W, b, R = _x(M, K, dt, M + K), _w(N, K, N), _vec(N, dt, 3), _x(M, N, dt, 4)
    acts = [None, "relu", "gelu_tanh", "gelu_erf", "silu"]
    act = acts[(M + N) % 5]
    ref.check(int8_linear(X, W, b, act, residual=R), ref.linear(X, W, b, act, R), "dynamic")
    plain = int8_linear(X, W, kernel="decode")
    assert nat.last_launch_plan().startswith("int8_tile"), nat.last_launch_plan()
    ref.check(plain, ref.linear(X, W), "tile")
    pair = quantize_rows(X)
    ref.check(int8_linear(pair, W, b, act, dtype=dt), ref.linear(X, W, b, act), "8-bit X")
    Y = int8_linear(X, W, b, act, residual=R, kernel="umma")
    assert nat.last_launch_plan().startswith("int8_pair"), nat.last_launch_plan()
    assert _plan("tma_out") == (dtype != "f32" and N % 8 == 0)
    ref.check(Y, ref.linear(X, W, b, act, R), "pair")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_gated(M, K, N, dtype):
    dt = DT[dtype]
    X, Wg, Wu = _x(M, K, dt, M + K), _w(N, K, N), _w(N, K, N + 1)
    bg, bu = _vec(N, dt, 3), _vec(N, dt, 4)
    act = ["silu", None, "gelu_erf", "relu", "gelu_tanh"][(M + N) % 5]
    ref.check(int8_gated_linear(X, Wg, Wu, bg, bu, act), ref.gated(X, Wg, Wu, bg, bu, act), "auto")
    ref.check(int8_gated_linear(X, Wg, Wu, None, bu, act, kernel="decode"),
              ref.gated(X, Wg, Wu, None, bu, act), "tile")
    assert nat.last_launch_plan().startswith("int8_tile_gated"), nat.last_launch_plan()
    Y = int8_gated_linear(quantize_rows(X), Wg, Wu, bg, None, act, kernel="umma", dtype=dt)
    assert nat.last_launch_plan().startswith("int8_pair_gated"), nat.last_launch_plan()
    ref.check(Y, ref.gated(X, Wg, Wu, bg, None, act), "pair")


@pytest.mark.parametrize("M,K,N", [(600, 384, 2100), (1024, 520, 4096), (2048, 130, 2568),
                                   (1500, 96, 5003)])
def test_many_tiles(M, K, N):
    """More tiles than a wave of CTA pairs, and raster groups of several m-tiles."""
    X, W, W2 = _x(M, K, torch.bfloat16, 1), _w(N, K, 2), _w(N, K, 3)
    b = _vec(N, torch.bfloat16, 4)
    for kern in ("auto", "umma", "decode"):
        ref.check(int8_linear(X, W, b, "silu", kernel=kern), ref.linear(X, W, b, "silu"), kern)
        ref.check(int8_gated_linear(X, W, W2, b, kernel=kern), ref.gated(X, W, W2, b), kern)


@pytest.mark.parametrize("M,K,N", [(2560, 200, 2048), (4096, 128, 4040)])
def test_last_wave_in_halves(M, K, N):
    X, W, W2 = _x(M, K, torch.float16, 1), _w(N, K, 2), _w(N, K, 3)
    b, R = _vec(N, torch.float16, 4), _x(M, N, torch.float16, 5)
    ref.check(int8_linear(X, W, b, "relu", residual=R), ref.linear(X, W, b, "relu", R))
    assert _plan("full") < _plan("tiles"), nat.last_launch_plan()
    ref.check(int8_gated_linear(X, W, W2, b, None), ref.gated(X, W, W2, b, None))


@pytest.mark.parametrize("N", [28672, 28601, 20000, 37888])
def test_channels_per_tile_evened_out(N):
    X, W = _x(9, 256, torch.bfloat16, 1), _w(N, 256, 2)
    ref.check(int8_linear(X, W, None, "gelu_erf"), ref.linear(X, W, None, "gelu_erf"))
    ref.check(int8_gated_linear(X, Int8Rows(W.q[:N // 2], W.scale[:N // 2]),
                                int8_rows(W.q[N - N // 2:], W.scale[N - N // 2:])),
              ref.gated(X, (W.q[:N // 2], W.scale[:N // 2]),
                        (W.q[N - N // 2:], W.scale[N - N // 2:])))


def test_extreme_integers_do_not_overflow():
    K = 131071
    q = torch.full((2, K), -128, dtype=torch.int8, device=DEV)
    one = torch.ones(2, device=DEV)
    Y = int8_linear(int8_rows(q, one), int8_rows(q, one), dtype=torch.float32)
    assert torch.equal(Y.cpu(), torch.full((2, 2), float(K * 128 * 128)))
    with pytest.raises(nat.NativeError, match="overflow"):
        wide = torch.zeros((1, K + 1), dtype=torch.int8, device=DEV)
        int8_linear(int8_rows(wide, one[:1]), int8_rows(wide, one[:1]))


def test_nonfinite_rows_stay_in_their_rows():
    X, W = _x(20, 256, torch.bfloat16, 1), _w(136, 256, 2)
    clean = int8_linear(X, W, activation="relu")
    X2 = X.clone()
    X2[3, 7], X2[11, 200] = float("nan"), float("inf")
    for kern in ("decode", "umma"):
        Y = int8_linear(X2, W, activation="relu", kernel=kern)
        for m in (3, 11):
            assert torch.isnan(Y[m]).all()
        keep = [m for m in range(20) if m not in (3, 11)]
        assert torch.equal(Y[keep], clean[keep])


def test_strided_operands_outputs_and_untouched_rows():
    dt = torch.float16
    for M, K, N in ((5, 200, 136), (300, 200, 136)):
        X = _x(M, K, dt, 1, pitch=K + 8)
        W, b = _w(N, K, 2), _vec(N, dt, 3)
        for pitch in (N + 8, N + 3):
            buf = torch.full((M + 2, pitch), 9.0, dtype=dt, device=DEV)
            res = _x(M, N, dt, 6, pitch=pitch)
            Y = int8_linear(X, W, b, "gelu", residual=res, out=buf[:M, :N])
            assert Y.data_ptr() == buf.data_ptr()
            ref.check(Y, ref.linear(X, W, b, "gelu", res), f"pitch {pitch}")
            assert (buf[:, N:] == 9).all() and (buf[M:] == 9).all()
        inplace = _x(M, N, dt, 7)
        want = ref.linear(X, W, b, None, inplace)
        ref.check(int8_linear(X, W, b, residual=inplace, out=inplace), want, "in place")


def test_output_dtype_and_empty():
    X, W = _x(4, 64, torch.float32, 1), _w(24, 64, 2)
    for dt in DT.values():
        Y = int8_linear(X, W, dtype=dt)
        assert Y.dtype == dt
        ref.check(Y, ref.linear(X, W), str(dt))
    assert int8_linear(quantize_rows(X), W).dtype == torch.bfloat16
    assert int8_linear(X[:0], W).shape == (0, 24)
    empty = Int8Rows(W.q[:0], W.scale[:0])
    assert int8_linear(X, empty).shape == (4, 0)
    with pytest.raises(ValueError, match="differs from the output dtype"):
        int8_linear(X, W, bias=_vec(24, torch.float16, 1))
    with pytest.raises(ValueError, match="at least one column"):
        int8_linear(X[:, :0], Int8Rows(W.q[:, :0], W.scale))


def test_same_result_whatever_the_split_and_order():
    """Integer sums: every kernel, and a row alone or in a batch, gives the same bits."""
    X, W = _x(64, 4096, torch.bfloat16, 1), _w(512, 4096, 2)
    Y = int8_linear(X, W, activation="silu")
    assert torch.equal(Y, int8_linear(X, W, activation="silu", kernel="umma"))
    assert torch.equal(Y[:16], int8_linear(X[:16], W, activation="silu"))
    assert torch.equal(Y[5:6], int8_linear(X[5:6], W, activation="silu"))


def test_gated_ffn_chain_and_sharing_one_quantisation():
    """The layers as a model runs them: q/k/v-like projections of one quantised
    input, then the gated FFN on the sum, added to the residual stream."""
    dt = torch.bfloat16
    for M in (1, 24, 300):
        D, H = 264, 1000
        X = _x(M, D, dt, M)
        Wp, Wg, Wu, Wo = _w(D, D, 1), _w(H, D, 2), _w(H, D, 3), _w(D, H, 4)
        bg, bo = _vec(H, dt, 5), _vec(D, dt, 6)
        rows = quantize_rows(X)
        a, c = int8_linear(rows, Wp), int8_linear(rows, Wp, activation="relu")
        ref.check(a, ref.linear(X, Wp), "first")
        ref.check(c, ref.linear(X, Wp, None, "relu"), "second")
        h = torch.empty(M, H, dtype=dt, device=DEV)
        y = int8_gated_ffn(a, Wg, bg, Wu, None, Wo, bo, residual=X, hidden=h)
        ref.check(h, ref.gated(a, Wg, Wu, bg, None), "hidden")
        ref.check(y, ref.linear(h, Wo, bo, None, X), "chain")


def test_other_stream_and_graphs_sharing_nothing():
    """Two graphs captured on one stream, replayed at once on two: each has its own workspace."""
    X1, X2 = _x(8, 2048, torch.float16, 1), _x(300, 2048, torch.float16, 2)
    W = _w(1024, 2048, 3)
    want1, want2 = int8_linear(X1, W, activation="silu"), int8_linear(X2, W, activation="silu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = int8_linear(X1, W, activation="silu")
    side.synchronize()
    assert torch.equal(got, want1)
    graphs, outs = [], []
    for X in (X1, X2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(int8_linear(X, W, activation="silu"))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want1) and torch.equal(outs[1], want2)
    assert nat.device_status(torch.cuda.current_stream().cuda_stream) == 0


def test_product_reads_what_the_launch_before_it_wrote():
    """W, X, bias and residual written by the preceding kernels of the stream."""
    W = _w(512, 1024, 3)
    X = torch.zeros(4, 1024, dtype=torch.float16, device=DEV)
    new = _x(4, 1024, torch.float16, 9)
    q2 = torch.randint(-127, 128, tuple(W.q.shape), generator=_gen(8), device=DEV, dtype=torch.int8)
    for i in range(8):
        X.copy_(new * (i + 1))
        W.q.copy_(torch.roll(q2, i, 0))
        Y = int8_linear(X, W)
        ref.check(Y, ref.linear(X, W), f"step {i}")
        rows = quantize_rows(X)
        W.q.copy_(torch.roll(q2, -i - 1, 0))
        Y = int8_linear(rows, W, dtype=torch.float16)
        ref.check(Y, ref.linear(X, W), f"step {i}, 8-bit X")

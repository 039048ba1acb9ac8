"""The mixture-of-experts layer on the GPU against its definition in 64 bits (gpu).

Tolerances: moe_oracle.py."""
import pytest
import torch

import moe_oracle as ref
from deepx_op_gpukernelcompiler_b200 import (int8_gated_ffn, moe_ffn, quantize_rows,
                                             quantize_weight)
from deepx_op_gpukernelcompiler_b200 import _native as nat

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def make(T, D, H, E, dtype, seed=0, bias=False, residual=False):
    g = torch.Generator(device=DEV).manual_seed(seed + 7 * T + D + H + E)

    def n(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)

    t = {"X": n(T, D), "Wr": n(D, E, std=D ** -0.5), "Wg": n(E, D, H, std=D ** -0.5),
         "Wu": n(E, D, H, std=D ** -0.5), "Wo": n(E, H, D, std=H ** -0.5)}
    if bias:
        t |= {"br": n(E, std=0.3), "bg": n(E, H, std=0.3), "bu": n(E, H, std=0.3), "bo": n(E, D)}
    if residual:
        t["residual"] = n(T, D)
    return t


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("T,D,H,E,k", [
    (1, 8, 8, 1, 1), (1, 64, 128, 4, 2), (1, 512, 256, 8, 2), (2, 72, 40, 3, 3),
    (3, 264, 1000, 5, 2), (5, 1024, 136, 33, 7), (8, 512, 512, 16, 4), (9, 256, 128, 64, 8),
    (16, 136, 264, 20, 6), (17, 1032, 200, 6, 2), (31, 320, 128, 40, 5), (33, 512, 384, 8, 2),
    (64, 256, 256, 16, 4), (64, 128, 72, 256, 8), (64, 96, 64, 4, 1), (7, 2048, 512, 8, 2),
    (4, 8, 4096, 2, 1), (4, 4096, 8, 2, 1), (1, 48, 16, 32, 32),
])
def test_layer(T, D, H, E, k, dtype):
    t = make(T, D, H, E, DT[dtype], bias=(T + E) % 2 == 0, residual=T % 3 != 0)
    act = ["silu", "gelu", "gelu_erf", "relu", None][(T + D // 8) % 5]
    renorm = T % 4 != 1
    got = moe_ffn(**t, top_k=k, activation=act, renormalize=renorm, return_routing=True)
    assert nat.last_launch_plan().startswith("moe "), nat.last_launch_plan()
    ref.check(got, ref.moe(**t, top_k=k, activation=act, renormalize=renorm))
    assert nat.device_status(torch.cuda.current_stream().cuda_stream) == 0


def test_skewed_routing_and_ties():
    """Every token to the same experts; experts with equal logits: the lowest numbers."""
    t = make(40, 128, 256, 12, torch.bfloat16)
    t["Wr"].zero_()
    got = moe_ffn(**t, top_k=3, return_routing=True)
    assert (got[2] == torch.arange(3, device=DEV, dtype=torch.int32)).all()
    ref.check(got, ref.moe(**t, top_k=3))
    t["br"] = torch.zeros(12, dtype=torch.bfloat16, device=DEV)
    t["br"][[11, 4]] = 1.0
    got = moe_ffn(**t, top_k=3, return_routing=True)
    assert (got[2] == torch.tensor([4, 11, 0], device=DEV, dtype=torch.int32)).all()
    ref.check(got, ref.moe(**t, top_k=3))


def test_one_token_one_expert_each():
    t = make(16, 64, 64, 16, torch.float16)
    t["Wr"].zero_()
    t["X"][:, :16] = torch.eye(16, device=DEV, dtype=torch.float16)
    t["X"][:, 16:] *= 0.5
    t["Wr"][:16] = 4 * torch.eye(16, device=DEV, dtype=torch.float16).flip(0)
    got = moe_ffn(**t, top_k=1, return_routing=True)
    assert (got[2][:, 0].cpu() == torch.arange(15, -1, -1)).all()
    ref.check(got, ref.moe(**t, top_k=1))


def test_masked_experts_and_nonfinite_weights_stay_where_they_were_chosen():
    t = make(12, 128, 192, 6, torch.bfloat16)
    t["br"] = torch.zeros(6, dtype=torch.bfloat16, device=DEV)
    t["br"][2] = float("-inf")  # an expert that is switched off
    for name in ("Wg", "Wu", "Wo"):
        t[name][2] = float("nan")
    got = moe_ffn(**t, top_k=2, return_routing=True)
    assert not (got[2] == 2).any() and torch.isfinite(got[0]).all()
    clean = {k: v.clone() for k, v in t.items()}
    for name in ("Wg", "Wu", "Wo"):
        clean[name][2] = 0
    ref.check(got, ref.moe(**clean, top_k=2))
    # an expert with infinite weights: exactly the tokens that chose it are touched
    e = int(got[2][0, 0])
    t["Wo"][e] = float("inf")
    y = moe_ffn(**t, top_k=2)
    chose = (got[2] == e).any(1)
    assert not torch.isfinite(y[chose]).any()
    assert torch.equal(y[~chose], got[0][~chose])
    # a token with a NaN: its row alone
    t["Wo"][e] = clean["Wo"][e]
    t["X"][5, 3] = float("nan")
    y, w, ids = moe_ffn(**t, top_k=2, return_routing=True)
    assert torch.isnan(y[5]).all()
    keep = [m for m in range(12) if m != 5]
    assert torch.equal(y[keep], got[0][keep]) and torch.equal(ids[keep], got[2][keep])
    assert ((ids >= 0) & (ids < 6)).all()


def test_a_token_alone_or_in_a_batch_and_repeats_give_the_same_bits():
    t = make(24, 512, 640, 8, torch.bfloat16)
    y = moe_ffn(**t, top_k=2)
    for _ in range(5):
        assert torch.equal(moe_ffn(**t, top_k=2), y)


def test_strided_operands_untouched_rows_and_in_place():
    dt = torch.float16
    t = make(6, 136, 72, 5, dt, bias=True)
    want = ref.moe(**t, top_k=2)
    pad = {}
    for name in ("Wg", "Wu", "Wo"):
        E, R, C = t[name].shape
        buf = torch.full((E, R + 3, C + 8), float("nan"), dtype=dt, device=DEV)
        buf[:, :R, :C] = t[name]
        pad[name] = buf[:, :R, :C]
    wr = torch.full((136, 9), float("nan"), dtype=dt, device=DEV)
    wr[:, :5] = t["Wr"]
    for pitch in (144, 137):
        xb = torch.full((6, pitch), float("nan"), dtype=dt, device=DEV)
        xb[:, :136] = t["X"]
        ob = torch.full((8, pitch), 9.0, dtype=dt, device=DEV)
        args = t | pad | {"Wr": wr[:, :5], "X": xb[:, :136]}
        got = moe_ffn(**args, top_k=2, out=ob[:6, :136], return_routing=True)
        ref.check(got, want, f"pitch {pitch}")
        assert (ob[6:] == 9).all() and (ob[:, 136:] == 9).all()
    x = t["X"].clone()  # residual and output in X's place
    got = moe_ffn(**(t | {"X": x}), top_k=2, residual=x, out=x, return_routing=True)
    ref.check(got, ref.moe(**t, top_k=2, residual=t["X"]), "in place")


@pytest.mark.parametrize("T,D,H,E,k", [(3, 40072, 72, 3, 2), (2, 136, 20000, 3, 2)])
def test_whole_waves_of_tiles_in_either_phase(T, D, H, E, k):
    """More 256-column tiles of the output, or 128-column tiles of h, than SMs."""
    t = make(T, D, H, E, torch.bfloat16, bias=True, residual=True)
    got = moe_ffn(**t, top_k=k, return_routing=True)
    ref.check(got, ref.moe(**t, top_k=k))


@pytest.mark.parametrize("D,E", [(1024, 64), (1032, 64), (256, 200), (264, 200), (4096, 64)])
def test_routers_of_512_and_of_1024_threads(D, E):
    """The last width that 512 threads read in one step, the first that they do not, and
    one that takes 1024 threads two."""
    t = make(9, D, 40, E, torch.float16, bias=True)
    got = moe_ffn(**t, top_k=5, return_routing=True)
    ref.check(got, ref.moe(**t, top_k=5))


def test_one_expert_given_by_a_view():
    """E = 1: the expert pitch of a view plays no part."""
    t = make(3, 64, 40, 1, torch.bfloat16)
    for name in ("Wg", "Wu", "Wo"):
        t[name] = t[name][0].as_strided((1, *t[name].shape[1:]), (0, t[name].shape[2], 1))
    got = moe_ffn(**t, top_k=1, return_routing=True)
    ref.check(got, ref.moe(**t, top_k=1))


def test_empty_batch():
    t = make(1, 64, 64, 4, torch.bfloat16)
    t["X"] = t["X"][:0]
    y, w, ids = moe_ffn(**t, top_k=2, return_routing=True)
    assert y.shape == (0, 64) and w.shape == ids.shape == (0, 2)


def test_streams_graphs_and_calls_at_once():
    """Two layers at once on two streams, eager and as graphs captured on one stream."""
    a = make(8, 1024, 512, 16, torch.bfloat16, seed=1)
    b = make(64, 512, 256, 8, torch.float16, seed=2)
    want = [moe_ffn(**a, top_k=4), moe_ffn(**b, top_k=2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (t, k) in enumerate(((a, 4), (b, 2))):
            with torch.cuda.stream(streams[i]):
                got[i].append(moe_ffn(**t, top_k=k))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])
    graphs, outs = [], []
    for t, k in ((a, 4), (b, 2)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(moe_ffn(**t, top_k=k))
        graphs.append(g)
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    # new inputs in the captured buffers
    a["X"].copy_(a["X"].flip(0))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0].flip(0))
    assert nat.device_status(torch.cuda.current_stream().cuda_stream) == 0


def test_block_of_shared_and_routed_experts():
    """The FFN half of a block as it is served: an 8-bit shared expert on the tokens,
    added to the residual stream, and the routed experts on top."""
    dt = torch.bfloat16
    for T in (1, 20):
        D, H = 256, 384
        t = make(T, D, 128, 8, dt, bias=True)
        g = torch.Generator(device=DEV).manual_seed(T)
        ws = [quantize_weight((torch.randn(s, generator=g, device=DEV) / s[0] ** 0.5).to(dt))
              for s in ((D, H), (D, H), (H, D))]
        stream = (torch.randn(T, D, generator=g, device=DEV)).to(dt)
        shared = int8_gated_ffn(quantize_rows(t["X"]), ws[0], None, ws[1], None, ws[2], None,
                                residual=stream)
        got = moe_ffn(**t, top_k=2, residual=shared, return_routing=True)
        ref.check(got, ref.moe(**t, top_k=2, residual=shared), f"T={T}")

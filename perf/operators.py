"""Measured cases of the 8-bit linear layers and the mixture-of-experts layer.

``int8_linear`` and ``int8_gated_linear`` are the fused linear and the gated
dual GEMM with 8-bit integer operands (one scale per token and per channel);
``moe_ffn`` is a whole mixture-of-experts layer for a serving step's tokens.
A case names its operator, sizes, type and epilogue.  With ``own`` false each
is computed in elementary torch operations, with ``own`` true through this
package.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LIMIT = 2.0 ** -100  # a row is scaled as if its largest magnitude were at least this
EMAX = 30e8  # bytes of expert weights of the largest mixture-of-experts case


def listed():
    return [
        # One token through a square projection: latency, 16 MB of weights.
        _linear("linear_1x4096x4096_f16", 1, 4096, 4096, "f16", None, False, True),
        # A small decode batch through a wide up-projection: the weights' stream.
        _linear("linear_16x8192x28672_f16", 16, 8192, 28672, "f16", "gelu_erf", True, False),
        # Ragged sizes: rows that no tile, vector or descriptor divides.
        _linear("linear_333x1000x2049_f16", 333, 1000, 2049, "f16", "relu", True, False),
        # A square prefill projection.
        _linear("linear_4096x4096x4096_bf16", 4096, 4096, 4096, "bf16", "gelu_tanh", True, False),
        # The FFN's down-projection over a long prefill, added to the stream of hidden states.
        _linear("linear_8192x14336x4096_bf16", 8192, 14336, 4096, "bf16", None, True, True),
        # One token through the gate and up projections of a gated FFN.
        _gated("gated_1x4096x14336_bf16", 1, 4096, 14336, "bf16", "silu", False),
        # A batch of odd size, between the single-token and the prefill shapes.
        _gated("gated_77x2056x5464_f16", 77, 2056, 5464, "f16", "silu", True),
        # The gated FFN over a long prefill: the largest integer product.
        _gated("gated_8192x4096x14336_bf16", 8192, 4096, 14336, "bf16", "silu", True),
        # One token through few large experts: two of eight are read.
        _moe("moe_1_4096x14336_8_2_bf16", 1, 4096, 14336, 8, 2, "bf16", "silu", False, False),
        # A small batch through many small experts: most of them are read, one or two tokens each.
        _moe("moe_8_2048x1024_64_8_bf16", 8, 2048, 1024, 64, 8, "bf16", "silu", False, True),
        # An odd batch, sizes that end inside a tile, every bias.
        _moe("moe_33_1032x2824_16_4_f16", 33, 1032, 2824, 16, 4, "f16", "gelu_tanh", True, True),
        # The largest batch of the operator: every expert is read.
        _moe("moe_64_2048x1024_64_8_bf16", 64, 2048, 1024, 64, 8, "bf16", "silu", False, True),
    ]


def _linear(name, m, k, n, dtype, act, bias, residual):
    return {"name": name, "op": "linear", "M": m, "K": k, "N": n, "dtype": dtype, "act": act,
            "bias": bias, "residual": residual}


def _gated(name, m, k, n, dtype, act, bias):
    return {"name": name, "op": "gated", "M": m, "K": k, "N": n, "dtype": dtype, "act": act,
            "bias": bias, "residual": False}


def _moe(name, t, d, h, e, top, dtype, act, bias, residual):
    return {"name": name, "op": "moe", "T": t, "D": d, "H": h, "E": e, "top": top, "dtype": dtype,
            "act": act, "bias": bias, "residual": residual}


def _spread(rng, low, high, step=1):
    """A multiple of `step` in [low, high], even over its logarithm."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return min(high, max(low, step * round(v / step)))


def draw(rng):
    op = rng.choice(["linear", "gated", "moe"])
    act = rng.choice([None, "relu", "gelu_tanh", "gelu_erf", "silu"])
    bias, residual = rng.random() < 0.5, rng.random() < 0.5
    while True:
        if op == "moe":
            case = _moe("", _spread(rng, 1, 64), _spread(rng, 256, 4096, 8),
                        _spread(rng, 256, 14336, 8), _spread(rng, 2, 128), _spread(rng, 1, 8),
                        rng.choice(["f16", "bf16"]), act or "silu", bias, residual)
            pairs = case["T"] * case["top"]
            fits = (case["top"] <= case["E"] and 6 * case["E"] * case["D"] * case["H"] <= EMAX
                    and pairs * case["D"] * case["H"] <= 512 * 2048 * 1024)
        else:
            make = _linear if op == "linear" else _gated
            args = [_spread(rng, 1, 8192), _spread(rng, 64, 14336), _spread(rng, 64, 28672),
                    rng.choice(["f16", "bf16", "bf16", "f32"]), act, bias]
            case = make("", *args, residual) if op == "linear" else make("", *args)
            wide = 2 if op == "gated" else 1
            fits = wide * case["M"] * case["K"] * case["N"] <= 2 * 8192 * 4096 * 14336
        if fits:
            del case["name"]
            return case


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=gen, device=dev) * std).to(dt)

    def weight(n, k):
        # 8-bit weights as a checkpoint holds them: [channels, K] and a scale for each channel.
        q = torch.randn((n, k), generator=gen, device=dev).mul_(32).round_().clamp_(-127, 127)
        s = (torch.rand((n,), generator=gen, device=dev) + 0.5) / (32 * math.sqrt(k))
        return q.to(torch.int8), s

    if case["op"] == "moe":
        T, D, H, E = case["T"], case["D"], case["H"], case["E"]
        state = {"X": normal(T, D), "Wr": normal(D, E, std=D ** -0.5),
                 "Wg": normal(E, D, H, std=D ** -0.5), "Wu": normal(E, D, H, std=D ** -0.5),
                 "Wo": normal(E, H, D, std=H ** -0.5)}
        for name, size in (("br", (E,)), ("bg", (E, H)), ("bu", (E, H)), ("bo", (E, D))):
            state[name] = normal(*size, std=0.1) if case["bias"] else None
        state["residual"] = normal(T, D) if case["residual"] else None
        return {**state, "case": case}
    M, K, N = case["M"], case["K"], case["N"]
    # Hidden states: a few channels are several times as large as the rest.
    channel = torch.exp(0.7 * torch.randn((K,), generator=gen, device=dev))
    X = (torch.randn((M, K), generator=gen, device=dev) * channel).to(dt)
    state = {"case": case, "X": X, "W": weight(N, K), "bias": normal(N, std=0.1) if case["bias"] else None}
    if case["op"] == "gated":
        state["W2"] = weight(N, K)
        state["bias2"] = normal(N, std=0.1) if case["bias"] else None
    else:
        state["residual"] = normal(M, N) if case["residual"] else None
    return state


def run(state):
    case = state["case"]
    if own:
        import deepx_op_gpukernelcompiler_b200 as dx
        if case["op"] == "linear":
            return dx.int8_linear(state["X"], state["W"], state["bias"], case["act"],
                                  residual=state["residual"])
        if case["op"] == "gated":
            return dx.int8_gated_linear(state["X"], state["W"], state["W2"], state["bias"],
                                        state["bias2"], case["act"])
        return dx.moe_ffn(state["X"], state["Wr"], state["Wg"], state["Wu"], state["Wo"],
                          case["top"], br=state["br"], bg=state["bg"], bu=state["bu"],
                          bo=state["bo"], activation=case["act"], residual=state["residual"],
                          return_routing=True)
    if case["op"] == "moe":
        return _plain_moe(state, case)
    x = state["X"].double()  # in 64 bits: which integer is nearest is decided next to a border
    top = x.abs().amax(1, keepdim=True).clamp_min(LIMIT)
    q, scale = torch.round(x * 127 / top).float(), (top / 127).float()
    y = _plain_product(q, scale, state["W"], state["bias"])
    y = _plain_act(y, case["act"])
    if case["op"] == "gated":
        y = y * _plain_product(q, scale, state["W2"], state["bias2"])
    elif state["residual"] is not None:
        y = y + state["residual"].float()
    return y.to(state["X"].dtype)


def _plain_product(q, scale, weight, bias):
    y = (q @ weight[0].float().t()) * scale * weight[1]
    return y if bias is None else y + bias.float()


def _plain_act(y, act):
    if act == "relu":
        return torch.clamp_min(y, 0)
    if act == "silu":
        return y / (1 + torch.exp(-y))
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    if act == "gelu_erf":
        return 0.5 * y * torch.erfc(-y / math.sqrt(2))
    return y


def _plain_moe(state, case):
    X = state["X"]
    T, top = case["T"], case["top"]
    logits = X.double() @ state["Wr"].double()  # in 64 bits: the choice of experts is decided next to a border
    if state["br"] is not None:
        logits = logits + state["br"].double()
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :top]
    picked = torch.exp(torch.gather(logits, 1, order) - logits.amax(1, keepdim=True))
    weights = (picked / picked.sum(1, keepdim=True)).float()
    ids = order.reshape(-1)
    x = X.float().repeat_interleave(top, 0).unsqueeze(1)  # one row for each token and expert

    def product(rows, name, bias):
        y = torch.bmm(rows, state[name][ids].float())
        return y if state[bias] is None else y + state[bias][ids].float().unsqueeze(1)

    h = _plain_act(product(x, "Wg", "bg"), case["act"]) * product(x, "Wu", "bu")
    y = product(h, "Wo", "bo").reshape(T, top, -1)
    y = (y * weights.unsqueeze(2)).sum(1)
    if state["residual"] is not None:
        y = y + state["residual"].float()
    return y.to(X.dtype), weights, order.to(torch.int32)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "moe":
        T, D, H, E, top = (case[n] for n in ("T", "D", "H", "E", "top"))
        read = E * (1 - (1 - top / E) ** T)  # experts that some token goes to, on average
        bias = (E + read * (2 * H + D)) if case["bias"] else 0
        rows = T * D * (3 if case["residual"] else 2)
        return {"bytes": int(size * (read * 3 * D * H + D * E + rows + bias) + 8 * T * top),
                "flops": 6 * T * top * D * H + 2 * T * D * E}
    M, K, N = case["M"], case["K"], case["N"]
    wide = 2 if case["op"] == "gated" else 1
    rows = M * K + M * N * (2 if case["residual"] else 1) + (wide * N if case["bias"] else 0)
    return {"bytes": size * rows + wide * N * (K + 4), "flops": 2 * wide * M * K * N}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] != "moe":
        return _exact_int8(state, case)
    X = state["X"].double()
    logit = torch.matmul(X, state["Wr"].double())
    if state["br"] is not None:
        logit += state["br"].double()
    share = torch.softmax(logit, -1)
    y = state["residual"].double().clone() if state["residual"] is not None else torch.zeros_like(X)
    weights = torch.empty((case["T"], case["top"]), dtype=torch.float64, device=X.device)
    ids = torch.empty((case["T"], case["top"]), dtype=torch.int32, device=X.device)
    rows = share.tolist()
    for t in range(case["T"]):
        best = sorted(range(case["E"]), key=lambda e: (-rows[t][e], e))[:case["top"]]
        ids[t] = torch.tensor(best, dtype=torch.int32)
        weights[t] = share[t, best] / share[t, best].sum()
    for e in range(case["E"]):
        t, slot = torch.nonzero(ids == e, as_tuple=True)
        if not t.numel():
            continue
        gate, up = X[t] @ state["Wg"][e].double(), X[t] @ state["Wu"][e].double()
        if case["bias"]:
            gate, up = gate + state["bg"][e].double(), up + state["bu"][e].double()
        out = (_exact_act(gate, case["act"]) * up) @ state["Wo"][e].double()
        if case["bias"]:
            out = out + state["bo"][e].double()
        y[t] += weights[t, slot, None] * out
    return y, weights, ids


def _exact_act(v, act):
    f = torch.nn.functional
    return {None: lambda u: u, "relu": f.relu, "silu": f.silu,
            "gelu_tanh": lambda u: f.gelu(u, approximate="tanh"), "gelu_erf": f.gelu}[act](v)


def _exact_int8(state, case):
    X = state["X"].double()
    top = torch.maximum(X.abs().max(1).values, torch.full((), LIMIT, dtype=X.dtype, device=X.device))
    q = torch.round(torch.div(X.mul(127), top[:, None]))

    def product(weight, bias):
        v = torch.einsum("mk,nk->mn", q, weight[0].double())
        v = v * (top[:, None] * weight[1].double()[None, :] / 127)
        return v if bias is None else v + bias.double()[None, :]

    y = _exact_act(product(state["W"], state["bias"]), case["act"])
    if case["op"] == "gated":
        return y * product(state["W2"], state["bias2"])
    return y if state["residual"] is None else y + state["residual"].double()

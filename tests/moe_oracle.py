"""The mixture-of-experts layer from its definition, in 64 bits on the CPU.

Tolerance of an output y with u = eps / 2 of the working type:

    |got - y| <= u |y| + 2^-17 S + (fp16: 2^-24 sum_e w_e sum_n |Wo_e| + 2^-25)

S is the size of what was summed: sum_e w_e (sum_n |h_n| |Wo_n| + |bo|) + |r|,
each |h_n| bounded by |act'| G U with G, U the sums of magnitudes of its gate and up
products.  Per value: an fp32 accumulator of K terms is off by at most K 2^-24 of
the sum of magnitudes in the worst case; the tensor core adds in blocks and the
rounding errors do not all align, so 2^-18 (64 roundings) bounds K up to some
thousands; that enters once from each product.  h as hi + lo is off by u^2 |h| (bf16
2^-16: covered by S; fp16's lo is exact to 2^-25 absolute), weights by some 2^-21
(logits in fp32, expf).
"""
import torch

from int8_oracle import act64


def moe(X, Wr, Wg, Wu, Wo, top_k, br=None, bg=None, bu=None, bo=None, activation="silu",
        renormalize=True, residual=None):
    """-> (y, S, F, weights, ids); F is sum_e w_e sum_n |Wo_e| (for fp16's subnormals)."""
    def d(t):
        return None if t is None else t.detach().cpu().double()

    X, Wr, br, residual = d(X), d(Wr), d(br), d(residual)
    T, D = X.shape
    E = Wr.shape[1]
    logits = X @ Wr + (br if br is not None else 0)
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :top_k]
    p = torch.softmax(logits, 1)
    w = torch.gather(p, 1, order)
    if renormalize:
        w = w / w.sum(1, keepdim=True)
    y = residual.clone() if residual is not None else torch.zeros(T, D, dtype=torch.float64)
    size, floor = y.abs(), torch.zeros(T, D, dtype=torch.float64)
    for e in range(E):
        rows, slot = torch.nonzero(order == e, as_tuple=True)
        if not rows.numel():
            continue
        x, G, U, O = X[rows], d(Wg[e]), d(Wu[e]), d(Wo[e])
        g, u = x @ G, x @ U
        sg, su = x.abs() @ G.abs(), x.abs() @ U.abs()
        if bg is not None:
            g, sg = g + d(bg[e]), sg + d(bg[e]).abs()
        if bu is not None:
            u, su = u + d(bu[e]), su + d(bu[e]).abs()
        h = act64(g, activation) * u
        o, so = h @ O, (1.13 * sg * su) @ O.abs()
        if bo is not None:
            o, so = o + d(bo[e]), so + d(bo[e]).abs()
        ww = w[rows, slot][:, None]
        y.index_add_(0, rows, ww * o)
        size.index_add_(0, rows, ww * so)
        floor.index_add_(0, rows, ww * O.abs().sum(0, keepdim=True).expand(rows.numel(), D))
    return y, size, floor, w, order


def check(got, want, what=""):
    """got: (Y, weights, ids) of moe_ffn; want: moe()'s result."""
    Y, weights, ids = got
    y, size, floor, w, order = want
    assert torch.equal(ids.cpu().long(), order), f"{what}: other experts"
    # logits: fp32 sums; relative error of a weight = error of its logit
    assert (weights.cpu().double() - w).abs().max().item() <= 2.0 ** -18, what
    g = Y.detach().cpu().double()
    tol = torch.finfo(Y.dtype).eps / 2 * y.abs() + 2.0 ** -17 * size
    if Y.dtype == torch.float16:
        tol = tol + 2.0 ** -24 * floor + 2.0 ** -25
    bad = ~((g - y).abs() <= tol)
    if bad.any():
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; first at {i}: "
                             f"got {g[i].item()}, want {y[i].item()} +- {tol[i].item()}")
    # Far tighter on the whole: rounding to the output type dominates.
    off = (g - y).norm() / y.norm()
    assert off <= 0.6 * torch.finfo(Y.dtype).eps, f"{what}: {off.item()} off"

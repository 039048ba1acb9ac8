"""The 8-bit linear layers from their definition, in 64 bits on the CPU.

Tolerance of a product whose exact value is y, with S the size of what was
summed on the way (|s t sum| + |bias|, for the gated form the product of both
sides' sizes, plus |residual|):

    |got - y| <= u |y| + 2^-18 S + 2^-25

u = eps / 2 is the output type's rounding (2^-25 its half step among fp16's
subnormals).  Before it: the integer sum, the product of the scales and the
multiply-add round once each (3 * 2^-24 S), the activations' slope is below
1.13, and an activation is off by at most (|z| + 4) 2^-23 of its value, z <= 32
where that value is not itself below 2^-40 S: 2^-17.9 |y| at the very tail of
the range and below 2^-19 S wherever |z| < 12.
"""
import torch

LIMIT = 2.0 ** -100


def act64(v, act):
    f = torch.nn.functional
    if act in (None, "none"):
        return v
    if act == "relu":
        return f.relu(v)
    if act in ("silu", "swish"):
        return v * torch.sigmoid(v)
    if act in ("gelu", "gelu_tanh"):
        return f.gelu(v, approximate="tanh")
    return 0.5 * v * torch.special.erfc(-v / 2 ** 0.5)


def quantize(X):
    """(q int8, scale float32) of the rows of X, any floating type.

    127 x and the largest magnitude are exact in 64 bits and a quotient that is
    not a half lies further from one than the division rounds, so round() takes
    the nearest integer, halves to even."""
    x = X.detach().cpu().double()
    finite = torch.isfinite(x).all(1)
    x = torch.where(finite[:, None], x, torch.zeros_like(x))
    top = (x.abs().amax(1) if x.shape[1] else x.new_zeros(x.shape[0])).clamp_min(LIMIT)
    q = torch.round(127 * x / top[:, None]).to(torch.int8)
    scale = top.float() / torch.full_like(top, 127).float()
    return q, torch.where(finite, scale, torch.full_like(scale, float("nan")))


def _pre(q, scale, W, bias):
    wq, ws = (t.detach().cpu().double() for t in W)
    v = (q.double() @ wq.t()) * (scale.double()[:, None] * ws[None, :])
    size = v.abs()
    if bias is not None:
        b = bias.detach().cpu().double()
        v, size = v + b, size + b.abs()
    return v, size


def linear(X, W, bias=None, act=None, residual=None):
    """-> (y, S); X a float matrix or an (int8, scale) pair."""
    q, s = quantize(X) if isinstance(X, torch.Tensor) else (X[0].cpu(), X[1].cpu())
    v, size = _pre(q, s, W, bias)
    y = act64(v, act)
    if residual is not None:
        r = residual.detach().cpu().double()
        y, size = y + r, size + r.abs()
    return y, size


def gated(X, Wg, Wu, bg=None, bu=None, act="silu"):
    q, s = quantize(X) if isinstance(X, torch.Tensor) else (X[0].cpu(), X[1].cpu())
    g, sg = _pre(q, s, Wg, bg)
    u, su = _pre(q, s, Wu, bu)
    return act64(g, act) * u, sg * su


def check(got, want, what=""):
    y, size = want
    g = got.detach().cpu().double()
    assert g.shape == y.shape, (g.shape, y.shape)
    assert torch.equal(torch.isnan(g), torch.isnan(y)), f"{what}: NaN in other places"
    ok = ~torch.isnan(y)
    tol = torch.finfo(got.dtype).eps / 2 * y.abs() + 2.0 ** -18 * size + 2.0 ** -25
    bad = ok & ((g - y).abs() > tol)
    if bad.any():
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; first at {i}: "
                             f"got {g[i].item()}, want {y[i].item()} +- {tol[i].item()}")

"""8-bit linear layers: the fused linear and the gated dual GEMM on integers.

No reference counterpart; they stand beside ``fused_linear`` and
``fused_gated_linear`` (linear.py) for models whose weights are kept in 8 bits.
A matrix of 8-bit rows is an ``Int8Rows`` pair ``(q, scale)``: ``q`` int8 whose
rows start on 16 bytes, ``scale`` fp32 with one value per row, standing for
``q * scale[:, None]``.  Activations have a scale per token, weights one per
output channel and are held as [N, K]: the transpose of the 16-bit layers' W.

    quantize_rows(X)        X [M, K]            -> Int8Rows, one scale per token
    quantize_weight(W)      W [K, N]            -> Int8Rows [N, K], one per channel
    int8_rows(q, scale)     8-bit data at hand  -> Int8Rows (rows padded if needed)
    int8_linear             act(s_m t_n sum_k Xq Wq + bias) + residual
    int8_gated_linear       act(X Wg^T + bias_g) * (X Wu^T + bias_u)
    int8_gated_ffn          the gated FFN chain on both

X of a product is an Int8Rows pair or a floating-point matrix, which the call
quantises first (one launch of its own, whose end overlaps the product's first
loads of W).  A weight may be any pair of int8 rows and scales: rows that do not
start on 16 bytes are copied to rows that do by the call itself, in every call (one
launch, and N x K bytes of workspace); int8_rows does that once.  The sums are exact:
32-bit integers, rounded to fp32 once and to the output type once.  Inference only:
no gradients.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as nat
from .linear import DTYPE_CODES, _check_matrix, _ld, activation_code

# Kernel choices of the 8-bit products: CTA pairs, or one tile per CTA.
_KERNELS = {"auto": nat.DX_KERNEL_AUTO, "umma": nat.DX_KERNEL_UMMA, "decode": nat.DX_KERNEL_DECODE}


class Int8Rows(NamedTuple):
    """8-bit rows and their scales: the matrix ``q * scale[:, None]``."""

    q: torch.Tensor      # int8 [rows, K], rows starting on 16 bytes
    scale: torch.Tensor  # float32 [rows]

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        return (self.q.float() * self.scale[:, None]).to(dtype)


def _empty_rows(rows: int, K: int, device) -> torch.Tensor:
    pitch = -(-K // 16) * 16
    q = torch.empty((rows, pitch), dtype=torch.int8, device=device)
    return q if pitch == K else q[:, :K]


def quantize_rows(X: torch.Tensor) -> Int8Rows:
    """Each row of X [M, K] as 8-bit integers and a scale.

    With a = max(max |row|, 2^-100): scale = a / 127 and q = 127 x / a rounded
    to the nearest integer, halves to even, decided exactly.  A row that holds an
    infinity or a NaN gets the scale NaN, so that products with it are NaN."""
    if not isinstance(X, torch.Tensor):
        raise TypeError("X must be a torch tensor")
    if X.device.type != "cuda":
        raise ValueError("quantize_rows runs on CUDA tensors only (the engine has no CPU path)")
    if X.dtype not in DTYPE_CODES:
        raise ValueError(f"unsupported dtype {X.dtype}; expected float32, float16 or bfloat16")
    _check_matrix("X", X, None, None)
    M, K = X.shape
    q = _empty_rows(M, K, X.device)
    scale = X.new_empty(M, dtype=torch.float32)
    lib = nat.load()
    rc = _on_device(X.get_device(), lambda stream: lib.dx_quantize_rows(
        X.data_ptr(), q.data_ptr(), scale.data_ptr(), M, K, _ld(X), max(q.stride(0), K),
        DTYPE_CODES[X.dtype], stream))
    if rc:
        nat.check("dx_quantize_rows", rc)
    return Int8Rows(q, scale)


def quantize_weight(W: torch.Tensor) -> Int8Rows:
    """W [K, N] of a linear layer as Int8Rows [N, K], one scale per output channel."""
    _check_matrix("W", W, None, None)
    return quantize_rows(W.t().contiguous())


def int8_rows(q: torch.Tensor, scale: torch.Tensor) -> Int8Rows:
    """8-bit data at hand as Int8Rows; q is copied only where its rows do not
    start on 16 bytes."""
    if q.dtype != torch.int8 or scale.dtype != torch.float32:
        raise ValueError(f"q must be int8 and scale float32, got {q.dtype} and {scale.dtype}")
    if q.dim() != 2 or scale.shape != (q.shape[0],):
        raise ValueError(f"q must be [rows, K] with a scale per row, got {tuple(q.shape)} and "
                         f"{tuple(scale.shape)}")
    if (q.stride(1) != 1 or q.data_ptr() % 16
            or (q.shape[0] > 1 and (q.stride(0) % 16 or q.stride(0) < q.shape[1]))):
        padded = _empty_rows(q.shape[0], q.shape[1], q.device)
        padded.copy_(q)
        q = padded
    return Int8Rows(q, scale.contiguous())


def _pair(name: str, rows, K: int | None, n: int | None, any_rows: bool = False) -> tuple:
    """Checks an (int8 rows, scales) pair -> (q, scale, rows, K, pitch).  With
    `any_rows` its rows may start anywhere (_packed lays them out)."""
    if not isinstance(rows, tuple) or len(rows) != 2:
        raise TypeError(f"{name} must be a pair (int8 rows, float32 scales), see quantize_rows")
    q, scale = rows
    if q.dtype is not torch.int8 or scale.dtype is not torch.float32:
        raise ValueError(f"{name} must hold int8 rows and float32 scales, got {q.dtype} and "
                         f"{scale.dtype}")
    shape = q.shape
    if len(shape) != 2:
        raise ValueError(f"{name} must be 2-D, got shape {tuple(shape)}")
    rows_, cols = shape
    ld, unit = q.stride()
    if unit != 1 or ld < cols or (K is not None and cols != K) or (n is not None and rows_ != n):
        _check_matrix(name, q, n, K)  # raises, unless the stride of a lone row or column is odd
    if scale.shape != (rows_,) or (rows_ > 1 and scale.stride(0) != 1):
        raise ValueError(f"{name} needs one contiguous scale per row, got {tuple(scale.shape)}")
    if scale.get_device() != q.get_device():
        raise ValueError(f"{name}'s scales are on {scale.device}, its rows on {q.device}")
    if rows_ <= 1:
        ld = -(-cols // 16) * 16
    if not any_rows and (ld % 16 or q.data_ptr() % 16):
        raise ValueError(f"{name}'s rows must start on 16 bytes (pitch {ld}): int8_rows(q, scale) "
                         f"lays them out")
    return q, scale, rows_, cols, ld


def _packed(lib, q: torch.Tensor, rows: int, K: int, ld: int, stream) -> tuple:
    """Rows of a weight that start on 16 bytes -> (rows, address, pitch): its own, or
    a copy of this call's (to be kept until the product is launched)."""
    ptr = q.data_ptr()
    if not (ld % 16 or ptr % 16):
        return q, ptr, ld
    pitch = -(-K // 16) * 16
    space = q.new_empty(rows * pitch)
    rc = lib.dx_pack_int8_rows(ptr, space.data_ptr(), rows, K, max(ld, K), pitch, stream)
    if rc:
        nat.check("dx_pack_int8_rows", rc)
    return space, space.data_ptr(), pitch


def _float_or_pair(X, dtype):
    """X of a product -> (x, dtype code, scale, M, K, pitch, output dtype)."""
    if isinstance(X, torch.Tensor):
        x_dtype = X.dtype
        code = DTYPE_CODES.get(x_dtype)
        if code is None:
            raise ValueError(f"unsupported dtype {x_dtype}; expected float32, float16 or "
                             f"bfloat16, or a pair (int8 rows, scales)")
        shape = X.shape
        if len(shape) != 2:
            raise ValueError(f"X must be 2-D, got shape {tuple(shape)}")
        M, K = shape
        ld, unit = X.stride()
        if unit != 1 or ld < K:
            _check_matrix("X", X, None, None)
            ld = _ld(X)
        x, scale = X, None
        if dtype is None:
            dtype = x_dtype
    else:
        x, scale, M, K, ld = _pair("X", X, None, None)
        code = nat.DX_DTYPE_I8
        if dtype is None:
            dtype = torch.bfloat16
    if dtype not in DTYPE_CODES:
        raise ValueError(f"unsupported output dtype {dtype}; expected float32, float16 or "
                         f"bfloat16")
    if K < 1:
        raise ValueError("X must have at least one column")
    return x, code, scale, M, K, ld, dtype


def _kernel(kernel: str) -> int:
    code = _KERNELS.get(kernel)
    if code is None:
        raise ValueError(f"unknown kernel {kernel!r}; expected one of {list(_KERNELS)}")
    return code


def _same_device(x: torch.Tensor, index: int, *named) -> None:
    for name, t in named:
        if t.get_device() != index:
            raise ValueError(f"{name} is on {t.device}, X is on {x.device}")


def _output(name: str, out, x: torch.Tensor, M: int, N: int, dtype: torch.dtype):
    """-> (Y, its pitch)."""
    if not x.is_cuda:
        raise ValueError(f"{name} runs on CUDA tensors only (the engine has no CPU path)")
    if out is None:
        new = x.new_empty((M, N)) if x.dtype is dtype else x.new_empty((M, N), dtype=dtype)
        return new, max(N, 1)
    _check_matrix("out", out, M, N)
    _like("out", out, x, dtype)
    return out, _ld(out)


def _like(name: str, t: torch.Tensor, x: torch.Tensor, dtype: torch.dtype) -> None:
    if t.dtype is not dtype:
        raise ValueError(f"{name} dtype {t.dtype} differs from the output dtype {dtype}")
    if t.get_device() != x.get_device():
        raise ValueError(f"{name} is on {t.device}, X is on {x.device}")


def _vector(name: str, b: torch.Tensor | None, N: int, x: torch.Tensor, dtype: torch.dtype):
    """Checks a bias -> its address (None without one)."""
    if b is None:
        return None
    if b.shape != (N,) or not b.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor of shape ({N},)")
    _like(name, b, x, dtype)
    return b.data_ptr()


def _on_device(index: int, call):
    """call(stream) with device `index` current; `stream` is its current stream's handle."""
    # torch._C's own functions: building a Stream object takes 2 us a call.  Looked up
    # here, since a torch without CUDA does not have them.
    if index == torch._C._cuda_getDevice():
        return call(torch._C._cuda_getCurrentRawStream(index))
    with torch.cuda.device(index):
        return call(torch._C._cuda_getCurrentRawStream(index))


def int8_linear(X, W, bias: torch.Tensor | None = None, activation=None,
                residual: torch.Tensor | None = None, out: torch.Tensor | None = None,
                dtype: torch.dtype | None = None, kernel: str = "auto") -> torch.Tensor:
    """Y = act(X Wq^T + bias) + residual on 8-bit operands (dx_int8_linear).

    X: a floating-point matrix [M, K] (quantised here, a scale per token) or an
    Int8Rows pair.  W: a pair of int8 rows [N, K] and their scales (quantize_weight;
    rows that do not start on 16 bytes cost a copy in every call, see int8_rows).  Y
    has X's type, or `dtype` (bfloat16 by default where X is a pair); bias, residual
    and out have Y's."""
    act, kcode = activation_code(activation), _kernel(kernel)
    x, x_code, x_scale, M, K, ldx, dtype = _float_or_pair(X, dtype)
    wq, ws, N, _, ldw = _pair("W", W, K, None, True)
    out, ldy = _output("int8_linear", out, x, M, N, dtype)
    index = x.get_device()
    _same_device(x, index, ("W", wq))
    b_ptr = _vector("bias", bias, N, x, dtype)
    r_ptr, ldr = None, 0
    if residual is not None:
        _check_matrix("residual", residual, M, N)
        _like("residual", residual, x, dtype)
        r_ptr, ldr = residual.data_ptr(), _ld(residual)
    lib = nat.load()

    def call(stream):
        # The workspace is this call's alone, from the allocator of the current
        # stream or of the graph being captured: calls on other streams and other
        # graphs cannot share it, and it stays theirs until the launches are done.
        ws_ptr, ws_bytes, sx_ptr = None, 0, None
        if x_scale is not None:
            sx_ptr = x_scale.data_ptr()
        elif M:
            ws_bytes = lib.dx_int8_workspace_size(M, K)
            space = x.new_empty(ws_bytes, dtype=torch.uint8)
            ws_ptr = space.data_ptr()
        w_rows, w_ptr, w_ld = _packed(lib, wq, N, K, ldw, stream)
        return lib.dx_int8_linear(
            x.data_ptr(), x_code, sx_ptr, w_ptr, ws.data_ptr(), b_ptr, r_ptr,
            out.data_ptr(), M, N, K, ldx, w_ld, ldr, ldy, DTYPE_CODES[dtype], act, kcode, ws_ptr,
            ws_bytes, stream)

    rc = _on_device(index, call)
    if rc:
        nat.check("dx_int8_linear", rc)
    return out


def int8_gated_linear(X, Wg, Wu, bias_g: torch.Tensor | None = None,
                      bias_u: torch.Tensor | None = None, activation="silu",
                      out: torch.Tensor | None = None, dtype: torch.dtype | None = None,
                      kernel: str = "auto") -> torch.Tensor:
    """Y = act(X Wg^T + bias_g) * (X Wu^T + bias_u) on 8-bit operands, X read
    once for both weights (dx_int8_gated_linear).  Arguments as int8_linear."""
    act, kcode = activation_code(activation), _kernel(kernel)
    x, x_code, x_scale, M, K, ldx, dtype = _float_or_pair(X, dtype)
    gq, gs, N, _, ldg = _pair("Wg", Wg, K, None, True)
    uq, us, _, _, ldu = _pair("Wu", Wu, K, N, True)
    out, ldy = _output("int8_gated_linear", out, x, M, N, dtype)
    index = x.get_device()
    _same_device(x, index, ("Wg", gq), ("Wu", uq))
    bg_ptr = _vector("bias_g", bias_g, N, x, dtype)
    bu_ptr = _vector("bias_u", bias_u, N, x, dtype)
    lib = nat.load()

    def call(stream):
        ws_ptr, ws_bytes, sx_ptr = None, 0, None  # as in int8_linear
        if x_scale is not None:
            sx_ptr = x_scale.data_ptr()
        elif M:
            ws_bytes = lib.dx_int8_workspace_size(M, K)
            space = x.new_empty(ws_bytes, dtype=torch.uint8)
            ws_ptr = space.data_ptr()
        g_rows, g_ptr, g_ld = _packed(lib, gq, N, K, ldg, stream)
        u_rows, u_ptr, u_ld = _packed(lib, uq, N, K, ldu, stream)
        return lib.dx_int8_gated_linear(
            x.data_ptr(), x_code, sx_ptr, g_ptr, gs.data_ptr(), u_ptr,
            us.data_ptr(), bg_ptr, bu_ptr, out.data_ptr(), M, N, K, ldx, g_ld, u_ld, ldy,
            DTYPE_CODES[dtype], act, kcode, ws_ptr, ws_bytes, stream)

    rc = _on_device(index, call)
    if rc:
        nat.check("dx_int8_gated_linear", rc)
    return out


def int8_gated_ffn(X, Wg, bg: torch.Tensor | None, Wu, bu: torch.Tensor | None, Wo,
                   bo: torch.Tensor | None, activation="silu",
                   residual: torch.Tensor | None = None, hidden: torch.Tensor | None = None,
                   out: torch.Tensor | None = None,
                   dtype: torch.dtype | None = None) -> torch.Tensor:
    """Y = H Wo^T + bo + residual with H = act(X Wg^T + bg) * (X Wu^T + bu), all
    three weights in 8 bits.  H has Y's type between the two products (`hidden`
    optionally receives it) and is quantised per token again."""
    if isinstance(Wg, tuple) and isinstance(Wo, tuple) and Wo[0].shape[1] != Wg[0].shape[0]:
        raise ValueError(f"Wo must take the hidden width {Wg[0].shape[0]}, got "
                         f"{tuple(Wo[0].shape)}")
    H = int8_gated_linear(X, Wg, Wu, bg, bu, activation, out=hidden, dtype=dtype)
    return int8_linear(H, Wo, bo, None, residual=residual, out=out)

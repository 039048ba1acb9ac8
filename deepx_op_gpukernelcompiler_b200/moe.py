"""Mixture-of-experts layer for the tokens of a serving step.

``moe_ffn`` runs a whole layer — router, choice of experts, every chosen
expert's gated FFN, the weighted sum — in two launches (dx_moe,
include/deepx_fused.h) that read each chosen expert's weights once.  The
reference lists the chain as ``moe_ffn`` with status multi_kernel
(fusion.py:51-53) and never runs it.  It takes up to 64 tokens; the experts are
gated FFNs in the layout of ``gated_ffn`` (mlp.py), stacked: Wg, Wu [E, D, H],
Wo [E, H, D].  A shared expert's output, or the residual stream, goes in as
``residual``.  Inference only: no gradients.
"""
from __future__ import annotations

import ctypes
import struct

import torch

from . import _native as nat
from .int8 import _like, _on_device
from .linear import DTYPE_CODES as _CODES
from .linear import _check_matrix, _ld, activation_code

MAX_TOKENS, MAX_EXPERTS, MAX_TOP_K = 64, 256, 32


# dx_moe_args packed by struct: a third of the time of filling a ctypes.Structure
# (13 pointers, 15 int64, 3 int, padding, pointer, size_t).
_PACK = struct.Struct("@13P15q3i4xPN")
assert _PACK.size == ctypes.sizeof(nat.MoeArgs)


def _experts(name: str, W: torch.Tensor, E: int, rows: int, cols: int, X: torch.Tensor,
             index: int):
    """Checks stacked expert weights -> (address, row pitch, expert pitch)."""
    if W.shape != (E, rows, cols):
        raise ValueError(f"{name} must have shape {(E, rows, cols)}, got {tuple(W.shape)}")
    se, sr, sc = W.stride()
    if sc != 1 or sr < cols or (E > 1 and se < sr * rows):
        raise ValueError(f"{name} must be [E, rows, columns] with contiguous rows that do not "
                         f"overlap, got strides {W.stride()}")
    if W.dtype is not X.dtype or W.get_device() != index:
        _like(name, W, X, X.dtype)
    return W.data_ptr(), sr, se if E > 1 else sr * rows


def _bias(name: str, b: torch.Tensor | None, shape: tuple, X: torch.Tensor) -> int:
    if b is None:
        return 0
    if b.shape != shape or not b.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor of shape {shape}, got "
                         f"{tuple(b.shape)}")
    _like(name, b, X, X.dtype)
    return b.data_ptr()


def moe_ffn(X: torch.Tensor, Wr: torch.Tensor, Wg: torch.Tensor, Wu: torch.Tensor,
            Wo: torch.Tensor, top_k: int, br: torch.Tensor | None = None,
            bg: torch.Tensor | None = None, bu: torch.Tensor | None = None,
            bo: torch.Tensor | None = None, activation="silu", renormalize: bool = True,
            residual: torch.Tensor | None = None, out: torch.Tensor | None = None,
            return_routing: bool = False):
    """Y = residual + sum_e w_e ((act(X Wg_e + bg_e) * (X Wu_e + bu_e)) Wo_e + bo_e).

    X [T, D], T <= 64, fp16 or bf16; Wr [D, E]; D and H multiples of 8.  Each token
    goes to the top_k experts of the largest logits X Wr + br, summed in 64 bits (ties:
    the lowest number); w is the softmax over them, or over all experts with
    ``renormalize=False``.  With ``return_routing`` the result is (Y, w [T, top_k]
    float32, expert numbers [T, top_k] int32), largest first.  What an expert
    computes reaches only the tokens that chose it.  The gate, up and output products
    are sums in fp32.  The hidden values pass between them as two 16-bit values each:
    in bfloat16 with a relative error of 2^-17, in float16 of 2^-22 with a step of 2^-36
    at least, and there they must stay below 65504.  An infinity in Wo gives infinities
    or NaN.  Workspace, per call: 4 T H bytes for every
    expert that can be chosen (min(E, T top_k) of them), and some 450 KB a token."""
    act = activation_code(activation)
    if not isinstance(X, torch.Tensor):
        raise TypeError("X must be a torch tensor")
    dtype = X.dtype
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise ValueError(f"unsupported dtype {dtype}; moe_ffn takes float16 or bfloat16")
    _check_matrix("X", X, None, None)
    T, D = X.shape
    _check_matrix("Wr", Wr, D, None)
    E = Wr.shape[1]
    if Wg.dim() != 3:
        raise ValueError(f"Wg must be [E, D, H], got shape {tuple(Wg.shape)}")
    H = Wg.shape[2]
    if T > MAX_TOKENS:
        raise ValueError(f"moe_ffn is for at most {MAX_TOKENS} tokens, got {T}")
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"moe_ffn takes 1 to {MAX_EXPERTS} experts, got {E}")
    if not 1 <= top_k <= min(E, MAX_TOP_K):
        raise ValueError(f"top_k must be between 1 and {min(E, MAX_TOP_K)}, got {top_k}")
    if D % 8 or H % 8 or not D or not H:
        raise ValueError(f"D and H must be multiples of 8, got {D} and {H}")
    _like("Wr", Wr, X, dtype)
    index = X.get_device()
    wg, ldg, ldg_e = _experts("Wg", Wg, E, D, H, X, index)
    wu, ldu, ldu_e = _experts("Wu", Wu, E, D, H, X, index)
    wo, ldo, ldo_e = _experts("Wo", Wo, E, H, D, X, index)
    br_ptr, bg_ptr = _bias("br", br, (E,), X), _bias("bg", bg, (E, H), X)
    bu_ptr, bo_ptr = _bias("bu", bu, (E, H), X), _bias("bo", bo, (E, D), X)
    r_ptr = ldr = 0
    if residual is not None:
        _check_matrix("residual", residual, T, D)
        _like("residual", residual, X, dtype)
        r_ptr, ldr = residual.data_ptr(), _ld(residual)
    if not X.is_cuda:
        raise ValueError("moe_ffn runs on CUDA tensors only (the engine has no CPU path)")
    if out is None:
        out, ldy = X.new_empty((T, D)), D
    else:
        _check_matrix("out", out, T, D)
        _like("out", out, X, dtype)
        ldy = _ld(out)
    x_ptr, ldx = X.data_ptr(), _ld(X)
    if x_ptr % 16 or (T > 1 and ldx % 8):
        X = X.clone(memory_format=torch.contiguous_format)
        x_ptr, ldx = X.data_ptr(), D
    if T == 1:
        ldx = D
    weights = X.new_empty((T, top_k), dtype=torch.float32)
    ids = X.new_empty((T, top_k), dtype=torch.int32)
    lib = nat.load()

    def call(stream):
        # Of this call alone, from the allocator of the current stream or of the
        # graph being captured.
        size = lib.dx_moe_workspace_size(T, H, E, top_k)
        space = X.new_empty(size, dtype=torch.uint8)
        return lib.dx_moe(_PACK.pack(
            x_ptr, Wr.data_ptr(), br_ptr, wg, wu, wo, bg_ptr, bu_ptr, bo_ptr, r_ptr,
            out.data_ptr(), ids.data_ptr(), weights.data_ptr(), T, D, H, E, top_k, ldx, _ld(Wr),
            ldg, ldg_e, ldu, ldu_e, ldo, ldo_e, ldr, ldy, _CODES[dtype], act,
            1 if renormalize else 0, space.data_ptr(), size), stream)

    rc = _on_device(index, call)
    if rc:
        nat.check("dx_moe", rc)
    return (out, weights, ids) if return_routing else out

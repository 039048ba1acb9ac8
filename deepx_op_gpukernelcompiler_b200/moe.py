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

import torch

from . import _native as nat
from .int8 import _like, _on_device
from .linear import DTYPE_CODES, _check_matrix, _ld, activation_code

MAX_TOKENS, MAX_EXPERTS, MAX_TOP_K = 64, 256, 32


def _experts(name: str, W: torch.Tensor, shape: tuple, X: torch.Tensor) -> None:
    if W.dim() != 3 or tuple(W.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(W.shape)}")
    se, sr, sc = W.stride()
    if sc != 1 or sr < shape[2] or (shape[0] > 1 and se < sr * shape[1]):
        raise ValueError(f"{name} must be [E, rows, columns] with contiguous rows that do not "
                         f"overlap, got strides {W.stride()}")
    _like(name, W, X, X.dtype)


def _bias(name: str, b: torch.Tensor | None, shape: tuple, X: torch.Tensor):
    if b is None:
        return None
    if tuple(b.shape) != shape or not b.is_contiguous():
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
    goes to the top_k experts of the largest logits X Wr + br (ties: the lowest
    number); w is the softmax over them, or over all experts with
    ``renormalize=False``.  With ``return_routing`` the result is (Y, w [T, top_k]
    float32, expert numbers [T, top_k] int32), largest first."""
    act = activation_code(activation)
    if not isinstance(X, torch.Tensor):
        raise TypeError("X must be a torch tensor")
    code = DTYPE_CODES.get(X.dtype)
    if X.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"unsupported dtype {X.dtype}; moe_ffn takes float16 or bfloat16")
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
    _like("Wr", Wr, X, X.dtype)
    _experts("Wg", Wg, (E, D, H), X)
    _experts("Wu", Wu, (E, D, H), X)
    _experts("Wo", Wo, (E, H, D), X)
    br_ptr, bg_ptr = _bias("br", br, (E,), X), _bias("bg", bg, (E, H), X)
    bu_ptr, bo_ptr = _bias("bu", bu, (E, H), X), _bias("bo", bo, (E, D), X)
    r_ptr, ldr = None, 0
    if residual is not None:
        _check_matrix("residual", residual, T, D)
        _like("residual", residual, X, X.dtype)
        r_ptr, ldr = residual.data_ptr(), _ld(residual)
    if X.device.type != "cuda":
        raise ValueError("moe_ffn runs on CUDA tensors only (the engine has no CPU path)")
    if out is None:
        out = X.new_empty((T, D))
    else:
        _check_matrix("out", out, T, D)
        _like("out", out, X, X.dtype)
    if X.data_ptr() % 16 or (T > 1 and X.stride(0) % 8):
        X = X.contiguous() if not X.is_contiguous() else X.clone()
    routing = X.new_empty((2, T, top_k), dtype=torch.float32)
    weights, ids = routing[0], routing[1].view(torch.int32)
    lib = nat.load()

    def call(stream):
        # Of this call alone, from the allocator of the current stream or of the
        # graph being captured.
        size = lib.dx_moe_workspace_size(T, H, E, top_k)
        space = X.new_empty(size, dtype=torch.uint8)
        args = nat.MoeArgs(
            X.data_ptr(), Wr.data_ptr(), br_ptr, Wg.data_ptr(), Wu.data_ptr(), Wo.data_ptr(),
            bg_ptr, bu_ptr, bo_ptr, r_ptr, out.data_ptr(), ids.data_ptr(), weights.data_ptr(), T, D,
            H, E, top_k, _ld(X), _ld(Wr), Wg.stride(1), Wg.stride(0), Wu.stride(1), Wu.stride(0),
            Wo.stride(1), Wo.stride(0), ldr, _ld(out), code, act, 1 if renormalize else 0,
            space.data_ptr(), size)
        return lib.dx_moe(ctypes.addressof(args), stream)

    rc = _on_device(X.get_device(), call)
    if rc:
        nat.check("dx_moe", rc)
    return (out, weights, ids) if return_routing else out

"""Serving operators beside the reference's eight ops: FP8 operand preparation
(``quantize_fp8``, ``layernorm_fp8``) and the FP8 matrix product with one scale
per block of 128 (``gemm_fp8``). The reference has no counterpart.

They keep the manner of ``vit_cuda._C``: CUDA tensors on the current device
(RuntimeError otherwise), fresh outputs from PyTorch's caching allocator, work
launched asynchronously on the current stream, no workspace, capturable in a
CUDA graph. They are forward only, like every op of this package.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from ._C import _ptr, _same_device, _stream
from ._lib import lib

FP8 = torch.float8_e4m3fn
BLOCK = 128  # columns (and, for weights, rows) that share one scale

_TYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def _type_code(dtype: torch.dtype, what: str) -> int:
    code = _TYPES.get(dtype)
    if code is None:
        raise RuntimeError(f"{what} must be float32, float16 or bfloat16")
    return code


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """(tensor, rows, row stride in elements) of a tensor read as [rows, last
    dim]: as it is where one stride describes the rows, else a contiguous copy."""
    n = t.shape[-1]
    if t.dim() == 2 and (t.stride(1) == 1 or n == 1) and t.stride(0) >= n:
        return t, t.shape[0], t.stride(0)
    if not t.is_contiguous():
        # a padded [B, N, K] of code rows still has one stride
        if (t.dim() == 3 and t.stride(2) == 1 and t.stride(1) >= n
                and t.stride(0) == t.shape[1] * t.stride(1)):
            return t, t.shape[0] * t.shape[1], t.stride(1)
        t = t.contiguous()
    rows = 1
    for d in t.shape[:-1]:
        rows *= d
    return t, rows, n


def _codes_like(X: torch.Tensor) -> tuple[torch.Tensor, int]:
    """(empty codes of X's shape, row stride): rows a multiple of 16 bytes apart,
    as the matrix product's loads need them."""
    n = X.shape[-1]
    ld = (n + 15) // 16 * 16
    q = torch.empty((*X.shape[:-1], ld), dtype=FP8, device=X.device)
    return (q if ld == n else q[..., :n]), ld


# ---------------------------------------------------------------- ops
def quantize_fp8(X: torch.Tensor, block_rows: int = 1) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of X [..., K] (float32, float16 or bfloat16): e4m3 codes of
    X's shape and one float32 scale per block, X ~= codes * scale with
    scale = max|block| / 448. ``block_rows=1``: blocks of 128 columns of one row,
    scales [..., ceil(K/128)] (activations). ``block_rows=128``: blocks of
    128 x 128 of a 2-D X, scales [ceil(N/128), ceil(K/128)] (weights). Rows of the
    codes are 16 bytes or a multiple apart. A block holding a NaN or an infinity
    dequantises to NaN."""
    _same_device([X], "quantize_fp8")
    code = _type_code(X.dtype, "X")
    if X.dim() < 1 or X.shape[-1] < 1:
        raise RuntimeError("X must be [..., K] with K >= 1")
    if block_rows not in (1, BLOCK):
        raise RuntimeError("block_rows must be 1 or 128")
    if block_rows != 1 and X.dim() != 2:
        raise RuntimeError("X must be 2D for 128 x 128 blocks")
    Xc, M, ldx = _rows(X)
    K = X.shape[-1]
    q, ldq = _codes_like(X)
    lead = X.shape[:-1] if block_rows == 1 else (_blocks(M),)
    scales = torch.empty((*lead, _blocks(K)), dtype=torch.float32, device=X.device)
    _lib.check(lib.vitb200_quantize_fp8(Xc.data_ptr(), code, M, K, ldx, block_rows, q.data_ptr(),
                                        ldq, scales.data_ptr(), _stream()), "quantize_fp8")
    return q, scales


def layernorm_fp8(X: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor,
                  eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """``quantize_fp8(layernorm_forward(X, gamma, beta, eps))`` in one pass over X
    [..., K] (float32, float16 or bfloat16; gamma and beta float32): (codes, scales)."""
    _same_device([X, gamma, beta], "layernorm_fp8")
    code = _type_code(X.dtype, "X")
    if X.dim() < 1 or X.shape[-1] < 1:
        raise RuntimeError("X must be [..., K] with K >= 1")
    K = X.shape[-1]
    for t, name in ((gamma, "gamma"), (beta, "beta")):
        if t.dtype != torch.float32:
            raise RuntimeError(f"{name} must be float32")
        if t.numel() != K:
            raise RuntimeError(f"{name} size mismatch")
    Xc, M, ldx = _rows(X)
    gc, bc = gamma.contiguous(), beta.contiguous()
    q, ldq = _codes_like(X)
    scales = torch.empty((*X.shape[:-1], _blocks(K)), dtype=torch.float32, device=X.device)
    _lib.check(lib.vitb200_layernorm_fp8(Xc.data_ptr(), code, M, K, ldx, gc.data_ptr(),
                                         bc.data_ptr(), float(eps), q.data_ptr(), ldq,
                                         scales.data_ptr(), _stream()), "layernorm_fp8")
    return q, scales


def _code_rows(q: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """_rows of codes, with rows and base aligned to 16 bytes (a padded copy if not)."""
    t, rows, ld = _rows(q)
    if ld % 16 or t.data_ptr() % 16:
        c, ld = _codes_like(q)
        c.view(torch.uint8).copy_(q.view(torch.uint8))
        t = c
    return t, rows, ld


def gemm_fp8(X: torch.Tensor, X_scale: torch.Tensor, W: torch.Tensor, W_scale: torch.Tensor,
             B: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
             gelu: bool = False, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Y = residual + act(X W^T + B) of e4m3 operands as ``quantize_fp8`` makes
    them: X [N, K] or [B, N, K] with X_scale [..., ceil(K/128)], W [N_out, K] with
    W_scale [ceil(N_out/128), ceil(K/128)]; B [N_out] float32, act erf-GELU when
    ``gelu``, residual of Y's shape and type. Sums are float32, Y is rounded once
    to ``out_dtype`` (float32, float16 or bfloat16)."""
    tensors = [X, X_scale, W, W_scale]
    if B is not None:
        tensors.append(B)
    if residual is not None:
        tensors.append(residual)
    _same_device(tensors, "gemm_fp8")
    if X.dtype != FP8 or W.dtype != FP8:
        raise RuntimeError("X and W must be float8_e4m3fn")
    if X_scale.dtype != torch.float32 or W_scale.dtype != torch.float32:
        raise RuntimeError("X_scale and W_scale must be float32")
    code = _type_code(out_dtype, "out_dtype")
    if X.dim() not in (2, 3):
        raise RuntimeError("X must be [N, K] or [B, N, K]")
    if W.dim() != 2:
        raise RuntimeError("W must be [N_out, K]")
    K = X.shape[-1]
    N = W.shape[0]
    if K < 1:
        raise RuntimeError("K must be at least 1")
    if W.shape[1] != K:
        raise RuntimeError("W second dim must match K")
    kb = _blocks(K)
    if tuple(X_scale.shape) != (*X.shape[:-1], kb):
        raise RuntimeError(f"X_scale must be [..., {kb}] (one scale per row and 128 columns)")
    if tuple(W_scale.shape) != (_blocks(N), kb):
        raise RuntimeError(f"W_scale must be [{_blocks(N)}, {kb}] (one scale per 128 x 128 block)")
    if B is not None:
        if B.dtype != torch.float32:
            raise RuntimeError("B must be float32")
        if B.numel() != N:
            raise RuntimeError("bias size mismatch")
        B = B.contiguous()
    Y = torch.empty((*X.shape[:-1], N), dtype=out_dtype, device=X.device)
    ldr = 0
    if residual is not None:
        if residual.dtype != out_dtype:
            raise RuntimeError("residual must have out_dtype")
        if residual.shape != Y.shape:
            raise RuntimeError("residual shape mismatch")
        residual, _, ldr = _rows(residual)
    Xc, M, ldx = _code_rows(X)
    Wc, _, ldw = _code_rows(W)
    Xs, _, ldxs = _rows(X_scale)
    Ws, _, ldws = _rows(W_scale)
    _lib.check(lib.vitb200_gemm_fp8(Xc.data_ptr(), ldx, Xs.data_ptr(), ldxs, Wc.data_ptr(), ldw,
                                    Ws.data_ptr(), ldws, _ptr(B), _ptr(residual), ldr,
                                    Y.data_ptr(), N, code, M, K, N, 1 if gelu else 0, _stream()),
               "gemm_fp8")
    return Y


__all__ = ["quantize_fp8", "layernorm_fp8", "gemm_fp8"]

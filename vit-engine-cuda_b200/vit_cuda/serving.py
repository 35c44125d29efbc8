"""Serving operators beside the reference's eight ops: FP8 operand preparation
(``quantize_fp8``, ``layernorm_fp8``), the FP8 matrix product with one scale per
block of 128 (``gemm_fp8``) and attention to an encoder's states of another length
(``cross_attention``). The reference has no counterparts.

They keep the manner of ``vit_cuda._C``: CUDA tensors on the current device
(RuntimeError otherwise), fresh outputs from PyTorch's caching allocator, work
launched asynchronously on the current stream, no workspace, capturable in a
CUDA graph. They are forward only, like every op of this package.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _lib
from ._C import _same_device
from ._lib import lib

FP8 = torch.float8_e4m3fn
BLOCK = 128  # columns (and, for weights, rows) that share one scale

_TYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}

# A single token's step runs a few microseconds on the GPU, so an eager call
# must not cost tens on the host: the raw handle of the current stream is read
# without building a Stream object (0.1 us against 3.2), and every helper has a
# short way for contiguous tensors.
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _on_device(op: str, *tensors: Optional[torch.Tensor]) -> int:
    """The current device's index, after checking that every tensor given is on it."""
    try:
        device = _current_device()
        for t in tensors:
            if t is not None and t.get_device() != device:
                break
        else:
            return device
    except (AttributeError, RuntimeError):
        pass
    _same_device([t for t in tensors if t is not None], op)  # says what is wrong
    raise RuntimeError(f"{op}: all inputs must be on the current CUDA device")


def _type_code(dtype: torch.dtype, what: str) -> int:
    code = _TYPES.get(dtype)
    if code is None:
        raise RuntimeError(f"{what} must be float32, float16 or bfloat16")
    return code


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """(tensor, row stride in elements) of a tensor read as [rows, last dim]: as
    it is where one stride describes the rows, else a contiguous copy."""
    n = t.shape[-1]
    if t.is_contiguous():
        return t, n
    st = t.stride()
    if st[-1] == 1:
        if t.dim() == 2 and st[0] >= n:
            return t, st[0]
        # a padded [B, N, K] still has one stride
        if t.dim() == 3 and st[1] >= n and st[0] == t.shape[1] * st[1]:
            return t, st[1]
    return t.contiguous(), n


def _code_rows(q: torch.Tensor) -> tuple[torch.Tensor, int]:
    """_rows of codes, with rows and base aligned to 16 bytes (a padded copy if not)."""
    t, ld = _rows(q)
    if ld % 16 or t.data_ptr() % 16:
        c, ld = _codes_like(q)
        c.view(torch.uint8).copy_(q.view(torch.uint8))
        t = c
    return t, ld


def _codes_like(X: torch.Tensor) -> tuple[torch.Tensor, int]:
    """(empty codes of X's shape, row stride): rows a multiple of 16 bytes apart,
    as the matrix product's loads need them."""
    n = X.shape[-1]
    if n % 16 == 0:
        return torch.empty_like(X, dtype=FP8, memory_format=torch.contiguous_format), n
    ld = (n + 15) // 16 * 16
    return X.new_empty((*X.shape[:-1], ld), dtype=FP8)[..., :n], ld


# ---------------------------------------------------------------- ops
def quantize_fp8(X: torch.Tensor, block_rows: int = 1) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of X [..., K] (float32, float16 or bfloat16): e4m3 codes of
    X's shape and one float32 scale per block, X ~= codes * scale with
    scale = max|block| / 448. ``block_rows=1``: blocks of 128 columns of one row,
    scales [..., ceil(K/128)] (activations). ``block_rows=128``: blocks of
    128 x 128 of a 2-D X, scales [ceil(N/128), ceil(K/128)] (weights). Rows of the
    codes are 16 bytes or a multiple apart. A block holding a NaN or an infinity
    dequantises to NaN."""
    device = _on_device("quantize_fp8", X)
    code = _type_code(X.dtype, "X")
    shape = X.shape
    if not shape or shape[-1] < 1:
        raise RuntimeError("X must be [..., K] with K >= 1")
    K = shape[-1]
    M = X.numel() // K
    if block_rows == 1:
        lead = shape[:-1]
    elif block_rows != BLOCK:
        raise RuntimeError("block_rows must be 1 or 128")
    elif len(shape) != 2:
        raise RuntimeError("X must be 2D for 128 x 128 blocks")
    else:
        lead = (_blocks(M),)
    Xc, ldx = _rows(X)
    q, ldq = _codes_like(X)
    scales = X.new_empty((*lead, _blocks(K)), dtype=torch.float32)
    st = lib.vitb200_quantize_fp8(Xc.data_ptr(), code, M, K, ldx, block_rows, q.data_ptr(), ldq,
                                  scales.data_ptr(), _raw_stream(device))
    if st:
        _lib.check(st, "quantize_fp8")
    return q, scales


def layernorm_fp8(X: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor,
                  eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """``quantize_fp8(layernorm_forward(X, gamma, beta, eps))`` in one pass over X
    [..., K] (float32, float16 or bfloat16; gamma and beta float32): (codes, scales)."""
    device = _on_device("layernorm_fp8", X, gamma, beta)
    code = _type_code(X.dtype, "X")
    shape = X.shape
    if not shape or shape[-1] < 1:
        raise RuntimeError("X must be [..., K] with K >= 1")
    K = shape[-1]
    for t, name in ((gamma, "gamma"), (beta, "beta")):
        if t.dtype != torch.float32:
            raise RuntimeError(f"{name} must be float32")
        if t.numel() != K:
            raise RuntimeError(f"{name} size mismatch")
    Xc, ldx = _rows(X)
    gc, bc = gamma.contiguous(), beta.contiguous()
    q, ldq = _codes_like(X)
    scales = X.new_empty((*shape[:-1], _blocks(K)), dtype=torch.float32)
    st = lib.vitb200_layernorm_fp8(Xc.data_ptr(), code, X.numel() // K, K, ldx, gc.data_ptr(),
                                   bc.data_ptr(), eps, q.data_ptr(), ldq, scales.data_ptr(),
                                   _raw_stream(device))
    if st:
        _lib.check(st, "layernorm_fp8")
    return q, scales


def gemm_fp8(X: torch.Tensor, X_scale: torch.Tensor, W: torch.Tensor, W_scale: torch.Tensor,
             B: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
             gelu: bool = False, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Y = residual + act(X W^T + B) of e4m3 operands as ``quantize_fp8`` makes
    them: X [N, K] or [B, N, K] with X_scale [..., ceil(K/128)], W [N_out, K] with
    W_scale [ceil(N_out/128), ceil(K/128)]; B [N_out] float32, act erf-GELU when
    ``gelu``, residual of Y's shape and type. Sums are float32, Y is rounded once
    to ``out_dtype`` (float32, float16 or bfloat16)."""
    device = _on_device("gemm_fp8", X, X_scale, W, W_scale, B, residual)
    if X.dtype != FP8 or W.dtype != FP8:
        raise RuntimeError("X and W must be float8_e4m3fn")
    if X_scale.dtype != torch.float32 or W_scale.dtype != torch.float32:
        raise RuntimeError("X_scale and W_scale must be float32")
    code = _type_code(out_dtype, "out_dtype")
    xshape, wshape = X.shape, W.shape
    if len(xshape) not in (2, 3):
        raise RuntimeError("X must be [N, K] or [B, N, K]")
    if len(wshape) != 2:
        raise RuntimeError("W must be [N_out, K]")
    N, K = wshape
    lead = xshape[:-1]
    if K < 1:
        raise RuntimeError("K must be at least 1")
    if xshape[-1] != K:
        raise RuntimeError("W second dim must match K")
    kb = _blocks(K)
    if X_scale.shape != (*lead, kb):
        raise RuntimeError(f"X_scale must be [..., {kb}] (one scale per row and 128 columns)")
    if W_scale.shape != (_blocks(N), kb):
        raise RuntimeError(f"W_scale must be [{_blocks(N)}, {kb}] (one scale per 128 x 128 block)")
    yshape = (*lead, N)
    bias_ptr = res_ptr = None
    ldr = 0
    if B is not None:
        if B.dtype != torch.float32:
            raise RuntimeError("B must be float32")
        if B.numel() != N:
            raise RuntimeError("bias size mismatch")
        B = B.contiguous()
        bias_ptr = B.data_ptr()
    if residual is not None:
        if residual.dtype != out_dtype:
            raise RuntimeError("residual must have out_dtype")
        if residual.shape != yshape:
            raise RuntimeError("residual shape mismatch")
        residual, ldr = _rows(residual)
        res_ptr = residual.data_ptr()
    Xc, ldx = _code_rows(X)
    Wc, ldw = _code_rows(W)
    Xs, ldxs = _rows(X_scale)
    Ws, ldws = _rows(W_scale)
    Y = X.new_empty(yshape, dtype=out_dtype)
    st = lib.vitb200_gemm_fp8(Xc.data_ptr(), ldx, Xs.data_ptr(), ldxs, Wc.data_ptr(), ldw,
                              Ws.data_ptr(), ldws, bias_ptr, res_ptr, ldr, Y.data_ptr(), N, code,
                              X.numel() // K, K, N, 1 if gelu else 0, _raw_stream(device))
    if st:
        _lib.check(st, "gemm_fp8")
    return Y


def _attention_operand(t: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """(tensor, row stride, batch stride) of a [B, N, E] operand in elements: as it
    is where rows are contiguous and everything is 16-byte aligned, else a copy."""
    B, N, E = t.shape
    sb, sn, se = t.stride()
    if B == 1:
        sb = N * sn if N else E
    if N <= 1:
        sn = E
    # a stride of 0 (an expanded batch) is no stride of a copy descriptor's
    if se != 1 or sn < E or sn % 8 or sb < E or sb % 8 or t.data_ptr() % 16:
        return t.clone(memory_format=torch.contiguous_format), E, max(N, 1) * E
    return t, sn, sb


def cross_attention(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, scale: float, heads: int,
                    kv_heads: Optional[int] = None,
                    kv_lens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(Q K^T * scale) V of queries Q [B, Tq, heads * D] over another
    sequence's keys and values K, V [B, Tk, kv_heads * D] (float16 or bfloat16, D
    64 or 128): an encoder's states read by a decoder's prompt, by its single
    tokens (Tq = 1), or by a pooling head. ``heads`` is a multiple of ``kv_heads``
    (default: equal); query head h reads key head h // (heads // kv_heads).
    ``kv_lens`` [B] int32: the keys of each image, clamped to 0..Tk; keys past it
    may hold anything, and an image without keys gets zeros. K and V may be column
    ranges of one tensor (no copy is made)."""
    device = _on_device("cross_attention", Q, K, V, kv_lens)
    dtype = Q.dtype
    if dtype != torch.bfloat16 and dtype != torch.float16:
        raise RuntimeError("Q must be float16 or bfloat16 (flash_attn_2 takes float32)")
    if K.dtype != dtype or V.dtype != dtype:
        raise RuntimeError("Q, K and V must have the same type")
    qshape, kshape = Q.shape, K.shape
    if len(qshape) != 3:
        raise RuntimeError("Q must be [B, Tq, heads * D]")
    if len(kshape) != 3 or kshape[0] != qshape[0]:
        raise RuntimeError("K must be [B, Tk, kv_heads * D] with Q's B")
    if V.shape != kshape:
        raise RuntimeError("V shape must match K shape")
    if kv_heads is None:
        kv_heads = heads
    if heads < 1 or kv_heads < 1 or heads % kv_heads:
        raise RuntimeError("heads must be a positive multiple of kv_heads")
    B, Tq, E = qshape
    D = E // heads
    if D not in (64, 128) or E != heads * D:
        raise RuntimeError("Q's last dim must be heads * D with D 64 or 128")
    if kshape[2] != kv_heads * D:
        raise RuntimeError("K's last dim must be kv_heads * D with Q's D")
    lens_ptr = None
    if kv_lens is not None:
        if kv_lens.dtype != torch.int32:
            raise RuntimeError("kv_lens must be int32")
        if kv_lens.dim() != 1 or kv_lens.shape[0] != B:
            raise RuntimeError("kv_lens must be [B]")
        kv_lens = kv_lens.contiguous()
        lens_ptr = kv_lens.data_ptr()
    Qc, q_row, q_batch = _attention_operand(Q)
    Kc, k_row, k_batch = _attention_operand(K)
    Vc, v_row, v_batch = _attention_operand(V)
    O = Q.new_empty(qshape)
    st = lib.vitb200_cross_attention(Qc.data_ptr(), Kc.data_ptr(), Vc.data_ptr(), O.data_ptr(),
                                     _TYPES[dtype], B, Tq, kshape[1], heads, kv_heads, D, q_row,
                                     q_batch, k_row, k_batch, v_row, v_batch, lens_ptr, scale,
                                     _raw_stream(device))
    if st:
        _lib.check(st, "cross_attention")
    return O


__all__ = ["quantize_fp8", "layernorm_fp8", "gemm_fp8", "cross_attention"]

"""Serving operators beside the reference's eight ops: FP8 operand preparation
(``quantize_fp8``, ``layernorm_fp8``), the FP8 matrix product with one scale per
block of 128 (``gemm_fp8``) and attention to an encoder's states of another length
(``cross_attention``). The reference has no counterparts.

They keep the manner of ``vit_cuda._C``: CUDA tensors on the current device
(RuntimeError otherwise), fresh outputs from PyTorch's caching allocator, work
launched asynchronously on the current stream, scratch space from the caching
allocator too, so that they can be captured in a CUDA graph. They are forward
only, like every op of this package: an output of inputs that require a gradient
requires one too, and its backward raises.

Each op is registered as ``torch.ops.vit_cuda.<op>`` (vit_cuda/library.py). A plain
call goes past the dispatcher; one that a tracer, a dispatch or function mode, a
transform or autograd has to see goes through the registered op.

The checks and the call into libvitb200.so are compiled (csrc/bindings.cpp, built
as ``vit_cuda._serving``): in a single token's step the host's time per call is
what a user waits for.
"""
from __future__ import annotations

import ctypes
import threading
from typing import Optional

import torch

from . import _lib

FP8 = torch.float8_e4m3fn
BLOCK = 128  # columns (and, for weights, rows) that share one scale

_ops = None
_lock = threading.Lock()


def _raise_status(status: int, what: str) -> None:
    raise _lib.VitB200Error(what, status)


def direct():
    """The compiled module itself: what the registered ops run on the GPU."""
    return _ops or _load()


def _load():
    """Imports the compiled module and hands it libvitb200.so's entry points (on
    the first call, so that importing the package maps neither)."""
    global _ops
    with _lock:
        if _ops is None:
            try:
                from . import _serving
                built_for = getattr(_serving, "BUILT_FOR", "another version")
                if built_for != torch.__version__:
                    raise ImportError(f"built for PyTorch {built_for}, "
                                      f"and this is {torch.__version__}")
            except ImportError as e:
                raise ImportError("vit_cuda: vit_cuda/_serving.so is missing or does not match this "
                                  "PyTorch; build it with `python vit-engine-cuda_b200/build.py`"
                                  ) from e
            entries = (_lib.lib.vitb200_quantize_fp8, _lib.lib.vitb200_layernorm_fp8,
                       _lib.lib.vitb200_gemm_fp8, _lib.lib.vitb200_cross_attention,
                       _lib.lib.vitb200_cross_attention_workspace_bytes)
            _serving.bind(*(ctypes.cast(f, ctypes.c_void_p).value for f in entries), _raise_status)
            _ops = _serving
    return _ops


# ---------------------------------------------------------------- ops
def quantize_fp8(X: torch.Tensor, block_rows: int = 1) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of X [..., K] (float32, float16 or bfloat16): e4m3 codes of
    X's shape and one float32 scale per block, X ~= codes * scale with
    scale = max|block| / 448. ``block_rows=1``: blocks of 128 columns of one row,
    scales [..., ceil(K/128)] (activations). ``block_rows=128``: blocks of
    128 x 128 of a 2-D X, scales [ceil(N/128), ceil(K/128)] (weights). Rows of the
    codes are 16 bytes or a multiple apart. A block holding a NaN or an infinity
    dequantises to NaN."""
    if torch.compiler.is_compiling() or (_ops or _load()).watched(X):
        return torch.ops.vit_cuda.quantize_fp8(X, block_rows)
    return _ops.quantize_fp8(X, block_rows)


def layernorm_fp8(X: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor,
                  eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """``quantize_fp8(layernorm_forward(X, gamma, beta, eps))`` in one pass over X
    [..., K] (float32, float16 or bfloat16; gamma and beta float32): (codes, scales)."""
    if torch.compiler.is_compiling() or (_ops or _load()).watched(X, gamma, beta):
        return torch.ops.vit_cuda.layernorm_fp8(X, gamma, beta, eps)
    return _ops.layernorm_fp8(X, gamma, beta, eps)


def gemm_fp8(X: torch.Tensor, X_scale: torch.Tensor, W: torch.Tensor, W_scale: torch.Tensor,
             B: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
             gelu: bool = False, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Y = residual + act(X W^T + B) of e4m3 operands as ``quantize_fp8`` makes
    them: X [N, K] or [B, N, K] with X_scale [..., ceil(K/128)], W [N_out, K] with
    W_scale [ceil(N_out/128), ceil(K/128)]; B [N_out] float32, act erf-GELU when
    ``gelu``, residual of Y's shape and type. Sums are float32, Y is rounded once
    to ``out_dtype`` (float32, float16 or bfloat16)."""
    if torch.compiler.is_compiling() or (_ops or _load()).watched(X, X_scale, W, W_scale, B,
                                                                  residual):
        return torch.ops.vit_cuda.gemm_fp8(X, X_scale, W, W_scale, B, residual, gelu, out_dtype)
    return _ops.gemm_fp8(X, X_scale, W, W_scale, B, residual, gelu, out_dtype)


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
    if torch.compiler.is_compiling() or (_ops or _load()).watched(Q, K, V, kv_lens):
        return torch.ops.vit_cuda.cross_attention(Q, K, V, scale, heads, kv_heads, kv_lens)
    return _ops.cross_attention(Q, K, V, scale, heads, kv_heads, kv_lens)


__all__ = ["quantize_fp8", "layernorm_fp8", "gemm_fp8", "cross_attention"]

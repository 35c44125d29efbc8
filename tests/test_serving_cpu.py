"""Argument checks of the serving operators' C entry points and Python
functions that need no GPU: bad calls come back with a status or an error
before any device work."""
import ctypes

import pytest
import torch

import vit_cuda
from vit_cuda import _lib
from vit_cuda._lib import lib

P = 1 << 20  # a 16-byte aligned address; rejected calls never touch it


def quantize(x=P, type=0, rows=4, K=128, ldx=128, block_rows=1, q=P, ldq=128, scales=P):
    return lib.vitb200_quantize_fp8(x, type, rows, K, ldx, block_rows, q, ldq, scales, None)


def layernorm(x=P, type=0, rows=4, K=128, ldx=128, gamma=P, beta=P, q=P, ldq=128, scales=P):
    return lib.vitb200_layernorm_fp8(x, type, rows, K, ldx, gamma, beta, 1e-6, q, ldq, scales, None)


def gemm(X=P, ldx=128, xs=P, ldxs=1, W=P, ldw=128, ws=P, ldws=1, bias=None, residual=None, ldr=0,
         out=P, ldo=16, type=0, M=4, K=128, N=16):
    return lib.vitb200_gemm_fp8(X, ldx, xs, ldxs, W, ldw, ws, ldws, bias, residual, ldr, out, ldo,
                                type, M, K, N, 0, None)


@pytest.mark.parametrize("call", [quantize, layernorm])
def test_quantize_status(call):
    for kw in (dict(rows=-1), dict(K=0), dict(ldx=127), dict(ldq=112), dict(type=3), dict(type=-1),
               dict(x=None), dict(q=None), dict(scales=None)):
        assert call(**kw) == _lib.E_INVALID_ARG, kw
    for kw in (dict(ldq=136), dict(q=P + 8), dict(x=P + 2)):
        assert call(**kw) == _lib.E_ALIGNMENT, kw
    assert call(rows=0) == _lib.OK
    assert call(rows=0, x=None, scales=None) == _lib.OK


def test_quantize_block_rows_status():
    assert quantize(block_rows=64) == _lib.E_INVALID_ARG
    assert layernorm(gamma=None) == _lib.E_INVALID_ARG


def test_gemm_status():
    for kw in (dict(M=-1), dict(N=-1), dict(K=0), dict(type=3), dict(ldx=112), dict(ldw=112),
               dict(ldxs=0), dict(ldws=0), dict(ldo=15), dict(residual=P, ldr=15), dict(X=None),
               dict(W=None), dict(xs=None), dict(ws=None), dict(out=None), dict(M=1 << 40)):
        assert gemm(**kw) == _lib.E_INVALID_ARG, kw
    for kw in (dict(ldx=136), dict(ldw=136), dict(X=P + 8), dict(W=P + 1), dict(xs=P + 2),
               dict(out=P + 2), dict(bias=P + 1), dict(residual=P + 2, ldr=16)):
        assert gemm(**kw) == _lib.E_ALIGNMENT, kw
    assert gemm(M=0, X=None) == _lib.OK
    assert gemm(N=0, out=None) == _lib.OK


def cross(q=P, k=P, v=P, o=P, type=1, B=2, Tq=3, Tk=5, heads=4, kv_heads=2, D=64, qs=(256, 768),
          ks=(128, 640), vs=(128, 640), lens=None):
    return lib.vitb200_cross_attention(q, k, v, o, type, B, Tq, Tk, heads, kv_heads, D, *qs, *ks,
                                       *vs, lens, 0.125, None, 0, None)


def test_cross_attention_status():
    for kw in (dict(type=0), dict(type=3), dict(B=-1), dict(Tq=-1), dict(Tk=-1), dict(heads=0),
               dict(kv_heads=0), dict(kv_heads=3), dict(q=None), dict(k=None), dict(v=None),
               dict(o=None), dict(qs=(255, 768)), dict(ks=(64, 640)), dict(vs=(64, 640)),
               dict(ks=(128, -8))):
        assert cross(**kw) == _lib.E_INVALID_ARG, kw
    for kw in (dict(q=P + 8), dict(k=P + 2), dict(v=P + 4), dict(o=P + 8), dict(qs=(260, 780)),
               dict(ks=(132, 640)), dict(vs=(128, 644)), dict(lens=P + 2)):
        assert cross(**kw) == _lib.E_ALIGNMENT, kw
    assert cross(D=32) == cross(D=96) == _lib.E_UNSUPPORTED
    assert cross(B=0, q=None) == _lib.OK
    assert cross(Tq=0, o=None) == _lib.OK


def test_python_refuses_cpu_tensors():
    x = torch.randn(4, 128)
    q, s = x.to(torch.float8_e4m3fn), torch.ones(4, 1)
    for call in (lambda: vit_cuda.quantize_fp8(x), lambda: vit_cuda.gemm_fp8(q, s, q, s[:1]),
                 lambda: vit_cuda.layernorm_fp8(x, x[0], x[0], 1e-6),
                 lambda: vit_cuda.cross_attention(x[None], x[None], x[None], 0.1, 2)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_quantisers_refuse_unaligned_fp32():
    """An fp32 pointer off a 4-byte boundary would fault on the GPU."""
    for off in (1, 2, 3):
        assert quantize(scales=P + off) == layernorm(scales=P + off) == _lib.E_ALIGNMENT
        assert layernorm(gamma=P + off) == layernorm(beta=P + off) == _lib.E_ALIGNMENT
    assert layernorm(gamma=None, beta=P + 1) == _lib.E_INVALID_ARG

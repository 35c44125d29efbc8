"""One row, or one token of each sequence: dimensions of size one, whose strides say
nothing, are read in place. A copy would cost the single-token step an allocation and a
launch more than the operator itself."""
import pytest
import torch

import vit_cuda

pytestmark = pytest.mark.gpu


def randn(*shape, seed=0, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def allocations(f):
    """(result, allocations) of a call."""
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    y = f()
    return y, torch.cuda.memory_stats()["allocation.all.allocated"] - before


def same(a, b):
    return all(torch.equal(x.float(), y.float()) for x, y in zip(a, b))


@pytest.mark.parametrize("shape", [(1, 1000), (1, 1, 1000)])
def test_codes_of_one_row(cuda, shape):
    x, w = randn(*shape, seed=1), vit_cuda.quantize_fp8(randn(300, 1000, seed=2), 128)
    q, s = vit_cuda.quantize_fp8(x)
    y, n = allocations(lambda: vit_cuda.gemm_fp8(q, s, *w))
    assert n == 1  # the result
    many = vit_cuda.gemm_fp8(*vit_cuda.quantize_fp8(x.reshape(1, 1000).expand(3, -1)), *w)
    assert torch.equal(y.reshape(1, 300), many[:1])
    # an unaligned start is still copied
    wide = torch.zeros(1, 1100, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    part = wide[:, 3:1003]
    part.view(torch.uint8).copy_(q.view(torch.uint8).reshape(1, 1000))
    assert torch.equal(vit_cuda.gemm_fp8(part, s.reshape(1, -1), *w), many[:1])


@pytest.mark.parametrize("k", [256, 1000, 77])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_token_of_each_sequence(cuda, k, dtype):
    x, gamma, beta = randn(3, 9, k, seed=3, dtype=dtype), randn(k, seed=4), randn(k, seed=5)
    wq, ws = vit_cuda.quantize_fp8(randn(70, k, seed=6), 128)
    res = randn(3, 9, 70, seed=7)
    for part, r in ((x[:, 4:5], res[:, 4:5]), (x[1:2], res[1:2]), (x[1:2, 3:7], res[1:2, 3:7]),
                    (x[2:, 8:], res[2:, 8:])):
        c = part.contiguous()
        got, n = allocations(lambda: vit_cuda.quantize_fp8(part))
        assert n == 2 and same(got, vit_cuda.quantize_fp8(c))
        got, n = allocations(lambda: vit_cuda.layernorm_fp8(part, gamma, beta, 1e-6))
        assert n == 2 and same(got, vit_cuda.layernorm_fp8(c, gamma, beta, 1e-6))
        q, s = got
        y, n = allocations(lambda: vit_cuda.gemm_fp8(q, s, wq, ws, residual=r))
        assert n == 1
        assert torch.equal(y, vit_cuda.gemm_fp8(q, s, wq, ws, residual=r.contiguous()))
    # what one stride does not describe is copied
    got, n = allocations(lambda: vit_cuda.quantize_fp8(x[:, 2:5]))
    assert n == 3 and same(got, vit_cuda.quantize_fp8(x[:, 2:5].contiguous()))

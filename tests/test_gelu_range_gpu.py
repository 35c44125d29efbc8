"""gemm_fp8's GELU of sums that leave fp32's range: infinity stays infinity, and where
the sum is -infinity the result is GELU's limit, zero."""
import pytest
import torch

import vit_cuda

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n", [(3, 130), (3, 131), (2600, 1000)])
def test_infinite_sums(cuda, out, m, n):
    k = 256
    one = torch.ones(m, k, device="cuda").to(torch.float8_e4m3fn)
    w = torch.ones(n, k, device="cuda")
    w[1::3] = -1
    w[2::3] = 0
    w = w.to(torch.float8_e4m3fn)
    big, unit = torch.full((m, 2), 1e30, device="cuda"), torch.ones(-(-n // 128), 2, device="cuda")
    want = torch.zeros(m, n, device="cuda")
    want[:, 0::3] = float("inf")
    y = vit_cuda.gemm_fp8(one, big, w, unit * 1e8, gelu=True, out_dtype=out)
    assert torch.equal(y.float(), want)
    # by way of the bias
    bias = torch.full((n,), float("inf"), device="cuda")
    bias[1::3] = -float("inf")
    bias[2::3] = -1e6
    y = vit_cuda.gemm_fp8(one, torch.ones_like(big), w, unit, bias, gelu=True, out_dtype=out)
    assert torch.equal(y.float(), want)
    bias[:] = 0
    bias[0] = float("nan")
    y = vit_cuda.gemm_fp8(one, torch.ones_like(big), w, unit, bias, gelu=True, out_dtype=out)
    assert bool(y[:, 0].isnan().all()) and bool(y[:, 1:].isfinite().all())

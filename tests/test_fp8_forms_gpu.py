"""The forms of the FP8 quantisers that only large inputs reach: several loads a warp,
grids that stride over the work, a row per CTA with the next row's loads ahead. Codes
and values against 64 bits, with the checks of test_fp8_gpu."""
import pytest
import torch

import test_fp8_gpu as base
import vit_cuda

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", base.DTYPES)
@pytest.mark.parametrize("m,k", [
    (6000, 512), (6000, 520), (6000, 768), (10000, 1536), (12000, 771), (5000, 1024), (3000, 2304),
    (20000, 256), (40000, 130), (70000, 24)])
def test_quantize_rows(cuda, dtype, m, k):
    x = base.randn(m, k, seed=m + k) * torch.exp(0.5 * base.randn(m, 1, seed=1))
    x[:, k // 3] *= 16  # neighbouring blocks have different scales
    x = x.to(dtype)
    q, s = vit_cuda.quantize_fp8(x)
    base.check_codes(x, q, s, 1)


@pytest.mark.parametrize("dtype", base.DTYPES)
@pytest.mark.parametrize("m,k", [(5000, 4100), (5000, 4101), (9000, 2560)])
def test_quantize_blocks(cuda, dtype, m, k):
    x = base.randn(m, k, seed=m + k) * torch.exp(base.randn(m, 1, seed=1))
    x = x.to(dtype)
    q, s = vit_cuda.quantize_fp8(x, 128)
    base.check_codes(x, q, s, 128)


@pytest.mark.parametrize("dtype", base.DTYPES)
@pytest.mark.parametrize("m,k", [
    (10000, 128), (10000, 300), (10000, 768), (10000, 771), (9600, 1024), (1300, 1500), (1300, 2048),
    (1300, 3000), (1300, 4096), (1300, 6000), (1300, 8192), (1300, 8200)])
def test_layernorm(cuda, dtype, m, k):
    base.test_layernorm_fp8(cuda, dtype, m, k)

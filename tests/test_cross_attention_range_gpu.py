"""cross_attention at the ends of its types' ranges: fp16 probabilities far below the
largest."""
import pytest
import torch

import vit_cuda
from test_cross_attention_gpu import randn, reference

pytestmark = pytest.mark.gpu

# One form each, alone and with its keys shared out: up to 16 rows per key head, up to
# 128, above (one row tile, two).
SHAPES = [(1, 1, 300, 2, 2), (1, 1, 60000, 2, 1), (2, 40, 700, 2, 2), (1, 40, 20000, 2, 1),
          (1, 300, 20000, 2, 2), (20, 300, 1000, 8, 8), (1, 600, 100, 4, 4)]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("gap", [12, 20, 26, 30])
@pytest.mark.parametrize("b,tq,tk,heads,kv_heads", SHAPES)
def test_fp16_tails(cuda, d, gap, b, tq, tk, heads, kv_heads):
    """One key's probability is 2^gap times every other's, its value is zero, and the
    output is what the others add up to. Probabilities are rounded to fp16, 2^-11 of
    themselves; below fp16's normal range by half a step, 2^-25, of a scale in which the
    largest is 2^7 at least, so 2^-32 of it: n of those against values of up to 1. The
    scores are exact, the exponents are off by 2^-23 * gap, the sums as in the other
    tests, the output by half a step, 2^-25 where it is subnormal."""
    q = torch.zeros(b, tq, heads * d, dtype=torch.float16, device="cuda")
    q[..., ::d] = 1
    k = torch.zeros(b, tk, kv_heads * d, dtype=torch.float16, device="cuda")
    k[:, tk // 2, ::d] = gap
    v = (randn(b, tk, kv_heads * d, seed=1).abs() + 0.5).clamp(max=1).half()
    v[:, tk // 2] = 0
    ln2 = 0.6931471805599453
    o = vit_cuda.cross_attention(q, k, v, ln2, heads, kv_heads)
    ref, mag, _ = reference(q, k, v, ln2, heads, kv_heads)
    rel = 2.0 ** -11 + 2 * (2.0 ** -22 + gap * 2.0 ** -22) + (tk / 4 + tk / 16 + 32) * 2.0 ** -23
    tol = rel * mag + tk * 2.0 ** -32
    tol = tol + 2.0 ** -11 * (ref + tol) + 2.0 ** -25
    off = (o.double() - ref).abs()
    assert bool((off <= tol).all()), float((off / tol).max())

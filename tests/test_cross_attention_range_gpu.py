"""cross_attention at the ends of its types' ranges: fp16 probabilities far below the
largest, and scores so large that neighbouring fp32 numbers lie whole units apart."""
import pytest
import torch

import vit_cuda
from test_cross_attention_gpu import DTYPES, operands, randn, reference

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


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [10.0, 3e4, -1e5, 1e8, -1e15, 1e30])
@pytest.mark.parametrize("b,tq,tk,heads,kv_heads", SHAPES)
def test_huge_scores(cuda, dtype, scale, b, tq, tk, heads, kv_heads):
    """Scores are exact small integers times `scale`, so all but the largest have no
    weight and the output is the mean value of the keys that share it, wherever they lie:
    off by the rounding of a probability and of the output, half a step each, and by
    fp32 sums."""
    d = 64
    g = torch.Generator(device="cuda")
    g.manual_seed(tk)
    q, _, v = operands(b, tq, tk, heads, kv_heads, d, dtype, seed=2)
    q = torch.ones_like(q)
    r = torch.randint(-40, 40, (b, tk), generator=g, device="cuda")
    k = r[:, :, None].expand(b, tk, kv_heads * d).to(dtype)
    o = vit_cuda.cross_attention(q, k, v, scale, heads, kv_heads)
    top = r == (r.amax(1, keepdim=True) if scale > 0 else r.amin(1, keepdim=True))
    w = top.double() / top.sum(1, keepdim=True)
    want = torch.einsum("bs,bse->be", w, v.double())
    mag = torch.einsum("bs,bse->be", w, v.double().abs())

    def spread(t):  # key heads to the query heads that read them, to every query
        t = t.view(b, 1, kv_heads, 1, d).expand(b, tq, kv_heads, heads // kv_heads, d)
        return t.reshape(b, tq, heads * d)

    eps = torch.finfo(dtype).eps
    tol = spread((eps / 2 + 2.0 ** -21) * mag + 4 * tk * 2.0 ** -24 * mag)
    tol = tol + eps / 2 * (spread(want).abs() + tol) + torch.finfo(dtype).tiny
    off = (o.double() - spread(want)).abs()
    assert bool((off <= tol).all()), float((off / tol).max())

"""FP8 operators (quantize_fp8, layernorm_fp8, gemm_fp8) against plain 64-bit
restatements, at sizes, strides and values where they can go wrong."""
import pytest
import torch

import vit_cuda

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=gen(seed), device="cuda").to(dtype)


def e4m3(x):
    """x (float64) rounded to the nearest e4m3 value, ties to even."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -20))).clamp(min=-6.0)
    step = torch.exp2(e - 3.0)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def blocks(x, rows):
    """x [M, K] (float64) as zero-padded blocks [mb, rows, kb, 128]."""
    m, k = x.shape
    mb, kb = -(-m // rows), -(-k // 128)
    x = torch.nn.functional.pad(x, (0, kb * 128 - k, 0, mb * rows - m))
    return x.view(mb, rows, kb, 128)


def expand(s, rows, m, k):
    """Scales [mb, kb] spread over [m, k]."""
    return s.repeat_interleave(rows, 0)[:m].repeat_interleave(128, 1)[:, :k]


def check_codes(x, q, s, rows):
    """Codes and scales of x [M, K] against the definition in 64 bits. The scale
    is one correctly rounded division. The quotient 448 x / a is rounded to fp32
    before it is rounded to e4m3 (and 448 x as well when x is fp32: three half
    steps of 2^-24), so a code may only differ from the exact one's where the
    quotient lies within 2^-22 of midway; for 16-bit x a quotient of such short
    numbers is midway or further than that from it, and codes are exact."""
    m, k = x.shape
    a = blocks(x.double(), rows).abs().amax(dim=(1, 3)).clamp(min=float(torch.tensor(1e-30)))
    torch.testing.assert_close(s, (a / 448.0).float(), rtol=0, atol=0)
    quot = x.double() * 448.0 / expand(a, rows, m, k)
    if x.dtype != torch.float32:
        assert torch.equal(q.double(), e4m3(quot))
    lo = e4m3(quot * (1 - 2.0 ** -22))
    hi = e4m3(quot * (1 + 2.0 ** -22))
    assert bool(((q.double() >= torch.minimum(lo, hi)) & (q.double() <= torch.maximum(lo, hi))).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 127), (3, 128), (5, 129), (197, 768), (33, 1000),
                                 (130, 257), (1, 8192), (700, 36)])
@pytest.mark.parametrize("rows", [1, 128])
def test_quantize(cuda, dtype, m, k, rows):
    x = (randn(m, k, seed=m + k) * torch.exp(randn(m, 1, seed=1))).to(dtype)
    x[:, k // 2] *= 16
    q, s = vit_cuda.quantize_fp8(x, rows)
    assert q.shape == x.shape and q.dtype == torch.float8_e4m3fn
    assert s.shape == (-(-m // rows), -(-k // 128))
    assert q.stride(0) % 16 == 0
    check_codes(x, q, s, rows)


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_midpoints(cuda, dtype):
    """A power of two as the largest magnitude puts many quotients midway."""
    x = torch.arange(1, 257, device="cuda", dtype=torch.float32).repeat(4, 1)
    x = (x * torch.tensor([[1.0], [2.0 ** -9], [-4.0], [0.25]], device="cuda")).to(dtype)
    q, s = vit_cuda.quantize_fp8(x)
    check_codes(x, q, s, 1)


@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_special_values(cuda, rows):
    """Zeros, values below the floor, the largest finite ones, infinities and
    NaN: a bad value marks its own block and no other."""
    x = randn(384, 512, seed=3)
    x[0, :128] = 0
    x[130, 128:256] = 1e-38
    x[131, :] = 3.4e38
    q, s = vit_cuda.quantize_fp8(x, rows)
    v = q.double() * expand(s.double(), rows, 384, 512)
    assert bool(v.isfinite().all())
    if rows == 1:
        assert bool((v[0, :128] == 0).all()) and bool((v[130, 128:256] == 0).all())
        # 3.4e38 is its blocks' maximum: code 448 times the scale, off by the scale's half step
        assert bool(((v[131] - x[131].double()).abs() <= 2.0 ** -23 * 3.4e38).all())
    for bad in (float("nan"), float("inf"), float("-inf")):
        y = randn(384, 512, seed=4)
        clean_q, clean_s = vit_cuda.quantize_fp8(y, rows)
        y[140, 200] = bad
        q, s = vit_cuda.quantize_fp8(y, rows)
        v = q.double() * expand(s.double(), rows, 384, 512)
        hit = torch.zeros(384, 512, dtype=torch.bool, device="cuda")
        hit[(slice(140, 141) if rows == 1 else slice(128, 256)), 128:256] = True
        assert bool(v[hit].isnan().all())
        assert torch.equal(q.view(torch.uint8)[~hit], clean_q.view(torch.uint8)[~hit])
        assert int((s != clean_s).sum()) == 1


@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_strided_and_batched(cuda, rows):
    base = randn(200, 400, seed=5, dtype=torch.bfloat16)
    for x in (base[:, 8:264], base[:, 3:260], base.t(), base[::2], base[:1].expand(200, 400)):
        q, s = vit_cuda.quantize_fp8(x, rows)
        check_codes(x, q, s, rows)
    if rows == 1:
        x = randn(3, 7, 200, seed=6)
        q, s = vit_cuda.quantize_fp8(x)
        assert q.shape == x.shape and s.shape == (3, 7, 2)
        check_codes(x.view(21, 200), q.reshape(21, 200), s.view(21, 2), 1)
    q, s = vit_cuda.quantize_fp8(base[:0], rows)
    assert q.shape == (0, 400) and s.shape == (0, 4)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (4, 100), (3, 256), (197, 768), (50, 1000), (5, 1536),
                                 (2, 8192), (3, 8200), (9, 10001)])
def test_layernorm_fp8(cuda, dtype, m, k):
    """Each value against the 64-bit LayerNorm: half a code step (2^-4 of the
    value, or of the smallest normal code where it is subnormal: 2^-10 / 448 of
    the block's maximum) plus the fp32 arithmetic. That is sums of k values held
    to k/32 sequential steps of 2^-24 and a dozen roundings, on values of up to
    the row's largest |x - mean| * rstd * |gamma| + |beta|."""
    x = (randn(m, k, seed=k) * 2 + 0.5).to(dtype)
    g, b = torch.exp(0.3 * randn(k, seed=7)), 0.2 * randn(k, seed=8)
    q, s = vit_cuda.layernorm_fp8(x, g, b, 1e-6)
    assert q.shape == x.shape and s.shape == (m, -(-k // 128)) and q.stride(0) % 16 == 0
    xd = x.double()
    c = xd - xd.mean(1, keepdim=True)
    y = c / torch.sqrt((c * c).mean(1, keepdim=True) + 1e-6) * g.double() + b.double()
    a = blocks(y, 1).abs().amax(dim=(1, 3))
    # one column: x - mean is exactly zero only in 64 bits; fp32's mean of one value is exact too
    arith = (k / 32 + 16) * 2.0 ** -24 * (y.abs().amax(1, keepdim=True) + b.double().abs().max() + 1)
    got = q.double() * expand(s.double(), 1, m, k)
    bound = 2.0 ** -4 * y.abs() + expand(a, 1, m, k) * 2.0 ** -10 / 448 + 2 * arith
    assert bool(((got - y).abs() <= bound).all())
    assert bool(((s.double() * 448 - a).abs() <= arith + 2.0 ** -23 * a).all())


def test_layernorm_fp8_is_quantized_layernorm(cuda):
    """The fused operator against its two steps: both LayerNorms are fp32, so the
    scales agree to the arithmetic and the values to a code step."""
    x = randn(2, 197, 768, seed=9)
    g, b = torch.exp(0.3 * randn(768, seed=10)), 0.2 * randn(768, seed=11)
    q, s = vit_cuda.layernorm_fp8(x, g, b, 1e-6)
    q2, s2 = vit_cuda.quantize_fp8(vit_cuda.layernorm_forward(x, g, b, 1e-6))
    torch.testing.assert_close(s, s2, rtol=2.0 ** -18, atol=0)
    assert float((q.float() != q2.float()).double().mean()) < 1e-3
    with_nan = x.clone()
    with_nan[1, 5, 3] = float("nan")
    q3, s3 = vit_cuda.layernorm_fp8(with_nan, g, b, 1e-6)
    assert bool(s3[1, 5].isnan().all()) and bool(q3[1, 5].float().isnan().all())
    s3[1, 5] = s[1, 5]
    assert torch.equal(s3, s)


# ---------------------------------------------------------------- gemm
def operands(m, k, n, seed=0):
    x = randn(m, k, seed=seed) * torch.exp(0.5 * randn(m, 1, seed=seed + 1))
    w = randn(n, k, seed=seed + 2) * torch.exp(0.3 * randn(n, 1, seed=seed + 3)) * k ** -0.5
    return (*vit_cuda.quantize_fp8(x), *vit_cuda.quantize_fp8(w, 128))


def check_gemm(y, xq, xs, wq, ws, bias=None, residual=None, gelu=False, sample=None):
    """Against the 64-bit product of the dequantised operands. Products of codes
    are exact; the tensor core sums 128 of them in four steps of 32 aligned
    terms, each term cut to 24 bits or more below the largest, and adding the
    four: at most 36 steps of 2^-24 of the sum of magnitudes S. Two scales
    multiplied, one FMA per block, bias and residual: ceil(K/128) + 4 more. GELU's
    slope is at most 1.13, its own error 2e-6 of the result and 2.4e-7. The
    output's rounding is half a step."""
    m, k = xq.shape
    n = wq.shape[0]
    rows = torch.arange(m, device="cuda") if sample is None else sample
    x = xq.view(torch.uint8)[rows].view(torch.float8_e4m3fn).double() * expand(xs.double()[rows], 1, len(rows), k)
    w = wq.double() * expand(ws.double(), 128, n, k)
    ref, S = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        ref, S = ref + bias.double(), S + bias.double().abs()
    tol = (36 + -(-k // 128) + 4) * 2.0 ** -24 * S
    if gelu:
        ref = ref * 0.5 * torch.erfc(-ref * 0.5 ** 0.5)
        tol = 1.13 * tol + 2e-6 * ref.abs() + 2.4e-7
    if residual is not None:
        r = residual[rows].double()
        ref = ref + r
        tol = tol + 2.0 ** -24 * (ref.abs() + r.abs())
    tol = tol + torch.finfo(y.dtype).eps / 2 * (ref.abs() + tol) + torch.finfo(y.dtype).tiny
    bad = ((y[rows].double() - ref).abs() > tol)
    assert not bool(bad.any()), float(((y[rows].double() - ref).abs() / tol).max())


@pytest.mark.parametrize("m,k,n", [
    (1, 1, 1), (1, 128, 16), (3, 17, 5), (8, 4096, 1024), (16, 130, 130), (127, 256, 129),
    (128, 768, 768), (129, 1000, 100), (197, 768, 2304), (300, 2176, 64), (40, 8192, 24),
    (2600, 384, 1000), (2573, 129, 1001), (1280, 640, 4096), (5000, 16, 520), (257, 200, 16384)])
@pytest.mark.parametrize("out", DTYPES)
def test_gemm(cuda, m, k, n, out):
    ops = operands(m, k, n, seed=m)
    check_gemm(vit_cuda.gemm_fp8(*ops, out_dtype=out), *ops)


@pytest.mark.parametrize("m,k,n", [(1, 256, 64), (50, 300, 200), (197, 640, 777), (2600, 256, 1000),
                                   (2561, 140, 1003)])
@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("bias,gelu,residual", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 1)])
def test_gemm_epilogue(cuda, m, k, n, out, bias, gelu, residual):
    ops = operands(m, k, n, seed=n)
    b = randn(n, seed=20) if bias else None
    r = randn(m, n, seed=21, dtype=out) if residual else None
    y = vit_cuda.gemm_fp8(*ops, b, residual=r, gelu=bool(gelu), out_dtype=out)
    check_gemm(y, *ops, b, r, bool(gelu))


@pytest.mark.parametrize("m,n", [(130, 96), (2600, 1000)])
def test_gemm_strided_operands(cuda, m, n):
    """Column slices of wider codes, scales and residuals; unaligned ones are
    copied, not misread. Rows beside the slices stay as they were."""
    k = 256
    xq, xs, wq, ws = operands(m, k, n, seed=30)
    wide = torch.zeros(m, k + 64, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    for off in (0, 16, 7):
        part = wide[:, off:off + k]
        part.view(torch.uint8).copy_(xq.view(torch.uint8))
        scales = torch.zeros(m, 5, device="cuda")
        scales[:, 1:3] = xs
        res = randn(m, n + 9, seed=31, dtype=torch.bfloat16)
        for r in (res[:, :n], res[:, 3:3 + n]):
            y = vit_cuda.gemm_fp8(part, scales[:, 1:3], wq, ws, residual=r, out_dtype=torch.bfloat16)
            check_gemm(y, xq, xs, wq, ws, residual=r)


def test_gemm_batched_and_empty(cuda):
    xq, xs, wq, ws = operands(60, 100, 40, seed=32)
    ref = vit_cuda.gemm_fp8(xq, xs, wq, ws)
    buf = torch.zeros(3, 20, 112, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    buf[..., :100].view(torch.uint8).copy_(xq.view(torch.uint8).reshape(3, 20, 100))
    for x3 in (buf[..., :100], buf[..., :100].contiguous()):
        y = vit_cuda.gemm_fp8(x3, xs.view(3, 20, 1), wq, ws)
        assert y.shape == (3, 20, 40) and torch.equal(y.view(60, 40), ref)
    assert vit_cuda.gemm_fp8(xq[:0], xs[:0], wq, ws).shape == (0, 40)
    assert vit_cuda.gemm_fp8(xq, xs, wq[:0], ws[:0]).shape == (60, 0)


@pytest.mark.parametrize("m,n", [(130, 200), (2600, 1000)])
def test_gemm_nan_stays_in_its_row_and_column(cuda, m, n):
    xq, xs, wq, ws = operands(m, 256, n, seed=33)
    ref = vit_cuda.gemm_fp8(xq, xs, wq, ws)
    xq.view(torch.uint8)[70, 5] = 0x7F
    wq.view(torch.uint8)[140, 200] = 0xFF
    y = vit_cuda.gemm_fp8(xq, xs, wq, ws)
    nan = torch.zeros(m, n, dtype=torch.bool, device="cuda")
    nan[70], nan[:, 140] = True, True
    assert bool(y[nan].isnan().all()) and torch.equal(y[~nan], ref[~nan])


def test_gemm_same_result_every_time(cuda):
    ops = operands(24, 4096, 512, seed=34)
    ref = vit_cuda.gemm_fp8(*ops)
    for _ in range(5):
        assert torch.equal(vit_cuda.gemm_fp8(*ops), ref)


def test_gemm_output_past_32_bit_offsets(cuda):
    m, k, n = 70000, 32, 32768
    ops = operands(m, k, n, seed=35)
    y = vit_cuda.gemm_fp8(*ops, out_dtype=torch.bfloat16)
    sample = torch.tensor([0, 1, 32767, 65535, 65536, 69887, 69999], device="cuda")
    check_gemm(y, *ops, sample=sample)


def test_other_stream_and_graph(cuda):
    """quantise -> product -> quantise -> product on a side stream, then captured
    and replayed on new inputs: the same bits as eager calls."""
    w1, w2 = randn(512, 256, seed=40), randn(256, 512, seed=41)
    wq1, wq2 = vit_cuda.quantize_fp8(w1 * 0.06, 128), vit_cuda.quantize_fp8(w2 * 0.04, 128)
    g, b = torch.ones(256, device="cuda"), torch.zeros(256, device="cuda")
    bias = randn(512, seed=42)

    def mlp(x):
        h = vit_cuda.gemm_fp8(*vit_cuda.layernorm_fp8(x, g, b, 1e-6), *wq1, bias, gelu=True,
                              out_dtype=torch.bfloat16)
        return vit_cuda.gemm_fp8(*vit_cuda.quantize_fp8(h), *wq2, residual=x)

    xs = [randn(77, 256, seed=50 + i) for i in range(3)]
    refs = [mlp(x) for x in xs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        outs = [mlp(x) for x in xs]
    side.synchronize()
    assert all(torch.equal(o, r) for o, r in zip(outs, refs))
    static = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mlp(static)
    for x, r in zip(xs, refs):
        static.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, r)


def test_compiled(cuda):
    """torch.compile traces the operators without a graph break."""
    wq, ws = vit_cuda.quantize_fp8(randn(96, 100, seed=60), 128)
    g, b = torch.ones(100, device="cuda"), torch.zeros(100, device="cuda")

    def f(x):
        q, s = vit_cuda.quantize_fp8(x)
        q2, s2 = vit_cuda.layernorm_fp8(x, g, b, 1e-6)
        return vit_cuda.gemm_fp8(q, s, wq, ws), vit_cuda.gemm_fp8(q2, s2, wq, ws, gelu=True)

    x = randn(30, 100, seed=61)
    for got, ref in zip(torch.compile(f, fullgraph=True, backend="aot_eager")(x), f(x)):
        assert torch.equal(got, ref)


def test_refusals(cuda):
    x = randn(8, 256)
    q, s = vit_cuda.quantize_fp8(x)
    wq, ws = vit_cuda.quantize_fp8(randn(130, 256, seed=1), 128)
    ok = dict(X=q, X_scale=s, W=wq, W_scale=ws)

    def bad(match, **kw):
        with pytest.raises(RuntimeError, match=match):
            vit_cuda.gemm_fp8(**{**ok, **kw})

    bad("float8_e4m3fn", X=x)
    bad("float8_e4m3fn", W=wq.view(torch.uint8))
    bad("float32", X_scale=s.half())
    bad("X must be", X=q.view(2, 2, 2, 256))
    bad("match K", W=wq[:, :128])
    bad("X_scale must be", X_scale=s[:, :1])
    bad("W_scale must be", W_scale=ws[:1])
    bad("bias size", B=randn(131))
    bad("B must be float32", B=randn(130).half())
    bad("out_dtype", residual=randn(8, 130).half())
    bad("residual shape", residual=randn(8, 129))
    bad("out_dtype", out_dtype=torch.float64)
    bad("same CUDA device|CUDA", X_scale=s.cpu())
    bad("at least 1", X=q[:, :0], W=wq[:, :0])
    with pytest.raises(RuntimeError, match="block_rows"):
        vit_cuda.quantize_fp8(x, 64)
    with pytest.raises(RuntimeError, match="2D"):
        vit_cuda.quantize_fp8(x.view(2, 4, 256), 128)
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        vit_cuda.quantize_fp8(x.double())
    with pytest.raises(RuntimeError, match="K >= 1"):
        vit_cuda.quantize_fp8(x[:, :0])
    with pytest.raises(RuntimeError, match="gamma size"):
        vit_cuda.layernorm_fp8(x, randn(255), randn(256), 1e-6)
    with pytest.raises(RuntimeError, match="beta must be float32"):
        vit_cuda.layernorm_fp8(x, randn(256), randn(256).half(), 1e-6)

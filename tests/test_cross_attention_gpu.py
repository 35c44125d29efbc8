"""cross_attention against a plain 64-bit restatement, at the lengths, groups,
strides, masks and values where it can go wrong."""
import math

import pytest
import torch

import vit_cuda

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


def randn(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def operands(b, tq, tk, heads, kv_heads, d, dtype, seed=0):
    kv = randn(b, tk, 2 * kv_heads * d, seed=seed + 1, dtype=dtype)
    e = kv_heads * d
    return randn(b, tq, heads * d, seed=seed, dtype=dtype, scale=1.5), kv[..., :e], kv[..., e:]


def reference(q, k, v, scale, heads, kv_heads, lens=None):
    """(o, sum_s p |v|, largest |q| |k| scale sum) in 64 bits; images without keys are zeros."""
    b, tq, _ = q.shape
    tk, d, g = k.shape[1], q.shape[2] // heads, heads // kv_heads
    o = torch.zeros(b, tq, heads, d, dtype=torch.float64, device=q.device)
    mag, arg = torch.zeros_like(o), torch.zeros(b, tq, heads, dtype=torch.float64, device=q.device)
    for i in range(b):
        n = tk if lens is None else max(0, min(tk, int(lens[i])))
        if n == 0:
            continue
        for h in range(heads):
            j = h // g
            qh = q[i, :, h * d:(h + 1) * d].double()
            kh = k[i, :n, j * d:(j + 1) * d].double()
            vh = v[i, :n, j * d:(j + 1) * d].double()
            p = torch.softmax(qh @ kh.t() * scale, dim=1)
            o[i, :, h] = p @ vh
            mag[i, :, h] = p @ vh.abs()
            arg[i, :, h] = (qh.abs() @ kh.abs().t()).amax(1) * abs(scale)
    return o.view(b, tq, -1), mag.view(b, tq, -1), arg[..., None].expand_as(o).reshape(b, tq, -1)


def check(o, q, k, v, scale, heads, kv_heads, lens=None):
    """A probability is off by its rounding to the type (half a step, and for fp16
    half the smallest step where it is subnormal, against a sum of at least 1),
    by its argument (fp32 sums of D products in 8 steps of 16 aligned terms:
    (8 + 16) half steps of 2^-23 of the magnitudes, and two roundings) and by
    ex2.approx (2^-22). The normalising sum has the last two and n / 4 additions.
    The products with V are summed in fp32 in steps of 16 keys, cut toward zero:
    (n / 16 + 16) steps of 2^-23. All of it scales sum p |v|. The output is rounded
    by half a step."""
    ref, mag, arg = reference(q, k, v, scale, heads, kv_heads, lens)
    n, eps = k.shape[1], torch.finfo(o.dtype).eps
    rel = eps / 2 + 2 * (26 * 2.0 ** -23 * arg + 2.0 ** -22) + (n / 4 + n / 16 + 32) * 2.0 ** -23
    tol = rel * mag
    if o.dtype == torch.float16:
        tol = tol + 2.0 ** -25 * n * v.double().abs().nan_to_num(0, 0, 0).amax()
    tol = tol + eps / 2 * (ref.abs() + tol) + torch.finfo(o.dtype).tiny
    off = (o.double() - ref).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,tq,tk,heads,kv_heads", [
    (1, 1, 1, 1, 1), (2, 1, 5, 4, 4), (3, 1, 197, 12, 12), (2, 1, 1000, 8, 2), (1, 1, 5000, 6, 1),
    (2, 3, 128, 6, 2), (1, 5, 129, 7, 1), (2, 16, 255, 4, 4), (2, 17, 256, 8, 1), (1, 61, 577, 12, 12),
    (1, 128, 64, 2, 2), (1, 129, 300, 2, 2), (2, 300, 385, 3, 3), (1, 257, 1100, 8, 2),
    (1, 700, 130, 10, 2), (1, 20, 200, 65, 1), (1, 3, 200, 128, 1), (1, 2, 130, 130, 1),
    (40, 33, 50, 4, 4), (1, 2000, 2000, 4, 1)])
def test_lengths_and_groups(cuda, dtype, d, b, tq, tk, heads, kv_heads):
    q, k, v = operands(b, tq, tk, heads, kv_heads, d, dtype, seed=tq + tk)
    scale = d ** -0.5
    o = vit_cuda.cross_attention(q, k, v, scale, heads, kv_heads)
    assert o.shape == q.shape and o.dtype == dtype and o.is_contiguous()
    check(o, q, k, v, scale, heads, kv_heads)


@pytest.mark.parametrize("tq", [1, 4, 40, 150, 300])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -3.0e38, 3.0e38])
def test_keys_past_the_length_are_never_seen(cuda, tq, d, bad):
    """Lengths of every kind; what lies past them is NaN, infinite or the type's
    largest value, in keys and values alike."""
    heads, kv_heads, tk = 4, 2, 420
    lens = torch.tensor([0, 1, 16, 100, 127, 128, 129, 256, 300, 384, 419, 420, 421, -5, 10 ** 9],
                        dtype=torch.int32, device="cuda")
    b = len(lens)
    q, k, v = operands(b, tq, tk, heads, kv_heads, d, torch.bfloat16, seed=3)
    clean_k, clean_v = k.clone(), v.clone()
    for i, n in enumerate(lens.clamp(0, tk).tolist()):
        k[i, n:], v[i, n:] = bad, bad
    o = vit_cuda.cross_attention(q, k, v, d ** -0.5, heads, kv_heads, lens)
    check(o, q, clean_k, clean_v, d ** -0.5, heads, kv_heads, lens)
    assert bool((o[0] == 0).all()) and bool((o[13] == 0).all())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("tq,heads,kv_heads", [(1, 8, 2), (1, 1, 1), (3, 4, 4), (1, 16, 1), (20, 4, 2)])
@pytest.mark.parametrize("lens", [[0, 9000, 3, 4097, 17], [5, 0, 0, 0, 0], [0, 0, 0, 0, 0],
                                  [9000, 9000, 8999, 1, 9000], [0, 0, 16, 33, 2000]])
def test_long_ragged_lengths(cuda, d, tq, heads, kv_heads, lens):
    """Work that is cut evenly whatever the lengths: key heads shared by several
    CTAs, CTAs with several key heads, fewer steps than CTAs, empty images first,
    last and between."""
    lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q, k, v = operands(5, tq, 9000, heads, kv_heads, d, torch.bfloat16, seed=50)
    o = vit_cuda.cross_attention(q, k, v, d ** -0.5, heads, kv_heads, lens)
    check(o, q, k, v, d ** -0.5, heads, kv_heads, lens)
    assert bool((o[lens == 0] == 0).all())


def test_many_images(cuda):
    """More images than a warp scans at once."""
    lens = torch.arange(100, dtype=torch.int32, device="cuda") * 97 % 3001
    q, k, v = operands(100, 1, 3000, 4, 1, 64, torch.float16, seed=51)
    check(vit_cuda.cross_attention(q, k, v, 0.125, 4, 1, lens), q, k, v, 0.125, 4, 1, lens)


@pytest.mark.parametrize("tq", [1, 40, 300])
def test_bad_values_within_the_length(cuda, tq):
    """A NaN key or query makes its rows NaN, a NaN value its column; other
    images and heads keep theirs."""
    b, heads, d, tk = 2, 4, 64, 300
    q, k, v = operands(b, tq, tk, heads, 2, d, torch.float16, seed=5)
    ref = vit_cuda.cross_attention(q, k, v, 0.125, heads, 2)
    k2, v2, q2 = k.clone(), v.clone(), q.clone()
    k2[0, 200, 70] = float("nan")  # key head 1: query heads 2, 3
    o = vit_cuda.cross_attention(q, k2, v, 0.125, heads, 2)
    assert bool(o[0, :, 2 * d:].isnan().all())
    assert torch.equal(o[0, :, :2 * d], ref[0, :, :2 * d]) and torch.equal(o[1], ref[1])
    v2[1, 299, 3] = float("nan")  # key head 0, column 3: query heads 0, 1
    o = vit_cuda.cross_attention(q, k, v2, 0.125, heads, 2)
    nan = torch.zeros_like(o, dtype=torch.bool)
    nan[1, :, [3, d + 3]] = True
    assert bool(o[nan].isnan().all()) and torch.equal(o[~nan], ref[~nan])
    q2[0, 0, 0] = float("nan")
    o = vit_cuda.cross_attention(q2, k, v, 0.125, heads, 2)
    nan = torch.zeros_like(o, dtype=torch.bool)
    nan[0, 0, :d] = True
    assert bool(o[nan].isnan().all()) and torch.equal(o[~nan], ref[~nan])


@pytest.mark.parametrize("tq", [1, 40, 300])
@pytest.mark.parametrize("scale", [0.0, -0.2, 2.0, -3.0, 1e-4])
def test_scales(cuda, tq, scale):
    q, k, v = operands(2, tq, 333, 4, 4, 64, torch.bfloat16, seed=7)
    check(vit_cuda.cross_attention(q, k, v, scale, 4), q, k, v, scale, 4, 4)


@pytest.mark.parametrize("tq", [1, 40, 300])
def test_growing_scores(cuda, tq):
    """Scores that grow by tens from key tile to key tile: every tile's maximum
    replaces the one before, so each rescales what was summed; and the reverse."""
    d, tk = 64, 1200
    q = randn(1, tq, d, seed=8, dtype=torch.float16).abs() + 0.5
    k = randn(1, tk, d, seed=9, dtype=torch.float16, scale=0.05)
    ramp = (torch.arange(tk, device="cuda") // 64).to(torch.float16)[None, :, None]
    v = randn(1, tk, d, seed=10, dtype=torch.float16)
    for kk in (k + 0.5 * ramp, k - 0.5 * ramp, k + 0.5 * (ramp % 5)):
        check(vit_cuda.cross_attention(q, kk, v, 0.125, 1), q, kk, v, 0.125, 1, 1)


@pytest.mark.parametrize("tq", [1, 30, 200])
def test_one_key_is_its_value(cuda, tq):
    q, k, v = operands(3, tq, 1, 8, 2, 128, torch.bfloat16, seed=11)
    o = vit_cuda.cross_attention(q, k, v, 0.1, 8, 2).view(3, tq, 8, 128)
    want = v.view(3, 1, 2, 1, 128).expand(3, tq, 2, 4, 128).reshape(3, tq, 8, 128)
    assert torch.equal(o, want)


@pytest.mark.parametrize("tq", [1, 24, 260])
def test_strides(cuda, tq):
    """Column ranges, transposed head orders, expanded batches and unaligned
    starts give what contiguous copies give."""
    b, heads, kv_heads, d, tk = 2, 4, 2, 64, 200
    q, k, v = operands(b, tq, tk, heads, kv_heads, d, torch.bfloat16, seed=12)
    ref = vit_cuda.cross_attention(q.contiguous(), k.contiguous(), v.contiguous(), 0.125, heads,
                                   kv_heads)

    def same(q, k, v):
        assert torch.equal(vit_cuda.cross_attention(q, k, v, 0.125, heads, kv_heads), ref)

    same(q, k, v)
    wide = torch.zeros(b, tq, heads * d + 24, dtype=q.dtype, device="cuda")
    for off in (8, 3):
        view = wide[..., off:off + heads * d]
        view.copy_(q)
        same(view, k, v)
    same(q.transpose(0, 1).contiguous().transpose(0, 1), k.transpose(0, 1).contiguous().transpose(0, 1), v)
    same(q, k.transpose(1, 2).contiguous().transpose(1, 2), v)
    one_k, one_v = k[:1].expand(b, -1, -1), v[:1].expand(b, -1, -1)
    assert torch.equal(vit_cuda.cross_attention(q, one_k, one_v, 0.125, heads, kv_heads),
                       vit_cuda.cross_attention(q, one_k.contiguous(), one_v.contiguous(), 0.125,
                                                heads, kv_heads))
    rows = torch.zeros(b, 2 * tk, kv_heads * d, dtype=q.dtype, device="cuda")
    rows[:, ::2] = k
    same(q, rows[:, ::2], v)


def test_empty(cuda):
    q, k, v = operands(2, 3, 7, 2, 2, 64, torch.bfloat16)
    assert vit_cuda.cross_attention(q[:0], k[:0], v[:0], 0.1, 2).shape == (0, 3, 128)
    assert vit_cuda.cross_attention(q[:, :0], k, v, 0.1, 2).shape == (2, 0, 128)
    assert bool((vit_cuda.cross_attention(q, k[:, :0], v[:, :0], 0.1, 2) == 0).all())


@pytest.mark.parametrize("tq", [1, 9, 64])
def test_same_result_every_time_and_in_any_batch(cuda, tq):
    q, k, v = operands(1, tq, 3000, 4, 2, 128, torch.bfloat16, seed=13)
    ref = vit_cuda.cross_attention(q, k, v, 0.1, 4, 2)
    for _ in range(5):
        assert torch.equal(vit_cuda.cross_attention(q, k, v, 0.1, 4, 2), ref)


@pytest.mark.parametrize("tq", [1, 2])
def test_keys_past_32_bit_offsets(cuda, tq):
    """The last image's keys start beyond 2^31 elements."""
    heads, d, tk, b = 8, 128, 65536, 33
    q = randn(b, tq, heads * d, seed=14, dtype=torch.bfloat16)
    k = torch.zeros(b, tk, heads * d, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    k[-1] = randn(tk, heads * d, seed=15, dtype=torch.bfloat16)
    v[-1] = randn(tk, heads * d, seed=16, dtype=torch.bfloat16)
    o = vit_cuda.cross_attention(q, k, v, 0.08, heads)
    assert bool((o[:-1] == 0).all())
    check(o[-1:], q[-1:], k[-1:], v[-1:], 0.08, heads, heads)


@pytest.mark.parametrize("tq", [1, 50])
def test_other_stream_and_graph(cuda, tq):
    sets = [operands(2, tq, 600, 8, 2, 64, torch.bfloat16, seed=20 + i) for i in range(3)]
    lens = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([600, 17], [0, 300], [128, 600])]
    refs = [vit_cuda.cross_attention(*s, 0.125, 8, 2, n) for s, n in zip(sets, lens)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        outs = [vit_cuda.cross_attention(*s, 0.125, 8, 2, n) for s, n in zip(sets, lens)]
    side.synchronize()
    assert all(torch.equal(o, r) for o, r in zip(outs, refs))
    q, k, v = (t.clone() for t in sets[0])
    n = lens[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = vit_cuda.cross_attention(q, k, v, 0.125, 8, 2, n)
    for s, ln, r in zip(sets, lens, refs):
        for dst, src in zip((q, k, v, n), (*s, ln)):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, r)


def test_compiled(cuda):
    q, k, v = operands(2, 5, 40, 4, 2, 64, torch.bfloat16, seed=30)
    f = torch.compile(lambda q, k, v: vit_cuda.cross_attention(q, k, v, 0.125, 4, 2), fullgraph=True,
                      backend="aot_eager")
    assert torch.equal(f(q, k, v), vit_cuda.cross_attention(q, k, v, 0.125, 4, 2))


def test_refusals(cuda):
    q, k, v = operands(2, 5, 40, 4, 2, 64, torch.bfloat16)

    def bad(match, q=q, k=k, v=v, heads=4, kv_heads=2, lens=None):
        with pytest.raises(RuntimeError, match=match):
            vit_cuda.cross_attention(q, k, v, 0.125, heads, kv_heads, lens)

    bad("float16 or bfloat16", q=q.float(), k=k.float(), v=v.float())
    bad("same type", k=k.half())
    bad("Q must be", q=q[0])
    bad("K must be", k=k[:1], v=v[:1])
    bad("V shape", v=v[:, :39])
    bad("multiple of kv_heads", kv_heads=3)
    bad("multiple of kv_heads", heads=0)
    bad("D 64 or 128", heads=8)
    bad("D 64 or 128", q=q[..., :255])
    bad("kv_heads \\* D", kv_heads=4)
    bad("int32", lens=torch.tensor([1, 2], device="cuda"))
    bad("kv_lens must be", lens=torch.tensor([1], dtype=torch.int32, device="cuda"))
    bad("CUDA", k=k.cpu())


def test_decoder_layer(cuda):
    """The operators as a decoder's cross-attention layer runs them: the image
    tokens' keys and values are projected once in FP8; a prompt and then single
    tokens go through LayerNorm + FP8 query projection, attention, FP8 output
    projection and the residual. Against the same layer in 64 bits on the
    dequantised weights: the tokens, the LayerNorm and the attention output are
    rounded to e4m3, each by at most half a step (2^-4 of a value), whose effects
    on the sums are independent: sqrt(3) * 2^-4 in the 2-norm, and the first two
    enter through scores of order 1 as well; the bf16 roundings (2^-9) and fp32
    sums are far below. Held to 2^-3."""
    b, tk, e, heads, d = 3, 197, 256, 4, 64
    tokens, x = randn(b, tk, e, seed=40), randn(b, 12, e, seed=41)
    wq, wkv, wo = (randn(n, e, seed=42 + i) * e ** -0.5 for i, n in enumerate((e, 2 * e, e)))
    gamma, beta, bias = torch.exp(0.2 * randn(e, seed=46)), 0.1 * randn(e, seed=47), 0.1 * randn(e, seed=48)
    lens = torch.tensor([197, 60, 0], dtype=torch.int32, device="cuda")
    qw, kvw, ow = (vit_cuda.quantize_fp8(w, 128) for w in (wq, wkv, wo))

    def full(ws, n):
        return ws[0].double() * ws[1].double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :e]

    kv = vit_cuda.gemm_fp8(*vit_cuda.quantize_fp8(tokens), *kvw, out_dtype=torch.bfloat16)

    def layer(x):
        q = vit_cuda.gemm_fp8(*vit_cuda.layernorm_fp8(x, gamma, beta, 1e-6), *qw,
                              out_dtype=torch.bfloat16)
        a = vit_cuda.cross_attention(q, kv[..., :e], kv[..., e:], d ** -0.5, heads, kv_lens=lens)
        return vit_cuda.gemm_fp8(*vit_cuda.quantize_fp8(a), *ow, bias, residual=x)

    prompt = layer(x)
    steps = torch.cat([layer(x[:, t:t + 1]) for t in range(12)], dim=1)
    assert vit_cuda.device_error() == 0

    xd = x.double()
    c = xd - xd.mean(-1, keepdim=True)
    y = c / torch.sqrt((c * c).mean(-1, keepdim=True) + 1e-6) * gamma.double() + beta.double()
    kvd = tokens.double() @ full(kvw, 2 * e).t()
    att, _, _ = reference(y @ full(qw, e).t(), kvd[..., :e], kvd[..., e:], d ** -0.5, heads, heads, lens)
    delta = att @ full(ow, e).t() + bias.double()
    for got in (prompt, steps):
        off = got.double() - xd - delta
        for i in range(b):
            assert float(off[i].norm() / delta[i].norm()) < 2.0 ** -3
    assert torch.equal(prompt[2], (x[2] + bias))  # no keys: the residual and the bias alone

"""Guard bands around every buffer that the serving operators' C entry points write
(codes, scales, products, attention outputs and workspaces), at sizes where every tail
is partial; rows further apart than they are wide; a residual in place."""
import pytest
import torch

import test_cross_attention_gpu as cross
import test_fp8_gpu as fp8
from test_guard_band_gpu import bands_intact, guarded, stream

pytestmark = pytest.mark.gpu

TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
FILL = {torch.float32: 1234.5, torch.float16: 1234.0, torch.bfloat16: 1232.0}


def guard(n, device, dtype):
    fill = FILL.get(dtype, 165)
    buf, inside = guarded(n, device, dtype, fill)
    return lambda: bands_intact(buf, fill), inside


@pytest.mark.parametrize("dtype", fp8.DTYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (3, 129), (130, 257), (33, 1000), (5000, 390), (700, 36),
                                 (20, 8201)])
@pytest.mark.parametrize("rows", [1, 128, "norm"])
def test_quantisers(vlib, cuda, dtype, m, k, rows):
    x = fp8.randn(m, k + 3, seed=k, dtype=dtype)[:, :k]
    ldq = (k + 15) // 16 * 16 + 16
    block = rows if rows == 128 else 1
    mb, kb = -(-m // block), -(-k // 128)
    q_ok, q = guard((m - 1) * ldq + (k + 15) // 16 * 16, cuda, torch.uint8)
    s_ok, s = guard(mb * kb, cuda, torch.float32)
    if rows == "norm":
        g, b = fp8.randn(k, seed=1), fp8.randn(k, seed=2)
        vlib.check(vlib.lib.vitb200_layernorm_fp8(
            x.data_ptr(), TYPES[dtype], m, k, x.stride(0), g.data_ptr(), b.data_ptr(), 1e-6,
            q.data_ptr(), ldq, s.data_ptr(), stream()), "layernorm_fp8")
    else:
        vlib.check(vlib.lib.vitb200_quantize_fp8(
            x.data_ptr(), TYPES[dtype], m, k, x.stride(0), rows, q.data_ptr(), ldq, s.data_ptr(),
            stream()), "quantize_fp8")
    torch.cuda.synchronize()
    assert q_ok() and s_ok()
    assert not bool((s == FILL[torch.float32]).any())
    # between the rows: the last 16-byte chunk of each belongs to it, the rest to nobody
    gaps = torch.as_strided(q, (m - 1, 16), (ldq, 1), q.storage_offset() + ldq - 16)
    assert bool((gaps == 165).all())
    if rows != "norm":
        codes = torch.as_strided(q, (m, k), (ldq, 1), q.storage_offset()).view(torch.float8_e4m3fn)
        fp8.check_codes(x, codes, s.view(mb, kb), rows)


@pytest.mark.parametrize("out", fp8.DTYPES)
@pytest.mark.parametrize("m,k,n", [(1, 40, 3), (8, 1100, 130), (197, 300, 777), (300, 130, 64),
                                   (2600, 200, 1000), (2573, 129, 1001)])
@pytest.mark.parametrize("wide", [0, 24, 5])
def test_product(vlib, cuda, out, m, k, n, wide):
    """Into rows `wide` elements further apart than the result is, with the residual
    beside it and then in the result's own place."""
    xq, xs, wq, ws = fp8.operands(m, k, n, seed=m)
    bias, res = fp8.randn(n, seed=20), fp8.randn(m, n, seed=21, dtype=out)
    ld = n + wide

    def run(residual, ldr, y):
        vlib.check(vlib.lib.vitb200_gemm_fp8(
            xq.data_ptr(), max(xq.stride(0), (k + 15) // 16 * 16), xs.data_ptr(), xs.shape[1],
            wq.data_ptr(), max(wq.stride(0), (k + 15) // 16 * 16), ws.data_ptr(), ws.shape[1],
            bias.data_ptr(), residual.data_ptr(), ldr, y.data_ptr(), ld, TYPES[out], m, k, n, 1,
            stream()), "gemm_fp8")
        torch.cuda.synchronize()

    ok, y = guard((m - 1) * ld + n, cuda, out)
    run(res, n, y)
    assert ok()
    rows = torch.as_strided(y, (m, n), (ld, 1), y.storage_offset())
    fp8.check_gemm(rows.contiguous(), xq, xs, wq, ws, bias, res, True)
    if wide and m > 1:
        gaps = torch.as_strided(y, (m - 1, wide), (ld, 1), y.storage_offset() + n)
        assert bool((gaps == FILL[out]).all())
    ok, z = guard((m - 1) * ld + n, cuda, out)
    place = torch.as_strided(z, (m, n), (ld, 1), z.storage_offset())
    place.copy_(res)
    run(z, ld, z)
    assert ok() and torch.equal(place, rows)
    if wide and m > 1:
        gaps = torch.as_strided(z, (m - 1, wide), (ld, 1), z.storage_offset() + n)
        assert bool((gaps == FILL[out]).all())


@pytest.mark.parametrize("dtype", cross.DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,tq,tk,heads,kv_heads", [
    (2, 1, 197, 12, 12), (3, 1, 9000, 4, 2), (2, 3, 9001, 3, 1), (1, 16, 20000, 1, 1),
    (2, 61, 577, 3, 3), (1, 24, 5000, 2, 1), (2, 129, 1000, 2, 1), (1, 300, 4000, 3, 1),
    (1, 257, 100, 5, 5)])
def test_attention(vlib, cuda, dtype, d, b, tq, tk, heads, kv_heads):
    q, k, v = cross.operands(b, tq, tk, heads, kv_heads, d, dtype, seed=tk)
    lens = torch.tensor([tk, tk // 3, 0][:b], dtype=torch.int32, device="cuda")
    o_ok, o = guard(q.numel(), cuda, dtype)
    need = vlib.lib.vitb200_cross_attention_workspace_bytes(b, tq, tk, heads, kv_heads, d)
    w_ok, w = guard(max(1, need), cuda, torch.uint8)
    vlib.check(vlib.lib.vitb200_cross_attention(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), TYPES[dtype], b, tq, tk, heads,
        kv_heads, d, q.stride(1), q.stride(0), k.stride(1), k.stride(0), v.stride(1), v.stride(0),
        lens.data_ptr(), d ** -0.5, w.data_ptr() if need else None, need, stream()),
        "cross_attention")
    torch.cuda.synchronize()
    assert o_ok() and w_ok()
    cross.check(o.view(q.shape), q, k, v, d ** -0.5, heads, kv_heads, lens)


@pytest.mark.parametrize("tq", [1, 9, 64, 300])
def test_an_image_in_batches_of_other_images(cuda, tq):
    """A batch changes how an image's keys are shared out, and with it only the order of
    its sums: each result is within the check's bounds alone and in any batch."""
    import vit_cuda
    q, k, v = cross.operands(9, tq, 3000, 4, 2, 128, torch.bfloat16, seed=13)
    for n in (1, 2, 5, 9):
        o = vit_cuda.cross_attention(q[:n], k[:n], v[:n], 0.1, 4, 2)
        cross.check(o, q[:n], k[:n], v[:n], 0.1, 4, 2)
        assert torch.equal(o, vit_cuda.cross_attention(q[:n], k[:n], v[:n], 0.1, 4, 2))

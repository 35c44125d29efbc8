"""cross_attention of a batch that shares one image's keys and values (several beams or
questions over one image): a batch stride of 0, read in place."""
import pytest
import torch

import vit_cuda
from test_cross_attention_gpu import check, operands
from test_serving_rows_gpu import allocations

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tq", [1, 5, 40, 64, 300, 1100])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("ragged", [False, True])
def test_expanded_keys(cuda, tq, d, ragged):
    b, heads, kv_heads, tk = 6, 4, 2, 700
    q, k, v = operands(b, tq, tk, heads, kv_heads, d, torch.bfloat16, seed=tq)
    lens = None
    if ragged:
        lens = torch.tensor([700, 0, 1, 129, 512, 699], dtype=torch.int32, device="cuda")
    one_k, one_v, one_q = k[:1].expand(b, -1, -1), v[:1].expand(b, -1, -1), q[:1].expand(b, -1, -1)

    def run(q, k, v):
        return vit_cuda.cross_attention(q, k, v, d ** -0.5, heads, kv_heads, lens)

    o, n = allocations(lambda: run(q, one_k, one_v))
    _, plain = allocations(lambda: run(q, k, v))
    assert n == plain + (2 if tq * heads // kv_heads > 128 else 0)  # copies for prompts alone
    assert torch.equal(o, run(q, one_k.contiguous(), one_v.contiguous()))
    assert torch.equal(run(q, one_k, v), run(q, one_k.contiguous(), v))
    assert torch.equal(run(q, k, one_v), run(q, k, one_v.contiguous()))
    assert torch.equal(run(one_q, k, v), run(one_q.contiguous(), k, v))


@pytest.mark.parametrize("tq", [1, 40, 300])
def test_batch_stride_of_zero_from_c(vlib, cuda, tq):
    """The same through the C entry point, prompts too."""
    b, heads, kv_heads, d, tk = 5, 4, 2, 64, 700
    q, k, v = operands(b, tq, tk, heads, kv_heads, d, torch.bfloat16, seed=tq)
    o = torch.empty_like(q)
    need = vlib.lib.vitb200_cross_attention_workspace_bytes(b, tq, tk, heads, kv_heads, d)
    w = torch.empty(max(1, need), dtype=torch.uint8, device=cuda)
    vlib.check(vlib.lib.vitb200_cross_attention(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), vlib.BF16, b, tq, tk, heads, kv_heads,
        d, q.stride(1), 0, k.stride(1), 0, v.stride(1), 0, None, 0.125, w.data_ptr() if need else None,
        need, torch.cuda.current_stream().cuda_stream), "cross_attention")
    check(o, *(t[:1].expand(b, -1, -1) for t in (q, k, v)), 0.125, heads, kv_heads)

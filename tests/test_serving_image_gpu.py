"""From an image to a decoder's cross-attention, as the readme shows it: the encoder's
tokens through its final LayerNorm into FP8 keys and values, read by a prompt."""
import pytest
import torch

import vit_cuda
from test_cross_attention_gpu import reference
from vit_cuda.weights import synthetic_images, synthetic_state_dict

pytestmark = pytest.mark.gpu


def test_image_to_attention(cuda):
    """Against the same layer in 64 bits on the encoder's own tokens and the dequantised
    weights. The normalised tokens are rounded to e4m3, each by at most half a step (2^-4
    of a value), keys and values to bf16 (2^-9); through scores of order 1 and the values
    themselves that is sqrt(2) * 2^-4 in the 2-norm, held to 2^-3 as the decoder layer's
    test is."""
    E, heads, d, b = 768, 12, 64, 2
    state = synthetic_state_dict(seed=5, img_size=224, depth=2)
    model = vit_cuda.ViTCUDA(state_dict={k: v.to(cuda) for k, v in state.items()}).to(cuda).eval()
    images = synthetic_images(b, 224, seed=5).to(cuda)
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    w_kv = torch.randn(2 * E, E, generator=g, device="cuda") * E ** -0.5
    q = torch.randn(b, 9, E, generator=g, device="cuda").bfloat16()
    with torch.no_grad():
        model.prepare()
        tokens = model.embed(images)
        for i in range(len(model.blocks)):
            tokens = model.block(i, tokens)
        wq, ws = vit_cuda.quantize_fp8(w_kv, 128)
        kv = vit_cuda.gemm_fp8(
            *vit_cuda.layernorm_fp8(tokens, model.norm_gamma, model.norm_beta, model.eps), wq, ws,
            out_dtype=torch.bfloat16)
        a = vit_cuda.cross_attention(q, kv[..., :E], kv[..., E:], d ** -0.5, heads)
        logits = model.head(tokens)[0]
        torch.testing.assert_close(logits, model(images), atol=1e-4, rtol=1e-4)  # its tokens
    x = tokens.double()
    c = x - x.mean(-1, keepdim=True)
    y = c / torch.sqrt((c * c).mean(-1, keepdim=True) + model.eps)
    y = y * model.norm_gamma.double() + model.norm_beta.double()
    w = wq.double() * ws.double().repeat_interleave(128, 0).repeat_interleave(128, 1)
    full = y @ w.t()
    want, _, _ = reference(q, full[..., :E], full[..., E:], d ** -0.5, heads, heads)
    assert float((a.double() - want).norm() / want.norm()) < 2.0 ** -3

"""The serving operators under tracers, fake tensors, transforms and autograd: a
call that something has to see goes through the registered op, as the package's
other ops do, and never past it with a frozen or a gradientless answer."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

import vit_cuda
from vit_cuda import serving

FP8 = torch.float8_e4m3fn


def calls(device, k=100):
    """{op: (function of its first floating argument, that argument)}"""
    def t(*shape, dtype=torch.float32):
        return torch.randn(*shape, device=device).to(dtype)

    q, s = t(5, k).to(FP8), t(5, 1).abs()
    w, ws = t(30, k).to(FP8), t(1, 1).abs()
    kv = t(2, 7, 128, dtype=torch.bfloat16)
    ones = torch.ones(k, device=device)
    lens = torch.full((2,), 5, dtype=torch.int32, device=device)
    return {
        "quantize_fp8": (lambda x: vit_cuda.quantize_fp8(x), t(5, k)),
        "quantize_fp8_blocks": (lambda x: vit_cuda.quantize_fp8(x, 128), t(5, k)),
        "layernorm_fp8": (lambda x: vit_cuda.layernorm_fp8(x, ones, ones, 1e-6), t(2, 5, k)),
        "gemm_fp8": (lambda x: vit_cuda.gemm_fp8(q, s, w, ws, residual=x, gelu=True), t(5, 30)),
        "cross_attention": (lambda x: vit_cuda.cross_attention(x, kv, kv, 0.1, 4, 2, lens),
                            t(2, 3, 256, dtype=torch.bfloat16)),
    }


OPS = ["quantize_fp8", "quantize_fp8_blocks", "layernorm_fp8", "gemm_fp8", "cross_attention"]
SHAPES = {"quantize_fp8": [(5, 100), (5, 1)], "quantize_fp8_blocks": [(5, 100), (1, 1)],
          "layernorm_fp8": [(2, 5, 100), (2, 5, 1)], "gemm_fp8": [(5, 30)],
          "cross_attention": [(2, 3, 256)]}


def outputs(y):
    return list(y) if isinstance(y, (tuple, list)) else [y]


@pytest.mark.parametrize("op", OPS)
def test_fake_tensors(op):
    with FakeTensorMode(allow_non_fake_inputs=True):
        f, x = calls("cuda")[op]
        ys = outputs(f(x))
    assert [tuple(y.shape) for y in ys] == SHAPES[op]
    assert all(type(y) is type(x) and y.device == x.device for y in ys)


@pytest.mark.parametrize("op", OPS)
def test_meta_gradient_is_refused(op):
    """An input that requires a gradient never gives an output that looks like a
    constant."""
    f, x = calls("meta")[op]
    y = outputs(f(x.requires_grad_()))[-1]
    assert y.requires_grad
    with pytest.raises(RuntimeError, match="no autograd formula"):
        (y.float().sum() + x.float().sum()).backward()
    with torch.no_grad():
        assert not outputs(f(x))[-1].requires_grad


@pytest.mark.parametrize("op", OPS)
def test_meta_tensors(op):
    f, x = calls("meta")[op]
    ys = outputs(f(x))
    assert [tuple(y.shape) for y in ys] == SHAPES[op] and all(y.is_meta for y in ys)


def test_proxies():
    """torch.fx's symbolic trace records the op."""
    g = torch.fx.symbolic_trace(lambda x: vit_cuda.quantize_fp8(x)[1] + 1)
    assert any("quantize_fp8" in str(n.target) for n in g.graph.nodes)


# ---------------------------------------------------------------- on the GPU
@pytest.mark.gpu
@pytest.mark.parametrize("op", OPS)
def test_plain_calls_go_past_the_dispatcher(cuda, op):
    _, x = calls(cuda)[op]
    watched = serving.direct().watched
    assert not watched(x) and not watched(torch.nn.Parameter(x, requires_grad=False), None)
    assert watched(torch.nn.Parameter(x))
    with torch.no_grad():
        assert not watched(torch.nn.Parameter(x))
    with torch.inference_mode():
        assert not watched(x) and not watched(torch.ones(3, device=cuda))
    with torch.autocast("cuda"):
        assert not watched(x)
    with torch.cuda.stream(torch.cuda.Stream()):
        assert not watched(x)


@pytest.mark.gpu
@pytest.mark.parametrize("op", OPS)
def test_traced_calls_follow_their_inputs(cuda, op):
    """make_fx and torch.jit.trace: the traced function, given other inputs, gives
    what the function gives."""
    torch.manual_seed(0)
    f, x = calls(cuda)[op]
    other = x.flip(0) * 0.5 + 1
    want = outputs(f(other))

    def same(ys):
        assert all(torch.equal(y.view(torch.uint8) if y.dtype == FP8 else y,
                               w.view(torch.uint8) if w.dtype == FP8 else w)
                   for y, w in zip(outputs(ys), want))

    same(make_fx(f)(x)(other))

    def plus(x):  # something else that depends on the input
        ys = outputs(f(x))
        return ys[-1].float() + 0 * x.float().sum()

    traced = torch.jit.trace(plus, (x,), check_trace=False)
    torch.testing.assert_close(traced(other), want[-1].float(), rtol=0, atol=0)


@pytest.mark.gpu
@pytest.mark.parametrize("op", OPS)
def test_gradients_are_refused(cuda, op):
    f, x = calls(cuda)[op]
    x.requires_grad_()
    y = outputs(f(x))[-1]
    assert y.requires_grad
    with pytest.raises(RuntimeError, match="no autograd formula"):
        (y.float().sum() + x.float().sum()).backward()
    with torch.no_grad():
        plain = outputs(f(x))[-1]
        assert not plain.requires_grad and torch.equal(plain, y)
    with torch.no_grad(), forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="tangent"):
            f(forward_ad.make_dual(x.detach(), torch.ones_like(x)))


@pytest.mark.gpu
@pytest.mark.parametrize("op", OPS)
def test_transforms_and_negated_views(cuda, op):
    f, x = calls(cuda)[op]
    xs = torch.stack([x, x.flip(0) + 1])
    each = [outputs(f(t)) for t in xs]
    for i, y in enumerate(outputs(torch.func.vmap(f)(xs))):
        assert torch.equal(y.float(), torch.stack([e[i].float() for e in each]))
    for y, w in zip(outputs(f(torch._neg_view(x))), outputs(f(-x))):
        assert torch.equal(y.float(), w.float())


@pytest.mark.gpu
def test_opcheck(cuda):
    """The fake implementation of the registered ops, and (where no operand is FP8, of which
    the check itself multiplies) the schema."""
    ops, w = torch.ops.vit_cuda, torch.randn(130, 100, device=cuda)
    ones = torch.ones(100, device=cuda)
    cases = [(ops.quantize_fp8, (w, 1)), (ops.quantize_fp8, (w, 128)), (ops.quantize_fp8, (w[:1], 1)),
             (ops.layernorm_fp8, (w.view(10, 13, 100), ones, ones, 1e-6)),
             (ops.gemm_fp8, (*vit_cuda.quantize_fp8(w[:7]), *vit_cuda.quantize_fp8(w, 128), None, None,
                             False, torch.float16))]
    q, kv = (torch.randn(2, t, 128, device=cuda).half() for t in (3, 9))
    cases.append((ops.cross_attention, (q, kv, kv, 0.1, 2, None, None)))
    for op, args in cases:
        torch.library.opcheck(op, args, test_utils="test_faketensor")
    torch.library.opcheck(*cases[-1], test_utils="test_schema")

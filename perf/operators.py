"""The serving operators around the ViT encoder, measured one by one: FP8
operand preparation (``quantize_fp8``, ``layernorm_fp8``), the FP8 matrix
product with one scale per block of 128 (``gemm_fp8``) and attention to an
encoder's states of another length (``cross_attention``).

``run`` computes a case in its plain form (elementary torch operations in 32
bits) or, with ``own`` set, through ``vit_cuda``; ``exact`` restates it in 64
bits. Every case's inputs come from its seed alone.
"""
import math
import os
import sys

import torch

own = False

FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
AMAX_FLOOR = 1e-30  # a block whose largest magnitude is below this is scaled as if it were this
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------- cases
def listed():
    return [
        # The widest thing one image's decoder hands to a projection: odd width, half precision.
        {"name": "quantize-odd", "op": "quantize", "m": 577, "k": 1000, "block_rows": 1, "dtype": "fp16"},
        # A weight laid out once, when a model is loaded or its weights are replaced.
        {"name": "quantize-weight", "op": "quantize", "m": 4096, "k": 4096, "block_rows": 128, "dtype": "bf16"},
        # One 224 x 224 image's tokens before the qkv or the first MLP product.
        {"name": "norm-image", "op": "layernorm", "m": 197, "k": 768, "dtype": "fp32"},
        # The same for the batch of 256 images that the throughput benchmark runs.
        {"name": "norm-batch", "op": "layernorm", "m": 50432, "k": 768, "dtype": "fp32"},
        # One decoding step of eight sequences: a few rows against a wide weight.
        {"name": "gemm-token", "op": "gemm", "m": 8, "k": 4096, "n": 4096, "dtype": "bf16",
         "bias": False, "gelu": False, "residual": False},
        # The qkv product of one 224 x 224 image.
        {"name": "gemm-image", "op": "gemm", "m": 197, "k": 768, "n": 2304, "dtype": "fp32",
         "bias": True, "gelu": False, "residual": False},
        # Seven 384 x 384 images into 1000 columns from a width no block divides, added to a residual.
        {"name": "gemm-ragged", "op": "gemm", "m": 4039, "k": 1000, "n": 1000, "dtype": "fp16",
         "bias": True, "gelu": False, "residual": True},
        # A long prompt batch through an MLP's first product.
        {"name": "gemm-large", "op": "gemm", "m": 16384, "k": 4096, "n": 4096, "dtype": "bf16",
         "bias": True, "gelu": True, "residual": False},
        # One caption token of sixteen sequences, each over its own 224 x 224 image.
        {"name": "cross-token", "op": "cross", "b": 16, "tq": 1, "tk": 197, "heads": 12, "kv_heads": 12,
         "d": 64, "dtype": "bf16", "lens": False},
        # One token over long encoder states (video or audio), grouped heads, ragged lengths.
        {"name": "cross-token-long", "op": "cross", "b": 2, "tq": 1, "tk": 32768, "heads": 32,
         "kv_heads": 8, "d": 128, "dtype": "bf16", "lens": True},
        # Short prompts over 384 x 384 images, some of them padded.
        {"name": "cross-prompt", "op": "cross", "b": 32, "tq": 61, "tk": 577, "heads": 12, "kv_heads": 12,
         "d": 64, "dtype": "fp16", "lens": True},
        # Long prompts over long encoder states.
        {"name": "cross-large", "op": "cross", "b": 4, "tq": 4096, "tk": 4500, "heads": 16, "kv_heads": 4,
         "d": 128, "dtype": "bf16", "lens": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["quantize", "layernorm", "gemm", "gemm", "cross", "cross"])
    if op in ("quantize", "layernorm"):
        k = _log_int(rng, 16, 8192)
        m = _log_int(rng, 1, max(1, min(65536, 50432 * 768 // k)))
        case = {"op": op, "m": m, "k": k, "dtype": rng.choice(["fp32", "bf16", "fp16"])}
        if op == "quantize":
            case["block_rows"] = rng.choice([1, 1, 128])
        return case
    if op == "gemm":
        k, n = _log_int(rng, 64, 8192), _log_int(rng, 16, 8192)
        if rng.random() < 0.5:  # most widths are multiples of 64
            k, n = max(64, k // 64 * 64), max(64, n // 64 * 64)
        m = _log_int(rng, 1, max(1, min(65536, 16384 * 4096 * 4096 // (k * n), 16384 * 8192 // max(k, n))))
        return {"op": "gemm", "m": m, "k": k, "n": n, "dtype": rng.choice(["fp32", "bf16", "fp16"]),
                "bias": rng.random() < 0.7, "gelu": rng.random() < 0.3, "residual": rng.random() < 0.3}
    kv_heads = rng.choice([1, 2, 4, 8, 12, 16])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
    d = rng.choice([64, 128])
    tk = _log_int(rng, 1, 32768)
    tq = 1 if rng.random() < 0.4 else _log_int(rng, 2, 4096)
    # at most the work of the largest listed case, in scores and in bytes of keys
    most = max(1, min(64, 4 * 16 * 4096 * 4500 // (heads * tq * tk), 2 * 8 * 32768 * 128 // (kv_heads * tk * d)))
    if heads * tq * tk > 4 * 16 * 4096 * 4500:
        tq = max(1, 4 * 16 * 4096 * 4500 // (heads * tk))
    return {"op": "cross", "b": _log_int(rng, 1, most), "tq": tq, "tk": tk, "heads": heads,
            "kv_heads": kv_heads, "d": d, "dtype": rng.choice(["bf16", "fp16"]),
            "lens": rng.random() < 0.5}


# ---------------------------------------------------------------- inputs
def _blocks(k):
    return (k + 127) // 128


def _padded_rows(q, k):
    """Codes as ``quantize_fp8`` hands them out: rows 16 bytes apart or a multiple of it."""
    ld = (k + 15) // 16 * 16
    if ld == k:
        return q
    buf = torch.zeros(q.shape[0], ld, dtype=torch.uint8, device=q.device)
    buf[:, :k] = q.view(torch.uint8)
    return buf.view(FP8)[:, :k]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32)

    dt = DTYPES[case["dtype"]]
    if case["op"] in ("quantize", "layernorm"):
        m, k = case["m"], case["k"]
        # activations: rows of different sizes, a few columns much larger than the rest
        x = randn(m, k) * torch.exp(0.5 * randn(m, 1))
        if case["op"] == "quantize" and case["block_rows"] == 128:
            x = randn(m, k) * 0.02
        else:
            x[:, torch.randint(0, k, (max(1, k // 256),), generator=g, device=dev)] *= 8.0
        state = {"case": dict(case), "x": x.to(dt)}
        if case["op"] == "layernorm":
            state["gamma"] = torch.exp(0.3 * randn(k))
            state["beta"] = 0.2 * randn(k)
        return state
    if case["op"] == "gemm":
        m, k, n = case["m"], case["k"], case["n"]
        x = randn(m, k) * torch.exp(0.5 * randn(m, 1))
        w = randn(n, k) * (torch.exp(0.3 * randn(n, 1)) / math.sqrt(k))
        xq, xs = _plain_quantize(x, 1)
        wq, ws = _plain_quantize(w, 128)
        return {"case": dict(case), "xq": _padded_rows(xq, k), "xs": xs, "wq": _padded_rows(wq, k), "ws": ws,
                "bias": 0.1 * randn(n) if case["bias"] else None,
                "residual": randn(m, n).to(dt) if case["residual"] else None}
    b, tq, tk, d = case["b"], case["tq"], case["tk"], case["d"]
    q = (randn(b, tq, case["heads"] * d) * 1.5).to(dt)
    # keys and values as one projection leaves them: side by side in a row
    kv = torch.empty(b, tk, 2 * case["kv_heads"] * d, device=dev, dtype=dt)
    for i in range(b):
        kv[i] = randn(tk, 2 * case["kv_heads"] * d)
    lens = None
    if case["lens"]:
        u = torch.rand(b, generator=g, device=dev)
        lens = (tk * (0.5 + 0.5 * u)).ceil().to(torch.int32).clamp_(max=tk)
    return {"case": dict(case), "q": q, "k": kv[..., :case["kv_heads"] * d], "v": kv[..., case["kv_heads"] * d:],
            "lens": lens, "scale": 1.0 / math.sqrt(d)}


# ---------------------------------------------------------------- plain forms
def _plain_quantize(x, block_rows):
    m, k = x.shape
    kb, mb = _blocks(k), (m + block_rows - 1) // block_rows
    x = torch.nn.functional.pad(x.float(), (0, kb * 128 - k, 0, mb * block_rows - m))
    t = x.view(mb, block_rows, kb, 128)
    a = t.abs().amax(dim=(1, 3))
    a = torch.where(a < AMAX_FLOOR, torch.full_like(a, AMAX_FLOOR), a)
    # one division of exact operands for 16-bit inputs, whose quotients often lie midway between two codes
    q = (t * FP8_MAX / a[:, None, :, None]).to(FP8).view(mb * block_rows, kb * 128)
    return q[:m, :k], a / FP8_MAX


def _plain_layernorm(x, gamma, beta, eps):
    x = x.float()
    c = x - x.mean(dim=1, keepdim=True)
    return c / torch.sqrt((c * c).mean(dim=1, keepdim=True) + eps) * gamma + beta


def _plain_gemm(s):
    k, n = s["case"]["k"], s["case"]["n"]
    x = s["xq"].float() * s["xs"].repeat_interleave(128, dim=1)[:, :k]
    w = s["wq"].float() * s["ws"].repeat_interleave(128, dim=0)[:n].repeat_interleave(128, dim=1)[:, :k]
    y = x @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["case"]["gelu"]:
        y = 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    if s["residual"] is not None:
        y = s["residual"].float() + y
    return y.to(DTYPES[s["case"]["dtype"]])


def _plain_cross(s):
    c = s["case"]
    b, tq, tk, h, hk, d = c["b"], c["tq"], c["tk"], c["heads"], c["kv_heads"], c["d"]
    q = s["q"].float().view(b, tq, hk, h // hk, d).permute(0, 2, 3, 1, 4)
    k = s["k"].float().view(b, tk, hk, 1, d).permute(0, 2, 3, 4, 1)
    v = s["v"].float().view(b, tk, hk, 1, d).permute(0, 2, 3, 1, 4)
    x = torch.matmul(q, k) * s["scale"]
    if s["lens"] is not None:
        out = torch.arange(tk, device=x.device)[None] >= s["lens"][:, None]
        x = x.masked_fill(out[:, None, None, None, :], float("-inf"))
    p = torch.exp(x - x.amax(dim=-1, keepdim=True))
    o = torch.matmul(p, v) / p.sum(dim=-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4).reshape(b, tq, h * d).to(s["q"].dtype)


def _package():
    if "vit_cuda" not in sys.modules:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vit-engine-cuda_b200")
        if root not in sys.path:
            sys.path.insert(0, root)
    import vit_cuda
    return vit_cuda


def run(state):
    c = state["case"]
    if own:
        vit = _package()
        if c["op"] == "quantize":
            return vit.quantize_fp8(state["x"], c["block_rows"])
        if c["op"] == "layernorm":
            return vit.layernorm_fp8(state["x"], state["gamma"], state["beta"], 1e-6)
        if c["op"] == "gemm":
            return vit.gemm_fp8(state["xq"], state["xs"], state["wq"], state["ws"], state["bias"],
                                residual=state["residual"], gelu=c["gelu"], out_dtype=DTYPES[c["dtype"]])
        return vit.cross_attention(state["q"], state["k"], state["v"], state["scale"], c["heads"],
                                   kv_heads=c["kv_heads"], kv_lens=state["lens"])
    if c["op"] == "quantize":
        return _plain_quantize(state["x"], c["block_rows"])
    if c["op"] == "layernorm":
        return _plain_quantize(_plain_layernorm(state["x"], state["gamma"], state["beta"], 1e-6), 1)
    return _plain_gemm(state) if c["op"] == "gemm" else _plain_cross(state)


# ---------------------------------------------------------------- work
def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    if case["op"] in ("quantize", "layernorm"):
        m, k = case["m"], case["k"]
        rows = case.get("block_rows", 1)
        norm = case["op"] == "layernorm"
        return {"bytes": m * k * (es + 1) + 4 * _blocks(k) * ((m + rows - 1) // rows) + (8 * k if norm else 0),
                "flops": m * k * (8 if norm else 2)}
    if case["op"] == "gemm":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": m * k + n * k + 4 * _blocks(k) * (m + _blocks(n)) + m * n * es * (2 if case["residual"] else 1)
                + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    b, tq, tk, d = case["b"], case["tq"], case["tk"], case["d"]
    share = 0.75 if case["lens"] else 1.0  # lengths are spread evenly over the upper half
    return {"bytes": int(2 * es * b * tq * case["heads"] * d + 2 * es * b * tk * case["kv_heads"] * d * share),
            "flops": int(4 * b * tq * tk * case["heads"] * d * share)}


# ---------------------------------------------------------------- in 64 bits
def _e4m3(x):
    """x rounded to the nearest value of a sign, four exponent bits (bias 7) and three fraction bits."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -20))).clamp(min=-6.0)
    step = torch.exp2(e - 3.0)
    return (torch.round(x / step) * step).clamp(-FP8_MAX, FP8_MAX)


def _exact_quantize(x, block_rows):
    m, k = x.shape
    q = torch.empty(m, k, dtype=torch.float64, device=x.device)
    scales = torch.empty((m + block_rows - 1) // block_rows, _blocks(k), dtype=torch.float64, device=x.device)
    for j in range(_blocks(k)):
        cols = x[:, 128 * j:128 * j + 128]
        amax = cols.abs().max(dim=1).values
        if block_rows > 1:
            whole = torch.cat([amax, amax.new_zeros(-m % block_rows)])
            amax = whole.view(-1, block_rows).max(dim=1).values
        amax = amax.clamp(min=AMAX_FLOOR)
        scales[:, j] = amax / FP8_MAX
        per_row = amax.repeat_interleave(block_rows)[:m]
        q[:, 128 * j:128 * j + 128] = _e4m3(cols * FP8_MAX / per_row[:, None])
    return q, scales


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        return _exact_quantize(s["x"].double(), case["block_rows"])
    if case["op"] == "layernorm":
        x = s["x"].double()
        var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        y = (x - mean) * torch.rsqrt(var + 1e-6) * s["gamma"].double() + s["beta"].double()
        return _exact_quantize(y, 1)
    if case["op"] == "gemm":
        m, k, n = case["m"], case["k"], case["n"]
        y = torch.zeros(m, n, dtype=torch.float64, device=s["xq"].device)
        for j in range(_blocks(k)):
            cols = slice(128 * j, min(k, 128 * j + 128))
            part = s["xq"][:, cols].double() @ s["wq"][:, cols].double().t()
            part *= s["xs"][:, j].double()[:, None]
            part *= s["ws"][:, j].double().repeat_interleave(128)[:n]
            y += part
        if s["bias"] is not None:
            y += s["bias"].double()
        if case["gelu"]:
            y *= 0.5 * torch.erfc(-y / math.sqrt(2.0))
        if s["residual"] is not None:
            y += s["residual"].double()
        return y
    b, tq, d = case["b"], case["tq"], case["d"]
    group = case["heads"] // case["kv_heads"]
    o = torch.empty(b, tq, case["heads"], d, dtype=torch.float64, device=s["q"].device)
    for i in range(b):
        n = case["tk"] if s["lens"] is None else int(s["lens"][i])
        for j in range(case["kv_heads"]):
            k = s["k"][i, :n, j * d:(j + 1) * d].double()
            v = s["v"][i, :n, j * d:(j + 1) * d].double()
            for h in range(j * group, (j + 1) * group):
                x = (s["q"][i, :, h * d:(h + 1) * d].double() @ k.t()) * s["scale"]
                o[i, :, h] = torch.softmax(x, dim=1) @ v
    return o.view(b, tq, case["heads"] * d)

"""The serving operators' first use in a process inside a CUDA graph capture,
after vitb200_init alone, and calls from several threads and streams at once."""
import os
import subprocess
import sys
import threading

import pytest
import torch

import vit_cuda

pytestmark = pytest.mark.gpu

PKG = os.path.dirname(os.path.dirname(os.path.abspath(vit_cuda.__file__)))

CAPTURE = """
import torch, vit_cuda
from vit_cuda import _lib
_lib.check(_lib.lib.vitb200_init(), "init")
g = torch.Generator(device="cuda"); g.manual_seed(0)
def randn(*s): return torch.randn(*s, generator=g, device="cuda")
x, w, gamma, beta = randn(5, 200), randn(300, 200), torch.ones(200, device="cuda"), torch.zeros(200, device="cuda")
kv = randn(2, 5000, 256).bfloat16()
q1, q2, q3 = (randn(2, t, 128).bfloat16() for t in (1, 30, 300))
def step():
    wq, ws = vit_cuda.quantize_fp8(w, 128)
    a = vit_cuda.gemm_fp8(*vit_cuda.quantize_fp8(x), wq, ws)
    b = vit_cuda.gemm_fp8(*vit_cuda.layernorm_fp8(x, gamma, beta, 1e-6), wq, ws, gelu=True)
    return [a, b] + [vit_cuda.cross_attention(q, kv[..., :128], kv[..., 128:], 0.125, 2) for q in (q1, q2, q3)]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    outs = step()
graph.replay()
torch.cuda.synchronize()
for o, r in zip(outs, step()):
    assert torch.equal(o, r)
assert vit_cuda.device_error() == 0
print("same")
"""


def test_first_use_inside_a_capture(cuda):
    env = dict(os.environ, PYTHONPATH=PKG + os.pathsep + os.environ.get("PYTHONPATH", ""))
    r = subprocess.run([sys.executable, "-c", CAPTURE], capture_output=True, text=True, env=env,
                       timeout=240)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-2000:]


def test_threads_and_streams(cuda):
    """Every thread its own stream; workspaces and outputs are each call's own."""
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    kv = torch.randn(4, 9000, 256, generator=g, device="cuda").bfloat16()
    x = torch.randn(64, 512, generator=g, device="cuda")
    wq, ws = vit_cuda.quantize_fp8(torch.randn(1000, 512, generator=g, device="cuda"), 128)
    qs = [torch.randn(4, t, 256, generator=g, device="cuda").bfloat16() for t in (1, 2, 1, 40)]
    lens = torch.tensor([9000, 10, 0, 4000], dtype=torch.int32, device="cuda")

    def work(q):
        a = vit_cuda.cross_attention(q, kv[..., :128], kv[..., 128:], 0.125, 4, 2, lens)
        return a, vit_cuda.gemm_fp8(*vit_cuda.quantize_fp8(x), wq, ws)

    refs = [work(q) for q in qs]
    torch.cuda.synchronize()
    bad = []

    def thread(i):
        torch.cuda.set_device(cuda)
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                for o, r in zip(work(qs[i]), refs[i]):
                    if not torch.equal(o, r):
                        bad.append(i)

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(len(qs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not bad

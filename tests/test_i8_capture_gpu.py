"""After one call of any 8-bit operator on a device, every other one may be captured into a CUDA graph."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

CODE = r"""
import sys
import torch
import aegis_torch
ops = torch.ops.aegis
first = sys.argv[1]
g = torch.Generator(device="cuda").manual_seed(3)
x, r = (torch.randn(M, 256, device="cuda", generator=g).bfloat16() for M in (20, 20))
nw = torch.ones(256, device="cuda").bfloat16()
w1, w2 = (torch.randint(-127, 128, s, device="cuda", generator=g, dtype=torch.int8) for s in ((1024, 256), (256, 512)))
s1, s2 = torch.full((1024,), 1e-3, device="cuda"), torch.full((256,), 1e-3, device="cuda")
many, wide = torch.ones(4000, 256, device="cuda").bfloat16(), torch.ones(700, 12000, device="cuda").bfloat16()
calls = {
    "rmsnorm": lambda: ops.rmsnorm_i8(x, nw, 1e-5),
    "silu": lambda: ops.silu_mul_i8(x, r),
    "matmul": lambda: ops.matmul_i8(w2[:20, :256], w1, s2[:20], s1),  # the stream kernel
    "dot": lambda: ops.matmul_i8(w2[:1, :256], w1, s2[:1], s1),
    "unaligned": lambda: ops.matmul_i8(w2[:20, 1:200], w1[:, 3:202], s2[:20], s1),
    "pair": lambda: ops.matmul_i8(w1, w1, s1, s1),
    "many rows": lambda: ops.rmsnorm_i8(many, nw, 1e-5),
    "wide rows": lambda: ops.silu_mul_i8(wide, wide),
    "mlp": lambda: ops.mlp_i8(x, r, nw, 1e-5, w1, s1, w2, s2),
}
calls[first]()
torch.cuda.synchronize()
graphs = {}
for name, call in calls.items():
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    graphs[name] = graph, out
for name, (graph, out) in graphs.items():
    graph.replay()
    torch.cuda.synchronize()
    want = calls[name]()
    for a, b in zip(out if isinstance(out, tuple) else (out,), want if isinstance(want, tuple) else (want,)):
        assert torch.equal(a, b), name
print("ok")
"""


@pytest.mark.parametrize("first", ["rmsnorm", "silu", "matmul", "mlp"])
def test_any_first_call_readies_the_device(cuda, first):
    r = subprocess.run([sys.executable, "-c", CODE, first], capture_output=True, text=True, timeout=300,
                       env={**os.environ, "PYTHONPATH": os.path.join(ROOT, "aegis-core_b200")})
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stderr[-2000:]

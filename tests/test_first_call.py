"""The first call of a process, which sets the library up on the device, while a stream is being captured into a graph."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROGRAM = """
import sys
sys.path.insert(0, %r)
import torch
import beam

name = sys.argv[1]
g = torch.Generator(device="cuda").manual_seed(1)
x, w = (torch.randn(s, device="cuda", generator=g).half() for s in ((200, 512), (512, 512)))
c, dx, dw = torch.empty(200, 512, device="cuda").half(), torch.empty_like(x), torch.empty_like(w)
q, v = beam.mxfp4_empty(200, 512), torch.empty_like(x)
gamma, beta = torch.ones(512, device="cuda").half(), torch.zeros(512, device="cuda").half()


def call():
    if name == "gated":
        beam.gated_gemmrc(x, w, w, c)
    elif name == "few rows":
        beam.gated_gemmrc(x[:3], w, w, c[:3])
    elif name == "gradients":
        beam.gated_gemmrc_backward(x, x, w, w, x, x, da=dx, db_gate=dw)
    elif name == "mxfp4":
        beam.mxfp4_quantize(x, *q)
        beam.mxfp4_dequantize(*q, v)
        beam.mxfp4_gemmrc(*q, *q, c.view(-1)[:40000].view(200, 200))
    elif name == "product":
        beam.cutlass_gemmrc(x, w, c)
    elif name == "split-K":
        beam.cutlass_gemmrc_splitk(x, w, c)
    else:
        beam.cutlass_parallel_gemmrc_lnr(x, w, c, gamma, beta)


torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    call()
outs = (c, dx, dw, v)
for t in outs:
    t.fill_(3)
graph.replay()
torch.cuda.synchronize()
seen = [t.clone() for t in outs]
for t in outs:
    t.fill_(3)
call()
torch.cuda.synchronize()
assert all(torch.equal(s, t) for s, t in zip(seen, outs)) and any((t != 3).any() for t in outs)
assert beam.device_status() == (0, 0)
"""


@pytest.mark.gpu
@pytest.mark.parametrize("name", ("gated", "few rows", "gradients", "mxfp4", "product", "split-K", "layernorm"))
def test_first_call_is_captured(built_library, name):
    program = PROGRAM % os.path.join(ROOT, "general-nvgpu-testing_b200")
    done = subprocess.run([sys.executable, "-c", program, name], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]

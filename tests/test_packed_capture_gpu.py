"""The packed operators captured into a graph by a process that has called none of them before: a process each, as a warm thread hides it."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

SCRIPT = """
import sys
import torch
from system_lab_b200 import ops
from system_lab_b200.ops import cuda

what, backward = sys.argv[1], sys.argv[2] == "backward"
dev = torch.device("cuda", 0)
g = torch.Generator(device=dev)
g.manual_seed(0)
normal = lambda *shape: torch.randn(shape, device=dev, generator=g).bfloat16()
if what == "attention":
    leaves, dout = [normal(200, n, 64) for n in (4, 2, 2)], normal(200, 4, 64)
    cu = torch.tensor([0, 120, 200], dtype=torch.int32, device=dev)
    call = lambda: ops.packed_attention(*leaves, ops.pack_documents(cu, 200))
elif what == "embedding":
    leaves, dout = [normal(40000, 64)], normal(300, 64)
    tokens = torch.randint(0, 40000, (300,), device=dev, generator=g)
    call = lambda: ops.embedding(tokens, *leaves, scale=3.0)
else:
    leaves, dout = [normal(200, 64)], normal(200, 64)
    call = lambda: ops.dropout(*leaves, 0.3, 5)
for x in leaves:
    x.requires_grad_(backward)

def step():
    out = call()
    return (out.detach(), *torch.autograd.grad(out, leaves, dout)) if backward else (out,)

cuda.lib()
cuda.status_word(dev)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step()
graph.replay()
want = step()
torch.cuda.synchronize()
cuda.check_status(dev)
assert all(torch.equal(a, b) for a, b in zip(got, want))
"""


@pytest.mark.parametrize("way", ["forward", "backward"])
@pytest.mark.parametrize("what", ["attention", "embedding", "dropout"])
def test_first_call_is_captured(what, way):
    run = subprocess.run([sys.executable, "-c", SCRIPT, what, way], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True,
                         timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]

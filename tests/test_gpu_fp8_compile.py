"""The 8-bit operators next to torch.compile, and captured before anything else has run."""

import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from _util import DEV, randn

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent


def _f(a, b):
    import fma_b200 as fma

    y = fma.linear_fp8(a * 2, b)
    return fma.swiglu_fp8_checkpoint(y, y * 0.5) + 1


def _step(f, x, w, d):
    a, b = x.clone().requires_grad_(), w.clone().requires_grad_()
    y = f(a, b)
    return (y.detach(), *torch.autograd.grad(y, (a, b), d))


def test_compiled_code_breaks_around_the_operators():
    x, w = randn((40, 264), torch.bfloat16, 1).to(DEV), randn((136, 264), torch.bfloat16, 2).to(DEV)
    d = randn((40, 136), torch.bfloat16, 3).to(DEV)
    want = _step(_f, x, w, d)
    for one, other in zip(want, _step(torch.compile(_f, backend="aot_eager"), x, w, d)):
        assert torch.equal(one, other)
    torch._dynamo.reset()
    with pytest.raises(torch._dynamo.exc.Unsupported):
        torch.compile(_f, backend="aot_eager", fullgraph=True)(x, w)
    torch._dynamo.reset()


CHILD = """
import sys
sys.path[:0] = ["cute-kernels_b200", "tests"]
import torch, fma_b200 as fma
x = torch.ones(ROWS, 264, device="cuda", dtype=torch.bfloat16)
w = torch.ones(3, 136, 264, device="cuda", dtype=torch.bfloat16)
count = torch.tensor([ROWS // 2, 0, ROWS - ROWS // 2], device="cuda")
d = torch.ones(ROWS, 136, device="cuda", dtype=torch.bfloat16)
graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
torch.cuda.synchronize()
with torch.cuda.graph(graph, stream=stream):
    a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
    if TRAIN:
        y = fma.grouped_linear_fp8(a, b, count)
        out = (y.detach(), *torch.autograd.grad(y, (a, b), d))
    else:
        with torch.no_grad():
            out = (fma.grouped_linear_fp8(x, w, count), fma.quantize_fp8(x).dequantize(), fma.swiglu_fp8_checkpoint(x, x))
graph.replay()
torch.cuda.synchronize()
assert bool((out[0] == 264).all())
if TRAIN:
    assert bool((out[1] == 136).all()) and bool((out[2][1] == 0).all()) and bool((out[2][0] == ROWS // 2).all())
print("fine")
"""


@pytest.mark.parametrize("train", [True, False])
@pytest.mark.parametrize("rows", [8, 400])
def test_first_call_of_a_process_is_captured(rows, train):
    code = CHILD.replace("ROWS", str(rows)).replace("TRAIN", str(train))
    got = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=120, env=dict(os.environ))
    assert got.returncode == 0 and "fine" in got.stdout, got.stdout[-500:] + got.stderr[-1500:]


def test_unknown_types_are_refused():
    import fma_b200 as fma

    held = fma.quantize_fp8(torch.ones(4, 16, device=DEV))
    for dtype in ("float32", 3):
        with pytest.raises(TypeError):
            held.dequantize(dtype)
    with pytest.raises(RuntimeError, match="dtype"):
        held.dequantize(torch.int8)

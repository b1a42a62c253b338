"""MI355X: the first launches of the attention block's kernels that need more than 48 KB of LDS, by several threads at once, in a
process of its own where none of them has been launched before (their LDS attribute is set by the first launch).

Sorts in front of what initialises the GPU in this process: a child is started before any GPU call only."""
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = """
import threading
import torch
from tsdiff_amd import block_ops as B

def normal(seed, *shape, dtype):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).to("cuda:0")

def gated(dtype, rows, fin, out):
    t = [normal(k, *s, dtype=dtype) for k, s in enumerate(((rows, fin), (out, fin), (out, fin), (out,), (out,)))]
    return B.gated_linear, t, normal(9, rows, out, dtype=dtype)

def attention(dtype, nodes, dim):
    ptr = torch.tensor([0, nodes], dtype=torch.int32, device="cuda:0")
    t = [normal(k, nodes, 2, dim, dtype=dtype) for k in range(3)]
    return (lambda q, k, v: B.graph_attention(q, k, v, ptr)), t, normal(9, nodes, 2, dim, dtype=dtype)

bf, hf, f = torch.bfloat16, torch.float16, torch.float32
# 256 x 128 and 256 x 256 tiles of 16 bits, 128 x 128 of f32, tiles of 64 and 128 values a head
calls = [gated(bf, 56000, 240, 124), gated(hf, 56000, 240, 124), gated(f, 3601, 256, 1020), attention(bf, 500, 64),
         attention(hf, 500, 128), attention(f, 500, 128)] * 2
torch.cuda.synchronize()
barrier = threading.Barrier(len(calls))
got = [None] * len(calls)

def go(k):
    f, t, d = calls[k]
    leaves = [x.clone().requires_grad_() for x in t]
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda.synchronize()
        barrier.wait()
        try:
            y = f(*leaves)
            got[k] = (y.detach(),) + torch.autograd.grad(y, leaves, d)
        except Exception as e:
            got[k] = e

threads = [threading.Thread(target=go, args=(k,)) for k in range(len(calls))]
for t in threads:
    t.start()
for t in threads:
    t.join()
torch.cuda.synchronize()
for (f, t, d), g in zip(calls, got):
    assert not isinstance(g, Exception), g
    leaves = [x.clone().requires_grad_() for x in t]
    y = f(*leaves)
    want = (y.detach(),) + torch.autograd.grad(y, leaves, d)
    assert all(torch.equal(a, b) and a.isfinite().all() for a, b in zip(g, want))
print("same bits", len(calls))
"""


def test_first_launches_by_several_threads():
    if torch.cuda.device_count() < 1:
        pytest.skip("needs a GPU")
    if torch.cuda.is_initialized():
        pytest.skip("this process has initialised the GPU already: child programs are started before any GPU call only")
    out = subprocess.run([sys.executable, "-c", CHILD], cwd=ROOT, capture_output=True, text=True, timeout=110)
    assert out.returncode == 0 and "same bits 12" in out.stdout, out.stdout[-2000:] + out.stderr[-3000:]

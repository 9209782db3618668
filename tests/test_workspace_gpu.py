"""A captured graph goes on working when a later call needs a larger workspace.
In a process of its own, whose workspace is as small as the first calls leave it."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

CHILD = """
import numpy as np, torch
from cllm_inference_b200 import _lib, synth
from cllm_inference_b200.kv4 import KV4Cache

lib = _lib.load()
_lib.check(lib.cllm_cuda_init(0))
torch.manual_seed(0)
lens = [700, 3000, 64, 1500]
cache = KV4Cache.empty(1, 200, 64, 8, 128, 4, 64).fork(
    torch.full((4,), -1, dtype=torch.int32, device="cuda"), torch.tensor(lens, dtype=torch.int32, device="cuda"))
assert cache.lens.tolist() == lens
kv = torch.randn(sum(lens), 2 * 1024, device="cuda")
seq = torch.repeat_interleave(torch.arange(4), torch.tensor(lens)).int().cuda()
pos = torch.cat([torch.arange(n) for n in lens]).int().cuda()
cache.append(0, kv[:, :1024], kv[:, 1024:], seq, pos)
q = torch.randn(4, 4096, device="cuda")
w = torch.from_numpy(synth.make_weights(synth.Q4_K, 1000, 4096, 1)).cuda()
y = torch.empty(4, 1000, device="cuda")


def step():  # a layer's attention and a product of several rows, both of which use the workspace
    o = cache.attention(0, q)
    _lib.check(lib.cllm_cuda_matmul_quant(o.data_ptr(), w.data_ptr(), synth.Q4_K, None, 4096, 1000, 4, y.data_ptr(), 0,
                                          torch.cuda.current_stream().cuda_stream))
    return o


want = step().clone(), y.clone()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    o = step()
graph.replay()
torch.cuda.synchronize()
assert torch.equal(o, want[0]) and torch.equal(y, want[1])
many = torch.randn(1600, 4096, device="cuda")  # rows of prompts: a workspace several times larger
begin = torch.tensor([0, 300, 900, 900, 1600], dtype=torch.int32, device="cuda")
first = cache.attention(0, many, begin=begin).clone()
torch.cuda.synchronize()
other = [torch.full((1 << 20,), i, dtype=torch.int32, device="cuda") for i in range(64)]  # where freed memory would be
for _ in range(3):
    o.zero_()
    y.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, want[0]) and torch.equal(y, want[1])
    assert all(bool((t == i).all()) for i, t in enumerate(other))
    assert torch.equal(cache.attention(0, many, begin=begin), first)
_lib.check(lib.cllm_cuda_check_device_status())
print("fine")
"""


def test_a_captured_step_outlives_a_larger_call(cuda, lib):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", CHILD], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip() == "fine", done.stderr[-2000:]

"""Calls of the block-scaled KV cache's operators that depend on their surroundings."""
import subprocess
import sys

import numpy as np
import pytest
import torch

import kvb_ref as R
from kvb_ref64 import DEV, i32, make_cache
from torch2riscv_accelerator_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("default", [torch.float64, torch.bfloat16])
def test_another_default_type(default):
    """The calls' own tensors do not follow torch's default type."""
    import torch2riscv_accelerator_b200.torch_ops  # noqa: F401
    g = torch.Generator(device=DEV).manual_seed(1)
    cache = make_cache(g, 2, 2, 64, 32, 16)
    q = torch.randn(5, 4, 32, generator=g, device=DEV)
    pos, start = i32([3, 40]), i32([0, 2, 4])
    want = ops.kvb_read(cache, pos, start, 4), ops.kvb_attn_rows(q, cache, pos, start, out=torch.zeros_like(q))
    torch.set_default_dtype(default)
    try:
        read = torch.ops.w8a8.kvb_read(*cache, pos, start, 5)
        rows = torch.ops.w8a8.kvb_attn_rows(q, *cache, pos, start, None)
        empty = ops.kvb_cache(1, 1, 16, 16, block=16)
    finally:
        torch.set_default_dtype(torch.float32)
    assert all(torch.equal(a[:4], b) and (a[4] == 0).all() for a, b in zip(read, want[0]))
    assert torch.equal(rows, want[1])
    assert empty.k.dtype == torch.int8 and empty.k_scale.dtype == torch.float32


CAPTURE = """
import torch
from torch2riscv_accelerator_b200 import ops
i32 = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda")
cache, mass = ops.kvb_cache(3, 2, 8192, 128, 64), torch.zeros(3, 2, 8192, device="cuda")
x = torch.randn(200, 8, 128, device="cuda")
pos, start, n = i32(0, 0, 0), i32(0, 100, 150, 200), i32(100, 50, 50)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    ops.kvb_append(x[:, 4:6], x[:, 6:], cache, pos, start)
    rows = ops.kvb_attn_rows(x[:, :4], cache, pos, start, mass=mass)
    one = ops.kvb_attn(x[:3, :4], cache, n - 1, mass=mass)
    kept, left = ops.kvb_evict(cache, mass, n, 40)
    read = ops.kvb_read(cache, pos, None, 3)
graph.replay()
torch.cuda.synchronize()
assert rows.abs().sum() > 0 and one.abs().sum() > 0 and left.tolist() == [40, 40, 40]
assert ops.error_flags() == 0
print("captured")
"""


def test_the_first_calls_of_a_process_can_be_captured():
    """No call before the capture: nothing of it needs one."""
    got = subprocess.run([sys.executable, "-c", CAPTURE], capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and "captured" in got.stdout, got.stderr[-2000:]


@pytest.mark.parametrize("T,keep", [(40000, 7001), (33000, 32900)])
def test_eviction_of_more_weights_than_a_cta_holds(T, keep):
    rng = np.random.default_rng(T)
    H, hd, block = 2, 16, 64
    cap = -(-T // block) * block
    g = torch.Generator(device=DEV).manual_seed(T)
    cache = make_cache(g, 1, H, cap, hd, block)
    arrays = [t.cpu().numpy().copy() for t in cache]
    mass = (rng.integers(0, 5000, (1, H, cap)) / 7).astype(np.float32)
    m = torch.as_tensor(mass).to(DEV)
    kept, left = ops.kvb_evict(cache, m, i32([T]), keep, sink=4, recent=100)
    want, n = R.evict(*arrays, mass, [T], keep, 4, 100)
    assert np.array_equal(kept.cpu().numpy(), want) and left.tolist() == n.tolist()
    assert all(np.array_equal(t.cpu().numpy(), a) for t, a in zip(cache, arrays))
    assert np.array_equal(m.cpu().numpy(), mass)

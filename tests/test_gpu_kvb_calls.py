"""Calls of the block-scaled KV cache's operators that depend on their surroundings."""
import pytest
import torch

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

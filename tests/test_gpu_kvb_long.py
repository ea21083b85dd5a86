"""Prompt attention over the block-scaled 8-bit KV cache where one CTA takes many
tiles of one unit: accumulators that are moved out and begun anew, rescaled on
the way, scores and V scales that jump in the middle of a unit. Compared with
float64 on the same device (the bound: kvb_ref64.py)."""
import pytest
import torch

from kvb_ref64 import DEV, TYPES, attend, check, dz_of, i32, make_cache
from torch2riscv_accelerator_b200 import ops

pytestmark = pytest.mark.gpu


def rising(H, cap, block, every):
    """Scores whose spread grows by 1.8 (their largest by 4.5, 6.5 in log2) every `every` tiles of 128 tokens, each
    head at tiles of its own."""
    tile = torch.arange(cap // block, device=DEV) * block // 128
    return 0.3 + 1.8 * ((tile + torch.arange(H, device=DEV).view(-1, 1)) // every)


def growing(H, cap, block, times):
    """V scales that grow by 2^9 `times` times, each head at tiles of its own."""
    tiles = -(-cap // 128)
    tile = torch.arange(cap // block, device=DEV) * block // 128
    level = (tile + torch.arange(H, device=DEV).view(-1, 1)) * times // (tiles + H)
    return 2.0 ** (9.0 * level - 4.5 * times)


# one unit per KV head; its tiles (200 to 700) are shared out to 148 CTAs: 9 to 38 tiles of one unit in a CTA, more than
# the 3 (16-bit types: 32) between two move-outs
@pytest.mark.parametrize("heads,kv_heads,hd,block,dt,rows,prior,jumps", [
    (16, 8, 128, 64, "fp32", 37, 25001, "none"),
    (16, 8, 128, 64, "fp32", 37, 25001, "scores"),
    (16, 8, 128, 32, "fp32", 20, 25600, "values"),
    (8, 4, 64, 32, "fp32", 64, 51000, "scores"),
    (8, 4, 64, 16, "fp32", 3, 51000, "values"),
    (4, 4, 256, 64, "fp32", 70, 25555, "scores"),
    (4, 4, 208, 128, "fp32", 5, 25555, "values"),
    (8, 8, 64, 64, "bf16", 50, 90000, "scores"),
    (8, 8, 64, 64, "bf16", 2, 90000, "values"),
    (16, 8, 128, 128, "fp16", 40, 90011, "scores"),
    (4, 4, 256, 64, "bf16", 9, 90011, "scores")])
def test_a_long_unit_in_one_cta(heads, kv_heads, hd, block, dt, rows, prior, jumps):
    g = torch.Generator(device=DEV).manual_seed(heads * hd + rows)
    G, cap = heads // kv_heads, -(-(prior + rows) // block) * block
    every = 1 if dt == "fp32" else 8
    cache = make_cache(g, 1, kv_heads, cap, hd, block, rising(kv_heads, cap, block, every) if jumps == "scores" else None,
                       growing(kv_heads, cap, block, 12) if jumps == "values" else None)
    q = torch.randn(rows, heads, hd, generator=g, device=DEV).to(TYPES[dt])
    mass = torch.zeros(1, kv_heads, cap, device=DEV)
    pos, start = i32([prior]), i32([0, rows])
    out = ops.kvb_attn_rows(q, cache, pos, start, mass=mass)
    at = torch.arange(rows, device=DEV)
    for h in range(kv_heads):
        want, w, vabs, zabs, lost = attend(q[:, h * G:h * G + G], cache, 0, prior, at, h)
        check(out[:, h * G:h * G + G], want, vabs, zabs, lost, prior + rows, hd, dt)
        # a token's sum of probabilities: each off by 4 |dz| + ..., their addition by a step of 2^-24 a row
        rel = 4 * dz_of(zabs.max(), hd) + 2.0 ** -20 + ((prior + rows) / 32 + 16 + rows * G) * 2.0 ** -24
        sums = w.sum((0, 1))
        assert ((mass[0, h, :prior + rows].double() - sums).abs() <= rel * sums + 2.0 ** -126).all()
    assert ops.error_flags() == 0
    again = ops.kvb_attn_rows(q, cache, pos, start, mass=torch.zeros_like(mass))
    assert torch.equal(again, out)


@pytest.mark.parametrize("heads,kv_heads,hd,block,dt,rows,prior", [
    (4, 2, 128, 64, "fp32", 4096, 0),
    (9, 3, 64, 16, "fp32", 3000, 77),
    (3, 3, 256, 32, "fp32", 2500, 1),
    (8, 4, 64, 64, "bf16", 8192, 0),
    (8, 4, 112, 64, "fp16", 8000, 33)])
def test_a_long_causal_prompt(heads, kv_heads, hd, block, dt, rows, prior):
    """Rows at and beside the units' borders, and some between."""
    g = torch.Generator(device=DEV).manual_seed(heads * hd + rows)
    G, cap = heads // kv_heads, -(-(prior + rows) // block) * block
    cache = make_cache(g, 1, kv_heads, cap, hd, block)
    q = torch.randn(rows, heads, hd, generator=g, device=DEV).to(TYPES[dt])
    out = ops.kvb_attn_rows(q, cache, i32([prior]), i32([0, rows]))
    edge = torch.arange(0, rows, 128 // G if 128 % G == 0 else 128, device=DEV)[::3]
    at = torch.cat([edge, (edge - 1).clamp(min=0), torch.randint(0, rows, (64,), generator=g, device=DEV),
                    torch.tensor([rows - 1], device=DEV)]).unique()
    for h in range(kv_heads):
        want, _, vabs, zabs, lost = attend(q[at, h * G:h * G + G], cache, 0, prior, at, h)
        check(out[at, h * G:h * G + G], want, vabs, zabs, lost, prior + rows, hd, dt)
    assert ops.error_flags() == 0

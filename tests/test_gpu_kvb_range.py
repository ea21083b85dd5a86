"""Attention over the block-scaled 8-bit KV cache at the ends of fp32's range: blocks
of V far larger than the others that a row does not see or gives no weight, tiny and
huge values. Compared with float64 (the bound: kvb_ref64.py)."""
import pytest
import torch

from kvb_ref64 import DEV, TYPES, attend, check, i32, make_cache
from torch2riscv_accelerator_b200 import ops

pytestmark = pytest.mark.gpu


def compare(q, cache, pos, start, dt, hd, n, scale=None, rows=True):
    """Every row of every slot against float64."""
    if rows:
        out = ops.kvb_attn_rows(q, cache, i32(pos), i32(start), scale=scale)
    else:
        out = ops.kvb_attn(q, cache, i32(pos), scale=scale)
    H = cache.k.shape[1]
    G = q.shape[1] // H
    for b, p in enumerate(pos):
        a, e = (start[b], start[b + 1]) if rows else (b, b + 1)
        if e == a or p < 0:
            continue
        at = torch.arange(e - a, device=DEV)
        for h in range(H):
            want, _, vabs, zabs, lost = attend(q[a:e, h * G:h * G + G], cache, b, p, at, h, scale, not rows)
            check(out[a:e, h * G:h * G + G], want, vabs, zabs, lost, n, hd, dt)
    return out


@pytest.mark.parametrize("big", [2.0 ** 12, 2.0 ** 25, 2.0 ** 40, 2.0 ** 60, 1e35])
@pytest.mark.parametrize("heads,kv_heads,hd,block,dt", [
    (4, 2, 64, 16, "fp32"), (16, 8, 128, 64, "fp32"), (3, 3, 256, 32, "fp32"), (8, 2, 80, 64, "bf16"),
    (4, 4, 128, 16, "fp16")])
def test_a_large_block_behind_a_row_does_not_reach_it(heads, kv_heads, hd, block, dt, big):
    """The last block of each prompt holds V's far larger than the others: the rows before it do not see it."""
    if dt == "fp16" and big > 2.0 ** 12:
        pytest.skip("outputs of the rows that do see it leave fp16")
    g = torch.Generator(device=DEV).manual_seed(hd)
    cap = 320
    cache = make_cache(g, 3, kv_heads, cap, hd, block)
    counts, pos = [300, 130, 64], [0, 50, 200]
    for b in range(3):
        cache.v_scale[b, :, (pos[b] + counts[b] - 1) // block] *= big
    start = [0, 300, 430, 494]
    q = torch.randn(494, heads, hd, generator=g, device=DEV).to(TYPES[dt])
    compare(q, cache, pos, start, dt, hd, cap)


def test_an_infinity_in_the_last_value_leaves_earlier_rows():
    """Appended as the largest finite value: the rows of the blocks before give what they gave without it."""
    g = torch.Generator(device=DEV).manual_seed(1)
    q, k, v = (torch.randn(100, 2, 64, generator=g, device=DEV) for _ in range(3))
    bad = v.clone()
    bad[99, 0, 5] = float("inf")
    out = []
    for x in (v, bad):
        cache = ops.kvb_cache(1, 2, 128, 64, block=16)
        ops.kvb_append(k, x, cache, i32([0]), i32([0, 100]))
        out.append(compare(q, cache, [0], [0, 100], "fp32", 64, 100))
    assert (out[1][:96] - out[0][:96]).abs().max() < 1e-5
    assert out[1][99, 0, 5] > 1e30


@pytest.mark.parametrize("heads,kv_heads,hd,block,dt", [
    (4, 2, 64, 64, "fp32"), (16, 2, 128, 16, "fp32"), (2, 1, 256, 64, "fp32"), (8, 2, 64, 32, "bf16")])
@pytest.mark.parametrize("rows", [False, True])
@pytest.mark.parametrize("big", [2.0 ** 30, 2.0 ** 100])
def test_a_large_block_without_weight_does_not_count(heads, kv_heads, hd, block, dt, big, rows):
    """Every row sees the large block, but its scores lie so far below the others that its weights are 0."""
    g = torch.Generator(device=DEV).manual_seed(hd)
    cap = 640
    cache = make_cache(g, 2, kv_heads, cap, hd, block)
    n = 70 if rows else 1
    q = torch.rand(2 * n, heads, hd, generator=g, device=DEV).add_(0.5).to(TYPES[dt])
    for j in (1, 7):                                          # keys against the queries, all other scores near 0
        cache.k[:, :, j * block:(j + 1) * block] = -127
        cache.k_scale[:, :, j] = 2.0
        cache.v_scale[:, :, j] *= big
    compare(q, cache, [500, 512], [0, n, 2 * n], dt, hd, cap, rows=rows)


@pytest.mark.parametrize("rows", [False, True])
@pytest.mark.parametrize("tiny", [1e-30, 1e-34, 1e-36, 1e-38, 1e-41, 1e-42])
@pytest.mark.parametrize("heads,kv_heads,hd,block,dt", [
    (4, 2, 64, 16, "fp32"), (16, 2, 128, 64, "fp32"), (2, 2, 256, 32, "fp32"), (8, 2, 64, 32, "bf16")])
def test_tiny_values(heads, kv_heads, hd, block, dt, tiny, rows):
    """V of any size comes back at its size, subnormal scales too; a scale of 0 is no value at all."""
    g = torch.Generator(device=DEV).manual_seed(hd)
    cache = make_cache(g, 2, kv_heads, 256, hd, block)
    cache.v_scale.mul_(tiny)
    cache.v_scale[:, :, 1] = 0                                # a block of zeros
    n = 70 if rows else 1
    q = torch.randn(2 * n, heads, hd, generator=g, device=DEV).to(TYPES[dt])
    out = compare(q, cache, [180, 5], [0, n, 2 * n], dt, hd, 256, rows=rows)
    t = torch.finfo(TYPES[dt])
    assert out.abs().max() > tiny / 100 or tiny < 100 * t.smallest_normal * t.eps      # (the type's own end)


@pytest.mark.parametrize("rows", [False, True])
@pytest.mark.parametrize("hd,dt,cap", [(64, "fp32", 2048), (128, "fp32", 2048), (256, "fp32", 2048),
                                       (128, "bf16", 2048), (64, "fp32", 17024), (128, "fp32", 8256)])
def test_huge_values(hd, dt, cap, rows):
    """V up to the largest that append writes: finite outputs, wherever a row's parts are joined (single tokens: in a
    cluster, for the long caches by a second kernel)."""
    g = torch.Generator(device=DEV).manual_seed(hd)
    cache = make_cache(g, 1, 8, cap, hd, 64)
    cache.v_scale.fill_(2.6e36)
    cache.k_scale.mul_(torch.linspace(0.1, 3.0, cap // 64, device=DEV))  # maxima that rise
    n = 70 if rows else 1
    q = torch.randn(n, 16, hd, generator=g, device=DEV).to(TYPES[dt])
    compare(q, cache, [cap - n], [0, n], dt, hd, cap, rows=rows)


@pytest.mark.parametrize("rows", [False, True])
@pytest.mark.parametrize("size", [1e2, 1e4, 2e5])
@pytest.mark.parametrize("hd,dt", [(64, "fp32"), (128, "bf16"), (256, "fp32")])
def test_scores_in_which_a_scale_is_lost(hd, dt, size, rows):
    """One token far above all others, scores of up to 2^24, V scales of very different sizes: that token's values. Its weight
    cancels but for the logarithm of V's scale (at most 2^-18 off), the exponential and two halves (2^-20)."""
    g = torch.Generator(device=DEV).manual_seed(hd)
    cache = make_cache(g, 2, 2, 256, hd, 16)
    n = 6 if rows else 1
    q = torch.ones(2 * n, 4, hd, device=DEV, dtype=TYPES[dt])
    cache.k.clamp_(-20, 20)
    cache.k_scale.fill_(size / 36)
    cache.v_scale.mul_(2.0 ** torch.linspace(-60, 60, 16, device=DEV))
    cache.v_scale[1] = cache.v_scale[1].flip(-1)
    for t in (40, 130):                                       # the other tokens' sums are below hd * 20
        cache.k[:, :, t] = 127
        pos = i32([200, 150])
        out = ops.kvb_attn_rows(q, cache, pos, i32([0, n, 2 * n])) if rows else ops.kvb_attn(q, cache, pos)
        for b in range(2):
            want = (cache.v[b, :, t].double() * cache.v_scale[b, :, t // 16, None].double()).repeat_interleave(2, 0)
            off = (out[n * b:n * b + n].double() - want).abs()
            assert (off <= (2.0 ** -18 + 2.0 ** -20 + torch.finfo(TYPES[dt]).eps / 2) * want.abs()).all(), (b, t, off.max())
        cache.k[:, :, t] = 0


@pytest.mark.parametrize("rows", [False, True])
@pytest.mark.parametrize("tiny", [1e-18, 1e-25, 1e-33, 1e-36])
@pytest.mark.parametrize("heads,kv_heads,hd,block,dt", [
    (4, 2, 64, 16, "fp32"), (16, 2, 128, 64, "fp32"), (3, 1, 256, 32, "fp32"), (8, 2, 48, 32, "bf16"),
    (24, 2, 128, 32, "bf16")])
def test_tiny_queries(heads, kv_heads, hd, block, dt, tiny, rows):
    """Queries of any size against keys, or a scale, that bring the scores back; one head of another size beside them,
    zeros in the rows."""
    g = torch.Generator(device=DEV).manual_seed(hd)
    cache = make_cache(g, 3, kv_heads, 512, hd, block)
    counts = [40, 1, 9] if rows else [1, 1, 1]
    start, pos = [0, counts[0], counts[0] + counts[1], sum(counts)], [300, 17, 500]
    q = torch.randn(start[-1], heads, hd, generator=g, device=DEV) * tiny
    q[:, :, 1::3] = 0
    q[:, 1] *= 2.0 ** -12
    q = q.to(TYPES[dt])
    compare(q, cache, pos, start, dt, hd, 512, scale=0.25 / tiny, rows=rows)
    cache.k_scale.mul_(0.1 / tiny)
    compare(q, cache, pos, start, dt, hd, 512, scale=1.0, rows=rows)


def test_subnormal_queries_of_single_tokens():
    g = torch.Generator(device=DEV).manual_seed(3)
    cache = make_cache(g, 2, 2, 256, 64, 32)
    q = torch.randn(2, 8, 64, generator=g, device=DEV) * 1e-38 * 2.0 ** -torch.arange(0, 16, 2, device=DEV).view(8, 1)
    assert (q != 0).any(-1).all()
    compare(q, cache, [255, 100], None, "fp32", 64, 256, scale=1e38, rows=False)


@pytest.mark.parametrize("rows", [False, True])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_the_largest_scales(hd, rows):
    """Scales of up to 2^126 with codes whose values are still finite, beside ordinary ones."""
    g = torch.Generator(device=DEV).manual_seed(hd)
    cache = make_cache(g, 2, 2, 512, hd, 32)
    cache.v.clamp_(-2, 2)
    cache.v_scale[:, :, 1::2] = 2.0 ** 126
    n = 40 if rows else 1
    q = torch.randn(2 * n, 4, hd, generator=g, device=DEV)
    compare(q, cache, [470, 40], [0, n, 2 * n], "fp32", hd, 512, rows=rows)


@pytest.mark.parametrize("rows", [False, True])
@pytest.mark.parametrize("tiny", [1e-2, 1e-4, 1e-7])
@pytest.mark.parametrize("heads,kv_heads,hd,cap", [(16, 8, 128, 2048), (8, 2, 64, 2048), (8, 2, 64, 17024), (4, 4, 256, 640)])
def test_a_first_token_that_takes_the_weight(heads, kv_heads, hd, cap, tiny, rows):
    """Its own values tiny: every other block's scale is far over the heaviest weight's, its weights are not."""
    g = torch.Generator(device=DEV).manual_seed(hd)
    cache = make_cache(g, 2, kv_heads, cap, hd, 64)
    cache.k[:, :, 0] = 127
    cache.v_scale[:, :, 0] *= tiny
    n = 33 if rows else 1
    q = torch.randn(2 * n, heads, hd, generator=g, device=DEV) + 0.5
    compare(q, cache, [cap - n, cap // 2], [0, n, 2 * n], "fp32", hd, cap, rows=rows)

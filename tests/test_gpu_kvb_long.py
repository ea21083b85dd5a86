"""Prompt attention over the block-scaled 8-bit KV cache where one CTA takes many
tiles of one unit: accumulators that are moved out and begun anew, rescaled on
the way, scores and V scales that jump in the middle of a unit. Compared with
float64 on the same device.

The bound, from the kernel's arithmetic, all of it over the tokens that a row
sees. A query enters with an error of at most 2^-22 of itself, the products are
exact and summed in fp32, the result is scaled and taken from the maximum (two
roundings): |dz| <= (2^-21 + (D / 16 + 2) 2^-23) max_t sum|q k_t| scale. A weight
is off by 2 |dz|, and so is the sum that divides it; the exponential, V's scale in
it and its rounding to 21 bits add 2^-20. The tensor cores round each product's
running sum towards zero by at most 2^-23: two products for 16 tokens of the
FOLD tiles between two move-outs, 2 * FOLD * 128 / 16 of them (fewer where a tile
has 64 tokens); the moved-out sums and the weights' sum are added in fp32 over n
tokens in at most n / 32 + 16 steps of 2^-24. All are relative to sum p |v|:
|do| <= (4 |dz| + 2^-20 + 16 FOLD 2^-23 + (n / 32 + 16) 2^-24) sum p |v|, and half
a step of the output's type relative to it."""
import pytest
import torch

from torch2riscv_accelerator_b200 import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
FOLD = {"fp32": 3, "bf16": 32, "fp16": 32}


def i32(a):
    return torch.tensor(list(a), dtype=torch.int32, device=DEV)


def dz_of(zabs, hd):
    return (2.0 ** -21 + (hd / 16 + 2) * 2.0 ** -23) * zabs


def attend(q, cache, b, p, rows, h, scale=None):
    """Rows (indices i at positions p + i) of one slot and KV head in float64: q [n, G, D] of these rows -> their
    outputs, probabilities [n, G, T], sum p |v|, max sum|q k| scale over the tokens that each sees, and what subnormal
    halves may lose."""
    k, ks, v, vs = cache
    B, D = k.shape[2] // ks.shape[2], k.shape[3]
    T = p + int(rows.max()) + 1
    of = torch.arange(T, device=DEV) // B
    sv = vs[b, h].double()[of]
    kd, vd = k[b, h, :T].double() * ks[b, h].double()[of, None], v[b, h, :T].double() * sv[:, None]
    hidden = torch.arange(T, device=DEV) > (p + rows).view(-1, 1, 1)
    q = q.double()
    scale = D ** -0.5 if scale is None else scale
    w = torch.softmax((q @ kd.T * scale).masked_fill(hidden, -float("inf")), -1)
    zabs = ((q.abs() @ kd.abs().T) * abs(scale)).masked_fill(hidden, 0.0).amax(-1, keepdim=True)
    most = sv.expand_as(w).masked_fill(hidden, 0.0).amax(-1, keepdim=True)
    lost = torch.minimum(2 * w * sv, 2.0 ** -31 * most).masked_fill(hidden, 0.0) @ v[b, h, :T].double().abs()
    return w @ vd, w, w @ vd.abs(), zabs, lost


def check(got, want, vabs, zabs, lost, n, hd, dt):
    rel = 4 * dz_of(zabs, hd) + 2.0 ** -20 + 16 * FOLD[dt] * 2.0 ** -23 + (n / 32 + 16) * 2.0 ** -24
    t = torch.finfo(TYPES[dt])
    tol = rel * vabs + t.eps / 2 * want.abs() + lost + t.smallest_normal * t.eps / 2
    off = (got.double() - want).abs()
    assert got.isfinite().all()
    assert (off <= tol).all(), (off.max().item(), tol.flatten()[(off - tol).argmax()].item(), (off / tol).max().item())


def make_cache(g, S, H, cap, hd, block, k_std=None, v_scale=None):
    """Codes over the whole range; k_std, v_scale [H, blocks]: a head's scores' spread for unit queries, its V scales."""
    code = lambda: (torch.randn(S, H, cap, hd, generator=g, device=DEV) * 36).round().clamp(-127, 127).to(torch.int8)
    nb = cap // block
    plain = torch.exp(0.25 * torch.randn(S, H, nb, generator=g, device=DEV)) / 36
    ks = plain if k_std is None else (k_std / 36).expand(S, H, nb).contiguous()
    vs = torch.exp(0.25 * torch.randn(S, H, nb, generator=g, device=DEV)) / 36
    if v_scale is not None:
        vs = vs * v_scale
    return ops.KvBlocks(code(), ks.float(), code(), vs.float().contiguous())


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

"""The block-scaled 8-bit KV cache on the GPU: append and eviction bit for bit
with their float32 steps in NumPy, attention against float64.

The attention's bound, from its arithmetic: a query enters the products with an
error of at most 2^-22 of itself, the products are exact and summed in fp32
(at most one step of 2^-23 per 16 channels and two roundings of the result):
|dz| <= (2^-21 + (D / 16) 2^-23) sum|q k| scale, plus 2^-23 |z| of the scaling.
A weight exp(z - m) is then off by at most 2 |dz| (its own score and the
maximum's) and 2^-21 relative (the exponential, its rounding to 22 bits), the
sums over n tokens by (n / 16 + 8) 2^-23 relative to sum p |v|. Against
max |v|: |do| <= (4 |dz| + 2^-20 + (n / 16 + 8) 2^-22) max|v|, and half a step
of the output's type, eps / 2, relative to it."""
import numpy as np
import pytest
import torch

import kvb_ref as R
from torch2riscv_accelerator_b200 import ops

pytestmark = pytest.mark.gpu
F = np.float32
DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def cu(a, dt=None):
    return torch.as_tensor(np.ascontiguousarray(a)).to(DEV, dt)


def i32(a):
    return torch.tensor(list(a), dtype=torch.int32, device=DEV)


def host(t):
    torch.cuda.synchronize()
    return t.detach().cpu().numpy()


def random_cache(rng, slots, heads, cap, hd, block, spread=0.5):
    """Cache arrays (k, ks, v, vs) with codes over the whole range and scales of different sizes per block."""
    code = lambda: np.clip(np.rint(rng.standard_normal((slots, heads, cap, hd)) * 36), -127, 127).astype(np.int8)
    scale = lambda: (np.exp(spread * rng.standard_normal((slots, heads, cap // block))) / 36).astype(F)
    return code(), scale(), code(), scale()


def on_gpu(cache):
    return ops.KvBlocks(*(cu(a) for a in cache))


def same(got, want):
    for g, w in zip(got, want):
        g = host(g)
        assert g.dtype == w.dtype and np.array_equal(g, w), (g.shape, np.argwhere(g != w)[:4])


def rounded(rng, shape, dt, std=1.0):
    """Random rows of the type, and their values as float64."""
    t = torch.as_tensor(rng.standard_normal(shape) * std).to(dt)
    return t.to(DEV), t.double().numpy()


def check_attn(got, ref, q_dtype, n_tokens, hd):
    out, zabs, vmax = ref
    dz = (2.0 ** -21 + hd / 16 * 2.0 ** -23 + 2.0 ** -23) * zabs
    tol = (4 * dz + 2.0 ** -20 + (n_tokens / 16 + 8) * 2.0 ** -22) * vmax + torch.finfo(q_dtype).eps / 2 * np.abs(out)
    g = got.double().cpu().numpy()
    assert np.isfinite(g).all()
    bad = np.abs(g - out) > tol
    assert not bad.any(), (np.argwhere(bad)[:4], np.abs(g - out).max(), tol[bad][:4])


def check_mass(got, want, base, zabs_max, n_tokens, hd):
    """mass - base: a sum of probabilities, each off by (2 |dz| + 2^-20 + ...) of itself; the addition to the base rounds."""
    dz = (2.0 ** -21 + hd / 16 * 2.0 ** -23 + 2.0 ** -23) * zabs_max
    g = host(got).astype(np.float64)
    tol = (4 * dz + 2.0 ** -20 + (n_tokens / 16 + 8) * 2.0 ** -22) * (want - base) + 2.0 ** -22 * np.abs(want)
    assert (np.abs(g - want) <= tol).all(), np.abs(g - want).max()


# ----------------------------------------------------------------- append
@pytest.mark.parametrize("hd,block,dt", [(16, 16, "fp32"), (48, 32, "bf16"), (64, 64, "fp16"), (80, 128, "fp32"),
                                         (128, 64, "bf16"), (256, 16, "fp32")])
def test_append_rows_and_single_tokens(hd, block, dt):
    """Ragged prompts, then single tokens, over a cache with garbage in it: idle
    slots, an empty sequence, rows behind the last one, odd positions."""
    rng = np.random.default_rng(hd + block)
    S, H, cap = 5, 3, 3 * block
    cache = random_cache(rng, S, H, cap, hd, block)
    dev = on_gpu(cache)
    pos = [0, 7, -1, block + 3, block - 1]
    counts = [2 * block + 5, 1, 2, 0, block + 2]
    start = np.concatenate([[0], np.cumsum(counts)])
    rows = start[-1] + 3
    wide, w64 = rounded(rng, (rows, 3 * H, hd), TYPES[dt], 2.0)          # k and v as slices of wider rows
    w32 = w64.astype(F)
    ops.kvb_append(wide[:, H:2 * H], wide[:, 2 * H:], dev, i32(pos), i32(start))
    R.append(w32[:start[-1], H:2 * H], cache[0], cache[1], pos, start)
    R.append(w32[:start[-1], 2 * H:], cache[2], cache[3], pos, start)
    same(dev, cache)
    at = [p + n for p, n in zip(pos, counts)]
    at[2] = -1
    for step in range(3):                                                # growing values: the older codes are rescaled
        k, k64 = rounded(rng, (S, H, hd), TYPES[dt], 2.0 ** step)
        v, v64 = rounded(rng, (S, H, hd), TYPES[dt], 0.5)
        ops.kvb_append(k, v, dev, i32(at))
        R.append(k64.astype(F), cache[0], cache[1], at)
        R.append(v64.astype(F), cache[2], cache[3], at)
        same(dev, cache)
        at = [p + 1 if p >= 0 else p for p in at]
    assert ops.error_flags() == 0


def test_append_values_out_of_the_ordinary():
    """NaN, infinities, zeros, subnormal rows and exact halves of a code."""
    S, H, hd, block = 6, 1, 16, 16
    x = np.zeros((S, H, hd), F)
    x[0, 0, :4] = [np.nan, 1.0, -2.0, 0.5]
    x[1, 0, :3] = [np.inf, -np.inf, 3e38]
    x[3, 0, :3] = [1e-45, -3e-45, 2e-44]
    x[4, 0] = np.arange(16) * 0.5 - 4 + 0.0
    x[4, 0, 0] = 127.0
    x[5, 0] = (np.arange(16) - 8) * 1.0000001
    cache = tuple(np.zeros((S, H, block, hd), np.int8) if i % 2 == 0 else np.zeros((S, H, 1), F) for i in range(4))
    dev = on_gpu(cache)
    ops.kvb_append(cu(x), cu(-x), dev, i32([0] * S))
    R.append(x, cache[0], cache[1], [0] * S)
    R.append(-x, cache[2], cache[3], [0] * S)
    same(dev, cache)
    k, v = ops.kvb_read(dev, i32([0] * S), None, S)
    assert np.isfinite(host(k)).all() and (host(k)[2] == 0).all()


def test_rows_past_the_capacity_are_skipped_and_flagged():
    rng = np.random.default_rng(3)
    S, H, hd, block = 2, 2, 32, 16
    cache = random_cache(rng, S, H, 2 * block, hd, block)
    dev = on_gpu(cache)
    ops.error_flags()
    x, x64 = rounded(rng, (20, H, hd), torch.float32)
    pos, start = [20, 2 ** 31 - 5], [0, 14, 20]
    ops.kvb_append(x, x, dev, i32(pos), i32(start))
    R.append(x64.astype(F), cache[0], cache[1], pos, start)
    R.append(x64.astype(F), cache[2], cache[3], pos, start)
    same(dev, cache)
    assert ops.error_flags() == 128
    q, q64 = rounded(rng, (20, 4, hd), torch.float32)
    out = ops.kvb_attn_rows(q, dev, i32(pos), i32(start))
    check_attn(out, R.attend(q64, *cache, pos, start), torch.float32, 32, hd)
    assert (host(out)[12:] == 0).all() and ops.error_flags() == 128
    k, _ = ops.kvb_read(dev, i32(pos), i32(start), 20)
    assert (host(k)[12:] == 0).all() and (host(k)[:12] != 0).any() and ops.error_flags() == 128
    # offsets out of order or out of range lead nowhere
    bad = i32([0, 9999, -5])
    ops.kvb_append(x, x, dev, i32([0, 0]), bad)
    ops.kvb_attn_rows(q, dev, i32([0, 0]), bad)
    ops.error_flags()


@pytest.mark.parametrize("dt", list(TYPES))
def test_read_gives_the_values(dt):
    rng = np.random.default_rng(8)
    cache = random_cache(rng, 3, 2, 96, 48, 32)
    dev = on_gpu(cache)
    pos, start = [5, -1, 90], [0, 11, 13, 19]
    k = torch.full((22, 2, 48), 7.0, dtype=TYPES[dt], device=DEV)
    v = torch.full((22, 2, 48), 7.0, dtype=TYPES[dt], device=DEV)
    ops.kvb_read(dev, i32(pos), i32(start), 22, dtype=TYPES[dt], k=k, v=v)
    for got, c, s in ((k, cache[0], cache[1]), (v, cache[2], cache[3])):
        val = torch.as_tensor(c.astype(F) * np.repeat(s, 32, 2)[..., None]).to(TYPES[dt])
        assert torch.equal(got[:11].cpu(), val[0, :, 5:16].transpose(0, 1))
        assert (got[11:13] == 0).all() and (got[19:] == 7).all()
        assert torch.equal(got[13:19].cpu(), val[2, :, 90:].transpose(0, 1))


# -------------------------------------------------------------- attention
@pytest.mark.parametrize("heads,kv_heads,hd,block,dt,lens", [
    (4, 2, 64, 64, "fp32", [1, 2, 63, 64, 65, 0, 200]),
    (16, 8, 128, 64, "fp32", [1000, 999, 1]),
    (9, 3, 64, 16, "bf16", [130, 17, 16, 15, 0]),
    (6, 6, 48, 32, "fp16", [256, 31, 33, 5]),
    (8, 1, 80, 128, "fp32", [300, 128, 129]),
    (16, 1, 96, 32, "bf16", [70, 500]),
    (10, 1, 16, 16, "fp32", [3, 90]),
    (4, 2, 256, 64, "fp32", [260, 64, 1]),
    (2, 2, 112, 16, "fp16", [1, 3000]),
    (24, 1, 32, 64, "fp32", [77])])
def test_step_attention_and_mass(heads, kv_heads, hd, block, dt, lens):
    rng = np.random.default_rng(heads * hd + block)
    S = len(lens)
    cap = -(-max(lens) // block) * block + block
    cache = random_cache(rng, S, kv_heads, cap, hd, block)
    for b, n in enumerate(lens):                                          # blocks past the length are never read
        cache[1][b, :, -(-n // block):] = np.nan
        cache[3][b, :, -(-n // block):] = np.nan
    dev = on_gpu(cache)
    pos = [n - 1 for n in lens]
    qkv, q64 = rounded(rng, (S, heads + 2 * kv_heads, hd), TYPES[dt], 1.5)
    base = rng.random((S, kv_heads, cap)).astype(F)
    mass = cu(base)
    out = ops.kvb_attn(qkv[:, :heads], dev, i32(pos), mass=mass)
    want_mass = base.astype(np.float64)
    ref = R.attend(q64[:, :heads], *cache, pos, mass=want_mass)
    check_attn(out, ref, TYPES[dt], max(lens), hd)
    check_mass(mass, want_mass, base, ref[1].max(), max(lens), hd)
    assert all((host(out.float())[b] == 0).all() for b, n in enumerate(lens) if n == 0)
    again = ops.kvb_attn(qkv[:, :heads], dev, i32(pos))                   # without mass: the same rows, every time
    assert torch.equal(again, out) and torch.equal(ops.kvb_attn(qkv[:, :heads], dev, i32(pos)), out)


@pytest.mark.parametrize("heads,kv_heads,hd,block,dt,pos,counts,pad", [
    (4, 2, 64, 64, "fp32", [0], [1], 0),
    (4, 2, 64, 64, "fp32", [0, 5, -1, 63], [130, 0, 3, 70], 5),
    (16, 8, 128, 64, "fp32", [100], [256], 0),
    (9, 3, 64, 16, "bf16", [0, 77, 15], [33, 200, 1], 2),
    (6, 6, 48, 32, "fp16", [31, 0], [64, 129], 0),
    (8, 1, 80, 128, "fp32", [0, 127], [100, 30], 1),
    (16, 1, 96, 32, "bf16", [3], [150], 0),
    (10, 1, 16, 16, "fp32", [200], [18], 0),
    (4, 2, 256, 64, "fp32", [70, 0], [65, 31], 0),
    (2, 1, 112, 32, "fp16", [0], [513], 0),
    (3, 1, 32, 128, "fp32", [900, 10], [17, 300], 3)])
def test_prompt_attention_and_mass(heads, kv_heads, hd, block, dt, pos, counts, pad):
    rng = np.random.default_rng(heads * hd + block + sum(counts))
    S, lens = len(pos), [p + n if p >= 0 else 0 for p, n in zip(pos, counts)]
    cap = -(-max(lens) // block) * block + block
    cache = random_cache(rng, S, kv_heads, cap, hd, block)
    for b, n in enumerate(lens):
        cache[1][b, :, -(-n // block):] = np.nan
        cache[3][b, :, -(-n // block):] = np.nan
    dev = on_gpu(cache)
    start = np.concatenate([[0], np.cumsum(counts)])
    rows = start[-1] + pad
    qkv, q64 = rounded(rng, (rows, heads + 2 * kv_heads, hd), TYPES[dt], 1.5)
    base = rng.random((S, kv_heads, cap)).astype(F)
    mass, out = cu(base), torch.full((rows, heads, hd), 7.0, dtype=TYPES[dt], device=DEV)
    ops.kvb_attn_rows(qkv[:, :heads], dev, i32(pos), i32(start), out=out, mass=mass)
    want_mass = base.astype(np.float64)
    ref = R.attend(q64[:start[-1], :heads], *cache, pos, start, mass=want_mass)
    check_attn(out[:start[-1]], ref, TYPES[dt], max(lens), hd)
    assert (host(out.float())[start[-1]:] == 7).all()
    live = np.array([n > 0 and p >= 0 for p, n in zip(pos, counts)])
    assert np.array_equal(host(mass)[~live], base[~live])
    check_mass(mass, want_mass, base, ref[1].max(), max(lens), hd)
    again = torch.full_like(out, 7.0)
    ops.kvb_attn_rows(qkv[:, :heads], dev, i32(pos), i32(start), out=again)
    assert torch.equal(again, out)


@pytest.mark.parametrize("rows", [False, True])
def test_scores_far_apart_and_a_given_scale(rows):
    """Scores of +-thousands: the running maximum rises late, early weights vanish; scale 0 weighs all tokens alike."""
    rng = np.random.default_rng(11)
    cache = list(random_cache(rng, 1, 1, 512, 64, 64))
    cache[1][0, 0] = [1e-3, 1e-3, 0.0, 10.0, 0.1, 30.0, 1e-3, 1.0]
    cache[3][0, 0, 2] = 0.0
    dev = on_gpu(cache)
    n = 17 if rows else 1
    q, q64 = rounded(rng, (n, 2, 64), torch.float32, 3.0)
    pos, start = [511 - n + 1], [0, n]
    for scale in (None, 0.0, 1.0):
        if rows:
            out = ops.kvb_attn_rows(q, dev, i32(pos), i32(start), scale=scale)
        else:
            out = ops.kvb_attn(q, dev, i32(pos), scale=scale)
        ref = R.attend(q64, *cache, pos, start, scale=scale)
        check_attn(out, ref, torch.float32, 512, 64)


def test_strided_slots_and_a_long_head():
    """One layer of a [slots, layers, ...] cache, and codes past 2^31 from the cache's start."""
    rng = np.random.default_rng(5)
    S, L, H, cap, hd, B = 3, 2, 2, 128, 64, 32
    whole = random_cache(rng, S * L, H, cap, hd, B)
    big = [cu(a).view(S, L, *a.shape[1:]) for a in whole]
    layer = tuple(t[:, 1] for t in big)
    arrays = tuple(host(t).copy() for t in layer)
    q, q64 = rounded(rng, (S, 4, hd), torch.float32)
    pos = [100, 3, 127]
    check_attn(ops.kvb_attn(q, layer, i32(pos)), R.attend(q64, *arrays, pos), torch.float32, 128, hd)
    k, k64 = rounded(rng, (S, H, hd), torch.float32, 3.0)
    other = [t[:, 0].clone() for t in big]
    ops.kvb_append(k, k, layer, i32(pos))
    for c, s in ((arrays[0], arrays[1]), (arrays[2], arrays[3])):
        R.append(k64.astype(F), c, s, pos)
    same(layer, arrays)
    assert all(torch.equal(t[:, 0], o) for t, o in zip(big, other))
    del big, layer, other

    cap, H = 1 << 21, 9                                                   # 9 heads x 2^21 tokens x 128 codes > 2^31
    cache = ops.kvb_cache(1, H, cap, 128, 128)
    k, k64 = rounded(rng, (1, H, 128), torch.float32)
    v, v64 = rounded(rng, (1, H, 128), torch.float32)
    ops.kvb_append(k, v, cache, i32([cap - 1]))
    rk, rv = ops.kvb_read(cache, i32([cap - 1]), None, 1)
    vals = host(rv)[0].astype(np.float64)
    assert np.abs(host(rk)[0] - k64[0]).max() <= np.abs(k64).max() / 127
    q = torch.as_tensor(k64 * 4).to(torch.float32).to(DEV)               # the last token against 2^21 - 1 zeros
    out = host(ops.kvb_attn(q, cache, i32([cap - 1])).double())[0]
    z = (host(q)[0].astype(np.float64) * host(rk)[0].astype(np.float64)).sum(1) / np.sqrt(128)
    w = np.exp(z) / (np.exp(z) + cap - 1)
    # sums over 2^21 weights; the weight itself is off by 2 |dz|
    assert np.abs(out - w[:, None] * vals).max() <= np.abs(vals).max() * 2.0 ** -13


# ----------------------------------------------------------------- evict
@pytest.mark.parametrize("hd,block,keep,sink,recent,counts", [
    (64, 64, 100, 4, 32, [256, 100, 99, 0, 101, 255]),
    (128, 16, 33, 0, 0, [200, 34]),
    (48, 32, 64, 0, 64, [65, 96]),
    (16, 128, 1, 0, 0, [256, 1]),
    (256, 64, 129, 129, 0, [200, 250]),
    (80, 16, 250, 3, 5, [256, 251, -1]),
    (112, 32, 256, 1, 1, [256, 300])])
@pytest.mark.parametrize("inplace", [True, False])
def test_evict(hd, block, keep, sink, recent, counts, inplace):
    rng = np.random.default_rng(hd + keep)
    S, H, cap = len(counts), 2, 256
    cache = random_cache(rng, S, H, cap, hd, block)
    mass = (rng.random((S, H, cap)) ** 4).astype(F)
    mass[:, :, 10:60] = np.where(rng.random((S, H, 50)) < 0.5, 0.0, -0.0)  # ties, signed zeros
    mass[:, 0, 5:9] = [np.nan, np.inf, -np.inf, np.nan]
    dev, m = on_gpu(cache), cu(mass)
    if inplace:
        kept, left = ops.kvb_evict(dev, m, i32(counts), keep, sink=sink, recent=recent)
        want, n = R.evict(*cache, mass, counts, keep, sink, recent)
        same(dev, cache)
    else:
        dst = random_cache(rng, S, H, 256, hd, block)
        dmass = rng.random((S, H, 256)).astype(F)
        d, dm = on_gpu(dst), cu(dmass)
        before = [t.clone() for t in dev] + [m.clone()]
        kept, left = ops.kvb_evict(dev, m, i32(counts), keep, sink=sink, recent=recent, dst=d, dst_mass=dm)
        want, n = R.evict(*cache, mass, counts, keep, sink, recent, dst, dmass)
        same(d, dst)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip([*dev, m], before))
        m, mass = dm, dmass
    assert np.array_equal(host(kept), want) and np.array_equal(host(left), n)
    assert np.array_equal(host(m), mass, equal_nan=True)
    assert ops.error_flags() == (128 if max(counts) > cap else 0)


@pytest.mark.parametrize("T,keep", [(6000, 2999), (20000, 512), (16384, 16000)])
def test_evict_long(T, keep):
    """Long slots: segments of many tokens per CTA and several compaction rounds, into a smaller cache and in place."""
    rng = np.random.default_rng(T)
    S, H, hd, block = 2, 1, 32, 32
    cap = -(-T // block) * block
    cache = random_cache(rng, S, H, cap, hd, block)
    mass = (rng.integers(0, 400, (S, H, cap)) / 7).astype(F)               # many ties
    counts = [T, T - 77]
    dev, m = on_gpu(cache), cu(mass)
    small = ops.kvb_cache(S, H, keep, hd, block)
    dm = torch.full((S, H, small.k.shape[2]), 5.0, device=DEV)
    kept2, _ = ops.kvb_evict(dev, m, i32(counts), keep, sink=4, recent=100, dst=small, dst_mass=dm)
    kept, _ = ops.kvb_evict(dev, m, i32(counts), keep, sink=4, recent=100)
    want, _ = R.evict(*cache, mass, counts, keep, 4, 100)
    same(dev, cache)
    assert np.array_equal(host(kept), want) and torch.equal(kept, kept2) and np.array_equal(host(m), mass)
    nb = -(-keep // block)
    assert torch.equal(small.k[:, :, :keep], dev.k[:, :, :keep]) and torch.equal(small.v_scale, dev.v_scale[:, :, :nb])
    assert torch.equal(dm[:, :, :keep], m[:, :, :keep])


# ------------------------------------------------------- used together
def test_prompt_steps_and_eviction_together():
    """As a serving loop uses them: prompts in chunks with their weights
    gathered, single steps, a cut to a budget, more steps after it."""
    rng = np.random.default_rng(21)
    S, heads, H, hd, block, keep = 3, 6, 2, 64, 32, 70
    cap = 192
    dev, mass = ops.kvb_cache(S, H, cap, hd, block), torch.zeros(S, H, cap, device=DEV)
    cache = [host(t).copy() for t in dev]
    m64 = np.zeros((S, H, cap))
    pos = [0, 0, 0]
    zmax = 0.0

    def put(counts, start):
        nonlocal zmax
        rows = sum(counts)
        qkv, x64 = rounded(rng, (rows, heads + 2 * H, hd), torch.float32, 1.2)
        st = None if start is None else i32(start)
        ops.kvb_append(qkv[:, heads:heads + H], qkv[:, heads + H:], dev, i32(pos), st)
        R.append(x64[:, heads:heads + H].astype(F), cache[0], cache[1], pos, start)
        R.append(x64[:, heads + H:].astype(F), cache[2], cache[3], pos, start)
        if start is None:
            out = ops.kvb_attn(qkv[:, :heads], dev, i32(pos), mass=mass)
        else:
            out = ops.kvb_attn_rows(qkv[:, :heads], dev, i32(pos), st, mass=mass)
        ref = R.attend(x64[:, :heads], *cache, pos, start, mass=m64)
        check_attn(out, ref, torch.float32, cap, hd)
        zmax = max(zmax, ref[1].max())
        for b in range(S):
            pos[b] += counts[b]

    for counts in ([50, 3, 90], [33, 64, 1]):
        put(counts, np.concatenate([[0], np.cumsum(counts)]))
    for _ in range(4):
        put([1, 1, 1], None)
    same(dev, cache)
    check_mass(mass, m64, np.zeros_like(m64), zmax, cap, hd)
    m32 = host(mass).copy()                                               # the cut goes by the weights as gathered
    kept, left = ops.kvb_evict(dev, mass, i32(pos), keep, sink=2, recent=16)
    want, n = R.evict(*cache, m32, pos, keep, 2, 16)
    same(dev, cache)
    assert np.array_equal(host(kept), want) and np.array_equal(host(left), n)
    m64 = m32.astype(np.float64)
    pos = list(n)
    for _ in range(3):
        put([1, 1, 1], None)
    same(dev, cache)


def test_graph_replay_streams_and_two_calls_at_once():
    """A captured step (append, attention with weights) replayed with new
    inputs; the same calls on two streams at once, each with its own scratch."""
    rng = np.random.default_rng(31)
    S, heads, H, hd, block, cap = 4, 8, 2, 128, 64, 512
    arrays = random_cache(rng, S, H, cap, hd, block)
    a, b = on_gpu(arrays), on_gpu(arrays)
    qkv = torch.zeros(S, heads + 2 * H, hd, device=DEV)
    pos, mass, out = i32([0] * S), torch.zeros(S, H, cap, device=DEV), torch.zeros(S, heads, hd, device=DEV)

    def step(cache, q, p, m, o):
        ops.kvb_append(q[:, heads:heads + H], q[:, heads + H:], cache, p)
        ops.kvb_attn(q[:, :heads], cache, p, mass=m, out=o)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(a, qkv, pos, mass, out)
    torch.cuda.current_stream().wait_stream(side)
    for t, w in zip(a, arrays):
        t.copy_(cu(w))
    mass.zero_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(a, qkv, pos, mass, out)
    m2 = torch.zeros_like(mass)
    for i in range(3):
        x = torch.randn(S, heads + 2 * H, hd, device=DEV)
        p = i32([100 * i, 5, -1, 300 + i])
        qkv.copy_(x)
        pos.copy_(p)
        g.replay()
        o2 = torch.empty_like(out)
        step(b, x, p, m2, o2)
        assert torch.equal(out, o2) and torch.equal(mass, m2)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    p = i32([511, 200, 64, 0])
    q = torch.randn(S, heads, hd, device=DEV)
    want = ops.kvb_attn(q, a, p)
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for s in (s1, s2):
            with torch.cuda.stream(s):
                got.append(ops.kvb_attn(q, a, p))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


def test_torch_ops():
    """torch.ops.w8a8.kvb_* do what the ops calls do."""
    import torch2riscv_accelerator_b200.torch_ops  # noqa: F401
    rng = np.random.default_rng(41)
    arrays = random_cache(rng, 2, 2, 96, 32, 32)
    a, b = on_gpu(arrays), on_gpu(arrays)
    k = torch.randn(9, 2, 32, device=DEV)
    q = torch.randn(9, 4, 32, device=DEV)
    pos, start = i32([3, 60]), i32([0, 4, 8])
    m1, m2 = torch.zeros(2, 2, 96, device=DEV), torch.zeros(2, 2, 96, device=DEV)
    ops.kvb_append(k, -k, a, pos, start)
    torch.ops.w8a8.kvb_append(k, -k, *b, pos, start)
    want = ops.kvb_attn_rows(q, a, pos, start, mass=m1, out=torch.zeros_like(q))
    assert torch.equal(torch.ops.w8a8.kvb_attn_rows(q, *b, pos, start, m2), want) and torch.equal(m1, m2)
    assert torch.equal(torch.ops.w8a8.kvb_attn(q[:2], *b, pos, None), ops.kvb_attn(q[:2], a, pos))
    got, want = torch.ops.w8a8.kvb_read(*b, pos, start, 9), ops.kvb_read(a, pos, start, 9)
    assert all(torch.equal(x[:8], y[:8]) and (x[8] == 0).all() for x, y in zip(got, want))
    got, want = torch.ops.w8a8.kvb_evict(*b, m2, i32([7, 64]), 6, 1, 2), ops.kvb_evict(a, m1, i32([7, 64]), 6, 1, 2)
    assert all(torch.equal(x, y) for x, y in zip(got, want)) and all(torch.equal(x, y) for x, y in zip(a, b))
    assert torch.equal(m1, m2)


# ------------------------------------------------------- the forms for many units
@pytest.mark.parametrize("heads,kv_heads,hd,block,dt,S,cap,mass", [
    (6, 3, 64, 32, "fp32", 120, 192, True),
    (8, 2, 64, 64, "bf16", 150, 128, False),
    (12, 4, 128, 64, "fp32", 60, 320, True),
    (16, 2, 128, 16, "fp16", 70, 208, True),
    (9, 9, 112, 16, "fp32", 40, 160, False),
    (4, 2, 256, 64, "fp32", 40, 256, True),
    (12, 1, 208, 16, "bf16", 90, 96, True),
    (4, 2, 64, 128, "fp32", 1, 20096, True),
    (2, 1, 128, 128, "fp16", 2, 16512, False),
    (4, 2, 128, 64, "fp32", 2, 4160, True),
    (2, 1, 32, 16, "fp32", 700, 48, True)])
def test_step_attention_of_many_slots_and_long_ones(heads, kv_heads, hd, block, dt, S, cap, mass):
    """Sequences of every length up to the capacity, idle ones between them."""
    rng = np.random.default_rng(heads * hd + S)
    cache = random_cache(rng, S, kv_heads, cap, hd, block)
    pos = rng.integers(0, cap, S)
    pos[-1], pos[:S // 5] = cap - 1, -1
    dev = on_gpu(cache)
    q, q64 = rounded(rng, (S, heads, hd), TYPES[dt], 1.5)
    m, want = torch.zeros(S, kv_heads, cap, device=DEV), np.zeros((S, kv_heads, cap))
    out = ops.kvb_attn(q, dev, i32(pos), mass=m if mass else None)
    ref = R.attend(q64, *cache, pos, mass=want)
    check_attn(out, ref, TYPES[dt], cap, hd)
    assert (host(out.float())[pos < 0] == 0).all()
    if mass:
        check_mass(m, want, np.zeros_like(want), ref[1].max(), cap, hd)
    assert torch.equal(ops.kvb_attn(q, dev, i32(pos)), out)
    scratch = ops.kvb_attn_scratch(dev, heads, S, start=False, mass=True, dtype=TYPES[dt])
    scratch.fill_(255)                                                    # its contents do not matter
    again = torch.zeros_like(m)
    assert torch.equal(ops.kvb_attn(q, dev, i32(pos), mass=again, scratch=scratch), out)
    assert not mass or torch.equal(again, m)


@pytest.mark.parametrize("heads,kv_heads,hd,block,dt,S,cap", [
    (4, 2, 64, 64, "fp32", 160, 128), (6, 2, 128, 32, "bf16", 150, 160), (3, 3, 80, 16, "fp32", 110, 144),
    (2, 1, 256, 64, "fp16", 80, 256), (2, 1, 32, 16, "fp32", 700, 48),
    (24, 12, 48, 16, "bf16", 48, 64)])
def test_prompt_attention_of_many_slots(heads, kv_heads, hd, block, dt, S, cap):
    """Prompts of a few rows each, idle and empty ones between them."""
    rng = np.random.default_rng(heads * hd + S)
    cache = random_cache(rng, S, kv_heads, cap, hd, block)
    counts = rng.integers(0, 9, S)
    pos = rng.integers(0, cap - 8, S)
    pos[::7], counts[::5] = -1, 0
    start = np.concatenate([[0], np.cumsum(counts)])
    dev = on_gpu(cache)
    q, q64 = rounded(rng, (start[-1] + 2, heads, hd), TYPES[dt], 1.5)
    m, want = torch.zeros(S, kv_heads, cap, device=DEV), np.zeros((S, kv_heads, cap))
    scratch = ops.kvb_attn_scratch(dev, heads, q.shape[0], mass=True, dtype=TYPES[dt])
    scratch.fill_(255)
    out = torch.full_like(q, 7.0)
    ops.kvb_attn_rows(q, dev, i32(pos), i32(start), mass=m, out=out, scratch=scratch)
    ref = R.attend(q64[:start[-1]], *cache, pos, start, mass=want)
    check_attn(out[:start[-1]], ref, TYPES[dt], cap, hd)
    assert (host(out.float())[start[-1]:] == 7).all()
    check_mass(m, want, np.zeros_like(want), ref[1].max(), cap, hd)


@pytest.mark.parametrize("rows", [False, True])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_a_bad_query_row_stays_alone(rows, hd):
    """A row with a NaN or an infinity gives NaN, its neighbours what they gave without it; a negative scale."""
    rng = np.random.default_rng(hd)
    cache = random_cache(rng, 3, 2, 128, hd, 64)
    dev = on_gpu(cache)
    counts = [5, 20, 1] if rows else [1, 1, 1]
    start = np.concatenate([[0], np.cumsum(counts)])
    pos = [3, 100, 60]
    q, q64 = rounded(rng, (start[-1], 4, hd), torch.float32)
    call = lambda x: (ops.kvb_attn_rows(x, dev, i32(pos), i32(start), scale=-0.1) if rows else
                      ops.kvb_attn(x, dev, i32(pos), scale=-0.1))
    want = call(q)
    check_attn(want, R.attend(q64, *cache, pos, start, scale=-0.1), torch.float32, 128, hd)
    bad = q.clone()
    bad[1, 0, 3], bad[1, 3, 0] = float("nan"), float("-inf")
    got = call(bad)
    assert got[1, 0].isnan().all() and got[1, 3].isnan().all()
    keep = torch.ones(q.shape[:2], dtype=torch.bool, device=DEV)
    keep[1, 0] = keep[1, 3] = False
    assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("rows", [False, True])
def test_nothing_to_attend(rows):
    """Only idle slots, or no rows at all: zeros, and nothing else is touched."""
    rng = np.random.default_rng(3)
    dev = on_gpu(random_cache(rng, 3, 2, 64, 64, 64))
    m = torch.ones(3, 2, 64, device=DEV)
    if rows:
        q = torch.randn(6, 4, 64, device=DEV)
        out = torch.full_like(q, 7.0)
        ops.kvb_attn_rows(q, dev, i32([-1, -5, -1]), i32([0, 2, 2, 4]), mass=m, out=out)
        assert (out[:4] == 0).all() and (out[4:] == 7).all()
        out.fill_(7.0)
        ops.kvb_attn_rows(q, dev, i32([0, 3, 63]), i32([0, 0, 0, 0]), mass=m, out=out)
        assert (out == 7).all()
        assert ops.kvb_attn_rows(q[:0], dev, i32([0, 3, 63]), i32([0, 0, 0, 0])).shape == (0, 4, 64)
    else:
        assert (ops.kvb_attn(torch.randn(3, 4, 64, device=DEV), dev, i32([-1, -7, -1]), mass=m) == 0).all()
    assert (m == 1).all()


def test_prompts_and_eviction_captured_and_on_two_streams():
    """A captured prompt (append, attention with weights, cut in place, read-back)
    replayed with other lengths; prompt attention and many-slot steps on two
    streams at once."""
    rng = np.random.default_rng(37)
    S, heads, H, hd, block, cap, R0, keep = 3, 6, 2, 64, 32, 256, 160, 48
    arrays = random_cache(rng, S, H, cap, hd, block)
    a, b = on_gpu(arrays), on_gpu(arrays)
    qkv = torch.zeros(R0, heads + 2 * H, hd, device=DEV)
    pos, start, count = i32([0] * S), i32([0] * (S + 1)), i32([0] * S)
    mass, out, zero = torch.zeros(S, H, cap, device=DEV), torch.zeros(R0, heads, hd, device=DEV), i32([0] * S)

    def step(c, x, p, st, n, m, o):
        ops.kvb_append(x[:, heads:heads + H], x[:, heads + H:], c, p, st)
        ops.kvb_attn_rows(x[:, :heads], c, p, st, mass=m, out=o)
        kept, left = ops.kvb_evict(c, m, n, keep, sink=1, recent=9)
        return kept, left, *ops.kvb_read(c, zero, None, S)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(a, qkv, pos, start, count, mass, out)
    torch.cuda.current_stream().wait_stream(side)
    for t, w in zip(a, arrays):
        t.copy_(cu(w))
    mass.zero_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = step(a, qkv, pos, start, count, mass, out)
    m2 = torch.zeros_like(mass)
    p = [0, 0, 0]
    for counts in ([150, 3, 0], [1, 60, 99], [40, 40, 40]):
        x = torch.randn(R0, heads + 2 * H, hd, device=DEV)
        st = np.concatenate([[0], np.cumsum(counts)])
        n = [u + v for u, v in zip(p, counts)]
        for t, w in ((qkv, x), (pos, i32(p)), (start, i32(st)), (count, i32(n))):
            t.copy_(w)
        out.zero_()
        g.replay()
        o2 = torch.zeros_like(out)
        got = step(b, x, i32(p), i32(st), i32(n), m2, o2)
        assert torch.equal(out, o2) and torch.equal(mass, m2)
        assert all(torch.equal(u, v) for u, v in zip(held, got))
        assert all(torch.equal(u, v) for u, v in zip(a, b))
        p = host(got[1]).tolist()
        assert p == [min(v, keep) for v in n]
    many = on_gpu(random_cache(rng, 100, 4, 128, 64, 64))
    q1, p1 = torch.randn(100, 8, 64, device=DEV), i32(rng.integers(0, 128, 100))
    q2, p2, s2 = torch.randn(300, heads, hd, device=DEV), i32([5, 100, 0]), i32([0, 130, 200, 300])
    calls = [lambda: ops.kvb_attn(q1, many, p1), lambda: ops.kvb_attn_rows(q2[:, :, :], a, p2, s2),
             lambda: ops.kvb_attn(q2[:S], a, p2)]
    want = [f() for f in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for i in range(24):
        with torch.cuda.stream(streams[i % 3]):
            got.append((i // 3 % 3, calls[i // 3 % 3]()))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i, x in got)

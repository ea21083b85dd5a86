"""Attention over the block-scaled KV cache in float64 on the GPU, and the bound of
the kernels' outputs, all of it over the tokens that a row sees.

A query enters with an error of at most 2^-22 of itself, the products are exact and
summed in fp32, the result is scaled and taken from the maximum (two roundings):
|dz| <= (2^-21 + (D / 16 + 2) 2^-23) max_t sum|q k_t| scale. A weight is off by 2 |dz|,
and so is the sum that divides it; the exponential and its rounding to 21 bits add
2^-20, V's scale as a logarithm (up to 128 in size, rounded once) 2^-18. The tensor
cores round each product's running sum towards zero by at most 2^-23: two products for
16 tokens of the FOLD tiles of 128 between two move-outs, 2 * FOLD * 128 / 16 of them;
the moved-out sums and the weights' sum are added in fp32 over n tokens in at most
n / 32 + 16 steps of 2^-24. All are relative to sum p |v|:
(4 |dz| + 2^-20 + 2^-18 + 16 FOLD 2^-23 + (n / 32 + 16) 2^-24) sum p |v|.

A weight times V's scale, over a reference of at most twice the row's largest such (four
times for single tokens), enters as two halves that stand for 2^7 of it (2^5). Where they
are subnormal each is off by half a step of 2^-24, 2^-24 / 2^7 of the reference together,
but a weight by no more than itself: sum_t min(2^-30 max_t p_t s_t, 2 p_t s_t) |code_t|
(2^-27). The reference is at least 2^-126 of the largest weight (2^-119, and 2^-120 of it
times the largest scale). (A channel where the heaviest token holds 0 has nothing but
such weights.) The output's type rounds by half a step, relative to it and of its
smallest subnormal; parts of a row that are joined round once more."""
import torch

from torch2riscv_accelerator_b200 import ops

DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
FOLD = {"fp32": 3, "bf16": 32, "fp16": 32}


def i32(a):
    return torch.tensor(list(a), dtype=torch.int32, device=DEV)


def dz_of(zabs, hd):
    return (2.0 ** -21 + (hd / 16 + 2) * 2.0 ** -23) * zabs


def attend(q, cache, b, p, rows, h, scale=None, single=False):
    """Rows (indices i at positions p + i) of one slot and KV head in float64: q [n, G, D] of these rows -> their
    outputs, probabilities [n, G, T], sum p |v|, max sum|q k| scale, and what subnormal halves may lose."""
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
    least, step = (2.0 ** -119, 2.0 ** -27) if single else (2.0 ** -126, 2.0 ** -30)
    ref = torch.maximum((w * sv).amax(-1, keepdim=True), least * w.amax(-1, keepdim=True))
    if single:
        ref = torch.maximum(ref, 2.0 ** -120 * sv.max() * w.amax(-1, keepdim=True))
    lost = torch.minimum(2 * w * sv, step * ref) @ v[b, h, :T].double().abs()
    return w @ vd, w, w @ vd.abs(), zabs, lost


def check(got, want, vabs, zabs, lost, n, hd, dt):
    rel = 4 * dz_of(zabs, hd) + 2.0 ** -20 + 2.0 ** -18 + 16 * FOLD[dt] * 2.0 ** -23 + (n / 32 + 16) * 2.0 ** -24
    t = torch.finfo(TYPES[dt])
    tol = rel * vabs + t.eps / 2 * want.abs() + lost + t.smallest_normal * t.eps
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

"""Measured cases of the operators over a key / value cache held in 8 bits with one scale for each block of tokens
and KV head: append, attention of one row per sequence, attention of prompt rows, eviction by accumulated attention
weight (and the read-back of what the cache holds, with append and eviction).

The cache of one layer is four tensors: codes k, v int8 [slots, kv_heads, capacity, head_dim] and scales k_scale,
v_scale fp32 [slots, kv_heads, capacity / block]; a token's key is code * scale of its block. Rows of several
sequences lie one behind the other: sequence b's are start[b] .. start[b + 1] - 1, its first one at cache position
pos[b] (a negative position: an idle slot).
"""
import math
import random

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------ the cases
def _case(name, op, dtype, slots, heads, kv_heads, head_dim, block, **kw):
    c = {"name": name, "op": op, "dtype": dtype, "slots": slots, "heads": heads, "kv_heads": kv_heads,
         "head_dim": head_dim, "block": block, "ragged": False, "idle": 0, "mass": False, "pad": 0, "prior": 0,
         "rows": 1, "longest": 0, "keep": 0, "sink": 0, "recent": 0}
    c.update(kw)
    return c


def listed():
    return [
        # one new token of each of 128 sequences (16 / 8 heads of 128), caches about 2,000 tokens long
        _case("append_step_128", "append", "fp32", 128, 16, 8, 128, 64, prior=2031, ragged=True),
        # prompts of up to 2,000 tokens written behind an odd shared prefix, 64-dim heads
        _case("append_prompts", "append", "bf16", 6, 32, 8, 64, 32, rows=2000, prior=77, ragged=True, pad=9),
        # one sequence, one token, in the middle of a chat: the smallest call, latency counts
        _case("step_one", "step", "fp32", 1, 16, 8, 128, 64, longest=2032),
        # batched decode at the length of the decode benchmark
        _case("step_128", "step", "fp32", 128, 16, 8, 128, 64, longest=2032),
        # a few long documents, 64-dim heads in groups of four
        _case("step_long", "step", "bf16", 4, 32, 8, 64, 64, longest=32768, ragged=True),
        # decode that also gathers each token's attention weight, sequences of mixed lengths and idle slots,
        # three query heads per KV head
        _case("step_mass", "step", "fp32", 24, 9, 3, 64, 16, longest=8191, ragged=True, idle=3, mass=True),
        # one prefill chunk of a prompt in progress
        _case("rows_chunk", "rows", "fp32", 1, 16, 8, 128, 64, rows=256, prior=1760),
        # several prompts of mixed lengths in one launch, a padded row count
        _case("rows_prompts", "rows", "bf16", 6, 32, 8, 64, 32, rows=2000, prior=77, ragged=True, pad=9),
        # a prompt that gathers the attention weights that the eviction after it goes by
        _case("rows_mass", "rows", "fp32", 2, 9, 3, 64, 64, rows=1500, ragged=True, mass=True),
        # one long prompt at once: the largest case
        _case("rows_long", "rows", "fp32", 1, 16, 8, 128, 64, rows=8192),
        # one sequence cut to half its length
        _case("evict_one", "evict", "fp32", 1, 16, 8, 128, 64, longest=2048, keep=1024, sink=4, recent=256),
        # a batch of sequences of mixed lengths cut to an odd budget, some of them shorter than it
        _case("evict_batch", "evict", "fp32", 16, 32, 8, 64, 32, longest=8192, keep=3001, sink=4, recent=500,
              ragged=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["append", "step", "step", "rows", "rows", "evict"])
    kv_heads, group = rng.choice([1, 2, 3, 4, 6, 8]), rng.choice([1, 2, 3, 4, 8])
    hd, block = rng.choice([16, 48, 64, 80, 96, 128]), rng.choice([16, 32, 64, 128])
    kw = {"ragged": rng.random() < 0.7}
    row = 2 * kv_heads * hd                                   # bytes of one cached token
    if op == "append":
        slots, rows = _log_int(rng, 1, 64), 1 if rng.random() < 0.5 else _log_int(rng, 2, 2000)
        rows = max(1, min(rows, (64 << 20) // (slots * row)))
        kw.update(rows=rows, prior=rng.randint(0, 2000), pad=rng.randint(0, 15) if rows > 1 else 0,
                  idle=rng.randint(0, slots // 4))
    elif op == "step":
        slots = _log_int(rng, 1, 128)
        longest = max(1, min(_log_int(rng, 1, 32768), (512 << 20) // (slots * row)))
        kw.update(longest=longest, idle=rng.randint(0, slots // 4), mass=rng.random() < 0.3)
    elif op == "rows":
        slots, rows, prior = _log_int(rng, 1, 8), _log_int(rng, 1, 4000), rng.randint(0, 2500)
        while slots * kv_heads * group * rows * (rows + prior) > 1 << 29:
            rows = max(1, rows * 2 // 3)
            prior = prior * 2 // 3
        kw.update(rows=rows, prior=prior, pad=rng.randint(0, 15), idle=rng.randint(0, slots // 4),
                  mass=rng.random() < 0.3)
    else:
        slots = _log_int(rng, 1, 24)
        longest = max(2, min(_log_int(rng, 16, 16384), (192 << 20) // (slots * row)))
        keep = rng.randint(1, longest)
        sink = rng.randint(0, min(8, keep))
        kw.update(longest=longest, keep=keep, sink=sink, recent=rng.randint(0, (keep - sink) // 2))
    c = _case("", op, rng.choice(["fp32", "fp32", "bf16", "fp16"]), slots, kv_heads * group, kv_heads, hd, block,
              **kw)
    del c["name"]
    return c


# ------------------------------------------------------------------ lengths
def _lengths(c):
    """Per slot (tokens before the call, new rows; step and evict: tokens held, 0), from the case alone."""
    r = random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))
    S, out = c["slots"], []
    for b in range(S):
        first = b == 0                                       # slot 0 has the longest
        if c["op"] in ("append", "rows"):
            n = c["rows"] if first or not c["ragged"] else r.randint(0 if c["rows"] > 1 else 1, c["rows"])
            p = c["prior"] if first or not c["ragged"] else r.randint(0, c["prior"])
            out.append((p, n))
        else:
            out.append((c["longest"] if first or not c["ragged"] else r.randint(1, c["longest"]), 0))
    for b in r.sample(range(1, S), c["idle"]) if c["idle"] else []:
        out[b] = (-1, 0)
    return out


def _capacity(c):
    need = max(c["longest"], c["rows"] + c["prior"], c["keep"])
    return -(-need // c["block"]) * c["block"]


def _fill(c, g, dev):
    """Codes as they lie after quantization (a block's largest at +-127 or near), and their blocks' scales."""
    S, H, T, D, B = c["slots"], c["kv_heads"], _capacity(c), c["head_dim"], c["block"]
    codes = torch.empty(S, H, T, D, dtype=torch.int8, device=dev)
    for b in range(S):
        codes[b] = torch.randn(H, T, D, generator=g, device=dev).mul_(36).round_().clamp_(-127, 127).to(torch.int8)
    scale = torch.exp(0.25 * torch.randn(S, H, T // B, generator=g, device=dev)) / 36
    return codes, scale


def prepare(case, seed):
    c, dev = case, "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    dt, S, lens = DTYPES[c["dtype"]], c["slots"], _lengths(c)
    k, ks = _fill(c, g, dev)
    v, vs = _fill(c, g, dev)
    s = {"case": c, "cache": (k, ks, v, vs)}
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)
    new = [n for _, n in lens]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    rows = S if c["op"] == "step" else starts[-1] + c["pad"]
    randn = lambda *z: torch.randn(*z, generator=g, device=dev).to(dt)
    if c["op"] == "step":
        s["pos"] = i32([p - 1 if p >= 0 else -1 for p, _ in lens])
        s["q"] = randn(rows, c["heads"], c["head_dim"])
    elif c["op"] == "rows":
        s["pos"], s["start"] = i32([p for p, _ in lens]), i32(starts)
        s["q"] = randn(rows, c["heads"], c["head_dim"])
        s["out"] = torch.zeros_like(s["q"])                   # rows behind the last sequence stay as they are
        s["most_rows"], s["most"] = max(new), max(p + n for p, n in lens)
    elif c["op"] == "append":
        s["pos"], s["start"] = i32([p for p, _ in lens]), i32(starts)
        s["k_new"], s["v_new"] = (randn(rows, c["kv_heads"], c["head_dim"]) for _ in range(2))
        # the rows to read back: every token of the blocks that the new rows fall into, up to the last new one
        B = c["block"]
        lo = [p // B * B if n else 0 for p, n in lens]
        back = [0]
        for (p, n), f in zip(lens, lo):
            back.append(back[-1] + (p + n - f if n else 0))
        s["back_pos"], s["back_start"], s["back_rows"] = i32(lo), i32(back), back[-1]
        s["blocks"] = sum((p + n - 1) // B - p // B + 1 for p, n in lens if n)
    else:
        s["count"] = i32([p for p, _ in lens])
        s["dst"] = tuple(torch.zeros_like(t) for t in s["cache"])
        s["back_pos"], s["back_start"] = i32([0] * S), i32([b * c["keep"] for b in range(S + 1)])
        s["dst_mass"] = torch.zeros(S, c["kv_heads"], k.shape[2], device=dev)
    if c["mass"] or c["op"] == "evict":
        s["mass"] = torch.rand(S, c["kv_heads"], k.shape[2], generator=g, device=dev).pow_(4)
        # a prompt's first tokens gather most, and weights that ran to nothing tie at zero
        s["mass"][:, :, :4] += 3
        s["mass"][s["mass"] < 1e-4] = 0
    return s


# ------------------------------------------------------------------ the plain forms
def _expand(codes, scale, block):
    S, H, T, D = codes.shape
    return (codes.float().view(S, H, T // block, block, D) * scale.view(S, H, -1, 1, 1)).view(S, H, T, D)


def _softmax_out(scores, vd):
    """exp / sum over the last axis, masked scores at -inf; rows that see nothing give zeros."""
    m = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    total = e.sum(-1, keepdim=True)
    total = torch.where(total > 0, total, torch.ones_like(total))
    return e @ vd / total, e, total


def _plain_step(s):
    c, (k, ks, v, vs), pos = s["case"], s["cache"], s["pos"].long()
    S, H, D, T = c["slots"], c["kv_heads"], c["head_dim"], c["longest"]
    kd, vd = _expand(k, ks, c["block"])[:, :, :T], _expand(v, vs, c["block"])[:, :, :T]
    q = s["q"].float().view(S, H, -1, D)
    scores = q @ kd.transpose(2, 3) / math.sqrt(D)
    hidden = torch.arange(T, device=q.device) > pos.view(S, 1, 1, 1)
    out, e, total = _softmax_out(scores.masked_fill(hidden, -math.inf), vd)
    got = {"out": out.reshape(S, c["heads"], D).to(s["q"].dtype)}
    if c["mass"]:
        s["mass"][:, :, :T] += (e / total).sum(2)
        got["mass"] = s["mass"]
    return got


def _row_places(s, rows):
    """Each row's slot and its index in the slot's rows."""
    start, at = s["start"].long(), torch.arange(rows, device=s["pos"].device)
    slot = torch.searchsorted(start, at, right=True) - 1
    return slot, at - start[slot]


def _plain_rows(s):
    c, (k, ks, v, vs), pos = s["case"], s["cache"], s["pos"].long()
    S, H, D, N, T = c["slots"], c["kv_heads"], c["head_dim"], s["most_rows"], s["most"]
    G = c["heads"] // H
    rows = s["q"].shape[0] - c["pad"]
    slot, i = _row_places(s, rows)
    q = torch.zeros(S, N, H, G, D, device=pos.device)
    q[slot, i] = s["q"][:rows].float().view(rows, H, G, D)
    q = q.permute(0, 2, 3, 1, 4).reshape(S, H, G * N, D)
    kd, vd = _expand(k, ks, c["block"])[:, :, :T], _expand(v, vs, c["block"])[:, :, :T]
    scores = (q @ kd.transpose(2, 3)).view(S, H, G, N, T) / math.sqrt(D)
    n = (s["start"][1:] - s["start"][:-1]).long()
    at = torch.arange(N, device=pos.device)
    last = torch.where(at < n.view(S, 1), pos.view(S, 1) + at, -1)      # the last token that a row sees
    hidden = torch.arange(T, device=pos.device) > last.view(S, 1, 1, N, 1)
    out, e, total = _softmax_out(scores.masked_fill_(hidden, -math.inf), vd.unsqueeze(2))
    out = out.permute(0, 3, 1, 2, 4)[slot, i].reshape(rows, c["heads"], D)
    s["out"][:rows] = out.to(s["out"].dtype)
    got = {"out": s["out"]}
    if c["mass"]:
        s["mass"][:, :, :T] += (e / total).sum((2, 3))
        got["mass"] = s["mass"]
    return got


def _read_back(cache, block, pos, start, rows):
    k, ks, v, vs = cache
    at = torch.arange(rows, device=pos.device)
    slot = torch.searchsorted(start.long(), at, right=True) - 1
    t = pos.long()[slot] + at - start.long()[slot]
    read = lambda x, xs: x[slot, :, t].float() * xs[slot, :, t // block].unsqueeze(-1)
    return read(k, ks), read(v, vs)


def _plain_append_one(s, x, codes, scale):
    """Rows into their blocks: a block's scale grows to its new rows' largest value times F(1/127), its older codes with it."""
    c, pos = s["case"], s["pos"].long()
    S, H, D, B = c["slots"], c["kv_heads"], c["head_dim"], c["block"]
    rows, total = x.shape[0] - c["pad"], s["blocks"]
    x = torch.nan_to_num(x[:rows].float())
    n = (s["start"][1:] - s["start"][:-1]).long()
    first = pos.clamp(min=0) // B
    touched = torch.where(n > 0, (pos + n - 1).div(B, rounding_mode="floor") - first + 1, 0)
    offset = torch.cumsum(touched, 0) - touched
    owner = torch.repeat_interleave(torch.arange(S, device=x.device), touched, output_size=total)
    blk = first[owner] + torch.arange(total, device=x.device) - offset[owner]
    slot, i = _row_places(s, rows)
    t = pos[slot] + i
    pair = offset[slot] + t // B - first[slot]
    new = torch.zeros(total, B, H, D, device=x.device)
    new[pair, t % B] = x
    token = blk.unsqueeze(1) * B + torch.arange(B, device=x.device)
    is_old = (token < pos[owner].unsqueeze(1)).view(total, 1, B, 1)
    is_new = (token >= pos[owner].unsqueeze(1)) & (token < (pos + n)[owner].unsqueeze(1))
    new, is_new = new.transpose(1, 2), is_new.view(total, 1, B, 1)
    blocks, scales = codes.view(S, H, -1, B, D), scale
    old = blocks[owner, :, blk].float()
    s_old = scales[owner, :, blk] * (blk * B < pos[owner]).unsqueeze(1)
    s_new = torch.maximum(s_old, new.abs().amax((2, 3)) * (1 / 127))
    a, b = s_old.view(total, H, 1, 1), s_new.view(total, H, 1, 1)
    keep = torch.where(a == b, old, torch.round(old * a / b))
    put = torch.where(b > 0, torch.round(new / b).clamp(-127, 127), 0.0)
    got = torch.where(is_new, put, torch.where(is_old, keep, old))
    blocks[owner, :, blk] = got.to(torch.int8)
    scales[owner, :, blk] = s_new


def _plain_append(s):
    k, ks, v, vs = s["cache"]
    _plain_append_one(s, s["k_new"], k, ks)
    _plain_append_one(s, s["v_new"], v, vs)
    return _read_back(s["cache"], s["case"]["block"], s["back_pos"], s["back_start"], s["back_rows"])


def _plain_evict(s):
    c, count, mass = s["case"], s["count"].long(), s["mass"]
    S, H, T = mass.shape
    B, D, K = c["block"], c["head_dim"], c["keep"]
    at = torch.arange(T, device=mass.device)
    n = count.view(S, 1, 1)
    score = torch.where(torch.isnan(mass), -math.inf, mass)
    # order: sink and recent tokens first, then the middle by weight, then what is not held; ties by index
    always = (at < c["sink"]) | (at >= n - c["recent"])
    rank = torch.where(at >= n, 2, torch.where(always, 0, 1)).expand(S, H, T)
    by_weight = torch.sort(score, dim=-1, descending=True, stable=True).indices
    order = torch.gather(by_weight, 2, torch.sort(torch.gather(rank, 2, by_weight), dim=-1, stable=True).indices)
    left = torch.clamp(count, max=K)
    place = torch.arange(K, device=mass.device)
    chosen = torch.where(place < left.view(S, 1, 1), order[:, :, :K], T).sort(-1).values
    held = chosen < T
    idx = chosen.clamp(max=T - 1)
    evicts = (count > K).view(S, 1, 1)
    new_mass = torch.where(at < n, 0.0, s["dst_mass"])
    new_mass[:, :, :K] = torch.where(held, torch.gather(mass, 2, idx), new_mass[:, :, :K])
    s["dst_mass"].copy_(new_mass)
    NB = -(-K // B)
    for codes, scale, to, to_scale in ((s["cache"][0], s["cache"][1], s["dst"][0], s["dst"][1]),
                                       (s["cache"][2], s["cache"][3], s["dst"][2], s["dst"][3])):
        q = torch.gather(codes, 2, idx.unsqueeze(-1).expand(S, H, K, D)).float()
        s_old = torch.gather(scale, 2, idx // B).unsqueeze(-1)
        x = torch.zeros(S, H, NB * B, D, device=q.device)
        x[:, :, :K] = q * s_old * held.unsqueeze(-1)
        x = x.view(S, H, NB, B, D)
        s_new = x.abs().amax((3, 4)) * (1 / 127)
        r = s_new.view(S, H, NB, 1, 1)
        y = torch.where(r > 0, torch.round(x / r).clamp(-127, 127), 0.0).view(S, H, NB * B, D)[:, :, :K]
        y = torch.where(evicts.unsqueeze(-1), y, q).to(torch.int8)
        to[:, :, :K] = torch.where(held.unsqueeze(-1), y, to[:, :, :K])
        has = torch.arange(NB, device=q.device) * B < left.view(S, 1, 1)
        s_new = torch.where(evicts, s_new, scale[:, :, :NB])
        to_scale[:, :, :NB] = torch.where(has, s_new, to_scale[:, :, :NB])
    back = _read_back(s["dst"], B, s["back_pos"], s["back_start"], S * K)
    kept = torch.where(held, chosen, -1).to(torch.int32)
    return {"kept": kept, "count": left.to(torch.int32), "mass": s["dst_mass"], "k": back[0], "v": back[1]}


# ------------------------------------------------------------------ one pass
def run(state):
    s, c = state, state["case"]
    if own:
        from torch2riscv_accelerator_b200 import ops
        if c["op"] == "step":
            out = ops.kvb_attn(s["q"], s["cache"], s["pos"], mass=s["mass"] if c["mass"] else None)
            return {"out": out, "mass": s["mass"]} if c["mass"] else {"out": out}
        if c["op"] == "rows":
            out = ops.kvb_attn_rows(s["q"], s["cache"], s["pos"], s["start"], out=s["out"],
                                    mass=s["mass"] if c["mass"] else None)
            return {"out": out, "mass": s["mass"]} if c["mass"] else {"out": out}
        if c["op"] == "append":
            ops.kvb_append(s["k_new"], s["v_new"], s["cache"], s["pos"], s["start"])
            return _append_outputs(s, ops.kvb_read(s["cache"], s["back_pos"], s["back_start"], s["back_rows"]))
        kept, count = ops.kvb_evict(s["cache"], s["mass"], s["count"], c["keep"], sink=c["sink"],
                                    recent=c["recent"], dst=s["dst"], dst_mass=s["dst_mass"])
        k, v = ops.kvb_read(s["dst"], s["back_pos"], s["back_start"], c["slots"] * c["keep"])
        return {"kept": kept, "count": count, "mass": s["dst_mass"], "k": k, "v": v}
    if c["op"] == "append":
        return _append_outputs(s, _plain_append(s))
    return {"step": _plain_step, "rows": _plain_rows, "evict": _plain_evict}[c["op"]](s)


def _append_outputs(s, back):
    return {"k": back[0], "v": back[1], "k_scale": s["cache"][1], "v_scale": s["cache"][3]}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c, lens = case, _lengths(case)
    e = 4 if c["dtype"] == "fp32" else 2
    H, D, B, G = c["kv_heads"], c["head_dim"], c["block"], c["heads"] // c["kv_heads"]
    token, blk = 2 * H * D, 2 * H * 4                         # bytes of a cached token, of a block's scales
    if c["op"] == "step":
        t = sum(max(p, 0) for p, _ in lens)
        b = sum(-(-max(p, 0) // B) for p, _ in lens)
        io = 2 * sum(p > 0 for p, _ in lens) * c["heads"] * D * e
        return {"bytes": t * token + b * blk + io + (8 * t * H if c["mass"] else 0), "flops": 4 * t * H * G * D}
    if c["op"] == "rows":
        t = sum(p + n for p, n in lens if n)
        b = sum(-(-(p + n) // B) for p, n in lens if n)
        pairs = sum(n * p + n * (n + 1) // 2 for p, n in lens if n)
        io = 2 * sum(n for _, n in lens) * c["heads"] * D * e
        return {"bytes": t * token + b * blk + io + (8 * t * H if c["mass"] else 0), "flops": 4 * pairs * H * G * D}
    if c["op"] == "append":                                   # rows in, codes out; touched blocks read back as fp32
        n = sum(n for _, n in lens)
        back = sum(p + n - p // B * B for p, n in lens if n)
        touched = sum((p + n - 1) // B - p // B + 1 for p, n in lens if n)
        return {"bytes": n * 2 * H * D * e + back * token + touched * 2 * blk + back * token * 4, "flops": 0}
    t, left = sum(p for p, _ in lens), sum(min(p, c["keep"]) for p, _ in lens)
    b = sum(-(-min(p, c["keep"]) // B) for p, _ in lens)
    return {"bytes": t * H * 8 + left * (2 * token + 8 * H) + 2 * b * blk + c["slots"] * c["keep"] * token * 4,
            "flops": 0}


# ------------------------------------------------------------------ the definition in 64 bits
def _values64(codes, scale, b, h, n, block):
    t = torch.arange(n, device=codes.device)
    return codes[b, h, :n].double() * scale[b, h].double()[t // block].unsqueeze(1)


def _attend64(q, k, v, last):
    """q [n, D] sees tokens 0 .. last[i]: output rows and the sum of the probabilities of each token."""
    z = q @ k.T * (k.shape[1] ** -0.5)
    z[torch.arange(k.shape[0], device=q.device).unsqueeze(0) > last.unsqueeze(1)] = -math.inf
    p = torch.softmax(z, 1)
    return p @ v, p.sum(0)


def exact(case, seed):
    s, c, lens = prepare(case, seed), case, _lengths(case)
    k, ks, v, vs = s["cache"]
    H, G, B = c["kv_heads"], c["heads"] // c["kv_heads"], c["block"]
    if c["op"] in ("step", "rows"):
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        mass = s["mass"].double() if c["mass"] else None
        at = 0
        for b, (p, n) in enumerate(lens):
            p, n, row = (p - 1, 1, b) if c["op"] == "step" else (p, n, at)
            if p < 0 or n == 0:
                continue
            last = p + torch.arange(n, device="cuda")
            for h in range(H):
                kd, vd = _values64(k, ks, b, h, p + n, B), _values64(v, vs, b, h, p + n, B)
                for j in range(h * G, h * G + G):
                    out[row:row + n, j], w = _attend64(s["q"][row:row + n, j].double(), kd, vd, last)
                    if mass is not None:
                        mass[b, h, :p + n] += w
            at += n
        return {"out": out, "mass": mass} if c["mass"] else {"out": out}
    if c["op"] == "append":
        # the codes follow from roundings in single precision: the scales have a value in 64 bits
        got = []
        for x, scale in ((s["k_new"], ks.double()), (s["v_new"], vs.double())):
            at = 0
            for b, (p, n) in enumerate(lens):
                for j in range(p // B, (p + n - 1) // B + 1) if n else ():
                    lo, hi = max(j * B, p), min((j + 1) * B, p + n)
                    most = x[at + lo - p:at + hi - p].double().abs().amax((0, 2)) / 127
                    scale[b, :, j] = torch.maximum(scale[b, :, j], most) if j * B < p else most
                at += n
            got.append(scale)
        return {"k": None, "v": None, "k_scale": got[0], "v_scale": got[1]}
    kept = torch.full((c["slots"], H, c["keep"]), -1, dtype=torch.int64)
    mass = s["dst_mass"].double()
    for b, (n, _) in enumerate(lens):
        for h in range(H):
            w = s["mass"][b, h, :n].tolist()
            if n > c["keep"]:
                middle = range(c["sink"], n - c["recent"])
                best = sorted(middle, key=lambda t: (-w[t], t))[:c["keep"] - c["sink"] - c["recent"]]
                ids = sorted([*range(c["sink"]), *best, *range(n - c["recent"], n)])
            else:
                ids = list(range(n))
            kept[b, h, :len(ids)] = torch.tensor(ids)
            mass[b, h, :len(ids)] = torch.tensor([w[t] for t in ids], dtype=torch.float64, device="cuda")
    count = torch.tensor([min(n, c["keep"]) for n, _ in lens], dtype=torch.int32)
    return {"kept": kept.to(torch.int32), "count": count, "mass": mass, "k": None, "v": None}

"""Plain NumPy forms of the block-scaled KV cache's operators for the tests:
append and eviction step by step in float32 (each step rounded once, so codes
and scales are compared bit for bit), attention in float64."""
import numpy as np

F = np.float32
INV127 = F(1.0 / 127.0)
FMAX = np.finfo(F).max


def spans(pos, start, slots, rows):
    """(slot, first row, rows, position of the first) of the slots with rows."""
    for b in range(slots):
        r0, r1 = (b, b + 1) if start is None else (start[b], start[b + 1])
        if r1 > r0:
            yield b, r0, r1 - r0, int(pos[b])


def codes_of(num, den):
    with np.errstate(all="ignore"):
        return np.clip(np.rint((num / den).astype(F)), -127, 127).astype(np.int8)


def append(x, codes, scale, pos, start=None):
    """Rows x [rows, H, D] float32 into codes [S, H, T, D], scale [S, H, T / B], in place."""
    S, H, T, D = codes.shape
    B = T // scale.shape[2]
    x = np.nan_to_num(x.astype(F), nan=0.0, posinf=FMAX, neginf=-FMAX)
    for b, r0, n, p in spans(pos, start, S, x.shape[0]):
        n = 0 if p < 0 else min(n, T - p)
        for j in range(p // B, (p + n - 1) // B + 1) if n > 0 else ():
            t0, t1 = max(j * B, p), min((j + 1) * B, p + n)
            for h in range(H):
                y = x[r0 + t0 - p:r0 + t1 - p, h]
                s_old = scale[b, h, j] if t0 > j * B else F(0)
                s_new = np.maximum(s_old, np.abs(y).max() * INV127)
                if t0 > j * B and s_new != s_old:
                    codes[b, h, j * B:t0] = codes_of(codes[b, h, j * B:t0].astype(F) * s_old, s_new)
                codes[b, h, t0:t1] = codes_of(y, s_new) if s_new > 0 else 0
                scale[b, h, j] = s_new


def values(codes, scale, b, h, n):
    B = codes.shape[2] // scale.shape[2]
    return codes[b, h, :n].astype(np.float64) * np.repeat(scale[b, h].astype(np.float64), B)[:n, None]


def attend(q, k, ks, v, vs, pos, start=None, scale=None, mass=None):
    """q [rows, heads, D] float64 -> out, the bound's sums: per row and head
    max_t sum_d |q_d k_td| * scale and max |v|; mass [S, H, T] float64 is added to."""
    rows, heads, D = q.shape
    S, H, T = k.shape[:3]
    G = heads // H
    scale = D ** -0.5 if scale is None else scale
    out, zabs, vmax = np.zeros(q.shape), np.zeros((rows, heads, 1)), np.zeros((rows, heads, 1))
    for b, r0, n, p in spans(pos, start, S, rows):
        n = 0 if p < 0 else min(n, T - p)
        if n <= 0:
            continue
        for h in range(H):
            kd, vd = values(k, ks, b, h, p + n), values(v, vs, b, h, p + n)
            hidden = np.arange(p + n)[None, :] > (p + np.arange(n))[:, None]
            for j in range(h * G, h * G + G):
                qj = q[r0:r0 + n, j]
                z = np.where(hidden, -np.inf, qj @ kd.T * scale)
                e = np.exp(z - z.max(1, keepdims=True))
                w = e / e.sum(1, keepdims=True)
                out[r0:r0 + n, j] = w @ vd
                zabs[r0:r0 + n, j, 0] = (np.abs(qj) @ np.abs(kd).T).max(1) * abs(scale)
                vmax[r0:r0 + n, j, 0] = np.abs(vd).max()
                if mass is not None:
                    mass[b, h, :p + n] += w.sum(0)
    return out, zabs, vmax


def keep_of(w, n, keep, sink, recent):
    """The kept positions of one slot and head."""
    if n <= keep:
        return list(range(n))
    key = [-np.inf if np.isnan(x) else x for x in w[:n]]
    mid = sorted(range(sink, n - recent), key=lambda t: (-key[t], t))[:keep - sink - recent]
    return sorted([*range(sink), *mid, *range(n - recent, n)])


def evict(k, ks, v, vs, mass, count, keep, sink, recent, dst=None, dst_mass=None):
    """In place (dst None) or into dst = (k, ks, v, vs) and dst_mass; returns kept, new counts."""
    S, H, T, D = k.shape
    B = T // ks.shape[2]
    src = [a.copy() for a in (k, ks, v, vs, mass)]
    to = (k, ks, v, vs) if dst is None else dst
    to_mass = mass if dst is None else dst_mass
    kept = np.full((S, H, keep), -1, np.int32)
    for b in range(S):
        n = min(max(int(count[b]), 0), T)
        for h in range(H):
            ids = keep_of(src[4][b, h], n, keep, sink, recent)
            kept[b, h, :len(ids)] = ids
            if dst is None and n <= keep:
                continue
            for c, sc, oc, osc in ((src[0], src[1], to[0], to[1]), (src[2], src[3], to[2], to[3])):
                for j in range(-(-len(ids) // B)):
                    part = ids[j * B:(j + 1) * B]
                    q, s = c[b, h, part], sc[b, h, [t // B for t in part]]
                    if n > keep:
                        x = q.astype(F) * s[:, None]
                        s_new = np.abs(x).max() * INV127
                        q = codes_of(x, s_new) if s_new > 0 else np.zeros_like(q)
                        osc[b, h, j] = s_new
                    else:
                        osc[b, h, j] = s[0]
                    oc[b, h, j * B:j * B + len(part)] = q
            to_mass[b, h, :len(ids)] = src[4][b, h, ids]
            to_mass[b, h, len(ids):n] = 0
    return kept, np.array([min(min(max(int(c), 0), T), keep) for c in count], np.int32)

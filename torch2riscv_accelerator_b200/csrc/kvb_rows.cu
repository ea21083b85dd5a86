// Attention of prompt rows over the block-scaled 8-bit KV cache on the
// 5th-generation tensor cores.
//
//   o_r = sum_t p_rt v_t,  p_rt = exp(z_rt - m_r) / sum_t exp(z_rt - m_r),
//   z_rt = scale * sk[t / B] * (q_r . k_t)     for the tokens t <= pos_r
//
// A unit is 128 rows of one (slot, KV head): row f of the slot's n * G is query
// row f / G and query head f % G of the KV head's group, so that a key tile
// serves the whole group. Its tokens up to the last row's position come in
// tiles of BN. All units' tiles, in order, are dealt out to the SMs in equal
// contiguous shares (causal units differ in length, and few rows must still
// fill the GPU); a CTA leaves at most two partial units, which kvb_rows_finish
// joins. kvb_rows_plan lists the units, since lengths are device data.
//
// Warps of a CTA (one CTA an SM, all 512 TMEM columns):
//   softmax   4 warps per stream, one row per thread. With two streams the even
//             tiles go to one and the odd ones to the other, each with its own
//             maximum, sum and output accumulator: no exchange before the end.
//   convert   4 warps: int8 codes -> exact halves (byte permutes, one
//             subtraction) in 128-byte-swizzled tiles, a tile ahead of the
//             products in registers; the query rows as hi + lo halves (22 bits)
//             of the row scaled by a power of two (16-bit queries are exact in
//             one half).
//   products  one thread: S = Q K^T (A, B from shared memory), O += P V (P from
//             TMEM, written over S: hi in columns 0-15, lo in 16-31 of every 32;
//             V as it lies, its rows being the contraction).
// Block scales do not touch the codes: K's multiplies the scores of its 16
// columns, V's goes into the weights, as exp(z - m) sv / sv_ref 2^7 with the
// lazily moved references of the one-row kernel (kvb_attn.cu), so that the
// accumulator is rescaled rarely.
#include "kvb.cuh"
#include "tc.cuh"

namespace w8a8 {

static __device__ unsigned int g_kvb_rows_errors;

unsigned int kvb_rows_read_clear_errors() {
    unsigned int v = 0, zero = 0;
    cudaMemcpyFromSymbol(&v, g_kvb_rows_errors, sizeof(v));
    cudaMemcpyToSymbol(g_kvb_rows_errors, &zero, sizeof(zero));
    return v;
}

namespace {

constexpr int kRows = 128;                       // rows of a unit (TMEM lanes)
constexpr int kSms = 148;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazyScore = 6.0f, kLazyScale = 4.0f, kWeightScale = 128.0f;
constexpr unsigned int kErrWait = 256u;          // error bit 8: a pipeline wait gave up
constexpr int kPlanThreads = 1024;
constexpr int kFinishThreads = 256;

template <int HD>
struct RowsCfg {
    static constexpr int BN = HD == 256 ? 64 : 128;
    static constexpr int STREAMS = HD == 256 ? 1 : 2;
    static constexpr int NBUF = HD == 256 ? 1 : 2;
    static constexpr int SLABS = HD / 64;        // 64-channel slabs of a tile
    static constexpr int QSLAB = kRows * 128, SLAB = BN * 128, TILE = SLABS * SLAB;   // bytes
    static constexpr int SOFT = STREAMS * 128;   // softmax threads
    static constexpr int THREADS = SOFT + 128 + 32;
    static constexpr size_t smem(bool q2) {
        return 1024 + (size_t)(q2 ? 2 : 1) * SLABS * QSLAB + (size_t)NBUF * 2 * TILE;
    }
    static constexpr size_t PART = (size_t)kRows * (HD + 2);   // floats of a partial unit
};

struct RowsPlan {                                // in scratch: total, units' count, units, slots' first units
    int* head;                                   // [4]: tiles of all units of one KV head, units
    int4* unit;                                  // slot, 128-row tile, tiles before, tiles
    int* first;                                  // [slots + 1]
};

__host__ __device__ inline int64_t max_units(const KvbCache& c, int heads, int rows) {
    return (int64_t)rows * (heads / c.heads) / kRows + (rows < c.slots ? rows : c.slots);
}

__device__ __forceinline__ int live_rows(const KvbSpan& s, int cap) { return s.p < 0 ? 0 : max(min(s.n, cap - s.p), 0); }

// exclusive scan over the CTA's kPlanThreads threads; *sum the total
__device__ __forceinline__ int block_scan(int x, int* sum) {
    __shared__ int w[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    int upto = x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += o;
    }
    if (lane == 31) w[warp] = upto;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        if (i < warp) before += w[i];
        all += w[i];
    }
    __syncthreads();
    *sum = all;
    return before + upto - x;
}

__global__ void __launch_bounds__(kPlanThreads) kvb_rows_plan(const KvbAttnArgs a, RowsPlan plan, int bn, int most) {
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, S = a.c.slots, G = a.heads / a.c.heads;
    int units = 0, sum;
    for (int b0 = 0; b0 < S; b0 += kPlanThreads) {
        const int b = b0 + tid;
        const int n = b < S ? (live_rows(kvb_span(a.r, b), a.c.cap) * G + kRows - 1) / kRows : 0;
        const int at = block_scan(n, &sum);
        if (b < S) plan.first[b] = units + at;
        units += sum;
    }
    if (tid == 0) plan.first[S] = units;
    __syncthreads();
    units = min(units, most);                    // more only with offsets out of order: rows are then left out
    int total = 0;
    for (int u0 = 0; u0 < units; u0 += kPlanThreads) {
        const int u = u0 + tid;
        int b = 0, m = 0, tiles = 0;
        if (u < units) {
            int hi = S;                          // the last slot with first <= u that has units
            while (hi - b > 1) {
                const int mid = (b + hi) >> 1;
                if (plan.first[mid] <= u) b = mid;
                else hi = mid;
            }
            m = u - plan.first[b];
            const KvbSpan sp = kvb_span(a.r, b);
            const int rows = live_rows(sp, a.c.cap) * G;
            tiles = (sp.p + min(m * kRows + kRows - 1, rows - 1) / G) / bn + 1;
        }
        const int at = block_scan(tiles, &sum);
        if (u < units) plan.unit[u] = make_int4(b, m, total + at, tiles);
        total += sum;
    }
    if (tid == 0) plan.head[0] = total, plan.head[1] = units;
}

// A run of tiles of one unit within a CTA's share [x, end).
struct Seg {
    int64_t x, end;
    int h, u, j, n, tiles;                       // KV head, unit; first tile, tiles here, tiles of the unit
    int slot, m, p, r0, rows;                    // rows: the slot's n * G live ones
    __device__ __forceinline__ void unit(const KvbAttnArgs& a, const RowsPlan& plan) {
        const int4 v = plan.unit[u];
        slot = v.x, m = v.y, tiles = v.w;
        const KvbSpan s = kvb_span(a.r, slot);
        p = s.p, r0 = s.r0, rows = live_rows(s, a.c.cap) * (a.heads / a.c.heads);
        n = (int)min((int64_t)(tiles - j), end - x);
    }
    __device__ __forceinline__ bool begin(const KvbAttnArgs& a, const RowsPlan& plan, int64_t x0, int64_t x1) {
        x = x0, end = x1;
        if (x >= end) return false;
        const int total = plan.head[0];
        h = (int)(x / total);
        const int at = (int)(x - (int64_t)h * total);
        int lo = 0, hi = plan.head[1];
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (plan.unit[mid].z <= at) lo = mid;
            else hi = mid;
        }
        u = lo, j = at - plan.unit[lo].z;
        unit(a, plan);
        return true;
    }
    __device__ __forceinline__ bool next(const KvbAttnArgs& a, const RowsPlan& plan) {
        x += n;
        if (x >= end) return false;
        if (++u == plan.head[1]) u = 0, ++h;
        j = 0;
        unit(a, plan);
        return true;
    }
};

__device__ __forceinline__ void rows_share(const RowsPlan& plan, int heads, int grid, int cta, int64_t* lo, int64_t* hi) {
    const int64_t total = (int64_t)plan.head[0] * heads, ctas = total < grid ? total : grid;
    *lo = *hi = 0;
    if (cta < ctas) *lo = total * cta / ctas, *hi = total * (cta + 1) / ctas;
}

// 16 codes as 16 halves in two 16-byte chunks of a swizzled row
__device__ __forceinline__ void put_codes(unsigned char* slab, int row, int ch, int odd, uint4 w) {
    const uint32_t x[4] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u};
    uint4 lo, hi;
    lo = make_uint4(halves_of(x[0], 0x4140), halves_of(x[0], 0x4342), halves_of(x[1], 0x4140), halves_of(x[1], 0x4342));
    hi = make_uint4(halves_of(x[2], 0x4140), halves_of(x[2], 0x4342), halves_of(x[3], 0x4140), halves_of(x[3], 0x4342));
    unsigned char* r = slab + row * 128;
    // lanes of the second slab store their second chunk first: other banks
    const int c0 = ((2 * ch + odd) ^ (row & 7)) * 16, c1 = ((2 * ch + (odd ^ 1)) ^ (row & 7)) * 16;
    *reinterpret_cast<uint4*>(r + c0) = odd ? hi : lo;
    *reinterpret_cast<uint4*>(r + c1) = odd ? lo : hi;
}

// HD: padded head size; Q2: queries as hi + lo (fp32), P2: weights as hi + lo
// (fp32 and fp16 outputs; bf16 outputs keep 8 bits, against the half's 11).
template <int HD, bool Q2, bool P2>
__global__ void __launch_bounds__(RowsCfg<HD>::THREADS, 1)
    kvb_rows_kernel(const KvbAttnArgs a, const RowsPlan plan, float* parts, float2* stats) {
    using C = RowsCfg<HD>;
    constexpr int BN = C::BN, NG = BN / 16;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* sq = sm;                                              // [hi, lo][slab][128 rows][128 B]
    unsigned char* sk = sm + (Q2 ? 2 : 1) * C::SLABS * C::QSLAB;         // [buffer][slab][BN][128 B]
    unsigned char* sv = sk + C::NBUF * C::TILE;
    __shared__ __align__(8) uint64_t q_full, q_free, k_full[2], k_free[2], v_full[2], v_free[2], s_full[2], p_full[2],
        o_full, drained;
    __shared__ uint32_t tmem_base;
    __shared__ int dead;
    __shared__ float s_scale[4][2 * NG];         // K, V scales of a tile's 16-token groups
    __shared__ float s_row[2][kRows];            // score factors of the unit's rows
    __shared__ float s_stat[2][C::STREAMS][3][kRows];
    const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    const int hd = a.c.hd, G = a.heads / a.c.heads, B = a.c.block;
    if (tid == 0) {
        dead = 0;
        mbar_init(&q_full, 128), mbar_init(&q_free, 1), mbar_init(&o_full, 1), mbar_init(&drained, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], 128), mbar_init(&k_free[i], 1), mbar_init(&v_full[i], 128), mbar_init(&v_free[i], 1);
            mbar_init(&s_full[i], 1), mbar_init(&p_full[i], 128);
        }
        mbar_fence_init();
    }
    // every earlier kernel of the stream is complete before this one takes the
    // SM's tensor memory, and the next ones start only once every CTA has it
    pdl_wait();
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)),
                     "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_trigger();
    const uint32_t tmem = tmem_base;
    constexpr uint32_t kO = C::STREAMS == 2 ? 2 * BN : 256;              // first output column
    auto wait = [&](uint64_t* bar, uint32_t parity, bool spin = false) {
        if (*(volatile int*)&dead) return;
        if (!(spin ? mbar_wait_spin(bar, parity) : mbar_wait(bar, parity))) {
            dead = 1;
            atomicOr(&g_kvb_rows_errors, kErrWait);
        }
    };
    Seg seg;
    int64_t lo, hi;
    rows_share(plan, a.c.heads, gridDim.x, blockIdx.x, &lo, &hi);
    const bool any = seg.begin(a, plan, lo, hi);
    int J = 0, sn = 0;                           // tiles and units of this CTA so far

    if (warp * 32 >= C::SOFT + 128) {
        // ------------------------------------------------------- products
        if (lane == 0 && any) {
            constexpr uint32_t id_s = idesc_f16(kRows, BN, false), id_o = idesc_f16(kRows, HD, true);
            do {
                wait(&q_full, sn & 1, true);
                auto scores = [&](int jj) {
                    const int T = J + jj, kb = T % C::NBUF;
                    wait(&k_full[kb], (T / C::NBUF) & 1, true);
                    tc_fence_after();
                    const uint32_t d = tmem + (T & 1) * BN;
#pragma unroll
                    for (int s = 0; s < C::SLABS; ++s) {
                        const uint64_t da = smem_desc(sq + s * C::QSLAB), db = smem_desc(sk + kb * C::TILE + s * C::SLAB);
                        const uint64_t dl = smem_desc(sq + (C::SLABS + s) * C::QSLAB);
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk) {
                            mma_f16_ss(d, da + 2 * kk, db + 2 * kk, id_s, s > 0 || kk > 0);
                            if (Q2) mma_f16_ss(d, dl + 2 * kk, db + 2 * kk, id_s, 1u);
                        }
                    }
                    mma_commit(&k_free[kb]);
                    mma_commit(&s_full[T & 1]);
                    if (jj == seg.n - 1) mma_commit(&q_free);
                };
                scores(0);
                if (seg.n > 1) scores(1);
                for (int jj = 0; jj < seg.n; ++jj) {
                    const int T = J + jj, vb = T % C::NBUF;
                    wait(&v_full[vb], (T / C::NBUF) & 1, true);
                    wait(&p_full[T & 1], (T >> 1) & 1, true);
                    tc_fence_after();
                    const uint32_t d = tmem + kO + (C::STREAMS == 2 ? (T & 1) * HD : 0), ap = tmem + (T & 1) * BN;
                    const uint64_t db = smem_desc_mn(sv + vb * C::TILE, C::SLAB);
                    const uint32_t more = jj >= C::STREAMS;              // the stream's first tile writes
#pragma unroll
                    for (int s = 0; s < BN / 16; ++s) {
                        const uint32_t at = ap + 32 * (s >> 1) + 8 * (s & 1);
                        mma_f16_ts(d, at, db + 128 * s, id_o, more || s > 0);
                        if (P2) mma_f16_ts(d, at + 16, db + 128 * s, id_o, 1u);
                    }
                    mma_commit(&v_free[vb]);
                    if (jj == seg.n - 1) mma_commit(&o_full);
                    if (jj + 2 < seg.n) scores(jj + 2);
                }
                J += seg.n, ++sn;
            } while (seg.next(a, plan));
            mma_commit(&drained);
            mbar_wait(&drained, 0u);             // also after a wait that gave up: nothing in flight below
        }
    } else if (tid >= C::SOFT) {
        // -------------------------------------------------------- convert
        const int c = tid - C::SOFT;
        constexpr int CH = HD / 16, PER = BN * CH / 128;                 // 16-code chunks of a row, of a thread
        if (any) {
            // A tile's K, then its V: the next of them on its way in registers
            // while this one is converted (one loop body: code that several
            // roles run at once has to stay within the instruction cache).
            Seg ld = seg;
            int lj = 0, lz = 0;                  // what is loaded next: tile of the unit, K or V
            bool more = true;
            uint4 cur[PER], nxt[PER];
            auto load = [&]() {
                if (!more) return;
                const int t0 = (ld.j + lj) * BN, len = ld.p + ld.rows / G;
                const int8_t* base = (lz ? a.c.v : a.c.k) + ld.slot * a.c.slot_stride +
                                     ((int64_t)ld.h * a.c.cap + t0) * hd;
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    const int idx = i * 128 + c, row = idx / CH, ch = idx % CH;
                    nxt[i] = make_uint4(0, 0, 0, 0);
                    if (t0 + row < len && ch * 16 < hd)
                        nxt[i] = *reinterpret_cast<const uint4*>(base + row * hd + ch * 16);
                }
                if ((lz ^= 1) == 0 && ++lj == ld.n) lj = 0, more = ld.next(a, plan);
            };
            load();
            do {
                // the unit's rows: row c of it
                if (sn > 0) wait(&q_free, (sn - 1) & 1);
                {
                    const int f = seg.m * kRows + c;
                    const bool live = f < seg.rows;
                    const int64_t at = (int64_t)(seg.r0 + f / G) * a.q_stride + (int64_t)(seg.h * G + f % G) * hd;
                    float mx = 0.0f;
                    bool bad = false;
                    if (live)
                        for (int d = 0; d < hd; d += 16) {
                            float y[16];
                            load16(a.q, a.type, at + d, y);
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                mx = fmaxf(mx, fabsf(y[i])), bad |= !(fabsf(y[i]) <= 3.402823466e38f);
                        }
                    // the largest element to [2^13, 2^14)
                    const int e = mx > 0.0f && !bad ? min(max(13 - ilogbf(mx), -120), 120) : 0;
                    const float up = a.scale < 0.0f ? -exp2f((float)e) : exp2f((float)e);
                    s_row[sn & 1][c] = bad ? NAN : fabsf(a.scale) * kLog2e * exp2f((float)-e);
                    for (int d = 0; d < HD; d += 16) {
                        float y[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) y[i] = 0.0f;
                        if (live && !bad && d < hd) load16(a.q, a.type, at + d, y);
                        uint32_t hh[8], ll[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float y0 = y[2 * i] * up, y1 = y[2 * i + 1] * up;
                            const __half2 h2 = __floats2half2_rn(y0, y1);
                            const float2 b2 = __half22float2(h2);
                            hh[i] = bits(h2);
                            if (Q2) ll[i] = bits(__floats2half2_rn(y0 - b2.x, y1 - b2.y));
                        }
                        const int slab = d / 64, ch = d % 64 / 8;
                        unsigned char* r = sq + slab * C::QSLAB + c * 128;
                        const int c0 = (ch ^ (c & 7)) * 16, c1 = ((ch + 1) ^ (c & 7)) * 16;
                        *reinterpret_cast<uint4*>(r + c0) = make_uint4(hh[0], hh[1], hh[2], hh[3]);
                        *reinterpret_cast<uint4*>(r + c1) = make_uint4(hh[4], hh[5], hh[6], hh[7]);
                        if (Q2) {
                            r += C::SLABS * C::QSLAB;
                            *reinterpret_cast<uint4*>(r + c0) = make_uint4(ll[0], ll[1], ll[2], ll[3]);
                            *reinterpret_cast<uint4*>(r + c1) = make_uint4(ll[4], ll[5], ll[6], ll[7]);
                        }
                    }
                }
                fence_async_smem();
                mbar_arrive(&q_full);
                const int n = seg.n;
#pragma unroll 1
                for (int jz = 0; jz < 2 * n; ++jz) {
                    const int z = jz & 1, T = J + (jz >> 1), kb = T % C::NBUF;
#pragma unroll
                    for (int i = 0; i < PER; ++i) cur[i] = nxt[i];
                    load();
                    if (z == 0 && c < 2 * NG) {
                        const int t = (seg.j + (jz >> 1)) * BN + c % NG * 16;
                        const float* s = (c < NG ? a.c.ks : a.c.vs) + seg.slot * a.c.scale_stride +
                                         (int64_t)seg.h * (a.c.cap / B);
                        // tile T - 4's readers are done: V of tile T - 1 went in after their weights
                        s_scale[T & 3][c] = t < seg.p + seg.rows / G ? s[t / B] : 0.0f;
                    }
                    if (T >= C::NBUF) wait(z ? &v_free[kb] : &k_free[kb], ((T - C::NBUF) / C::NBUF) & 1);
                    unsigned char* tile = (z ? sv : sk) + kb * C::TILE;
#pragma unroll
                    for (int i = 0; i < PER; ++i) {
                        const int idx = i * 128 + c, row = idx / CH, ch = idx % CH;
                        put_codes(tile + (ch / 4) * C::SLAB, row, ch % 4, (ch / 4) & 1, cur[i]);
                    }
                    fence_async_smem();
                    mbar_arrive(z ? &v_full[kb] : &k_full[kb]);
                }
                J += n, ++sn;
            } while (seg.next(a, plan));
        }
    } else if (any) {
        // -------------------------------------------------------- softmax
        const int w = C::STREAMS == 2 ? warp / 4 : 0, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        do {
            const int f = seg.m * kRows + row;
            const bool live = f < seg.rows;
            const int lim = seg.p + (live ? f : seg.rows - 1) / G;       // the last token that the row sees
            const int all_see = seg.p + seg.m * kRows / G;               // ... that every row sees
            float m = -INFINITY, l = 0.0f, svr = 0.0f, rsv = 0.0f;
            bool has = false;                                            // the stream's accumulator is written
            for (int jj = 0; jj < seg.n; ++jj) {
                const int T = J + jj;
                if (C::STREAMS == 2 && (T & 1) != w) continue;
                const int t0 = (seg.j + jj) * BN;
                const bool cut = t0 + BN - 1 > all_see;                  // some row does not see the whole tile
                const uint32_t ts = tmem + lanes + (T & 1) * BN;
                wait(&s_full[T & 1], (T >> 1) & 1);
                tc_fence_after();
                const float qs = s_row[sn & 1][row];
                const float* sc = s_scale[T & 3];
                float x = -INFINITY, xs = 0.0f;
#pragma unroll 1
                for (int c = 0; c < BN / 32; ++c) {
                    uint32_t v[32];
                    tmem_ld32(ts + c * 32, v);
                    tmem_ld_wait();
                    if (cut) {
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (t0 + c * 32 + i > lim) v[i] = 0xff800000u;
                    }
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        float y = __uint_as_float(v[16 * g]);
#pragma unroll
                        for (int i = 1; i < 16; ++i) y = fmaxf(y, __uint_as_float(v[16 * g + i]));
                        if (y != -INFINITY) x = fmaxf(x, y * (sc[2 * c + g] * qs));
                        xs = fmaxf(xs, sc[NG + 2 * c + g]);
                    }
                }
                if (__any_sync(0xffffffffu, x > m + kLazyScore || xs > svr * kLazyScale)) {
                    const float xm = fmaxf(x, m), xv = fmaxf(xs, svr);
                    const float el = xm == m ? 1.0f : ex2(m - xm), eo = el * (xv > 0.0f ? svr / xv : 0.0f);
                    if (has) {
                        if (C::STREAMS == 1 && T > 0) {                  // the products of the tile before
                            wait(&v_free[(T - 1) % C::NBUF], ((T - 1) / C::NBUF) & 1);
                            tc_fence_after();
                        }
                        const uint32_t to = tmem + lanes + kO + (C::STREAMS == 2 ? w * HD : 0);
#pragma unroll 1
                        for (int c = 0; c < HD / 16; ++c) {
                            uint32_t v[16];
                            tmem_ld16(to + c * 16, reinterpret_cast<int*>(v));
#pragma unroll
                            for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * eo);
                            tmem_st16(to + c * 16, v);
                        }
                    }
                    l *= el, m = xm, svr = xv;
                    rsv = svr > 1e-33f ? kWeightScale / svr : 0.0f;      // values below count as 0
                }
                has = true;
#pragma unroll 1
                for (int c = 0; c < BN / 32; ++c) {
                    uint32_t v[32], ph[16], pl[16];
                    tmem_ld32(ts + c * 32, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        const float fz = sc[2 * c + g] * qs, fv = sc[NG + 2 * c + g] * rsv;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const int k = 16 * g + 2 * i;
                            float e0 = ex2(fmaf(__uint_as_float(v[k]), fz, -m));
                            float e1 = ex2(fmaf(__uint_as_float(v[k + 1]), fz, -m));
                            if (cut) {
                                if (t0 + c * 32 + k > lim) e0 = 0.0f;
                                if (t0 + c * 32 + k + 1 > lim) e1 = 0.0f;
                            }
                            l += e0 + e1;
                            const float w0 = e0 * fv, w1 = e1 * fv;
                            const __half2 h2 = __floats2half2_rn(w0, w1);
                            ph[8 * g + i] = bits(h2);
                            if (P2) {
                                const float2 b2 = __half22float2(h2);
                                pl[8 * g + i] = bits(__floats2half2_rn(w0 - b2.x, w1 - b2.y));
                            }
                        }
                    }
                    tmem_st16(ts + c * 32, ph);
                    if (P2) tmem_st16(ts + c * 32 + 16, pl);
                }
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(&p_full[T & 1]);
            }
            // the unit's rows: both streams' accumulators joined
            float(*st)[3][kRows] = s_stat[sn & 1];
            st[w][0][row] = m, st[w][1][row] = l, st[w][2][row] = has ? svr * (1.0f / kWeightScale) : 0.0f;
            wait(&o_full, sn & 1);
            tc_fence_after();
            named_barrier_sync(1, C::SOFT);
            float mm = st[0][0][row];
            if (C::STREAMS == 2) mm = fmaxf(mm, st[C::STREAMS - 1][0][row]);
            float fo[2] = {0.0f, 0.0f}, ll = 0.0f;
#pragma unroll
            for (int s = 0; s < C::STREAMS; ++s) {
                const float e = st[s][0][row] == -INFINITY ? 0.0f : ex2(st[s][0][row] - mm);
                ll = fmaf(st[s][1][row], e, ll), fo[s] = st[s][2][row] * e;
            }
            // an accumulator that no tile of the unit went into holds what was there before
            const bool two = C::STREAMS == 2 && seg.n > 1;
            const int w0 = J & 1;                                        // the first tile's stream
            const bool whole = seg.j == 0 && seg.n == seg.tiles;
            const float inv = whole ? 1.0f / ll : 1.0f;
            const int64_t orow = (int64_t)(seg.r0 + f / G) * a.heads + seg.h * G + f % G;
            float* pt = parts + ((int64_t)blockIdx.x * 2 + (seg.j == 0)) * C::PART;
            constexpr int COLS = HD / C::STREAMS;
#pragma unroll 1
            for (int c = w * COLS; c < (w + 1) * COLS; c += 16) {
                int o0[16], o1[16];
                const uint32_t to = tmem + lanes + kO + c;
                tmem_ld16(to + (C::STREAMS == 2 ? w0 * HD : 0), o0);
                if (two) tmem_ld16(to + (w0 ^ 1) * HD, o1);
                float y[16];
                const float f0 = fo[C::STREAMS == 2 ? w0 : 0] * inv, f1 = fo[C::STREAMS == 2 ? w0 ^ 1 : 0] * inv;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    y[i] = __int_as_float(o0[i]) * f0;
                    if (two) y[i] = fmaf(__int_as_float(o1[i]), f1, y[i]);
                }
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<float4*>(pt + row * HD + c + 4 * i) =
                            make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
                } else if (live && c < hd) {
                    if (a.type == KVB_F32) {
                        float4* o = reinterpret_cast<float4*>(static_cast<float*>(a.out) + orow * hd + c);
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[i] = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
                    } else {
                        uint32_t q[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            if (a.type == KVB_BF16) {
                                const __nv_bfloat162 z = __floats2bfloat162_rn(y[2 * i], y[2 * i + 1]);
                                q[i] = *reinterpret_cast<const uint32_t*>(&z);
                            } else {
                                q[i] = bits(__floats2half2_rn(y[2 * i], y[2 * i + 1]));
                            }
                        }
                        uint4* o = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + orow * hd + c);
                        o[0] = make_uint4(q[0], q[1], q[2], q[3]), o[1] = make_uint4(q[4], q[5], q[6], q[7]);
                    }
                }
            }
            if (w == 0) {
                if (!whole) pt[kRows * HD + row] = mm, pt[kRows * (HD + 1) + row] = ll;
                else if (stats && live) stats[orow] = make_float2(mm, 1.0f / ll);
            }
            tc_fence_before();
            named_barrier_sync(1, C::SOFT);      // the accumulators may be overwritten
            tc_fence_after();
            J += seg.n, ++sn;
        } while (seg.next(a, plan));
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// Joins the units that shares cut: CTA c those whose first cut lies at the
// begin of share c. Also the rows without tokens: zeros.
template <int HD>
__global__ void __launch_bounds__(kFinishThreads) kvb_rows_finish(const KvbAttnArgs a, const RowsPlan plan,
                                                                const float* parts, float2* stats, int grid) {
    using C = RowsCfg<HD>;
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, hd = a.c.hd, G = a.heads / a.c.heads;
    for (int b = blockIdx.x; b < a.c.slots; b += gridDim.x) {
        const KvbSpan s = kvb_span(a.r, b);
        const int live = live_rows(s, a.c.cap);
        if (s.p >= 0 && live < s.n && tid == 0) atomicOr(&g_kvb_rows_errors, kKvbErrCapacity);
        const int64_t e0 = (int64_t)(s.r0 + live) * a.heads * hd, e1 = (int64_t)(s.r0 + s.n) * a.heads * hd;
        for (int64_t i = e0 + tid; i < e1; i += kFinishThreads) store1(a.out, a.type, i, 0.0f);
    }
    int64_t lo, hi, plo, phi;
    if (blockIdx.x == 0) return;
    rows_share(plan, a.c.heads, grid, blockIdx.x, &lo, &hi);
    rows_share(plan, a.c.heads, grid, blockIdx.x - 1, &plo, &phi);
    if (lo >= hi) return;
    Seg s;
    s.begin(a, plan, lo, hi);
    if (s.j == 0 || plo > lo - s.j) return;      // not cut here, or first cut before
    const int64_t end = lo - s.j + s.tiles;
    int last = blockIdx.x;                       // the last share with a part of the unit
    for (int64_t e = hi; e < end;) {
        int64_t l2, h2;
        rows_share(plan, a.c.heads, grid, ++last, &l2, &h2);
        e = h2;
    }
    const int c0 = blockIdx.x - 1;
    __shared__ float s_m[kRows], s_i[kRows];
    auto at = [&](int c) { return parts + ((int64_t)c * 2 + (c == c0)) * C::PART; };
    if (tid < kRows) {
        float m = -INFINITY, l = 0.0f;
        for (int c = c0; c <= last; ++c) m = fmaxf(m, at(c)[kRows * HD + tid]);
        for (int c = c0; c <= last; ++c) {
            const float mc = at(c)[kRows * HD + tid];
            if (mc != -INFINITY) l = fmaf(at(c)[kRows * (HD + 1) + tid], ex2(mc - m), l);
        }
        s_m[tid] = m, s_i[tid] = 1.0f / l;
        const int f = s.m * kRows + tid;
        if (stats && f < s.rows)
            stats[(int64_t)(s.r0 + f / G) * a.heads + s.h * G + f % G] = make_float2(m, 1.0f / l);
    }
    __syncthreads();
    for (int i = tid; i < kRows * HD / 4; i += kFinishThreads) {
        const int row = i / (HD / 4), d = i % (HD / 4) * 4, f = s.m * kRows + row;
        if (f >= s.rows || d >= hd) continue;
        const float m = s_m[row], inv = s_i[row];
        float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int c = c0; c <= last; ++c) {
            const float mc = at(c)[kRows * HD + row];
            if (mc == -INFINITY) continue;
            const float e = ex2(mc - m);
            const float4 x = *reinterpret_cast<const float4*>(at(c) + row * HD + d);
            y.x = fmaf(x.x, e, y.x), y.y = fmaf(x.y, e, y.y), y.z = fmaf(x.z, e, y.z), y.w = fmaf(x.w, e, y.w);
        }
        const int64_t o = ((int64_t)(s.r0 + f / G) * a.heads + s.h * G + f % G) * hd + d;
        store1(a.out, a.type, o, y.x * inv), store1(a.out, a.type, o + 1, y.y * inv);
        store1(a.out, a.type, o + 2, y.z * inv), store1(a.out, a.type, o + 3, y.w * inv);
    }
}

// mass[t] += the probabilities of token t over the rows and the query heads of
// its KV head: one thread per token, in row order.
constexpr int kMassThreads = 128;
__global__ void __launch_bounds__(kMassThreads) kvb_rows_mass(const KvbAttnArgs a, const float2* stats) {
    pdl_wait();
    pdl_trigger();
    const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, t = blockIdx.x * kMassThreads + tid;
    const KvbSpan sp = kvb_span(a.r, b);
    const int n = live_rows(sp, a.c.cap), hd = a.c.hd, G = a.heads / a.c.heads, B = a.c.block;
    if (n <= 0 || blockIdx.x * kMassThreads >= sp.p + n) return;
    __shared__ __align__(16) float q[kKvbMaxHd];
    const int64_t head = b * a.c.slot_stride + (int64_t)h * a.c.cap * hd;
    const float sk = t < sp.p + n ? a.c.ks[b * a.c.scale_stride + (int64_t)h * (a.c.cap / B) + t / B] : 0.0f;
    float sum = 0.0f;
    for (int i = 0; i < n; ++i) {
        for (int g = 0; g < G; ++g) {
            const int64_t r = sp.r0 + i;
            __syncthreads();
            for (int d = tid * 16; d < hd; d += kMassThreads * 16) {
                load16(a.q, a.type, r * a.q_stride + (int64_t)(h * G + g) * hd + d, q + d);
#pragma unroll
                for (int e = 0; e < 16; ++e) q[d + e] *= a.scale * kLog2e;
            }
            __syncthreads();
            if (t > sp.p + i) continue;
            const uint4* row = reinterpret_cast<const uint4*>(a.c.k + head + (int64_t)t * hd);
            float z = 0.0f;
            for (int c = 0; c < hd / 16; ++c) {
                const uint4 w = row[c];
                const int8_t* k = reinterpret_cast<const int8_t*>(&w);
#pragma unroll
                for (int e = 0; e < 16; ++e) z = fmaf((float)k[e], q[c * 16 + e], z);
            }
            const float2 st = stats[r * a.heads + h * G + g];
            sum = fmaf(ex2(z * sk - st.x), st.y, sum);
        }
    }
    if (t < sp.p + n) a.mass[((int64_t)b * a.c.heads + h) * a.c.cap + t] += sum;
}

int rows_hd(int hd) { return hd <= 64 ? 64 : hd <= 128 ? 128 : 256; }

size_t up16(size_t x) { return (x + 15) & ~(size_t)15; }

struct RowsLayout {                              // byte offsets in the scratch
    size_t unit, first, parts, stats, total;
    RowsLayout(const KvbCache& c, int heads, int rows, bool mass) {
        const int hd = rows_hd(c.hd);
        unit = 16;
        first = unit + (size_t)max_units(c, heads, rows) * sizeof(int4);
        parts = up16(first + ((size_t)c.slots + 1) * sizeof(int));
        stats = parts + (size_t)kSms * 2 * kRows * (hd + 2) * sizeof(float);
        total = stats + (mass ? (size_t)rows * heads * sizeof(float2) : 0);
    }
};

template <int HD>
cudaError_t rows_launch(const KvbAttnArgs& a, cudaStream_t st) {
    using C = RowsCfg<HD>;
    const RowsLayout L(a.c, a.heads, a.r.rows, a.mass != nullptr);
    char* s = static_cast<char*>(a.scratch);
    const RowsPlan plan{reinterpret_cast<int*>(s), reinterpret_cast<int4*>(s + L.unit), reinterpret_cast<int*>(s + L.first)};
    float* parts = reinterpret_cast<float*>(s + L.parts);
    float2* stats = a.mass ? reinterpret_cast<float2*>(s + L.stats) : nullptr;
    cudaError_t e = launch_k(kvb_rows_plan, dim3(1), dim3(kPlanThreads), 0, st, a, plan, C::BN,
                             (int)max_units(a.c, a.heads, a.r.rows));
    if (e != cudaSuccess) return e;
    const bool q2 = a.type == KVB_F32;
    const auto kern = a.type == KVB_F32    ? kvb_rows_kernel<HD, true, true>
                      : a.type == KVB_BF16 ? kvb_rows_kernel<HD, false, false>
                                           : kvb_rows_kernel<HD, false, true>;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::smem(q2));
    if (e != cudaSuccess) return e;
    e = launch_k(kern, dim3(kSms), dim3(C::THREADS), C::smem(q2), st, a, plan, parts, stats);
    if (e != cudaSuccess) return e;
    e = launch_k(kvb_rows_finish<HD>, dim3(kSms), dim3(kFinishThreads), 0, st, a, plan, (const float*)parts, stats, kSms);
    if (e != cudaSuccess || !stats) return e;
    return launch_k(kvb_rows_mass, dim3((a.c.cap + kMassThreads - 1) / kMassThreads, a.c.heads, a.c.slots),
                    dim3(kMassThreads), 0, st, a, (const float2*)stats);
}

}  // namespace

size_t kvb_rows_scratch(const KvbCache& c, int heads, int rows, bool mass) {
    return RowsLayout(c, heads, rows, mass).total;
}

cudaError_t launch_kvb_rows(const KvbAttnArgs& a, cudaStream_t st) {
    switch (rows_hd(a.c.hd)) {
        case 64: return rows_launch<64>(a, st);
        case 128: return rows_launch<128>(a, st);
        default: return rows_launch<256>(a, st);
    }
}

}  // namespace w8a8

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
// joins. plan_rows lists the units on the device, since lengths are device data.
//
// Warps of a CTA (one CTA an SM, all 512 TMEM columns):
//   softmax   8 warps: a row's columns are split between two threads, which meet
//             at one reducing barrier a tile (does any score pass its reference?).
//   convert   7 warps: int8 codes -> exact halves (byte permutes, one
//             subtraction) in 128-byte-swizzled tiles, the next tile's codes on
//             their way in registers; the query rows as hi + lo halves (22 bits)
//             of the row scaled by a power of two (16-bit queries are exact in
//             one half), in TMEM where it has room (head sizes up to 128), which
//             halves what the score products read from shared memory.
//   products  one thread: S = Q K^T for the tile after next, then O += P V (P from
//             TMEM, written over S: hi in columns 0-7, lo in 8-15 of every 16;
//             V as it lies, its rows being the contraction).
// Block scales do not touch the codes: K's multiplies the scores of its 16
// columns, V's goes into the weights, exp(z - m) sv / 2^r 2^7 by one
// exponential. m is the row's largest score and 2^r its largest exp(z - m) sv,
// both over the tokens that it sees and lazily moved, so that the accumulator is
// rescaled rarely; blocks that the row does not see, or gives no weight, leave the
// others' halves their bits, however large their values are.
//
// Bound by two chains that run beside each other: the softmax warps (wait, read 64
// scores, exponentials, write the weights; two warps a scheduler, half of all issue
// slots) and the products' thread (for fp32 2,048 cycles of products a tile, the rest
// hand-overs). 8,192 causal rows, 16 heads on 8 KV heads of 128, fp32: 650 us of a
// call's 690, 0.42 PFLOP/s of the formula's operations and 0.84 of those done (hi and
// lo); the tensor pipe is active 42 % of the time, 2.5 % of the DRAM's rate is used.
// Four softmax threads a row (24 warps) took 7 to 11 % longer; two groups that take
// turns on the tiles with an accumulator each (64-channel heads) 35 %. Head sizes above
// 128 have room for one buffer and one tile on its way: 4,096 fp32 rows, 16 heads on
// 8 KV heads of 256, 668 us (0.2 PFLOP/s, tensor pipe 19 %).
#include <type_traits>

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
// log2 of: how far a score may pass m, the most that a weight as a half should come to, and
// what its reference stands for
constexpr float kLazyScore = 6.0f, kMostWeight = 15.0f, kWeightLog = 7.0f;
constexpr float kLeastLog = -126.0f;             // the least reference: a normal number
constexpr unsigned int kErrWait = 256u;          // error bit 8: a pipeline wait gave up
// The tensor cores round each product's running sum towards zero: an accumulator
// is moved out and begun anew every kFold tiles (fp32, relative error of an output over
// 8,192 tokens: 6.3e-6 never moved, 1.8e-6 every 8, 1.0e-6 every 4, 8e-7 every 3,
// 6.4e-7 every 2; moving out every 2 tiles instead of 4 costs 11 % of the time).
template <typename T>
constexpr int kFold = sizeof(T) == 4 ? 3 : 32;   // (16-bit outputs round by 2e-4 and more)
constexpr int kFinishThreads = 256;

template <int HD>
struct RowsCfg {
    static constexpr int BN = HD == 256 ? 64 : 128;
    static constexpr int NBUF = HD == 256 ? 1 : 2;
    static constexpr bool QT = HD <= 128;        // queries in TMEM
    static constexpr int SLABS = HD / 64;        // 64-channel slabs of a tile
    static constexpr int QSLAB = kRows * 128, SLAB = BN * 128, TILE = SLABS * SLAB;   // bytes
    static constexpr int SOFT = 256;             // softmax threads
    static constexpr int CONV = 224;             // converting threads
    static constexpr int THREADS = 32 + SOFT + CONV;   // 16 warps: 128 registers a thread
    static constexpr int RAW = BN * HD, NRAW = HD == 256 ? 1 : 4;   // bytes of a tile's codes; tiles on their way
    // a prepared query row: halves (hi, lo), its score factor in 16 bytes more
    // (lanes that read one row each then meet no bank conflicts)
    static constexpr int qrow(int qbytes) { return HD * qbytes + 16; }
    static constexpr int stage(int qbytes) { return QT && 32 * qrow(qbytes) > RAW ? 32 * qrow(qbytes) : RAW; }
    static constexpr size_t smem(int qbytes) {
        return 1024 + (QT ? 0 : (size_t)(qbytes == 4 ? 2 : 1) * SLABS * QSLAB) + (size_t)NBUF * 2 * TILE +
               (size_t)NRAW * stage(qbytes);
    }
    // floats of a partial unit, and of a CTA's moved-out accumulator: channels in
    // fours, [HD / 4][row][4], then maxima and sums of the rows
    static constexpr size_t PART = (size_t)kRows * (HD + 2), ACC = (size_t)kRows * HD;
};

struct RowsPlan {                                // in scratch
    int64_t* head;                               // [2]: cost of all units of one KV head, units
    RowsUnit* unit;
    int* first;                                  // [slots + 1]: the slots' first units
    RowsShare* share;                            // [kSms]
};

__host__ __device__ inline int64_t max_units(const KvbCache& c, int heads, int rows) {
    return (int64_t)rows * (heads / c.heads) / kRows + (rows < c.slots ? rows : c.slots);
}

__device__ __forceinline__ int live_rows(const KvbSpan& s, int cap) { return s.p < 0 ? 0 : max(min(s.n, cap - s.p), 0); }

// exclusive scan over the CTA's NT threads; *sum the total
template <int NT>
__device__ __forceinline__ int64_t block_scan(int64_t x, int64_t* sum) {
    __shared__ int64_t w[NT / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
    int64_t upto = x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t o = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += o;
    }
    if (lane == 31) w[warp] = upto;
    __syncthreads();
    int64_t before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < NT / 32; ++i) {
        if (i < warp) before += w[i];
        all += w[i];
    }
    __syncthreads();
    *sum = all;
    return before + upto - x;
}

// The plan, by one CTA of NT threads.
template <int NT>
__device__ __forceinline__ void plan_rows(const KvbAttnArgs& a, const RowsPlan& plan, int bn, int most) {
    const int tid = threadIdx.x, S = a.c.slots, G = a.heads / a.c.heads;
    __shared__ int64_t s_before[NT];             // the first units' costs before them
    int64_t counted = 0, sum;
    // (offsets out of order may count more than `most` units: rows are then left out)
    for (int b0 = 0; b0 < S; b0 += NT) {
        const int b = b0 + tid;
        const int n = b < S ? (live_rows(kvb_span(a.r, b), a.c.cap) * G + kRows - 1) / kRows : 0;
        const int64_t at = block_scan<NT>(n, &sum);
        if (b < S) plan.first[b] = (int)min(counted + at, (int64_t)most + 1);
        counted += sum;
    }
    const int units = (int)min(counted, (int64_t)most);
    if (tid == 0) plan.first[S] = units;
    __syncthreads();
    int64_t total = 0;
    for (int u0 = 0; u0 < units; u0 += NT) {
        const int u = u0 + tid;
        RowsUnit v{};
        if (u < units) {
            int b = 0;
            int hi = S;                          // the last slot with first <= u that has units
            while (hi - b > 1) {
                const int mid = (b + hi) >> 1;
                if (plan.first[mid] <= u) b = mid;
                else hi = mid;
            }
            const KvbSpan sp = kvb_span(a.r, b);
            v.slot = b, v.m = u - plan.first[b], v.p = sp.p, v.r0 = sp.r0, v.rows = live_rows(sp, a.c.cap) * G;
            v.tiles = (sp.p + min(v.m * kRows + kRows - 1, v.rows - 1) / G) / bn + 1;
        }
        v.before = total + block_scan<NT>(u < units ? v.tiles + kUnitCost : 0, &sum);
        if (u < units) plan.unit[u] = v;
        if (u0 == 0) s_before[tid] = v.before;
        total += sum;
    }
    if (tid == 0) plan.head[0] = total, plan.head[1] = units;
    __syncthreads();
    // the shares, and where they begin (searched here once: a search through
    // global memory in every CTA of two kernels took 1.5 us in each)
    auto before = [&](int u) { return u < NT ? s_before[u] : plan.unit[u].before; };
    auto tiles = [&](int u) { return plan.unit[u].tiles; };
    for (int c = tid; c < kSms; c += NT) plan.share[c] = share_of(c, kSms, total, a.c.heads, units, before, tiles);
}

// A run of tiles of one unit within a CTA's share [x, end) of the cost.
struct Seg {
    int64_t x, end, begin_x;                     // begin_x: where the unit's cost begins
    int h, u, j, n, tiles;                       // KV head, unit; first tile, tiles here, tiles of the unit
    int slot, m, p, r0, rows;                    // rows: the slot's n * G live ones
    __device__ __forceinline__ void unit(const RowsPlan& plan) {
        const RowsUnit v = plan.unit[u];
        slot = v.slot, m = v.m, tiles = v.tiles, p = v.p, r0 = v.r0, rows = v.rows;
        // a unit's own cost comes before its tiles
        j = (int)max(x - begin_x - kUnitCost, (int64_t)0);
        n = (int)(min(max(end - begin_x - kUnitCost, (int64_t)0), (int64_t)tiles) - j);
    }
    __device__ __forceinline__ bool begin(const RowsPlan& plan, int cta) {
        const RowsShare w = plan.share[cta];
        x = w.lo, end = w.hi;
        if (x >= end) return false;
        h = w.h, u = w.u;
        begin_x = h * plan.head[0] + plan.unit[u].before;
        unit(plan);
        return n > 0 || next(plan);              // a share may end before the unit's first tile
    }
    __device__ __forceinline__ bool next(const RowsPlan& plan) {
        do {
            x = begin_x + kUnitCost + tiles;
            if (x >= end) return false;
            if (++u == (int)plan.head[1]) u = 0, ++h;
            begin_x = x;                         // units lie side by side
            unit(plan);
        } while (n <= 0);
        return true;
    }
};

// 16 codes as 16 halves in two 16-byte chunks of a swizzled row (`more`: rows
// that the slab pointer is already past)
__device__ __forceinline__ void put_codes(unsigned char* slab, int row, int ch, int odd, uint4 w, int more) {
    const uint32_t x[4] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u};
    uint4 lo, hi;
    lo = make_uint4(halves_of(x[0], 0x4140), halves_of(x[0], 0x4342), halves_of(x[1], 0x4140), halves_of(x[1], 0x4342));
    hi = make_uint4(halves_of(x[2], 0x4140), halves_of(x[2], 0x4342), halves_of(x[3], 0x4140), halves_of(x[3], 0x4342));
    unsigned char* r = slab + row * 128;
    // lanes of the second slab store their second chunk first: other banks
    const int sw = (row + more) & 7, c0 = ((2 * ch + odd) ^ sw) * 16, c1 = ((2 * ch + (odd ^ 1)) ^ sw) * 16;
    *reinterpret_cast<uint4*>(r + c0) = odd ? hi : lo;
    *reinterpret_cast<uint4*>(r + c1) = odd ? lo : hi;
}

template <typename T>
__device__ __forceinline__ void load_row16(const T* p, float* y) {
    kvb_load8<T>(p, y);
    kvb_load8<T>(p + 8, y + 8);
}

// Whether the mbarrier phase with the given parity is over.
__device__ __forceinline__ bool mbar_done(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}

// Bounded; once one wait has given up nobody waits any more, so that every role
// runs to its end (the result is then worthless, the error bit is set). Out of
// line: the roles' loops together have to fit the instruction cache.
__device__ __noinline__ void wait_long(uint64_t* bar, uint32_t parity, int* dead) {
    if (*(volatile int*)dead) return;
    if (!mbar_wait(bar, parity)) {
        *(volatile int*)dead = 1;
        atomicOr(&g_kvb_rows_errors, kErrWait);
    }
}

// log2 of a scale, its exponent and its mantissa (in [1, 2)) apart: off by 2^-22 and the
// rounding of the sum (for scales from 2^-16 to 2^16 2^-21, at most 2^-18), where the
// logarithm of the whole may be off by 2 ulp. (As an integer with 22 bits behind the point
// it would keep 2^-22 at any size: 4 % of the time, in registers that spill.)
__device__ __forceinline__ float log2_scale(float s) {
    const bool small = s < 1.17549435e-38f;      // subnormal
    const uint32_t u = __float_as_uint(small ? s * 16777216.0f : s);
    const float y = (float)((int)(u >> 23) - (small ? 151 : 127)) + __log2f(__uint_as_float((u & 0x7fffffu) | 0x3f800000u));
    return u ? y : -INFINITY;
}

__device__ __forceinline__ float exp2_int(float e) { return __int_as_float((127 + (int)e) << 23); }   // -126 .. 127

// Barrier `id` among n threads, and whether x holds for any of them.
__device__ __forceinline__ bool barrier_any(int id, int n, bool x) {
    uint32_t r;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.u32 p, %3, 0;\n barrier.cta.red.or.pred q, %1, %2, p;\n"
        " selp.u32 %0, 1, 0, q;\n}\n"
        : "=r"(r)
        : "r"(id), "r"(n), "r"((uint32_t)x)
        : "memory");
    return r != 0;
}

// Powers of two that bring a row's largest element (bits of |x|) to [2^13, 2^14),
// and its score factor; rows with a NaN or an infinity (and bad set) give NaN.
__device__ __forceinline__ float row_factor(uint32_t top, float scale, float* up, bool* bad) {
    *bad = top >= 0x7f800000u;
    const int e = top && !*bad ? min(140 - (int)(top >> 23), 120) : 0;
    *up = __int_as_float((127 + e) << 23) * (scale < 0.0f ? -1.0f : 1.0f);
    return *bad ? NAN : fabsf(scale) * kLog2e * __int_as_float((127 - e) << 23);
}

// The plan alone: where the query rows need no preparation, or the slots are many.
constexpr int kPlanThreads = 256;
// A few slots: the plan in the queries' kernel, whose CTAs then each count the
// slots (1 slot, 32 rows of 16 heads 14.9 -> 13.3 us and a launch less of the host;
// 64 slots 37.3 -> 36.0, 128 slots 57.8 -> 58.7, 512 slots 204 -> 250).
constexpr int kFoldSlots = 64;
constexpr int kFullUnits = 4 * kSms;
__global__ void __launch_bounds__(kPlanThreads) kvb_rows_plan(const KvbAttnArgs a, const RowsPlan plan, int bn, int most) {
    pdl_wait();
    pdl_trigger();
    plan_rows<kPlanThreads>(a, plan, bn, most);
}

// The units' query rows as the products take them, 32 rows at a time, a lane per 8
// channels: halves in unit order, so that a stage of the main kernel's ring is
// one run of memory. (Converted there, row by row, they cost each unit 12,000
// cycles of cold code and scattered loads between two streams of products.)
// With bn (tokens of a tile) the first CTA makes the plan and the others find
// their unit by themselves; else the plan is there.
template <int HD, typename T>
__global__ void __launch_bounds__(HD / 8 * 32) kvb_rows_queries(const KvbAttnArgs a, const RowsPlan plan,
                                                              unsigned char* out, int units, int bn, int per) {
    pdl_wait();
    pdl_trigger();
    constexpr int RS = RowsCfg<HD>::qrow(sizeof(T)), LPR = HD / 8;       // bytes, lanes of a row
    const int x0 = ((int)blockIdx.x - (bn > 0)) * per, u = x0 / 4, h = blockIdx.y, G = a.heads / a.c.heads;
    if (x0 < 0) {
        if (h == 0) plan_rows<HD / 8 * 32>(a, plan, bn, units);
        return;
    }
    __shared__ int s_slot, s_m;
    if (bn == 0) {
        if (threadIdx.x == 0) {
            const bool ok = u < plan.head[1];
            s_slot = ok ? plan.unit[u].slot : -1, s_m = ok ? plan.unit[u].m : 0;
        }
    } else if (threadIdx.x < 32) {               // unit u: the slots' units counted through
        const int lane = threadIdx.x;
        if (lane == 0) s_slot = -1;
        __syncwarp();
        int before = 0;
        for (int b0 = 0; b0 < a.c.slots && before <= u; b0 += 128) {     // four slots a lane in flight
            int n[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int b = b0 + 32 * i + lane;
                n[i] = b < a.c.slots ? (live_rows(kvb_span(a.r, b), a.c.cap) * G + kRows - 1) / kRows : 0;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (b0 + 32 * i >= a.c.slots) break;
                int upto = n[i];
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int o = __shfl_up_sync(0xffffffffu, upto, d);
                    if (lane >= d) upto += o;
                }
                const int at = u - before - (upto - n[i]);
                if (at >= 0 && at < n[i]) s_slot = b0 + 32 * i + lane, s_m = at;
                before += __shfl_sync(0xffffffffu, upto, 31);
            }
        }
    }
    __syncthreads();
    if (s_slot < 0) return;
    const KvbSpan sp = kvb_span(a.r, s_slot);
    const int rows = live_rows(sp, a.c.cap) * G, r = threadIdx.x / LPR, d = threadIdx.x % LPR * 8;
    for (int part = x0 % 4; part < x0 % 4 + per; ++part) {
        const int f = s_m * kRows + part * 32 + r;
        float x[8];
        uint32_t top = 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = 0.0f;
        if (f < rows && d < a.c.hd)
            kvb_load8<T>(static_cast<const T*>(a.q) + (int64_t)(sp.r0 + f / G) * a.q_stride + (int64_t)(h * G + f % G) * a.c.hd + d, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
        for (int i = 1; i < LPR; i <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, i));
        float up;
        bool bad;
        const float factor = row_factor(top, a.scale, &up, &bad);
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float y0 = bad ? 0.0f : x[2 * i] * up, y1 = bad ? 0.0f : x[2 * i + 1] * up;
            const __half2 h2 = __floats2half2_rn(y0, y1);
            const float2 b2 = __half22float2(h2);
            hi[i] = bits(h2), lo[i] = bits(__floats2half2_rn(y0 - b2.x, y1 - b2.y));
        }
        unsigned char* to = out + ((((int64_t)h * units + u) * 4 + part) * 32 + r) * RS;
        *reinterpret_cast<uint4*>(to + d * 2) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if (sizeof(T) == 4) *reinterpret_cast<uint4*>(to + HD * 2 + d * 2) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        if (d == 0) *reinterpret_cast<float*>(to + HD * (int)sizeof(T)) = factor;
    }
}

// HD: padded head size. Queries enter as hi + lo for fp32 (Q2), the weights
// always: one half would lose as much as a 16-bit output's rounding, and saves
// 8 % of the time.
template <int HD, typename T>
__global__ void __launch_bounds__(RowsCfg<HD>::THREADS, 1)
    kvb_rows_kernel(const KvbAttnArgs a, const RowsPlan plan, const unsigned char* queries, int units, float* parts,
                    float* accs, float2* stats) {
    using C = RowsCfg<HD>;
    constexpr int BN = C::BN, NG = BN / 16;
    constexpr int RAWS = C::stage(sizeof(T));
    constexpr bool Q2 = sizeof(T) == 4;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* sq = sm;                                              // [hi, lo][slab][128 rows][128 B]
    unsigned char* sk = sm + (C::QT ? 0 : (Q2 ? 2 : 1) * C::SLABS * C::QSLAB);   // [buffer][slab][BN][128 B]
    unsigned char* sv = sk + C::NBUF * C::TILE;
    unsigned char* raw = sv + C::NBUF * C::TILE;                         // [NRAW] codes as they lie in the cache, or query rows
    __shared__ __align__(8) uint64_t q_full, q_free, k_full[2], k_free[2], v_full[2], v_free[2], s_full[2], p_full[2],
        o_full, drained, raw_full[C::NRAW];
    __shared__ uint32_t tmem_base;
    __shared__ int dead;
    __shared__ float s_row[2][kRows];            // score factors of the unit's rows
    // a row's half, for its other thread: largest score (at the end the sum), largest log2 of a weight
    __shared__ float s_half[2][kRows], s_top[2][kRows];
    const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31;
    const int hd = a.c.hd, G = a.heads / a.c.heads;
    if (tid == 0) {
        dead = 0;
        mbar_init(&q_full, 128), mbar_init(&q_free, 1), mbar_init(&o_full, 1), mbar_init(&drained, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], C::CONV), mbar_init(&k_free[i], 1);
            mbar_init(&v_full[i], C::CONV), mbar_init(&v_free[i], 1);
            mbar_init(&s_full[i], 1), mbar_init(&p_full[i], C::SOFT);
        }
        for (int i = 0; i < C::NRAW; ++i) mbar_init(&raw_full[i], 1);
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
    constexpr uint32_t kO = 256, kQ = 384;       // columns: two score tiles, outputs, queries (hi, lo)
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (!mbar_done(bar, parity)) wait_long(bar, parity, &dead);
    };
    Seg seg;
    const bool any = seg.begin(plan, blockIdx.x);
    int J = 0, sn = 0;                           // tiles and units of this CTA so far

    if (warp == 0) {
        // ------------------------------------------------------- products
        if (any) {                               // the whole warp, one lane issuing
            const uint32_t lead = lane == 0;
            constexpr uint32_t id_s = idesc_f16(kRows, BN, false), id_o = idesc_f16(kRows, HD, true);
            do {
                wait(&q_full, sn & 1);
                auto scores = [&](int jj) {
                    const int tl = J + jj, kb = tl % C::NBUF;
                    wait(&k_full[kb], (tl / C::NBUF) & 1);
                    tc_fence_after();
                    const uint32_t d = tmem + (tl & 1) * BN;
                    // the lo halves first: every product rounds the running sum towards
                    // zero, and theirs is small
#pragma unroll
                    for (int part = Q2 ? 1 : 0; part >= 0; --part)
#pragma unroll
                        for (int s = 0; s < C::SLABS; ++s) {
                            const uint64_t db = smem_desc(sk + kb * C::TILE + s * C::SLAB);
                            const uint64_t da = smem_desc(sq + (part * C::SLABS + s) * C::QSLAB);
                            const uint32_t at = tmem + kQ + part * 64 + s * 32;
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk) {
                                const bool more = part != (Q2 ? 1 : 0) || s > 0 || kk > 0;
                                if constexpr (C::QT) mma_f16_ts(d, at + 8 * kk, db + 2 * kk, id_s, more, lead);
                                else mma_f16_ss(d, da + 2 * kk, db + 2 * kk, id_s, more, lead);
                            }
                        }
                    mma_commit(&s_full[tl & 1], lead);
                    mma_commit(&k_free[kb], lead);
                    if (jj == seg.n - 1) mma_commit(&q_free, lead);
                };
                scores(0);
                if (seg.n > 1) scores(1);
                for (int jj = 0; jj < seg.n; ++jj) {
                    const int tl = J + jj, vb = tl % C::NBUF;
                    wait(&v_full[vb], (tl / C::NBUF) & 1);
                    wait(&p_full[tl & 1], (tl >> 1) & 1);
                    tc_fence_after();
                    const uint32_t d = tmem + kO, ap = tmem + (tl & 1) * BN;
                    const uint64_t db = smem_desc_mn(sv + vb * C::TILE, C::SLAB);
#pragma unroll
                    for (int s = 0; s < BN / 16; ++s) {                  // 16 tokens: 8 columns hi, 8 lo
                        const uint32_t at = ap + 16 * s;
                        mma_f16_ts(d, at, db + 128 * s, id_o, jj % kFold<T> > 0 || s > 0, lead);
                        mma_f16_ts(d, at + 8, db + 128 * s, id_o, 1u, lead);
                    }
                    mma_commit(&v_free[vb], lead);
                    if (jj == seg.n - 1) mma_commit(&o_full, lead);
                    if (jj + 2 < seg.n) scores(jj + 2);
                }
                J += seg.n, ++sn;
            } while (seg.next(plan));
            mma_commit(&drained, lead);
            mbar_wait(&drained, 0u);             // also after a wait that gave up: nothing in flight below
        }
    } else if (tid >= 32 + C::SOFT) {
        // -------------------------------------------------------- convert
        const int c = tid - 32 - C::SOFT;
        if (any) {
            // A tile's K, then its V, in one loop body (see wait_long). A tile's codes
            // are one run of the cache: one bulk copy each, NRAW of them on their way
            // (what lies behind the slot's last token is finite and masked). A unit's
            // prepared query rows come the same way before its first tile, 32 rows a
            // stage.
            constexpr int CH = HD / 16, STEP = C::CONV / CH;             // 16-code chunks of a row; rows between a thread's
            constexpr int PER = (BN + STEP - 1) / STEP;                  // ... chunks of a thread
            constexpr int NQ = C::QT ? kRows / 32 : 0;                   // stages of query rows
            constexpr int RS = C::qrow(sizeof(T));
            Seg ld = seg;                        // first thread: the unit of the next copy, its place in the unit
            int li = 0, lq = 0;
            bool more = c == 0;
            const int row0 = c / CH, ch = c % CH;
            const bool live_ch = ch * 16 < hd;
            auto copy = [&]() {
                if (!more) return;
                uint64_t* bar = &raw_full[lq % C::NRAW];
                unsigned char* to = raw + lq % C::NRAW * RAWS;
                if (li < NQ) {
                    mbar_expect_tx(bar, 32 * RS);
                    bulk_g2s(to, queries + (((int64_t)ld.h * units + ld.u) * NQ + li) * 32 * RS, 32 * RS, bar);
                } else {
                    const int t0 = (ld.j + (li - NQ) / 2) * BN, n = min(BN, ld.p + ld.rows / G - t0);
                    const int8_t* at = ((li - NQ) & 1 ? a.c.v : a.c.k) + ld.slot * a.c.slot_stride +
                                       ((int64_t)ld.h * a.c.cap + t0) * hd;
                    mbar_expect_tx(bar, n * hd);
                    bulk_g2s(to, at, n * hd, bar);
                }
                ++lq;
                if (++li == NQ + 2 * ld.n) li = 0, more = ld.next(plan);
            };
            int at = 0;                          // stages of the ring used so far
#pragma unroll 1
            for (int i = 0; i < C::NRAW; ++i) copy();
            do {
                // the unit's rows, one per thread of four warps
                if (c < kRows) {
                    const int qr = (warp & 3) * 32 + lane;
                    if (sn > 0) wait(&q_free, (sn - 1) & 1);
                    tc_fence_after();
                    if constexpr (C::QT) {       // this warp's 32 TMEM lanes are its rows
                        const int x = at + (warp & 3);
                        wait(&raw_full[x % C::NRAW], (x / C::NRAW) & 1);
                        const unsigned char* mine = raw + x % C::NRAW * RAWS + lane * RS;
                        s_row[sn & 1][qr] = *reinterpret_cast<const float*>(mine + HD * sizeof(T));
#pragma unroll 1
                        for (int d = 0; d < HD * (int)sizeof(T); d += 64) {
                            uint32_t v[16];
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                *reinterpret_cast<uint4*>(v + 4 * i) = *reinterpret_cast<const uint4*>(mine + d + 16 * i);
                            // lo halves begin 64 columns further
                            tmem_st16(tmem + ((uint32_t)((warp & 3) * 32) << 16) + kQ + (d < HD * 2 ? d / 4 : 64 + (d - HD * 2) / 4), v);
                        }
                        tmem_st_wait();
                    } else {                     // head sizes above 128: straight from the rows
                        const int f = seg.m * kRows + qr;
                        const bool live = f < seg.rows;
                        const T* q = static_cast<const T*>(a.q) + (int64_t)(seg.r0 + f / G) * a.q_stride +
                                     (int64_t)(seg.h * G + f % G) * hd;
                        uint32_t top = 0u;
#pragma unroll 1
                        for (int d = 0; live && d < hd; d += 16) {
                            float y[16];
                            load_row16<T>(q + d, y);
#pragma unroll
                            for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(y[i]) & 0x7fffffffu);
                        }
                        float up;
                        bool bad;
                        s_row[sn & 1][qr] = row_factor(top, a.scale, &up, &bad);
#pragma unroll 1
                        for (int d = 0; d < HD; d += 16) {
                            float y[16];
#pragma unroll
                            for (int i = 0; i < 16; ++i) y[i] = 0.0f;
                            if (live && !bad && d < hd) load_row16<T>(q + d, y);
                            uint32_t hh[8], ll[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                const float y0 = y[2 * i] * up, y1 = y[2 * i + 1] * up;
                                const __half2 h2 = __floats2half2_rn(y0, y1);
                                const float2 b2 = __half22float2(h2);
                                hh[i] = bits(h2), ll[i] = bits(__floats2half2_rn(y0 - b2.x, y1 - b2.y));
                            }
                            unsigned char* r = sq + d / 64 * C::QSLAB + qr * 128;
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                const int at16 = ((d % 64 / 8 + x) ^ (qr & 7)) * 16;
                                *reinterpret_cast<uint4*>(r + at16) =
                                    make_uint4(hh[4 * x], hh[4 * x + 1], hh[4 * x + 2], hh[4 * x + 3]);
                                if (Q2)
                                    *reinterpret_cast<uint4*>(r + C::SLABS * C::QSLAB + at16) =
                                        make_uint4(ll[4 * x], ll[4 * x + 1], ll[4 * x + 2], ll[4 * x + 3]);
                            }
                        }
                        fence_async_smem();
                    }
                    tc_fence_before();
                    mbar_arrive(&q_full);
                }
                if (C::QT) {
                    at += NQ;
                    named_barrier_sync(3, C::CONV);
#pragma unroll 1
                    for (int i = 0; i < NQ; ++i) copy();
                }
                const int n = seg.n;
#pragma unroll 1
                for (int jz = 0; jz < 2 * n; ++jz) {
                    const int z = jz & 1, tl = J + (jz >> 1), kb = tl % C::NBUF;
                    wait(&raw_full[at % C::NRAW], (at / C::NRAW) & 1);
                    const unsigned char* codes = raw + at % C::NRAW * RAWS + row0 * hd + ch * 16;
                    uint4 x[PER];
#pragma unroll
                    for (int i = 0; i < PER; ++i) {
                        x[i] = make_uint4(0, 0, 0, 0);
                        if (live_ch && ((i + 1) * STEP <= BN || row0 + i * STEP < BN))
                            x[i] = *reinterpret_cast<const uint4*>(codes + i * STEP * hd);
                    }
                    if (tl >= C::NBUF) wait(z ? &v_free[kb] : &k_free[kb], ((tl - C::NBUF) / C::NBUF) & 1);
                    unsigned char* tile = (z ? sv : sk) + kb * C::TILE + (ch / 4) * C::SLAB;
#pragma unroll
                    for (int i = 0; i < PER; ++i)
                        if ((i + 1) * STEP <= BN || row0 + i * STEP < BN)
                            put_codes(tile + i * STEP * 128, row0, ch % 4, (ch / 4) & 1, x[i], STEP % 8 ? i * STEP : 0);
                    fence_async_smem();
                    mbar_arrive(z ? &v_full[kb] : &k_full[kb]);
                    named_barrier_sync(3, C::CONV);                      // everybody has read the codes
                    ++at;
                    copy();
                }
                J += n, ++sn;
            } while (seg.next(plan));
        }
    } else if (any) {
        // -------------------------------------------------------- softmax
        const int w = (warp - 1) / 4, row = (warp & 3) * 32 + lane;           // this thread's half of the columns, its row
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        constexpr int HC = BN / 2;
        const int bsh = 31 - __clz(a.c.block);
        do {
            const int f = seg.m * kRows + row;
            const bool live = f < seg.rows;
            const int lim = seg.p + (live ? f : seg.rows - 1) / G;       // the last token that the row sees
            const int all_see = seg.p + seg.m * kRows / G;               // ... that every row sees
            float m = -INFINITY, l = 0.0f, lr = 0.0f;                    // lr: an integer, log2 of the reference less kWeightLog
            float acc_f = 1.0f;                  // rescaling of the moved-out accumulator since it was moved
            float4* acc = reinterpret_cast<float4*>(accs + (int64_t)blockIdx.x * C::ACC) + w * (HD / 8) * kRows + row;
            // scales of a tile's 16-token groups, loaded a tile ahead: lanes 0-15
            // K's, lanes 16-31 log2 of V's
            const float* sc = (lane < 16 ? a.c.ks : a.c.vs) + seg.slot * a.c.scale_stride +
                              (int64_t)seg.h * (a.c.cap >> bsh);
            auto scale_of = [&](int t0) {
                const int t = t0 + lane % 16 * 16;
                return lane % 16 < NG && t < seg.p + seg.rows / G ? sc[t >> bsh] : 0.0f;
            };
            float coming = scale_of(seg.j * BN);
            for (int jj = 0; jj < seg.n; ++jj) {
                const int tl = J + jj, t0 = (seg.j + jj) * BN;
                const uint32_t ts = tmem + lanes + (tl & 1) * BN + w * HC;
                // this half's groups: K's scales, log2 of V's; ready before the scores are
                const float scale = lane < 16 ? coming : log2_scale(coming);
                if (jj + 1 < seg.n) coming = scale_of(t0 + BN);
                float fk[NG / 2], fv[NG / 2];
#pragma unroll
                for (int g = 0; g < NG / 2; ++g) {
                    fk[g] = __shfl_sync(0xffffffffu, scale, w * (NG / 2) + g);
                    fv[g] = __shfl_sync(0xffffffffu, scale, 16 + w * (NG / 2) + g);
                }
                float most = fv[0];
#pragma unroll
                for (int g = 1; g < NG / 2; ++g) most = fmaxf(most, fv[g]);
                wait(&s_full[tl & 1], (tl >> 1) & 1);
                tc_fence_after();
                const float qs = s_row[sn & 1][row];
#pragma unroll
                for (int g = 0; g < NG / 2; ++g) fk[g] *= qs;            // score factors
                // the scores are read once (a TMEM load waits long while products run)
                uint32_t v[HC];
#pragma unroll
                for (int c = 0; c < HC / 32; ++c) tmem_ld32(ts + c * 32, v + c * 32);
                tmem_ld_wait();
                float z[NG / 2], x = -INFINITY;  // the groups' largest scores, and theirs
                // seen: how many of this thread's columns the row sees, where some row does not see all
                auto largest = [&](auto cut, int seen) {
#pragma unroll
                    for (int g = 0; g < HC / 16; ++g) {
                        if (cut) {
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                if (16 * g + i >= seen) v[16 * g + i] = 0xff800000u;
                        }
                        float y = __uint_as_float(v[16 * g]);
#pragma unroll
                        for (int i = 1; i < 15; i += 2)
                            y = fmaxf(fmaxf(y, __uint_as_float(v[16 * g + i])), __uint_as_float(v[16 * g + i + 1]));
                        y = fmaxf(y, __uint_as_float(v[16 * g + 15]));
                        z[g] = cut && y == -INFINITY ? y : y * fk[g];
                        x = fmaxf(x, z[g]);
                    }
                };
                auto weights = [&](auto cut, int seen) {
#pragma unroll
                    for (int g = 0; g < HC / 16; ++g) {
                        uint32_t p[16];          // hi, lo
                        // sv / 2^lr joins the exponent; the sum of the weights without it
                        const float lv = fmaxf(fv[g] - lr, -40.0f), fz = fk[g], off = lv - m;
                        const uint64_t fz2 = pack2(fz, fz), off2 = pack2(off, off);
                        uint64_t sum = 0;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const int k = 16 * g + 2 * i;
                            float z0, z1;
                            unpack2(fma2(pack2(__uint_as_float(v[k]), __uint_as_float(v[k + 1])), fz2, off2), z0, z1);
                            float w0 = ex2(z0), w1 = ex2(z1);
                            if (cut) {
                                if (k >= seen) w0 = 0.0f;
                                if (k + 1 >= seen) w1 = 0.0f;
                            }
                            const uint64_t w2 = pack2(w0, w1);
                            sum = add2(sum, w2);
                            // hi: 11 bits, lo: the rest, 21 together
                            const float h0 = __uint_as_float(__float_as_uint(w0) & 0xffffe000u);
                            const float h1 = __uint_as_float(__float_as_uint(w1) & 0xffffe000u);
                            float r0, r1;
                            unpack2(sub2(w2, pack2(h0, h1)), r0, r1);
                            p[i] = bits(__floats2half2_rn(h0, h1));
                            p[8 + i] = bits(__floats2half2_rn(r0, r1));
                        }
                        float a0, a1;
                        unpack2(sum, a0, a1);
                        l = fmaf(a0 + a1, ex2(-lv), l);
                        tmem_st16(ts + g * 16, p);
                    }
                };
                const bool cut = t0 + BN - 1 > all_see;
                const int seen = lim + 1 - t0 - w * HC;
                if (cut) largest(std::true_type{}, seen);
                else largest(std::false_type{}, 0);
                // (x - m + most is no less than what the reference goes by; all of it relative to a
                // maximum, since scores may be so large that a scale is lost in them)
                if (barrier_any(1, C::SOFT, x > m + kLazyScore || x - m + most > lr + kMostWeight)) {
                    s_half[w][row] = x;
                    named_barrier_sync(2, C::SOFT);
                    const float xm = fmaxf(fmaxf(x, s_half[w ^ 1][row]), m);
                    float top = -INFINITY;       // log2 of the largest weight times V's scale (a NaN, -inf less -inf, is passed over)
#pragma unroll
                    for (int g = 0; g < NG / 2; ++g) top = fmaxf(top, z[g] - xm + fv[g]);
                    s_top[w][row] = top;
                    named_barrier_sync(2, C::SOFT);
                    top = fmaxf(fmaxf(top, s_top[w ^ 1][row]), m - xm + lr + kWeightLog);
                    // (a row that has seen nothing yet stays as it is)
                    const float xr = xm == -INFINITY ? lr : fminf(fmaxf(ceilf(top), kLeastLog), 127.0f) - kWeightLog;
                    const float dm = xm == m ? 0.0f : m - xm, el = ex2(dm), eo = ex2(dm + (lr - xr));
                    if (jj > 0) {                // the products of the tile before are in
                        wait(&v_free[(tl - 1) % C::NBUF], ((tl - 1) / C::NBUF) & 1);
                        tc_fence_after();
                        const uint32_t to = tmem + lanes + kO + w * (HD / 2);
#pragma unroll 1
                        for (int c = 0; c < HD / 32; ++c) {
                            uint32_t v[16];
                            tmem_ld16(to + c * 16, reinterpret_cast<int*>(v));
#pragma unroll
                            for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * eo);
                            tmem_st16(to + c * 16, v);
                        }
                        tmem_st_wait();          // a tile that moves the accumulator out reads these columns below
                    }
                    l *= el, acc_f *= eo, m = xm, lr = xr;
                }
                if (cut) weights(std::true_type{}, seen);
                else weights(std::false_type{}, 0);
                if (jj % kFold<T> == 0 && jj > 0) { // the last tiles' outputs move out
                    wait(&v_free[(tl - 1) % C::NBUF], ((tl - 1) / C::NBUF) & 1);
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < HD / 2; c += HD / 4) {           // half of them in flight at a time
                        float4 y[HD / 16];
#pragma unroll
                        for (int i = 0; i < HD / 16; ++i)
                            y[i] = jj == kFold<T> ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : acc[(c / 4 + i) * kRows];
#pragma unroll
                        for (int x = 0; x < HD / 4; x += 16) {
                            int o[16];
                            tmem_ld16(tmem + lanes + kO + w * (HD / 2) + c + x, o);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                float4& z = y[x / 4 + i];
                                z.x = fmaf(z.x, acc_f, __int_as_float(o[4 * i]));
                                z.y = fmaf(z.y, acc_f, __int_as_float(o[4 * i + 1]));
                                z.z = fmaf(z.z, acc_f, __int_as_float(o[4 * i + 2]));
                                z.w = fmaf(z.w, acc_f, __int_as_float(o[4 * i + 3]));
                                acc[((c + x) / 4 + i) * kRows] = z;
                            }
                        }
                    }
                    acc_f = 1.0f;
                }
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(&p_full[tl & 1]);
            }
            // the unit's rows; what needs no outputs while the last products run
            barrier_any(1, C::SOFT, false);      // s_half is free
            s_half[w][row] = l;
            named_barrier_sync(2, C::SOFT);
            l += s_half[w ^ 1][row];
            const bool whole = seg.j == 0 && seg.n == seg.tiles;
            // parts are divided by their own sums, so that none passes the largest value
            // (a part that the row sees nothing of: 0; 1 / NaN stays)
            const float fo = exp2_int(-kWeightLog) * (l == 0.0f ? 0.0f : 1.0f / l), fr = exp2_int(lr + kWeightLog);
            const int64_t orow = (int64_t)(seg.r0 + f / G) * a.heads + seg.h * G + f % G;
            float* pt = parts + ((int64_t)blockIdx.x * 2 + (seg.j == 0)) * C::PART;
            wait(&o_full, sn & 1);
            tc_fence_after();
#pragma unroll 1
            for (int c = w * (HD / 2); c < (w + 1) * (HD / 2); c += 16) {
                int o[16];
                tmem_ld16(tmem + lanes + kO + c, o);
                float y[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) y[i] = __int_as_float(o[i]);
                if (seg.n > kFold<T>) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float4 x = acc[((c - w * (HD / 2)) / 4 + i) * kRows];
                        y[4 * i] = fmaf(x.x, acc_f, y[4 * i]), y[4 * i + 1] = fmaf(x.y, acc_f, y[4 * i + 1]);
                        y[4 * i + 2] = fmaf(x.z, acc_f, y[4 * i + 2]), y[4 * i + 3] = fmaf(x.w, acc_f, y[4 * i + 3]);
                    }
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) y[i] = y[i] * fo * fr;
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        reinterpret_cast<float4*>(pt)[(c / 4 + i) * kRows + row] =
                            make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
                } else if (live && c < hd) {
                    T* to = static_cast<T*>(a.out) + orow * hd + c;
                    if constexpr (Q2) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            reinterpret_cast<float4*>(to)[i] = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
                    } else {
                        T q[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) q[i] = kvb_t<T>(y[i]);
                        reinterpret_cast<uint4*>(to)[0] = reinterpret_cast<const uint4*>(q)[0];
                        reinterpret_cast<uint4*>(to)[1] = reinterpret_cast<const uint4*>(q)[1];
                    }
                }
            }
            if (w == 0) {
                if (!whole) pt[kRows * HD + row] = m, pt[kRows * (HD + 1) + row] = l;
                else if (stats && live) stats[orow] = make_float2(m, 1.0f / l);
            }
            tc_fence_before();                   // the next unit's first weights let the accumulator go
            J += seg.n, ++sn;
        } while (seg.next(plan));
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// Joins the units that shares cut: CTA (c, y) 16 rows of the unit whose first
// cut lies at the begin of share c (one CTA a unit took 57 us for 32 units in
// five parts each). Also the rows without tokens: zeros.
constexpr int kJoinRows = 16;
template <int HD>
__global__ void __launch_bounds__(kFinishThreads) kvb_rows_finish(const KvbAttnArgs a, const RowsPlan plan,
                                                                const float* parts, float2* stats) {
    using C = RowsCfg<HD>;
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, hd = a.c.hd, G = a.heads / a.c.heads;
    for (int b = blockIdx.x * gridDim.y + blockIdx.y; b < a.c.slots; b += gridDim.x * gridDim.y) {
        const KvbSpan s = kvb_span(a.r, b);
        const int live = live_rows(s, a.c.cap);
        if (s.p >= 0 && live < s.n && tid == 0) atomicOr(&g_kvb_rows_errors, kKvbErrCapacity);
        const int64_t e0 = (int64_t)(s.r0 + live) * a.heads * hd, e1 = (int64_t)(s.r0 + s.n) * a.heads * hd;
        for (int64_t i = e0 + tid; i < e1; i += kFinishThreads) store1(a.out, a.type, i, 0.0f);
    }
    const RowsShare w = plan.share[blockIdx.x];
    const int last = w.join;
    if (last < 0) return;                        // no unit's first cut
    const RowsUnit s = plan.unit[w.u];
    const int c0 = blockIdx.x - 1;
    const int r0 = blockIdx.y * kJoinRows;
    __shared__ float s_m[kJoinRows], s_i[kJoinRows], s_o[kJoinRows][HD + 1];   // maxima, 1 / sums
    auto at = [&](int c) { return parts + ((int64_t)c * 2 + (c == c0)) * C::PART; };
    {
        static_assert(kFinishThreads == 16 * kJoinRows, "16 threads a row");
        const int row = r0 + tid / 16;           // 16 threads share a row's parts
        float m = -INFINITY, l = 0.0f;
        for (int c = c0 + tid % 16; c <= last; c += 16) {
            const float mc = at(c)[kRows * HD + row], lc = at(c)[kRows * (HD + 1) + row], top = fmaxf(m, mc);
            l = (m == -INFINITY ? l : l * ex2(m - top)) + (mc == -INFINITY ? lc : lc * ex2(mc - top));
            m = top;
        }
        float top = m;
#pragma unroll
        for (int d = 8; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        if (m != -INFINITY) l *= ex2(m - top);
        m = top;
#pragma unroll
        for (int d = 8; d; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
        if (tid % 16 == 0) {
            s_m[tid / 16] = m, s_i[tid / 16] = 1.0f / l;
            const int f = s.m * kRows + row;
            if (stats && f < s.rows)
                stats[(int64_t)(s.r0 + f / G) * a.heads + w.h * G + f % G] = make_float2(m, 1.0f / l);
        }
    }
    __syncthreads();
    for (int i = tid; i < kJoinRows * HD / 4; i += kFinishThreads) {
        const int r = i % kJoinRows, row = r0 + r, d4 = i / kJoinRows;
        const float m = s_m[r], inv = s_i[r];
        float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int c = c0; c <= last; ++c) {
            const float mc = at(c)[kRows * HD + row], lc = at(c)[kRows * (HD + 1) + row];
            const float e = (mc == -INFINITY ? 0.0f : ex2(mc - m) * lc) * inv;
            const float4 x = reinterpret_cast<const float4*>(at(c))[d4 * kRows + row];
            y.x = fmaf(x.x, e, y.x), y.y = fmaf(x.y, e, y.y), y.z = fmaf(x.z, e, y.z), y.w = fmaf(x.w, e, y.w);
        }
        float* o = &s_o[r][4 * d4];
        o[0] = y.x, o[1] = y.y, o[2] = y.z, o[3] = y.w;
    }
    __syncthreads();
    for (int i = tid; i < kJoinRows * HD; i += kFinishThreads) {
        const int r = i / HD, d = i % HD, f = s.m * kRows + r0 + r;
        if (f < s.rows && d < hd)
            store1(a.out, a.type, ((int64_t)(s.r0 + f / G) * a.heads + w.h * G + f % G) * hd + d, s_o[r][d]);
    }
}

// mass[t] += the probabilities of token t over the rows and the query heads of
// its KV head, from the rows' maxima and sums: the scores once more, tokens as
// the 16 rows of mma m16n8k16 (the codes as halves in registers for the whole
// kernel), the prepared queries as its columns (hi and lo into one accumulator).
// A warp holds 16 TG tokens; with few token tiles the CTA's warps hold the same
// ones and share out the rows (kvb_rows_mass_few), else four warps hold four tiles
// and share the queries they read. Sums run in a fixed order: over a warp's rows,
// then over the warps. Sixteen prompts of up to 1,500 rows, 9 heads on 3 KV heads of 64:
// 328 us, issue slots 14 %, warps 10 %: bound by the CTAs of the first tokens, which
// every row sees, while the others are done.
constexpr int kMassThreads = 128;

template <int HD, bool Q2>
struct MassCfg {
    static constexpr int TG = HD == 256 ? 1 : 2;
    static constexpr int RS = RowsCfg<HD>::qrow(Q2 ? 4 : 2), CHUNK = 32 * RS;
    // kvb_rows_mass_few: rows of a step, groups of them in a warp's ring (208 KB in 16)
    static constexpr int STEP = HD == 64 ? 16 : 8, GROUP = STEP * RS;
    static constexpr int STAGES = HD == 256 ? 1 : 3;
};

__device__ __forceinline__ void mma_halves(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A warp's 16 TG tokens from t0 on: channels 32 x + 8 t + 0..7 of rows g and g + 8,
// and the 16 tokens' scale.
template <int TG, int KB>
__device__ __forceinline__ void mass_tokens(const KvbAttnArgs& a, int b, int h, int t0, int len, int g, int t,
                                            uint32_t (&k)[TG][KB][2][4], float (&sk)[TG]) {
    const int hd = a.c.hd;
#pragma unroll
    for (int j = 0; j < TG; ++j) {
        sk[j] = 0.0f;
#pragma unroll
        for (int x = 0; x < KB; ++x) {
            uint2 w[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int tok = t0 + 16 * j + 8 * r + g;
                w[r] = make_uint2(0, 0);
                if (tok < len && 32 * x + 8 * t < hd)
                    w[r] = *reinterpret_cast<const uint2*>(a.c.k + b * a.c.slot_stride +
                                                           ((int64_t)h * a.c.cap + tok) * hd + 32 * x + 8 * t);
                w[r].x ^= 0x80808080u, w[r].y ^= 0x80808080u;
            }
            k[j][x][0][0] = halves_of(w[0].x, 0x4140), k[j][x][0][1] = halves_of(w[1].x, 0x4140);
            k[j][x][0][2] = halves_of(w[0].x, 0x4342), k[j][x][0][3] = halves_of(w[1].x, 0x4342);
            k[j][x][1][0] = halves_of(w[0].y, 0x4140), k[j][x][1][1] = halves_of(w[1].y, 0x4140);
            k[j][x][1][2] = halves_of(w[0].y, 0x4342), k[j][x][1][3] = halves_of(w[1].y, 0x4342);
        }
        if (t0 + 16 * j < len)                   // 16 tokens lie in one block
            sk[j] = a.c.ks[b * a.c.scale_stride + (int64_t)h * (a.c.cap / a.c.block) + (t0 + 16 * j) / a.c.block];
    }
}

// Scores of 8 rows (qr: row g's channels from 8 t on) and the warp's tokens.
template <int HD, bool Q2>
__device__ __forceinline__ void mass_scores(const unsigned char* qr, const uint32_t (&k)[MassCfg<HD, Q2>::TG][HD / 32][2][4],
                                            float (&z)[MassCfg<HD, Q2>::TG][4]) {
    constexpr int TG = MassCfg<HD, Q2>::TG, KB = HD / 32;
#pragma unroll
    for (int j = 0; j < TG; ++j) z[j][0] = z[j][1] = z[j][2] = z[j][3] = 0.0f;
#pragma unroll
    for (int x = 0; x < KB; ++x)
#pragma unroll
        for (int y = 0; y < (Q2 ? 2 : 1); ++y) {
            const uint4 w = *reinterpret_cast<const uint4*>(qr + y * HD * 2 + x * 64);
#pragma unroll
            for (int j = 0; j < TG; ++j) {
                mma_halves(z[j], k[j][x][0], w.x, w.y);
                mma_halves(z[j], k[j][x][1], w.z, w.w);
            }
        }
}

template <int HD, bool Q2>
__global__ void __launch_bounds__(kMassThreads) kvb_rows_mass(const KvbAttnArgs a, const RowsPlan plan,
                                                            const unsigned char* queries, int units, const float2* stats) {
    using M = MassCfg<HD, Q2>;
    constexpr int TG = M::TG, RS = M::RS, KB = HD / 32, TOK = 16 * TG;   // 32-channel blocks; tokens of a warp
    extern __shared__ __align__(128) unsigned char smem[];               // [2][CHUNK]
    __shared__ __align__(8) uint64_t full[2];
    __shared__ float2 s_stat[2][32];
    const int tid = threadIdx.x, warp = tid / 32, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int h = blockIdx.y, b = blockIdx.z, G = a.heads / a.c.heads;
    if (tid == 0) {
        mbar_init(&full[0], 1), mbar_init(&full[1], 1);
        mbar_fence_init();
    }
    pdl_wait();
    pdl_trigger();
    const KvbSpan sp = kvb_span(a.r, b);
    const int n = live_rows(sp, a.c.cap), len = sp.p + n, rows = n * G;
    const int tile = blockIdx.x * TOK * 4, t0 = tile + warp * TOK;       // the CTA's, the warp's first token
    if (n == 0 || tile >= len) return;
    if (plan.first[b] + (rows + kRows - 1) / kRows > plan.head[1]) return;   // only with offsets out of order
    __syncthreads();

    uint32_t k[TG][KB][2][4];
    float sk[TG];
    mass_tokens<TG, KB>(a, b, h, t0, len, g, t, k, sk);
    // chunks of 32 rows (f = query row * G + head), from the first that sees the tile
    const unsigned char* src = queries + ((int64_t)h * units + plan.first[b]) * 4 * M::CHUNK;
    const int c0 = max(tile - sp.p, 0) * G / 32, c1 = (rows + 31) / 32;
    auto fetch = [&](int step) {                 // a chunk and its rows' maxima and sums
        const int s = step & 1, c = c0 + step;
        if (c >= c1) return;
        if (tid == 0) {
            mbar_expect_tx(&full[s], M::CHUNK);
            bulk_g2s(smem + s * M::CHUNK, src + (int64_t)c * M::CHUNK, M::CHUNK, &full[s]);
        }
        if (tid < 32) {
            const int f = c * 32 + tid;          // rows past the last weigh nothing
            s_stat[s][tid] =
                f < rows ? stats[(int64_t)(sp.r0 + f / G) * a.heads + h * G + f % G] : make_float2(0.0f, 0.0f);
        }
    };
    fetch(0);
    fetch(1);
    float sum[TG][2];
#pragma unroll
    for (int j = 0; j < TG; ++j) sum[j][0] = sum[j][1] = 0.0f;
    for (int c = c0; c < c1; ++c) {
        const int step = c - c0, s = step & 1;
        if (!mbar_wait(&full[s], (step >> 1) & 1) && lane == 0) atomicOr(&g_kvb_rows_errors, kErrWait);
        __syncthreads();                         // s_stat as well
        const unsigned char* q = smem + s * M::CHUNK;
        const bool cut = sp.p + c * 32 / G < t0 + TOK - 1;               // some row does not see every token
        float part[TG][2];
#pragma unroll
        for (int j = 0; j < TG; ++j) part[j][0] = part[j][1] = 0.0f;
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {            // 8 rows
            float z[TG][4];
            mass_scores<HD, Q2>(q + (i * 8 + g) * RS + 16 * t, k, z);
            // columns: rows c * 32 + 8 i + 2 t + e
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int col = i * 8 + 2 * t + e, f = c * 32 + col;
                const float fq = *reinterpret_cast<const float*>(q + col * RS + (RS - 16));
                const float2 st = s_stat[s][col];
                const int lim = f < rows ? sp.p + f / G : -1;
#pragma unroll
                for (int j = 0; j < TG; ++j)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        float w = ex2(fmaf(z[j][2 * r + e], sk[j] * fq, -st.x)) * st.y;
                        if ((cut || f >= rows) && t0 + 16 * j + 8 * r + g > lim) w = 0.0f;
                        part[j][r] += w;
                    }
            }
        }
#pragma unroll
        for (int j = 0; j < TG; ++j) sum[j][0] += part[j][0], sum[j][1] += part[j][1];
        __syncthreads();
        fetch(step + 2);
    }
#pragma unroll
    for (int j = 0; j < TG; ++j)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            sum[j][r] += __shfl_xor_sync(0xffffffffu, sum[j][r], 1);
            sum[j][r] += __shfl_xor_sync(0xffffffffu, sum[j][r], 2);
            const int tok = t0 + 16 * j + 8 * r + g;
            if (t == 0 && tok < len) a.mass[((int64_t)b * a.c.heads + h) * a.c.cap + tok] += sum[j][r];
        }
}

// Few token tiles: sixteen warps on the same 16 TG tokens, each taking every
// sixteenth group of STEP rows through a ring of its own, so that no barrier stands
// in the loop and four warps a scheduler cover the products' latency. 1,500 rows
// of 9 heads on 3 KV heads of 64, two sequences: 31 us (38 with 8 rows a step, 57 with
// half the warps) against 100 with four warps that met at each 32 rows. Issue slots are
// 24 % used, the tensor pipe 14 %: bound by latencies and by the second wave of CTAs.
constexpr int kFewWarps = 16;

template <int HD, bool Q2>
__global__ void __launch_bounds__(kFewWarps * 32) kvb_rows_mass_few(const KvbAttnArgs a, const RowsPlan plan,
                                                                  const unsigned char* queries, int units,
                                                                  const float2* stats) {
    using M = MassCfg<HD, Q2>;
    constexpr int TG = M::TG, RS = M::RS, KB = HD / 32, TOK = 16 * TG;
    constexpr int STEP = M::STEP, GROUP = M::GROUP, STAGES = M::STAGES;
    extern __shared__ __align__(128) unsigned char smem[];               // [kFewWarps][STAGES][GROUP]
    __shared__ __align__(8) uint64_t full[kFewWarps][STAGES];
    __shared__ float s_sum[kFewWarps][TOK];
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int h = blockIdx.x, b = blockIdx.y, G = a.heads / a.c.heads;
    if (lane == 0) {
        for (int i = 0; i < STAGES; ++i) mbar_init(&full[warp][i], 1);
        mbar_fence_init();
    }
    __syncwarp();
    pdl_wait();
    pdl_trigger();
    const KvbSpan sp = kvb_span(a.r, b);
    const int n = live_rows(sp, a.c.cap), len = sp.p + n, rows = n * G, t0 = blockIdx.z * TOK;   // the longest first
    if (n == 0 || t0 >= len) return;
    if (plan.first[b] + (rows + kRows - 1) / kRows > plan.head[1]) return;   // only with offsets out of order

    // groups of STEP rows (f = query row * G + head), from the first that sees the tile
    const unsigned char* src = queries + ((int64_t)h * units + plan.first[b]) * 4 * M::CHUNK;
    const int c0 = max(t0 - sp.p, 0) * G / STEP + warp, c1 = (rows + STEP - 1) / STEP;
    unsigned char* ring = smem + warp * STAGES * GROUP;
    auto fetch = [&](int c, int s) {
        if (lane == 0 && c < c1) {
            mbar_expect_tx(&full[warp][s], GROUP);
            bulk_g2s(ring + s * GROUP, src + (int64_t)c * GROUP, GROUP, &full[warp][s]);
        }
    };
    // lane STEP x + i: row i of the group, its maximum, 1 / sum and last visible token
    auto load_stat = [&](int c, int* lim) {
        const int f = c * STEP + (lane & (STEP - 1)), i = f / G;
        *lim = f < rows ? sp.p + i : -1;
        return f < rows ? stats[(int64_t)(sp.r0 + i) * a.heads + h * G + (f - i * G)] : make_float2(0.0f, 0.0f);
    };
#pragma unroll
    for (int i = 0; i < STAGES; ++i) fetch(c0 + i * kFewWarps, i);
    uint32_t k[TG][KB][2][4];
    float sk[TG], sum[TG][2];
    mass_tokens<TG, KB>(a, b, h, t0, len, g, t, k, sk);
#pragma unroll
    for (int j = 0; j < TG; ++j) sum[j][0] = sum[j][1] = 0.0f;
    int s = 0, phase = 0, lim_next;
    float2 st_next = load_stat(c0, &lim_next);
    for (int c = c0; c < c1; c += kFewWarps) {
        const float2 st = st_next;
        const int lim = lim_next;
        st_next = load_stat(c + kFewWarps, &lim_next);
        if (!mbar_wait(&full[warp][s], phase) && lane == 0) atomicOr(&g_kvb_rows_errors, kErrWait);
        const unsigned char* q = ring + s * GROUP;
        float z[STEP / 8][TG][4], fq[STEP / 8][2];
#pragma unroll
        for (int i = 0; i < STEP / 8; ++i) {
            mass_scores<HD, Q2>(q + (8 * i + g) * RS + 16 * t, k, z[i]);
#pragma unroll
            for (int e = 0; e < 2; ++e) fq[i][e] = *reinterpret_cast<const float*>(q + (8 * i + 2 * t + e) * RS + (RS - 16));
        }
        __syncwarp();                            // the stage is read
        fetch(c + STAGES * kFewWarps, s);
        if (++s == STAGES) s = 0, phase ^= 1;
        const bool cut = sp.p + c * STEP / G < t0 + TOK - 1 || (c + 1) * STEP > rows;    // some row does not see every token
#pragma unroll
        for (int i = 0; i < STEP / 8; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {        // column 2 t + e: row STEP c + 8 i + 2 t + e
                const int from = 8 * i + 2 * t + e;
                const float mx = __shfl_sync(0xffffffffu, st.x, from), inv = __shfl_sync(0xffffffffu, st.y, from);
                const int last = cut ? __shfl_sync(0xffffffffu, lim, from) : 0;
#pragma unroll
                for (int j = 0; j < TG; ++j)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        float w = ex2(fmaf(z[i][j][2 * r + e], sk[j] * fq[i][e], -mx)) * inv;
                        if (cut && t0 + 16 * j + 8 * r + g > last) w = 0.0f;
                        sum[j][r] += w;
                    }
            }
    }
#pragma unroll
    for (int j = 0; j < TG; ++j)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            sum[j][r] += __shfl_xor_sync(0xffffffffu, sum[j][r], 1);
            sum[j][r] += __shfl_xor_sync(0xffffffffu, sum[j][r], 2);
            if (t == 0) s_sum[warp][16 * j + 8 * r + g] = sum[j][r];
        }
    __syncthreads();
    if (threadIdx.x < TOK && t0 + threadIdx.x < len) {
        float y = 0.0f;
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) y += s_sum[w][threadIdx.x];
        a.mass[((int64_t)b * a.c.heads + h) * a.c.cap + t0 + threadIdx.x] += y;
    }
}

template <int HD, bool Q2>
cudaError_t mass_launch(const KvbAttnArgs& a, const RowsPlan& plan, const unsigned char* queries, int units,
                        const float2* stats, cudaStream_t st) {
    using M = MassCfg<HD, Q2>;
    constexpr int TOK = 16 * M::TG;
    const int64_t tiles = (a.c.cap + TOK - 1) / TOK;
    // four tiles a CTA, which reads a quarter of the queries, once that still gives
    // every SM two CTAs (by the capacity: the lengths are device data)
    const bool share = tiles / 4 * a.c.heads * a.c.slots >= 2 * kSms;
    const auto kern = share ? kvb_rows_mass<HD, Q2> : kvb_rows_mass_few<HD, Q2>;
    const size_t smem = share ? (size_t)2 * M::CHUNK : (size_t)kFewWarps * M::STAGES * M::GROUP;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    const unsigned n = (unsigned)(share ? (tiles + 3) / 4 : tiles);
    return launch_k(kern, share ? dim3(n, a.c.heads, a.c.slots) : dim3(a.c.heads, a.c.slots, n),
                    dim3(share ? kMassThreads : kFewWarps * 32), smem, st, a, plan, queries, units, stats);
}

int rows_hd(int hd) { return hd <= 64 ? 64 : hd <= 128 ? 128 : 256; }

size_t up16(size_t x) { return (x + 15) & ~(size_t)15; }

struct RowsLayout {                              // byte offsets in the scratch
    size_t share, unit, first, parts, accs, stats, queries, total;
    RowsLayout(const KvbCache& c, int heads, int rows, bool mass, int qbytes) {
        const int hd = rows_hd(c.hd);
        share = 16;
        unit = share + kSms * sizeof(RowsShare);
        first = unit + (size_t)max_units(c, heads, rows) * sizeof(RowsUnit);
        parts = up16(first + ((size_t)c.slots + 1) * sizeof(int));
        accs = parts + (size_t)kSms * 2 * kRows * (hd + 2) * sizeof(float);
        stats = accs + (size_t)kSms * kRows * hd * sizeof(float);
        queries = up16(stats + (mass ? (size_t)rows * heads * sizeof(float2) : 0));
        total = queries + (hd <= 128 || mass ? (size_t)max_units(c, heads, rows) * c.heads * kRows * (hd * qbytes + 16) : 0);
    }
};

template <int HD>
cudaError_t rows_launch(const KvbAttnArgs& a, cudaStream_t st) {
    using C = RowsCfg<HD>;
    const int qbytes = a.type == KVB_F32 ? 4 : 2, units = (int)max_units(a.c, a.heads, a.r.rows);
    const RowsLayout L(a.c, a.heads, a.r.rows, a.mass != nullptr, qbytes);
    char* s = static_cast<char*>(a.scratch);
    const RowsPlan plan{reinterpret_cast<int64_t*>(s), reinterpret_cast<RowsUnit*>(s + L.unit), reinterpret_cast<int*>(s + L.first),
                        reinterpret_cast<RowsShare*>(s + L.share)};
    float* parts = reinterpret_cast<float*>(s + L.parts);
    float2* stats = a.mass ? reinterpret_cast<float2*>(s + L.stats) : nullptr;
    unsigned char* queries = reinterpret_cast<unsigned char*>(s + L.queries);
    const bool prepared = C::QT || a.mass, fold = prepared && a.c.slots <= kFoldSlots;
    if (!fold) {
        const cudaError_t e = launch_k(kvb_rows_plan, dim3(1), dim3(kPlanThreads), 0, st, a, plan, C::BN, units);
        if (e != cudaSuccess) return e;
    }
    cudaError_t e = cudaSuccess;
    if (prepared) {
        const auto prep = a.type == KVB_F32    ? kvb_rows_queries<HD, float>
                          : a.type == KVB_BF16 ? kvb_rows_queries<HD, __nv_bfloat16>
                                               : kvb_rows_queries<HD, __half>;
        // a unit a CTA once that fills the SMs (3,000 units of 64 channels 25.7 -> 19.4 us), else a quarter
        const int per = (int64_t)units * a.c.heads >= kFullUnits ? 4 : 1;
        e = launch_k(prep, dim3(units * (4 / per) + fold, a.c.heads), dim3(HD / 8 * 32), 0, st, a, plan, queries, units,
                     fold ? C::BN : 0, per);
        if (e != cudaSuccess) return e;
    }
    const auto kern = a.type == KVB_F32    ? kvb_rows_kernel<HD, float>
                      : a.type == KVB_BF16 ? kvb_rows_kernel<HD, __nv_bfloat16>
                                           : kvb_rows_kernel<HD, __half>;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::smem(qbytes));
    if (e != cudaSuccess) return e;
    e = launch_k(kern, dim3(kSms), dim3(C::THREADS), C::smem(qbytes), st, a, plan,
                 (const unsigned char*)queries, units, parts,
                 reinterpret_cast<float*>(s + L.accs), stats);
    if (e != cudaSuccess) return e;
    e = launch_k(kvb_rows_finish<HD>, dim3(kSms, kRows / kJoinRows), dim3(kFinishThreads), 0, st, a, plan, (const float*)parts, stats);
    if (e != cudaSuccess || !stats) return e;
    return qbytes == 4 ? mass_launch<HD, true>(a, plan, queries, units, stats, st)
                       : mass_launch<HD, false>(a, plan, queries, units, stats, st);
}

}  // namespace

size_t kvb_rows_scratch(const KvbCache& c, int heads, int rows, bool mass, int qbytes) {
    return RowsLayout(c, heads, rows, mass, qbytes).total;
}

cudaError_t launch_kvb_rows(const KvbAttnArgs& a, cudaStream_t st) {
    switch (rows_hd(a.c.hd)) {
        case 64: return rows_launch<64>(a, st);
        case 128: return rows_launch<128>(a, st);
        default: return rows_launch<256>(a, st);
    }
}

}  // namespace w8a8

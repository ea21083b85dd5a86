// Attention of one row per slot over the block-scaled 8-bit KV cache (prompt
// rows: kvb_rows.cu).
//
//   o = sum_t p_t v_t,  p_t = exp(z_t - m) / sum exp(z_t - m),
//   z_t = scale * sk[t / B] * (q . k_t),  v_t = sv[t / B] * code
//
// for the tokens t <= pos of each row; a row of an idle slot gives zeros.
#include <cooperative_groups.h>

#include "kvb.cuh"

namespace w8a8 {

static __device__ unsigned int g_kvb_attn_errors;

unsigned int kvb_attn_read_clear_errors() {
    unsigned int v = 0, zero = 0;
    cudaMemcpyFromSymbol(&v, g_kvb_attn_errors, sizeof(v));
    cudaMemcpyToSymbol(g_kvb_attn_errors, &zero, sizeof(zero));
    return v;
}

namespace {

constexpr int kThreads = 128;
constexpr float kLog2e = 1.4426950408889634f;

// ---------------------------------------------------------------- one row per slot
// The cache is streamed once; everything else is small, so DRAM bounds it: 128
// sequences of 2,032 tokens, 8 KV heads of 128 (535 MB): 104 us, 5.1 TB/s, 5 us of it
// the joins; 94 MB of four ragged sequences: 27.7 us with the joins (start and end
// of the stream). For one sequence of 2,032 tokens the chain of latencies is all (8.9 us).
//
// Work: a unit is one (slot, KV head, group of GC query heads); its tokens come
// in tiles of 64 KT. All units' tiles, in order, are dealt out in equal
// contiguous shares to a fixed grid, so that lengths of any mix load every SM
// alike and the partial results do not grow with the capacity: a CTA leaves at most
// two (its first unit and its last), which kvb_step_finish joins. (Weights to gather
// do take a score for every head and place of the capacity.) Every CTA, and every
// joined row, counts the slots through by itself: for hundreds of them, not many thousands.
//
// A warp takes 16 KT tokens of a tile through its own ring of shared-memory
// stages (cp.async, no block barrier in the loop) and keeps its own maxima,
// sums and outputs. The cache is the 16-row operand of both products, the
// query heads are their 8 columns:
//   scores   mma m16n8k32 on the int8 codes as they lie (16 tokens x 32
//            channels). The query row is taken to 24-bit fixed point of its
//            largest element; its three signed 8-bit digits make three
//            products (column n: head n % GC), whose integer sums are exact.
//            (A row below 2^-64 is taken up by 2^64 for it; its factor has 2^11
//            that K's scales give, so that rows down to 1e-33 and scales down to
//            1e-34 keep all their bits.)
//   outputs  mma m16n8k16 in fp16 with fp32 sums (16 channels x 16 tokens): the
//            codes become halves exactly (byte permutes and one subtraction),
//            the weights enter as hi + lo halves (22 bits), in columns of
//            their own where GC leaves room.
// The weights are exp(z - m) sv / 2^r 2^5: m is the warp's largest score of the head,
// 2^r its largest exp(z - m) sv, an integer power of two, so that a block without weight
// leaves the others' halves their bits, however large its values are. Both move lazily:
// a warp looks when a score passes m by 2^5 or a block's V scale 2^r by 2^5, and rescales
// where a weight would pass 2^15. A warp's outputs are divided by its own sum before
// they are joined, so that none passes the largest value.
namespace cg = cooperative_groups;
constexpr int kStepWarps = 4;
constexpr int kClusterMost = 16;                 // CTAs of a cluster
constexpr int kMaxParts = 2;                     // partial units per CTA
constexpr float kLazyScore = 5.0f, kLazyScale = 1024.0f;   // 2^5, and the weights' 2^5
constexpr float kMostWeight = 32768.0f;
constexpr int kWeightLog = 5, kLeastLog = -119, kMostLog = 128;   // the references' range: 2^(5 - r) and its inverse are normal

template <int HD, int GC>
struct StepCfg {
    static constexpr int KT = HD == 64 ? 2 : 1;  // 16-token steps per warp and tile
    static constexpr int TOK = 16 * KT;          // tokens per warp and tile
    static constexpr int TILE = TOK * kStepWarps;
    static constexpr int CTAS = HD == 256 ? 2 : GC == 8 && HD == 128 ? 3 : 4;
    static constexpr int NST = HD == 256 ? 2 : 3;
    static constexpr int STAGE = 2 * TOK * HD;   // bytes: K rows, V rows
    static constexpr int RING = NST * STAGE;     // per warp
    static constexpr int NP = GC == 8 ? 2 : 1;   // column tiles of the weights
    static constexpr size_t PART = (size_t)GC * (HD + 2);   // floats of a partial unit: outputs, maximum, sum
    static constexpr size_t smem(bool cluster) { return (size_t)kStepWarps * RING + (kStepWarps + cluster) * PART * sizeof(float); }
};

// CTAs with a share: two tiles or more each where there are few (one sequence of
// 2,032 tokens, 8 KV heads of 128: 13.3 us with one tile, 11.7 us with two).
__device__ __forceinline__ int64_t step_ctas(int64_t total, int grid) { return (total + 1) / 2 < grid ? (total + 1) / 2 : grid; }

__device__ __forceinline__ int step_len(const KvbAttnArgs& a, int b) {
    const int p = a.r.pos[b];
    return p < 0 || p >= a.c.cap ? 0 : p + 1;
}

// Tiles of the slots before slot b (*before, for every thread) and of all slots.
__device__ __forceinline__ int64_t step_scan(const KvbAttnArgs& a, int tile, int b, int64_t* before) {
    __shared__ int s_sum[2][kThreads / 32];
    int all = 0, pre = 0;
    for (int i = threadIdx.x; i < a.c.slots; i += kThreads) {
        const int n = (step_len(a, i) + tile - 1) / tile;
        all += n;
        if (i < b) pre += n;
    }
    all = __reduce_add_sync(0xffffffffu, all), pre = __reduce_add_sync(0xffffffffu, pre);
    if ((threadIdx.x & 31) == 0) s_sum[0][threadIdx.x / 32] = all, s_sum[1][threadIdx.x / 32] = pre;
    __syncthreads();
    int64_t x = 0, y = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) x += s_sum[0][w], y += s_sum[1][w];
    *before = y;
    return x;
}

// 2^(5 - r) of a reference r, and back
__device__ __forceinline__ float ref_factor(int r) { return __int_as_float((127 + kWeightLog - r) << 23); }
__device__ __forceinline__ int ref_of(float factor) { return 127 + kWeightLog - (__float_as_int(factor) >> 23); }
__device__ __forceinline__ float inverse_of(float factor) { return __int_as_float((254 << 23) - __float_as_int(factor)); }
// 1 / x within 2^-23, for the sums of weights (a division is a subroutine)
__device__ __forceinline__ float rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// An integer above log2(s)
__device__ __forceinline__ float log2_above(float s) { return (float)(max(__float_as_int(s) >> 23, 1) - 126); }

// A head's maximum m and reference (as factor) moved for a tile whose 16 KT tokens' largest
// scores on this lane are x[k]: what the sums and the outputs are to be multiplied by.
template <int KT>
__device__ __forceinline__ float2 move_refs(const float (&x)[KT], const float (&fs)[KT], float& m, float& factor) {
    float xm = x[0];
    if constexpr (KT == 2) xm = fmaxf(xm, x[1]);
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) xm = fmaxf(xm, __shfl_xor_sync(0xffffffffu, xm, d));
    xm = fmaxf(xm, m);
    float top = -INFINITY;                       // (-inf less -inf, a NaN, is passed over)
#pragma unroll
    for (int k = 0; k < KT; ++k) {               // (a scale over 2^r 2^5 stays below 2^126)
        const float e = log2_above(fs[k]);
        top = fmaxf(top, fmaxf(x[k] - xm + e, e - 121.0f));
    }
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const int r = ref_of(factor);
    top = fmaxf(top, m - xm + (float)r);
    const int to = xm == -INFINITY ? r : min(max(__float2int_ru(top), kLeastLog), kMostLog);
    const float dm = xm == m ? 0.0f : m - xm;
    m = xm, factor = ref_factor(to);
    return make_float2(ex2(dm), ex2(dm + (float)(r - to)));
}

__device__ __forceinline__ void mma_s8(int* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// an 8 x 8 matrix of halves transposed across the warp
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// A tile among the units: slot b, KV head h, head group gt, tile of the slot.
struct StepIter {
    int b, h, gt, tile, tiles, len;
    int64_t head;                                // first code of (b, h)
    __device__ __forceinline__ void load(const KvbAttnArgs& a, int tile_tokens) {
        len = step_len(a, b);
        tiles = (len + tile_tokens - 1) / tile_tokens;
        head = b * a.c.slot_stride + (int64_t)h * a.c.cap * a.c.hd;
    }
    // the next unit; false past the last one
    __device__ __forceinline__ bool next_unit(const KvbAttnArgs& a, int GT, int tile_tokens) {
        tile = 0;
        if (++gt < GT) return true;
        gt = 0;
        if (++h < a.c.heads) {
            head += (int64_t)a.c.cap * a.c.hd;
            return true;
        }
        h = 0;
        do {
            if (++b >= a.c.slots) return false;
            load(a, tile_tokens);
        } while (tiles == 0);
        return true;
    }
};

// EXACT: the head fills HD channels (the copies' offsets are then constants:
// a third of the loop's address arithmetic).
// CLUSTER: few units of a small capacity (step_cluster): a unit's tiles go to the
// CTAs of one cluster in equal runs, whose results meet through distributed shared
// memory, without a look at the other slots, scratch or a second kernel. One
// sequence of 2,032 tokens, 8 KV heads: 11.7 -> 8.7 us, and 3 us less of the host.
// With weights to gather and one unit a KV head, a CTA also adds its own tokens' (24
// sequences of up to 8,191 tokens, 9 heads on 3: 23.3 -> 20.5 us).
template <int HD, int GC, bool EXACT, bool CLUSTER>
__global__ void __launch_bounds__(kThreads, StepCfg<HD, GC>::CTAS) kvb_step_kernel(const KvbAttnArgs a, float* parts,
                                                                                 float* scores) {
    using C = StepCfg<HD, GC>;
    constexpr int KT = C::KT, CH = HD / 16, MT = HD / 16;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int s_b, s_off;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32, g = lane >> 2, t = lane & 3;
    const int hd = EXACT ? HD : a.c.hd, G = a.heads / a.c.heads, GT = (G + GC - 1) / GC, units = a.c.heads * GT;
    unsigned char* ring = smem + warp * C::RING;
    float* merge = reinterpret_cast<float*>(smem + kStepWarps * C::RING);
    if (!EXACT) {                                // channels past the head stay zero
        uint4* z = reinterpret_cast<uint4*>(ring);
        for (int i = lane; i < C::RING / 16; i += 32) z[i] = make_uint4(0, 0, 0, 0);
        __syncwarp();
    }
    pdl_wait();
    pdl_trigger();

    StepIter in, it;                             // the next tile to fetch, the tile at work
    int fetch, todo;
    if constexpr (CLUSTER) {
        it.b = blockIdx.z, it.h = blockIdx.y / GT, it.gt = blockIdx.y - it.h * GT;
        it.load(a, C::TILE);
        if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0 && a.r.pos[it.b] >= a.c.cap)
            atomicOr(&g_kvb_attn_errors, kKvbErrCapacity);
        it.tile = it.tiles * (int)blockIdx.x / (int)gridDim.x;
        fetch = todo = it.tiles * ((int)blockIdx.x + 1) / (int)gridDim.x - it.tile;
    } else {
        // this CTA's share [lo, hi) of the tiles, and the slot it begins in
        int64_t none;
        const int64_t total = step_scan(a, C::TILE, 0, &none) * units;
        const int64_t ctas = step_ctas(total, gridDim.x);
        if (blockIdx.x >= ctas) return;
        const int64_t lo = div64(total * blockIdx.x, ctas), hi = div64(total * (blockIdx.x + 1), ctas);
        if (warp == 0) {
            const int per = (a.c.slots + 31) / 32, b0 = lane * per, b1 = min(b0 + per, a.c.slots);
            int64_t mine = 0;
            for (int b = b0; b < b1; ++b) mine += (step_len(a, b) + C::TILE - 1) / C::TILE;
            int64_t upto = mine;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int64_t o = __shfl_up_sync(0xffffffffu, upto, d);
                if (lane >= d) upto += o;
            }
            int64_t at = lo - (upto - mine) * units;
            if (at >= 0 && at < mine * units)
                for (int b = b0; b < b1; ++b) {
                    const int64_t n = (int64_t)((step_len(a, b) + C::TILE - 1) / C::TILE) * units;
                    if (at < n) {
                        s_b = b, s_off = (int)at;
                        break;
                    }
                    at -= n;
                }
        }
        __syncthreads();
        it.b = s_b;
        it.h = 0;
        it.load(a, C::TILE);
        {
            const int u = s_off / it.tiles;
            it.tile = s_off - u * it.tiles;
            it.h = u / GT, it.gt = u - it.h * GT;
            it.head += (int64_t)it.h * a.c.cap * hd;
        }
        fetch = todo = (int)(hi - lo);
    }
    in = it;

    // Places in a stage without bank conflicts. K (a row's 16-byte chunk ch): the
    // halves of odd rows' 128-byte lines are swapped, so that the two rows that
    // eight lanes read together lie in different banks. V: ch ^ (row & 6), for
    // eight lanes that read two neighbouring chunks of rows 0, 2, 4 and 6; with
    // 64-byte rows two rows share a line and the line's number is folded in.
    constexpr int RPI = 32 / CH;                 // rows per copy instruction of the warp
    const int crow = lane / CH, ch = lane % CH;
    const bool live_ch = EXACT || ch * 16 < hd;
    const uint32_t kdst = crow * HD + (HD == 64 ? ch : ch ^ ((crow & 1) << 2)) * 16;
    const uint32_t vdst = HD == 64 ? (crow >> 1) * 128 + ((((crow & 1) * 4 + ch) ^ ((crow >> 1 & 3) << 1)) * 16)
                                   : crow * HD + (ch ^ (crow & 6)) * 16;
    const int lane_off = crow * hd + ch * 16;
    auto issue = [&](int stage) {
        if (fetch > 0) {
            const uint32_t dst = smem_u32(ring) + stage * C::STAGE;
            const int t0 = in.tile * C::TILE + warp * C::TOK;
            const int64_t at = in.head + (int64_t)t0 * hd + lane_off;
            const int8_t *k = a.c.k + at, *v = a.c.v + at;
            if (live_ch) {
                if (t0 + C::TOK <= in.len) {
#pragma unroll
                    for (int i = 0; i < C::TOK / RPI; ++i) {
                        cp16(dst + kdst + i * RPI * HD, k + i * RPI * hd);
                        cp16(dst + C::TOK * HD + i * RPI * HD + (vdst ^ (HD == 64 ? 0 : ((i * RPI) & 6) * 16)),
                             v + i * RPI * hd);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < C::TOK / RPI; ++i) {
                        const bool ok = t0 + i * RPI + crow < in.len;
                        cp16z(dst + kdst + i * RPI * HD, ok ? k + i * RPI * hd : a.c.k, ok);
                        cp16z(dst + C::TOK * HD + i * RPI * HD + (vdst ^ (HD == 64 ? 0 : ((i * RPI) & 6) * 16)),
                              ok ? v + i * RPI * hd : a.c.v, ok);
                    }
                }
            }
            --fetch;
            if (++in.tile == in.tiles) in.next_unit(a, GT, C::TILE);
        }
        cp_commit();
    };
    const int bsh = 31 - __clz(a.c.block);
    // the fragments' places: lane (g, t) reads K chunk 4 c + t of row g, V's
    // run of channels g of rows 2t, 2t + 1, 2t + 8, 2t + 9
    const int kfrag = g * HD + (HD == 64 ? t : t ^ ((g & 1) << 2)) * 16;
    const int vfrag = HD == 64 ? t * 128 + (((g >> 1) ^ (t << 1)) * 16) + (g & 1) * 8 : 2 * t * HD + (g ^ (2 * t)) * 16;
#pragma unroll
    for (int i = 0; i < C::NST - 1; ++i) issue(i);

    int stage = 0;
    for (bool once = CLUSTER; todo > 0 || once; once = false) {
        // one unit, or what of it lies in this share
        const int b = it.b, h = it.h, j0 = it.gt * GC, first = it.tile;
        const int live = min(G - j0, GC), jg = g % GC;         // heads of the unit; the one this lane quantizes
        const int n_it = min(todo, it.tiles - first);
        const bool whole = first == 0 && n_it == it.tiles;
        const int64_t sc = b * a.c.scale_stride + (int64_t)h * (a.c.cap / a.c.block);
        const int len = it.len;

        uint32_t qd[3][HD / 64][2][2];           // digit (high first), 64 channels, k step, operand word
        float qsa, qsb;                          // score factors of this lane's columns' heads
        {
            const int64_t qr = b * a.q_stride + (int64_t)(h * G + j0 + jg) * hd;
            float mx = 0.0f;
            bool nan = false;
#pragma unroll
            for (int c = 0; c < HD / 64; ++c)
                if (jg < live && c * 64 + t * 16 < hd) {
                    float y[16];
                    load16(a.q, a.type, qr + c * 64 + t * 16, y);
#pragma unroll
                    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, fabsf(y[i])), nan |= !(fabsf(y[i]) <= 3.402823466e38f);
                }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const unsigned int bad = __ballot_sync(0xffffffffu, nan);
            const float pre = mx < 0x1p-64f ? 0x1p64f : 1.0f;
            mx *= pre;
            const float up = mx > 0.0f ? 8355711.0f / mx : 0.0f;         // 0x7F7F7F: the largest three digits
            float qs = mx * (2048.0f / 8355711.0f) * a.scale * kLog2e * (1.0f / pre);
            if (bad >> (lane & ~3) & 15u) qs = NAN;                      // a NaN or infinite row gives NaN
            qsa = __shfl_sync(0xffffffffu, qs, (2 * t) % GC * 4);
            qsb = __shfl_sync(0xffffffffu, qs, (2 * t + 1) % GC * 4);
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) {
                float y[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) y[i] = 0.0f;
                if (jg < live && c * 64 + t * 16 < hd) load16(a.q, a.type, qr + c * 64 + t * 16, y);
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float x = fminf(fmaxf(y[w * 4 + i] * pre * up, -8355711.0f), 8355711.0f);
                        v[i] = ((uint32_t)__float2int_rn(x) + 0x808080u) ^ 0x808080u;   // three signed digits
                    }
                    const uint32_t x01 = __byte_perm(v[0], v[1], 0x5140), x23 = __byte_perm(v[2], v[3], 0x5140);
                    qd[2][c][w >> 1][w & 1] = __byte_perm(x01, x23, 0x5410);
                    qd[1][c][w >> 1][w & 1] = __byte_perm(x01, x23, 0x7632);
                    qd[0][c][w >> 1][w & 1] =
                        __byte_perm(__byte_perm(v[0], v[1], 0x0062), __byte_perm(v[2], v[3], 0x0062), 0x5410);
                }
            }
        }

        // outputs: channel tile i, column tile; maxima and sums of the lane's two heads
        float o[MT][C::NP][4], ma = -INFINITY, mb = -INFINITY, la = 0.0f, lb = 0.0f;
        float ra = 1.0f, rb = 1.0f;              // the references as factors 2^(5 - r)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int x = 0; x < C::NP; ++x) o[i][x][0] = o[i][x][1] = o[i][x][2] = o[i][x][3] = 0.0f;

        const float *ksc = a.c.ks + sc, *vsc = a.c.vs + sc;
        float sk[KT], sv[KT];                    // a step's 16 tokens lie in one block; loaded a tile ahead
        auto scales = [&](int t0) {
#pragma unroll
            for (int k = 0; k < KT; ++k) {
                const bool in_len = t0 + k * 16 < len;
                sk[k] = in_len ? ksc[(t0 + k * 16) >> bsh] : 0.0f;
                sv[k] = in_len ? vsc[(t0 + k * 16) >> bsh] : 0.0f;
            }
        };
        scales(first * C::TILE + warp * C::TOK);
        for (int n = 0; n < n_it; ++n) {
            const int t0 = (first + n) * C::TILE + warp * C::TOK;
            float fk[KT], fs[KT];
#pragma unroll
            for (int k = 0; k < KT; ++k) fk[k] = sk[k] * 0x1p-11f, fs[k] = sv[k];
            if (n + 1 < n_it) scales(t0 + C::TILE);
            cp_wait<C::NST - 2>();
            __syncwarp();                        // this stage has landed, the one before it is free
            int fill = stage + C::NST - 1;
            if (fill >= C::NST) fill -= C::NST;
            issue(fill);
            if (t0 < len) {
                const unsigned char* ks = ring + stage * C::STAGE;
                const unsigned char* vs = ks + C::TOK * HD;
                float z[KT][4];                  // tokens g, g + 8 of step k: first head, second head
#pragma unroll
                for (int k = 0; k < KT; ++k) {
                    int c0[4] = {0, 0, 0, 0}, c1[4] = {0, 0, 0, 0}, c2[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int c = 0; c < HD / 64; ++c) {
                        const unsigned char* kr = ks + k * 16 * HD + (c >> 1) * 128 + (kfrag ^ ((c & 1) * 64));
                        const uint4 u = *reinterpret_cast<const uint4*>(kr);
                        const uint4 w = *reinterpret_cast<const uint4*>(kr + 8 * HD);
                        mma_s8(c0, u.x, w.x, u.y, w.y, qd[0][c][0][0], qd[0][c][0][1]);
                        mma_s8(c1, u.x, w.x, u.y, w.y, qd[1][c][0][0], qd[1][c][0][1]);
                        mma_s8(c2, u.x, w.x, u.y, w.y, qd[2][c][0][0], qd[2][c][0][1]);
                        mma_s8(c0, u.z, w.z, u.w, w.w, qd[0][c][1][0], qd[0][c][1][1]);
                        mma_s8(c1, u.z, w.z, u.w, w.w, qd[1][c][1][0], qd[1][c][1][1]);
                        mma_s8(c2, u.z, w.z, u.w, w.w, qd[2][c][1][0], qd[2][c][1][1]);
                    }
                    const float fa = fk[k] * qsa, fb = fk[k] * qsb;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        z[k][e] = fmaf((float)c0[e], 65536.0f, (float)(c1[e] * 256 + c2[e])) * (e & 1 ? fb : fa);
                }
                if (t0 + C::TOK > len) {
#pragma unroll
                    for (int k = 0; k < KT; ++k)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (t0 + k * 16 + (e >> 1) * 8 + g >= len) z[k][e] = -INFINITY;
                }
                if (scores) {
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        if (2 * t + e < live) {
                            float* zr = scores + ((int64_t)b * a.heads + h * G + j0 + 2 * t + e) * a.c.cap + t0 + g;
#pragma unroll
                            for (int k = 0; k < KT; ++k)
                                if (t0 + k * 16 < len) zr[k * 16] = z[k][e], zr[k * 16 + 8] = z[k][2 + e];
                        }
                }
                float xa = fmaxf(z[0][0], z[0][2]), xb = fmaxf(z[0][1], z[0][3]), xs = fs[0];
                if constexpr (KT == 2) {
                    xa = fmaxf(xa, fmaxf(z[1][0], z[1][2])), xb = fmaxf(xb, fmaxf(z[1][1], z[1][3]));
                    xs = fmaxf(xs, fs[1]);
                }
                const bool up = xa > ma + kLazyScore || xb > mb + kLazyScore;
                const float over = xs * fmaxf(ra, rb);
                if (__any_sync(0xffffffffu, up || over > kLazyScale)) {
                    // a large scale counts only with its weight (a first token that takes most of it, its
                    // own values tiny, would else have every tile rescaled: 128 sequences 106 -> 117 us)
                    float ya[KT], yb[KT];
                    bool move = up || over > 0x1p126f;
#pragma unroll
                    for (int k = 0; k < KT; ++k) {
                        ya[k] = fmaxf(z[k][0], z[k][2]), yb[k] = fmaxf(z[k][1], z[k][3]);
                        move |= ex2(ya[k] - ma) * (fs[k] * ra) > kMostWeight || ex2(yb[k] - mb) * (fs[k] * rb) > kMostWeight;
                    }
                    if (__any_sync(0xffffffffu, move)) {
                        const float2 ea = move_refs<KT>(ya, fs, ma, ra), eb = move_refs<KT>(yb, fs, mb, rb);
                        la *= ea.x, lb *= eb.x;
#pragma unroll
                        for (int i = 0; i < MT; ++i)
#pragma unroll
                            for (int x = 0; x < C::NP; ++x)
                                o[i][x][0] *= ea.y, o[i][x][1] *= eb.y, o[i][x][2] *= ea.y, o[i][x][3] *= eb.y;
                    }
                }
#pragma unroll
                for (int k = 0; k < KT; ++k) {
                    const float fa = fs[k] * ra, fb = fs[k] * rb;
                    uint32_t pb[C::NP][2];       // the weights as the products' columns
#pragma unroll
                    for (int j = 0; j < 2; ++j) {                        // tokens g, then g + 8
                        const float ea = ex2(z[k][2 * j] - ma), eb = ex2(z[k][2 * j + 1] - mb);
                        la += ea, lb += eb;
                        const float wa = ea * fa, wb = eb * fb;
                        const __half2 hi = __floats2half2_rn(wa, wb);
                        const float2 back = __half22float2(hi);
                        const __half2 lo = __floats2half2_rn(wa - back.x, wb - back.y);
                        if constexpr (GC == 8) {
                            pb[0][j] = transpose8(bits(hi)), pb[1][j] = transpose8(bits(lo));
                        } else {                 // columns [0, GC): hi, [GC, 2 GC): lo
                            const uint32_t x = t * 2 < GC ? bits(hi) : t * 2 < 2 * GC ? bits(lo) : 0u;
                            pb[0][j] = transpose8(x);
                        }
                    }
                    // V rows 2t, 2t + 1, 2t + 8, 2t + 9 of this step, RUN channels each
                    constexpr int RUN = HD == 64 ? 8 : 16, RUNS = HD == 256 ? 2 : 1;
#pragma unroll
                    for (int r = 0; r < RUNS; ++r) {
                        uint32_t v[4][RUN / 4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            if constexpr (HD == 64) {
                                const uint2 w = *reinterpret_cast<const uint2*>(vs + k * 1024 + (q >> 1) * 512 +
                                                                                (vfrag ^ ((q & 1) * 64)));
                                v[q][0] = w.x ^ 0x80808080u, v[q][1] = w.y ^ 0x80808080u;
                            } else {
                                const uint4 w = *reinterpret_cast<const uint4*>(
                                    vs + (k * 16 + (q & 1) + (q >> 1) * 8) * HD + r * 128 + vfrag);
                                v[q][0] = w.x ^ 0x80808080u, v[q][1] = w.y ^ 0x80808080u;
                                v[q][2] = w.z ^ 0x80808080u, v[q][3] = w.w ^ 0x80808080u;
                            }
                        }
#pragma unroll
                        for (int w = 0; w < RUN / 4; ++w) {
                            // a product's 16 rows: two channels of every lane group, tokens in pairs
                            const uint32_t a01 = __byte_perm(v[0][w], v[1][w], 0x5140);
                            const uint32_t a23 = __byte_perm(v[0][w], v[1][w], 0x7362);
                            const uint32_t b01 = __byte_perm(v[2][w], v[3][w], 0x5140);
                            const uint32_t b23 = __byte_perm(v[2][w], v[3][w], 0x7362);
                            const uint32_t x0 = halves_of(a01, 0x4140), x1 = halves_of(a01, 0x4342);
                            const uint32_t x2 = halves_of(b01, 0x4140), x3 = halves_of(b01, 0x4342);
                            const uint32_t y0 = halves_of(a23, 0x4140), y1 = halves_of(a23, 0x4342);
                            const uint32_t y2 = halves_of(b23, 0x4140), y3 = halves_of(b23, 0x4342);
#pragma unroll
                            for (int x = 0; x < C::NP; ++x) {
                                mma_f16(o[r * 8 + 2 * w][x], x0, x1, x2, x3, pb[x][0], pb[x][1]);
                                mma_f16(o[r * 8 + 2 * w + 1][x], y0, y1, y2, y3, pb[x][0], pb[x][1]);
                            }
                        }
                    }
                }
            }
            if (++stage == C::NST) stage = 0;
        }

        // the warps' states joined: merge[warp][head][HD | maximum, sum]
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
            la += __shfl_xor_sync(0xffffffffu, la, d);
            lb += __shfl_xor_sync(0xffffffffu, lb, d);
        }
        __syncthreads();                         // the last unit's readers are done
        {
            // 1 / sum (no tokens: 0; 1 / NaN stays), then 2^(r - 5)
            const float ia = la == 0.0f ? 0.0f : rcp(la), ib = lb == 0.0f ? 0.0f : rcp(lb), fa = inverse_of(ra), fb = inverse_of(rb);
            constexpr int RUN = HD == 64 ? 8 : 16;
            float* wa = merge + (warp * GC + (2 * t) % GC) * (HD + 2);
            const bool mine = 2 * t < GC;        // the columns of the lo halves are added to the hi ones'
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                float y[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (GC == 8) y[e] = o[i][0][e] + o[i][1][e];
                    else y[e] = o[i][0][e] + __shfl_down_sync(0xffffffffu, o[i][0][e], GC / 2);
                }
                float* w = wa + (i / 8) * 128 + RUN * g + 2 * (i % 8);
                if (mine) {
                    *reinterpret_cast<float2*>(w) = make_float2(y[0] * ia * fa, y[2] * ia * fa);
                    *reinterpret_cast<float2*>(w + HD + 2) = make_float2(y[1] * ib * fb, y[3] * ib * fb);
                }
            }
            if (mine && g == 0) wa[HD] = ma, wa[HD + 1] = la, wa[2 * HD + 2] = mb, wa[2 * HD + 3] = lb;
        }
        __syncthreads();
        float* pt = parts + ((int64_t)blockIdx.x * kMaxParts + (first == 0)) * C::PART;
        for (int i = tid; i < live * HD; i += kThreads) {
            const int j = i / HD, d = i - j * HD;
            const float* w = merge + j * (HD + 2);
            constexpr int WS = GC * (HD + 2);
            float mm = w[HD];
#pragma unroll
            for (int x = 1; x < kStepWarps; ++x) mm = fmaxf(mm, w[x * WS + HD]);
            float acc = 0.0f, ll = 0.0f, f[kStepWarps];
#pragma unroll
            for (int x = 0; x < kStepWarps; ++x) {
                f[x] = w[x * WS + HD] == -INFINITY ? 0.0f : ex2(w[x * WS + HD] - mm);
                f[x] *= w[x * WS + HD + 1], ll += f[x];
            }
            const float inv = ll == 0.0f ? 0.0f : rcp(ll);
#pragma unroll
            for (int x = 0; x < kStepWarps; ++x) acc = fmaf(w[x * WS + d], f[x] * inv, acc);
            const int64_t row = (int64_t)b * a.heads + h * G + j0 + j;
            if constexpr (CLUSTER) {
                float* p = merge + kStepWarps * C::PART + j * (HD + 2);
                p[d] = acc;
                if (d == 0) p[HD] = mm, p[HD + 1] = ll;
            } else if (!whole) {
                pt[j * (HD + 2) + d] = acc;
                if (d == 0) pt[j * (HD + 2) + HD] = mm, pt[j * (HD + 2) + HD + 1] = ll;
            } else {
                if (d < hd) store1(a.out, a.type, row * hd + d, acc);
                if (scores && d == 0) {
                    float* ml = scores + (int64_t)a.c.slots * a.heads * a.c.cap + 2 * row;
                    ml[0] = mm, ml[1] = ll;
                }
            }
        }
        if constexpr (CLUSTER) {
            cg::cluster_group cl = cg::this_cluster();
            cl.sync();
            const float* own = merge + kStepWarps * C::PART;
            const int n = cl.num_blocks();
            for (int i = cl.block_rank() * kThreads + tid; i < live * hd; i += n * kThreads) {
                const int j = i / hd, d = i - j * hd;
                float2 ml[kClusterMost];         // the CTAs' maxima and sums
                float mm = -INFINITY, acc = 0.0f, ll = 0.0f;
#pragma unroll
                for (int r = 0; r < kClusterMost; ++r) {
                    ml[r] = make_float2(-INFINITY, 0.0f);
                    if (r < n) ml[r] = *reinterpret_cast<const float2*>(cl.map_shared_rank(own, r) + j * (HD + 2) + HD);
                    mm = fmaxf(mm, ml[r].x);
                }
#pragma unroll
                for (int r = 0; r < kClusterMost; ++r) {
                    ml[r].y *= ml[r].x == -INFINITY ? 0.0f : ex2(ml[r].x - mm);
                    ll += ml[r].y;
                }
                const float inv = rcp(ll);
#pragma unroll
                for (int r = 0; r < kClusterMost; ++r)
                    if (r < n) acc = fmaf(cl.map_shared_rank(own, r)[j * (HD + 2) + d], ml[r].y * inv, acc);
                // a slot without tokens: zeros
                const int64_t row = (int64_t)b * a.heads + h * G + j0 + j;
                store1(a.out, a.type, row * hd + d, len > 0 ? acc : 0.0f);
                if (scores && GT > 1 && d == 0) {
                    float* ml = scores + (int64_t)a.c.slots * a.heads * a.c.cap + 2 * row;
                    ml[0] = mm, ml[1] = ll;
                }
            }
            if (scores && GT == 1) {
                // this CTA's tokens' weights, from the scores that it stored (a KV head in
                // several units: kvb_step_mass)
                float* ml = reinterpret_cast<float*>(smem);              // the ring is read: [GC] maxima, 1 / sums
                if (tid < live) {
                    float mm = -INFINITY, ll = 0.0f;
                    for (int r = 0; r < n; ++r) mm = fmaxf(mm, cl.map_shared_rank(own, r)[tid * (HD + 2) + HD]);
                    for (int r = 0; r < n; ++r) {
                        const float* p = cl.map_shared_rank(own, r) + tid * (HD + 2) + HD;
                        ll = fmaf(p[1], p[0] == -INFINITY ? 0.0f : ex2(p[0] - mm), ll);
                    }
                    ml[tid] = mm, ml[GC + tid] = 1.0f / ll;
                }
                __syncthreads();
                // four tokens at a time (of 16 in one block, so that none lies past the capacity)
                const int end = min((first + n_it) * C::TILE, len);
                for (int x = first * C::TILE + 4 * tid; x < end; x += 4 * kThreads) {
                    const float* z = scores + ((int64_t)b * a.heads + h * G) * a.c.cap + x;
                    float4* to = reinterpret_cast<float4*>(a.mass + ((int64_t)b * a.c.heads + h) * a.c.cap + x);
                    float4 w[GC], y = *to;
#pragma unroll
                    for (int j = 0; j < GC; ++j)
                        if (j < live) w[j] = *reinterpret_cast<const float4*>(z + (int64_t)j * a.c.cap);
                    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (int j = 0; j < GC; ++j)
                        if (j < live) {
                            const float mx = ml[j], inv = ml[GC + j];
                            sum.x = fmaf(ex2(w[j].x - mx), inv, sum.x), sum.y = fmaf(ex2(w[j].y - mx), inv, sum.y);
                            sum.z = fmaf(ex2(w[j].z - mx), inv, sum.z), sum.w = fmaf(ex2(w[j].w - mx), inv, sum.w);
                        }
                    y.x += sum.x;
                    if (x + 1 < end) y.y += sum.y;
                    if (x + 2 < end) y.z += sum.z;
                    if (x + 3 < end) y.w += sum.w;
                    *to = y;
                }
            }
            cl.sync();                           // the others have read this CTA's results
            break;
        }
        todo -= n_it;
        it.next_unit(a, GT, C::TILE);            // a unit that is cut ends the share
    }
    cp_wait<0>();
}

// Joins the partial units: W warps per (slot, query head), a lane per HD / 32
// channels; W = 4 where there are few rows, so that a row's many parts are read
// at once. A row that one CTA saw whole is written already; a slot without
// tokens gets zeros. With weights to gather, the joined maximum and sum go where
// the whole rows' are.
template <int HD, int GC, int W>
__global__ void __launch_bounds__(kThreads) kvb_step_finish(const KvbAttnArgs a, const float* parts, float* scores,
                                                          int grid) {
    using C = StepCfg<HD, GC>;
    constexpr int V = HD / 32;
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31, hd = a.c.hd;
    const int j = blockIdx.x * (kThreads / 32 / W) + warp / W, b = blockIdx.y;
    if (j >= a.heads) return;
    __shared__ float s_o[W > 1 ? kThreads / 32 : 1][W > 1 ? HD : 1];
    const int G = a.heads / a.c.heads, GT = (G + GC - 1) / GC, units = a.c.heads * GT;
    int all = 0, pre = 0;
    for (int i = lane; i < a.c.slots; i += 32) {
        const int n = (step_len(a, i) + C::TILE - 1) / C::TILE;
        all += n;
        if (i < b) pre += n;
    }
    const int len = step_len(a, b), tiles = (len + C::TILE - 1) / C::TILE;
    if (j == 0 && lane == 0 && a.r.pos[b] >= a.c.cap) atomicOr(&g_kvb_attn_errors, kKvbErrCapacity);
    const int64_t out = ((int64_t)b * a.heads + j) * hd;
    if (len == 0) {
        for (int d = threadIdx.x % (32 * W); d < hd; d += 32 * W) store1(a.out, a.type, out + d, 0.0f);
        return;
    }
    all = __reduce_add_sync(0xffffffffu, all), pre = __reduce_add_sync(0xffffffffu, pre);
    const int64_t total = (int64_t)all * units, ctas = step_ctas(total, grid);
    const int h = j / G, u = h * GT + (j - h * G) / GC, row = (j - h * G) % GC;
    const int64_t x0 = (int64_t)pre * units + (int64_t)u * tiles;
    const int c0 = (int)div64((x0 + 1) * ctas - 1, total), c1 = (int)div64((x0 + tiles) * ctas - 1, total);
    if (c0 == c1) return;
    // the part of CTA c: its last unit (index 1) if the unit begins there, else its first (index 0)
    const float* p0 = parts + row * (HD + 2);
    auto at = [&](int c) { return p0 + ((int64_t)c * kMaxParts + (c == c0)) * C::PART; };
    float m = -INFINITY, l = 0.0f, o[V];
    for (int c = c0 + lane; c <= c1; c += 32) {
        const float2 x = *reinterpret_cast<const float2*>(at(c) + HD);   // maximum, sum
        const float top = fmaxf(m, x.x);
        l = (m == -INFINITY ? l : l * ex2(m - top)) + x.y * ex2(x.x - top);
        m = top;
    }
    float top = m;
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (m != -INFINITY) l *= ex2(m - top);
    m = top;
#pragma unroll
    for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
    const float inv = rcp(l);
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = 0.0f;
    for (int cc = c0 + warp % W; cc <= c1; cc += 32 * W) {               // this warp: every W-th part
        const int n = min(32, (c1 - cc) / W + 1);
        float w = 0.0f;
        if (lane < n) {
            const float2 x = *reinterpret_cast<const float2*>(at(cc + lane * W) + HD);
            w = ex2(x.x - m) * x.y * inv;
        }
#pragma unroll 8
        for (int i = 0; i < n; ++i) {
            const float* p = at(cc + i * W) + lane * V;
            const float f = __shfl_sync(0xffffffffu, w, i);
#pragma unroll
            for (int v = 0; v < V; v += 2) {
                const float2 y = *reinterpret_cast<const float2*>(p + v);
                o[v] = fmaf(y.x, f, o[v]), o[v + 1] = fmaf(y.y, f, o[v + 1]);
            }
        }
    }
    if constexpr (W > 1) {
#pragma unroll
        for (int v = 0; v < V; ++v) s_o[warp][lane * V + v] = o[v];
        __syncthreads();                         // one row per CTA: every warp comes here
        for (int d = threadIdx.x; d < hd; d += kThreads) {
            float y = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) y += s_o[w][d];
            store1(a.out, a.type, out + d, y);
        }
        if (warp) return;
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (lane * V + v < hd) store1(a.out, a.type, out + lane * V + v, o[v]);
    }
    if (scores && lane == 0) {
        float* ml = scores + (int64_t)a.c.slots * a.heads * a.c.cap + 2 * ((int64_t)b * a.heads + j);
        ml[0] = m, ml[1] = l;
    }
}

// mass[t] += sum over the KV head's query heads of exp(z_t - m) / l, from the
// stored scores: one thread per token.
__global__ void __launch_bounds__(kThreads) kvb_step_mass(const KvbAttnArgs a, const float* scores) {
    pdl_wait();
    pdl_trigger();
    const int t = blockIdx.x * kThreads + threadIdx.x, h = blockIdx.y, b = blockIdx.z, G = a.heads / a.c.heads;
    if (t >= step_len(a, b)) return;
    const float* ml = scores + (int64_t)a.c.slots * a.heads * a.c.cap;
    float sum = 0.0f;
    for (int j = h * G; j < h * G + G; ++j) {
        const int64_t r = (int64_t)b * a.heads + j;
        sum += ex2(scores[r * a.c.cap + t] - ml[2 * r]) / ml[2 * r + 1];
    }
    a.mass[((int64_t)b * a.c.heads + h) * a.c.cap + t] += sum;
}

constexpr int kSms = 148;

int step_hd(int hd) { return hd <= 64 ? 64 : hd <= 128 ? 128 : 256; }
int step_gc(int G) { return G <= 2 ? 2 : G <= 4 ? 4 : 8; }

template <int HD, int GC>
size_t step_parts() {
    return (size_t)kSms * StepCfg<HD, GC>::CTAS * kMaxParts * StepCfg<HD, GC>::PART;
}

// CTAs of a unit's cluster, 0: in shares. By capacity, since the lengths are
// device data. Clusters win while every unit's fits on the device at once and no
// CTA gets a long run (a unit has at most 16 CTAs): 32 query heads on 8 KV heads
// of 128, full slots, shares / clusters of 8 / of 16 in us, caches in L2:
//   1 x 512 tokens 10.3 / 7.2 / 8.6    1 x 8,192 22 / 15.2 / 13.3   1 x 65,536 49 / 76 / 51
//   4 x 2,048      19.3 / 11.3 / 20    4 x 8,192 31 / 21.7 / 28     8 x 4,096  31 / 27 / 27
//   8 x 512        12.8 / 16.0 / 16    (the one range above that clusters lose)
template <int HD, int GC>
int step_cluster(const KvbCache& c, int heads) {
    const int64_t units = (int64_t)c.heads * ((heads / c.heads + GC - 1) / GC) * c.slots;
    const int64_t room = (int64_t)kSms * StepCfg<HD, GC>::CTAS;
    if (units * 16 <= room / 2 && c.cap >= 4096 && c.cap <= 16384) return 16;
    return units * 8 <= room && c.cap <= 8192 ? 8 : 0;
}

template <int HD, int GC>
size_t step_scratch(const KvbCache& c, int heads, bool mass) {
    return ((step_cluster<HD, GC>(c, heads) ? 0 : step_parts<HD, GC>()) + (mass ? (size_t)c.slots * heads * (c.cap + 2) : 0)) * sizeof(float);
}

template <int HD, int GC>
cudaError_t step_launch(const KvbAttnArgs& a, cudaStream_t st) {
    using C = StepCfg<HD, GC>;
    const int cluster = step_cluster<HD, GC>(a.c, a.heads);
    const bool exact = a.c.hd == HD;
    const int GT = (a.heads / a.c.heads + GC - 1) / GC, grid = kSms * C::CTAS;
    float* parts = static_cast<float*>(a.scratch);
    float* scores = a.mass ? parts + (cluster ? 0 : step_parts<HD, GC>()) : nullptr;
    const auto kern = cluster ? (exact ? kvb_step_kernel<HD, GC, true, true> : kvb_step_kernel<HD, GC, false, true>)
                              : (exact ? kvb_step_kernel<HD, GC, true, false> : kvb_step_kernel<HD, GC, false, false>);
    const size_t smem = C::smem(cluster > 0);
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    if (cluster) {
        if (cluster > 8) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(cluster, a.c.heads * GT, a.c.slots);
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = st;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = cluster;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = g_use_pdl ? 2 : 1;
        e = cudaLaunchKernelEx(&cfg, kern, a, parts, scores);
    } else {
        e = launch_k(kern, dim3(grid), dim3(kThreads), smem, st, a, parts, scores);
        if (e != cudaSuccess) return e;
        if ((int64_t)a.heads * a.c.slots <= 2 * kSms)
            e = launch_k(kvb_step_finish<HD, GC, 4>, dim3(a.heads, a.c.slots), dim3(kThreads), 0, st, a,
                         (const float*)parts, scores, grid);
        else
            e = launch_k(kvb_step_finish<HD, GC, 1>, dim3((a.heads + kThreads / 32 - 1) / (kThreads / 32), a.c.slots),
                         dim3(kThreads), 0, st, a, (const float*)parts, scores, grid);
    }
    if (e != cudaSuccess || !scores || (cluster && GT == 1)) return e;
    return launch_k(kvb_step_mass, dim3((a.c.cap + kThreads - 1) / kThreads, a.c.heads, a.c.slots), dim3(kThreads), 0, st,
                    a, (const float*)scores);
}

// f<HD, GC>() for a head size and group
#define KVB_STEP_PICK(f, hd, G, ...)                                                                          \
    (step_hd(hd) == 64    ? (step_gc(G) == 2 ? f<64, 2>(__VA_ARGS__)                                          \
                             : step_gc(G) == 4 ? f<64, 4>(__VA_ARGS__) : f<64, 8>(__VA_ARGS__))               \
     : step_hd(hd) == 128 ? (step_gc(G) == 2 ? f<128, 2>(__VA_ARGS__)                                         \
                             : step_gc(G) == 4 ? f<128, 4>(__VA_ARGS__) : f<128, 8>(__VA_ARGS__))             \
                          : (step_gc(G) == 2 ? f<256, 2>(__VA_ARGS__)                                         \
                             : step_gc(G) == 4 ? f<256, 4>(__VA_ARGS__) : f<256, 8>(__VA_ARGS__)))

}  // namespace

size_t kvb_attn_scratch(const KvbCache& c, int heads, int rows, bool one_row, bool mass, int qbytes) {
    if (one_row) return KVB_STEP_PICK(step_scratch, c.hd, heads / c.heads, c, heads, mass);
    return kvb_rows_scratch(c, heads, rows, mass, qbytes);
}

cudaError_t launch_kvb_attn(const KvbAttnArgs& a, cudaStream_t st) {
    if (a.r.start) return launch_kvb_rows(a, st);
    return KVB_STEP_PICK(step_launch, a.c.hd, a.heads / a.c.heads, a, st);
}

}  // namespace w8a8

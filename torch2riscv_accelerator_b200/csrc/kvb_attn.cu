// Attention over the block-scaled 8-bit KV cache.
//
//   o = sum_t p_t v_t,  p_t = exp(z_t - m) / sum exp(z_t - m),
//   z_t = scale * sk[t / B] * (q . k_t),  v_t = sv[t / B] * code
//
// for the tokens t <= pos of each row; a row of an idle slot gives zeros.
#include <cfloat>

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

__device__ __forceinline__ float dot16(const uint4 w, const float* q) {
    const int8_t* c = reinterpret_cast<const int8_t*>(&w);
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < 16; ++j) s = fmaf((float)c[j], q[j], s);
    return s;
}

// One CTA per (row, query head): tiles of one token per thread, the running
// maximum and sum in registers, outputs by channel.
template <typename T>
__global__ void __launch_bounds__(kThreads) kvb_attn_kernel(const KvbAttnArgs a) {
    pdl_wait();
    pdl_trigger();
    const int r = blockIdx.x, j = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid / 32;
    const int b = kvb_slot_of(a.r, a.c.slots, r);
    if (b < 0) return;
    const KvbSpan sp = kvb_span(a.r, b);
    const int hd = a.c.hd, h = j / (a.heads / a.c.heads), B = a.c.block;
    const bool idle = sp.p < 0, over = !idle && r - sp.r0 >= a.c.cap - sp.p;
    if (over && tid == 0) atomicOr(&g_kvb_attn_errors, kKvbErrCapacity);
    const int n = idle || over ? 0 : sp.p + (r - sp.r0) + 1;
    __shared__ __align__(16) float q[kKvbMaxHd];
    __shared__ float p[kThreads], red[kThreads / 32];
    const T* qr = static_cast<const T*>(a.q) + r * a.q_stride + j * hd;
    for (int d = tid; d < hd; d += kThreads) q[d] = kvb_f<T>(qr[d]) * (a.scale * kLog2e);
    __syncthreads();
    const int64_t head = b * a.c.slot_stride + (int64_t)h * a.c.cap * hd;
    const int64_t sc = b * a.c.scale_stride + (int64_t)h * (a.c.cap / B);
    float m = -INFINITY, l = 0.0f, o[kKvbMaxHd / kThreads] = {0.0f, 0.0f};
    for (int t0 = 0; t0 < n; t0 += kThreads) {
        const int t = t0 + tid;
        float z = -INFINITY;
        if (t < n) {
            const uint4* row = reinterpret_cast<const uint4*>(a.c.k + head + (int64_t)t * hd);
            z = 0.0f;
            for (int c = 0; c < hd / 16; ++c) z += dot16(row[c], q + c * 16);
            z *= a.c.ks[sc + t / B];
        }
        float mx = z;
        for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        if (lane == 0) red[warp] = mx;
        __syncthreads();
        mx = m;
        for (int w = 0; w < kThreads / 32; ++w) mx = fmaxf(mx, red[w]);
        const float fix = mx == -INFINITY ? 1.0f : exp2f(m - mx);
        const float e = t < n && mx != -INFINITY ? exp2f(z - mx) : 0.0f;
        m = mx;
        p[tid] = t < n ? e * a.c.vs[sc + t / B] : 0.0f;
        float su = e;
        for (int d = 16; d; d >>= 1) su += __shfl_xor_sync(0xffffffffu, su, d);
        __syncthreads();
        if (lane == 0) red[warp] = su;
        __syncthreads();
        l *= fix;
        for (int w = 0; w < kThreads / 32; ++w) l += red[w];
        const int cnt = min(kThreads, n - t0);
#pragma unroll
        for (int i = 0; i < kKvbMaxHd / kThreads; ++i) {
            const int d = tid + i * kThreads;
            if (d >= hd) continue;
            const int8_t* col = a.c.v + head + (int64_t)t0 * hd + d;
            float s = 0.0f;
            for (int t2 = 0; t2 < cnt; ++t2) s = fmaf(p[t2], (float)col[(int64_t)t2 * hd], s);
            o[i] = fmaf(o[i], fix, s);
        }
        __syncthreads();
    }
    T* out = static_cast<T*>(a.out) + ((int64_t)r * a.heads + j) * hd;
#pragma unroll
    for (int i = 0; i < kKvbMaxHd / kThreads; ++i)
        if (tid + i * kThreads < hd) out[tid + i * kThreads] = kvb_t<T>(l > 0.0f ? o[i] / l : 0.0f);
    if (a.mass && tid == 0) static_cast<float*>(a.scratch)[(int64_t)r * a.heads + j] = n ? m + log2f(l) : INFINITY;
}

// mass[t] += the probabilities of token t over the rows and the query heads of
// its KV head, from the rows' log2-sum-exp: one thread per token, in row order.
template <typename T>
__global__ void __launch_bounds__(kThreads) kvb_mass_kernel(const KvbAttnArgs a) {
    pdl_wait();
    pdl_trigger();
    const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, t = blockIdx.x * kThreads + tid;
    const KvbSpan sp = kvb_span(a.r, b);
    if (sp.p < 0 || sp.n == 0) return;
    const int n = min(sp.n, a.c.cap - sp.p), hd = a.c.hd, G = a.heads / a.c.heads, B = a.c.block;
    if (n <= 0 || blockIdx.x * kThreads >= sp.p + n) return;
    __shared__ __align__(16) float q[kKvbMaxHd];
    const int64_t head = b * a.c.slot_stride + (int64_t)h * a.c.cap * hd;
    const float sk = t < a.c.cap ? a.c.ks[b * a.c.scale_stride + (int64_t)h * (a.c.cap / B) + t / B] : 0.0f;
    const float* lse = static_cast<const float*>(a.scratch);
    float sum = 0.0f;
    for (int i = 0; i < n; ++i) {
        for (int g = 0; g < G; ++g) {
            const int64_t r = sp.r0 + i;
            const T* qr = static_cast<const T*>(a.q) + r * a.q_stride + (h * G + g) * hd;
            __syncthreads();
            for (int d = tid; d < hd; d += kThreads) q[d] = kvb_f<T>(qr[d]) * (a.scale * kLog2e);
            __syncthreads();
            if (t > sp.p + i) continue;
            const uint4* row = reinterpret_cast<const uint4*>(a.c.k + head + (int64_t)t * hd);
            float z = 0.0f;
            for (int c = 0; c < hd / 16; ++c) z += dot16(row[c], q + c * 16);
            sum += exp2f(z * sk - lse[r * a.heads + h * G + g]);
        }
    }
    if (t < sp.p + n) a.mass[((int64_t)b * a.c.heads + h) * a.c.cap + t] += sum;
}

// ---------------------------------------------------------------- one row per slot
// The cache is streamed once; everything else is small, so DRAM bounds it.
//
// Work: a unit is one (slot, KV head, group of 8 query heads); its tokens come
// in tiles of 64 KT. All units' tiles, in order, are dealt out in equal
// contiguous shares to a fixed grid, so that lengths of any mix load every SM
// alike and the scratch does not grow with the capacity: a CTA leaves at most
// two partial units (its first and its last), which kvb_step_finish joins.
//
// A warp takes 16 KT tokens of a tile through its own ring of shared-memory
// stages (cp.async, no block barrier in the loop) and keeps its own running
// maximum, sum and outputs:
//   scores   mma m16n8k32 on the int8 codes as they lie. The query row is taken
//            to 24-bit fixed point of its largest element, its three signed
//            8-bit digits are rows of the A operand (hi: rows 0-7, mid: 8-15 of
//            the first product, lo: rows 0-7 of a second): integer sums are exact
//            and the codes need no conversion.
//   outputs  mma m16n8k16 in fp16 with fp32 sums: the codes become fp16 exactly
//            (byte permutes), the weights 2^15 p sv / sv_max enter as hi + lo
//            halves (22 bits) in rows 0-7 and 8-15; sv_max is the warp's
//            largest V scale so far, so that weights stay in fp16's range.
constexpr int kStepWarps = 4;
constexpr int kGroup = 8;                        // query heads of a unit (rows of the products)
constexpr int kMaxParts = 2;                     // partial units per CTA

template <int HD>
struct StepCfg {
    static constexpr int KT = HD == 64 ? 2 : 1;  // 16-token steps per warp and tile
    static constexpr int TOK = 16 * KT;          // tokens per warp and tile
    static constexpr int TILE = TOK * kStepWarps;
    static constexpr int NST = HD == 256 ? 2 : 3;
    static constexpr int STAGE = 2 * TOK * HD;   // bytes: K rows, V rows
    static constexpr int RING = NST * STAGE;     // per warp
    static constexpr int CTAS = HD == 256 ? 2 : 3;
    static constexpr size_t SMEM = (size_t)kStepWarps * RING + kStepWarps * kGroup * (HD + 2) * sizeof(float);
};

// CTAs with a share: each at least one tile.
__device__ __forceinline__ int64_t step_ctas(int64_t total, int grid) { return total < grid ? total : grid; }

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

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// zeros instead of the source where it is not to be read
__device__ __forceinline__ void cp16z(uint32_t dst, const void* src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma_s8(int* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two codes (biased by 128, bytes lo and lo + 1 of x) as exact halves
__device__ __forceinline__ uint32_t halves_of(uint32_t x, uint32_t sel) {
    const uint32_t h = __byte_perm(x, 0x64646464u, sel);                // 1024 + byte
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&h), __float2half2_rn(1152.0f));
    return *reinterpret_cast<const uint32_t*>(&r);
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

__host__ __device__ __forceinline__ size_t step_part_floats(int hd_pad) { return (size_t)kGroup * (hd_pad + 2); }

template <int HD, typename T>
__global__ void __launch_bounds__(kThreads, StepCfg<HD>::CTAS) kvb_step_kernel(const KvbAttnArgs a, float* parts,
                                                                             float* scores) {
    using C = StepCfg<HD>;
    constexpr int KT = C::KT, NV = HD / 8, CH = HD / 16;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int s_b, s_off;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid / 32, g = lane >> 2, t = lane & 3;
    const int hd = a.c.hd, G = a.heads / a.c.heads, GT = (G + kGroup - 1) / kGroup, units = a.c.heads * GT;
    unsigned char* ring = smem + warp * C::RING;
    float* merge = reinterpret_cast<float*>(smem + kStepWarps * C::RING);
    if (hd < HD) {                               // channels past the head stay zero
        uint4* z = reinterpret_cast<uint4*>(ring);
        for (int i = lane; i < C::RING / 16; i += 32) z[i] = make_uint4(0, 0, 0, 0);
        __syncwarp();
    }
    pdl_wait();
    pdl_trigger();

    // this CTA's share [lo, hi) of the tiles, and the slot it begins in
    int64_t none;
    const int64_t total = step_scan(a, C::TILE, 0, &none) * units;
    const int64_t ctas = step_ctas(total, gridDim.x);
    if (blockIdx.x >= ctas) return;
    const int64_t lo = total * blockIdx.x / ctas, hi = total * (blockIdx.x + 1) / ctas;
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
    StepIter in, it;                             // the next tile to fetch, the tile at work
    it.b = s_b;
    it.h = 0;
    it.load(a, C::TILE);
    {
        const int u = s_off / it.tiles;
        it.tile = s_off - u * it.tiles;
        it.h = u / GT, it.gt = u - it.h * GT;
        it.head += (int64_t)it.h * a.c.cap * hd;
    }
    in = it;
    int fetch = (int)(hi - lo), todo = fetch;

    // Places in a stage without bank conflicts. K (a row's 16-byte chunk ch): the
    // halves of odd rows' 128-byte lines are swapped, so that the two rows that
    // eight lanes read together lie in different banks. V: ch ^ (row & 6), for
    // eight lanes that read two neighbouring chunks of rows 0, 2, 4 and 6; with
    // 64-byte rows two rows share a line and the line's number is folded in.
    constexpr int RPI = 32 / CH;                 // rows per copy instruction of the warp
    const int crow = lane / CH, ch = lane % CH;
    const bool live_ch = ch * 16 < hd;
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
    while (todo > 0) {
        // one unit, or what of it lies in this share
        const int b = it.b, h = it.h, j0 = it.gt * kGroup, first = it.tile;
        const int live = min(G - j0, kGroup), head = h * G + j0 + g;
        const int n_it = min(todo, it.tiles - first);
        const bool whole = first == 0 && n_it == it.tiles;
        const int64_t sc = b * a.c.scale_stride + (int64_t)h * (a.c.cap / a.c.block);
        const int len = it.len;

        uint32_t qh[HD / 64][2][4], ql[HD / 64][2][2];
        float qs;
        {
            const T* qr = static_cast<const T*>(a.q) + b * a.q_stride + (int64_t)head * hd;
            float mx = 0.0f;
            bool nan = false;
#pragma unroll
            for (int c = 0; c < HD / 64; ++c)
                if (g < live && c * 64 + t * 16 < hd) {
                    float y[16];
                    kvb_load8<T>(qr + c * 64 + t * 16, y);
                    kvb_load8<T>(qr + c * 64 + t * 16 + 8, y + 8);
#pragma unroll
                    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, fabsf(y[i])), nan |= isnan(y[i]);
                }
            if (nan) mx = NAN;
            const float m1 = __shfl_xor_sync(0xffffffffu, mx, 1);
            mx = isnan(mx) || isnan(m1) ? NAN : fmaxf(mx, m1);
            const float m2 = __shfl_xor_sync(0xffffffffu, mx, 2);
            mx = isnan(mx) || isnan(m2) ? NAN : fmaxf(mx, m2);
            const float up = mx > 0.0f ? 8355711.0f / mx : 0.0f;         // 0x7F7F7F: the largest three digits
            qs = mx * (1.0f / 8355711.0f) * a.scale * kLog2e;            // NaN and infinite rows give NaN
            if (isinf(mx)) qs = NAN;
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) {
                float y[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) y[i] = 0.0f;
                if (g < live && c * 64 + t * 16 < hd) {
                    kvb_load8<T>(qr + c * 64 + t * 16, y);
                    kvb_load8<T>(qr + c * 64 + t * 16 + 8, y + 8);
                }
                uint32_t d[3][4];
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float x = fminf(fmaxf(y[w * 4 + i] * up, -8355711.0f), 8355711.0f);
                        v[i] = ((uint32_t)__float2int_rn(x) + 0x808080u) ^ 0x808080u;   // three signed digits
                    }
                    const uint32_t x01 = __byte_perm(v[0], v[1], 0x5140), x23 = __byte_perm(v[2], v[3], 0x5140);
                    d[2][w] = __byte_perm(x01, x23, 0x5410);             // low digits of the four
                    d[1][w] = __byte_perm(x01, x23, 0x7632);             // middle ones
                    d[0][w] = __byte_perm(__byte_perm(v[0], v[1], 0x0062), __byte_perm(v[2], v[3], 0x0062), 0x5410);
                }
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    qh[c][s][0] = d[0][2 * s], qh[c][s][1] = d[1][2 * s];
                    qh[c][s][2] = d[0][2 * s + 1], qh[c][s][3] = d[1][2 * s + 1];
                    ql[c][s][0] = d[2][2 * s], ql[c][s][1] = d[2][2 * s + 1];
                }
            }
        }

        float o[NV][4], m = -INFINITY, l = 0.0f, svm = 0.0f, rsv = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;

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
            for (int k = 0; k < KT; ++k) fk[k] = sk[k] * qs, fs[k] = sv[k];
            if (n + 1 < n_it) scales(t0 + C::TILE);
            cp_wait<C::NST - 2>();
            __syncwarp();                        // this stage has landed, the one before it is free
            int fill = stage + C::NST - 1;
            if (fill >= C::NST) fill -= C::NST;
            issue(fill);
            if (t0 < len) {
                const unsigned char* ks = ring + stage * C::STAGE;
                const unsigned char* vs = ks + C::TOK * HD;
                float z[KT][4];                  // [k][2 j + e]: token 16 k + 8 j + 2 t + e of head g
#pragma unroll
                for (int k = 0; k < KT; ++k)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        int c1[4] = {0, 0, 0, 0}, c2[4] = {0, 0, 0, 0};
#pragma unroll
                        for (int c = 0; c < HD / 64; ++c) {
                            const uint4 w = *reinterpret_cast<const uint4*>(ks + (k * 16 + j * 8) * HD + (c >> 1) * 128 +
                                                                             (kfrag ^ ((c & 1) * 64)));
                            mma_s8(c1, qh[c][0][0], qh[c][0][1], qh[c][0][2], qh[c][0][3], w.x, w.y);
                            mma_s8(c1, qh[c][1][0], qh[c][1][1], qh[c][1][2], qh[c][1][3], w.z, w.w);
                            mma_s8(c2, ql[c][0][0], 0u, ql[c][0][1], 0u, w.x, w.y);
                            mma_s8(c2, ql[c][1][0], 0u, ql[c][1][1], 0u, w.z, w.w);
                        }
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            z[k][2 * j + e] = fmaf((float)c1[e], 65536.0f, (float)(c1[2 + e] * 256 + c2[e])) * fk[k];
                    }
                if (t0 + C::TOK > len) {
#pragma unroll
                    for (int k = 0; k < KT; ++k)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (t0 + k * 16 + (e >> 1) * 8 + 2 * t + (e & 1) >= len) z[k][e] = -INFINITY;
                }
                if (scores && g < live) {
                    float* zr = scores + ((int64_t)b * a.heads + head) * a.c.cap + t0 + 2 * t;
#pragma unroll
                    for (int k = 0; k < KT; ++k)
#pragma unroll
                        for (int j = 0; j < 2; ++j)
                            if (t0 + k * 16 < len)
                                *reinterpret_cast<float2*>(zr + k * 16 + j * 8) =
                                    make_float2(z[k][2 * j], z[k][2 * j + 1]);
                }
                float mx = m, smx = svm;
#pragma unroll
                for (int k = 0; k < KT; ++k) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx = fmaxf(mx, z[k][e]);
                    smx = fmaxf(smx, fs[k]);
                }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                if (__any_sync(0xffffffffu, mx != m || smx != svm)) {
                    const float el = ex2(m - mx), eo = smx > 0.0f ? el * (svm / smx) : 0.0f;
                    l *= el;
#pragma unroll
                    for (int i = 0; i < NV; ++i) o[i][0] *= eo, o[i][1] *= eo, o[i][2] *= eo, o[i][3] *= eo;
                    m = mx, svm = smx;
                    rsv = svm > 1e-33f ? 32768.0f / svm : 0.0f;   // values below count as 0
                }
#pragma unroll
                for (int k = 0; k < KT; ++k) {
                    const float fv = fs[k] * rsv;
                    uint32_t p[4];               // hi | lo of tokens 2t, 2t + 1, then of 8 + 2t, 8 + 2t + 1
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float e0 = ex2(z[k][2 * j] - m), e1 = ex2(z[k][2 * j + 1] - m);
                        l += e0 + e1;
                        const float w0 = e0 * fv, w1 = e1 * fv;
                        const __half2 hi2 = __floats2half2_rn(w0, w1);
                        const float2 back = __half22float2(hi2);
                        const __half2 lo2 = __floats2half2_rn(w0 - back.x, w1 - back.y);
                        p[2 * j] = *reinterpret_cast<const uint32_t*>(&hi2);
                        p[2 * j + 1] = *reinterpret_cast<const uint32_t*>(&lo2);
                    }
                    // V rows 2t, 2t + 1, 2t + 8, 2t + 9 of this step, NV channels each (HD / 128 runs of 16, or 8)
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
                            const uint32_t a01 = __byte_perm(v[0][w], v[1][w], 0x5140);
                            const uint32_t a23 = __byte_perm(v[0][w], v[1][w], 0x7362);
                            const uint32_t b01 = __byte_perm(v[2][w], v[3][w], 0x5140);
                            const uint32_t b23 = __byte_perm(v[2][w], v[3][w], 0x7362);
                            float(*oo)[4] = o + r * 16 + w * 4;
                            mma_f16(oo[0], p, halves_of(a01, 0x4140), halves_of(b01, 0x4140));
                            mma_f16(oo[1], p, halves_of(a01, 0x4342), halves_of(b01, 0x4342));
                            mma_f16(oo[2], p, halves_of(a23, 0x4140), halves_of(b23, 0x4140));
                            mma_f16(oo[3], p, halves_of(a23, 0x4342), halves_of(b23, 0x4342));
                        }
                    }
                }
            }
            if (++stage == C::NST) stage = 0;
        }

        // the warps' states joined: merge[warp][head][HD | m, l]
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        __syncthreads();                         // the last unit's readers are done
        if (g < live) {
            float* w = merge + (warp * kGroup + g) * (HD + 2);
            const float f = svm * (1.0f / 32768.0f);
            constexpr int RUN = HD == 64 ? 8 : 16;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    w[(i / RUN) * 128 + RUN * (2 * t + e) + i % RUN] = (o[i][e] + o[i][2 + e]) * f;
            if (t == 0) w[HD] = m, w[HD + 1] = l;
        }
        __syncthreads();
        float* pt = parts + ((int64_t)blockIdx.x * kMaxParts + (first == 0)) * step_part_floats(HD);
        for (int i = tid; i < live * HD; i += kThreads) {
            const int j = i / HD, d = i - j * HD;
            const float* w = merge + j * (HD + 2);
            constexpr int WS = kGroup * (HD + 2);
            float mm = w[HD];
#pragma unroll
            for (int x = 1; x < kStepWarps; ++x) mm = fmaxf(mm, w[x * WS + HD]);
            float acc = 0.0f, ll = 0.0f;
#pragma unroll
            for (int x = 0; x < kStepWarps; ++x) {
                const float f = w[x * WS + HD] == -INFINITY ? 0.0f : ex2(w[x * WS + HD] - mm);
                acc = fmaf(w[x * WS + d], f, acc), ll = fmaf(w[x * WS + HD + 1], f, ll);
            }
            if (whole) {
                if (d < hd)
                    static_cast<T*>(a.out)[((int64_t)b * a.heads + h * G + j0 + j) * hd + d] = kvb_t<T>(acc / ll);
            } else {
                pt[j * (HD + 2) + d] = acc;
            }
            if (d == 0 && (!whole || scores)) pt[j * (HD + 2) + HD] = mm, pt[j * (HD + 2) + HD + 1] = ll;
            if (whole && scores && d == 0) {
                float* ml = scores + (int64_t)a.c.slots * a.heads * a.c.cap + 2 * ((int64_t)b * a.heads + h * G + j0 + j);
                ml[0] = mm, ml[1] = ll;
            }
        }
        todo -= n_it;
        it.next_unit(a, GT, C::TILE);            // a unit that is cut ends the share
    }
    cp_wait<0>();
}

// Joins the partial units: one CTA per (query head, slot, chunk of tokens); the
// first chunk's CTA writes the output row (zeros for a slot without tokens),
// and with weights to gather every CTA of a KV head's first query head adds its
// chunk's probabilities, from the stored scores.
constexpr int kMassChunk = 1024;

template <int HD, typename T>
__global__ void __launch_bounds__(kThreads) kvb_step_finish(const KvbAttnArgs a, const float* parts,
                                                          const float* scores, int grid) {
    using C = StepCfg<HD>;
    pdl_wait();
    pdl_trigger();
    const int j = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, hd = a.c.hd;
    const int G = a.heads / a.c.heads, GT = (G + kGroup - 1) / kGroup, units = a.c.heads * GT;
    const int len = step_len(a, b);
    if (blockIdx.z == 0 && j == 0 && tid == 0 && a.r.pos[b] >= a.c.cap) atomicOr(&g_kvb_attn_errors, kKvbErrCapacity);
    T* out = static_cast<T*>(a.out) + ((int64_t)b * a.heads + j) * hd;
    if (len == 0) {
        if (blockIdx.z == 0)
            for (int d = tid; d < hd; d += kThreads) out[d] = kvb_t<T>(0.0f);
        return;
    }
    const int t0 = blockIdx.z * kMassChunk;
    if (blockIdx.z > 0 && (t0 >= len || j % G)) return;
    int64_t before;
    const int64_t total = step_scan(a, C::TILE, b, &before) * units, ctas = step_ctas(total, grid);
    const int tiles = (len + C::TILE - 1) / C::TILE;
    const int heads_here = scores && j % G == 0 ? G : 1;     // whose maxima and sums are needed
    __shared__ float s_m[kThreads], s_l[kThreads];
    __shared__ float s_mass[kMassChunk];
    if (scores && j % G == 0)
        for (int i = tid; i < kMassChunk; i += kThreads) s_mass[i] = 0.0f;
    for (int i = 0; i < heads_here; ++i) {
        const int jj = j + i, h = jj / G, u = h * GT + (jj - h * G) / kGroup, row = (jj - h * G) % kGroup;
        const int64_t x0 = before * units + (int64_t)u * tiles, x1 = x0 + tiles;
        const int c0 = (int)(((x0 + 1) * ctas - 1) / total), c1 = (int)((x1 * ctas - 1) / total);
        float m = -INFINITY, l = 0.0f;
        if (c0 == c1) {
            if (!scores) return;                 // written whole by its CTA
            const float* ml = scores + (int64_t)a.c.slots * a.heads * a.c.cap + 2 * ((int64_t)b * a.heads + jj);
            m = ml[0], l = ml[1];
        } else {
            // part of CTA c: its last unit (index 1) if the unit begins there, else its first (index 0)
            const float* p0 = parts + row * (HD + 2);
            auto at = [&](int c) { return p0 + ((int64_t)c * kMaxParts + (c == c0 ? 1 : 0)) * step_part_floats(HD); };
            float mine = -INFINITY;
            for (int c = c0 + tid; c <= c1; c += kThreads) mine = fmaxf(mine, at(c)[HD]);
            s_m[tid] = mine;
            __syncthreads();
            for (int w = 0; w < kThreads; w += 4) m = fmaxf(fmaxf(fmaxf(s_m[w], s_m[w + 1]), s_m[w + 2]), fmaxf(m, s_m[w + 3]));
            float sum = 0.0f;
            for (int c = c0 + tid; c <= c1; c += kThreads) sum = fmaf(at(c)[HD + 1], ex2(at(c)[HD] - m), sum);
            s_l[tid] = sum;
            __syncthreads();
            for (int w = 0; w < kThreads; ++w) l += s_l[w];
            if (blockIdx.z == 0 && i == 0)
                for (int d = tid; d < hd; d += kThreads) {
                    float acc = 0.0f;
                    for (int c = c0; c <= c1; ++c) acc = fmaf(at(c)[d], ex2(at(c)[HD] - m), acc);
                    out[d] = kvb_t<T>(acc / l);
                }
            __syncthreads();
        }
        if (scores && j % G == 0) {
            const float* z = scores + ((int64_t)b * a.heads + jj) * a.c.cap;
            const float r = 1.0f / l;
            for (int x = tid; x < kMassChunk && t0 + x < len; x += kThreads) s_mass[x] += ex2(z[t0 + x] - m) * r;
        }
    }
    if (scores && j % G == 0) {
        float* mass = a.mass + ((int64_t)b * a.c.heads + j / G) * a.c.cap + t0;
        for (int x = tid; x < kMassChunk && t0 + x < len; x += kThreads) mass[x] += s_mass[x];
    }
}

constexpr int kSms = 148;

int step_hd(int hd) { return hd <= 64 ? 64 : hd <= 128 ? 128 : 256; }

template <int HD, typename T>
cudaError_t step_launch(const KvbAttnArgs& a, cudaStream_t st) {
    using C = StepCfg<HD>;
    const int grid = kSms * C::CTAS;
    float* parts = static_cast<float*>(a.scratch);
    float* scores = a.mass ? parts + (size_t)grid * kMaxParts * step_part_floats(HD) : nullptr;
    cudaError_t e = cudaFuncSetAttribute(kvb_step_kernel<HD, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM);
    if (e != cudaSuccess) return e;
    e = launch_k(kvb_step_kernel<HD, T>, dim3(grid), dim3(kThreads), C::SMEM, st, a, parts, scores);
    if (e != cudaSuccess) return e;
    const int chunks = a.mass ? (a.c.cap + kMassChunk - 1) / kMassChunk : 1;
    return launch_k(kvb_step_finish<HD, T>, dim3(a.heads, a.c.slots, chunks), dim3(kThreads), 0, st, a,
                    (const float*)parts, (const float*)scores, grid);
}

template <typename T>
cudaError_t step_launch_hd(const KvbAttnArgs& a, cudaStream_t st) {
    switch (step_hd(a.c.hd)) {
        case 64: return step_launch<64, T>(a, st);
        case 128: return step_launch<128, T>(a, st);
        default: return step_launch<256, T>(a, st);
    }
}

template <typename T>
cudaError_t attn_launch(const KvbAttnArgs& a, cudaStream_t st) {
    const cudaError_t e = launch_k(kvb_attn_kernel<T>, dim3(a.r.rows, a.heads), dim3(kThreads), 0, st, a);
    if (e != cudaSuccess || !a.mass) return e;
    return launch_k(kvb_mass_kernel<T>, dim3((a.c.cap + kThreads - 1) / kThreads, a.c.heads, a.c.slots), dim3(kThreads),
                    0, st, a);
}

}  // namespace

size_t kvb_attn_scratch(const KvbCache& c, int heads, int rows, bool one_row, bool mass) {
    if (one_row) {
        const int hd = step_hd(c.hd), grid = kSms * (hd == 256 ? StepCfg<256>::CTAS : StepCfg<64>::CTAS);
        const size_t parts = (size_t)grid * kMaxParts * step_part_floats(hd);
        return (parts + (mass ? (size_t)c.slots * heads * (c.cap + 2) : 0)) * sizeof(float);
    }
    return mass ? (size_t)rows * heads * sizeof(float) : 0;
}

cudaError_t launch_kvb_attn(const KvbAttnArgs& a, cudaStream_t st) {
    if (!a.r.start)
        return a.type == KVB_F32    ? step_launch_hd<float>(a, st)
               : a.type == KVB_BF16 ? step_launch_hd<__nv_bfloat16>(a, st)
                                    : step_launch_hd<__half>(a, st);
    return a.type == KVB_F32    ? attn_launch<float>(a, st)
           : a.type == KVB_BF16 ? attn_launch<__nv_bfloat16>(a, st)
                                : attn_launch<__half>(a, st);
}

}  // namespace w8a8

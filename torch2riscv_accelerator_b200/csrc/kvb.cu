// The block-scaled 8-bit KV cache: append, read-back and eviction.
#include <cooperative_groups.h>

#include "kvb.cuh"

namespace w8a8 {

static __device__ unsigned int g_kvb_errors;

unsigned int kvb_read_clear_errors() {
    unsigned int v = 0, zero = 0;
    cudaMemcpyFromSymbol(&v, g_kvb_errors, sizeof(v));
    cudaMemcpyToSymbol(g_kvb_errors, &zero, sizeof(zero));
    return v;
}

namespace {

constexpr float kInv127 = (float)(1.0 / 127.0);

// ------------------------------------------------------------------ append
// One CTA per (touched block, KV head). A block's scale is
//   s' = max(s, max|new rows| * F(1/127))   (s = 0 for a block without older tokens)
// the new codes are rint(x / s') and, where s' grew, the older codes
// rint((q * s) / s'): each step rounded once, so that the codes do not depend
// on how the kernel is split. Values are first made finite (NaN 0, infinities
// the largest finite value), so that one bad element does not void its block.
// Bound by the chain span -> scale -> older codes -> store: one token of each of
// 128 sequences, 8 KV heads of 128, fp32: 7.1 us; prompts of up to 2,000 bf16 rows,
// 8 KV heads of 64: 15 us.
constexpr int kAppThreads = 256;                 // half of them for K, half for V

__device__ __forceinline__ int touched_blocks(const KvbSpan& s, int cap, int sh) {
    const int n = s.p < 0 ? 0 : min(s.n, cap - s.p);
    return n > 0 ? ((s.p + n - 1) >> sh) - (s.p >> sh) + 1 : 0;
}

__device__ __forceinline__ float finite_of(float x) {
    if (isnan(x)) return 0.0f;
    return fminf(fmaxf(x, -3.402823466e38f), 3.402823466e38f);
}

template <typename T>
__global__ void __launch_bounds__(kAppThreads) kvb_append_kernel(const KvbAppendArgs a) {
    pdl_wait();
    pdl_trigger();
    constexpr int H = kAppThreads / 2;
    __shared__ int s_slot, s_index;
    __shared__ unsigned int s_max[kAppThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, S = a.c.slots, B = a.c.block, sh = 31 - __clz(B);
    if (tid < 32) {                              // work item blockIdx.x: the slots' touched blocks counted through
        if (lane == 0) s_slot = -1;
        __syncwarp();
        int before = 0;
        bool over = false;
        for (int b0 = 0; b0 < S; b0 += 128) {    // four slots a lane in flight
            int n[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int b = b0 + 32 * i + lane;
                n[i] = 0;
                if (b < S) {
                    const KvbSpan s = kvb_span(a.r, b);
                    n[i] = touched_blocks(s, a.c.cap, sh);
                    over |= s.p >= 0 && s.n > 0 && s.n > a.c.cap - s.p;
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                int upto = n[i];
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int o = __shfl_up_sync(0xffffffffu, upto, d);
                    if (lane >= d) upto += o;
                }
                const int at = (int)blockIdx.x - before - (upto - n[i]);
                if (at >= 0 && at < n[i]) s_slot = b0 + 32 * i + lane, s_index = at;
                before += __shfl_sync(0xffffffffu, upto, 31);
            }
            if (before > (int)blockIdx.x && blockIdx.x + blockIdx.y > 0) break;
        }
        if (over && blockIdx.x == 0 && blockIdx.y == 0) atomicOr(&g_kvb_errors, kKvbErrCapacity);
    }
    __syncthreads();
    const int b = s_slot;
    if (b < 0) return;
    const KvbSpan sp = kvb_span(a.r, b);
    const int n = min(sp.n, a.c.cap - sp.p), hd = a.c.hd, h = blockIdx.y, ht = tid % H;
    const int blk = (sp.p >> sh) + s_index, t0 = max(blk * B, sp.p), t1 = min((blk + 1) * B, sp.p + n);
    const bool is_v = tid >= H;
    const int64_t stride = is_v ? a.v_stride : a.k_stride;
    const T* x = static_cast<const T*>(is_v ? a.v : a.k) + (int64_t)(sp.r0 + t0 - sp.p) * stride + h * hd;
    int8_t* codes = (is_v ? a.c.v : a.c.k) + b * a.c.slot_stride + (int64_t)h * a.c.cap * hd;
    float* scale = (is_v ? a.c.vs : a.c.ks) + b * a.c.scale_stride + (int64_t)h * (a.c.cap >> sh) + blk;
    const bool older = t0 > blk * B;
    const float s_old = older ? *scale : 0.0f;

    // the thread's vectors of 8: number ht, ht + H, ... of the rows' hd / 8 each
    const int nv = hd / 8, items = (t1 - t0) * nv, step_r = H / nv, step_v = H % nv;
    unsigned int m = 0;                          // max|x| as bits: non-negative floats order as integers
    int row = ht / nv, v = ht % nv;
    for (int i = ht; i < items; i += H) {
        float y[8];
        kvb_load8<T>(x + row * stride + v * 8, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(fabsf(finite_of(y[j]))));
        row += step_r, v += step_v;
        if (v >= nv) v -= nv, ++row;
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) s_max[tid / 32] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < H / 32; ++w) m = max(m, s_max[(is_v ? H / 32 : 0) + w]);
    const float s_new = fmaxf(s_old, __fmul_rn(__uint_as_float(m), kInv127));
    const float rcp = 1.0f / s_new;
    if (older && s_new != s_old) {
        const int olds = (t0 - blk * B) * (hd / 16);
        uint4* q = reinterpret_cast<uint4*>(codes + (int64_t)blk * B * hd);
        for (int i = ht; i < olds; i += H) q[i] = kvb_requant16(q[i], s_old, s_new, rcp);
    }
    row = ht / nv, v = ht % nv;
    for (int i = ht; i < items; i += H) {
        float y[8];
        kvb_load8<T>(x + row * stride + v * 8, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = finite_of(y[j]);
        uint32_t w[2] = {0u, 0u};
        if (s_new > 0.0f) kvb_codes<8>(y, s_new, rcp, w);
        *reinterpret_cast<uint2*>(codes + (int64_t)(t0 + row) * hd + v * 8) = make_uint2(w[0], w[1]);
        row += step_r, v += step_v;
        if (v >= nv) v -= nv, ++row;
    }
    __syncthreads();                             // every thread has read the old scale
    if (ht == 0) *scale = s_new;
}

// -------------------------------------------------------------------- read
// A warp per row, 4 codes a lane: one full 512-byte (16-bit: 256-byte) run of
// values per store. Bound by the values' stores: 49 million codes to fp32 in 49 us,
// 5.0 TB/s read and written.
constexpr int kReadWarps = 8;

template <typename T>
__global__ void __launch_bounds__(kReadWarps * 32) kvb_read_kernel(const KvbReadArgs a) {
    pdl_wait();
    pdl_trigger();
    const int r = blockIdx.x * kReadWarps + threadIdx.x / 32, lane = threadIdx.x & 31;
    if (r >= a.r.rows) return;
    const int b = kvb_slot_of(a.r, a.c.slots, r);
    if (b < 0) return;
    const KvbSpan sp = kvb_span(a.r, b);
    const int hd = a.c.hd, n4 = hd / 4, sh = 31 - __clz(a.c.block);
    const bool idle = sp.p < 0, over = !idle && r - sp.r0 >= a.c.cap - sp.p, none = idle || over;
    const int t = none ? 0 : sp.p + (r - sp.r0);
    if (over && lane == 0) atomicOr(&g_kvb_errors, kKvbErrCapacity);
    const int64_t head = (int64_t)a.c.cap * hd, first = b * a.c.slot_stride + (int64_t)t * hd;
    const int64_t shead = a.c.cap >> sh, sfirst = b * a.c.scale_stride + (t >> sh);
    const int64_t to = (int64_t)r * a.c.heads * hd;
    int h = lane / n4, d = lane % n4;
    const int step_h = 32 / n4, step_d = 32 % n4;
#pragma unroll 4
    for (int i = lane; i < a.c.heads * n4; i += 32) {
        const int64_t at = first + h * head + d * 4, sat = sfirst + h * shead;
        char4 q[2] = {make_char4(0, 0, 0, 0), make_char4(0, 0, 0, 0)};
        float s[2] = {0.0f, 0.0f};
        if (!none) {
            q[0] = *reinterpret_cast<const char4*>(a.c.k + at), q[1] = *reinterpret_cast<const char4*>(a.c.v + at);
            s[0] = a.c.ks[sat], s[1] = a.c.vs[sat];
        }
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            T y[4] = {kvb_t<T>(q[z].x * s[z]), kvb_t<T>(q[z].y * s[z]), kvb_t<T>(q[z].z * s[z]), kvb_t<T>(q[z].w * s[z])};
            T* p = static_cast<T*>(z ? a.v : a.k) + to + i * 4;
            if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(y);
            else *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(y);
        }
        h += step_h, d += step_d;
        if (d >= n4) d -= n4, ++h;
    }
}

// ------------------------------------------------------------------- evict
// 1. Selection, one CTA per (slot, KV head): the (keep - sink - recent)-th largest
//    weight of the middle tokens by four 8-bit radix passes over order-preserving
//    keys (in shared memory up to 32,768 of them), then the kept indices in order:
//    a token stays if its key is above the threshold, or equal to it and among the
//    first equal ones.
// 2. Compaction, 128 tokens a CTA: each block's new scale is its largest held
//    value * F(1/127). A kept token moves to a place at or before its own, so in
//    place the CTAs of a (slot, KV head) form one cluster and go in rounds: a round
//    may be stored once every CTA has read its sources (one cluster barrier).
// Sixteen sequences of up to 8,192 tokens to 3,001, 8 KV heads of 64, into another
// cache: selection 22 us (128 CTAs, bound by the passes' barriers), compaction 44 us
// for 98 MB of codes read and written (bound by the requantizing instructions: half
// of all issue slots).
namespace cg = cooperative_groups;
constexpr int kSelThreads = 1024;
constexpr int kSelKeys = 32768;                  // keys held in shared memory
constexpr int kEvThreads = 512;
constexpr int kEvUnit = 128;                     // tokens per CTA and round (a multiple of every block size)

__device__ __forceinline__ unsigned int weight_key(float w) {
    const unsigned int u = __float_as_uint(isnan(w) ? -INFINITY : w + 0.0f);   // -0 ties with +0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int evict_count(const KvbEvictArgs& a, int b) { return max(min(a.count[b], a.src.cap), 0); }

__global__ void __launch_bounds__(kSelThreads) kvb_select_kernel(const KvbEvictArgs a, int cached) {
    pdl_wait();
    pdl_trigger();
    extern __shared__ unsigned int keys[];
    __shared__ unsigned int hist[256], s_prefix, s_left;
    __shared__ int w_gt[kSelThreads / 32], w_eq[kSelThreads / 32];
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid / 32, keep = a.keep;
    const int n = evict_count(a, b), left = min(n, keep);
    if (h == 0 && tid == 0) {
        if (a.count[b] > a.src.cap) atomicOr(&g_kvb_errors, kKvbErrCapacity);
        a.count_out[b] = left;
    }
    const int64_t head = (int64_t)b * a.src.heads + h;
    const float* mass = a.mass + head * a.src.cap;
    int32_t* kept = a.kept + head * keep;
    const bool cut = n > keep;
    for (int i = tid; i < keep; i += kSelThreads)
        if (!cut) kept[i] = i < n ? i : -1;
        else if (i < a.sink) kept[i] = i;
        else if (i >= keep - a.recent) kept[i] = n - keep + i;
    const int mid = n - a.recent - a.sink, want = keep - a.sink - a.recent;
    if (!cut || want == 0) return;
    mass += a.sink;
    const bool in_smem = mid <= cached;
    if (in_smem)
        for (int t = tid; t < mid; t += kSelThreads) keys[t] = weight_key(mass[t]);
    auto key = [&](int t) { return in_smem ? keys[t] : weight_key(mass[t]); };
    const int rounds = (mid + kSelThreads - 1) / kSelThreads;
    unsigned int prefix = 0, need = want;
    for (int pass = 0; pass < 4; ++pass) {
        const int sh = 24 - 8 * pass;
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int i = 0; i < rounds; ++i) {       // equal digits of a warp count once
            const int t = i * kSelThreads + tid;
            const unsigned int k = t < mid ? key(t) : 0u;
            const bool in = t < mid && (pass == 0 || (k >> (sh + 8)) == prefix);
            const unsigned int digit = in ? (k >> sh) & 255u : 256u, same = __match_any_sync(0xffffffffu, digit);
            if (in && lane == __ffs(same) - 1) atomicAdd(&hist[digit], (unsigned int)__popc(same));
        }
        __syncthreads();
        if (warp == 0) {                         // digit 255 - 8 lane - j: from the largest down
            unsigned int c[8], sum = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) c[j] = hist[255 - 8 * lane - j], sum += c[j];
            unsigned int upto = sum;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const unsigned int o = __shfl_up_sync(0xffffffffu, upto, d);
                if (lane >= d) upto += o;
            }
            unsigned int above = upto - sum;
            if (above < need && need <= upto) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (above < need && need <= above + c[j]) {
                        s_prefix = (prefix << 8) | (255 - 8 * lane - j);
                        s_left = need - above;
                    }
                    above += c[j];
                }
            }
        }
        __syncthreads();
        prefix = s_prefix, need = s_left;
    }
    int gt0 = 0, eq0 = 0;                        // above / at the threshold so far
    for (int i = 0; i < rounds; ++i) {
        const int t = i * kSelThreads + tid;
        const unsigned int k = t < mid ? key(t) : 0u;
        const bool g = t < mid && k > prefix, e = t < mid && k == prefix;
        const unsigned int bg = __ballot_sync(0xffffffffu, g), be = __ballot_sync(0xffffffffu, e);
        if (lane == 0) w_gt[warp] = __popc(bg), w_eq[warp] = __popc(be);
        __syncthreads();
        int cg_ = w_gt[lane], ce = w_eq[lane], ug = cg_, ue = ce;        // the warps' counts, scanned
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int og = __shfl_up_sync(0xffffffffu, ug, d), oe = __shfl_up_sync(0xffffffffu, ue, d);
            if (lane >= d) ug += og, ue += oe;
        }
        const int pg = gt0 + __shfl_sync(0xffffffffu, ug - cg_, warp) + __popc(bg & ((1u << lane) - 1u));
        const int pe = eq0 + __shfl_sync(0xffffffffu, ue - ce, warp) + __popc(be & ((1u << lane) - 1u));
        gt0 += __shfl_sync(0xffffffffu, ug, 31), eq0 += __shfl_sync(0xffffffffu, ue, 31);
        if (g || (e && pe < (int)need)) kept[a.sink + pg + min(pe, (int)need)] = a.sink + t;
        __syncthreads();
    }
}

// ITEMS: 16-code chunks per thread and round, 2 (K, V) * kEvUnit * hd / 16 / kEvThreads
template <int ITEMS, bool INPLACE>
__global__ void __launch_bounds__(kEvThreads) kvb_compact_kernel(const KvbEvictArgs a) {
    pdl_wait();
    pdl_trigger();
    const int CN = gridDim.x, rank = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    __shared__ unsigned int s_amax[2][kEvUnit / 16];
    const int n = evict_count(a, b), keep = a.keep, left = min(n, keep), cap = a.src.cap;
    const bool cut = n > keep;
    if (INPLACE && !cut) return;                 // nothing moves
    const int64_t head = (int64_t)b * a.src.heads + h;
    const float* mass = a.mass + head * cap;
    float* dmass = a.dst_mass + head * a.dst.cap;
    const int32_t* kept = a.kept + head * keep;
    const int hd = a.src.hd, B = a.src.block, sh = 31 - __clz(B), nc = hd / 16;
    const int64_t s_head = b * a.src.slot_stride + (int64_t)h * cap * hd;
    const int64_t d_head = b * a.dst.slot_stride + (int64_t)h * a.dst.cap * hd;
    const int64_t ss = b * a.src.scale_stride + (int64_t)h * (cap >> sh);
    const int64_t ds = b * a.dst.scale_stride + (int64_t)h * (a.dst.cap >> sh);
    const int per = kEvUnit * nc;
    for (int base = rank * kEvUnit; base < (INPLACE ? (left + CN * kEvUnit - 1) / (CN * kEvUnit) * (CN * kEvUnit) : left);
         base += CN * kEvUnit) {
        const int have = min(max(left - base, 0), kEvUnit);
        uint4 q[ITEMS];
        float s_old[ITEMS], w = 0.0f;
        if (tid < 2 * (kEvUnit / 16)) (&s_amax[0][0])[tid] = 0u;
        __syncthreads();
        if (tid < have) w = mass[kept[base + tid]];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int item = tid + i * kEvThreads, z = item >= per, at = (item - z * per) / nc, ch = item - z * per - at * nc;
            s_old[i] = 0.0f;
            if (item < 2 * per && at < have) {
                const int t = kept[base + at];
                q[i] = *reinterpret_cast<const uint4*>((z ? a.src.v : a.src.k) + s_head + (int64_t)t * hd + ch * 16);
                s_old[i] = (z ? a.src.vs : a.src.ks)[ss + (t >> sh)];
            }
        }
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int item = tid + i * kEvThreads, z = item >= per, at = (item - z * per) / nc;
            if (item < 2 * per && at < have) {
                unsigned int m4 = __vabsdiffs4(q[i].x, 0u);
                m4 = __vmaxu4(m4, __vabsdiffs4(q[i].y, 0u));
                m4 = __vmaxu4(m4, __vabsdiffs4(q[i].z, 0u));
                m4 = __vmaxu4(m4, __vabsdiffs4(q[i].w, 0u));
                const unsigned int m = max(max(m4 & 255u, (m4 >> 8) & 255u), max((m4 >> 16) & 255u, m4 >> 24));
                atomicMax(&s_amax[z][at >> sh], __float_as_uint(__fmul_rn((float)m, s_old[i])));
            }
        }
        if (INPLACE) cg::this_cluster().sync();  // the cluster's sources of this round are in registers
        else __syncthreads();
        if (tid < have) dmass[base + tid] = w;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int item = tid + i * kEvThreads, z = item >= per, at = (item - z * per) / nc, ch = item - z * per - at * nc;
            if (item < 2 * per && at < have) {
                uint4 o = q[i];
                float s_new = s_old[i];
                if (cut) {
                    s_new = __fmul_rn(__uint_as_float(s_amax[z][at >> sh]), kInv127);
                    o = s_new > 0.0f ? kvb_requant16(o, s_old[i], s_new, 1.0f / s_new) : make_uint4(0, 0, 0, 0);
                }
                if (ch == 0 && (at & (B - 1)) == 0) (z ? a.dst.vs : a.dst.ks)[ds + ((base + at) >> sh)] = s_new;
                *reinterpret_cast<uint4*>((z ? a.dst.v : a.dst.k) + d_head + (int64_t)(base + at) * hd + ch * 16) = o;
            }
        }
        __syncthreads();                         // s_amax is free
    }
    if (INPLACE) cg::this_cluster().sync();      // every weight has been read
    const int end = min(n, a.dst.cap);
    for (int i = left + rank * kEvThreads + tid; i < end; i += CN * kEvThreads) dmass[i] = 0.0f;
}

template <int ITEMS>
cudaError_t compact_launch(const KvbEvictArgs& a, cudaStream_t st) {
    const int units = (a.keep + kEvUnit - 1) / kEvUnit;
    if (!a.in_place)
        return launch_k(kvb_compact_kernel<ITEMS, false>, dim3(units, a.src.heads, a.src.slots), dim3(kEvThreads), 0, st, a);
    int cn = 8;                                  // the portable cluster size
    while (cn > 1 && cn / 2 >= units) cn >>= 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(cn, a.src.heads, a.src.slots);
    cfg.blockDim = dim3(kEvThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cn;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = g_use_pdl ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kvb_compact_kernel<ITEMS, true>, a);
}

}  // namespace

cudaError_t launch_kvb_append(const KvbAppendArgs& a, cudaStream_t st) {
    // every touched block holds a new row, and a slot's rows touch at most
    // n / block + 2 of them
    const int64_t rows = a.r.rows, some = rows < a.c.slots ? rows : a.c.slots;
    const int64_t by_size = rows / a.c.block + 2 * some;
    const dim3 grid((unsigned)(rows < by_size ? rows : by_size), a.c.heads);
    auto kern = a.type == KVB_F32    ? kvb_append_kernel<float>
                : a.type == KVB_BF16 ? kvb_append_kernel<__nv_bfloat16>
                                     : kvb_append_kernel<__half>;
    return launch_k(kern, grid, dim3(kAppThreads), 0, st, a);
}

cudaError_t launch_kvb_read(const KvbReadArgs& a, cudaStream_t st) {
    auto kern = a.type == KVB_F32    ? kvb_read_kernel<float>
                : a.type == KVB_BF16 ? kvb_read_kernel<__nv_bfloat16>
                                     : kvb_read_kernel<__half>;
    return launch_k(kern, dim3((a.r.rows + kReadWarps - 1) / kReadWarps), dim3(kReadWarps * 32), 0, st, a);
}

cudaError_t launch_kvb_evict(const KvbEvictArgs& a, cudaStream_t st) {
    const int cached = a.src.cap < kSelKeys ? a.src.cap : kSelKeys;
    cudaError_t e = cudaSuccess;
    if (cached * 4 > 40960)                      // what a CTA may have anyway, less the static arrays
        e = cudaFuncSetAttribute(kvb_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSelKeys * 4);
    if (e != cudaSuccess) return e;
    e = launch_k(kvb_select_kernel, dim3(a.src.heads, a.src.slots), dim3(kSelThreads), (size_t)cached * 4, st, a, cached);
    if (e != cudaSuccess) return e;
    const int items = (2 * kEvUnit * (a.src.hd / 16) + kEvThreads - 1) / kEvThreads;
    if (items <= 1) return compact_launch<1>(a, st);
    if (items <= 2) return compact_launch<2>(a, st);
    if (items <= 4) return compact_launch<4>(a, st);
    return compact_launch<8>(a, st);
}

}  // namespace w8a8

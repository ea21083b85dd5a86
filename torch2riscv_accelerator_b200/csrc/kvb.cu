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
// One CTA per (touched block, KV head, K or V). A block's scale is
//   s' = max(s, max|new rows| * F(1/127))   (s = 0 for a block without older tokens)
// the new codes are rint(x / s') and, where s' grew, the older codes
// rint((q * s) / s'): each step rounded once, so that the codes do not depend
// on how the kernel is split. Values are first made finite (NaN 0, infinities
// the largest finite value), so that one bad element does not void its block.
constexpr int kAppThreads = 128;

__device__ __forceinline__ int touched_blocks(const KvbSpan& s, int cap, int block) {
    const int n = s.p < 0 ? 0 : min(s.n, cap - s.p);
    return n > 0 ? (s.p + n - 1) / block - s.p / block + 1 : 0;
}

__device__ __forceinline__ float finite_of(float x) {
    if (isnan(x)) return 0.0f;
    return fminf(fmaxf(x, -3.402823466e38f), 3.402823466e38f);
}

template <typename T>
__global__ void __launch_bounds__(kAppThreads) kvb_append_kernel(const KvbAppendArgs a) {
    pdl_wait();
    pdl_trigger();
    __shared__ int s_slot, s_index;
    __shared__ unsigned int s_max[kAppThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, S = a.c.slots, B = a.c.block;
    if (tid < 32) {                              // work item blockIdx.x: the slots' touched blocks counted through
        const int per = (S + 31) / 32, b0 = lane * per, b1 = min(b0 + per, S);
        int mine = 0;
        for (int b = b0; b < b1; ++b) mine += touched_blocks(kvb_span(a.r, b), a.c.cap, B);
        int upto = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += o;
        }
        int left = (int)blockIdx.x - (upto - mine);
        if (lane == 0) s_slot = -1;
        __syncwarp();
        if (left >= 0 && left < mine) {
            for (int b = b0; b < b1; ++b) {
                const int n = touched_blocks(kvb_span(a.r, b), a.c.cap, B);
                if (left < n) {
                    s_slot = b, s_index = left;
                    break;
                }
                left -= n;
            }
        }
        if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0) {
            bool over = false;
            for (int b = b0; b < b1; ++b) {
                const KvbSpan s = kvb_span(a.r, b);
                over |= s.p >= 0 && s.n > 0 && s.n > a.c.cap - s.p;
            }
            if (over) atomicOr(&g_kvb_errors, kKvbErrCapacity);
        }
    }
    __syncthreads();
    const int b = s_slot;
    if (b < 0) return;
    const KvbSpan sp = kvb_span(a.r, b);
    const int n = min(sp.n, a.c.cap - sp.p), hd = a.c.hd, h = blockIdx.y;
    const int blk = sp.p / B + s_index, t0 = max(blk * B, sp.p), t1 = min((blk + 1) * B, sp.p + n);
    const bool is_v = blockIdx.z != 0;
    const int64_t stride = is_v ? a.v_stride : a.k_stride;
    const T* x = static_cast<const T*>(is_v ? a.v : a.k) + (int64_t)(sp.r0 + t0 - sp.p) * stride + h * hd;
    int8_t* codes = (is_v ? a.c.v : a.c.k) + b * a.c.slot_stride + (int64_t)h * a.c.cap * hd;
    float* scale = (is_v ? a.c.vs : a.c.ks) + b * a.c.scale_stride + (int64_t)h * (a.c.cap / B) + blk;

    const int nv = hd / 8, items = (t1 - t0) * nv;
    unsigned int m = 0;                          // max|x| as bits: non-negative floats order as integers
    for (int i = tid; i < items; i += kAppThreads) {
        float y[8];
        kvb_load8<T>(x + (i / nv) * stride + (i % nv) * 8, y);
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(fabsf(finite_of(y[j]))));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if (lane == 0) s_max[tid / 32] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kAppThreads / 32; ++w) m = max(m, s_max[w]);
    const bool older = t0 > blk * B;
    const float s_old = older ? *scale : 0.0f;
    const float s_new = fmaxf(s_old, __fmul_rn(__uint_as_float(m), kInv127));
    const float rcp = 1.0f / s_new;
    if (older && s_new != s_old) {
        const int olds = (t0 - blk * B) * (hd / 16);
        uint4* q = reinterpret_cast<uint4*>(codes + (int64_t)blk * B * hd);
        for (int i = tid; i < olds; i += kAppThreads) {
            uint4 w = q[i];
            int8_t* c = reinterpret_cast<int8_t*>(&w);
#pragma unroll
            for (int j = 0; j < 16; ++j) c[j] = (int8_t)kvb_code(__fmul_rn((float)c[j], s_old), s_new, rcp);
            q[i] = w;
        }
    }
    for (int i = tid; i < items; i += kAppThreads) {
        const int row = i / nv, d = (i % nv) * 8;
        float y[8];
        kvb_load8<T>(x + row * stride + d, y);
        uint2 w;
        int8_t* c = reinterpret_cast<int8_t*>(&w);
#pragma unroll
        for (int j = 0; j < 8; ++j) c[j] = s_new > 0.0f ? (int8_t)kvb_code(finite_of(y[j]), s_new, rcp) : (int8_t)0;
        *reinterpret_cast<uint2*>(codes + (int64_t)(t0 + row) * hd + d) = w;
    }
    __syncthreads();                             // every thread has read the old scale
    if (tid == 0) *scale = s_new;
}

// -------------------------------------------------------------------- read
// One warp per row: 4 codes per lane, one full 128-byte (16-bit: 64-byte) run
// of values per store.
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
    const int hd = a.c.hd, n4 = hd / 4;
    const bool idle = sp.p < 0, over = !idle && r - sp.r0 >= a.c.cap - sp.p;
    const int t = idle || over ? 0 : sp.p + (r - sp.r0);
    if (over && lane == 0) atomicOr(&g_kvb_errors, kKvbErrCapacity);
    T* out[2] = {static_cast<T*>(a.k), static_cast<T*>(a.v)};
    for (int i = lane; i < a.c.heads * n4; i += 32) {
        const int h = i / n4, d = (i % n4) * 4;
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            char4 q = make_char4(0, 0, 0, 0);
            float s = 0.0f;
            if (!idle && !over) {
                const int8_t* codes = (z ? a.c.v : a.c.k) + b * a.c.slot_stride;
                q = *reinterpret_cast<const char4*>(codes + ((int64_t)h * a.c.cap + t) * hd + d);
                s = (z ? a.c.vs : a.c.ks)[b * a.c.scale_stride + (int64_t)h * (a.c.cap / a.c.block) + t / a.c.block];
            }
            T y[4] = {kvb_t<T>(q.x * s), kvb_t<T>(q.y * s), kvb_t<T>(q.z * s), kvb_t<T>(q.w * s)};
            T* p = out[z] + ((int64_t)r * a.c.heads + h) * hd + d;
            if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<uint4*>(y);
            else *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(y);
        }
    }
}

// ------------------------------------------------------------------- evict
// One thread-block cluster per (slot, KV head).
//  1. Selection: the (keep - sink - recent)-th largest weight of the middle
//     tokens by four 8-bit radix passes over order-preserving keys; the CTAs
//     count their segments and add the histograms up through distributed
//     shared memory (integers: the same in every order).
//  2. The kept indices in order: a token stays if its key is above the
//     threshold, or equal to it and among the first equal ones.
//  3. Compaction in rounds of one unit of tokens per CTA. A kept token moves
//     to a place at or before its own, so in place a round may be stored once
//     every CTA of the cluster has read its sources: one cluster barrier per
//     round. A block's new scale is its largest held value * F(1/127).
namespace cg = cooperative_groups;
constexpr int kEvThreads = 512;
constexpr int kEvUnit = 128;                     // tokens per CTA and round (a multiple of every block size)

__device__ __forceinline__ unsigned int weight_key(float w) {
    const unsigned int u = __float_as_uint(isnan(w) ? -INFINITY : w + 0.0f);   // -0 ties with +0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// ITEMS: 16-code chunks per thread and round, 2 (K, V) * kEvUnit * hd / 16 / kEvThreads
template <int ITEMS>
__global__ void __launch_bounds__(kEvThreads) kvb_evict_kernel(const KvbEvictArgs a) {
    pdl_wait();
    pdl_trigger();
    cg::cluster_group cl = cg::this_cluster();
    const int CN = (int)cl.num_blocks(), rank = (int)cl.block_rank();
    const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid / 32;
    __shared__ unsigned int hist[2][256];
    __shared__ unsigned int s_prefix, s_left;
    __shared__ int s_gt, s_eq;                   // this CTA's counts above / at the threshold
    __shared__ int w_gt[kEvThreads / 32], w_eq[kEvThreads / 32];
    __shared__ unsigned int s_amax[2][kEvUnit / 16];
    const int keep = a.keep, cap = a.src.cap;
    int n = a.count[b];
    if (n > cap) {
        if (tid == 0 && rank == 0 && h == 0) atomicOr(&g_kvb_errors, kKvbErrCapacity);
        n = cap;
    }
    n = max(n, 0);
    const int64_t head = (int64_t)b * a.src.heads + h;
    const float* mass = a.mass + head * cap;
    float* dmass = a.dst_mass + head * a.dst.cap;
    int32_t* kept = a.kept + head * keep;
    const bool cut = n > keep;
    const int left = min(n, keep);
    if (rank == 0 && h == 0 && tid == 0) a.count_out[b] = left;
    for (int i = rank * kEvThreads + tid; i < keep; i += CN * kEvThreads)
        if (!cut) kept[i] = i < n ? i : -1;
        else if (i < a.sink) kept[i] = i;
        else if (i >= keep - a.recent) kept[i] = n - keep + i;
    if (cut) {
        const int mid = n - a.recent - a.sink, want = keep - a.sink - a.recent;
        const int seg = (mid + CN - 1) / CN, lo = a.sink + min(rank * seg, mid), hi = a.sink + min((rank + 1) * seg, mid);
        unsigned int prefix = 0, need = want;
        if (want > 0) {
            for (int pass = 0; pass < 4; ++pass) {
                const int sh = 24 - 8 * pass;
                unsigned int* hg = hist[pass & 1];
                if (tid < 256) hg[tid] = 0;
                __syncthreads();
                for (int t = lo + tid; t < hi; t += kEvThreads) {
                    const unsigned int k = weight_key(mass[t]);
                    if (pass == 0 || (k >> (sh + 8)) == prefix) atomicAdd(&hg[(k >> sh) & 255u], 1u);
                }
                cl.sync();
                if (warp == 0) {                 // digit 255 - 8 lane - j: from the largest down
                    unsigned int c[8], sum = 0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) c[j] = 0;
                    for (int r = 0; r < CN; ++r) {
                        const unsigned int* o = cl.map_shared_rank(hg, r);
#pragma unroll
                        for (int j = 0; j < 8; ++j) c[j] += o[255 - 8 * lane - j];
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) sum += c[j];
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
                // the buffer of pass + 1 was last read remotely before this pass's barrier
            }
        }
        // counts of this segment, then its place among the cluster's
        int gt = 0, eq = 0;
        if (want > 0)
            for (int t = lo + tid; t < hi; t += kEvThreads) {
                const unsigned int k = weight_key(mass[t]);
                gt += k > prefix, eq += k == prefix;
            }
        gt = __reduce_add_sync(0xffffffffu, gt), eq = __reduce_add_sync(0xffffffffu, eq);
        if (lane == 0) w_gt[warp] = gt, w_eq[warp] = eq;
        __syncthreads();
        if (tid == 0) {
            int g = 0, e = 0;
            for (int w = 0; w < kEvThreads / 32; ++w) g += w_gt[w], e += w_eq[w];
            s_gt = g, s_eq = e;
        }
        cl.sync();
        int gt0 = 0, eq0 = 0;
        for (int r = 0; r < rank; ++r) gt0 += *cl.map_shared_rank(&s_gt, r), eq0 += *cl.map_shared_rank(&s_eq, r);
        if (want > 0)
            for (int c0 = lo; c0 < hi; c0 += kEvThreads) {
                const int t = c0 + tid;
                const unsigned int k = t < hi ? weight_key(mass[t]) : 0u;
                const bool g = t < hi && k > prefix, e = t < hi && k == prefix;
                const unsigned int bg = __ballot_sync(0xffffffffu, g), be = __ballot_sync(0xffffffffu, e);
                __syncthreads();
                if (lane == 0) w_gt[warp] = __popc(bg), w_eq[warp] = __popc(be);
                __syncthreads();
                int pg = gt0, pe = eq0;
                for (int w = 0; w < kEvThreads / 32; ++w) {
                    if (w < warp) pg += w_gt[w], pe += w_eq[w];
                    gt0 += w_gt[w], eq0 += w_eq[w];
                }
                pg += __popc(bg & ((1u << lane) - 1u)), pe += __popc(be & ((1u << lane) - 1u));
                if (g || (e && pe < (int)need)) kept[a.sink + pg + min(pe, (int)need)] = t;
            }
    }
    cl.sync();                                   // the kept indices are written (and no histogram is read any more)

    // compaction; nothing to do in place for a slot within its budget
    if (!cut && a.in_place) return;
    const int hd = a.src.hd, B = a.src.block, nc = hd / 16, NBs = cap / B, NBd = a.dst.cap / B;
    const int64_t s_head = b * a.src.slot_stride + (int64_t)h * cap * hd;
    const int64_t d_head = b * a.dst.slot_stride + (int64_t)h * a.dst.cap * hd;
    const int8_t* src[2] = {a.src.k + s_head, a.src.v + s_head};
    int8_t* dst[2] = {a.dst.k + d_head, a.dst.v + d_head};
    const int64_t ss = b * a.src.scale_stride + (int64_t)h * NBs, ds = b * a.dst.scale_stride + (int64_t)h * NBd;
    const float* sscale[2] = {a.src.ks + ss, a.src.vs + ss};
    float* dscale[2] = {a.dst.ks + ds, a.dst.vs + ds};
    const int rounds = (left + CN * kEvUnit - 1) / (CN * kEvUnit), per = kEvUnit * nc;
    for (int round = 0; round < rounds; ++round) {
        const int base = (round * CN + rank) * kEvUnit, have = min(max(left - base, 0), kEvUnit);
        uint4 q[ITEMS];
        float s_old[ITEMS], w = 0.0f;
        if (tid < 2 * (kEvUnit / 16)) (&s_amax[0][0])[tid] = 0u;
        __syncthreads();
        if (tid < have) w = mass[__ldcg(kept + base + tid)];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int item = tid + i * kEvThreads, z = item >= per, at = (item - z * per) / nc, ch = item - z * per - at * nc;
            s_old[i] = 0.0f;
            if (item < 2 * per && at < have) {
                const int t = __ldcg(kept + base + at);
                q[i] = *reinterpret_cast<const uint4*>(src[z] + (int64_t)t * hd + ch * 16);
                s_old[i] = sscale[z][t / B];
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
                atomicMax(&s_amax[z][at / B], __float_as_uint(__fmul_rn((float)m, s_old[i])));
            }
        }
        if (a.in_place) cl.sync();               // the cluster's sources of this round are in registers
        else __syncthreads();
        if (tid < have) dmass[base + tid] = w;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int item = tid + i * kEvThreads, z = item >= per, at = (item - z * per) / nc, ch = item - z * per - at * nc;
            if (item < 2 * per && at < have) {
                uint4 o = q[i];
                if (cut) {
                    const float s_new = __fmul_rn(__uint_as_float(s_amax[z][at / B]), kInv127), rcp = 1.0f / s_new;
                    int8_t* c = reinterpret_cast<int8_t*>(&o);
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        c[j] = s_new > 0.0f ? (int8_t)kvb_code(__fmul_rn((float)c[j], s_old[i]), s_new, rcp) : (int8_t)0;
                    if (ch == 0 && at % B == 0) dscale[z][(base + at) / B] = s_new;
                } else if (ch == 0 && at % B == 0) {
                    dscale[z][(base + at) / B] = s_old[i];
                }
                *reinterpret_cast<uint4*>(dst[z] + (int64_t)(base + at) * hd + ch * 16) = o;
            }
        }
        __syncthreads();                         // s_amax is free
    }
    if (a.in_place) cl.sync();                   // every weight has been read
    const int end = min(n, a.dst.cap);
    for (int i = left + rank * kEvThreads + tid; i < end; i += CN * kEvThreads) dmass[i] = 0.0f;
}

template <int ITEMS>
cudaError_t evict_launch(const KvbEvictArgs& a, int cn, cudaStream_t st) {
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
    return cudaLaunchKernelEx(&cfg, kvb_evict_kernel<ITEMS>, a);
}

}  // namespace

cudaError_t launch_kvb_append(const KvbAppendArgs& a, cudaStream_t st) {
    // every touched block holds a new row, and a slot's rows touch at most
    // n / block + 2 of them
    const int64_t rows = a.r.rows, some = rows < a.c.slots ? rows : a.c.slots;
    const int64_t by_size = rows / a.c.block + 2 * some;
    const dim3 grid((unsigned)(rows < by_size ? rows : by_size), a.c.heads, 2);
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
    int cn = 8;
    while (cn > 1 && ((int64_t)a.src.slots * a.src.heads * cn > 296 || cn * kEvUnit > a.src.cap * 2)) cn >>= 1;
    const int items = (2 * kEvUnit * (a.src.hd / 16) + kEvThreads - 1) / kEvThreads;
    if (items <= 1) return evict_launch<1>(a, cn, st);
    if (items <= 2) return evict_launch<2>(a, cn, st);
    if (items <= 4) return evict_launch<4>(a, cn, st);
    return evict_launch<8>(a, cn, st);
}

}  // namespace w8a8

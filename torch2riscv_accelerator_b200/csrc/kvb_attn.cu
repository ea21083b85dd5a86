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

template <typename T>
cudaError_t attn_launch(const KvbAttnArgs& a, cudaStream_t st) {
    const cudaError_t e = launch_k(kvb_attn_kernel<T>, dim3(a.r.rows, a.heads), dim3(kThreads), 0, st, a);
    if (e != cudaSuccess || !a.mass) return e;
    return launch_k(kvb_mass_kernel<T>, dim3((a.c.cap + kThreads - 1) / kThreads, a.c.heads, a.c.slots), dim3(kThreads),
                    0, st, a);
}

}  // namespace

size_t kvb_attn_scratch(const KvbCache&, int heads, int rows, bool, bool mass) {
    return mass ? (size_t)rows * heads * sizeof(float) : 0;
}

cudaError_t launch_kvb_attn(const KvbAttnArgs& a, cudaStream_t st) {
    return a.type == KVB_F32    ? attn_launch<float>(a, st)
           : a.type == KVB_BF16 ? attn_launch<__nv_bfloat16>(a, st)
                                : attn_launch<__half>(a, st);
}

}  // namespace w8a8

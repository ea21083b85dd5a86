// The block-scaled 8-bit KV cache (kvb.cu, kvb_attn.cu, kvb_rows.cu): codes int8
// [slots][kv_heads][cap][hd] for K and V, one fp32 scale per (slot, KV head,
// block of tokens): the value held is code * scale.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "kvb_plan.cuh"
#include "pdl.cuh"

namespace w8a8 {

constexpr int kKvbMaxHd = 256;
enum KvbType { KVB_F32 = 0, KVB_BF16 = 1, KVB_F16 = 2 };
constexpr unsigned int kKvbErrCapacity = 128u;   // error bit 7: a row or a length past the capacity

struct KvbCache {
    int8_t* k;
    int8_t* v;
    float* ks;
    float* vs;
    int slots, heads, cap, hd, block;
    int64_t slot_stride;                         // codes between slots
    int64_t scale_stride;                        // scales between slots
};

// Rows of several sequences: slot b's are r0 .. r0 + n - 1, the first at cache
// position pos[b]; start null: row b alone.
struct KvbRows {
    int rows;
    const int32_t* pos;
    const int32_t* start;
};

struct KvbSpan {
    int r0, n, p;                                // first row, rows, position of the first (negative: idle)
};

// The offsets are data: clamped into [0, rows], so that no order of them
// leads out of the row arrays.
__device__ __forceinline__ KvbSpan kvb_span(const KvbRows& r, int b) {
    KvbSpan s;
    s.p = r.pos[b];
    if (r.start) {
        const int a = min(max(r.start[b], 0), r.rows), e = min(max(r.start[b + 1], 0), r.rows);
        s.r0 = a, s.n = max(e - a, 0);
    } else {
        s.r0 = b, s.n = 1;
    }
    return s;
}

// The slot whose rows hold row r, or -1 (a row behind the last sequence):
// the last b with start[b] <= r.
__device__ __forceinline__ int kvb_slot_of(const KvbRows& w, int slots, int r) {
    if (!w.start) return r;
    int lo = 0, hi = slots;                      // start[lo] <= r < start[hi], if any
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (w.start[mid] <= r) lo = mid;
        else hi = mid;
    }
    return w.start[lo] <= r && r < w.start[lo + 1] ? lo : -1;
}

struct KvbAppendArgs {
    KvbCache c;
    KvbRows r;
    const void* k;
    const void* v;
    int64_t k_stride, v_stride;                  // elements between rows
    int type;
};
struct KvbReadArgs {
    KvbCache c;
    KvbRows r;
    void* k;
    void* v;
    int type;
};
struct KvbAttnArgs {
    KvbCache c;
    KvbRows r;
    const void* q;                               // [rows][heads][hd], q_stride elements between rows
    int64_t q_stride;
    void* out;                                   // [rows][heads][hd]
    int heads, type;
    float scale;
    float* mass;                                 // [slots][kv_heads][cap] or null
    void* scratch;
};
struct KvbEvictArgs {
    KvbCache src, dst;
    const float* mass;                           // [slots][kv_heads][src.cap]
    float* dst_mass;                             // [slots][kv_heads][dst.cap]
    const int32_t* count;
    int keep, sink, recent;
    int32_t* kept;                               // [slots][kv_heads][keep]
    int32_t* count_out;
    int in_place;
};

cudaError_t launch_kvb_append(const KvbAppendArgs& a, cudaStream_t st);
cudaError_t launch_kvb_read(const KvbReadArgs& a, cudaStream_t st);
cudaError_t launch_kvb_evict(const KvbEvictArgs& a, cudaStream_t st);
size_t kvb_attn_scratch(const KvbCache& c, int heads, int rows, bool one_row, bool mass, int qbytes);
cudaError_t launch_kvb_attn(const KvbAttnArgs& a, cudaStream_t st);
size_t kvb_rows_scratch(const KvbCache& c, int heads, int rows, bool mass, int qbytes);
cudaError_t launch_kvb_rows(const KvbAttnArgs& a, cudaStream_t st);
unsigned int kvb_rows_read_clear_errors();
unsigned int kvb_read_clear_errors();
unsigned int kvb_attn_read_clear_errors();

template <typename T>
__device__ __forceinline__ float kvb_f(T x);
template <>
__device__ __forceinline__ float kvb_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ float kvb_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float kvb_f<__half>(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T kvb_t(float x);
template <>
__device__ __forceinline__ float kvb_t<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 kvb_t<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half kvb_t<__half>(float x) { return __float2half_rn(x); }

// 8 consecutive elements (16- or 32-byte aligned) as floats
template <typename T>
__device__ __forceinline__ void kvb_load8(const T* p, float* x) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        T h[8];
        *reinterpret_cast<uint4*>(h) = a;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = kvb_f<T>(h[i]);
    }
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

__device__ __forceinline__ uint32_t bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
// 16 consecutive elements of a row of type `type`
__device__ __forceinline__ void load16(const void* base, int type, int64_t at, float* y) {
    if (type == KVB_F32) {
        kvb_load8<float>(static_cast<const float*>(base) + at, y);
        kvb_load8<float>(static_cast<const float*>(base) + at + 8, y + 8);
    } else if (type == KVB_BF16) {
        kvb_load8<__nv_bfloat16>(static_cast<const __nv_bfloat16*>(base) + at, y);
        kvb_load8<__nv_bfloat16>(static_cast<const __nv_bfloat16*>(base) + at + 8, y + 8);
    } else {
        kvb_load8<__half>(static_cast<const __half*>(base) + at, y);
        kvb_load8<__half>(static_cast<const __half*>(base) + at + 8, y + 8);
    }
}
__device__ __forceinline__ void store1(void* base, int type, int64_t at, float y) {
    if (type == KVB_F32) static_cast<float*>(base)[at] = y;
    else if (type == KVB_BF16) static_cast<__nv_bfloat16*>(base)[at] = __float2bfloat16_rn(y);
    else static_cast<__half*>(base)[at] = __float2half_rn(y);
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

// pairs of floats in one instruction
__device__ __forceinline__ uint64_t pack2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t r, float& x, float& y) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(r));
}
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}
__device__ __forceinline__ uint64_t sub2(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}

// rint(num / den) saturated to +-127, the quotient correctly rounded before the
// rounding to an integer.
__device__ __forceinline__ int kvb_code(float num, float den) {
    return (int)fminf(fmaxf(rintf(__fdiv_rn(num, den)), -127.0f), 127.0f);
}

// The codes of N values num (N even): codes = rint(num / den), |num| <= 127 den
// up to rounding. The product with rcp ~ 1 / den is within 2 ulp of the quotient
// (3e-5 for |quotient| <= 128), so only where some value lies that close to a
// half (its distance d to the next integer: |d^2 - 1/4| < 2e-4) is the division
// itself needed. Adding 1.5 * 2^23 rounds to an integer whose low byte is the
// code. Scales below 2^-120 (their quotients could leave the range) divide too.
template <int N>
__device__ __forceinline__ void kvb_codes(const float* num, float den, float rcp, uint32_t* out) {
    constexpr float kMagic = 12582912.0f;
    const uint64_t r2 = pack2(rcp, rcp), m2 = pack2(kMagic, kMagic), q2 = pack2(-0.25f, -0.25f);
    float near = 1.0f;
    uint32_t t[N];
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const uint64_t y = mul2(pack2(num[i], num[i + 1]), r2), s = add2(y, m2), d = sub2(y, sub2(s, m2));
        float a, b;
        unpack2(fma2(d, d, q2), a, b);
        near = fminf(near, fminf(fabsf(a), fabsf(b)));
        t[i] = (uint32_t)s, t[i + 1] = (uint32_t)(s >> 32);
    }
    if (!(near > 2e-4f) || den < 7.5e-37f) {
#pragma unroll 1
        for (int w = 0; w < N / 4; ++w) {
            uint32_t c = 0;
#pragma unroll
            for (int i = 0; i < N; ++i)          // (registers: no indexing by w)
                if (i / 4 == w) c |= ((uint32_t)kvb_code(num[i], den) & 255u) << (8 * (i % 4));
#pragma unroll
            for (int i = 0; i < N / 4; ++i)
                if (i == w) out[i] = c;
        }
        return;
    }
#pragma unroll
    for (int w = 0; w < N / 4; ++w)
        out[w] = __byte_perm(__byte_perm(t[4 * w], t[4 * w + 1], 0x0040), __byte_perm(t[4 * w + 2], t[4 * w + 3], 0x0040), 0x5410);
}

// 16 codes of one scale in another: rint((q * s_old) / s_new)
__device__ __forceinline__ uint4 kvb_requant16(uint4 w, float s_old, float s_new, float rcp) {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
    const uint64_t bias2 = pack2(8388736.0f, 8388736.0f), s2 = pack2(s_old, s_old);
    uint32_t o[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float num[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {            // biased bytes as the low bits of 2^23 + b + 128
            const uint32_t y = x[2 * h + i / 2] ^ 0x80808080u;
            const uint64_t f = pack2(__uint_as_float(__byte_perm(y, 0x4b000000u, i % 2 ? 0x7442 : 0x7440)),
                                     __uint_as_float(__byte_perm(y, 0x4b000000u, i % 2 ? 0x7443 : 0x7441)));
            unpack2(mul2(sub2(f, bias2), s2), num[2 * i], num[2 * i + 1]);
        }
        kvb_codes<8>(num, s_new, rcp, o + 2 * h);
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
}

}  // namespace w8a8

// How prompt attention over the block-scaled KV cache (kvb_rows.cu) deals its
// units out to the CTAs: arithmetic for the device and for tests on the host.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define W8A8_HD __host__ __device__ __forceinline__
#else
#define W8A8_HD inline
#endif

namespace w8a8 {

// Shares are equal in tiles plus kUnitCost for each unit begun: a unit's first
// queries and last outputs cost about as much as two tiles (by tiles alone the
// CTA with a causal prompt's short units took 20 % longer than the others).
constexpr int kUnitCost = 2;

struct alignas(16) RowsUnit {
    int slot, m;                                 // 128-row tile of the slot
    int64_t before;                              // cost of the units before (a million rows of 64 heads on one pass 2^31)
    int tiles, p, r0, rows;                      // tiles, position of the slot's first row, its row, the slot's n * G live rows
};
struct alignas(16) RowsShare {                   // a CTA's share [lo, hi) of the cost
    int64_t lo, hi;
    int h, u, join, pad;                         // KV head and unit where it begins; if that unit is cut there for the
};                                               // first time, the last share with a part of it, else -1

// x / y for x >= 0, y > 0; 32-bit where both fit (a 64-bit division is a subroutine)
W8A8_HD int64_t div64(int64_t x, int64_t y) { return (x | y) >> 32 ? x / y : (int64_t)((uint32_t)x / (uint32_t)y); }

// Share c of at most `most` CTAs: total the cost of one KV head's units, before(u)
// of those before unit u, tiles(u) the unit's own.
template <class Before, class Tiles>
W8A8_HD RowsShare share_of(int c, int most, int64_t total, int heads, int units, Before before, Tiles tiles) {
    RowsShare w{};
    w.join = -1;
    const int64_t all = total * heads, ctas = all < most ? all : most;
    if (c >= ctas) return w;
    w.lo = div64(all * c, ctas), w.hi = div64(all * (c + 1), ctas);
    w.h = (int)div64(w.lo, total);
    const int64_t at = w.lo - w.h * total;
    int u = 0, hi = units;                       // the last unit that begins at or before `at`
    while (hi - u > 1) {
        const int mid = (u + hi) >> 1;
        if (before(mid) <= at) u = mid;
        else hi = mid;
    }
    w.u = u;
    const int64_t begin = w.h * total + before(u), end = begin + kUnitCost + tiles(u);
    if (w.lo > begin + kUnitCost && div64(all * (c - 1), ctas) <= begin + kUnitCost)
        w.join = (int)div64(end * ctas - 1, all);
    return w;
}

}  // namespace w8a8

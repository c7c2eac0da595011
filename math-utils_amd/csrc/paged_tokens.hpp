// paged_tokens.hpp - what the kernels over paged caches share: where a token's rows lie.
#pragma once

#include "device.hpp"
#include "kernels.hpp"

namespace aigpu {

namespace {

constexpr uint32_t THREADS = 256;
constexpr uint32_t NOWHERE = 0xFFFFFFFFu;

/* x, hidden from the compiler: what is derived from it is formed where it is
   used. Unrolled loops would otherwise hold every address and mask of their
   rare parts in registers: a hundred of the decode's, spilled, and twenty of
   append's, which cost it two of its six workgroups a CU. */
__device__ __forceinline__ int fresh_lane(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

/* sum over the LPR lanes of a row: a power of two times 1 or 3 */
template <int LPR>
__device__ __forceinline__ float row_sum(float x, int lane) {
    constexpr int P = LPR & -LPR;
#pragma unroll
    for (int o = P / 2; o > 0; o >>= 1) x += __shfl_xor(x, o, WAVE);
    if constexpr (LPR == P) {
        return x;
    } else {
        static_assert(LPR == 3 * P, "rows of 2^n or 3 2^n lanes");
        const int first = lane / LPR * LPR;
        return __shfl(x, first, WAVE) + __shfl(x, first + P, WAVE) + __shfl(x, first + 2 * P, WAVE);
    }
}

constexpr uint32_t MAX_TOKENS = 16;

/* A workgroup's token of a lane: sequence, position and page of token t0 + own. A wave
   takes every NW-th of the workgroup's nt <= MAX_TOKENS tokens, its lane l the l-th of
   those; all of a wave's lanes call it. */
struct Token {
    bool finds;                      // the lane has a token
    bool live;                       // which belongs to a sequence
    uint32_t own, pos, at, page;     // page NOWHERE: no place in the table; at: the row in it
};
template <int NW>
__device__ __forceinline__ Token find_token(const PagedCache& c, const uint32_t* starts, uint64_t t0, uint32_t nt,
                                            int w, int lane) {
    constexpr int MINE = MAX_TOKENS / NW;
    uint32_t before[MINE] = {};
    if (starts) {
        for (uint32_t k = 0; k <= c.batch; k += WAVE) {
            const bool in = k + lane <= c.batch;
            const uint32_t start = in ? starts[k + lane] : 0u;
#pragma unroll
            for (int i = 0; i < MINE; ++i) before[i] += __popcll(__ballot(in && start <= t0 + w + i * NW));
        }
    }
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < MINE; ++i) mine = lane == i ? before[i] : mine;
    Token x{};
    x.page = NOWHERE;
    x.own = w + lane * NW;
    x.finds = lane < MINE && x.own < nt;
    if (x.finds) {
        const uint64_t t = t0 + x.own;
        uint32_t b = uint32_t(t);
        uint64_t back = 1;                           // it is the sequence's back-th newest
        x.live = true;
        if (starts) {
            x.live = mine > 0 && mine <= c.batch;
            b = x.live ? mine - 1 : 0;
            const uint64_t end = starts[b + 1];
            x.live = x.live && end > t;
            back = x.live ? end - t : 1;
        }
        const uint64_t len = c.lengths[b];
        x.pos = uint32_t(len - back);
        const uint32_t slot = x.pos / c.pageSize;
        x.at = x.pos - slot * c.pageSize;
        if (x.live && len >= back && slot < c.tableWidth) x.page = c.table[b * c.tableStride + slot];
    }
    return x;
}

} // namespace

} // namespace aigpu

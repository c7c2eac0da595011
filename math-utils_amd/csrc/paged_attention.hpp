// paged_attention.hpp - one token's attention over a paged cache: the kernel of
// its forms (plain, scored, 4-bit pages), each compiled by a file of its own.
#pragma once

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "context.hpp"
#include "device.hpp"
#include "kernels.hpp"
#include "paged_tokens.hpp"

namespace aigpu {

namespace {

/*
    One token's attention over the pages.

    The batch is cut into slabs of 32 positions of one sequence, one kv head and
    up to 16 of its query heads (a pair: sequence, heads), listed pair by pair,
    and the list into one even run a wave: whatever the lengths, every wave reads
    as many slabs, within one, and the work is bounded by the keys and values,
    read once (HBM). paged_attention_kernel works a run off as one software
    pipeline over its slabs, whichever pair they belong to: page ids are read two
    slabs ahead, keys (registers) and values (DMA into LDS) one slab ahead, so
    loads stay in flight while a pair ends and the next one's queries are
    prepared.
      scores   v_mfma_f32_16x16x32_bf16, 16 keys as A, the heads' queries as B, in
               three terms of 8 bits each (x = hi + mid + lo exactly: fp32 is 24
               bits), so the products are fp32's; three instructions a tile cost
               11% of the matrix rate at full HBM bandwidth
      softmax  a running maximum and sum a head; lane l holds head l % 16
      p v      the weights in three terms likewise, as A, exactly the scores the
               lane holds; values as B through ds_read_b64_tr_b16
    A pair wholly in one run is written at once. What is left at the end of a run
    is joined over the workgroup's waves in LDS; pairs that span workgroups leave
    (max, sum, weighted values) records, two a wave at most, that are joined in
    their order, so results do not depend on timing: by the workgroup that finds
    itself the last of the pair's (a counter that it sets back to zero), or, where
    sequences of one length would leave a pair more records than one workgroup
    should read, by paged_merge_kernel.

    32 sequences of 1k to 32k under 32/4 heads of 128 (1.11 GB): 190 us, 5.8 TB/s,
    where a copy of 256 or 512 MB moves 5.9. Small calls are a chain of about 15 us:
    dispatch, lengths and list 4, page ids and queries 2, a first slab 3, its
    weights 1, the joins 5 (one sequence of 4096 under 16/8 heads, 16.8 MB: 15).

    The forms are kernels of their own, so that the plain one keeps its registers: scored
    (a cap's tanh, a bias by distance), and codes, the scored one over 4-bit pages:
      slabs    64 positions (9.2 KB of 128 channels), as 16 rows of a group are read
               transposed at once (ds_read_b64_tr_b4) and four groups read together
      keys     codes to registers, unpacked there into exact fp16; a lane takes a quarter
               of a row, so its scales are two at most
      values   codes through registers into LDS, read back transposed, unpacked per column
      products v_mfma_f32_16x16x32_f16: the pages' values exactly, q and the weights in two
               fp16 terms (22 bits), brought to a power of two where both hold down to
               2^-38 and 2^-40 of the largest
    32 sequences of 1k to 32k under 32/4 heads of 128 (312 MB): 86 to 89 us, 3.5 to 3.6 TB/s;
    11 us with a position or two each, 4.4 us a slab of each wave on top. A slab is some 650
    vector instructions of a wave (420 of them unpack), 2.6 of those 4.4 us for a SIMD's two
    waves, and 64 matrix ones: the 1.8 that are left, 30 us in all, are loads that two waves of
    one slab each do not cover (a slab's keys are asked for behind the scores). One workgroup a
    CU takes 114 us, three (128 channels) spill and take twice the time; of 64 channels three
    fit.
*/
constexpr bool scored(int form) { return form != PAGED_PLAIN; }
// positions of a slab: 4-bit rows are read 64 at a time, as their values are transposed in LDS
constexpr int slab_rows(int form) { return form == PAGED_CODES ? 64 : 32; }
constexpr int WAVES = 4;
constexpr int ROWS = 16;             // query heads of a group
constexpr uint32_t MAXB = 512;       // sequences of a launch
constexpr uint32_t MAX_RUNS = 4096;
// A pair's queries and its end cost about what a slab's loads do when many are
// short, so the list counts a unit for them before its slabs' units.
constexpr uint32_t OPENING = 1;

struct DecodeArgs {
    PagedDecodeParams p;
    uint32_t* arrived;               // [runs] by a pair's last run; zero between calls
    uint32_t* plan;                  // [MAXB + 1] units before each sequence, and in all; null: joined in the kernel
    float* records;                  // [runs][2] of record_floats
    uint32_t groups, perGroup;       // of one kv head's query heads
    uint32_t pageMagic, pageShift;   // pos / pageSize = pos pageMagic >> pageShift (pos below 2^31)
    float scaleLog2;                 // of q: the scores in units of ln 2; with a cap, as its fractions
    float capLog2;                   // the cap in units of ln 2, 0: none
    float series[6];                 // of the cap's tanh, times that
    int wideQ;                       // q rows can be read 16 bytes at a time
};

typedef __bf16 bf16v4 __attribute__((__vector_size__(4 * sizeof(__bf16))));

/* ds_read_b64_tr_b16: within each 16-lane group, lane i receives element i % 4
   of the 8-byte rows addressed by lanes i/4, i/4 + 4, i/4 + 8, i/4 + 12 */
__device__ __forceinline__ bf16v4 read_transposed(const uint16_t* lds) {
    typedef __attribute__((address_space(3))) bf16v4 lds_bf16v4;
    return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16v4*)(lds));
}

/* a wave's 64 blocks of 16 bytes into LDS, one after the other; cache policy 2: nontemporal
   (each value is read once) */
__device__ __forceinline__ void value_to_lds(const uint16_t* from, uint16_t* to) {
    __builtin_amdgcn_global_load_lds(from, (__attribute__((address_space(3))) void*)to, 16, 0, 2);
}

/* s_waitcnt vmcnt(N) alone */
template <int N>
__device__ __forceinline__ void wait_loads() {
    static_assert(N >= 0 && N < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
}

__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }


/* the eight rows of 32 bytes that 32 lanes read transposed lie in distinct
   banks (64 of 4 bytes): block x of 16 bytes of row r sits at x ^ this */
template <int D>
__device__ __forceinline__ int value_swizzle(int r) {
    if constexpr (D % 128 == 0) return 2 * (r & 7);        // rows start in the same bank
    else if constexpr (D % 64 == 0) return 2 * ((r >> 1) & 3);
    else return 2 * ((r >> 2) & 1);
}

__device__ __forceinline__ uint32_t first_of(const PagedDecodeParams& p, uint32_t len) {
    return p.window && len > p.window ? uint32_t(len - p.window) : 0u;
}

template <int SLAB>
__device__ __forceinline__ uint32_t slabs_of(const PagedDecodeParams& p, uint32_t len) {
    return len == 0 || len > p.maxLength ? 0u : (len + SLAB - 1) / SLAB - first_of(p, len) / SLAB;
}

/* the even cut of `total` units into runs: run w's first unit, and a unit's run */
struct Cut {
    uint32_t runs, each, extra;      // the first `extra` runs have one more
    __device__ __forceinline__ Cut(uint32_t total, uint32_t waves) {
        runs = total < waves ? total : waves;
        each = runs ? total / runs : 0;
        extra = runs ? total % runs : 0;
    }
    __device__ __forceinline__ uint32_t begin(uint32_t w) const {
        return w < runs ? w * each + (w < extra ? w : extra) : runs * each + extra;
    }
    __device__ __forceinline__ uint32_t run_of(uint32_t unit) const {
        const uint32_t longer = extra * (each + 1);
        return unit < longer ? unit / (each + 1) : extra + (unit - longer) / each;
    }
};

/* a record: the rows' maxima and sums, padded to 16 bytes, then [perGroup][D] */
__host__ __device__ constexpr uint32_t record_heads(uint32_t rows) { return (2 * rows + 3) / 4 * 4; }
__host__ __device__ constexpr uint32_t record_floats(uint32_t rows, uint32_t D) { return record_heads(rows) + rows * D; }

/* The parts of a pair whose units are begin .. end - 1: `joined` records of
   workgroups wg, wg + 1, ... over their runs, then one of run `to` if that went
   on to another pair. Of one part alone there is no record: its wave or its
   workgroup wrote the output. */
struct Parts {
    uint32_t from, to, joined, total;
    Parts() = default;
    __device__ __forceinline__ Parts(const Cut& cut, uint32_t begin, uint32_t end) {
        from = cut.run_of(begin + OPENING);
        to = cut.run_of(end - 1);
        const bool toEnd = end + OPENING >= cut.begin(to + 1);     // no later slab in run `to`
        const uint32_t wg = from / WAVES, last = to / WAVES;
        joined = last - wg + (toEnd || to % WAVES > (last == wg ? from % WAVES : 0u) ? 1 : 0);
        total = joined + (toEnd ? 0 : 1);
        if (from == to) total = 1;
    }
    // the place of part k's record in [runs][2]
    __device__ __forceinline__ uint32_t slot(uint32_t k) const {
        return k == joined ? to * 2 : ((from / WAVES + k) * WAVES + (k ? 0 : from % WAVES)) * 2 + 1;
    }
};

/* Records go from one workgroup to another within a launch, perhaps between
   XCDs, whose L2s do not see each other's lines: written and read past the L2
   (device scope), which spares the fences that would write back and invalidate
   it whole. Their order: the writer's stores are waited for before it counts
   itself in, and the reader reads after the last count. */
constexpr int PAST_L2 = 16;          // the buffer instructions' sc1 bit
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(float* base) {
    return __builtin_amdgcn_make_buffer_rsrc(base, 0, -1, 0x00027000);
}

struct Piece {
    uint32_t begin, end;             // the pair's units; begin NOWHERE: none
    uint32_t b, head, rows;          // its query heads: head .. head + rows - 1 of sequence b
};

struct Slab {
    uint32_t b, pair;                // pair: kv head * groups + group
    uint32_t pos, first, len;        // its first position; the attended range
    uint32_t is;                     // of BEGINS .. CLOSES
};
enum : uint32_t {
    BEGINS = 1, ENDS = 2,            // the pair's first slab, its last
    OPENS = 4, CLOSES = 8,           // the first of the pair in this run, the last
};

/* fp32 to three bf16 terms whose sum it is: each takes the next 8 bits */
__device__ __forceinline__ void split3(const float (&x)[8], u32x4 (&t)[3]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
            t[k][i] = __builtin_amdgcn_perm(ub, ua, 0x07060302);    // the high halves
            a -= __uint_as_float(ua & 0xFFFF0000u);
            b -= __uint_as_float(ub & 0xFFFF0000u);
        }
    }
}

/* x times sigmoid of the gate half of its q row when the output gate is on */
__device__ __forceinline__ float gated(const PagedDecodeParams& p, uint32_t b, uint32_t head, uint32_t d, float x) {
    if (!p.outputGate) return x;
    return x * sigmoid_of(load_elem(p.q, b * p.qTokenStride + head * p.qStride + p.c.dim + d, p.inType));
}

/*
    Joins rows `row0` .. of a pair's records into the output of query heads
    `head` .. of sequence b, by a whole workgroup or, with `alone`, by a wave: the
    same sums in the same order. A thread takes four columns of a row and adds the
    parts up, TILE of them (one trip to memory) at a time; or, where that takes
    fewer trips, the parts are dealt to WAVES shares, a wave of the workgroup each
    (a wave alone takes them one after the other), that meet in `room`.
*/
constexpr int JOIN_FLOATS = 6;
template <int D, uint32_t TILE>
__device__ __forceinline__ void join_parts(const DecodeArgs& a, const Parts& parts, uint32_t b, uint32_t head,
                                           uint32_t row0, uint32_t rows, bool alone, float* room) {
    const PagedDecodeParams& p = a.p;
    const uint32_t size = record_floats(a.perGroup, D), skip = record_heads(a.perGroup), units = rows * (D / 4);
    const auto records = buffer_of(a.records);
    auto word = [&](uint32_t at) {
        return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(records, at * 4, 0, PAST_L2));
    };
    const uint32_t lane = threadIdx.x % WAVE, wave = alone ? 0 : uniform(threadIdx.x / WAVE);
    const uint32_t waves = alone ? 1 : WAVES;
    const uint32_t trips = (units + THREADS - 1) / THREADS * ((parts.total + TILE - 1) / TILE);
    const uint32_t shared = (units + WAVE - 1) / WAVE * ((parts.total + WAVES * TILE - 1) / (WAVES * TILE));
    const uint32_t shares = trips <= shared ? 1 : WAVES;
    // without shares the waves take the columns in turn, with them the shares
    const uint32_t stepU = shares == 1 ? waves * WAVE : WAVE;
#pragma unroll 1
    for (uint32_t u0 = shares == 1 ? wave * WAVE : 0; u0 < units; u0 += stepU) {
        const uint32_t unit = u0 + lane;
        const bool live = unit < units;
        const uint32_t row = row0 + unit / (D / 4), d = unit % (D / 4) * 4;
        float top = -INFINITY, sum = 0.0f;
        floatx4 x = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
        for (uint32_t q = shares == 1 ? 0 : wave; q < shares; q += waves) {
            top = -INFINITY;
            sum = 0.0f;
            x = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
            for (uint32_t k0 = q; k0 < parts.total && live; k0 += shares * TILE) {
                float mk[TILE], lk[TILE];
                u32x4 xk[TILE];
#pragma unroll
                for (uint32_t i = 0; i < TILE; ++i) {
                    const uint32_t k = k0 + i * shares, at = parts.slot(k < parts.total ? k : k0) * size;
                    mk[i] = word(at + row);
                    lk[i] = word(at + a.perGroup + row);
                    xk[i] = __builtin_amdgcn_raw_buffer_load_b128(records, (at + skip + row * D + d) * 4, 0, PAST_L2);
                }
                float next = top;
#pragma unroll
                for (uint32_t i = 0; i < TILE; ++i)
                    if (k0 + i * shares < parts.total) next = fmaxf(next, mk[i]);
                const float base = next == -INFINITY ? 0.0f : next, keep = exp2f(top - base);
                sum *= keep;
                x *= keep;
#pragma unroll
                for (uint32_t i = 0; i < TILE; ++i) {
                    if (k0 + i * shares >= parts.total) break;
                    const float f = exp2f(mk[i] - base);
                    sum += lk[i] * f;
                    x += __builtin_bit_cast(floatx4, xk[i]) * f;
                }
                top = next;
            }
            if (shares == 1) break;
            float* mine = room + (q * WAVE + lane) * JOIN_FLOATS;
            mine[0] = top;
            mine[1] = sum;
#pragma unroll
            for (int i = 0; i < 4; ++i) mine[2 + i] = x[i];
        }
        if (shares > 1) {
            if (alone) wave_sync();
            else __syncthreads();
            if (wave == 0) {
                top = -INFINITY;
                sum = 0.0f;
                x = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
                for (uint32_t o = 0; o < WAVES; ++o) {
                    const float* theirs = room + (o * WAVE + lane) * JOIN_FLOATS;
                    const float next = fmaxf(top, theirs[0]), base = next == -INFINITY ? 0.0f : next;
                    const float keep = exp2f(top - base), f = exp2f(theirs[0] - base);
                    sum = sum * keep + theirs[1] * f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = x[i] * keep + theirs[2 + i] * f;
                    top = next;
                }
            }
        }
        if (live && (shares == 1 || wave == 0)) {
            const uint32_t h = head + row - row0;
            const float by = 1.0f / sum;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                p.out[(size_t(b) * p.heads + h) * D + d + i] = gated(p, b, h, d + i, x[i] * by);
        }
        if (shares > 1) {            // the room is free again
            if (alone) wave_sync();
            else __syncthreads();
        }
    }
}

/* workgroups a CU: what registers and LDS hold (fp32 queries over 4-bit pages spill 5 registers at
   128 channels and 10 at 256) */
constexpr int occupancy(int D, int form) { return form == PAGED_CODES && D == 64 ? 3 : (D <= 128 ? 2 : 1); }

/*
    4-bit rows. An element is s (c - 8) with c its code and s its block's scale, an
    fp16 number of 8 significant bits: the product has at most 11, so fp16 holds it
    exactly. Eight codes of a word become four pairs (elements i and i + 4): each
    code moves to the top of a significand whose exponent makes it 16 + c, and one
    packed product and sum takes that to s (16 + c) - 24 s, rounded once: not at all.
*/
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef float float2v __attribute__((ext_vector_type(2)));

/* a scale for both elements of a pair, and what takes the 24 off */
__device__ __forceinline__ half2v scale_of(uint16_t bits, half2v& off) {
    const _Float16 s = __builtin_bit_cast(_Float16, bits);
    off = half2v{s, s} * half2v{_Float16(-24.0f), _Float16(-24.0f)};
    return half2v{s, s};
}
/* the unpacking's constants, in registers: an instruction takes no two literals */
struct Unpack {
    uint32_t mask = 0x03C003C0u, sixteen = 0x4C004C00u;
    __device__ __forceinline__ Unpack() { asm("" : "+v"(mask), "+s"(sixteen)); }
    __device__ __forceinline__ half2v pair(uint32_t at) const {
        return __builtin_bit_cast(half2v, (at & mask) | sixteen);
    }
};
__device__ __forceinline__ half8 joined(half2v a, half2v b, half2v c, half2v d) {
    return half8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ half8 values_of(const Unpack& u, uint32_t word, half2v by, half2v off) {
    return joined(__builtin_elementwise_fma(u.pair(word << 6), by, off), __builtin_elementwise_fma(u.pair(word << 2), by, off),
                  __builtin_elementwise_fma(u.pair(word >> 2), by, off), __builtin_elementwise_fma(u.pair(word >> 6), by, off));
}
/* a word of eight rows' codes of one column, with their scales in pairs alike */
__device__ __forceinline__ half8 values_of(const Unpack& u, uint32_t word, const half2v (&by)[4], const half2v (&off)[4]) {
    return joined(__builtin_elementwise_fma(u.pair(word << 6), by[0], off[0]), __builtin_elementwise_fma(u.pair(word << 2), by[1], off[1]),
                  __builtin_elementwise_fma(u.pair(word >> 2), by[2], off[2]), __builtin_elementwise_fma(u.pair(word >> 6), by[3], off[3]));
}
__device__ __forceinline__ void scales_of(u32x4 scales, half2v (&by)[4], half2v (&off)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t pair = scales[i];             // (the cast of an element in place takes the first one)
        by[i] = __builtin_bit_cast(half2v, pair);
        off[i] = by[i] * half2v{_Float16(-24.0f), _Float16(-24.0f)};
    }
}
/* the largest of lanes c, c + 16, c + 32 and c + 48, by swaps of lanes that need no LDS */
__device__ __forceinline__ float over_groups(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const uint32_t y = __float_as_uint(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
    const auto b = __builtin_amdgcn_permlane32_swap(y, y, false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

/* two fp32 values as pairs of fp16 terms: the nearest, then what it leaves */
__device__ __forceinline__ u32x2 split_f16(float a, float b) {
    const half2v hi = __builtin_convertvector(float2v{a, b}, half2v);
    const half2v lo = __builtin_convertvector(float2v{fmaf(float(hi[0]), -1.0f, a), fmaf(float(hi[1]), -1.0f, b)}, half2v);
    return u32x2{__builtin_bit_cast(uint32_t, hi), __builtin_bit_cast(uint32_t, lo)};
}
/* the same of their products with `up`, which only the terms round (taken for q too, this
   form costs a small call 0.3 us) */
__device__ __forceinline__ u32x2 split_f16(float a, float b, float up) {
    const half2v hi = __builtin_convertvector(float2v{a * up, b * up}, half2v);
    const half2v lo = __builtin_convertvector(float2v{fmaf(a, up, -float(hi[0])), fmaf(b, up, -float(hi[1]))}, half2v);
    return u32x2{__builtin_bit_cast(uint32_t, hi), __builtin_bit_cast(uint32_t, lo)};
}
/* N words of a row from an address of 4 bytes' alignment */
template <int N>
__device__ __forceinline__ void read_words(const char* at, u32x4* to) {
    typedef uint32_t words2 __attribute__((ext_vector_type(2), aligned(4)));
    typedef uint32_t words3 __attribute__((ext_vector_type(3), aligned(4)));
    typedef uint32_t words4 __attribute__((ext_vector_type(4), aligned(4)));
    if constexpr (N >= 4) {
        to[0] = *reinterpret_cast<const words4*>(at);
        if constexpr (N > 4) read_words<N - 4>(at + 16, to + 1);
    } else if constexpr (N == 3) {
        const words3 x = *reinterpret_cast<const words3*>(at);
        to[0] = u32x4{x[0], x[1], x[2], 0u};
    } else {
        static_assert(N == 2, "rows of 2, 3, 4, 6 or 8 blocks");
        const words2 x = *reinterpret_cast<const words2*>(at);
        to[0] = u32x4{x[0], x[1], 0u, 0u};
    }
}
/* a row's N scales, two a register */
template <int N>
__device__ __forceinline__ void read_scales(const uint16_t* at, uint32_t* to) {
    if constexpr (N % 2) {               // 6 bytes a row: no word starts every row
#pragma unroll
        for (int i = 0; i < N; i += 2) to[i / 2] = at[i] | (i + 1 < N ? uint32_t(at[i + 1]) << 16 : 0u);
    } else {
        u32x4 x[2];
        if constexpr (N == 2) {
            to[0] = *reinterpret_cast<const uint32_t*>(at);
        } else {
            read_words<N / 2>(reinterpret_cast<const char*>(at), x);
#pragma unroll
            for (int i = 0; i < N / 2; ++i) to[i] = x[0][i];
        }
    }
}
/* ds_read_b64_tr_b4: within each 16-lane group, lane i receives 4-bit element i of the
   8-byte rows addressed by lanes 0 .. 15, row n's as its own element n */
__device__ __forceinline__ u32x2 read_codes(const uint16_t* lds) {
    typedef int int2v __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) int2v lds_int2v;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_int2v*)(lds)));
}
/* the 16 rows that a group reads transposed, 16 a + b for a and b of 0 .. 3, in distinct
   banks where the row's length allows: block x of 16 bytes of row r sits at x ^ this */
template <int D>
__device__ __forceinline__ int code_swizzle(int r) {
    if constexpr (D == 256) return (r >> 4 & 3) * 2 + (r >> 1 & 1);
    else if constexpr (D == 128) return r >> 4 & 3;
    else if constexpr (D == 64 || D == 192) return r >> 4 & 1;
    else return 0;
}

/* The kernel's arguments, read where they are used: kept in scalar registers over the
   loop, those that it does not need push out (through vector lanes) those that it does. */
__device__ __forceinline__ const DecodeArgs& arguments() {
    typedef const __attribute__((address_space(4))) DecodeArgs constant_args;
    constant_args* at = (constant_args*)__builtin_amdgcn_kernarg_segment_ptr();
    asm("" : "+s"(at));
    return *(const DecodeArgs*)at;
}

template <int D, bool BF, int FORM>
__global__ __launch_bounds__(THREADS, occupancy(D, FORM)) void paged_attention_kernel(DecodeArgs a) {
    constexpr bool CODES = FORM == PAGED_CODES;
    constexpr int SLAB = slab_rows(FORM);
    constexpr int DB = D / 32, CT = D / 16, BPR = D / 8;
    constexpr int VLOADS = SLAB * BPR / WAVE;
    // a lane's 8 elements of the scores' step db start at first_at(g) + STEP db: of 4-bit
    // rows a lane reads a quarter of one
    constexpr int STEP = CODES ? 8 : 32;
    auto first_at = [](int g) { return CODES ? 8 * DB * g : 8 * g; };
    constexpr int HALF = CODES ? (16 * D > 1536 ? 16 * D : 1536) : SLAB * D;   // of vbuf; 6 KB a wave are the joins' room
    const PagedDecodeParams& p = a.p;
    const PagedCache& c = p.c;
    const int lane = threadIdx.x & 63, w = int(uniform(threadIdx.x >> 6));
    const uint32_t B = c.batch, pairs = c.kvHeads * a.groups, G = p.heads / c.kvHeads;

    __shared__ uint32_t pre[MAXB + 1], lens[MAXB], sums[WAVES];
    __shared__ uint64_t place[WAVES][SLAB];
    __shared__ float2 turns[WAVES][D / 2];
    __shared__ float gamma[D];
    __shared__ float wm[WAVES][ROWS], wl[WAVES][ROWS], total[ROWS];
    // pairs that waves leave in parts: [w] in the record of a run that went on to
    // another pair, [WAVES + w] open at the run's end
    __shared__ Piece pieces[2 * WAVES];
    __shared__ Parts joins[2 * WAVES];            // those that this workgroup joins; total 0: none
    __shared__ uint32_t leftEnds[WAVES];          // bit 0: from the pair's first slab, bit 1: to its last
    __shared__ __attribute__((aligned(16))) uint16_t vbuf[WAVES][2][HALF];
    // a slab's scales: the keys' [row][block], the values' [block][pair of rows]
    __shared__ __attribute__((aligned(16))) uint16_t kscales[CODES ? WAVES : 1][CODES ? SLAB * DB : 8];
    __shared__ __attribute__((aligned(16))) uint32_t vscales[CODES ? WAVES : 1][CODES ? DB * SLAB / 2 : 4];

    // ---- the list: units before each sequence ----
    {
        uint32_t own[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t b = 2 * threadIdx.x + i;
            const uint32_t len = b < B ? c.lengths[b] : 0u;
            if (b < B) lens[b] = len;
            const uint32_t slabs = slabs_of<SLAB>(p, len);
            own[i] = slabs ? (slabs + OPENING) * pairs : 0u;
        }
        if (p.gamma)
            for (int d = threadIdx.x; d < D; d += THREADS) gamma[d] = p.gamma[d] + p.offset;
        if (lane < 2) pieces[w + lane * WAVES].begin = NOWHERE;
        uint32_t x = own[0] + own[1];
#pragma unroll
        for (int o = 1; o < WAVE; o <<= 1) {
            const uint32_t y = __shfl_up(x, o, WAVE);
            if (lane >= o) x += y;
        }
        if (lane == 63) sums[w] = x;
        __syncthreads();
        uint32_t before = x - own[0] - own[1];
        for (int k = 0; k < w; ++k) before += sums[k];
        const uint32_t b = 2 * threadIdx.x;
        if (b <= B) pre[b] = before;
        if (b + 1 <= B) pre[b + 1] = before + own[0];
        if (threadIdx.x == THREADS - 1 && B == MAXB) pre[B] = before + own[0] + own[1];
        __syncthreads();
    }
    if (a.plan && blockIdx.x == 0)
        for (uint32_t i = threadIdx.x; i <= B; i += THREADS) a.plan[i] = pre[i];
    // sequences without a slab: empty ones, and those that cannot be
    for (uint32_t b = blockIdx.x; b < B; b += gridDim.x) {
        if (pre[b] != pre[b + 1]) continue;
        const float x = lens[b] ? __builtin_nanf("") : 0.0f;
        for (uint32_t i = threadIdx.x; i < p.heads * D; i += THREADS) p.out[size_t(b) * p.heads * D + i] = x;
    }

    const Cut cut(uniform(pre[B]), gridDim.x * WAVES);
    const uint32_t run = blockIdx.x * WAVES + w;
    const uint32_t runEnd = cut.begin(run + 1);
    uint32_t at = cut.begin(run);                 // the next slab's unit
    uint32_t seq = 0, pair = 0, slab = 0, slabs = 1, len = 0, fresh = OPENS;
    // to the next pair's first slab, if the run reaches it
    auto next_pair = [&] {
        at += OPENING;
        slab = 0;
        if (at < runEnd && ++pair == pairs) {
            pair = 0;
            do ++seq;                             // at < pre[B]: a later sequence has slabs
            while (uniform(pre[seq]) == uniform(pre[seq + 1]));
            len = uniform(lens[seq]);
            slabs = slabs_of<SLAB>(p, len);
        }
    };
    if (at < runEnd) {
        uint32_t lo = 0, hi = B;                  // pre[lo] <= at < pre[hi]
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (uniform(pre[mid]) <= at) lo = mid;
            else hi = mid;
        }
        seq = lo;
        len = uniform(lens[seq]);
        slabs = slabs_of<SLAB>(p, len);
        const uint32_t in = at - uniform(pre[seq]);
        pair = in / (slabs + OPENING);
        slab = in % (slabs + OPENING);
        if (slab < OPENING) at += OPENING - slab, slab = 0;
        else slab -= OPENING;
    }
    auto list = [&](Slab& s) -> bool {
        if (at >= runEnd) return false;
        s.b = seq;
        s.pair = pair;
        s.first = first_of(p, len);
        s.len = len;
        s.pos = (s.first / SLAB + slab) * SLAB;
        s.is = fresh | (slab == 0 ? BEGINS | OPENS : 0u) | (slab + 1 == slabs ? ENDS | CLOSES : 0u) |
               (at + 1 >= runEnd ? CLOSES : 0u);
        fresh = 0;
        ++at;
        if (++slab == slabs) next_pair();
        return true;
    };

    auto cold = [&]() -> const DecodeArgs& {
        if constexpr (CODES) return arguments();
        else return a;
    };

    // ---- the stages of a slab ----
    // its page ids: lane r (of SLAB) holds row r's; rows outside the attended
    // range stand at its ends, so that nothing else is read
    struct Rows { uint32_t page, row; };
    auto find = [&](const Slab& s, Rows& r) {
        const DecodeArgs& a = cold();
        const PagedCache& c = a.p.c;
        uint32_t pos = s.pos + (lane & (SLAB - 1));
        pos = pos < s.first ? s.first : (pos < s.len ? pos : s.len - 1);
        const uint32_t slot = CODES ? uint32_t(uint64_t(pos) * a.pageMagic >> a.pageShift) : pos / c.pageSize;
        r.row = pos - slot * c.pageSize;
        r.page = c.table[s.b * c.tableStride + slot];
    };
    // its keys into registers (A operands: row lane % 16, 8 elements a lane),
    // its values into LDS; false where a page lies outside the pool (its rows
    // are then read from page 0)
    struct Chunk {                   // the j-th 16 bytes of a lane among a slab's rows of DB each
        uint32_t row, block;
        __device__ __forceinline__ Chunk(uint32_t j, uint32_t lane) {
            if constexpr (WAVE % DB == 0) row = WAVE / DB * j + lane / DB, block = lane % DB;
            else row = (WAVE * j + lane) / DB, block = (WAVE * j + lane) % DB;
        }
    };
    constexpr int KRB = CODES ? 4 : 2, KRD = CODES ? (DB + 3) / 4 : DB;
    u32x4 kr[KRB][KRD];              // keys: rows 16 rb + lane % 16
    u32x4 vr[CODES ? DB : 1];        // 4-bit values: 16 bytes a lane, row after row
    uint32_t ksr[CODES ? (DB + 1) / 2 : 1], vsr[CODES ? (DB + 1) / 2 : 1];   // row `lane`'s scales
    auto issue = [&](uint32_t pair, Rows r, int half) -> bool {
        const DecodeArgs& a = cold();
        const PagedDecodeParams& p = a.p;
        const PagedCache& c = p.c;
        const int lane = fresh_lane(threadIdx.x & 63), g = lane >> 4, c16 = lane & 15;
        const bool ok = r.page < c.pages;
        const uint64_t mine = (ok ? uint64_t(r.page) * c.pageStride + uint64_t(r.row) * c.rowStride : 0) +
                              uint64_t(pair / a.groups) * c.headStride;
        wave_sync();
        if (lane < SLAB) place[w][lane] = CODES ? mine * (D / 2) : mine;
        wave_sync();
        if constexpr (CODES) {
            const char* values = reinterpret_cast<const char*>(c.values);
#pragma unroll
            for (int j = 0; j < DB; ++j) {
                const Chunk at(j, lane);
                vr[j] = *reinterpret_cast<const u32x4*>(values + place[w][at.row] + 16 * at.block);
            }
            read_scales<DB>(p.keyScales + mine * DB, ksr);
            read_scales<DB>(p.valueScales + mine * DB, vsr);
        } else {
#pragma unroll
            for (int rb = 0; rb < 2; ++rb) {
                const uint16_t* k = c.keys + place[w][16 * rb + c16] + 8 * g;
#pragma unroll
                for (int db = 0; db < DB; ++db) kr[rb][db] = *reinterpret_cast<const u32x4*>(k + 32 * db);
            }
            uint16_t* to = vbuf[w][half];
#pragma unroll
            for (int j = 0; j < VLOADS; ++j) {
                const int i = j * WAVE + lane, row = i / BPR, block = (i % BPR) ^ value_swizzle<D>(row);
                value_to_lds(c.values + place[w][row] + 8 * block, to + j * WAVE * 8);
            }
        }
        return __all(ok);
    };
    // 4-bit rows: the keys apart, as the scores free their registers later
    auto issue_keys = [&] {
        const PagedCache& c = cold().p.c;
        const int lane = fresh_lane(threadIdx.x & 63), g = lane >> 4, c16 = lane & 15;
        const char* keys = reinterpret_cast<const char*>(c.keys) + g * (D / 8);
#pragma unroll
        for (int rb = 0; rb < KRB; ++rb) read_words<DB>(keys + place[w][16 * rb + c16], kr[rb]);
    };
    // 4-bit rows: the values and both scales from the registers into LDS
    auto stage = [&] {
        if constexpr (CODES) {
#pragma unroll
            for (int j = 0; j < DB; ++j) {
                const Chunk at(j, lane);
                *reinterpret_cast<u32x4*>(vbuf[w][0] + (at.row * DB + (at.block ^ code_swizzle<D>(at.row))) * 8) = vr[j];
            }
            if constexpr (DB % 2 == 0) {
#pragma unroll
                for (int i = 0; i < DB / 2; ++i) reinterpret_cast<uint32_t*>(kscales[w] + lane * DB)[i] = ksr[i];
            } else {
#pragma unroll
                for (int b = 0; b < DB; ++b) kscales[w][lane * DB + b] = uint16_t(ksr[b / 2] >> 16 * (b & 1));
            }
            uint16_t* pairs = reinterpret_cast<uint16_t*>(vscales[w]);
#pragma unroll
            for (int b = 0; b < DB; ++b) {
                // rows 16 rb + 4 g + i of even and odd rb are pairs
                pairs[((b * 2 + (lane >> 5)) * 16 + (lane & 15)) * 2 + (lane >> 4 & 1)] =
                    uint16_t(vsr[b / 2] >> 16 * (b & 1));
            }
            wave_sync();
        }
    };
    // the raw queries of a pair, lane (c16, g) holding head c16's elements
    // first_at(g) + STEP db + 0..7: the B operand's layout
    constexpr int RAW = BF ? 1 : 2;
    u32x4 raw[DB][RAW];
    auto ask = [&](const Slab& s) {
        const DecodeArgs& a = cold();
        const PagedDecodeParams& p = a.p;
        const int lane = fresh_lane(threadIdx.x & 63), g = lane >> 4, c16 = lane & 15;
        const uint32_t group = s.pair % a.groups, kvh = s.pair / a.groups;
        const uint32_t h = group * a.perGroup + c16;
        const uint32_t head = kvh * G + (uint32_t(c16) < a.perGroup && h < G ? h : group * a.perGroup);
        const size_t row = s.b * p.qTokenStride + head * p.qStride + first_at(g);
        if (a.wideQ) {
            const u32x4* src = reinterpret_cast<const u32x4*>(static_cast<const char*>(p.q) + row * (BF ? 2 : 4));
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < RAW; ++i) raw[db][i] = src[db * (STEP / 8) * RAW + i];
        } else if constexpr (BF) {
            const uint16_t* src = static_cast<const uint16_t*>(p.q) + row;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    raw[db][0][i] = src[STEP * db + 2 * i] | uint32_t(src[STEP * db + 2 * i + 1]) << 16;
        } else {
            const uint32_t* src = static_cast<const uint32_t*>(p.q) + row;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 8; ++i) raw[db][i / 4][i % 4] = src[STEP * db + i];
        }
    };
    const uint32_t rot = p.freqs ? uint32_t(p.rot) : 0;
    float freq[(D / 2 + WAVE - 1) / WAVE];
#pragma unroll
    for (uint32_t i = 0; i < sizeof(freq) / 4; ++i) freq[i] = lane + i * WAVE < rot / 2 ? p.freqs[lane + i * WAVE] : 0.0f;

    typedef std::conditional_t<CODES, half8, bf16x8> operand;
    operand qb[DB][CODES ? 2 : 3];
    float qpow = 1.0f;               // 4-bit rows: head c16's power of two, taken out of its queries
    float slope = 0.0f;              // of head c16
    uint32_t turned = NOWHERE;
    // raw to the three-term B operands: norm, rotation at len - 1, scale.
    // `spare` holds 16 rows in LDS, element d of row r at d ^ 4 (r % 8), so that
    // a column of them is spread over the banks
    auto prepare = [&](const Slab& s, float* spare) {
        const DecodeArgs& a = cold();
        const PagedDecodeParams& p = a.p;
        const int lane = fresh_lane(threadIdx.x & 63), g = lane >> 4, c16 = lane & 15;
        const uint32_t group = s.pair % a.groups;
        const bool live = uint32_t(c16) < a.perGroup && group * a.perGroup + c16 < G;
        float x[DB][8];
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                uint32_t bits;
                if constexpr (BF) bits = e & 1 ? raw[db][0][e / 2] & 0xFFFF0000u : raw[db][0][e / 2] << 16;
                else bits = raw[db][e / 4][e % 4];
                x[db][e] = live ? __uint_as_float(bits) : 0.0f;
            }
        if (p.gamma) {
            float ss = 0.0f;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int e = 0; e < 8; ++e) ss += x[db][e] * x[db][e];
            ss += __shfl_xor(ss, 16, WAVE);
            ss += __shfl_xor(ss, 32, WAVE);
            const float inv = 1.0f / sqrtf(ss / float(D) + p.eps);
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int e = 0; e < 8; ++e) x[db][e] = x[db][e] * inv * gamma[first_at(g) + STEP * db + e];
        }
        if (rot) {
            const uint32_t half = rot / 2;
            if (turned != s.b) {
                wave_sync();
#pragma unroll
                for (uint32_t i = 0; i < sizeof(freq) / 4; ++i) {
                    float cs, sn;
                    rotation_at(s.len - 1, freq[i], cs, sn);
                    if (lane + i * WAVE < half) turns[w][lane + i * WAVE] = float2{cs * p.amplitude, sn * p.amplitude};
                }
                turned = s.b;
            }
            wave_sync();
            if (p.interleaved) {
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const uint32_t d = first_at(g) + STEP * db + e;
                        const float2 cs = turns[w][d / 2];
                        const float u = x[db][e], v = x[db][e + 1];
                        x[db][e] = d < rot ? u * cs.x - v * cs.y : u;
                        x[db][e + 1] = d < rot ? v * cs.x + u * cs.y : v;
                    }
            } else if (CODES && half == D / 2) {
                // the partner is that of the lane two quarters on
                const int d0 = first_at(g & 1);
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float2 cs = turns[w][d0 + 8 * db + e];
                        const float other = __shfl_xor(x[db][e], 32, WAVE);
                        x[db][e] = x[db][e] * cs.x + (g < 2 ? -other : other) * cs.y;
                    }
            } else if (!CODES && DB % 2 == 0 && half == D / 2) {
                // the partner D / 2 elements on is this lane's too
#pragma unroll
                for (int db = 0; db < DB / 2; ++db)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float2 cs = turns[w][32 * db + 8 * g + e];
                        const float u = x[db][e], v = x[db + DB / 2][e];
                        x[db][e] = u * cs.x - v * cs.y;
                        x[db + DB / 2][e] = v * cs.x + u * cs.y;
                    }
            } else {
                // elsewhere it is another lane's: through LDS (whose reads wait
                // for the values on their way there)
                const int sw = 4 * (c16 & 7);
                float* row = spare + c16 * D;
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        *reinterpret_cast<floatx4*>(row + ((first_at(g) + STEP * db + 4 * i) ^ sw)) =
                            floatx4{x[db][4 * i], x[db][4 * i + 1], x[db][4 * i + 2], x[db][4 * i + 3]};
                wave_sync();
#pragma unroll 8
                for (uint32_t j = g; j < half; j += 4) {      // the row's pairs, a quarter a lane
                    float* u = row + (j ^ sw);
                    float* v = row + ((j + half) ^ sw);
                    const float2 cs = turns[w][j];
                    const float xu = *u, xv = *v;
                    *u = xu * cs.x - xv * cs.y;
                    *v = xv * cs.x + xu * cs.y;
                }
                wave_sync();
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const floatx4 y = *reinterpret_cast<const floatx4*>(row + ((first_at(g) + STEP * db + 4 * i) ^ sw));
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[db][4 * i + e] = y[e];
                    }
                wave_sync();
            }
        }
        if constexpr (scored(FORM)) {
            if (p.slopes) slope = p.slopes[s.pair / a.groups * G + (live ? group * a.perGroup + c16 : 0)] * LOG2E;
        }
        if constexpr (CODES) {
            // fp32 as two fp16 terms of 11 bits each (what is left, 2^-23 of the value, is
            // below the products' fp32), the largest element brought to 2^13 .. 2^14, so
            // that the second term of small ones stays above fp16's least
            float top = 0.0f;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(x[db][e] *= a.scaleLog2));
            top = fmaxf(top, __shfl_xor(top, 16, WAVE));
            top = fmaxf(top, __shfl_xor(top, 32, WAVE));
            int power = 14 - __builtin_amdgcn_frexp_expf(top);
            power = power > 100 ? 100 : power;       // -114 for fp32's largest
            const float up = ldexpf(1.0f, power);
            qpow = ldexpf(1.0f, -power);
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                u32x4 hi, lo;
#pragma unroll
                for (int i = 0; i < 4; ++i) {    // elements i and i + 4, as the codes are unpacked
                    const u32x2 t = split_f16(x[db][i] * up, x[db][i + 4] * up);
                    hi[i] = t[0];
                    lo[i] = t[1];
                }
                qb[db][0] = __builtin_bit_cast(half8, hi);
                qb[db][1] = __builtin_bit_cast(half8, lo);
            }
        } else {
#pragma unroll
            for (int db = 0; db < DB; ++db) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[db][e] *= a.scaleLog2;
                u32x4 t[3];
                split3(x[db], t);
#pragma unroll
                for (int k = 0; k < 3; ++k) qb[db][k] = __builtin_bit_cast(bf16x8, t[k]);
            }
        }
    };

    float m = -INFINITY, l = 0.0f;   // of head c16; l of this lane's positions
    floatx4 acc[CT];                 // [tile][r]: head 4 g + r, column 16 tile + c16
    bool bad = false, begun = false;
    float sv[KRB][4];                // scores: of head c16 at positions 16 rb + 4 g + i
    float svBy = 1.0f;
    auto score = [&](const Slab& s) {
        const Unpack unpack;
        const int lane = fresh_lane(threadIdx.x & 63), g = lane >> 4, c16 = lane & 15;
#pragma unroll
        for (int rb = 0; rb < KRB; ++rb) {
            floatx4 sc = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (CODES) {
                const uint16_t* scales = kscales[w] + (16 * rb + c16) * DB;
                half2v by = {}, off = {};
#pragma unroll
                for (int db = 0; db < DB; ++db) {
                    // word g DB + db of the row, of block (g DB + db) / 4
                    if (db == 0 || (DB % 4 == 0 ? db % 4 == 0 : DB != 2)) by = scale_of(scales[(g * DB + db) / 4], off);
                    const half8 k = values_of(unpack, kr[rb][db / 4][db % 4], by, off);
                    sc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qb[db][1], sc, 0, 0, 0);
                    sc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qb[db][0], sc, 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int k = 2; k >= 0; --k)
#pragma unroll
                    for (int db = 0; db < DB; ++db)
                        sc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kr[rb][db]), qb[db][k],
                                                                     sc, 0, 0, 0);
            }
            if constexpr (CODES) {
#pragma unroll
                for (int i = 0; i < 4; ++i) sv[rb][i] = sc[i];
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t pos = s.pos + 16 * rb + 4 * g + i;
                    float x = sc[i];
                    if constexpr (scored(FORM)) {
                        if (a.capLog2 != 0.0f) x = a.capLog2 * tanh_of(x);
                        if (p.slopes) x -= slope * float(s.len - 1 - pos);
                    }
                    sv[rb][i] = pos >= s.first && pos < s.len ? x : -INFINITY;
                }
            }
        }
        if constexpr (CODES) {
            svBy = qpow;             // what takes sv to scores: left to the exponentials where nothing comes between
            if (a.capLog2 != 0.0f || p.slopes) {
                svBy = 1.0f;
                const float apart = float(s.len - 1 - s.pos - 4 * g);
#pragma unroll
                for (int i = 0; i < 16; ++i) sv[i >> 2][i & 3] *= qpow;
                if (a.capLog2 != 0.0f) {
                    float most = 0.0f;
#pragma unroll
                    for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(sv[i >> 2][i & 3]));
                    if (__all(most <= TANH_WITHIN)) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float x = sv[i >> 2][i & 3];
                            sv[i >> 2][i & 3] = x * tanh_series<6>(x * x, a.series);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) sv[i >> 2][i & 3] = a.capLog2 * tanh_of(sv[i >> 2][i & 3]);
                    }
                }
                if (p.slopes) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) sv[i >> 2][i & 3] -= slope * (apart - float(16 * (i >> 2) + (i & 3)));
                }
            }
            if (s.pos < s.first || s.pos + SLAB > s.len) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const uint32_t pos = s.pos + 16 * (i >> 2) + 4 * g + (i & 3);
                    sv[i >> 2][i & 3] = pos >= s.first && pos < s.len ? sv[i >> 2][i & 3] : -INFINITY;
                }
            }
        }
    };
    auto weigh = [&](int bufHalf, bool nextInFlight) {
        const int lane = fresh_lane(threadIdx.x & 63), g = lane >> 4, c16 = lane & 15;
        if constexpr (CODES) {
            const Unpack unpack;
            float top = sv[0][0];
#pragma unroll
            for (int i = 1; i < 16; ++i) top = fmaxf(top, sv[i >> 2][i & 3]);
            top = over_groups(top) * svBy;
            // Weights, 1 at most, are taken times 2^15: their terms are whole numbers of 2^-24, so
            // that a weight is off by its 22 bits or by 2^-40 of the largest, which many small ones
            // add up to no more than fp32's own roundings do. (As part of the exponent, 15 would take
            // four bits of its argument: results 1.25 times as far from float64. Raising the maximum
            // only by 2^8 at a time, which leaves 2^-31, takes the same times.)
            constexpr float UP = 0x1p15f;
            const bool grow = top > m;
            const float next = grow ? top : m;
            if (__any(grow)) {
                const float keep = grow ? __builtin_amdgcn_exp2f(m - next) : 1.0f;
                l *= keep;
                float rk[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) rk[r] = __shfl(keep, 4 * g + r, WAVE);
#pragma unroll
                for (int t = 0; t < CT; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[t][r] *= rk[r];
            }
            // (the accumulators stay where they are on both ways here)
#pragma unroll
            for (int t = 0; t < CT; ++t) asm("" : "+v"(acc[t]));
            m = next;
            const float base = next == -INFINITY ? 0.0f : next;
            float pv[16], sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                pv[i] = __builtin_amdgcn_exp2f(fmaf(sv[i >> 2][i & 3], svBy, -base));
                sum += pv[i];
            }
            l = fmaf(sum, UP, l);
            u32x4 hi[2], lo[2];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const u32x2 t = split_f16(pv[8 * h + i], pv[8 * h + 4 + i], UP);
                    hi[h][i] = t[0];
                    lo[h][i] = t[1];
                }
            // lane c16 of group g gets element 16 t + c16 of the 16 rows 16 rb + 4 g + i
            const int row = 16 * (c16 >> 2) + 4 * g + (c16 & 3);
            const uint16_t* codes = vbuf[w][0] + row * DB * 8;
#pragma unroll
            for (int b = 0; b < DB; ++b) {           // a block's two tiles of 16 columns
                u32x2 col[2];
#pragma unroll
                for (int t = 0; t < 2; ++t) col[t] = read_codes(codes + (b ^ code_swizzle<D>(row)) * 8 + 4 * t);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    half2v by[4], off[4];
                    scales_of(*reinterpret_cast<const u32x4*>(vscales[w] + (b * 2 + h) * 16 + 4 * g), by, off);
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const half8 v = values_of(unpack, col[t][h], by, off);
                        floatx4& x = acc[2 * b + t];
                        x = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, lo[h]), v, x, 0, 0, 0);
                        x = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, hi[h]), v, x, 0, 0, 0);
                    }
                }
            }
            return;
        }
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, sv[i >> 2][i & 3]);
        top = fmaxf(top, __shfl_xor(top, 16, WAVE));
        top = fmaxf(top, __shfl_xor(top, 32, WAVE));
        const float next = fmaxf(m, top), base = next == -INFINITY ? 0.0f : next;
        const float keep = exp2f(m - base);
        float pv[8], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            pv[i] = exp2f(sv[i >> 2][i & 3] - base);
            sum += pv[i];
        }
        l = l * keep + sum;
        m = next;
        float rk[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) rk[r] = __shfl(keep, 4 * g + r, WAVE);
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[t][r] *= rk[r];
        u32x4 pa[3];
        split3(pv, pa);
        // this slab's values have landed: at most the next slab's loads are out
        if (nextInFlight) wait_loads<2 * DB + VLOADS>();
        else wait_loads<0>();
        wave_sync();
        // lane c16 of group g gets column 16 t + c16 of rows 4 g + 0..3, then 16 + 4 g + 0..3
        const uint16_t* vs = vbuf[w][bufHalf];
        const int r0 = 4 * g + (c16 >> 2), r1 = r0 + 16, x0 = (c16 >> 1) & 1, sub = 4 * (c16 & 1);
        constexpr int BATCH = CT % 4 == 0 ? 4 : 2;       // tiles whose reads go out together
#pragma unroll
        for (int t0 = 0; t0 < CT; t0 += BATCH) {
            bf16v4 lo[BATCH], hi[BATCH];
#pragma unroll
            for (int t = 0; t < BATCH; ++t) {
                const int x = 2 * (t0 + t) + x0;
                lo[t] = read_transposed(vs + r0 * D + 8 * (x ^ value_swizzle<D>(r0)) + sub);
                hi[t] = read_transposed(vs + r1 * D + 8 * (x ^ value_swizzle<D>(r1)) + sub);
            }
#pragma unroll
            for (int k = 2; k >= 0; --k)
#pragma unroll
                for (int t = 0; t < BATCH; ++t)
                    acc[t0 + t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                        __builtin_bit_cast(bf16x8, pa[k]), __builtin_shufflevector(lo[t], hi[t], 0, 1, 2, 3, 4, 5, 6, 7),
                        acc[t0 + t], 0, 0, 0);
        }
    };
    // a pair's last slab of this run: the sum over lanes, then its output or,
    // where other runs have parts of it, a record (the run's last stays in the
    // registers, for the workgroup's join)
    const auto records = buffer_of(a.records);
    auto piece_of = [&](const Slab& s) {
        const DecodeArgs& a = cold();
        const PagedDecodeParams& p = a.p;
        const uint32_t h0 = s.pair % a.groups * a.perGroup, units = slabs_of<SLAB>(p, s.len) + OPENING;
        const uint32_t begin = uniform(pre[s.b]) + s.pair * units;
        return Piece{begin, begin + units, s.b, s.pair / a.groups * G + h0,
                     a.perGroup < G - h0 ? a.perGroup : G - h0};
    };
    auto finish = [&](const Slab& s, bool last) {
        const DecodeArgs& a = cold();
        const PagedDecodeParams& p = a.p;
        const int lane = fresh_lane(threadIdx.x & 63), g = lane >> 4, c16 = lane & 15;
        l += __shfl_xor(l, 16, WAVE);
        l += __shfl_xor(l, 32, WAVE);
        if (bad) l = __builtin_nanf("");
        const bool whole = begun && (s.is & ENDS);
        if (last && !whole) return;
        const Piece piece = piece_of(s);
        const uint32_t rows = piece.rows;
        if (!whole) {
            const auto records = buffer_of(a.records);
            const uint32_t rec = run * 2 * record_floats(a.perGroup, D);
            auto put = [&](uint32_t at, float x) {
                __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x), records, (rec + at) * 4, 0, PAST_L2);
            };
            if (g == 0 && uint32_t(c16) < rows) {
                put(c16, m);
                put(a.perGroup + c16, l);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (4 * g + r < rows) {
#pragma unroll
                    for (int t = 0; t < CT; ++t)
                        put(record_heads(a.perGroup) + (4 * g + r) * D + 16 * t + c16, acc[t][r]);
                }
            if (lane == 0) pieces[w] = piece;
            return;
        }
        float* to = p.out + (size_t(s.b) * p.heads + piece.head) * D;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint32_t row = 4 * g + r;
            const float by = 1.0f / __shfl(l, row, WAVE);
            if (row < rows) {
#pragma unroll
                for (int t = 0; t < CT; ++t) to[row * D + 16 * t + c16] = acc[t][r] * by;
            }
        }
        if (p.outputGate) {
#pragma unroll 1
            for (uint32_t i = c16; i < 4 * D; i += 16) {      // this lane's own elements again
                const uint32_t row = 4 * g + i / D, d = i % D;
                if (row < rows) to[row * D + d] = gated(p, s.b, piece.head + row, d, to[row * D + d]);
            }
        }
    };

    // ---- the pipeline ----
    Slab s0{}, s1{}, s2{};           // computed, in flight, its pages asked for
    Rows r0{}, r1{}, r2{};
    bool ok0 = true;
    const bool any = list(s0);
    bool more = false, moreThen = false;
    if (any) {
        find(s0, r0);
        more = list(s1);
        if (more) find(s1, r1);
        ask(s0);
        ok0 = issue(s0.pair, r0, 0);
        if constexpr (CODES) issue_keys();
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll 1
    for (int buf = 0; any; buf ^= 1) {
        wave_sync();                 // the other buffer's reads are done
        if (s0.is & OPENS) {
            prepare(s0, reinterpret_cast<float*>(vbuf[w][CODES ? 0 : buf ^ 1]));
            m = -INFINITY;
            l = 0.0f;
#pragma unroll
            for (int t = 0; t < CT; ++t) acc[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
            bad = false;
            begun = s0.is & BEGINS;
        }
        bad |= !ok0;
        auto ahead = [&] {
            if (more) {
                moreThen = list(s2);
                if (moreThen) find(s2, r2);
                if (s1.is & OPENS) ask(s1);
                if constexpr (!CODES) ok0 = issue(s1.pair, r1, buf ^ 1);
            }
            // after the last slab this one's rows are asked for again: were there a way on which
            // nothing is asked for, the wait for the keys, counted for all ways, would be one for
            // the next slab's values too
            if constexpr (CODES) {
                const uint32_t pair = more ? s1.pair : s0.pair;
                ok0 = issue(pair, Rows{more ? r1.page : r0.page, more ? r1.row : r0.row}, 0);
            }
        };
        if constexpr (CODES) {
            stage();
            __builtin_amdgcn_sched_barrier(0);
            ahead();
            __builtin_amdgcn_sched_barrier(0);
            score(s0);
            __builtin_amdgcn_sched_barrier(0);
            issue_keys();
        } else {
            score(s0);
            __builtin_amdgcn_sched_barrier(0);
            ahead();
        }
        __builtin_amdgcn_sched_barrier(0);
        weigh(buf, more);
        if (s0.is & CLOSES) finish(s0, !more);
        if (!more) break;
        s0 = s1;
        s1 = s2;
        if constexpr (CODES) r0 = r1;
        r1 = r2;
        more = moreThen;
    }

    // ---- the runs' open ends, joined over the workgroup ----
    const bool open = any && !(begun && (s0.is & ENDS));
    if (lane == 0) {
        if (open) pieces[WAVES + w] = piece_of(s0);
        leftEnds[w] = (begun ? 1u : 0u) | (s0.is & ENDS ? 2u : 0u);
    }
    if (open) {
        const int g = lane >> 4, c16 = lane & 15;
        if (g == 0) wm[w][c16] = m, wl[w][c16] = l;
        float* rows = reinterpret_cast<float*>(vbuf[w]);
        wave_sync();
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) rows[(4 * g + r) * D + 16 * t + c16] = acc[t][r];
    }
    __syncthreads();
    const Piece* open_ends = pieces + WAVES;
    bool recorded[WAVES] = {};       // open_ends[w] leads a record of the workgroup's
#pragma unroll
    for (int from = 0; from < WAVES; ++from) {
        const uint32_t id = uniform(open_ends[from].begin);
        if (id == NOWHERE || (from && uniform(open_ends[from - 1].begin) == id)) continue;
        int to = from + 1;
        while (to < WAVES && uniform(open_ends[to].begin) == id) ++to;
        const bool whole = uniform((leftEnds[from] & 1) && (leftEnds[to - 1] & 2));
        recorded[from] = !whole;
        const uint32_t b = uniform(open_ends[from].b), head = uniform(open_ends[from].head),
                       rows = uniform(open_ends[from].rows);
        const uint32_t rec = ((blockIdx.x * WAVES + from) * 2 + 1) * record_floats(a.perGroup, D);
        if (threadIdx.x < rows) {    // each wave's factor, and the sum
            const uint32_t row = threadIdx.x;
            float top = -INFINITY, sum = 0.0f;
            for (int k = from; k < to; ++k) top = fmaxf(top, wm[k][row]);
            const float base = top == -INFINITY ? 0.0f : top;
            for (int k = from; k < to; ++k) {
                const float f = exp2f(wm[k][row] - base);
                sum += wl[k][row] * f;
                wm[k][row] = f;
            }
            total[row] = sum;
            if (!whole) {
                __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(top), records, (rec + row) * 4, 0, PAST_L2);
                __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(sum), records, (rec + a.perGroup + row) * 4, 0,
                                                      PAST_L2);
            }
        }
        __syncthreads();
#pragma unroll 1
        for (uint32_t i = threadIdx.x; i < rows * (D / 4); i += THREADS) {
            const uint32_t row = i / (D / 4), d = i % (D / 4) * 4;
            floatx4 x = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < WAVES; ++k)
                if (k >= from && k < to)
                    x += *reinterpret_cast<const floatx4*>(reinterpret_cast<const float*>(vbuf[k]) + 4 * i) * wm[k][row];
            if (whole) {
                const float by = 1.0f / total[row];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    p.out[(size_t(b) * p.heads + head + row) * D + d + e] = gated(p, b, head + row, d + e, x[e] * by);
            } else {
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), records,
                                                       (rec + record_heads(a.perGroup) + 4 * i) * 4, 0, PAST_L2);
            }
        }
        __syncthreads();             // total and the factors are read
    }
    if (a.plan) return;

    // ---- pairs that span workgroups: the last one to arrive joins them ----
    wait_loads<0>();                 // this wave's records are out
    __syncthreads();
    bool mine = false;
    Parts parts{};
    if (threadIdx.x < 2 * WAVES) {
        const Piece& piece = pieces[threadIdx.x];
        bool counts = piece.begin != NOWHERE;
#pragma unroll
        for (int k = 0; k < WAVES; ++k)
            if (threadIdx.x == WAVES + k) counts = recorded[k];
        if (counts) {
            parts = Parts(cut, piece.begin, piece.end);
            uint32_t* arrived = a.arrived + parts.to;
            const uint32_t before = __hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            mine = before + 1 == parts.total;
            if (mine) __hip_atomic_store(arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        joins[threadIdx.x] = mine ? parts : Parts{};
    }
    const int count = __syncthreads_count(mine);
    if (count == 0) return;
    // several, of no more columns than a wave takes at once: a wave each
    const bool apart = count > 1 && a.perGroup * (D / 4) <= WAVE;
#pragma unroll 1
    for (int k = apart ? w : 0; k < 2 * WAVES; k += apart ? WAVES : 1) {
        if (uniform(joins[k].total) == 0) continue;
        const Piece& piece = pieces[k];
        join_parts<D, 8>(a, joins[k], piece.b, piece.head, 0, piece.rows, apart,
                      reinterpret_cast<float*>(vbuf[apart ? w : 0]));
    }
}

/* joins the records of one (sequence, query head) a workgroup */
template <int D>
__global__ __launch_bounds__(THREADS) void paged_merge_kernel(DecodeArgs a, uint32_t runs) {
    __shared__ __attribute__((aligned(16))) float room[THREADS * JOIN_FLOATS];
    const PagedDecodeParams& p = a.p;
    const uint32_t b = blockIdx.x / p.heads, head = blockIdx.x % p.heads, G = p.heads / p.c.kvHeads;
    const uint32_t pairs = p.c.kvHeads * a.groups, pair = head / G * a.groups + head % G / a.perGroup;
    const uint32_t before = a.plan[b], units = (a.plan[b + 1] - before) / pairs;
    if (units == 0) return;
    const uint32_t begin = before + pair * units;
    const Parts parts(Cut(a.plan[p.c.batch], runs), begin, begin + units);
    if (parts.total > 1) join_parts<D, 16>(a, parts, b, head, head % G % a.perGroup, 1, false, room);
}

/* how a decode is launched */
struct DecodeShape {
    uint32_t groups, perGroup;       // of a kv head's query heads
    uint32_t slice;                  // sequences of a launch; 0: one is too much
    uint32_t grid;
};

/* the workgroups that the chip holds at once */
uint32_t full_grid(uint32_t dim, int form) {
    const int cus = Context::instance().cus ? Context::instance().cus : 256;
    return std::min(uint32_t(cus) * occupancy(int(dim), form), MAX_RUNS / WAVES);
}

DecodeShape decode_shape(const PagedDecodeParams& p) {
    DecodeShape s{};
    const uint32_t G = p.heads / p.c.kvHeads;
    s.groups = (G + ROWS - 1) / ROWS;
    s.perGroup = (G + s.groups - 1) / s.groups;
    const uint64_t SLAB = slab_rows(p.form);
    uint64_t slabs = (uint64_t(p.maxLength) + SLAB - 1) / SLAB;
    if (p.window && p.window / SLAB + 2 < slabs) slabs = p.window / SLAB + 2;
    const uint64_t each = (slabs + OPENING) * p.c.kvHeads * s.groups, most = uint64_t(1) << 31;   // units are counted in 32 bits
    uint64_t slice = p.c.batch < MAXB ? p.c.batch : MAXB;
    if (each && slice > most / each) slice = most / each;
    s.slice = uint32_t(slice);
    const uint64_t want = (slice * each + WAVES - 1) / WAVES, fills = full_grid(p.c.dim, p.form);
    s.grid = uint32_t(want < fills ? (want ? want : 1) : fills);
    return s;
}

// A pair's records that one workgroup joins within the attention's launch; past
// it, a workgroup a query head of a second launch. At 133 KB (131072 positions,
// 8 x 4 heads of 128) joining within takes 113 us in all, the second launch 109;
// at 33 KB (4096 positions, 8 x 2 heads) both 16; with few records of many pairs
// (256 sequences of 1 to 700, 4 KB) 78 against 92, most of whose workgroups find
// nothing to join. The host does not know the lengths, so the records are counted
// as if all places held as many positions. One long sequence among short or empty
// places leaves more than that, which one workgroup then reads alone: 131072
// positions under 16/1 heads of 256 take 197 us among 127 empty places and 44 by
// themselves, under 32/4 heads of 128 among 15 places 73 and 59.
constexpr uint64_t JOIN_BYTES = 64 << 10;
bool joins_in_kernel(const PagedDecodeParams& p, const DecodeShape& s, uint32_t batch) {
    const uint64_t parts = s.grid / (uint64_t(batch) * p.c.kvHeads * s.groups) + 1;
    return parts * s.perGroup * p.c.dim * sizeof(float) <= JOIN_BYTES;
}

// workspace: a place for arrivals that no call's records overlap, the plan, the records
constexpr size_t ARRIVED_BYTES = MAX_RUNS * 4, PLAN_BYTES = (MAXB + 1) * 4 + 252 & ~size_t(255);
size_t workspace_of(uint32_t grid, uint32_t perGroup, uint32_t dim) {
    return ARRIVED_BYTES + PLAN_BYTES + size_t(grid) * WAVES * 2 * record_floats(perGroup, dim) * sizeof(float);
}

/* one of the forms, launched */
template <int FORM>
bool launch_decode_as(const char* name, const PagedDecodeParams& p, void* work, hipStream_t stream) {
    Context& ctx = Context::instance();
    if (p.c.batch == 0) return true;
    const DecodeShape s = decode_shape(p);
    DecodeArgs a{};
    a.p = p;
    a.arrived = static_cast<uint32_t*>(work);
    a.records = reinterpret_cast<float*>(static_cast<char*>(work) + ARRIVED_BYTES + PLAN_BYTES);
    a.groups = s.groups;
    a.perGroup = s.perGroup;
    a.capLog2 = scored(FORM) ? p.cap * LOG2E : 0.0f;
    a.scaleLog2 = a.capLog2 != 0.0f ? p.scale / p.cap : p.scale * LOG2E;
    for (int i = 0; i < 6; ++i) a.series[i] = float(TANH6[i] * a.capLog2);
    // division by multiplication, exact below 2^31: the least power of two that holds the
    // page, and 2^31 times it over the page
    uint32_t log = 0;
    while ((uint64_t(1) << log) < p.c.pageSize) ++log;
    a.pageShift = 31 + log;
    a.pageMagic = uint32_t((uint64_t(1) << a.pageShift) / p.c.pageSize + 1);
    const size_t es = p.inType == 1 ? 2 : 4;
    a.wideQ = (reinterpret_cast<uintptr_t>(p.q) & 15) == 0 && (p.heads == 1 || p.qStride % (16 / es) == 0) &&
              (p.c.batch == 1 || p.qTokenStride % (16 / es) == 0);
    for (uint32_t b0 = 0; b0 < p.c.batch; b0 += s.slice) {
        a.p.c.batch = p.c.batch - b0 < s.slice ? p.c.batch - b0 : s.slice;
        a.p.c.table = p.c.table + b0 * p.c.tableStride;
        a.p.c.lengths = p.c.lengths + b0;
        a.p.q = static_cast<const char*>(p.q) + b0 * p.qTokenStride * es;
        a.p.out = p.out + size_t(b0) * p.heads * p.c.dim;
        a.plan = joins_in_kernel(p, s, a.p.c.batch)
                     ? nullptr
                     : reinterpret_cast<uint32_t*>(static_cast<char*>(work) + ARRIVED_BYTES);
        auto go = [&](auto attention, auto merge) {
            return ctx.launch(name, stream, [&] {
                       hipLaunchKernelGGL(attention, dim3(s.grid), dim3(THREADS), 0, stream, a);
                   }) &&
                   (!a.plan || ctx.launch("paged_merge_kernel", stream, [&] {
                       hipLaunchKernelGGL(merge, dim3(a.p.c.batch * p.heads), dim3(THREADS), 0, stream, a,
                                          s.grid * WAVES);
                   }));
        };
        bool ok = false;
        auto of = [&](auto dim) {
            constexpr int D = decltype(dim)::value;
            ok = p.inType == 1 ? go(paged_attention_kernel<D, true, FORM>, paged_merge_kernel<D>)
                               : go(paged_attention_kernel<D, false, FORM>, paged_merge_kernel<D>);
        };
        switch (p.c.dim) {
            case 64: of(std::integral_constant<int, 64>{}); break;
            case 96: of(std::integral_constant<int, 96>{}); break;
            case 128: of(std::integral_constant<int, 128>{}); break;
            case 192: of(std::integral_constant<int, 192>{}); break;
            default: of(std::integral_constant<int, 256>{}); break;
        }
        if (!ok) return false;
    }
    return true;
}

} // namespace

} // namespace aigpu

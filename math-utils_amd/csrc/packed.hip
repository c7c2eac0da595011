// packed.hip - attention of many documents' tokens in one call: a document mask, scores
// capped or biased, a prefix that all of a document's tokens see, a window.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "context.hpp"
#include "device.hpp"
#include "kernels.hpp"

namespace aigpu {

namespace {

/*
    A row of work is a (token, query head) of one document and kv head: the G heads of a
    token lie next to each other, so that the heads which share keys share their loads. A
    workgroup takes ROWS_WG = 128 consecutive rows, a wave 32 of them, and walks the keys
    that any of its rows sees in tiles of BN, two stages of LDS filled by DMA: past a tile's
    one barrier it has landed for every wave, and every wave has left the tile before, whose
    stage is then refilled. Per tile and 32 keys
      S^T = K Q^T      32 x 32 MFMA, keys as rows: a lane holds 16 keys' scores of one row
      softmax          a running maximum and sum a row, in the lane and the one 32 lanes on
      O^T += V^T P^T   the weights as they lie in the lane, V transposed out of LDS
    The rows of a key tile stand in LDS in the order that makes a lane's 16 scores two runs
    of 8 keys, which is how the second product takes them.

    bf16 in, bf16 out: the weights round to bf16, and the sum adds up the rounded ones. Next to
    the result's own rounding (1.6e-3 of it rms, 2.0e-3 with both for a prompt of 2048) a second
    term would spare little and cost 30%: 695 us in place of 535 for 8192 tokens of 128-wide
    heads. Who needs the weights whole takes fp32 out.
    bf16 in, fp32 out: the weights in three bf16 terms, whose sum they are (two
    leave 2^-16 of a weight, more than fp32's own roundings do).
    fp32 in: fp32 products (v_mfma_f32_32x32x2_f32), for which the keys' order is the plain one.

    bf16 is bounded by the matrix cores and the softmax's vector instructions, which take turns
    in a wave and overlap between the two workgroups of a CU. A causal prompt of 8192 under 32/8
    heads: heads of 64 330 to 345 us (800 to 840 TFLOP/s), 96 450 to 460 (900), 128 535 to 565
    (970 to 1030), 192 775 to 815 (1010 to 1065), 256 1050 to 1140 (965 to 1045, eight registers
    of the queries in scratch); capped 620 to 660 (835 to 885), 980 where every tile has scores
    past the series; biased 620 to 640; to fp32 865 to 915 (600 to 635; its products are double).
    fp32 is bounded by the matrix cores alone, whose products take eight times the softmax: 2048
    tokens of 64 channels 197 us (87 TFLOP/s of 154), 96 243 (106), 128 327 (105). From 96
    channels on one workgroup fits a CU, and nothing runs there while it waits at a tile's barrier.
*/
constexpr int WAVES = 4, THREADS = 64 * WAVES, ROWS_WG = 32 * WAVES;
enum Kind { BF16_OUT = 0, BF16_F32 = 1, FULL = 2 };

struct PackedArgs {
    PackedParams p;
    float* records;                  // of split keys, or null: [(slot, kv head)][split] of record floats
    uint32_t group, slots, splits;   // query heads of a kv head; 128-row slots over all documents
    uint32_t groupMagic, groupShift; // row / group = row groupMagic >> groupShift (rows below 2^31)
    float factor;                    // the product to the scores' fractions of the cap, or to units of ln 2
    float capLog2;
    float series[6];                 // capped scores in units of ln 2: s (series[0] + s^2 (series[1] + ...)) ...
    float within;                    // ... for products s up to this
    uint32_t fits;                   // tiles' rows lie within 31 bits of their first
    int wide;                        // out's rows can be written four elements at a time
};

template <int D>
constexpr uint32_t record_floats() { return ROWS_WG * (D + 2); }

__device__ __forceinline__ uint32_t scalar(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
}

/* row i of 32 in a key tile is this key: lane group g's 16 accumulators are keys 16 g + r */
__device__ __forceinline__ int key_of_row(int i) { return 16 * ((i >> 2) & 1) + 4 * (i >> 3) + (i & 3); }

/* LDS swizzles: block x of 16 bytes of a tile's row i sits at x ^ this. Keys are read a row a
   lane, values (bf16) four rows of 64 bytes at once: each in distinct banks (64 of 4 bytes). */
template <int BYTES>
__device__ __forceinline__ int key_swizzle(int i) {
    if constexpr (BYTES % 256 == 0) return i & 15;
    else if constexpr (BYTES % 128 == 0) return (i >> 1) & 7;
    else return (i >> 2) & 3;
}
template <int BYTES>
__device__ __forceinline__ int value_swizzle(int i) {
    if constexpr (BYTES % 256 == 0) return 4 * (i & 3);
    else if constexpr (BYTES % 128 == 0) return 4 * ((i >> 1) & 1);
    else return 0;
}

typedef __bf16 bf16v4 __attribute__((__vector_size__(4 * sizeof(__bf16))));
__device__ __forceinline__ bf16x8 read_transposed(const uint16_t* a0, const uint16_t* a1) {
    typedef __attribute__((address_space(3))) bf16v4 lds_bf16v4;
    const bf16v4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16v4*)(a0));
    const bf16v4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_bf16v4*)(a1));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

constexpr int series_terms(int kind) { return kind == BF16_OUT ? 4 : 6; }

/* acc plus both halves of a pair of bf16 values */
__device__ __forceinline__ float add_pair(uint32_t pair, float acc) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), __builtin_bit_cast(bf16x2, 0x3F803F80u), acc, false);
}

/* A workgroup's document and rows. Document b owns the slots from starts[b] G / 128 + b on
   (rounded down), one more than its rows may need; a slot past its rows does nothing. */
struct Work {
    uint32_t first, tokens;          // the document's tokens: q and out rows first ..
    uint32_t key0, keys;             // its keys
    int32_t shift;                   // a token's position less its number in the document
    uint32_t prefix;
    uint32_t row0, rows;             // the workgroup's first row, the document's rows
};
__device__ __forceinline__ uint32_t token_of(const PackedArgs& a, uint32_t row) {
    return uint32_t(uint64_t(row) * a.groupMagic >> a.groupShift);
}
__device__ __forceinline__ bool find_work(const PackedArgs& a, uint32_t slot, int lane, Work& x) {
    const PackedParams& p = a.p;
    uint32_t b = 0;
    uint64_t slot0 = 0;
    if (p.starts) {
        uint32_t before = 0;         // documents whose slots start at or before this one
        for (uint32_t k = 0; k < p.documents; k += WAVE) {
            const bool in = k + lane < p.documents;
            const uint64_t at = in ? uint64_t(p.starts[k + lane]) * a.group / ROWS_WG + k + lane : ~uint64_t(0);
            before += __popcll(__ballot(at <= slot));
        }
        before = scalar(before);
        if (before == 0) return false;
        b = before - 1;
        const uint32_t s0 = scalar(p.starts[b]), s1 = scalar(p.starts[b + 1]);
        slot0 = uint64_t(s0) * a.group / ROWS_WG + b;
        x.first = s0;
        x.tokens = s1 > s0 && s1 <= p.count ? s1 - s0 : 0;
        x.key0 = s0;
        x.keys = x.tokens;
    } else {
        x.first = x.key0 = 0;
        x.tokens = p.count;
        x.keys = p.keyCount;
    }
    if (p.keyStarts) {
        const uint32_t s0 = scalar(p.keyStarts[b]), s1 = scalar(p.keyStarts[b + 1]);
        x.key0 = s0;
        x.keys = s1 > s0 && s1 <= p.keyCount ? s1 - s0 : 0;
    }
    x.prefix = p.prefix ? scalar(p.prefix[b]) : 0;
    x.prefix = x.prefix < x.keys ? x.prefix : x.keys;
    x.shift = int32_t(x.keys) - int32_t(x.tokens);
    x.rows = x.tokens * a.group;
    x.row0 = uint32_t(slot - slot0) * ROWS_WG;
    return slot - slot0 < (x.rows + ROWS_WG - 1) / ROWS_WG;
}

/* What a row's weighted values are multiplied by for its weights' sum l. A token sees its own
   position, if that is not before its keys, and the prefix: zeros where that is nothing. Scores
   that are all -infinity leave no weights: NaN, as in the paged decode. */
__device__ __forceinline__ float share_of(const Work& x, uint32_t token, float l) {
    if (x.shift + int32_t(token) < 0 && x.prefix == 0) return 0.0f;
    return l == 0.0f ? NAN : 1.0f / l;
}

/* whether a value's bits (two bf16 or one fp32) are not all finite: an exponent of ones */
template <bool BF>
__device__ __forceinline__ uint32_t unbounded(uint32_t x) {
    constexpr uint32_t EXPONENT = BF ? 0x7F807F80u : 0x7F800000u, ONE = BF ? 0x00800080u : 0x00800000u;
    return ((x & EXPONENT) + ONE) & (BF ? 0x80008000u : 0x80000000u);
}

/* the same bits with zeros for the values that are not finite */
template <bool BF>
__device__ __forceinline__ uint32_t bounded(uint32_t x) {
    return x & ~((unbounded<BF>(x) >> (BF ? 15 : 31)) * (BF ? 0xFFFFu : 0xFFFFFFFFu));
}

/* four elements of a row of values */
__device__ __forceinline__ void get4(const uint16_t* at, float (&x)[4]) {
    const u32x2 two = *reinterpret_cast<const u32x2*>(at);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(i & 1 ? two[i / 2] & 0xFFFF0000u : two[i / 2] << 16);
}
__device__ __forceinline__ void get4(const float* at, float (&x)[4]) {
    const floatx4 four = *reinterpret_cast<const floatx4*>(at);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = four[i];
}

/* four elements of an out row */
__device__ __forceinline__ void put4(const PackedArgs& a, uint64_t at, const float (&x)[4]) {
    if (a.p.outType == 1) {
        uint16_t* out = static_cast<uint16_t*>(a.p.out) + at;
        const u32x2 two = {pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])};
        if (a.wide) {
            *reinterpret_cast<u32x2*>(out) = two;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] = uint16_t(two[i / 2] >> 16 * (i & 1));
        }
    } else {
        float* out = static_cast<float*>(a.p.out) + at;
        if (a.wide) {
            *reinterpret_cast<floatx4*>(out) = floatx4{x[0], x[1], x[2], x[3]};
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] = x[i];
        }
    }
}

/* Keys of a tile and workgroups a CU: the most that LDS and registers hold for two:
   256-wide heads at one took 247 us for seven prompts of up to 3001, at two 232, and 172 once
   the tiles were asked for behind the scores */
constexpr int tile_keys(int D, int kind) { return kind == FULL ? (D <= 96 ? 64 : 32) : (D <= 128 ? 64 : 32); }
constexpr int workgroups(int D, int kind) { return D <= (kind == FULL ? 64 : 256) ? 2 : 1; }

template <int D, int KIND>
__global__ __launch_bounds__(THREADS, workgroups(D, KIND)) void packed_attention_kernel(PackedArgs a) {
    typedef std::conditional_t<KIND == FULL, float, uint16_t> elem;
    constexpr int ES = sizeof(elem), BYTES = D * ES;       // of a row
    constexpr int BN = tile_keys(D, KIND), KB = BN / 32;   // keys of a tile, their blocks of 32
    constexpr int DT = D / 32;                             // 32-wide tiles of the output
    constexpr int BPR = BYTES / 16;                        // 16-byte blocks of a row
    constexpr int BLOCKS = BN * BPR / WAVE / WAVES;        // DMA blocks (1 KB) of a wave and tile, K or V
    constexpr int QV = KIND == FULL ? D / 8 : D / 16;      // 16-byte pieces of a lane's half query
    static_assert(BN * BPR % (WAVE * WAVES) == 0 && BLOCKS * WAVE % BPR == 0, "whole rows of a tile are the waves' alike");
    // The queries of 256 do not all stay in registers: three pieces wait in what LDS is left,
    // and what the scores read back from scratch must not wait for a tile that was asked for
    // before it.
    constexpr bool LATE = D == 256 && KIND != FULL;
    typedef std::conditional_t<BN == 64, uint16_t, uint8_t> flags;  // a bit each of the BN / WAVES rows of a wave's blocks
    __shared__ __attribute__((aligned(16))) elem ktile[2][BN * D], vtile[2][BN * D];
    __shared__ __attribute__((aligned(8))) flags wild[2][WAVES];
    constexpr int HELD = LATE ? 3 : 0;                     // pieces of the queries that wait in LDS
    __shared__ u32x4 held[HELD ? HELD : 1][HELD ? THREADS : 1];
    const PackedParams& p = a.p;
    const int lane = threadIdx.x & 63, w = int(scalar(threadIdx.x >> 6)), g = lane >> 5, c = lane & 31;

    // consecutive workgroups go round the 8 XCDs: give each XCD a run of them, so that
    // the rows that share a kv head's keys share an L2, where the grid is a multiple of 8 (8 kv
    // heads always; others go round as they come). Late rows, which see most, go first.
    uint32_t id = blockIdx.x;
    if (gridDim.x % 8 == 0) id = id % 8 * (gridDim.x / 8) + id / 8;
    const uint32_t split = id % a.splits, kvh = id / a.splits / a.slots, slot = a.slots - 1 - id / a.splits % a.slots;
    Work x;
    if (!find_work(a, slot, lane, x)) return;

    // a lane's row
    struct Row {
        bool live;
        uint32_t token, head;
    };
    auto row_of = [&](int c) {
        const uint32_t row = x.row0 + 32 * w + c, held = row < x.rows ? row : x.rows - 1, token = token_of(a, held);
        return Row{row < x.rows, token, kvh * a.group + held - token * a.group};
    };
    const uint32_t token = row_of(c).token, head = row_of(c).head;
    const int32_t pos = x.shift + int32_t(token);          // negative: before every key
    const uint32_t lastRow = x.row0 + ROWS_WG - 1 < x.rows ? x.row0 + ROWS_WG - 1 : x.rows - 1;
    const int32_t pos0 = x.shift + int32_t(token_of(a, x.row0)), pos1 = x.shift + int32_t(token_of(a, lastRow));

    // the keys that any row sees: [kbeg, kend), in whole tiles from a multiple of BN on
    uint32_t kend = pos1 < 0 ? 0 : uint32_t(pos1) + 1;
    kend = kend > x.prefix ? kend : x.prefix;
    uint32_t kbeg = 0;
    if (p.window && pos0 >= 0 && uint64_t(pos0) + 1 > p.window) kbeg = uint32_t(pos0 + 1 - int64_t(p.window)) / BN * BN;
    uint32_t tiles = kend > kbeg ? (kend - kbeg + BN - 1) / BN : 0;
    if (a.splits > 1) {
        const uint32_t t0 = uint32_t(uint64_t(tiles) * split / a.splits), t1 = uint32_t(uint64_t(tiles) * (split + 1) / a.splits);
        kbeg += t0 * BN;
        tiles = t1 - t0;
    }
    // a row sees keys [lo, hi)
    int32_t hi = pos + 1;
    hi = hi > int32_t(x.prefix) ? hi : int32_t(x.prefix);
    const int32_t lo = p.window && pos >= 0 && uint64_t(pos) + 1 > p.window ? int32_t(pos + 1 - int64_t(p.window)) : 0;
    // what every row of the wave sees
    const uint32_t waveFirst = x.row0 + 32 * w < x.rows ? x.row0 + 32 * w : x.rows - 1;
    const uint32_t waveLast = waveFirst + 31 < x.rows ? waveFirst + 31 : x.rows - 1;
    const int32_t p0 = x.shift + int32_t(token_of(a, waveFirst)), p1 = x.shift + int32_t(token_of(a, waveLast));
    int32_t hi0 = p0 + 1;
    hi0 = hi0 > int32_t(x.prefix) ? hi0 : int32_t(x.prefix);
    const int32_t lo1 = p.window && p1 >= 0 && uint64_t(p1) + 1 > p.window ? int32_t(p1 + 1 - int64_t(p.window)) : 0;
    int32_t hi1 = p1 + 1;
    hi1 = hi1 > int32_t(x.prefix) ? hi1 : int32_t(x.prefix);
    const int32_t lo0 = p.window && p0 >= 0 && uint64_t(p0) + 1 > p.window ? int32_t(p0 + 1 - int64_t(p.window)) : 0;
    const bool busy = x.row0 + 32 * w < x.rows;            // the wave has rows
    // what every row of the workgroup sees
    int32_t hiAll = pos0 + 1;
    hiAll = hiAll > int32_t(x.prefix) ? hiAll : int32_t(x.prefix);
    const int32_t loAll = p.window && pos1 >= 0 && uint64_t(pos1) + 1 > p.window ? int32_t(pos1 + 1 - int64_t(p.window)) : 0;

    // the query: elements 16 db + 8 g .. of bf16, D / 2 g .. of fp32
    u32x4 q[QV - HELD];
    {
        const elem* src = static_cast<const elem*>(p.q) + (uint64_t(x.first) + token) * p.qTokenStride + head * p.qHeadStride;
#pragma unroll
        for (int i = 0; i < QV; ++i) {
            const u32x4 piece = *reinterpret_cast<const u32x4*>(src + (KIND == FULL ? D / 2 * g + 4 * i : 16 * i + 8 * g));
            if (i < QV - HELD) q[i] = piece;
            else held[i - (QV - HELD)][threadIdx.x] = piece;
        }
    }
    const float slope = p.slopes ? p.slopes[head] * LOG2E : 0.0f;

    const elem* keys = static_cast<const elem*>(p.k) + x.key0 * p.kTokenStride + kvh * p.kHeadStride;
    const elem* values = static_cast<const elem*>(p.v) + x.key0 * p.vTokenStride + kvh * p.vHeadStride;
    // Byte offsets of this lane's blocks from a tile's first row. Of 256 channels a block is two
    // rows, 2 n and 2 n + 1 of the wave's eight, and its place is found anew each time, which
    // spares registers (offsets kept in scratch are read back between the tile's blocks, and
    // each waits for those before: 1.98 ms at 8192 tokens of 32/8 heads in place of 1.17).
    static_assert(!LATE || (BLOCKS == 4 && BPR == 32 && BN == 32), "as the offsets are found");
    uint32_t koff[LATE ? 1 : BLOCKS], voff[LATE ? 1 : BLOCKS];
    if constexpr (!LATE) {
#pragma unroll
        for (int n = 0; n < BLOCKS; ++n) {
            const uint32_t i = (w * BLOCKS + n) * WAVE + lane, r = i / BPR, at = i % BPR;
            const uint32_t kr = KIND == FULL ? r : (r & ~31u) + key_of_row(r & 31);
            koff[n] = uint32_t(kr * p.kTokenStride * ES) + 16 * (at ^ key_swizzle<BYTES>(r));
            voff[n] = uint32_t(r * p.vTokenStride * ES) + 16 * (KIND == FULL ? at : at ^ value_swizzle<BYTES>(r));
        }
    }
    auto issue = [&](uint32_t k0, int stage) {
        const uint32_t kl = scalar(lds_address(ktile[stage])) + w * BLOCKS * 1024, vl = scalar(lds_address(vtile[stage])) + w * BLOCKS * 1024;
        if (a.fits && k0 + BN <= x.keys) {
            const elem* kt = keys + k0 * p.kTokenStride;
            const elem* vt = values + k0 * p.vTokenStride;
            if constexpr (LATE) {
                uint32_t at = threadIdx.x & 63;
                asm volatile("" : "+v"(at));
                const uint32_t late = at >> 5;           // of the two rows
                at = 16 * (at & 31);
                // row 8 w + 2 n + late of keys is key 4 w + 16 (n >> 1) + 2 (n & 1) + late
                const uint32_t ka = at ^ 16 * (8 * (w & 1) + late), kl0 = late * uint32_t(p.kTokenStride * ES);
                const uint32_t va = at ^ 64 * late, vl0 = late * uint32_t(p.vTokenStride * ES);
#pragma unroll
                for (int n = 0; n < BLOCKS; ++n)
                    dma_block(kt + (4 * w + 16 * (n >> 1) + 2 * (n & 1)) * p.kTokenStride, (ka ^ 32 * n) + kl0, kl + n * 1024);
#pragma unroll
                for (int n = 0; n < BLOCKS; ++n)
                    dma_block(vt + (8 * w + 2 * n) * p.vTokenStride, (va ^ 128 * (n & 1)) + vl0, vl + n * 1024);
            } else {
#pragma unroll
                for (int n = 0; n < BLOCKS; ++n) dma_block(kt, koff[n], kl + n * 1024);
#pragma unroll
                for (int n = 0; n < BLOCKS; ++n) dma_block(vt, voff[n], vl + n * 1024);
            }
            return;
        }
        // rows past the document's last key hold that one again
        uint32_t lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));
#pragma unroll
        for (int n = 0; n < BLOCKS; ++n) {
            const uint32_t i = (w * BLOCKS + n) * WAVE + lane, r = i / BPR, at = i % BPR;
            uint32_t key = k0 + (KIND == FULL ? r : (r & ~31u) + key_of_row(r & 31));
            key = key < x.keys ? key : x.keys - 1;
            dma_block(keys + key * p.kTokenStride + 16 / ES * (at ^ key_swizzle<BYTES>(r)), kl + n * 1024);
        }
#pragma unroll
        for (int n = 0; n < BLOCKS; ++n) {
            const uint32_t i = (w * BLOCKS + n) * WAVE + lane, r = i / BPR, at = i % BPR;
            uint32_t key = k0 + r;
            key = key < x.keys ? key : x.keys - 1;
            dma_block(values + key * p.vTokenStride + 16 / ES * (KIND == FULL ? at : at ^ value_swizzle<BYTES>(r)), vl + n * 1024);
        }
    };

    // A weight of 0 does not take a value that is not finite out of the product. In a tile that
    // some row does not see whole, each wave makes zeros of such elements among its own blocks',
    // notes their rows, and the rows that see them get them back by themselves: their own channels
    // alone, as in a tile that all see (1% of the time of 8192 tokens, 2% of 32 documents of
    // 1000, whose tiles are cut more often).
    auto tame = [&](int stage) {
        uint32_t at = lane;              // (its own, so that nothing of this is kept over the loop)
        asm volatile("" : "+v"(at)::"memory");
        u32x4* blocks = reinterpret_cast<u32x4*>(vtile[stage]) + w * BLOCKS * WAVE + at;
        uint32_t found = 0;
#pragma unroll
        for (int n = 0; n < BLOCKS; ++n) {
            const u32x4 x = blocks[n * WAVE];
            const uint32_t some = unbounded<KIND != FULL>(x[0]) | unbounded<KIND != FULL>(x[1]) |
                                  unbounded<KIND != FULL>(x[2]) | unbounded<KIND != FULL>(x[3]);
            if (some) found |= 1u << ((n * WAVE + at) / BPR);
        }
        if (__any(found != 0)) {
            uint32_t all = 0;
#pragma unroll 1
            for (int i = 0; i < BN / WAVES; ++i) all |= uint32_t(__any(found >> i & 1)) << i;
            found = all;
#pragma unroll 1
            for (int n = 0; n < BLOCKS; ++n)
                if (found >> ((n * WAVE + at) / BPR) & 1) {
                    u32x4 x = blocks[n * WAVE];
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = bounded<KIND != FULL>(x[i]);
                    blocks[n * WAVE] = x;
                }
        }
        if (at == 0) wild[stage][w] = flags(found);
    };

    floatx16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] = 0.0f;
    float m = -INFINITY, l = 0.0f;

    if (tiles) issue(kbeg, 0);
#pragma unroll 1
    for (uint32_t it = 0; it < tiles; ++it) {
        const uint32_t k0 = kbeg + it * BN;
        const int stage = it & 1;
        wait_vmcnt<0>();
        const bool partial = int32_t(k0 + BN) > hiAll || int32_t(k0) < loAll;
        if (partial) tame(stage);
        lds_barrier();
        const bool idle = !busy || int32_t(k0) >= hi1 || int32_t(k0 + BN) <= lo0;
        if ((!LATE || idle) && it + 1 < tiles) issue(k0 + BN, stage ^ 1);
        if (idle) continue;
        floatx16 s[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[kb][r] = 0.0f;
#pragma unroll
        for (int i = 0; i < QV; ++i)
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                const int block = KIND == FULL ? QV * g + i : 2 * i + g;
                const u32x4 k = *reinterpret_cast<const u32x4*>(ktile[stage] + (32 * kb + c) * D + 16 / ES * (block ^ key_swizzle<BYTES>(c)));
                const u32x4 qi = i < QV - HELD ? q[i] : held[i - (QV - HELD)][threadIdx.x];
                if constexpr (KIND == FULL) {
                    const floatx4 kf = __builtin_bit_cast(floatx4, k), qf = __builtin_bit_cast(floatx4, qi);
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[kb] = __builtin_amdgcn_mfma_f32_32x32x2f32(kf[j], qf[j], s[kb], 0, 0, 0);
                } else {
                    s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, k),
                                                                    __builtin_bit_cast(bf16x8, qi), s[kb], 0, 0, 0);
                }
            }
        if (LATE && it + 1 < tiles) {
            __builtin_amdgcn_sched_barrier(0);
            issue(k0 + BN, stage ^ 1);
            __builtin_amdgcn_sched_barrier(0);
        }
        // register r of block kb is key k0 + 32 kb + key(r)
        auto key = [&](int r) { return KIND == FULL ? (r & 3) + 8 * (r >> 2) + 4 * g : 16 * g + r; };
        // what takes s to units of ln 2: left to the exponentials where nothing comes between
        float by = a.factor;
        if (a.capLog2 != 0.0f) {
            float most = 0.0f;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(s[kb][r]));
            if (__all(most <= a.within)) {
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const float y = s[kb][r], t = y * y;
                        s[kb][r] = y * tanh_series<series_terms(KIND)>(t, a.series);
                    }
            } else {
                float C[6];
#pragma unroll
                for (int i = 0; i < 6; ++i) {
                    C[i] = float(TANH6[i]);
                    if constexpr (LATE) asm volatile("" : "+v"(C[i]));     // (not kept over the loop)
                }
#pragma unroll
                for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const float y = s[kb][r] * a.factor;
                        if constexpr (KIND == BF16_OUT) {
                            // tanh_of without its branch and division, which would take registers
                            const float large = 1.0f - 2.0f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(2.0f * LOG2E * fabsf(y)) + 1.0f);
                            s[kb][r] = a.capLog2 * (fabsf(y) <= TANH_WITHIN ? y * tanh_series<6>(y * y, C) : copysignf(large, y));
                        } else {
                            s[kb][r] = a.capLog2 * tanh_of(y);
                        }
                        if constexpr (LATE) __builtin_amdgcn_sched_barrier(0);   // (one after the other, for the registers)
                    }
            }
            by = 1.0f;
        }
        if (p.slopes) {
            const float apart = float(pos - int32_t(k0) - key(0));
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    s[kb][r] = fmaf(-slope, fabsf(apart - float(32 * kb + key(r) - key(0))), s[kb][r] * by);
            by = 1.0f;
        }
        if (int32_t(k0 + BN) > hi0 || int32_t(k0) < lo1) {
            const int32_t from = lo - int32_t(k0) - key(0), to = hi - int32_t(k0) - key(0);
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int32_t j = 32 * kb + key(r) - key(0);
                    s[kb][r] = j >= from && j < to ? s[kb][r] : -INFINITY;
                }
        }
        float top = s[0][0];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, s[kb][r]);
        {
            const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
            top = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1])) * by;
        }
        // weights may grow to 2^8 before the maximum is taken up anew
        const bool grow = top > m + 8.0f;
        const float next = grow ? top : m, base = next == -INFINITY ? 0.0f : next;
        const float keep = grow ? __builtin_amdgcn_exp2f(m - next) : 1.0f;
        m = next;
        if (__any(grow)) {
            l *= keep;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[dt][r] *= keep;
        }
        // (the accumulators stay where they are on both ways here)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) asm("" : "+v"(o[dt]));
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            if constexpr (KIND == FULL) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float e = __builtin_amdgcn_exp2f(fmaf(s[kb][r], by, -base));
                    l += e;
                    const float* vr = vtile[stage] + (32 * kb + key(r)) * D + c;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
                        o[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(vr[32 * dt], e, o[dt], 0, 0, 0);
                }
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    constexpr int TERMS = KIND == BF16_F32 ? 3 : 1;
                    u32x4 term[TERMS];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float e0 = __builtin_amdgcn_exp2f(fmaf(s[kb][8 * h + 2 * j], by, -base));
                        const float e1 = __builtin_amdgcn_exp2f(fmaf(s[kb][8 * h + 2 * j + 1], by, -base));
                        if constexpr (KIND == BF16_F32) {
                            l += e0 + e1;
                            float f0 = e0, f1 = e1;          // each term takes the next 8 bits
#pragma unroll
                            for (int t = 0; t < TERMS; ++t) {
                                const uint32_t u0 = __float_as_uint(f0), u1 = __float_as_uint(f1);
                                term[t][j] = __builtin_amdgcn_perm(u1, u0, 0x07060302);
                                f0 -= __uint_as_float(u0 & 0xFFFF0000u);
                                f1 -= __uint_as_float(u1 & 0xFFFF0000u);
                            }
                        } else {
                            const uint32_t both = pack_bf16(e0, e1);
                            term[0][j] = both;
                            l = add_pair(both, l);
                        }
                    }
                    // V^T rows 32 dt + c: lane q16 of each 16 addresses row 16 g + 8 h + q16 / 4, and 4 on
                    const int q16 = lane & 15, vr = 32 * kb + 16 * g + 8 * h + (q16 >> 2);
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) {
                        const int d = 32 * dt + 16 * (lane >> 4 & 1) + 4 * (q16 & 3);
                        const uint16_t* at = vtile[stage] + vr * D + 8 * ((d >> 3) ^ value_swizzle<BYTES>(vr)) + (d & 7);
                        const bf16x8 v = read_transposed(at, at + 4 * D);
#pragma unroll
                        for (int t = TERMS - 1; t >= 0; --t)
                            o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, __builtin_bit_cast(bf16x8, term[t]), o[dt], 0, 0, 0);
                    }
                }
            }
        }
        if (partial) {
            typedef std::conditional_t<BN == 64, uint64_t, uint32_t> bits;
            bits rows = *reinterpret_cast<const bits*>(wild[stage]);
            if (__any(rows != 0)) {
                int half = threadIdx.x >> 5 & 1;                 // g (its own, so that nothing of this is kept over the loop)
                asm volatile("" : "+v"(half));
#pragma unroll 1
                for (; rows; rows &= rows - 1) {
                    const int32_t at = int32_t(k0) + (BN == 64 ? __builtin_ctzll(rows) : __builtin_ctz(uint32_t(rows)));
                    if (at < lo || at >= hi) continue;
                    const elem* row = values + uint32_t(at) * p.vTokenStride + 4 * half;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float y[4];
                            get4(row + 32 * dt + 8 * i, y);
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (unbounded<false>(__float_as_uint(y[e]))) o[dt][4 * i + e] += y[e];
                            __builtin_amdgcn_sched_barrier(0);   // (one after the other, for the registers)
                        }
                }
            }
        }
    }

    l += __shfl_xor(l, 32, WAVE);
    // (found anew: over the loop it would take registers)
    int again = c;
    asm volatile("" : "+v"(again));
    const Row r0 = row_of(again);
    if (!r0.live) return;
    // register r of tile dt is element 32 dt + (r & 3) + 8 (r >> 2) + 4 g
    if (a.records) {
        float* rec = a.records + ((uint64_t(slot) * p.kvHeads + kvh) * a.splits + split) * record_floats<D>();
        const uint32_t at = 32 * w + c;
        if (g == 0) {
            rec[at] = m;
            rec[ROWS_WG + at] = l;
        }
        float* to = rec + 2 * ROWS_WG + at * D + 4 * g;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<floatx4*>(to + 32 * dt + 8 * i) =
                    floatx4{o[dt][4 * i], o[dt][4 * i + 1], o[dt][4 * i + 2], o[dt][4 * i + 3]};
        return;
    }
    const float by = share_of(x, r0.token, l);
    const uint64_t to = (uint64_t(x.first) + r0.token) * p.outTokenStride + r0.head * p.outHeadStride + 4 * g;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float y[4] = {o[dt][4 * i] * by, o[dt][4 * i + 1] * by, o[dt][4 * i + 2] * by, o[dt][4 * i + 3] * by};
            put4(a, to + 32 * dt + 8 * i, y);
        }
}

/* joins the records of the splits: a workgroup 128 rows of one kv head, a thread four
   elements of a row */
template <int D>
__global__ __launch_bounds__(THREADS) void packed_merge_kernel(PackedArgs a) {
    const PackedParams& p = a.p;
    const uint32_t slot = blockIdx.x, kvh = blockIdx.y;
    Work x;
    if (!find_work(a, slot, threadIdx.x & 63, x)) return;
    const float* rec = a.records + (uint64_t(slot) * p.kvHeads + kvh) * a.splits * record_floats<D>();
    const uint32_t unit = blockIdx.z * THREADS + threadIdx.x, r = unit / (D / 4), d = unit % (D / 4) * 4;
    if (r >= ROWS_WG || x.row0 + r >= x.rows) return;
    float m = -INFINITY;
    for (uint32_t i = 0; i < a.splits; ++i) m = fmaxf(m, rec[i * record_floats<D>() + r]);
    const float base = m == -INFINITY ? 0.0f : m;
    float l = 0.0f;
    floatx4 o = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (uint32_t i = 0; i < a.splits; ++i) {
        const float* at = rec + i * record_floats<D>();
        const float f = exp2f(at[r] - base);
        l += at[ROWS_WG + r] * f;
        o += *reinterpret_cast<const floatx4*>(at + 2 * ROWS_WG + r * D + d) * f;
    }
    const uint32_t row = x.row0 + r, token = token_of(a, row), head = kvh * a.group + row - token * a.group;
    const float by = share_of(x, token, l);
    const float y[4] = {o[0] * by, o[1] * by, o[2] * by, o[3] * by};
    put4(a, (uint64_t(x.first) + token) * p.outTokenStride + head * p.outHeadStride + d, y);
}

struct Shape { uint64_t slots, splits; };

/* Few rows over many keys leave CUs idle: their keys are split over workgroups, two a CU of
   256 (fp32 rows from 96 channels on run one after the other there), whose records a second
   launch joins. How rows and keys lie in documents only the device knows: a document is taken
   to have one slot and the average's keys, so places without tokens and one long history among
   short ones are split less than they could be. */
Shape shape_of(const PackedParams& p) {
    const uint64_t group = p.heads / p.kvHeads, full = (uint64_t(p.count) * group + ROWS_WG - 1) / ROWS_WG;
    Shape s{};
    s.slots = p.starts ? uint64_t(p.count) * group / ROWS_WG + p.documents : full;
    const uint64_t busy = std::max<uint64_t>(full, std::min(p.documents, p.count)) * p.kvHeads, want = 512;
    s.splits = 1;
    // A split of 512 keys at the least, were the documents alike: of those that a window leaves
    // a document's tokens. Us with splits and without,
    // 32/8 heads of 128, bf16 to fp32: four documents of 5 to 27 tokens behind 30011 keys 115 and
    // 865, 8 of 64 behind 2000 47 and 69, 512 behind 8000 141 and 252; 1000 alone 41.7 and 38, 512
    // alone 28 and 21, as the second launch costs what 500 keys do. Half or twice as many workgroups
    // take 148 and 122 for the first.
    if (busy && busy * 2 <= want) {
        uint64_t keys = p.keyCount / p.documents;
        if (p.window && p.window < keys) keys = std::min<uint64_t>(keys, p.window + p.count / p.documents);
        s.splits = std::max<uint64_t>(std::min<uint64_t>(want / busy, keys / 512), 1);
    }
    return s;
}

} // namespace

bool check_packed_attention(const PackedParams& p) {
    Context& ctx = Context::instance();
    if (p.dim != 64 && p.dim != 96 && p.dim != 128 && p.dim != 192 && p.dim != 256)
        return ctx.fail("packed attention: dim must be 64, 96, 128, 192 or 256");
    if (p.inType < 0 || p.outType < 0) return ctx.fail("packed attention: unknown element type");
    if (p.heads == 0 || p.kvHeads == 0 || p.heads % p.kvHeads)
        return ctx.fail("packed attention: heads must be a multiple of kvHeads");
    if (!p.starts && p.documents != 1) return ctx.fail("packed attention: without starts there is one document");
    if (!p.starts && p.keyStarts) return ctx.fail("packed attention: keyStarts without starts");
    if (p.starts && !p.keyStarts && p.keyCount != p.count)
        return ctx.fail("packed attention: without keyStarts there are as many keys as tokens");
    if (!(p.scale > 0.0f) || !std::isfinite(p.scale))
        return ctx.fail("packed attention: the scale must be positive and finite");
    if (!cap_ok(p.cap)) return ctx.fail("packed attention: the cap must be 0, or 1e-6 .. 1e6");
    if (p.cap > 0.0f && !std::isnormal(p.scale / p.cap)) return ctx.fail("packed attention: the scale does not suit the cap");
    for (uint64_t s : {p.qTokenStride, p.qHeadStride, p.kTokenStride, p.kHeadStride, p.vTokenStride, p.vHeadStride,
                       p.outTokenStride, p.outHeadStride})
        if (s >= (uint64_t(1) << 40)) return ctx.fail("packed attention: a stride is out of range");
    if (p.count == 0 || p.documents == 0) return true;
    if (!p.q || !p.out || (p.keyCount && (!p.k || !p.v))) return ctx.fail("packed attention: null tensor");
    const uint64_t es = p.inType == 1 ? 2 : 4, os = p.outType == 1 ? 2 : 4;
    const uintptr_t in = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v);
    const uint64_t strides = p.qTokenStride | p.qHeadStride | p.kTokenStride | p.kHeadStride | p.vTokenStride | p.vHeadStride;
    if ((in & 15) || strides * es % 16) return ctx.fail("packed attention: rows of q, k and v must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(p.out) & (os - 1)) return ctx.fail("packed attention: out must be aligned to its elements");
    if ((reinterpret_cast<uintptr_t>(p.starts) | reinterpret_cast<uintptr_t>(p.keyStarts) |
         reinterpret_cast<uintptr_t>(p.prefix) | reinterpret_cast<uintptr_t>(p.slopes)) & 3)
        return ctx.fail("packed attention: the vectors must be aligned to their elements");
    const uint64_t ot = p.outTokenStride, oh = p.outHeadStride, D = p.dim;
    const bool tokensApart = (p.count == 1 || ot >= (p.heads - 1) * oh + D) && (p.heads == 1 || oh >= D);
    const bool headsApart = (p.heads == 1 || oh >= (p.count - 1) * ot + D) && (p.count == 1 || ot >= D);
    if (!tokensApart && !headsApart) return ctx.fail("packed attention: the rows of out overlap");
    const Extent out{reinterpret_cast<uintptr_t>(p.out), p.count, ot * os, p.heads, oh * os, D * os};
    for (const Extent& e : {Extent{reinterpret_cast<uintptr_t>(p.q), p.count, p.qTokenStride * es, p.heads, p.qHeadStride * es, D * es},
                            Extent{reinterpret_cast<uintptr_t>(p.k), p.keyCount, p.kTokenStride * es, p.kvHeads, p.kHeadStride * es, D * es},
                            Extent{reinterpret_cast<uintptr_t>(p.v), p.keyCount, p.vTokenStride * es, p.kvHeads, p.vHeadStride * es, D * es}})
        if (may_meet(out, e)) return ctx.fail("packed attention: out overlaps q, k or v");
    const Shape s = shape_of(p);
    if (uint64_t(p.count) * (p.heads / p.kvHeads) >= (uint64_t(1) << 31) - ROWS_WG ||
        s.slots * s.splits * p.kvHeads >= (uint64_t(1) << 32) / THREADS)     // a launch's threads
        return ctx.fail("packed attention: too many rows");
    return true;
}

size_t packed_attention_workspace(const PackedParams& p) {
    if (p.count == 0 || p.documents == 0) return 0;
    const Shape s = shape_of(p);
    return s.splits > 1 ? s.slots * p.kvHeads * s.splits * ROWS_WG * (p.dim + 2) * sizeof(float) : 0;
}

bool launch_packed_attention(const PackedParams& p, void* work, hipStream_t stream) {
    Context& ctx = Context::instance();
    if (p.count == 0 || p.documents == 0) return true;
    const Shape s = shape_of(p);
    PackedArgs a{};
    a.p = p;
    a.group = p.heads / p.kvHeads;
    uint32_t log = 0;
    while ((1u << log) < a.group) ++log;
    a.groupShift = 31 + log;
    a.groupMagic = uint32_t((uint64_t(1) << a.groupShift) / a.group + 1);
    a.slots = uint32_t(s.slots);
    a.splits = uint32_t(s.splits);
    a.records = s.splits > 1 ? static_cast<float*>(work) : nullptr;
    a.capLog2 = p.cap * LOG2E;
    a.factor = p.cap > 0.0f ? p.scale / p.cap : p.scale * LOG2E;
    const int kind = p.inType != 1 ? FULL : (p.outType == 1 ? BF16_OUT : BF16_F32);
    if (p.cap > 0.0f) {
        double power = double(p.cap) * 1.4426950408889634 * a.factor;
        for (int i = 0; i < series_terms(kind); ++i, power *= double(a.factor) * a.factor)
            a.series[i] = float((kind == BF16_OUT ? TANH4[i] : TANH6[i]) * power);
        float within = TANH_WITHIN;
        // four terms are off by 7e-6 of a score: kept below 2^-10, a quarter of a weight's
        // rounding to bf16 (six terms for all: the same errors in three digits, 655 us in place of 620 at 8192)
        if (kind == BF16_OUT) within = std::min(within, 0x1p-10f / 7e-6f / p.cap);
        a.within = within / a.factor;
        // a cap far from 1 may leave terms that fp32 does not hold: then none are used
        for (int i = 0; i < series_terms(kind); ++i)
            if (!std::isnormal(a.series[i])) a.within = -1.0f;
    }
    const uint64_t es = p.inType == 1 ? 2 : 4;
    a.fits = (uint64_t(64) * (p.kTokenStride > p.vTokenStride ? p.kTokenStride : p.vTokenStride) + p.dim) * es < (uint64_t(1) << 31);
    const uint64_t piece = p.outType == 1 ? 8 : 16, os = piece / 4;
    a.wide = (reinterpret_cast<uintptr_t>(p.out) | p.outTokenStride * os | p.outHeadStride * os) % piece == 0;
    const uint32_t grid = a.slots * p.kvHeads * a.splits;
    auto of = [&](auto dim) {
        constexpr int D = decltype(dim)::value;
        auto go = [&](auto kernel) {
            return ctx.launch("packed_attention_kernel", stream, [&] {
                       hipLaunchKernelGGL(kernel, dim3(grid), dim3(THREADS), 0, stream, a);
                   }) &&
                   (!a.records || ctx.launch("packed_merge_kernel", stream, [&] {
                       hipLaunchKernelGGL(packed_merge_kernel<D>, dim3(a.slots, p.kvHeads, ROWS_WG * (D / 4) / THREADS),
                                          dim3(THREADS), 0, stream, a);
                   }));
        };
        if (p.inType != 1) return go(packed_attention_kernel<D, FULL>);
        return p.outType == 1 ? go(packed_attention_kernel<D, BF16_OUT>) : go(packed_attention_kernel<D, BF16_F32>);
    };
    switch (p.dim) {
        case 64: return of(std::integral_constant<int, 64>{});
        case 96: return of(std::integral_constant<int, 96>{});
        case 128: return of(std::integral_constant<int, 128>{});
        case 192: return of(std::integral_constant<int, 192>{});
        default: return of(std::integral_constant<int, 256>{});
    }
}

} // namespace aigpu

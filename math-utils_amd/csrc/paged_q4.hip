// paged_q4.hip - a paged cache of 4-bit codes: appending the newest tokens, reading rows
// back, and one token's attention over the pages.
#include "paged_attention.hpp"

namespace aigpu {

namespace {

/*
    The rows of a 4-bit cache. A block is 32 elements of a row; its scale s is the least
    fp16 number of at most 8 significant bits with 7 s >= the block's largest magnitude,
    at most 2720 (24 s, which the readers form, is then finite in fp16), and an element's
    code c = floor(x / s + 1/2), from -7 to 7: within s / 2 of the value up to 19040. The
    code is stored plus 8, two a byte, the first in the low half. A block with a value
    that is not finite has a NaN for a scale.

    Next to a border between two codes (or two scales) the last bit of x decides, so that
    the codes do not depend on how x was computed: keys are normed and turned in 64 bits,
    and a border is compared with, exactly (it has 8 + 5 bits), after fp32 has said which.
*/
constexpr int BLOCK_LANES = 4;       // of 8 elements each
constexpr float MOST_SCALE = 2720.0f;
constexpr uint16_t NAN_SCALE = 0x7E00;

/* x of the lane one or two on, within fours */
template <int OFF>
__device__ __forceinline__ uint32_t neighbour(uint32_t x) {
    return __builtin_amdgcn_mov_dpp(x, OFF == 1 ? 0xB1 : 0x4E, 0xF, 0xF, true);
}
template <int OFF>
__device__ __forceinline__ double neighbour(double x) {
    const u32x2 b = __builtin_bit_cast(u32x2, x);
    const uint32_t lo = b[0], hi = b[1];
    return __builtin_bit_cast(double, u32x2{neighbour<OFF>(lo), neighbour<OFF>(hi)});
}

/* What the elements x of a lane are, for their codes: T double or float, and whether they
   are bf16 values. `encode` gives the codes 4 bits each, element j at 4 j, and the scale's
   fp16 bits. The lanes of a block call it together. */
template <typename T, bool BF>
__device__ __forceinline__ uint32_t encode(const T (&x)[8], uint16_t& scale) {
    float f[8];
    T top = T(0);
    uint32_t bits = 0;               // the largest magnitude's: not finite from 0x7F800000 on
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        f[j] = float(x[j]);
        bits = max(bits, __float_as_uint(f[j]) & 0x7FFFFFFFu);
        if constexpr (sizeof(T) == 8) top = fmax(top, fabs(x[j]));
    }
    bits = max(bits, neighbour<1>(bits));
    bits = max(bits, neighbour<2>(bits));
    if constexpr (sizeof(T) == 8) {
        top = fmax(top, neighbour<1>(top));
        top = fmax(top, neighbour<2>(top));
    } else {
        top = __uint_as_float(bits);
    }
    // A seventh of it less 2^-22 of itself, so that the next number of 8 bits (a bf16) is the
    // scale or the one before, which the exact product tells. Below 2^-17 fp16's least is the unit.
    const float about = __uint_as_float(bits) * (0.14285714f * (1.0f - 0x1p-22f));
    const uint32_t up = (__float_as_uint(about) + 0xFFFFu) & 0xFFFF0000u;
    float s = __uint_as_float(T(7.0f * __uint_as_float(up)) < top ? up + 0x10000u : up);
    if (__any(about < 0x1p-17f)) {
        float small = ceilf(about * 0x1p24f) * 0x1p-24f;
        if (T(7.0f * small) < top) small += 0x1p-24f;
        s = about < 0x1p-17f ? small : s;
    }
    s = fminf(s, MOST_SCALE);
    scale = bits >= 0x7F800000u ? NAN_SCALE : __builtin_bit_cast(uint16_t, _Float16(s));
    const float by = __builtin_amdgcn_rcpf(s);
    float c[8];
    if constexpr (BF) {
        // x / s, of two numbers of 8 bits, is a border or 2^-10 away from it at least
#pragma unroll
        for (int j = 0; j < 8; ++j) c[j] = floorf(fmaf(f[j], by, 0.5f + 0x1p-12f));
    } else {
        float edge = 0.0f;           // how far from the middle between two borders, at most
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float t = fmaf(f[j], by, 0.5f);
            c[j] = floorf(t);
            edge = fmaxf(edge, fabsf(t - c[j] - 0.5f));
        }
        // t (at most 8) is off by 8 (2^-23 + 2 2^-24): nearer borders are decided by the exact ones
        if (__any(edge > 0.5f - 4e-6f)) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (T((c[j] + 0.5f) * s) <= x[j]) c[j] += 1.0f;
                else if (T((c[j] - 0.5f) * s) > x[j]) c[j] -= 1.0f;
            }
        }
    }
    // four codes, and the eights, in a sum of fp32
    uint32_t word[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float sum = 34952.0f;        // 0x8888
#pragma unroll
        for (int j = 0; j < 4; ++j)
            sum = fmaf(__builtin_amdgcn_fmed3f(c[4 * h + j], -7.0f, 7.0f), float(1 << 4 * j), sum);
        word[h] = uint32_t(sum);
    }
    return bits == 0 || bits >= 0x7F800000u ? 0x88888888u : word[0] | word[1] << 16;
}

/* cos and sin of a = pos * freq radians in 64 bits: a less a whole number of quarter
   turns (pi / 2 in two parts), then the series on a quarter's half. The terms left out
   are below 5e-17. */
__device__ __forceinline__ void rotation64_at(uint32_t pos, float freq, double& cs, double& sn) {
    const double a = double(pos) * double(freq);
    const double quarters = rint(a * 0.63661977236758134);
    const double r = fma(-quarters, 6.123233995736766e-17, fma(-quarters, 1.5707963267948966, a)), t = r * r;
    double s = -1.0 / 1307674368000.0, c = 1.0 / 20922789888000.0;
    constexpr double S[] = {1.0 / 6227020800.0, -1.0 / 39916800.0, 1.0 / 362880.0, -1.0 / 5040.0, 1.0 / 120.0, -1.0 / 6.0};
    constexpr double C[] = {-1.0 / 87178291200.0, 1.0 / 479001600.0, -1.0 / 3628800.0, 1.0 / 40320.0, -1.0 / 720.0,
                            1.0 / 24.0, -0.5};
#pragma unroll
    for (int i = 0; i < 6; ++i) s = fma(s, t, S[i]);
#pragma unroll
    for (int i = 0; i < 7; ++i) c = fma(c, t, C[i]);
    s = fma(r * t, s, r);
    c = fma(t, c, 1.0);
    const uint32_t turn = uint32_t(int64_t(quarters)) & 3u;
    cs = turn == 0 ? c : (turn == 1 ? -s : (turn == 2 ? -c : s));
    sn = turn == 0 ? s : (turn == 1 ? c : (turn == 2 ? -s : -c));
}

/* 1 / sqrt(x) in 64 bits: the instruction's 26 bits or so, twice improved; 0 for infinity,
   which the steps would make NaN of: an element that is infinite is its own block's alone */
__device__ __forceinline__ double inverse_root(double x) {
    double y = __builtin_amdgcn_rsq(x);
#pragma unroll
    for (int i = 0; i < 2; ++i) y = fma(y * 0.5, fma(-x * y, y, 1.0), y);
    return x == INFINITY ? 0.0 : y;
}

/* where a token's turn j stands: those that neighbouring lanes read together, together */
__host__ __device__ constexpr uint32_t turnsOf(uint32_t half) { return (half + 7) / 8 * 8; }
__device__ __forceinline__ uint32_t turn_slot(uint32_t j, uint32_t half) { return j % 8 * ((half + 7) / 8) + j / 8; }

/* sum over the LPR lanes of a row, in 64 bits */
template <int LPR>
__device__ __forceinline__ double row_sum64(double x, int lane) {
    constexpr int P = LPR & -LPR;
#pragma unroll
    for (int o = P / 2; o > 0; o >>= 1) x += __shfl_xor(x, o, WAVE);
    if constexpr (LPR == P) return x;
    const int first = lane / LPR * LPR;
    return __shfl(x, first, WAVE) + __shfl(x, first + P, WAVE) + __shfl(x, first + 2 * P, WAVE);
}

/*
    Appending. A workgroup takes a few tokens, D / 8 lanes a row of k or v, 8 elements
    each: read, normed and turned (keys), encoded and stored, a word and a quarter of a
    scale a lane. A row's loads go out while the one before it is encoded.

    8199 tokens of 8 heads of 128, bf16, normed and turned (34 MB in, 9 MB out): 26 us,
    1.6 TB/s; without norm and rotation, whose 64 bits the keys take, 20. What bounds it is
    a workgroup's chain (starts, lengths, page ids, angles, then four rows a lane one after
    the other), which its registers let four workgroups a CU run at once: five and six spill
    (36 thousand tokens and their reading back 137 and 146 us against 130). The norm's
    weights wait in LDS, as in registers they spilled (141). 32 tokens: 5 us, that chain once.
*/
struct AppendQ4Args {
    PagedAppendQ4Params p;
    uint32_t headMagic, headShift;   // n / kvHeads = n headMagic >> headShift
    uint32_t tokens;                 // of a workgroup, at most MAX_TOKENS
    int wide;                        // k and v rows can be read 16 bytes at a time
};

template <int D, bool BF>
__global__ __launch_bounds__(THREADS, 4) void paged_append_q4_kernel(AppendQ4Args a) {
    constexpr int LPR = D / 8, RPW = WAVE / LPR, NW = THREADS / WAVE, RAW = BF ? 1 : 2;
    extern __shared__ __attribute__((aligned(16))) double2 turns64[];   // [tokens][rot / 2]
    __shared__ double rows[NW][8][WAVE];             // element e of each lane's eight
    __shared__ uint64_t base[MAX_TOKENS];            // row of kv head 0, ~0: not written
    __shared__ uint32_t place[MAX_TOKENS];
    __shared__ double gammas[8][LPR];                // element 8 l + e at [e][l]
    const PagedAppendParams& p = a.p.a;
    const PagedCache& c = p.c;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const uint64_t t0 = (uint64_t(blockIdx.y) * gridDim.x + blockIdx.x) * a.tokens;
    if (t0 >= p.count) return;
    const uint32_t nt = p.count - t0 < a.tokens ? uint32_t(p.count - t0) : a.tokens;
    const uint32_t keys = nt * c.kvHeads, total = 2 * keys;             // k's rows, then v's
    const int sub = lane / LPR, d0 = (lane % LPR) * 8;
    // row r of the workgroup: its token and kv head, and its elements of this lane
    struct Place { uint32_t t, h; } here{};
    u32x4 raw[RAW] = {};
    auto load = [&](uint32_t r) {
        const bool isKey = r < keys;
        if (sub >= RPW || r >= total) return;
        const uint32_t rest = isKey ? r : r - keys;
        here.t = uint32_t(uint64_t(rest) * a.headMagic >> a.headShift);
        here.h = rest - here.t * c.kvHeads;
        const char* src = static_cast<const char*>(isKey ? p.k : p.v) +
                          ((t0 + here.t) * (isKey ? p.kStride : p.vStride) + size_t(here.h) * D + d0) * (BF ? 2 : 4);
        if (a.wide) {
#pragma unroll
            for (int i = 0; i < RAW; ++i) raw[i] = reinterpret_cast<const u32x4*>(src)[i];
        } else if constexpr (BF) {
            const uint16_t* e = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
            for (int i = 0; i < 4; ++i) raw[0][i] = e[2 * i] | uint32_t(e[2 * i + 1]) << 16;
        } else {
            const uint32_t* e = reinterpret_cast<const uint32_t*>(src);
#pragma unroll
            for (int i = 0; i < 8; ++i) raw[i / 4][i % 4] = e[i];
        }
    };
    load(w * RPW + sub);             // the first row is on its way while its place is found
    const Token mine = find_token<NW>(c, p.starts, t0, nt, w, lane);
    if (mine.finds) {
        place[mine.own] = mine.pos;
        base[mine.own] = mine.page < c.pages ? mine.page * c.pageStride + mine.at * c.rowStride : ~uint64_t(0);
    }
    __syncthreads();
    if (p.gamma && threadIdx.x < D) gammas[threadIdx.x % 8][threadIdx.x / 8] = double(p.gamma[threadIdx.x]) + double(p.offset);
    const uint32_t half = p.freqs ? p.rot / 2 : 0;
    for (uint32_t i = threadIdx.x; i < nt * half; i += THREADS) {
        double cs, sn;
        rotation64_at(place[i / half], p.freqs[i % half], cs, sn);
        turns64[i / half * turnsOf(half) + turn_slot(i % half, half)] = double2{cs * double(p.amplitude), sn * double(p.amplitude)};
    }
    __syncthreads();

    // every lane of a wave stays in the loop: the sums and blocks shuffle over all of it
#pragma unroll 1
    for (uint32_t wave = w * RPW; wave < total; wave += NW * RPW) {
        const uint32_t r = wave + sub;
        const bool in = sub < RPW && r < total, isKey = r < keys;
        const uint32_t t = here.t, h = here.h;
        const uint64_t to = base[t];
        const bool live = in && to != ~uint64_t(0);
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (BF) x[e] = __uint_as_float(e & 1 ? raw[0][e / 2] & 0xFFFF0000u : raw[0][e / 2] << 16);
            else x[e] = __uint_as_float(raw[e / 4][e % 4]);
            if (!live) x[e] = 0.0f;
        }
        load(r + NW * RPW);          // the next row's, on its way meanwhile
        uint32_t word;
        uint16_t scale;
        if (wave < keys && (p.gamma || half)) {      // keys among the wave's rows
            double y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = double(x[e]);
            if (p.gamma) {
                double ss = 0.0;
#pragma unroll
                for (int e = 0; e < 8; ++e) ss += y[e] * y[e];
                const double inv = inverse_root(row_sum64<LPR>(ss, lane) * (1.0 / D) + double(p.eps));
                if (live && isKey) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] = y[e] * inv * gammas[e][lane % LPR];
                }
            }
            if (half) {
#pragma unroll
                for (int e = 0; e < 8; ++e) rows[w][e][lane] = y[e];
                wave_sync();
                const double2* cs = turns64 + t * turnsOf(half);
                if (live && isKey) {
                    if (p.interleaved) {
#pragma unroll
                        for (int e = 0; e < 8; e += 2) {
                            if (uint32_t(d0 + e) >= 2 * half) break;
                            const double2 by = cs[turn_slot((d0 + e) / 2, half)];
                            const double u = y[e], v = y[e + 1];
                            y[e] = u * by.x - v * by.y;
                            y[e + 1] = v * by.x + u * by.y;
                        }
                    } else if (half % 8 == 0) {          // all eight partners in one lane
                        if (uint32_t(d0) < 2 * half) {
                            const bool late = uint32_t(d0) >= half;
                            const int other = late ? lane - int(half / 8) : lane + int(half / 8);
                            const uint32_t j0 = late ? d0 - half : d0;
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const double2 by = cs[turn_slot(j0 + e, half)];
                                const double v = rows[w][e][other];
                                y[e] = y[e] * by.x + (late ? v : -v) * by.y;
                            }
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const uint32_t d = d0 + e;
                            if (d >= 2 * half) break;
                            const bool late = d >= half;
                            const uint32_t o = late ? d - half : d + half;
                            const double2 by = cs[turn_slot(late ? o : d, half)];
                            const double v = rows[w][o % 8][lane - lane % LPR + o / 8];
                            y[e] = y[e] * by.x + (late ? v : -v) * by.y;
                        }
                    }
                }
                wave_sync();
            }
            word = encode<double, false>(y, scale);
        } else {
            word = encode<float, BF>(x, scale);
        }
        if (live) {
            const uint64_t at = to + h * c.headStride;
            reinterpret_cast<uint32_t*>(isKey ? c.keys : c.values)[at * LPR + lane % LPR] = word;
            if (lane % LPR % BLOCK_LANES == 0)
                (isKey ? a.p.keyScales : a.p.valueScales)[at * (D / 32) + lane % LPR / BLOCK_LANES] = scale;
        }
    }
}

/*
    Reading back: the rows that the tokens of a ragged batch have in the pages, as the
    values that their codes stand for. The workgroups and lanes are append's; rows are
    independent, four of them in flight a lane. 8199 tokens of 8 heads of 128 to bf16
    (9 MB in, 34 MB out): 11 us, 3.9 TB/s, the search of the tokens' sequences included.
*/
struct ReadQ4Args {
    PagedReadQ4Params p;
    uint32_t headMagic, headShift;
    uint32_t tokens;
    int wide;                        // k and v rows can be written 16 bytes at a time
};

template <int D, bool BF>
__global__ __launch_bounds__(THREADS) void paged_read_q4_kernel(ReadQ4Args a) {
    constexpr int LPR = D / 8, RPW = WAVE / LPR, NW = THREADS / WAVE;
    __shared__ uint64_t base[MAX_TOKENS];            // row of kv head 0
    __shared__ uint32_t state[MAX_TOKENS];           // 0: no sequence's, 1: no place in the pool, 2: read
    const PagedReadQ4Params& p = a.p;
    const PagedCache& c = p.c;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const uint64_t t0 = (uint64_t(blockIdx.y) * gridDim.x + blockIdx.x) * a.tokens;
    if (t0 >= p.count) return;
    const uint32_t nt = p.count - t0 < a.tokens ? uint32_t(p.count - t0) : a.tokens;
    const uint32_t keys = nt * c.kvHeads, total = 2 * keys;
    const Token mine = find_token<NW>(c, p.starts, t0, nt, w, lane);
    if (mine.finds) {
        base[mine.own] = mine.page < c.pages ? mine.page * c.pageStride + mine.at * c.rowStride : 0;
        state[mine.own] = !mine.live ? 0 : (mine.page < c.pages ? 2 : 1);
    }
    __syncthreads();
    const int sub = lane / LPR, d0 = (lane % LPR) * 8;
    if (sub >= RPW) return;
#pragma unroll 4
    for (uint32_t r = w * RPW + sub; r < total; r += NW * RPW) {
        const bool isKey = r < keys;
        const uint32_t rest = isKey ? r : r - keys, t = uint32_t(uint64_t(rest) * a.headMagic >> a.headShift),
                       h = rest - t * c.kvHeads;
        if (state[t] == 0) continue;
        const uint64_t at = base[t] + h * c.headStride;
        const uint32_t word = reinterpret_cast<const uint32_t*>(isKey ? c.keys : c.values)[at * LPR + lane % LPR];
        const uint16_t bits = (isKey ? p.keyScales : p.valueScales)[at * (D / 32) + lane % LPR / BLOCK_LANES];
        const float s = state[t] == 2 ? float(__builtin_bit_cast(_Float16, bits)) : __builtin_nanf("");
        const uint32_t even = word & 0x0F0F0F0Fu, odd = word >> 4 & 0x0F0F0F0Fu;
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)      // s (c - 8), exact
            x[e] = fmaf(float((e & 1 ? odd : even) >> 8 * (e / 2) & 255u), s, -8.0f * s);
        const size_t to = (t0 + t) * (isKey ? p.kStride : p.vStride) + size_t(h) * D + d0;
        if constexpr (BF) {
            uint16_t* out = static_cast<uint16_t*>(isKey ? p.k : p.v) + to;
            const u32x4 packed = {pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])};
            if (a.wide) {
                *reinterpret_cast<u32x4*>(out) = packed;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) out[e] = uint16_t(packed[e / 2] >> 16 * (e & 1));
            }
        } else {
            float* out = static_cast<float*>(isKey ? p.k : p.v) + to;
            if (a.wide) {
                reinterpret_cast<floatx4*>(out)[0] = floatx4{x[0], x[1], x[2], x[3]};
                reinterpret_cast<floatx4*>(out)[1] = floatx4{x[4], x[5], x[6], x[7]};
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) out[e] = x[e];
            }
        }
    }
}

/* As many tokens as the lanes take four rows of, eight where the workgroups are many (16
   rounds of them: 36 thousand tokens of 8 heads of 128 121 us against 130, 8 thousand 39
   against 38), fewer where that leaves CUs idle. */
uint32_t tokens_of(uint64_t count, uint32_t kvHeads, uint32_t dim) {
    const uint32_t rows = THREADS / WAVE * (WAVE / (dim / 8)) * 4;
    const uint64_t spread = count / 512;
    uint32_t tokens = rows / (2 * kvHeads);
    if (tokens && count / tokens > 4096) tokens *= 2;
    if (tokens > spread) tokens = uint32_t(spread);
    return tokens < 1 ? 1 : (tokens > MAX_TOKENS ? MAX_TOKENS : tokens);
}

/* division by multiplication, exact below 2^31 */
void divide_by(uint32_t d, uint32_t& magic, uint32_t& shift) {
    uint32_t log = 0;
    while ((1u << log) < d) ++log;
    shift = 31 + log;
    magic = uint32_t((uint64_t(1) << shift) / d + 1);
}

template <typename Of>
void by_dim(uint32_t dim, Of of) {
    switch (dim) {
        case 64: of(std::integral_constant<int, 64>{}); break;
        case 96: of(std::integral_constant<int, 96>{}); break;
        case 128: of(std::integral_constant<int, 128>{}); break;
        case 192: of(std::integral_constant<int, 192>{}); break;
        default: of(std::integral_constant<int, 256>{}); break;
    }
}

bool tokens_ok(Context& ctx, const std::string& who, const PagedCache& c, const void* k, const void* v, int type,
               const uint32_t* starts, uint64_t count, uint64_t kStride, uint64_t vStride) {
    if (type != 0 && type != 1) return ctx.fail(who + ": unknown type of k and v");
    if (!k || !v) return ctx.fail(who + ": null tensor");
    if (!starts && count != c.batch) return ctx.fail(who + ": without starts there is one token a sequence");
    if (count >= (uint64_t(1) << 31)) return ctx.fail(who + ": too many tokens");
    if (kStride < uint64_t(c.kvHeads) * c.dim || vStride < uint64_t(c.kvHeads) * c.dim)
        return ctx.fail(who + ": the rows of k or v overlap");
    const uintptr_t at = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v);
    if (at & (type == 1 ? 1 : 3)) return ctx.fail(who + ": k and v must be aligned to their elements");
    return true;
}

} // namespace

bool codes_ok(Context& ctx, const char* who, const PagedCache& c, const void* keyScales, const void* valueScales) {
    const std::string w = std::string(who) + ": ";
    if (c.dim != 64 && c.dim != 96 && c.dim != 128 && c.dim != 192 && c.dim != 256)
        return ctx.fail(w + "dim must be 64, 96, 128, 192 or 256");
    if (!c.keys || !c.values || !keyScales || !valueScales || !c.table || !c.lengths) return ctx.fail(w + "null tensor");
    if ((reinterpret_cast<uintptr_t>(c.keys) | reinterpret_cast<uintptr_t>(c.values) |
         reinterpret_cast<uintptr_t>(keyScales) | reinterpret_cast<uintptr_t>(valueScales)) & 15)
        return ctx.fail(w + "the pages must be 16-byte aligned");
    return true;
}

bool check_paged_append_q4(const PagedAppendQ4Params& q) {
    Context& ctx = Context::instance();
    const PagedAppendParams& p = q.a;
    if (!codes_ok(ctx, "paged append", p.c, q.keyScales, q.valueScales)) return false;
    if (!rotation_ok(ctx, "paged append", p.freqs, p.rot, p.c.dim, p.amplitude)) return false;
    if (!tokens_ok(ctx, "paged append", p.c, p.k, p.v, p.inType, p.starts, p.count, p.kStride, p.vStride)) return false;
    if (!rows_apart(p.c, 1)) return ctx.fail("paged append: the rows of the pages overlap");
    return true;
}

bool launch_paged_append_q4(const PagedAppendQ4Params& q, hipStream_t stream) {
    Context& ctx = Context::instance();
    const PagedAppendParams& p = q.a;
    if (p.count == 0 || p.c.batch == 0) return true;
    const uint32_t es = p.inType == 1 ? 2 : 4;
    const uintptr_t at = reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v);
    AppendQ4Args a{};
    a.p = q;
    a.wide = (at & 15) == 0 && (p.count == 1 || (p.kStride | p.vStride) % (16 / es) == 0);
    a.tokens = tokens_of(p.count, p.c.kvHeads, p.c.dim);
    divide_by(p.c.kvHeads, a.headMagic, a.headShift);
    // 16 tokens of 128 turns are 32 KB
    const size_t each = p.freqs ? size_t(turnsOf(p.rot / 2)) * sizeof(double2) : 0;
    const Tiles tiles((p.count + a.tokens - 1) / a.tokens);
    return ctx.launch("paged_append_q4_kernel", stream, [&] {
        by_dim(p.c.dim, [&](auto dim) {
            constexpr int D = decltype(dim)::value;
            auto go = [&](auto kernel) {
                hipLaunchKernelGGL(kernel, dim3(tiles.side, tiles.sides), dim3(THREADS), a.tokens * each, stream, a);
            };
            if (p.inType == 1) go(paged_append_q4_kernel<D, true>);
            else go(paged_append_q4_kernel<D, false>);
        });
    });
}

bool check_paged_read_q4(const PagedReadQ4Params& p) {
    Context& ctx = Context::instance();
    if (!codes_ok(ctx, "paged read", p.c, p.keyScales, p.valueScales) ||
        !tokens_ok(ctx, "paged read", p.c, p.k, p.v, p.outType, p.starts, p.count, p.kStride, p.vStride))
        return false;
    const uint64_t es = p.outType == 1 ? 2 : 4, row = uint64_t(p.c.kvHeads) * p.c.dim * es;
    const Extent k{reinterpret_cast<uintptr_t>(p.k), p.count, p.kStride * es, 1, row, row};
    const Extent v{reinterpret_cast<uintptr_t>(p.v), p.count, p.vStride * es, 1, row, row};
    if (may_meet(k, v)) return ctx.fail("paged read: k and v overlap");
    return true;
}

bool launch_paged_read_q4(const PagedReadQ4Params& p, hipStream_t stream) {
    Context& ctx = Context::instance();
    if (p.count == 0 || p.c.batch == 0) return true;
    const uint32_t es = p.outType == 1 ? 2 : 4;
    const uintptr_t at = reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v);
    ReadQ4Args a{};
    a.p = p;
    a.wide = (at & 15) == 0 && (p.count == 1 || (p.kStride | p.vStride) % (16 / es) == 0);
    a.tokens = tokens_of(p.count, p.c.kvHeads, p.c.dim);
    divide_by(p.c.kvHeads, a.headMagic, a.headShift);
    const Tiles tiles((p.count + a.tokens - 1) / a.tokens);
    return ctx.launch("paged_read_q4_kernel", stream, [&] {
        by_dim(p.c.dim, [&](auto dim) {
            constexpr int D = decltype(dim)::value;
            auto go = [&](auto kernel) {
                hipLaunchKernelGGL(kernel, dim3(tiles.side, tiles.sides), dim3(THREADS), 0, stream, a);
            };
            if (p.outType == 1) go(paged_read_q4_kernel<D, true>);
            else go(paged_read_q4_kernel<D, false>);
        });
    });
}

bool launch_paged_codes(const PagedDecodeParams& p, void* work, hipStream_t stream) {
    return launch_decode_as<PAGED_CODES>("paged_codes_kernel", p, work, stream);
}

} // namespace aigpu

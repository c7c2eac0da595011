// rotary.hip - rotary positions of dense or strided heads, and the frequency
// tables they take.
//
// One pass over the data: 2 bytes moved per byte of x and 3 flops an element,
// so HBM bounds it, or the launch where x is small. A workgroup takes a tile of
// tokens and heads. A thread owns a unit of every row it takes: 16 bytes that
// turn within themselves (interleaved), the two 16-byte pieces whose elements
// pair up (half layout), or a piece to copy. Its first rows' loads go out, then
// the tokens' cosines and sines are formed into LDS, one evaluation a (token,
// pair) for all heads of the tile (the 64-bit angle and the two functions take
// about 100 instructions, as many as rotating 15 heads' pairs), then the rows
// are turned and stored. 8192 tokens of 32 bf16 heads of 128 (134 MB): 23.7 us,
// 5.7 TB/s, where a plain copy of as much takes 24; 1999 tokens of 40 fp32 heads
// of 192 (123 MB): 23.1 us, 5.3 TB/s; one token: 2.2 us, the launch.
#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "context.hpp"
#include "device.hpp"
#include "kernels.hpp"

namespace aigpu {

namespace {

constexpr uint32_t THREADS = 256;
constexpr uint32_t PIECES = 4;          // pieces a thread has in flight
constexpr uint32_t TABLE_BYTES = 32 << 10;

struct RotaryArgs {
    RotaryParams p;
    uint32_t tokens, headsTile;         // of one tile
    uint32_t units, turned;             // units of one row, and how many of them turn
    uint32_t across;                    // threads side by side over a row's units
};

/* V elements: 16 bytes, or one */
template <int V>
struct Piece {
    u32x4 bits;
};
template <>
struct Piece<1> {
    uint32_t bits;
};

template <int V, bool BF>
__device__ __forceinline__ void load_piece(const void* base, size_t at, Piece<V>& x) {
    // nontemporal: x is read once. (Storing out so too gains 5 us of 26 alone at
    // 67 MB, and costs whoever reads it next 9: not done.)
    if constexpr (V > 1)
        x.bits = __builtin_nontemporal_load(
            reinterpret_cast<const u32x4*>(static_cast<const char*>(base) + at * (BF ? 2 : 4)));
    else if constexpr (BF) x.bits = uint32_t(static_cast<const uint16_t*>(base)[at]) << 16;
    else x.bits = static_cast<const uint32_t*>(base)[at];
}

template <int V, bool BF>
__device__ __forceinline__ void store_piece(void* base, size_t at, const Piece<V>& x) {
    if constexpr (V > 1) *reinterpret_cast<u32x4*>(static_cast<char*>(base) + at * (BF ? 2 : 4)) = x.bits;
    else if constexpr (BF) static_cast<uint16_t*>(base)[at] = uint16_t(x.bits >> 16);
    else static_cast<uint32_t*>(base)[at] = x.bits;
}

template <int V, bool BF>
__device__ __forceinline__ void widen(const Piece<V>& x, float (&y)[V]) {
    if constexpr (V == 1) {
        y[0] = __uint_as_float(x.bits);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (BF) {
                y[2 * i] = bf16_bits_to_float(x.bits[i] & 0xFFFFu);
                y[2 * i + 1] = __uint_as_float(x.bits[i] & 0xFFFF0000u);
            } else {
                y[i] = __uint_as_float(x.bits[i]);
            }
        }
    }
}

template <int V, bool BF>
__device__ __forceinline__ void narrow(const float (&y)[V], Piece<V>& x) {
    if constexpr (V == 1) {
        x.bits = BF ? pack_bf16(0.0f, y[0]) : __float_as_uint(y[0]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (BF) x.bits[i] = pack_bf16(y[2 * i], y[2 * i + 1]);
            else x.bits[i] = __float_as_uint(y[i]);
        }
    }
}

/* V: elements of a piece (16 bytes of BF ? bf16 : fp32, or 1); IL: interleaved
   pairs. A unit is two pieces, but for interleaved ones of 16 bytes, whose pairs
   lie within one. */
template <int V, bool BF, bool IL>
__global__ __launch_bounds__(THREADS) void rotary_kernel(RotaryArgs a) {
    constexpr bool TWO = !IL || V == 1;
    constexpr uint32_t ROWS = TWO ? PIECES / 2 : PIECES;
    // [tokens][rot / 2]: cos, sin times the amplitude
    extern __shared__ __attribute__((aligned(16))) float2 turns[];
    const RotaryParams& p = a.p;
    const uint32_t half = p.rot / 2, dim = uint32_t(p.dim);
    const uint64_t t0 = (uint64_t(blockIdx.z) * gridDim.x + blockIdx.x) * a.tokens;
    if (t0 >= p.count) return;
    const uint32_t h0 = blockIdx.y * a.headsTile;
    const uint32_t nt = p.count - t0 < a.tokens ? uint32_t(p.count - t0) : a.tokens;
    const uint32_t nh = uint32_t(p.heads) - h0 < a.headsTile ? uint32_t(p.heads) - h0 : a.headsTile;
    const uint32_t deep = THREADS / a.across, rows = nt * nh;      // rows of one pass over the threads
    const uint32_t u0 = threadIdx.x % a.across, r0 = threadIdx.x / a.across;
    const uint32_t stepT = deep / nh, stepH = deep % nh;

    struct At {
        uint32_t t, h;
    };
    Piece<V> x[ROWS], y[ROWS];
    // the elements of unit u: piece one at d, piece two at d2 (kept out of rows of odd length)
    auto first = [&](uint32_t u) { return IL ? u * (V == 1 ? 2 : V) : (u < a.turned ? u * V : p.rot + (u - a.turned) * V); };
    auto second = [&](uint32_t u) { return IL ? u * 2 + 1 : u * V + half; };
    auto paired = [&](uint32_t u) { return IL ? u * 2 + 1 < dim : u < a.turned; };
    auto load = [&](uint32_t u, uint32_t r, At at) {
#pragma unroll
        for (uint32_t k = 0; k < ROWS; ++k) {
            if (r + k * deep < rows && u < a.units) {
                const size_t from = (t0 + at.t) * p.tokenStride + (h0 + at.h) * p.headStride;
                load_piece<V, BF>(p.x, from + first(u), x[k]);
                if (TWO && paired(u)) load_piece<V, BF>(p.x, from + second(u), y[k]);
            }
            at.t += stepT;
            at.h += stepH;
            if (at.h >= nh) at.h -= nh, ++at.t;
        }
    };
    At at{r0 / nh, r0 % nh};
    if (r0 < deep) load(u0, r0, at);

    for (uint32_t i = threadIdx.x; i < nt * half; i += THREADS) {
        const uint32_t t = i / half, j = i % half;
        const uint32_t pos = p.positions ? p.positions[t0 + t] : uint32_t(p.start + t0 + t);
        float cs, sn;
        rotation_at(pos, p.freqs[j], cs, sn);
        turns[i] = float2{cs * p.amplitude, (p.transpose ? -sn : sn) * p.amplitude};
    }
    __syncthreads();
    if (r0 >= deep) return;             // threads beyond the last whole row
    for (uint32_t u = u0; u < a.units; u += a.across) {
        At here = At{r0 / nh, r0 % nh};
        for (uint32_t r = r0; r < rows; r += ROWS * deep) {
            if (u != u0 || r != r0) load(u, r, here);
#pragma unroll
            for (uint32_t k = 0; k < ROWS; ++k) {
                if (r + k * deep < rows) {
                    if (u < a.turned) {
                        // (a unit's turns start on 16 bytes: its pairs are a piece's, or half of one's)
                        constexpr int PAIRS = TWO ? V : V / 2;
                        float2 turn[PAIRS];
                        const float2* cells = turns + here.t * half + (IL ? first(u) / 2 : first(u));
                        if constexpr (PAIRS == 1) {
                            turn[0] = cells[0];
                        } else {
#pragma unroll
                            for (int i = 0; i < PAIRS; i += 2) {
                                const floatx4 two = *reinterpret_cast<const floatx4*>(cells + i);
                                turn[i] = float2{two[0], two[1]};
                                turn[i + 1] = float2{two[2], two[3]};
                            }
                        }
                        float b[V], c[V];
                        widen<V, BF>(x[k], b);
                        if constexpr (TWO) {
                            widen<V, BF>(y[k], c);
#pragma unroll
                            for (int e = 0; e < V; ++e) {
                                const float2 cs = turn[e];
                                const float v = b[e];
                                b[e] = v * cs.x - c[e] * cs.y;
                                c[e] = c[e] * cs.x + v * cs.y;
                            }
                            narrow<V, BF>(c, y[k]);
                        } else {
#pragma unroll
                            for (int e = 0; e < V; e += 2) {
                                const float2 cs = turn[e / 2];
                                const float v = b[e];
                                b[e] = v * cs.x - b[e + 1] * cs.y;
                                b[e + 1] = b[e + 1] * cs.x + v * cs.y;
                            }
                        }
                        narrow<V, BF>(b, x[k]);
                    }
                    const size_t to = (t0 + here.t) * p.outTokenStride + (h0 + here.h) * p.outHeadStride;
                    store_piece<V, BF>(p.out, to + first(u), x[k]);
                    if (TWO && paired(u)) store_piece<V, BF>(p.out, to + second(u), y[k]);
                }
                here.t += stepT;
                here.h += stepH;
                if (here.h >= nh) here.h -= nh, ++here.t;
            }
        }
    }
}

/* [0, bytes) of the elements that a tensor of these strides spans */
size_t span(uint64_t count, uint64_t heads, uint64_t dim, uint64_t ts, uint64_t hs) {
    return (count - 1) * ts + (heads - 1) * hs + dim;
}

bool in_place(const RotaryParams& p) {
    return p.x == p.out && (p.count == 1 || p.tokenStride == p.outTokenStride) &&
           (p.heads == 1 || p.headStride == p.outHeadStride);
}

/* whether a row of x and one of out share an element, where out has x's strides and starts `apart` elements on */
bool rows_meet(const RotaryParams& p, int64_t apart) {
    const int64_t dim = int64_t(p.dim), ts = int64_t(p.tokenStride), mostT = int64_t(p.count) - 1,
                  mostH = int64_t(p.heads) - 1;
    for (int64_t dh = -mostH; dh <= mostH; ++dh) {
        const int64_t from = apart + dh * int64_t(p.headStride);    // between rows of one token
        // the token distance that brings them nearest, from either side
        const int64_t near = mostT ? -from / ts : 0;
        for (int64_t dt : {near - 1, near, near + 1}) {
            dt = std::max(-mostT, std::min(mostT, dt));
            if (std::abs(from + dt * ts) < dim) return true;
        }
    }
    return false;
}

} // namespace

bool check_rotary(const RotaryParams& p) {
    Context& ctx = Context::instance();
    constexpr uint64_t LIMIT = uint64_t(1) << 31;
    if (p.type != 0 && p.type != 1) return ctx.fail("rotary: unknown element type");
    if (p.dim == 0 || p.dim > 4096 || p.heads >= 65536) return ctx.fail("rotary: dim must be 1..4096, heads below 65536");
    if (p.rot < 2 || p.rot > p.dim || (p.rot & 1)) return ctx.fail("rotary: rotaryDims must be even and within dim");
    if (!(p.amplitude > 0.0f) || !std::isfinite(p.amplitude))
        return ctx.fail("rotary: the amplitude must be positive and finite");
    if (p.count >= LIMIT || (!p.positions && (p.start >= 2 * LIMIT || p.start + p.count > 2 * LIMIT)))
        return ctx.fail("rotary: positions must fit 32 bits");
    for (uint64_t s : {p.tokenStride, p.headStride, p.outTokenStride, p.outHeadStride})
        if (s >= (uint64_t(1) << 40)) return ctx.fail("rotary: a stride is out of range");
    if (p.count == 0 || p.heads == 0) return true;
    if (!p.x || !p.out || !p.freqs) return ctx.fail("rotary: null tensor");
    // out's rows must not overlap each other, nor x's unless they are x's
    const uint64_t ots = p.outTokenStride, ohs = p.outHeadStride;
    const bool tokensApart = (p.count == 1 || ots >= (p.heads - 1) * ohs + p.dim) && (p.heads == 1 || ohs >= p.dim);
    const bool headsApart = (p.heads == 1 || ohs >= (p.count - 1) * ots + p.dim) && (p.count == 1 || ots >= p.dim);
    if (!tokensApart && !headsApart) return ctx.fail("rotary: the rows of out overlap");
    const size_t es = p.type == 1 ? 2 : 4;
    const uintptr_t xb = reinterpret_cast<uintptr_t>(p.x), ob = reinterpret_cast<uintptr_t>(p.out);
    if ((xb | ob) & (es - 1)) return ctx.fail("rotary: x and out must be aligned to their elements");
    const size_t xs = span(p.count, p.heads, p.dim, p.tokenStride, p.headStride) * es;
    const size_t os = span(p.count, p.heads, p.dim, ots, ohs) * es;
    if (!in_place(p) && xb < ob + os && ob < xb + xs) {
        // rows of one token side by side in the same wider rows do not meet
        const uint64_t row = p.tokenStride * es;
        const uint64_t xr = ((p.heads - 1) * p.headStride + p.dim) * es, orow = ((p.heads - 1) * ohs + p.dim) * es;
        const uint64_t gap = row ? (ob >= xb ? (ob - xb) % row : (row - (xb - ob) % row) % row) : 0;
        const bool sideBySide = p.tokenStride == ots && row && gap >= xr && row - gap >= orow;
        // nor do equal lattices of rows that lie between one another (the halves of wider heads)
        const bool equal = (p.count == 1 || p.tokenStride == ots) && (p.heads == 1 || p.headStride == ohs);
        if (!sideBySide && (!equal || rows_meet(p, (int64_t(ob) - int64_t(xb)) / int64_t(es))))
            return ctx.fail("rotary: out overlaps x without being x");
    }

    return true;
}

bool launch_rotary(const RotaryParams& p, hipStream_t stream) {
    Context& ctx = Context::instance();
    if (p.count == 0 || p.heads == 0) return true;
    const size_t es = p.type == 1 ? 2 : 4;
    const uint64_t ots = p.outTokenStride, ohs = p.outHeadStride;
    const uintptr_t xb = reinterpret_cast<uintptr_t>(p.x), ob = reinterpret_cast<uintptr_t>(p.out);
    const bool inPlace = in_place(p);

    // 16-byte pieces where every row starts on 16 bytes and no pair straddles
    // a piece; single elements elsewhere
    const uint32_t piece = uint32_t(16 / es);
    uint64_t strides = 0;
    if (p.count > 1) strides |= p.tokenStride | ots;
    if (p.heads > 1) strides |= p.headStride | ohs;
    const uint32_t grain = p.interleaved ? p.rot : p.rot / 2;
    const bool wide = ((xb | ob) & 15) == 0 && strides % piece == 0 && p.dim % piece == 0 && grain % piece == 0;
    const uint32_t V = wide ? piece : 1;
    RotaryArgs a{};
    a.p = p;
    if (p.interleaved) {
        const uint32_t w = V == 1 ? 2 : V;
        a.units = uint32_t((p.dim + w - 1) / w);
        a.turned = p.rot / w;
    } else {
        a.turned = p.rot / 2 / V;
        a.units = a.turned + uint32_t((p.dim - p.rot) / V);
    }
    if (inPlace) a.units = a.turned;   // the rest is where it belongs
    // a tile of as many rows as the threads hold at once, of whole tokens if
    // that is more than one token's heads
    a.across = a.units < THREADS ? a.units : THREADS;
    const uint32_t heads = uint32_t(p.heads), rows = THREADS / a.across * (p.interleaved && V > 1 ? PIECES : PIECES / 2);
    a.headsTile = heads < rows ? heads : rows;
    const uint32_t most = TABLE_BYTES / (p.rot / 2 * uint32_t(sizeof(float2)));
    a.tokens = rows / a.headsTile;
    a.tokens = a.tokens > most ? most : a.tokens;
    if (a.tokens > p.count) a.tokens = uint32_t(p.count);
    const Tiles tiles((p.count + a.tokens - 1) / a.tokens);
    const dim3 grid(tiles.side, (heads + a.headsTile - 1) / a.headsTile, tiles.sides);
    const size_t lds = size_t(a.tokens) * (p.rot / 2) * sizeof(float2);
    const int which = (V > 1 ? 4 : 0) | (p.type == 1 ? 2 : 0) | (p.interleaved ? 1 : 0);
    return ctx.launch("rotary_kernel", stream, [&] {
        auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(THREADS), lds, stream, a); };
        switch (which) {
            case 0: go(rotary_kernel<1, false, false>); break;
            case 1: go(rotary_kernel<1, false, true>); break;
            case 2: go(rotary_kernel<1, true, false>); break;
            case 3: go(rotary_kernel<1, true, true>); break;
            case 4: go(rotary_kernel<4, false, false>); break;
            case 5: go(rotary_kernel<4, false, true>); break;
            case 6: go(rotary_kernel<8, true, false>); break;
            default: go(rotary_kernel<8, true, true>); break;
        }
    });
}

bool rotary_frequencies(const AiGpuRotaryScaling& s, float* out, float* amplitude) {
    Context& ctx = Context::instance();
    const uint32_t n = s.dims / 2;
    if (s.kind > AIGPU_ROTARY_YARN) return ctx.fail("rotary frequencies: unknown kind");
    if (s.dims < 2 || s.dims > 4096 || (s.dims & 1))
        return ctx.fail("rotary frequencies: dims must be even, 2 .. 4096");
    if (!(s.base > 1.0) || !std::isfinite(s.base)) return ctx.fail("rotary frequencies: base must exceed 1");
    if (s.kind != AIGPU_ROTARY_NONE && (!(s.factor >= 1.0) || !std::isfinite(s.factor)))
        return ctx.fail("rotary frequencies: factor must be at least 1");
    if (s.kind == AIGPU_ROTARY_NTK && s.dims < 4) return ctx.fail("rotary frequencies: this kind needs dims >= 4");
    if (s.kind >= AIGPU_ROTARY_LLAMA3 &&
        (!(s.original > 0.0) || !std::isfinite(s.original) || !(s.low > 0.0) || !(s.high > s.low) ||
         !std::isfinite(s.high)))
        return ctx.fail("rotary frequencies: original must be positive, and 0 < low < high");
    constexpr double TAU = 6.283185307179586;
    double base = s.base, first = 0.0, last = 0.0;
    if (s.kind == AIGPU_ROTARY_NTK) base *= std::pow(s.factor, double(s.dims) / (s.dims - 2.0));
    if (s.kind == AIGPU_ROTARY_YARN) {
        // the pair index whose wave makes `turns` turns over the trained context
        auto pair_of = [&](double turns) {
            return s.dims * std::log(s.original / (turns * TAU)) / (2.0 * std::log(base));
        };
        first = std::fmax(std::floor(pair_of(s.high)), 0.0);
        last = std::fmin(std::ceil(pair_of(s.low)), s.dims - 1.0);
        // no pair between: those from `last` on (all, where none makes `low` turns) are divided
        if (!(last - first >= 0.001)) first = last - 1.0;
    }
    for (uint32_t j = 0; j < n; ++j) {
        double f = std::pow(base, -2.0 * j / s.dims);
        if (s.kind == AIGPU_ROTARY_LINEAR) f /= s.factor;
        if (s.kind == AIGPU_ROTARY_LLAMA3) {
            const double wave = TAU / f;
            if (wave > s.original / s.low) {
                f /= s.factor;
            } else if (wave >= s.original / s.high) {
                const double blend = (s.original / wave - s.low) / (s.high - s.low);
                f *= (1.0 - blend) / s.factor + blend;
            }
        }
        if (s.kind == AIGPU_ROTARY_YARN) {
            const double ramp = std::fmin(std::fmax((j - first) / (last - first), 0.0), 1.0);
            f = f / s.factor * ramp + f * (1.0 - ramp);
        }
        out[j] = float(f);
    }
    *amplitude = s.kind == AIGPU_ROTARY_YARN ? float(0.1 * std::log(s.factor) + 1.0) : 1.0f;
    return true;
}

} // namespace aigpu

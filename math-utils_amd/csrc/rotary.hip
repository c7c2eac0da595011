// rotary.hip - rotary positions of dense or strided heads, and the frequency
// tables they take.
//
// One pass over the data: 2 bytes moved per byte of x and 3 flops an element,
// so HBM bounds it, or the launch where x is small. A workgroup takes a tile of
// tokens and heads. Its tokens' cosines and sines go to LDS first, one
// evaluation a (token, pair) for all the heads of the tile: the 64-bit angle
// and the two functions cost about 60 instructions, as much as rotating 20
// heads' pairs. Then each thread turns units of 16 bytes (half layout: the two
// 16-byte pieces whose elements pair up; interleaved: one piece, its pairs
// within) and copies the pieces that stay as they are.
#include <cmath>

#include "context.hpp"
#include "device.hpp"
#include "kernels.hpp"

namespace aigpu {

namespace {

constexpr uint32_t THREADS = 256;
constexpr uint32_t TILE_UNITS = 1024;   // units a workgroup aims at: four a thread
constexpr uint32_t MAX_TOKENS = 32;     // tokens of a tile: at most this, and a 32 KB table

struct RotaryArgs {
    RotaryParams p;
    uint32_t tokens, headsTile;         // of one tile
    uint32_t units, turned;             // units of one head, and how many of them turn
};

/* V elements (16 bytes, or one) as fp32 */
template <int V, bool BF>
__device__ __forceinline__ void load_piece(const void* base, size_t at, float (&x)[V]) {
    if constexpr (V == 1) {
        x[0] = load_elem(base, at, BF ? 1 : 0);
    } else {
        const u32x4 raw = *reinterpret_cast<const u32x4*>(static_cast<const char*>(base) + at * (BF ? 2 : 4));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (BF) {
                x[2 * i] = bf16_bits_to_float(raw[i] & 0xFFFFu);
                x[2 * i + 1] = __uint_as_float(raw[i] & 0xFFFF0000u);
            } else {
                x[i] = __uint_as_float(raw[i]);
            }
        }
    }
}

template <int V, bool BF>
__device__ __forceinline__ void store_piece(void* base, size_t at, const float (&x)[V]) {
    if constexpr (V == 1) {
        if constexpr (BF) static_cast<uint16_t*>(base)[at] = float_to_bf16_bits(x[0]);
        else static_cast<float*>(base)[at] = x[0];
    } else {
        u32x4 raw;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (BF)
                raw[i] = float_to_bf16_bits(x[2 * i]) | uint32_t(float_to_bf16_bits(x[2 * i + 1])) << 16;
            else
                raw[i] = __float_as_uint(x[i]);
        }
        *reinterpret_cast<u32x4*>(static_cast<char*>(base) + at * (BF ? 2 : 4)) = raw;
    }
}

/* V: elements of a piece (16 bytes of BF ? bf16 : fp32, or 1); IL: interleaved
   pairs, where a piece of one element comes with its partner */
template <int V, bool BF, bool IL>
__global__ __launch_bounds__(THREADS) void rotary_kernel(RotaryArgs a) {
    extern __shared__ float2 turns[];   // [tokens][rot / 2]: cos, sin times the amplitude
    const RotaryParams& p = a.p;
    const uint32_t half = p.rot / 2;
    const uint64_t t0 = uint64_t(blockIdx.x) * a.tokens;
    const uint32_t h0 = blockIdx.y * a.headsTile;
    const uint32_t nt = p.count - t0 < a.tokens ? uint32_t(p.count - t0) : a.tokens;
    const uint32_t nh = uint32_t(p.heads) - h0 < a.headsTile ? uint32_t(p.heads) - h0 : a.headsTile;
    for (uint32_t i = threadIdx.x; i < nt * half; i += THREADS) {
        const uint32_t t = i / half, j = i % half;
        const uint32_t pos = p.positions ? p.positions[t0 + t] : uint32_t(p.start + t0 + t);
        float cs, sn;
        rotation_at(pos, p.freqs[j], cs, sn);
        turns[i] = float2{cs * p.amplitude, (p.transpose ? -sn : sn) * p.amplitude};
    }
    __syncthreads();
    const uint32_t total = nt * nh * a.units;
    for (uint32_t i = threadIdx.x; i < total; i += THREADS) {
        const uint32_t u = i % a.units, th = i / a.units, h = th % nh, t = th / nh;
        const size_t from = (t0 + t) * p.tokenStride + (h0 + h) * p.headStride;
        const size_t to = (t0 + t) * p.outTokenStride + (h0 + h) * p.outHeadStride;
        const float2* turn = turns + t * half;
        if constexpr (IL) {
            constexpr int W = V == 1 ? 2 : V;
            const uint32_t d = u * W;
            float x[W];
            if constexpr (V == 1) {
                float one[1];
                load_piece<1, BF>(p.x, from + d, one), x[0] = one[0];
                if (d + 1 < p.dim) load_piece<1, BF>(p.x, from + d + 1, one);
                x[1] = one[0];
            } else {
                load_piece<V, BF>(p.x, from + d, x);
            }
            if (u < a.turned) {
#pragma unroll
                for (int i2 = 0; i2 < W; i2 += 2) {
                    const float2 cs = turn[d / 2 + i2 / 2];
                    const float b = x[i2], c = x[i2 + 1];
                    x[i2] = b * cs.x - c * cs.y;
                    x[i2 + 1] = c * cs.x + b * cs.y;
                }
            }
            if constexpr (V == 1) {
                store_piece<1, BF>(p.out, to + d, {x[0]});
                if (d + 1 < p.dim) store_piece<1, BF>(p.out, to + d + 1, {x[1]});
            } else {
                store_piece<V, BF>(p.out, to + d, x);
            }
        } else {
            if (u < a.turned) {
                const uint32_t d = u * V;
                float x[V], y[V];
                load_piece<V, BF>(p.x, from + d, x);
                load_piece<V, BF>(p.x, from + d + half, y);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float2 cs = turn[d + e];
                    const float b = x[e], c = y[e];
                    x[e] = b * cs.x - c * cs.y;
                    y[e] = c * cs.x + b * cs.y;
                }
                store_piece<V, BF>(p.out, to + d, x);
                store_piece<V, BF>(p.out, to + d + half, y);
            } else {
                const uint32_t d = p.rot + (u - a.turned) * V;
                float x[V];
                load_piece<V, BF>(p.x, from + d, x);
                store_piece<V, BF>(p.out, to + d, x);
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
        if (p.tokenStride != ots || !row || gap < xr || row - gap < orow)
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
    const uint32_t heads = uint32_t(p.heads);
    a.headsTile = TILE_UNITS / a.units;
    a.headsTile = a.headsTile < 1 ? 1 : (a.headsTile > heads ? heads : a.headsTile);
    a.tokens = TILE_UNITS / (a.headsTile * a.units);
    const uint32_t table = (32u << 10) / (p.rot / 2 * 8);
    const uint32_t most = table < 1 ? 1 : (table < MAX_TOKENS ? table : MAX_TOKENS);
    a.tokens = a.tokens < 1 ? 1 : (a.tokens > most ? most : a.tokens);
    if (a.tokens > p.count) a.tokens = uint32_t(p.count);
    const dim3 grid(unsigned((p.count + a.tokens - 1) / a.tokens), (heads + a.headsTile - 1) / a.headsTile);
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
        if (!(last - first >= 0.001)) last = first + 0.001;
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

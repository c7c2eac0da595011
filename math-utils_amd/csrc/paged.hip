// paged.hip - a paged KV cache: appending the newest tokens, and one token's
// attention over each sequence's pages.
#include <cmath>

#include "context.hpp"
#include "device.hpp"
#include "kernels.hpp"

namespace aigpu {

namespace {

constexpr uint32_t THREADS = 256;
constexpr uint32_t NOWHERE = 0xFFFFFFFFu;

/* element offset of (page, row) for kv head h, or ~0 where the sequence's table
   does not lead to a page of the pool */
__device__ __forceinline__ uint64_t row_offset(const PagedCache& c, uint32_t b, uint64_t pos, uint32_t h) {
    const uint64_t slot = pos / c.pageSize;
    if (slot >= c.tableWidth) return ~uint64_t(0);
    const uint32_t page = c.table[b * c.tableStride + slot];
    if (page >= c.pages) return ~uint64_t(0);
    return page * c.pageStride + h * c.headStride + (pos - slot * c.pageSize) * c.rowStride;
}

/*
    Appending. A workgroup takes `tokens` tokens; a wave works out each one's
    sequence (the count of starts at or before it: one round of loads, where a
    binary search would take one a step), its position and its page, and the
    workgroup their cosines and sines, once for all kv heads. Then D / 8 lanes
    take a row of k or v, 8 elements each. HBM bounds it: rows are read once and
    written once, 16 bytes a lane.
*/
struct AppendArgs {
    PagedAppendParams p;
    uint32_t tokens;
    int wide;                   // k and v rows can be read 16 bytes at a time
};

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

template <int D>
__global__ __launch_bounds__(THREADS) void paged_append_kernel(AppendArgs a) {
    constexpr int LPR = D / 8, RPW = WAVE / LPR;     // lanes of a row, rows of a wave
    extern __shared__ float2 turns[];                // [tokens][rot / 2]
    __shared__ float rows[THREADS / WAVE][RPW][D];
    __shared__ uint64_t base[32];                    // of head 0, ~0: not written
    __shared__ uint32_t place[32];
    const PagedAppendParams& p = a.p;
    const PagedCache& c = p.c;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const uint64_t t0 = uint64_t(blockIdx.x) * a.tokens;
    const uint32_t nt = p.count - t0 < a.tokens ? uint32_t(p.count - t0) : a.tokens;
    for (uint32_t i = w; i < nt; i += THREADS / WAVE) {
        const uint64_t t = t0 + i;
        uint32_t b = uint32_t(t);
        uint64_t back = 1;      // t is the sequence's back-th newest token
        bool live = true;
        if (p.starts) {
            uint32_t before = 0;
            for (uint32_t k = lane; k <= c.batch; k += WAVE) before += p.starts[k] <= t ? 1u : 0u;
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) before += __shfl_xor(before, o, WAVE);
            live = before > 0 && before <= c.batch;
            b = live ? before - 1 : 0;
            const uint64_t end = p.starts[b + 1];
            live = live && end > t;
            back = live ? end - t : 1;
        }
        if (lane == 0) {
            const uint64_t len = c.lengths[b];
            const uint64_t pos = len - back;
            place[i] = uint32_t(pos);
            base[i] = live && len >= back ? row_offset(c, b, pos, 0) : ~uint64_t(0);
        }
    }
    __syncthreads();
    const uint32_t half = p.freqs ? p.rot / 2 : 0;
    for (uint32_t i = threadIdx.x; i < nt * half; i += THREADS) {
        float cs, sn;
        rotation_at(place[i / half], p.freqs[i % half], cs, sn);
        turns[i] = float2{cs * p.amplitude, sn * p.amplitude};
    }
    __syncthreads();
    const int r = lane / LPR, d0 = (lane % LPR) * 8;
    const uint32_t total = nt * c.kvHeads * 2;      // k's rows of a token, then v's
    // every lane of a wave stays in the loop: the row sums shuffle over all of it
    for (uint32_t first = w * RPW; first < total; first += THREADS / WAVE * RPW) {
        const uint32_t i = first + r;
        const bool in = r < RPW && i < total;
        const uint32_t t = in ? i / (2 * c.kvHeads) : 0, rest = in ? i % (2 * c.kvHeads) : 0;
        const bool isKey = rest < c.kvHeads;
        const uint32_t h = isKey ? rest : rest - c.kvHeads;
        const uint64_t to = base[t];
        const bool live = in && to != ~uint64_t(0);
        float x[8] = {};
        if (live) {
            const void* src = isKey ? p.k : p.v;
            const size_t at = (t0 + t) * (isKey ? p.kStride : p.vStride) + size_t(h) * D + d0;
            if (!a.wide) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = load_elem(src, at + e, p.inType);
            } else if (p.inType == 1) {
                const u32x4 raw = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(src) + at);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[2 * e] = bf16_bits_to_float(raw[e] & 0xFFFFu);
                    x[2 * e + 1] = __uint_as_float(raw[e] & 0xFFFF0000u);
                }
            } else {
                const floatx4* f = reinterpret_cast<const floatx4*>(static_cast<const float*>(src) + at);
                const floatx4 lo = f[0], hi = f[1];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = lo[e], x[4 + e] = hi[e];
            }
        }
        if (p.gamma) {
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
            const float inv = 1.0f / sqrtf(row_sum<LPR>(ss, lane) / float(D) + p.eps);
            if (live && isKey) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * (p.gamma[d0 + e] + p.offset);
            }
        }
        if (half) {
            // a half-layout partner sits in another lane: through LDS
            float* row = rows[w][r < RPW ? r : 0];
            if (!p.interleaved && live && isKey) {
#pragma unroll
                for (int e = 0; e < 8; ++e) row[d0 + e] = x[e];
            }
            wave_sync();
            if (live && isKey) {
                const float2* turn = turns + t * half;
                float y[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t d = d0 + e;
                    y[e] = x[e];
                    if (d < 2 * half) {
                        if (p.interleaved) {
                            const float2 cs = turn[d / 2];
                            y[e] = d & 1 ? x[e] * cs.x + x[e ^ 1] * cs.y : x[e] * cs.x - x[e ^ 1] * cs.y;
                        } else {
                            const bool late = d >= half;
                            const float2 cs = turn[late ? d - half : d];
                            const float other = row[late ? d - half : d + half];
                            y[e] = late ? x[e] * cs.x + other * cs.y : x[e] * cs.x - other * cs.y;
                        }
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = y[e];
            }
            wave_sync();
        }
        if (live) {
            u32x4 raw;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                raw[e] = float_to_bf16_bits(x[2 * e]) | uint32_t(float_to_bf16_bits(x[2 * e + 1])) << 16;
            *reinterpret_cast<u32x4*>((isKey ? c.keys : c.values) + to + h * c.headStride + d0) = raw;
        }
    }
}

/*
    One token's attention, the plain way: a workgroup a (sequence, query head),
    its four waves taking every fourth position, each with a running maximum and
    sum, joined at the end.
*/
__global__ __launch_bounds__(THREADS) void paged_decode_kernel(PagedDecodeParams p) {
    constexpr int WAVES = THREADS / WAVE, PER = 4;   // elements of a row a lane holds at most
    __shared__ float q[256], acc[WAVES][256], wm[WAVES], wl[WAVES];
    __shared__ int bad;
    const PagedCache& c = p.c;
    const uint32_t b = blockIdx.x / p.heads, head = blockIdx.x % p.heads, D = c.dim;
    const uint32_t kvh = head / (p.heads / c.kvHeads);
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const uint32_t len = c.lengths[b];
    float* out = p.out + (size_t(b) * p.heads + head) * D;
    if (len == 0 || len > p.maxLength) {
        for (uint32_t d = threadIdx.x; d < D; d += THREADS) out[d] = len ? __builtin_nanf("") : 0.0f;
        return;
    }
    const size_t qrow = b * p.qTokenStride + head * p.qStride;
    if (threadIdx.x == 0) bad = 0;
    if (w == 0) {
        float ss = 0.0f;
        for (uint32_t d = lane; d < D; d += WAVE) {
            q[d] = load_elem(p.q, qrow + d, p.inType);
            ss += q[d] * q[d];
        }
        if (p.gamma) {
            const float inv = 1.0f / sqrtf(wave_sum(ss) / float(D) + p.eps);
            for (uint32_t d = lane; d < D; d += WAVE) q[d] = q[d] * inv * (p.gamma[d] + p.offset);
        }
        wave_sync();
        const uint32_t half = p.freqs ? p.rot / 2 : 0;
        for (uint32_t j = lane; j < half; j += WAVE) {
            const uint32_t i0 = p.interleaved ? 2 * j : j, i1 = p.interleaved ? 2 * j + 1 : j + half;
            float cs, sn;
            rotation_at(len - 1, p.freqs[j], cs, sn);
            const float u = q[i0], v = q[i1];
            q[i0] = (u * cs - v * sn) * p.amplitude;
            q[i1] = (v * cs + u * sn) * p.amplitude;
        }
        wave_sync();
        for (uint32_t d = lane; d < D; d += WAVE) q[d] *= p.scale * LOG2E;
    }
    __syncthreads();
    const uint32_t first = p.window && len > p.window ? uint32_t(len - p.window) : 0u;
    float m = -INFINITY, l = 0.0f, o[PER] = {};
    for (uint64_t pos = first + w; pos < len; pos += WAVES) {
        const uint64_t at = row_offset(c, b, pos, kvh);
        if (at == ~uint64_t(0)) {
            if (lane == 0) bad = 1;
            continue;
        }
        float s = 0.0f;
        for (uint32_t d = lane; d < D; d += WAVE) s += q[d] * bf16_bits_to_float(c.keys[at + d]);
        s = wave_sum(s);
        const float top = fmaxf(m, s), keep = exp2f(m - top), weight = exp2f(s - top);
        l = l * keep + weight;
        for (uint32_t i = 0; i < PER; ++i) {
            const uint32_t d = lane + i * WAVE;
            if (d < D) o[i] = o[i] * keep + weight * bf16_bits_to_float(c.values[at + d]);
        }
        m = top;
    }
    for (uint32_t i = 0; i < PER; ++i)
        if (lane + i * WAVE < D) acc[w][lane + i * WAVE] = o[i];
    if (lane == 0) wm[w] = m, wl[w] = l;
    __syncthreads();
    const float top = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
    for (uint32_t d = threadIdx.x; d < D; d += THREADS) {
        float sum = 0.0f, x = 0.0f;
        for (int k = 0; k < WAVES; ++k) {
            const float f = wm[k] == -INFINITY ? 0.0f : exp2f(wm[k] - top);
            sum += wl[k] * f;
            x += acc[k][d] * f;
        }
        x = bad ? __builtin_nanf("") : x / sum;
        if (p.outputGate) x *= sigmoid_of(load_elem(p.q, qrow + D + d, p.inType));
        out[d] = x;
    }
}

bool rotation_ok(Context& ctx, const char* who, const float* freqs, int rot, uint32_t dim, float amplitude) {
    if (!freqs) return true;
    if (rot < 2 || uint32_t(rot) > dim || (rot & 1))
        return ctx.fail(std::string(who) + ": rotaryDims must be even and within dim");
    if (!(amplitude > 0.0f) || !std::isfinite(amplitude))
        return ctx.fail(std::string(who) + ": the amplitude must be positive and finite");
    return true;
}

bool cache_ok(Context& ctx, const char* who, const PagedCache& c) {
    const std::string w = std::string(who) + ": ";
    if (c.dim != 64 && c.dim != 96 && c.dim != 128 && c.dim != 192 && c.dim != 256)
        return ctx.fail(w + "dim must be 64, 96, 128, 192 or 256");
    if (!c.keys || !c.values || !c.table || !c.lengths) return ctx.fail(w + "null tensor");
    if ((reinterpret_cast<uintptr_t>(c.keys) | reinterpret_cast<uintptr_t>(c.values)) & 15)
        return ctx.fail(w + "the pages must be 16-byte aligned");
    if ((c.pageStride | c.headStride | c.rowStride) % 8) return ctx.fail(w + "page strides must be multiples of 8");
    if (c.rowStride < c.dim) return ctx.fail(w + "the rows of a page overlap");
    return true;
}

} // namespace

bool check_paged_append(const PagedAppendParams& p) {
    Context& ctx = Context::instance();
    if (!cache_ok(ctx, "paged append", p.c)) return false;
    if (!rotation_ok(ctx, "paged append", p.freqs, p.rot, p.c.dim, p.amplitude)) return false;
    if (p.inType != 0 && p.inType != 1) return ctx.fail("paged append: unknown input type");
    if (!p.k || !p.v) return ctx.fail("paged append: null tensor");
    if (!p.starts && p.count != p.c.batch)
        return ctx.fail("paged append: without starts there is one token a sequence");
    if (p.count >= (uint64_t(1) << 31)) return ctx.fail("paged append: too many tokens");
    if (p.kStride < uint64_t(p.c.kvHeads) * p.c.dim || p.vStride < uint64_t(p.c.kvHeads) * p.c.dim)
        return ctx.fail("paged append: the rows of k or v overlap");
    const uintptr_t at = reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v);
    if (at & (p.inType == 1 ? 1 : 3)) return ctx.fail("paged append: k and v must be aligned to their elements");
    return true;
}

bool launch_paged_append(const PagedAppendParams& p, hipStream_t stream) {
    Context& ctx = Context::instance();
    if (p.count == 0 || p.c.batch == 0) return true;
    const uint32_t es = p.inType == 1 ? 2 : 4;
    const uintptr_t at = reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v);
    AppendArgs a{};
    a.p = p;
    a.wide = (at & 15) == 0 && (p.count == 1 || (p.kStride | p.vStride) % (16 / es) == 0);
    // one round of the workgroup's rows, but no more tokens than a wave a token
    const uint32_t rows = THREADS / WAVE * (WAVE / (p.c.dim / 8));
    a.tokens = rows / (2 * p.c.kvHeads);
    a.tokens = a.tokens < 1 ? 1 : (a.tokens > 16 ? 16 : a.tokens);
    const unsigned grid = unsigned((p.count + a.tokens - 1) / a.tokens);
    const size_t lds = p.freqs ? size_t(a.tokens) * (p.rot / 2) * sizeof(float2) : 0;
    return ctx.launch("paged_append_kernel", stream, [&] {
        auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(grid), dim3(THREADS), lds, stream, a); };
        switch (p.c.dim) {
            case 64: go(paged_append_kernel<64>); break;
            case 96: go(paged_append_kernel<96>); break;
            case 128: go(paged_append_kernel<128>); break;
            case 192: go(paged_append_kernel<192>); break;
            default: go(paged_append_kernel<256>); break;
        }
    });
}

bool check_paged_decode(const PagedDecodeParams& p) {
    Context& ctx = Context::instance();
    if (!cache_ok(ctx, "paged decode", p.c)) return false;
    if (!rotation_ok(ctx, "paged decode", p.freqs, p.rot, p.c.dim, p.amplitude)) return false;
    if (p.inType != 0 && p.inType != 1) return ctx.fail("paged decode: unknown input type");
    if (!p.q || !p.out) return ctx.fail("paged decode: null tensor");
    if ((reinterpret_cast<uintptr_t>(p.q) & (p.inType == 1 ? 1 : 3)) || (reinterpret_cast<uintptr_t>(p.out) & 3))
        return ctx.fail("paged decode: q and out must be aligned to their elements");
    if (p.heads == 0 || p.heads % p.c.kvHeads) return ctx.fail("paged decode: heads must be a multiple of kvHeads");
    if (p.qStride < p.c.dim) return ctx.fail("paged decode: qStride < dim");
    if (p.outputGate && p.qStride < 2 * uint64_t(p.c.dim))
        return ctx.fail("paged decode: the output gate needs qStride >= 2 dim");
    if (!(p.scale > 0.0f) || !std::isfinite(p.scale))
        return ctx.fail("paged decode: the scale must be positive and finite");
    if (p.maxLength > uint64_t(p.c.tableWidth) * p.c.pageSize)
        return ctx.fail("paged decode: maxLength exceeds the positions of the table");
    return true;
}

size_t paged_decode_workspace(const PagedDecodeParams& p) { return 0; }

bool launch_paged_decode(const PagedDecodeParams& p, void* work, hipStream_t stream) {
    Context& ctx = Context::instance();
    if (p.c.batch == 0) return true;
    const unsigned grid = p.c.batch * p.heads;
    return ctx.launch("paged_decode_kernel", stream, [&] {
        hipLaunchKernelGGL(paged_decode_kernel, dim3(grid), dim3(THREADS), 0, stream, p);
    });
}

} // namespace aigpu

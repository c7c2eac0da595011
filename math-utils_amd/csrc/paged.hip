// paged.hip - a paged KV cache: appending the newest tokens, and one token's
// attention over each sequence's pages.
#include "paged_attention.hpp"

namespace aigpu {

namespace {

/*
    Appending. A workgroup takes a few tokens; D / 8 lanes take a row of k or v, 8
    elements each, up to PASSES rows a lane. Their loads go out first. Meanwhile
    a wave works out each token's sequence (the count of starts at or before it:
    one round of loads, where a binary search would take one a step), its position
    and its page, and the workgroup the tokens' cosines and sines, once for all kv
    heads. Then k's rows are normed and turned, and all rows rounded and stored.
    Rows are read once and written once, 16 bytes a lane, which HBM would bound;
    what does is a workgroup's chain of starts, lengths, table and angles, of
    which as many run at once as a CU's registers hold (74 a thread: six; at 106,
    four, 12% slower): 8199 bf16 tokens of 8 heads of 128 (67 MB) take 16.8 us,
    4.0 TB/s; 32 tokens 4.1 us.
*/
constexpr int PASSES = 4;
struct AppendArgs {
    PagedAppendParams p;
    uint32_t tokens;                // of a workgroup, at most MAX_TOKENS
    int wide;                       // k and v rows can be read 16 bytes at a time
};

template <int D, bool BF>
__global__ __launch_bounds__(THREADS) void paged_append_kernel(AppendArgs a) {
    constexpr int LPR = D / 8, RPW = WAVE / LPR;     // lanes of a row, rows of a wave
    constexpr int NW = THREADS / WAVE, DEEP = NW * RPW, RAW = BF ? 1 : 2;
    extern __shared__ __attribute__((aligned(16))) float2 turns[];   // [tokens][rot / 2]
    __shared__ __attribute__((aligned(16))) float rows[NW][RPW][D];
    __shared__ __attribute__((aligned(16))) float gammas[D];
    __shared__ uint64_t base[MAX_TOKENS];            // of kv head 0, ~0: not written
    __shared__ uint32_t place[MAX_TOKENS];
    const PagedAppendParams& p = a.p;
    const PagedCache& c = p.c;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const uint64_t t0 = (uint64_t(blockIdx.y) * gridDim.x + blockIdx.x) * a.tokens;
    if (t0 >= p.count) return;
    const uint32_t nt = p.count - t0 < a.tokens ? uint32_t(p.count - t0) : a.tokens;
    const uint32_t keys = nt * c.kvHeads, total = 2 * keys;      // k's rows, then v's
    const int sub = lane / LPR, d0 = (lane % LPR) * 8;
    const uint32_t r0 = w * RPW + sub;               // of the lanes that have a row (sub < RPW)

    u32x4 raw[PASSES][RAW];
    uint32_t which[PASSES];                          // token << 16 | kv head; NOWHERE: no row
    auto load = [&](uint32_t first) {
#pragma unroll
        for (int k = 0; k < PASSES; ++k) {
            const uint32_t r = first + k * DEEP;
            which[k] = NOWHERE;
            if (sub >= RPW || r >= total) continue;
            const bool isKey = r < keys;
            const uint32_t rest = isKey ? r : r - keys, t = rest / c.kvHeads, h = rest - t * c.kvHeads;
            which[k] = t << 16 | h;
            const char* src = static_cast<const char*>(isKey ? p.k : p.v) +
                              ((t0 + t) * (isKey ? p.kStride : p.vStride) + size_t(h) * D + d0) * (BF ? 2 : 4);
            if (a.wide) {
#pragma unroll
                for (int i = 0; i < RAW; ++i) raw[k][i] = reinterpret_cast<const u32x4*>(src)[i];
            } else if constexpr (BF) {
                const uint16_t* e = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
                for (int i = 0; i < 4; ++i) raw[k][0][i] = e[2 * i] | uint32_t(e[2 * i + 1]) << 16;
            } else {
                const uint32_t* e = reinterpret_cast<const uint32_t*>(src);
#pragma unroll
                for (int i = 0; i < 8; ++i) raw[k][i / 4][i % 4] = e[i];
            }
        }
    };
    load(r0);
    if (p.gamma && threadIdx.x < D) gammas[threadIdx.x] = p.gamma[threadIdx.x] + p.offset;

    // ---- each token's sequence, position and page: a wave takes every NW-th,
    //      lane l < MINE its l-th; the page id is on its way during the angles ----
    const Token mine = find_token<NW>(c, p.starts, t0, nt, w, lane);
    if (mine.finds) place[mine.own] = mine.pos;
    __syncthreads();
    const uint32_t half = p.freqs ? p.rot / 2 : 0;
    for (uint32_t i = threadIdx.x; i < nt * half; i += THREADS) {
        float cs, sn;
        rotation_at(place[i / half], p.freqs[i % half], cs, sn);
        turns[i] = float2{cs * p.amplitude, sn * p.amplitude};
    }
    if (mine.finds) base[mine.own] = mine.page < c.pages ? mine.page * c.pageStride + mine.at * c.rowStride : ~uint64_t(0);
    __syncthreads();

    float* row = rows[w][sub < RPW ? sub : 0];
    // every lane of a wave stays in the loop: the row sums shuffle over all of it
#pragma unroll 1
    for (uint32_t first = r0, wave = w * RPW; wave < total; first += PASSES * DEEP, wave += PASSES * DEEP) {
        if (first != r0) load(first);
#pragma unroll
        for (int k = 0; k < PASSES; ++k) {
            const int d0 = fresh_lane((lane % LPR) * 8);
            const uint32_t r = first + k * DEEP;
            if (wave + k * DEEP >= total) break;     // no row of this wave's is left
            const bool in = which[k] != NOWHERE, isKey = r < keys;
            const uint32_t t = in ? which[k] >> 16 : 0, h = which[k] & 0xFFFFu;
            const uint64_t to = base[t];
            const bool live = in && to != ~uint64_t(0);
            u32x4 bits = raw[k][0];
            if (!BF || wave + k * DEEP < keys) {     // not only bf16 values, which are stored as they are
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if constexpr (BF) x[e] = __uint_as_float(e & 1 ? raw[k][0][e / 2] & 0xFFFF0000u : raw[k][0][e / 2] << 16);
                    else x[e] = __uint_as_float(raw[k][e / 4][e % 4]);
                }
                if (p.gamma) {
                    float ss = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
                    const float inv = 1.0f / sqrtf(row_sum<LPR>(ss, lane) / float(D) + p.eps);
                    if (live && isKey) {
                        const floatx4 ga = *reinterpret_cast<const floatx4*>(gammas + d0);
                        const floatx4 gb = *reinterpret_cast<const floatx4*>(gammas + d0 + 4);
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = x[e] * inv * (e < 4 ? ga[e] : gb[e - 4]);
                    }
                }
                if (half && p.interleaved) {
                    if (live && isKey) {
#pragma unroll
                        for (int e = 0; e < 8; e += 2) {
                            if (uint32_t(d0 + e) >= 2 * half) break;
                            const float2 cs = turns[t * half + (d0 + e) / 2];
                            const float u = x[e], v = x[e + 1];
                            x[e] = u * cs.x - v * cs.y;
                            x[e + 1] = v * cs.x + u * cs.y;
                        }
                    }
                } else if (half) {
                    // a half-layout partner sits in another lane: through LDS
                    if (live && isKey) {
                        *reinterpret_cast<floatx4*>(row + d0) = floatx4{x[0], x[1], x[2], x[3]};
                        *reinterpret_cast<floatx4*>(row + d0 + 4) = floatx4{x[4], x[5], x[6], x[7]};
                    }
                    wave_sync();
                    if (half % 8 == 0) {             // all eight partners in one lane
                        if (live && isKey && uint32_t(d0) < 2 * half) {
                            const bool late = uint32_t(d0) >= half;
                            const uint32_t o = late ? d0 - half : d0 + half;
                            const floatx4* cs = reinterpret_cast<const floatx4*>(turns + t * half + (late ? o : d0));
                            const float sign = late ? 1.0f : -1.0f;
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const floatx4 y = *reinterpret_cast<const floatx4*>(row + o + 4 * i);
                                const floatx4 c0 = cs[2 * i], c1 = cs[2 * i + 1];
                                x[4 * i] = x[4 * i] * c0[0] + sign * y[0] * c0[1];
                                x[4 * i + 1] = x[4 * i + 1] * c0[2] + sign * y[1] * c0[3];
                                x[4 * i + 2] = x[4 * i + 2] * c1[0] + sign * y[2] * c1[1];
                                x[4 * i + 3] = x[4 * i + 3] * c1[2] + sign * y[3] * c1[3];
                            }
                        }
                    } else {                         // the row's pairs, dealt to its lanes
                        if (live && isKey) {
#pragma unroll 1
                            for (uint32_t j = d0 / 8; j < half; j += LPR) {
                                const float2 cs = turns[t * half + j];
                                const float u = row[j], v = row[j + half];
                                row[j] = u * cs.x - v * cs.y;
                                row[j + half] = v * cs.x + u * cs.y;
                            }
                        }
                        wave_sync();
                        if (live && isKey) {
#pragma unroll
                            for (int e = 0; e < 8; ++e) x[e] = row[d0 + e];
                        }
                    }
                    wave_sync();
                }
                if (!BF || isKey) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) bits[e] = pack_bf16(x[2 * e], x[2 * e + 1]);
                }
            }
            // nontemporal: who reads the pages next is rarely on this XCD, whose L2
            // they would fill (8199 tokens stored plainly take 10% longer)
            if (live)
                __builtin_nontemporal_store(
                    bits, reinterpret_cast<u32x4*>((isKey ? c.keys : c.values) + to + h * c.headStride + d0));
        }
    }
}

} // namespace

bool rows_apart(const PagedCache& c, uint64_t row) {
    struct Axis { uint64_t stride, size; };
    Axis axes[3] = {{c.rowStride, c.pageSize}, {c.headStride, c.kvHeads}, {c.pageStride, c.pages}};
    std::sort(axes, axes + 3, [](const Axis& a, const Axis& b) { return a.stride < b.stride; });
    uint64_t extent = row;
    for (const Axis& a : axes) {
        if (a.size == 1) continue;
        if (a.stride < extent) return false;
        extent += (a.size - 1) * a.stride;
    }
    return true;
}

bool rotation_ok(Context& ctx, const char* who, const float* freqs, int rot, uint32_t dim, float amplitude) {
    if (!freqs) return true;
    if (rot < 2 || uint32_t(rot) > dim || (rot & 1))
        return ctx.fail(std::string(who) + ": rotaryDims must be even and within dim");
    if (!(amplitude > 0.0f) || !std::isfinite(amplitude))
        return ctx.fail(std::string(who) + ": the amplitude must be positive and finite");
    return true;
}

namespace {

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
    if (!rows_apart(p.c, p.c.dim)) return ctx.fail("paged append: the rows of the pages overlap");
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
    // as many tokens as the lanes hold rows of at once, fewer where workgroups
    // would be less than two a CU: the index chain is what small calls wait for
    const uint32_t rows = THREADS / WAVE * (WAVE / (p.c.dim / 8)) * PASSES;
    const uint64_t spread = p.count / 512;
    uint32_t tokens = rows / (2 * p.c.kvHeads);
    if (tokens > spread) tokens = uint32_t(spread);
    a.tokens = tokens < 1 ? 1 : (tokens > MAX_TOKENS ? MAX_TOKENS : tokens);
    const Tiles tiles((p.count + a.tokens - 1) / a.tokens);
    const size_t lds = p.freqs ? size_t(a.tokens) * (p.rot / 2) * sizeof(float2) : 0;
    return ctx.launch("paged_append_kernel", stream, [&] {
        auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(tiles.side, tiles.sides), dim3(THREADS), lds, stream, a); };
        auto of = [&](auto dim) {
            constexpr int D = decltype(dim)::value;
            if (p.inType == 1) go(paged_append_kernel<D, true>);
            else go(paged_append_kernel<D, false>);
        };
        switch (p.c.dim) {
            case 64: of(std::integral_constant<int, 64>{}); break;
            case 96: of(std::integral_constant<int, 96>{}); break;
            case 128: of(std::integral_constant<int, 128>{}); break;
            case 192: of(std::integral_constant<int, 192>{}); break;
            default: of(std::integral_constant<int, 256>{}); break;
        }
    });
}

bool check_paged_decode(const PagedDecodeParams& p) {
    Context& ctx = Context::instance();
    if (p.form == PAGED_CODES ? !codes_ok(ctx, "paged decode", p.c, p.keyScales, p.valueScales)
                              : !cache_ok(ctx, "paged decode", p.c))
        return false;
    if (!cap_ok(p.cap)) return ctx.fail("paged decode: the cap must be 0, or 1e-6 .. 1e6");
    if (reinterpret_cast<uintptr_t>(p.slopes) & 3)
        return ctx.fail("paged decode: the slopes must be aligned to their elements");
    if (!rotation_ok(ctx, "paged decode", p.freqs, p.rot, p.c.dim, p.amplitude)) return false;
    if (p.inType != 0 && p.inType != 1) return ctx.fail("paged decode: unknown input type");
    if (!p.q || !p.out) return ctx.fail("paged decode: null tensor");
    if ((reinterpret_cast<uintptr_t>(p.q) & (p.inType == 1 ? 1 : 3)) || (reinterpret_cast<uintptr_t>(p.out) & 3))
        return ctx.fail("paged decode: q and out must be aligned to their elements");
    if (p.heads == 0 || p.heads % p.c.kvHeads) return ctx.fail("paged decode: heads must be a multiple of kvHeads");
    if (p.qStride < p.c.dim) return ctx.fail("paged decode: qStride < dim");
    if (p.outputGate && p.qStride < 2 * uint64_t(p.c.dim))
        return ctx.fail("paged decode: the output gate needs qStride >= 2 dim");
    if (p.c.batch) {
        const uintptr_t q = reinterpret_cast<uintptr_t>(p.q), out = reinterpret_cast<uintptr_t>(p.out);
        const uint64_t row = (p.outputGate ? 2 : 1) * uint64_t(p.c.dim);
        const uint64_t last = (p.c.batch - 1) * p.qTokenStride + (p.heads - 1) * p.qStride + row;
        const uint64_t outBytes = uint64_t(p.c.batch) * p.heads * p.c.dim * sizeof(float);
        if (q < out + outBytes && out < q + last * (p.inType == 1 ? 2 : 4))
            return ctx.fail("paged decode: out overlaps q");
    }
    if (!(p.scale > 0.0f) || !std::isfinite(p.scale))
        return ctx.fail("paged decode: the scale must be positive and finite");
    if (p.cap > 0.0f && !std::isnormal(p.scale / p.cap)) return ctx.fail("paged decode: the scale does not suit the cap");
    if (p.maxLength > uint64_t(p.c.tableWidth) * p.c.pageSize)
        return ctx.fail("paged decode: maxLength exceeds the positions of the table");
    if (p.maxLength > (1u << 31)) return ctx.fail("paged decode: maxLength must be at most 2^31");
    if (p.c.batch && decode_shape(p).slice == 0) return ctx.fail("paged decode: one sequence is too much work");
    return true;
}

size_t paged_decode_workspace(const PagedDecodeParams& p) {
    if (p.c.batch == 0) return 0;
    const DecodeShape s = decode_shape(p);
    return workspace_of(s.grid, s.perGroup, p.c.dim);
}

size_t paged_decode_scratch(const PagedDecodeParams& p) {
    return workspace_of(full_grid(p.c.dim, p.form), decode_shape(p).perGroup, p.c.dim);
}

bool launch_paged_decode(const PagedDecodeParams& p, void* work, hipStream_t stream) {
    if (p.form == PAGED_SCORED) return launch_paged_scored(p, work, stream);
    if (p.form == PAGED_CODES) return launch_paged_codes(p, work, stream);
    return launch_decode_as<PAGED_PLAIN>("paged_attention_kernel", p, work, stream);
}

} // namespace aigpu

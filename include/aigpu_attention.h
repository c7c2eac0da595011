#ifndef AIGPU_ATTENTION_H
#define AIGPU_ATTENTION_H

/*
    aigpu_attention.h - the C ABI of the MI355X (gfx950) attention backend.

    Same conventions as the reference's device boundary
    (include/ai/gpu/DeviceABI.h in hday200202/math-utils):
      - plain C symbols with the aigpu_ prefix; scalars, pointers and POD
        structs only; structs go in by pointer, never by value
        (DeviceABI.h:59-65);
      - strings are borrowed from the backend (DeviceABI.h:79-83);
      - the allocator frees: device memory comes from aigpu_upload /
        aigpu_allocate and goes back through aigpu_release
        (DeviceABI.h:89-99);
      - every entry returns 1 on success and 0 on failure with the reason in
        aigpu_last_error(); aigpu_available() is safe to call first
        (DeviceABI.h:75-77);
      - calls are serialised on one process-wide lock, as the reference
        backend's Context::gate does (src/gpu/Kernels.hip:48-63);
      - AiGpuCounters separate kernel time from transfer time
        (DeviceABI.h:66-72).

    The attention entries replace these CPU call sites of the reference:
      kernels::attention     include/ai/Kernels.hpp:132-134, called at
                             include/ai/LocalModel.hpp:2657-2659
      norm -> RoPE -> append -> attention of attentionMixer
                             include/ai/LocalModel.hpp:2608-2659
      the per-token deltaStep loop of gatedDeltaNetMixer
                             include/ai/LocalModel.hpp:2802-2830 (deltaStep at
                             include/ai/Kernels.hpp:105-128)

    Layouts. Host-side tensors keep the reference's layouts: q
    [count][heads][qStride], k/v [count][kvHeads][dim], out
    [count][heads][dim] (Kernels.hpp:143-154). The device KV cache is
    head-major bf16: [kvHeads][capacity][dim] per sequence, so each KV head's
    history is one contiguous run in HBM.
*/

#include <stddef.h>
#include <stdint.h>

/*
    Shared with the reference's boundary. include/ai/gpu/DeviceABI.h
    (guard AI_GPU_DEVICE_ABI_H) defines AiGpuCounters, the AiGpuDense*
    structs and the device-management, projection and resident-decoder entry
    points that this backend implements too. Where that header is reachable
    (on the include path as ai/gpu/DeviceABI.h, or beside this file) it is
    included here and those definitions are taken from it, so both headers
    can share a translation unit in either order. Elsewhere this file
    declares the same types, with the same layouts, and the same entry
    points itself.
*/
#if !defined(AI_GPU_DEVICE_ABI_H) && defined(__has_include)
#if __has_include("ai/gpu/DeviceABI.h")
#include "ai/gpu/DeviceABI.h"
#elif __has_include("DeviceABI.h")
#include "DeviceABI.h"
#endif
#endif

#if defined(_WIN32)
#define AIGPU_ABI __declspec(dllexport)
#else
#define AIGPU_ABI __attribute__((visibility("default")))
#endif

#ifdef __cplusplus
extern "C" {
#endif

/* element types of tensors crossing the boundary */
enum { AIGPU_F32 = 0, AIGPU_BF16 = 1 };

#ifndef AI_GPU_DEVICE_ABI_H
/* DeviceABI.h:66-72 */
typedef struct AiGpuCounters {
    uint64_t launches;
    uint64_t hostToDeviceBytes;
    uint64_t deviceToHostBytes;
    double kernelSeconds;
    double transferSeconds;
} AiGpuCounters;

/* ---- device entry points, as DeviceABI.h:75-118 ---- */
AIGPU_ABI int aigpu_available(void);                               /* DeviceABI.h:77 */
AIGPU_ABI const char* aigpu_device_name(void);                     /* DeviceABI.h:82 */
AIGPU_ABI const char* aigpu_last_error(void);                      /* DeviceABI.h:83 */
AIGPU_ABI uint64_t aigpu_total_memory(void);                       /* DeviceABI.h:85 */
AIGPU_ABI uint64_t aigpu_free_memory(void);                        /* DeviceABI.h:86 */
AIGPU_ABI uint64_t aigpu_allocated_bytes(void);                    /* DeviceABI.h:87 */
AIGPU_ABI void* aigpu_upload(const void* host, uint64_t bytes);    /* DeviceABI.h:97 */
AIGPU_ABI void aigpu_release(void* device, uint64_t bytes);        /* DeviceABI.h:98 */
AIGPU_ABI int aigpu_download(void* host, const void* device, uint64_t bytes); /* DeviceABI.h:99 */
AIGPU_ABI void aigpu_synchronize(void);                            /* DeviceABI.h:115 */
AIGPU_ABI void aigpu_counters(AiGpuCounters* out);                 /* DeviceABI.h:117 */
AIGPU_ABI void aigpu_reset_counters(void);                         /* DeviceABI.h:118 */
#endif /* !AI_GPU_DEVICE_ABI_H */

/* New beside aigpu_upload: a zero-filled device allocation (KV caches,
   recurrent states) released by aigpu_release, and a host->device copy into
   an existing allocation at a byte offset. */
AIGPU_ABI void* aigpu_allocate(uint64_t bytes);
AIGPU_ABI int aigpu_write(void* device, uint64_t offset, const void* host, uint64_t bytes);

/* ------------------------------------------------------------------------ */
/* 1. Drop-in for kernels::attention (Kernels.hpp:132-134).                  */
/*    Host pointers, fp32, the reference's position-major KV                 */
/*    [pos][kvHeads][dim]; same argument list and meaning. Staged in,         */
/*    computed in fp32 on the GPU, copied back. Replaces the call at          */
/*    LocalModel.hpp:2657-2659 line for line.                                 */
/* ------------------------------------------------------------------------ */
AIGPU_ABI int aigpu_attention(const float* q, const float* keys, const float* values,
                              float* out, uint64_t count, uint64_t start, uint64_t heads,
                              uint64_t kvHeads, uint64_t dim, uint64_t qStride,
                              uint64_t window);

/* 2. The same computation on device pointers, with a dtype tag for q and for
      the KV history and explicit KV element strides, so one entry serves the
      reference's position-major layout (posStride = kvHeads*dim,
      headStride = dim) and the head-major cache (posStride = dim,
      headStride = capacity*dim). fp32 arithmetic; out is fp32. */
typedef struct AiGpuAttention {
    const void* q;            /* [count][heads][qStride], qType */
    const void* keys;         /* kvType, element (pos, head) at pos*posStride + head*headStride */
    const void* values;
    float* out;               /* [count][heads][dim] */
    uint32_t qType, kvType;
    uint64_t count, start, heads, kvHeads, dim, qStride, window;
    uint64_t posStride, headStride;
    void* stream;             /* hipStream_t; NULL = default stream */
} AiGpuAttention;
AIGPU_ABI int aigpu_attention_device(const AiGpuAttention* args);

/* ------------------------------------------------------------------------ */
/* 3. Prefill: attentionMixer's QK-RMSNorm -> RoPE -> KV append -> causal    */
/*    attention (LocalModel.hpp:2608-2659) for `count` new tokens at          */
/*    positions start..start+count-1, against a head-major bf16 cache that    */
/*    already holds positions [0, start). Flash-style kernel on fp16 MFMA     */
/*    with fp32 accumulation. dim must be 64 or 128. q, k, v (after norm,     */
/*    RoPE and q's scale) and the cached history go through fp16. A value     */
/*    fp16 cannot hold (|x| >= 65520) raises the call's range flag (below);   */
/*    the call has still written out and the new k, v rows of the cache.     */
/*    The device form is asynchronous: it launches on its stream and         */
/*    returns without waiting, and aigpu_range_status reports its flag. The   */
/*    host form waits for its kernels anyway and returns 0 with a reason.     */
/* ------------------------------------------------------------------------ */
typedef struct AiGpuPrefill {
    const void* q;            /* [count][heads][qStride], inType */
    const void* k;            /* [count][kvHeads][dim], inType */
    const void* v;            /* [count][kvHeads][dim], inType */
    float* out;               /* [count][heads][dim] fp32 */
    void* keyCache;           /* bf16 [kvHeads][capacity][dim] */
    void* valueCache;         /* bf16 [kvHeads][capacity][dim] */
    const float* qNorm;       /* [dim] gamma, NULL = no QK-norm (LocalModel.hpp:2609-2617) */
    const float* kNorm;       /* [dim] gamma, NULL = no QK-norm */
    const float* rotaryFrequencies; /* [rotaryDims/2] (LocalModel.hpp:807-820); NULL = no RoPE */
    float epsilon;            /* cfg.normEps */
    float normOffset;         /* spec.normWeightOffset (0 for qwen3) */
    uint32_t rotaryDims;
    uint32_t inType;
    uint32_t outputGate;      /* 1: out *= sigmoid(q[.. + dim + d]), the gate half of each q row
                                 (spec.attnOutputGate, LocalModel.hpp:2660-2665); needs qStride >= 2 dim */
    uint32_t reserved;
    uint64_t count, start, heads, kvHeads, dim, qStride, window, capacity;
    void* stream;
} AiGpuPrefill;
/* device pointers throughout */
AIGPU_ABI int aigpu_prefill_attention(const AiGpuPrefill* args);
/* q, k, v, out, qNorm, kNorm, rotaryFrequencies are host pointers (fp32 or
   bf16 per inType); the caches are device allocations. Staged in and out. */
AIGPU_ABI int aigpu_prefill_attention_host(const AiGpuPrefill* args);

/* A plain streaming copy of `bytes` between two device buffers (16-byte
   aligned, not overlapping) on `stream`. No counterpart in the reference's
   ABI: it measures what HBM delivers on this part, the ceiling beside the
   spec peak for the HBM-bound kernels (the reference's GPU testing measures
   bandwidth with a bf16 GEMV, src/gpu-testing.cpp:298-351). Asynchronous. */
AIGPU_ABI int aigpu_copy_device(void* dst, const void* src, uint64_t bytes, void* stream);

/* fp16 range flags of the asynchronous prefill calls (aigpu_prefill_attention,
   aigpu_prefill_mixer). No counterpart in the reference, whose calls are all
   synchronous on the host. Every prefill call takes the next ticket (1, 2,
   ...; aigpu_range_ticket returns the latest) and a flag word of its own,
   which its kernels raise when a value overflows fp16. aigpu_range_status
   waits for the device and returns 1 when no call since the previous query
   raised its flag; otherwise 0, with *ticket (when not NULL) the earliest
   raising call's ticket and aigpu_last_error naming it. Either way the flags
   are clear afterwards. A call captured into a graph has no ticket of its
   own: its replays raise a shared flag, reported as ticket UINT64_MAX. 255
   tickets share the flag words in turn, so a flag is lost only if 255 later
   calls are queued before its call runs. */
AIGPU_ABI uint64_t aigpu_range_ticket(void);
AIGPU_ABI int aigpu_range_status(uint64_t* ticket);

/* ------------------------------------------------------------------------ */
/* 4. Decode: one new token for each of `batch` sequences with ragged         */
/*    cached lengths. The new q and k get QK-RMSNorm and RoPE at position     */
/*    positions[b] inside the kernel ("on load"); the new k, v are appended   */
/*    to sequence b's cache at positions[b]; attention covers positions       */
/*    [first, positions[b]] (first from the window as Kernels.hpp:142).       */
/*    For batch 1 this is exactly attentionMixer with count = 1. Split-K,     */
/*    HBM-bound kernel; heads/kvHeads must be 1..8 and dim 64 or 128.         */
/* ------------------------------------------------------------------------ */
typedef struct AiGpuDecode {
    const void* q;            /* [batch][heads][qStride], inType */
    const void* k;            /* [batch][kvHeads][dim], inType */
    const void* v;            /* [batch][kvHeads][dim], inType */
    float* out;               /* [batch][heads][dim] fp32 */
    void* keyCache;           /* bf16, sequence b at b*batchStride: [kvHeads][capacity][dim] */
    void* valueCache;
    const uint32_t* positions;/* [batch] cached length of each sequence = new token position */
    const float* qNorm;
    const float* kNorm;
    const float* rotaryFrequencies;
    float epsilon;
    float normOffset;
    uint32_t rotaryDims;
    uint32_t inType;
    uint32_t maxPosition;     /* >= every positions[b]; sizes the launch */
    uint32_t outputGate;      /* as AiGpuPrefill::outputGate */
    uint64_t batch, heads, kvHeads, dim, qStride, window, capacity;
    uint64_t batchStride;     /* elements between sequences' caches; 0 = kvHeads*capacity*dim */
    void* stream;
} AiGpuDecode;
AIGPU_ABI int aigpu_decode_attention(const AiGpuDecode* args);
/* q, k, v, out, positions, qNorm, kNorm, rotaryFrequencies are host
   pointers; the caches are device allocations. */
AIGPU_ABI int aigpu_decode_attention_host(const AiGpuDecode* args);
/* aigpu_decode_attention without any allocation. No counterpart in the
   reference: it is for callers that cannot allocate device memory (code
   under HIP graph capture, serving loops that forbid hipMalloc). Its
   split-K records live in a fixed 32 MiB device array per GPU, held until
   the process ends; larger batches run in slices that fit it, and a call
   whose single sequence does not fit returns 0 with the reason. Every call
   on a GPU shares that array: calls on different streams are ordered by the
   backend, but replays of graphs captured from it that overlap on one GPU
   race on it. Make one call (or aigpu_available) before a capture: the
   first call of a process sets up the backend and looks up the array's
   address, which capture does not allow. Same arguments, kernels and
   results as aigpu_decode_attention. */
AIGPU_ABI int aigpu_decode_attention_static(const AiGpuDecode* args);

/* ------------------------------------------------------------------------ */
/* 5. Gated delta rule over a token range (the recurrence of                  */
/*    gatedDeltaNetMixer, LocalModel.hpp:2802-2830): for each token t and     */
/*    value head h (key head h / (valueHeads/keyHeads)):                      */
/*      S *= exp(g); delta = beta*(v - S^T k); S += k delta^T; out = S^T q    */
/*    computed as a chunked scan (WY form) with fp32 state.                   */
/* ------------------------------------------------------------------------ */
typedef struct AiGpuDeltaRule {
    const void* q;            /* [count][keyHeads][keyDim], inType */
    const void* k;            /* [count][keyHeads][keyDim], inType */
    const void* v;            /* [count][valueHeads][valueDim], inType */
    const float* g;           /* [count][valueHeads] log decay (used when aLog is NULL) */
    const float* beta;        /* [count][valueHeads] (used when aLog is NULL) */
    const float* a;           /* raw gate inputs [count][valueHeads] (used when aLog is set): */
    const float* b;           /*   g = -exp(aLog[h])*softplus(a + dtBias[h]), beta = sigmoid(b) */
    const float* aLog;        /* [valueHeads] (LocalModel.hpp:2820-2823) */
    const float* dtBias;      /* [valueHeads] */
    float* state;             /* [valueHeads][keyDim][valueDim] fp32, in/out */
    float* out;               /* [count][valueHeads][valueDim] fp32 */
    uint32_t inType;
    uint32_t normalize;       /* 1: l2normalise q,k (eps 1e-6) and q *= 1/sqrt(keyDim) */
    uint32_t chunk;           /* 64 (0 = 64) */
    uint32_t reserved;
    uint64_t count, keyHeads, valueHeads, keyDim, valueDim;
    void* stream;
} AiGpuDeltaRule;
AIGPU_ABI int aigpu_gated_delta_rule(const AiGpuDeltaRule* args);
/* every tensor a host pointer; state updated in place on the host */
AIGPU_ABI int aigpu_gated_delta_rule_host(const AiGpuDeltaRule* args);

/* ------------------------------------------------------------------------ */
/* 5b. Kimi Delta Attention's recurrence (kimiDeltaMixer,                    */
/*     LocalModel.hpp:2928-2947): the gated delta rule with one decay per    */
/*     KEY CHANNEL, deltaStep(perKeyDecay = true) (Kernels.hpp:105-128).     */
/* ------------------------------------------------------------------------ */
typedef struct AiGpuKda {
    const void* q;            /* [count][keyHeads][keyDim], inType */
    const void* k;            /* [count][keyHeads][keyDim], inType */
    const void* v;            /* [count][valueHeads][valueDim], inType */
    const float* g;           /* [count][valueHeads][keyDim] log decay (decay = exp(g) <= 1) */
    const float* beta;        /* [count][valueHeads] */
    /* raw gates, used when g and beta are NULL (LocalModel.hpp:2894-2905):  */
    /*   g = safeGate ? lowerBound sigmoid(exp(aLog) (f + dtBias))            */
    /*                : -exp(aLog) softplus(f + dtBias),  beta = sigmoid(b)   */
    const float* f;           /* [count][valueHeads][keyDim] decay projection (f_b output) */
    const float* b;           /* [count][valueHeads] write-strength projection */
    const float* aLog;        /* [valueHeads] */
    const float* dtBias;      /* [valueHeads][keyDim] */
    float lowerBound;         /* LocalConfig::linLowerBound, <= 0 */
    uint32_t safeGate;        /* LocalConfig::linSafeGate */
    float* state;             /* [valueHeads][keyDim][valueDim] fp32, in/out */
    float* out;               /* [count][valueHeads][valueDim] fp32 */
    uint32_t inType;
    uint32_t normalize;       /* 1: l2normalise q,k (eps 1e-6) and q *= 1/sqrt(keyDim) */
    uint64_t count, keyHeads, valueHeads, keyDim, valueDim;
    void* stream;
} AiGpuKda;
AIGPU_ABI int aigpu_kda_rule(const AiGpuKda* args);

/* ------------------------------------------------------------------------ */
/* 6. The Gated DeltaNet steps either side of the recurrence                 */
/*    (gatedDeltaNetMixer, LocalModel.hpp:2724-2844). No reference kernel    */
/*    exists for them: the mixer runs them inline on the host.               */
/* ------------------------------------------------------------------------ */
/* causalConvolution + SiLU (LocalModel.hpp:2678-2708) over the projection    */
/* rows, with the linFusedQKVZ de-interleave (:2739-2776) when `fused` is     */
/* set, writing the recurrence's dense inputs. The window carries the last   */
/* kernelSize-1 inputs between calls (LocalCache::convWindow), as fp32.      */
typedef struct AiGpuGdnConv {
    const void* in;           /* fused == 0: [count][CW] rows q | k | v (CW = 2 keyHeads keyDim
                                 + valueHeads valueDim); fused: [count][keyHeads][2 keyDim +
                                 2 G valueDim] (per key head q, k, its G value heads' v, their z) */
    const void* ba;           /* fused: [count][keyHeads][2 G], the G heads' b then their a */
    const float* kernel;      /* [CW][kernelSize] (LocalLayer::linConv) */
    float* window;            /* [kernelSize-1][CW] fp32, read then replaced */
    void* q;                  /* out [count][keyHeads][keyDim], outType */
    void* k;                  /* out [count][keyHeads][keyDim], outType */
    void* v;                  /* out [count][valueHeads][valueDim], outType */
    void* z;                  /* fused: out [count][valueHeads][valueDim], outType (not convolved) */
    float* a;                 /* fused: out [count][valueHeads] fp32 */
    float* b;                 /* fused: out [count][valueHeads] fp32 */
    uint32_t inType, outType; /* AIGPU_F32 / AIGPU_BF16 */
    uint32_t fused, reserved;
    uint64_t count, keyHeads, valueHeads, keyDim, valueDim, kernelSize;
    void* stream;
} AiGpuGdnConv;
AIGPU_ABI int aigpu_gdn_conv(const AiGpuGdnConv* args);

/* rmsNormRow of each (token, value head) row of the recurrence output, its  */
/* weight stored directly, then times SiLU(z) (LocalModel.hpp:2833-2841), or */
/* with gateKind 1 times sigmoid(z), kimiDeltaMixer's form (:2936-2945)      */
typedef struct AiGpuGdnGatedNorm {
    const float* x;           /* [count][valueHeads][valueDim] fp32 */
    const void* z;            /* [count][valueHeads][valueDim], zType */
    const float* gamma;       /* [valueDim] (LocalLayer::linNorm) */
    void* out;                /* [count][valueHeads][valueDim], outType */
    float epsilon;            /* LocalConfig::normEps */
    uint32_t zType, outType, gateKind; /* gateKind 0: SiLU, 1: sigmoid */
    uint64_t count, valueHeads, valueDim;
    void* stream;
} AiGpuGdnGatedNorm;
AIGPU_ABI int aigpu_gdn_gated_norm(const AiGpuGdnGatedNorm* args);

/* ------------------------------------------------------------------------ */
/* 5c. Multi-head latent attention (latentAttentionMixer,                    */
/*     LocalModel.hpp:3118-3158): per token and head, q folded through the  */
/*     head's key rows of kv_b_proj, softmax against the cached latents     */
/*     (all positions up to the token, or the indexer's sorted selection,   */
/*     KeySelection :1203-1206), the weighted latents through the value     */
/*     rows. Device pointers.                                               */
/* ------------------------------------------------------------------------ */
typedef struct AiGpuLatentAttention {
    const float* q;           /* [count][heads][nopeDim] (q_b_proj output, :3106) */
    const float* latent;      /* [startPos + count][kvLoraRank] cache, this call's rows included */
    const void* kvB;          /* [heads * (nopeDim + vDim)][kvLoraRank] kv_b_proj, kvBType */
    uint32_t kvBType;         /* AIGPU_F32 / AIGPU_BF16 */
    uint32_t reserved;
    const uint32_t* selStart; /* [count] or NULL (every token dense) */
    const uint32_t* selCount; /* [count], 0xFFFFFFFF for a dense token */
    const uint32_t* selKeys;  /* the concatenated sorted key lists */
    float* out;               /* [count][heads][vDim] fp32 */
    float scale;              /* 1/sqrt(qk_nope_head_dim + qk_rope_head_dim), :3116 */
    uint64_t count, startPos, heads, nopeDim, vDim, kvLoraRank;
    void* stream;
} AiGpuLatentAttention;
AIGPU_ABI int aigpu_latent_attention(const AiGpuLatentAttention* args);

/* ------------------------------------------------------------------------ */
/* 7. Projections (DeviceABI.h:101-112): c[m][n] = a[m][k] . b[n][k]^T, with */
/*    a and c host fp32 and b a device weight from aigpu_upload, in the     */
/*    reference's four encodings (Quant.hpp): fp32, bf16, Q8 (int8 codes,   */
/*    one fp32 scale per 32) and Q4 (two codes a byte, byte j of a block    */
/*    holding codes j and j+16, offset 8; one fp32 scale per 32). They      */
/*    return nothing, as the reference's do; failures set aigpu_last_error.  */
/* ------------------------------------------------------------------------ */
#ifndef AI_GPU_DEVICE_ABI_H
AIGPU_ABI void aigpu_matmul_nt(const float* a, const void* b, float* c,
                               uint64_t m, uint64_t k, uint64_t n);            /* DeviceABI.h:101 */
AIGPU_ABI void aigpu_matmul_nt_bf16(const float* a, const void* b, float* c,
                                    uint64_t m, uint64_t k, uint64_t n);       /* DeviceABI.h:104 */
AIGPU_ABI void aigpu_matmul_nt_q8(const float* a, const void* b, const void* scales, float* c,
                                  uint64_t m, uint64_t k, uint64_t n);         /* DeviceABI.h:107 */
AIGPU_ABI void aigpu_matmul_nt_q4(const float* a, const void* b, const void* scales, float* c,
                                  uint64_t m, uint64_t k, uint64_t n);         /* DeviceABI.h:111 */
#endif /* !AI_GPU_DEVICE_ABI_H */

/* The device form of the same product (no counterpart in the reference,
   whose matmul stages a and c through the host every call): every pointer
   is device memory, the bias is optional, and accumulate = 1 adds the
   product into c (a residual add). */
enum { AIGPU_W_F32 = 0, AIGPU_W_BF16 = 1, AIGPU_W_Q8 = 2, AIGPU_W_Q4 = 3 };
typedef struct AiGpuMatmul {
    const float* a;           /* [m][k] fp32 */
    const void* b;            /* [n][k] weights in `type` */
    const float* scales;      /* [n][k/32] for Q8 / Q4 */
    const float* bias;        /* [n] or NULL */
    float* c;                 /* [m][ldc] fp32 */
    uint32_t type;            /* AIGPU_W_* (AiGpuDenseWeight::type) */
    uint32_t accumulate;
    uint64_t m, k, n, ldc;    /* ldc 0 means n */
    void* stream;
} AiGpuMatmul;
AIGPU_ABI int aigpu_matmul_device(const AiGpuMatmul* args);

/* ------------------------------------------------------------------------ */
/* 8. The resident single-token decoder (DeviceABI.h:119-152), the same     */
/*    structs and entry points: a dense RMSNorm / RoPE / SwiGLU model kept   */
/*    on the device; LocalModel::residentDecode (LocalModel.hpp:3598-3645)   */
/*    is the caller. Weight codes and scales are device pointers (from      */
/*    aigpu_upload) and stay the caller's; norms, biases, rotary            */
/*    frequencies and the cache arrays are host pointers, copied in.        */
/* ------------------------------------------------------------------------ */
#ifndef AI_GPU_DEVICE_ABI_H
typedef struct AiGpuDenseWeight {       /* DeviceABI.h:122-127 */
    const void* codes;
    const void* scales;
    uint32_t type, inDim, outDim;       /* F32=0, BF16=1, Q8=2, Q4=3 */
    const float* bias;                  /* optional, copied at creation */
} AiGpuDenseWeight;
typedef struct AiGpuDenseLayer {        /* DeviceABI.h:128-135 */
    AiGpuDenseWeight q, k, v, o, gate, up, down;
    const float* inputNorm;
    const float* postNorm;
    const float* qNorm;
    const float* kNorm;
    uint32_t window;                    /* 0 = full causal attention */
} AiGpuDenseLayer;
typedef struct AiGpuDenseConfig {       /* DeviceABI.h:136-143 */
    uint32_t hidden, layers, heads, kvHeads, headDim, intermediate;
    uint32_t capacity, rotaryDims, vocab;
    float epsilon, theta;
    const float* finalNorm;
    AiGpuDenseWeight head;
    const float* rotaryFrequencies;     /* rotaryDims/2 entries; optional */
} AiGpuDenseConfig;
AIGPU_ABI int aigpu_dense_supported(void);                                      /* DeviceABI.h:144 */
AIGPU_ABI void* aigpu_dense_create(const AiGpuDenseConfig* config,
                                   const AiGpuDenseLayer* layers, const float* const* keys,
                                   const float* const* values, uint32_t length);  /* DeviceABI.h:145 */
AIGPU_ABI void aigpu_dense_release(void* context);                             /* DeviceABI.h:148 */
AIGPU_ABI void aigpu_dense_decode(void* context, const float* embedding,
                                  float* logits, uint32_t position);           /* DeviceABI.h:149 */
AIGPU_ABI void aigpu_dense_read_cache(void* context, float* const* keys,
                                      float* const* values, uint32_t length);  /* DeviceABI.h:151 */
#endif /* !AI_GPU_DEVICE_ABI_H */

/* ------------------------------------------------------------------------ */
/* 9. attentionMixer for a prefill in one call (LocalModel.hpp:2577-2667):  */
/*    the q, k, v projections of x (apply, :2604-2606), QK-RMSNorm -> RoPE  */
/*    -> KV append (:2608-2655) as the k and v projections' epilogue, the   */
/*    causal attention over the cache (:2657-2659), the output gate         */
/*    (:2660-2665) and the o projection (:2667) into out. The weights are   */
/*    AiGpuDenseWeight with every pointer on the device (bias included);    */
/*    qStride is dim, or 2 dim with outputGate (q_proj's per-head gate      */
/*    half). dim 64 or 128; codes 16-byte aligned.                          */
/* ------------------------------------------------------------------------ */
typedef struct AiGpuPrefillMixer {
    const float* x;                 /* [count][hidden] fp32, the normed hidden states */
    AiGpuDenseWeight q, k, v, o;    /* q [heads*qStride][hidden], k and v [kvHeads*dim][hidden],
                                       o [hidden][heads*dim] */
    float* out;                     /* [count][hidden] fp32 */
    void* keyCache;                 /* bf16 [kvHeads][capacity][dim], positions [0, start) valid */
    void* valueCache;
    const float* qNorm;             /* [dim] gamma or NULL (LocalModel.hpp:2609-2617) */
    const float* kNorm;
    const float* rotaryFrequencies; /* [rotaryDims/2] or NULL = no RoPE */
    float epsilon, normOffset;
    uint32_t rotaryDims, outputGate;
    uint32_t accumulate;            /* 1: out += the mixer's output (the residual add) */
    uint32_t reserved;
    uint64_t count, start, hidden, heads, kvHeads, dim, window, capacity;
    void* stream;
} AiGpuPrefillMixer;
/* asynchronous like aigpu_prefill_attention: values outside fp16's range
   raise the call's range flag (aigpu_range_status) */
AIGPU_ABI int aigpu_prefill_mixer(const AiGpuPrefillMixer* args);

/* ------------------------------------------------------------------------ */
/* 10. The sparse-attention indexer (selectKeys, LocalModel.hpp:2971-3068),  */
/*    GLM-5.3's pooled form: the call's index keys layer-normed into the     */
/*    key cache and folded, pool by pool, into pooled keys; each query token */
/*    scoring the pools wholly at or before it and keeping the topK / pool   */
/*    best, plus the unfinished pool with indexTail. The result is the       */
/*    selection aigpu_latent_attention takes. Among equal scores at the      */
/*    boundary the lower pool is kept (the reference's nth_element leaves    */
/*    that order unspecified). A score is fp32 work: within (dim + heads)    */
/*    2^-24 of its terms' magnitudes, whatever range q and the pools span.   */
/*    Device pointers throughout.                                            */
/* ------------------------------------------------------------------------ */
typedef struct AiGpuSelectKeys {
    const float* h;                 /* [count][hidden], latentAttentionMixer's input (the call, :3110) */
    const float* qResid;            /* [count][qRank], q_a_proj's normed output (:3097-3099) */
    AiGpuDenseWeight idxK;          /* [dim][hidden] */
    AiGpuDenseWeight idxGate;       /* [dim][hidden] */
    AiGpuDenseWeight idxQB;         /* [heads*dim][qRank] */
    AiGpuDenseWeight idxWeights;    /* [heads][hidden] */
    const float* kNorm;             /* [dim] layerNorm weight */
    const float* kNormBias;         /* [dim] or NULL */
    const float* ape;               /* [pool][dim] */
    float* indexKeys;               /* [capacity][dim]; positions < startPos valid */
    float* indexGates;              /* [capacity][dim] */
    float* poolKeys;                /* [capacity/pool + 1][dim] */
    uint32_t* selStart;             /* [count] */
    uint32_t* selCount;             /* [count]; UINT32_MAX: the token sees every key */
    uint32_t* selKeys;              /* [count][topK/pool*pool + pool], each token's keys sorted */
    float* scores;                  /* optional [count][(startPos+count)/pool]: sparse tokens' pool scores */
    uint32_t indexTail, reserved;
    uint64_t count, startPos, hidden, qRank, heads, dim, topK, pool, capacity;
    void* stream;
} AiGpuSelectKeys;
AIGPU_ABI int aigpu_select_keys(const AiGpuSelectKeys* args);

/* ------------------------------------------------------------------------ */
/* 11. Rotary positions (the inlined loop of LocalModel.hpp:2624-2648 as an  */
/*    operator of its own, for q and keys that go to aigpu_attention_device).*/
/*    Per token at position p and head, with n = rotaryDims / 2 and pair j   */
/*    made of elements (j, j + n), or (2j, 2j + 1) when interleaved:         */
/*      a = p frequencies[j]                                                 */
/*      (u, w) -> amplitude (u cos a - w sin a, w cos a + u sin a)           */
/*    and elements from rotaryDims on copied. transpose = 1 turns by -a (the */
/*    amplitude still multiplies): the gradient of x from the gradient of    */
/*    out. The angle is formed and reduced in 64 bits (the reference, and    */
/*    the entries above, round it to fp32 first: 3e-3 radians at position    */
/*    100000), good to 2^-51 of itself, and its cosine and sine, small ones  */
/*    too, to 3 units of fp32's last place; the amplitude and the rotation   */
/*    round in fp32, the result once to `type`. out may be x (same strides)  */
/*    or share no element with it. Asynchronous; needs no scratch, so calls  */
/*    on different streams are not ordered by the backend.                   */
/* ------------------------------------------------------------------------ */
typedef struct AiGpuRotary {
    const void* x;            /* element (token, head, d) at token*tokenStride + head*headStride + d, type */
    void* out;                /* the same with the out strides, type */
    const uint32_t* positions;/* [count], unsigned, or NULL: start, start + 1, ... */
    const float* frequencies; /* [rotaryDims/2] */
    float amplitude;          /* of cos and sin (scaled long contexts); 0 means 1 */
    uint32_t rotaryDims;      /* even, 2 .. dim */
    uint32_t type;            /* AIGPU_F32 / AIGPU_BF16 */
    uint32_t interleaved, transpose, reserved;
    uint64_t count, start, heads, dim;
    uint64_t tokenStride, headStride;       /* 0 mean heads*headStride and dim */
    uint64_t outTokenStride, outHeadStride; /* 0 likewise */
    void* stream;
} AiGpuRotary;
AIGPU_ABI int aigpu_rotary(const AiGpuRotary* args);

/* The frequency table that rotations take, on the host (LocalModel.hpp:807-820
   builds the first, second and fourth kind; computed here in 64 bits and
   rounded once). With f_j = base^(-2j / dims):
     NONE    f_j
     LINEAR  f_j / factor
     NTK     f_j with base * factor^(dims / (dims - 2)) as the base
     LLAMA3  f_j / factor where a turn takes more than original / low
             positions, f_j below original / high, blended between
     YARN    f_j / factor for pairs of at most `low` turns over `original`
             positions, f_j from `high` turns on, a ramp over the pair index
             between; amplitude 0.1 ln(factor) + 1
   *amplitude (optional) is what the rotations' amplitude takes. Needs no
   device. */
enum { AIGPU_ROTARY_NONE = 0, AIGPU_ROTARY_LINEAR = 1, AIGPU_ROTARY_NTK = 2, AIGPU_ROTARY_LLAMA3 = 3,
       AIGPU_ROTARY_YARN = 4 };
typedef struct AiGpuRotaryScaling {
    uint32_t kind;            /* AIGPU_ROTARY_* */
    uint32_t dims;            /* rotaryDims: even, at least 2 (4 for NTK) */
    double base;              /* ropeTheta, > 1 */
    double factor;            /* >= 1 (LINEAR and later) */
    double original;          /* trained context (LLAMA3, YARN) */
    double low, high;         /* LLAMA3: 1 and 4; YARN: 1 and 32 */
} AiGpuRotaryScaling;
AIGPU_ABI int aigpu_rotary_frequencies(const AiGpuRotaryScaling* scaling, float* frequencies, float* amplitude);

/* ------------------------------------------------------------------------ */
/* 12. A paged KV cache: the sequences of a batch keep their positions in    */
/*    pages of pageSize positions from one pool, found through a table.      */
/*    Position i of sequence b lies in page table[b][i / pageSize], row      */
/*    i % pageSize. No counterpart in the reference, whose cache is one      */
/*    contiguous run per layer. lengths[b] counts the cached positions with  */
/*    the newest token's, for both entries: a step adds its tokens to the    */
/*    lengths, then appends, then decodes. A length of 0 is an empty place   */
/*    of a padded batch. A table entry is read only where a position of the  */
/*    sequence needs it; the rest may hold anything.                         */
/* ------------------------------------------------------------------------ */
typedef struct AiGpuPagedCache {
    void* keys;               /* bf16; element (page, head, row, d) at page*pageStride +       */
    void* values;             /*   head*headStride + row*rowStride + d                         */
    const uint32_t* table;    /* [batch][tableStride], the first tableWidth of each row */
    const uint32_t* lengths;  /* [batch] */
    uint64_t batch, pages, pageSize, kvHeads, dim;  /* dim 64, 96, 128, 192 or 256 */
    uint64_t tableWidth, tableStride;               /* tableStride 0 means tableWidth */
    uint64_t pageStride, headStride, rowStride;     /* all 0: [pages][kvHeads][pageSize][dim] */
} AiGpuPagedCache;

/* The newest tokens' k (normed and rotated on the way) and v into the pages,
   rounded to bf16. Without `starts` there is one token a sequence (count =
   batch). With it, rows starts[b] .. starts[b + 1] - 1 of k and v are the last
   starts[b + 1] - starts[b] positions of sequence b, and rows before starts[0]
   or from starts[batch] on are left out. A token whose position is negative
   (a length below its new tokens), beyond the table or in a page outside the
   pool is not written; a decode over such a length answers NaN. No two
   tokens may share a row, nor a key one with a value: a page shared by
   sequences is copied before either writes to it, and strides that let rows of
   the pool overlap are refused (a decode reads such a pool). Asynchronous; needs
   no scratch, so calls on different streams are not ordered by the backend. */
typedef struct AiGpuPagedAppend {
    AiGpuPagedCache cache;
    const void* k;            /* [count][kvHeads][dim], inType; token t at t*kStride */
    const void* v;            /* the same at t*vStride */
    const uint32_t* starts;   /* [batch + 1], not decreasing, or NULL */
    const float* kNorm;       /* [dim] gamma, NULL = no norm (LocalModel.hpp:2609-2617) */
    const float* rotaryFrequencies; /* [rotaryDims/2], NULL = no rotation */
    float epsilon, normOffset;
    float amplitude;          /* as AiGpuRotary::amplitude */
    uint32_t rotaryDims, interleaved, inType;
    uint64_t count, kStride, vStride; /* strides 0 mean kvHeads*dim */
    void* stream;
} AiGpuPagedAppend;
AIGPU_ABI int aigpu_paged_append(const AiGpuPagedAppend* args);

/* Attention of the newest token of each sequence over its cached positions
   (its own included: append first), q normed and rotated at position
   lengths[b] - 1 on load. fp32 throughout but for the cache's bf16: q and the
   softmax's weights enter the products in three bf16 terms each. A sequence of
   length 0 gets zeros; one whose length exceeds maxLength, or that needs a page
   outside the pool, gets NaN. Attended rows have to be finite (one that is not
   makes the heads that read it NaN or infinite); rows that no position covers may hold
   anything. */
typedef struct AiGpuPagedDecode {
    AiGpuPagedCache cache;
    const void* q;            /* [batch][heads][qStride], inType; sequence b at b*qTokenStride */
    float* out;               /* [batch][heads][dim] fp32, apart from q */
    const float* qNorm;
    const float* rotaryFrequencies;
    float epsilon, normOffset, amplitude;
    float scale;              /* of the scores; 0 means 1/sqrt(dim) */
    uint32_t rotaryDims, interleaved, inType;
    uint32_t outputGate;      /* as AiGpuPrefill::outputGate */
    uint32_t maxLength;       /* >= every lengths[b], at most 2^31; sizes the launch */
    uint32_t reserved;
    uint64_t heads, qStride, qTokenStride;  /* qStride 0 means dim, qTokenStride 0 heads*qStride */
    uint64_t window;          /* the last `window` positions only; 0 = all */
    void* workspace;          /* device, 256-byte aligned, zero-filled at first; NULL: the backend's scratch */
    uint64_t workspaceBytes;
    void* stream;
} AiGpuPagedDecode;
AIGPU_ABI int aigpu_paged_decode(const AiGpuPagedDecode* args);
/* The workspace bytes that a call with these sizes needs at most (0: none),
   whatever the lengths hold. The workspace is zero-filled before its first use
   (as aigpu_allocate leaves it); every call leaves the part that matters zero
   again, so calls of any sizes may follow one another in it, but calls that may
   run at once need one each. A call captured into a graph has to bring one
   where this is not 0: the backend's scratch may move. That scratch, of one
   size for calls of the same heads and dim (34 MB at most), is a stream's own
   for the first eight streams that decode, so their calls are not ordered among
   one another (destroy such a stream only when its decodes have ended: its
   scratch goes with the handle); the calls of later streams share one, in turn,
   and so do those of the per-thread default stream, which return when their
   work is done. */
AIGPU_ABI uint64_t aigpu_paged_decode_workspace(const AiGpuPagedDecode* args);

/* aigpu_paged_decode with its scores capped or biased: with s the scaled product of a
   query of head h and the key `apart` positions before it,
     cap > 0   s = cap tanh(s / cap)
     slopes    s -= slopes[h] apart      (after the cap)
   before the softmax; cap 0 and slopes NULL leave them out. The workspace is
   aigpu_paged_decode_workspace's. */
typedef struct AiGpuScores {
    const float* slopes;      /* [heads] or NULL */
    float cap;                /* 0: none; otherwise 1e-6 .. 1e6 */
    uint32_t reserved;
} AiGpuScores;
AIGPU_ABI int aigpu_paged_decode_scored(const AiGpuPagedDecode* args, const AiGpuScores* scores);

/* ------------------------------------------------------------------------ */
/* 13. A paged cache held in 4 bits: the tables, lengths and rules of 12, a   */
/*    row being dim codes of 4 bits and a scale for every 32 of them, at      */
/*      row r = page*pageStride + head*headStride + row*rowStride             */
/*    (strides in rows) of the codes [r][dim / 2] bytes, element d in byte    */
/*    d / 2, the even one in the low half, and of the scales [r][dim / 32]    */
/*    fp16. An element's value is scale * (code - 8). An append makes the     */
/*    scale s of a block the least fp16 number of at most 8 significant bits  */
/*    with 7 s >= its largest magnitude, at most 2720, and a code             */
/*    floor(x / s + 1/2) + 8 within 1 .. 15: an element is off by s / 2 at    */
/*    most, or, past 7 * 2720 = 19040, becomes that. A block with an element  */
/*    that is not finite reads as NaN. Keys are normed and rotated in 64      */
/*    bits, so that their codes are those of the exact rows. The scales of a  */
/*    cache of other origin may be any fp16 numbers of at most 8 significant  */
/*    bits up to 2720, and its codes 0 .. 15: then every value is exact in    */
/*    fp16, which the decode's products take.                                 */
/* ------------------------------------------------------------------------ */
typedef struct AiGpuPagedCacheQ4 {
    void* keyCodes;           /* 16-byte aligned, as the other three */
    void* valueCodes;
    void* keyScales;
    void* valueScales;
    const uint32_t* table;    /* [batch][tableStride], the first tableWidth of each row */
    const uint32_t* lengths;  /* [batch] */
    uint64_t batch, pages, pageSize, kvHeads, dim;  /* dim 64, 96, 128, 192 or 256 */
    uint64_t tableWidth, tableStride;               /* tableStride 0 means tableWidth */
    uint64_t pageStride, headStride, rowStride;     /* in rows; all 0: [pages][kvHeads][pageSize] */
} AiGpuPagedCacheQ4;

/* as AiGpuPagedAppend, into 4-bit pages */
typedef struct AiGpuPagedAppendQ4 {
    AiGpuPagedCacheQ4 cache;
    const void* k;
    const void* v;
    const uint32_t* starts;
    const float* kNorm;
    const float* rotaryFrequencies;
    float epsilon, normOffset, amplitude;
    uint32_t rotaryDims, interleaved, inType;
    uint64_t count, kStride, vStride;
    void* stream;
} AiGpuPagedAppendQ4;
AIGPU_ABI int aigpu_paged_append_q4(const AiGpuPagedAppendQ4* args);

/* The rows of the newest tokens (which ones, `starts` says as an append's) read back:
   the values that their codes stand for, rounded once to outType. Rows of k and v
   before starts[0] or from starts[batch] on stay as they were; a token without a
   place in the pool reads as NaN. With the lengths summed up as starts this is every
   sequence whole, as aigpu_packed_attention takes the keys of a chunk's documents.
   k and v share no element (slices of the same rows do not). Asynchronous, without
   scratch. */
typedef struct AiGpuPagedReadQ4 {
    AiGpuPagedCacheQ4 cache;
    void* k;                  /* [count][kvHeads][dim], outType; token t at t*kStride */
    void* v;                  /* the same at t*vStride */
    const uint32_t* starts;   /* [batch + 1], not decreasing, or NULL: one token a sequence */
    uint32_t outType, reserved;
    uint64_t count, kStride, vStride; /* strides 0 mean kvHeads*dim */
    void* stream;
} AiGpuPagedReadQ4;
AIGPU_ABI int aigpu_paged_read_q4(const AiGpuPagedReadQ4* args);

/* As aigpu_paged_decode_scored, over 4-bit pages: fp32 throughout, the products taking
   the pages' values exactly, q and the weights in two fp16 terms each: 22 bits, but
   none below 2^-38 of the head's largest element of q and 2^-40 of its largest weight. */
typedef struct AiGpuPagedDecodeQ4 {
    AiGpuPagedCacheQ4 cache;
    const void* q;
    float* out;
    const float* qNorm;
    const float* rotaryFrequencies;
    const float* slopes;      /* as AiGpuScores */
    float epsilon, normOffset, amplitude, scale, cap;
    uint32_t rotaryDims, interleaved, inType, outputGate, maxLength;
    uint64_t heads, qStride, qTokenStride;
    uint64_t window;
    void* workspace;
    uint64_t workspaceBytes;
    void* stream;
} AiGpuPagedDecodeQ4;
AIGPU_ABI int aigpu_paged_decode_q4(const AiGpuPagedDecodeQ4* args);
AIGPU_ABI uint64_t aigpu_paged_decode_q4_workspace(const AiGpuPagedDecodeQ4* args);

/* ------------------------------------------------------------------------ */
/* 14. Attention of the tokens of many documents in one call (prompts, or the */
/*    new tokens of conversations behind their cached keys). Document b has    */
/*    tokens starts[b] .. starts[b + 1] - 1 of q and out and keys              */
/*    keyStarts[b] .. keyStarts[b + 1] - 1 of k and v; its tokens are the last */
/*    of its keys' positions, 0, 1, ... A token at position i sees the keys j  */
/*    of its own document with                                                 */
/*      (j <= i or j < prefix[b]) and (window = 0 or i - j < window)           */
/*    with the scores s = scale q.k, then cap > 0: s = cap tanh(s / cap), then */
/*    slopes: s -= slopes[head] |i - j|. A token that sees nothing gets zeros  */
/*    (more tokens than keys: the first ones). Rows of out that no document    */
/*    has stay as they were. The starts do not decrease, nor pass count and    */
/*    keyCount (nothing outside is touched where they do, but documents may be */
/*    left out). A value that is not finite makes NaN or an infinity of its    */
/*    channel of the tokens that see it, and of nothing else; a key that makes */
/*    a score NaN or +infinity makes NaN of the tokens that see it, and so do  */
/*    scores that are all -infinity (as in 12's and 13's decode). Rows of no   */
/*    document may hold anything.                                              */
/*    Types: q, k, v of inType, out of outType. bf16 to bf16 rounds the        */
/*    weights to bf16 (their sum adds the rounded ones) and the result once;   */
/*    bf16 to fp32 takes the weights whole, in three terms; fp32 is fp32       */
/*    throughout. Rows of q, k and v are 16-byte aligned. No counterpart in    */
/*    the reference, whose call is one sequence's. Asynchronous.               */
/* ------------------------------------------------------------------------ */
typedef struct AiGpuPackedAttention {
    const void* q;            /* element (token, head, d) at token*qTokenStride + head*qHeadStride + d */
    const void* k;            /* the same with heads = kvHeads */
    const void* v;
    void* out;                /* apart from q, k and v (slices of the same rows may be) */
    const uint32_t* starts;   /* [documents + 1], or NULL: one document of all tokens and keys */
    const uint32_t* keyStarts;/* [documents + 1], or NULL: starts (keyCount = count) */
    const uint32_t* prefix;   /* [documents], or NULL: none */
    const float* slopes;      /* [heads], or NULL: none */
    float cap;                /* 0: none; otherwise 1e-6 .. 1e6 */
    float scale;              /* 0 means 1/sqrt(dim) */
    uint32_t inType, outType;
    uint64_t count, keyCount, documents, heads, kvHeads, dim;   /* dim 64, 96, 128, 192 or 256 */
    uint64_t window;          /* 0 = all */
    uint64_t qTokenStride, qHeadStride, kTokenStride, kHeadStride;  /* 0 mean heads*headStride and dim */
    uint64_t vTokenStride, vHeadStride, outTokenStride, outHeadStride;
    void* workspace;          /* device, 256-byte aligned; NULL: the backend's scratch */
    uint64_t workspaceBytes;
    void* stream;
} AiGpuPackedAttention;
AIGPU_ABI int aigpu_packed_attention(const AiGpuPackedAttention* args);
/* The workspace bytes of a call with these sizes and this window, no more than without
   one (0: none; UINT64_MAX: refused, as the call would be): few tokens over many keys
   are split over workgroups. How far, the sizes alone decide, as the starts are on the
   device: keyCount / documents keys each, of which a window leaves its own, and one
   workgroup of rows a kv head for each place, also those without tokens. A long history
   among many short ones or many empty places is therefore split less or not at all, and
   takes longer than by itself; a batch of chunks is best given without empty places.
   The workspace need not be zero-filled; calls that may run at once need one each. A
   call captured into a graph has to bring one where this is not 0. */
AIGPU_ABI uint64_t aigpu_packed_attention_workspace(const AiGpuPackedAttention* args);

/* ------------------------------------------------------------------------ */
/* Per-kernel timing. With profiling on, every launch is bracketed by a pair */
/* of hipEvents on the stream it runs on; aigpu_profile_read synchronises    */
/* and reports the summed device time and launch count of kernels whose name */
/* contains `kernel` since the last reset.                                   */
/* ------------------------------------------------------------------------ */
AIGPU_ABI void aigpu_profile(int enable);
AIGPU_ABI int aigpu_profile_read(const char* kernel, double* milliseconds, uint64_t* launches);
AIGPU_ABI void aigpu_profile_reset(void);

#ifdef __cplusplus
}
#endif

#endif /* AIGPU_ATTENTION_H */

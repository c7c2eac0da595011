// paged_scored.hip - one token's attention over bf16 pages, its scores capped or biased.
// A form of its own, so that the plain one keeps its registers. Bounded by the cache's bytes,
// as that one is: 24 sequences of up to 16 thousand under 16/8 heads of 256, capped, 1.67 GB in
// 295 us (5.7 TB/s); 64 of up to 5 thousand under 12/12 heads of 64, fp32 queries, biased, a
// window of 1024, 169 MB in 37 us (4.6).
#include "paged_attention.hpp"

namespace aigpu {

bool launch_paged_scored(const PagedDecodeParams& p, void* work, hipStream_t stream) {
    return launch_decode_as<PAGED_SCORED>("paged_scored_kernel", p, work, stream);
}

} // namespace aigpu

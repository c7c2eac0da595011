// paged_scored.hip - one token's attention over bf16 pages, its scores capped or biased.
#include "paged_attention.hpp"

namespace aigpu {

bool launch_paged_scored(const PagedDecodeParams& p, void* work, hipStream_t stream) {
    return launch_decode_as<PAGED_SCORED>("paged_scored_kernel", p, work, stream);
}

} // namespace aigpu

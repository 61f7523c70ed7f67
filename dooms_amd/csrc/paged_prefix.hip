// The packed prompts' kernel over the keys that groups of sequences share.
#include "paged_prefill_kernel.hpp"

namespace mx {

hipError_t launch_paged_prefix(const PagedAttnParams & p, int head_dim, int dtype, bool e4m3, uint32_t grid, hipStream_t stream) {
    if (dtype == 1) e4m3 ? launch_prefix<F16, true>(p, head_dim, grid, stream) : launch_prefix<F16, false>(p, head_dim, grid, stream);
    else e4m3 ? launch_prefix<BF16, true>(p, head_dim, grid, stream) : launch_prefix<BF16, false>(p, head_dim, grid, stream);
    return hipGetLastError();
}

}  // namespace mx

// The packed prompts' kernel over pages of e4m3 codes.
#include "paged_prefill_kernel.hpp"

namespace mx {

hipError_t launch_paged_prefill_e4m3(const PagedAttnParams & p, int head_dim, int dtype, const PagedPrefillPlan & plan, hipStream_t stream) {
    if (dtype == 1) launch_hd<F16, true>(p, head_dim, plan, stream);
    else launch_hd<BF16, true>(p, head_dim, plan, stream);
    return hipGetLastError();
}

}  // namespace mx

// The partials of sequences that share prefixes, over pages of the query rows' type.
#include "paged_shared_kernel.hpp"

namespace mx {

hipError_t launch_paged_shared(const PagedAttnParams & p, int head_dim, int dtype, int rt, hipStream_t stream) {
    return launch_shared<false>(p, head_dim, dtype, rt, stream);
}

}  // namespace mx

// The partials of sequences that share prefixes, over pages of e4m3 codes.
#include "paged_shared_kernel.hpp"

namespace mx {

hipError_t launch_paged_shared_e4m3(const PagedAttnParams & p, int head_dim, int dtype, int rt, hipStream_t stream) {
    return launch_shared<true>(p, head_dim, dtype, rt, stream);
}

}  // namespace mx

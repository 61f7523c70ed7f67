// The paged decode kernel behind that of the shared prefixes, over pages of the query rows' type.
#include "paged_decode_kernel.hpp"

namespace mx {

hipError_t launch_paged_decode_shared(const PagedAttnParams & p, int head_dim, int dtype, int rt, hipStream_t stream) {
    if (dtype == 1) launch_hd<F16, false, true>(p, head_dim, rt, 4, stream);
    else launch_hd<BF16, false, true>(p, head_dim, rt, 4, stream);
    return hipGetLastError();
}

}  // namespace mx

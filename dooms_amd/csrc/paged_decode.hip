// The paged decode kernel over pages of the query rows' type.
#include "paged_decode_kernel.hpp"

namespace mx {

hipError_t launch_paged_decode(const PagedAttnParams & p, int head_dim, int dtype, int rt, int waves, hipStream_t stream) {
    if (dtype == 1) launch_hd<F16, false>(p, head_dim, rt, waves, stream);
    else launch_hd<BF16, false>(p, head_dim, rt, waves, stream);
    return hipGetLastError();
}

}  // namespace mx

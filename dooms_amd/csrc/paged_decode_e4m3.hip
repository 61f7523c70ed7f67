// The paged decode kernel over pages of e4m3 codes.
#include "paged_decode_kernel.hpp"

namespace mx {

hipError_t launch_paged_decode_e4m3(const PagedAttnParams & p, int head_dim, int dtype, int rt, int waves, hipStream_t stream) {
    if (dtype == 1) launch_hd<F16, true>(p, head_dim, rt, waves, stream);
    else launch_hd<BF16, true>(p, head_dim, rt, waves, stream);
    return hipGetLastError();
}

}  // namespace mx

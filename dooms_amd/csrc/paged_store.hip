// The append to pages of the queries' type.
#include "paged_store_kernel.hpp"

namespace mx {

hipError_t launch_paged_store(const PagedStoreParams & p, int head_dim, int in_dtype, int dtype, hipStream_t stream) {
    return dtype == 1 ? launch_hd<F16, false>(p, head_dim, in_dtype, stream) : launch_hd<BF16, false>(p, head_dim, in_dtype, stream);
}

}  // namespace mx

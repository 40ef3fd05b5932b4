// The tcgen05 paged attention kernel for fp16 caches (paged_tc.cuh).
#include "paged_tc.cuh"

namespace tfx {
template int launch_paged_tc<kCodeF16>(const tfx_paged_cache*, const Paged&, const PagedAttn&, int64_t,
                                 cudaStream_t);
}  // namespace tfx

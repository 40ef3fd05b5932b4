// The tcgen05 paged attention kernel for int8 caches (paged_tc.cuh).
#include "paged_tc.cuh"

namespace tfx {
template int launch_paged_tc<kCodeI8>(const tfx_paged_cache*, const Paged&, const PagedAttn&, int64_t,
                                 cudaStream_t);
}  // namespace tfx

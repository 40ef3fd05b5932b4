// The mma.sync paged attention kernel for int8 caches (paged_rows.cuh).
#include "paged_rows.cuh"

namespace tfx {
template int launch_paged_rows<kCodeI8>(const Paged&, const PagedAttn&, int, int, bool, int64_t,
                                         cudaStream_t);
}  // namespace tfx

// The mma.sync paged attention kernel for e4m3 caches (paged_rows.cuh).
#include "paged_rows.cuh"

namespace tfx {
template int launch_paged_rows<kCodeE4M3>(const Paged&, const PagedAttn&, int, int, bool, int64_t,
                                         cudaStream_t);
}  // namespace tfx

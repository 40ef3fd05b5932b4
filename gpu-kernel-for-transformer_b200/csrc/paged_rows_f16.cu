// The mma.sync paged attention kernel for fp16 caches (paged_rows.cuh).
#include "paged_rows.cuh"

namespace tfx {
template int launch_paged_rows<kCodeF16>(const Paged&, const PagedAttn&, int, int, bool, int64_t,
                                         cudaStream_t);
}  // namespace tfx

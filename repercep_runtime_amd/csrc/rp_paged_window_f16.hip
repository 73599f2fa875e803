// rp_paged_window.hip's kernels for fp16 queries and an fp16 cache.
#include "rp_paged_window_kernels.h"

template void rp::launch_window<rp::kInF16, RP_CACHE_F16>(const WindowArgs&, const PagedView&, int64_t,
                                                 const WindowLaunch&, hipStream_t);

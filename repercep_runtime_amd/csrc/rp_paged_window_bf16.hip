// rp_paged_window.hip's kernels for bf16 queries and a bf16 cache.
#include "rp_paged_window_kernels.h"

template void rp::launch_window<rp::kInBf16, RP_CACHE_BF16>(const WindowArgs&, const PagedView&, int64_t,
                                                 const WindowLaunch&, hipStream_t);

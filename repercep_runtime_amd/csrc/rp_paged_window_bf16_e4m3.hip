// rp_paged_window.hip's kernels for bf16 queries and an e4m3fn cache.
#include "rp_paged_window_kernels.h"

template void rp::launch_window<rp::kInBf16, RP_CACHE_E4M3>(const WindowArgs&, const PagedView&, int64_t,
                                                 const WindowLaunch&, hipStream_t);

// Both kernels of rp_paged_window.hip and their launch for one pair of types.
#pragma once

#include "rp_paged_few.h"
#include "rp_paged_prompt.h"

template <int QT, int CT>
void rp::launch_window(const WindowArgs& a, const PagedView& c, int64_t D, const WindowLaunch& l,
                       hipStream_t st) {
  if (l.columns) launch_few<QT, CT>(a, c, D, l.columns, l.stream, st);
  else launch_prompt<QT, CT>(a, c, D, l.waves, st);
}

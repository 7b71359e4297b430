// Instantiations of the attention kernels for one element type, a translation unit each.
#pragma once
#include "attn_bwd.h"
#include "attn_host.h"

namespace amoe {

// Heads are padded to 64, 96 or 128 elements in LDS and registers (zeros that no memory is read for).  Operands that are not
// in whole aligned 16-byte chunks take the 128 form with element-wise edges, whatever their size.
#define AMOE_ATTN_SIZES(LAUNCH, TYPE, P)                                 \
  do {                                                                   \
    if (!attn_whole_chunks(P, sizeof(TYPE))) LAUNCH(TYPE, 128, true);    \
    else if ((P).d <= 64) LAUNCH(TYPE, 64, false);                       \
    else if ((P).d <= 96) LAUNCH(TYPE, 96, false);                       \
    else LAUNCH(TYPE, 128, false);                                       \
  } while (0)

template <typename T>
int launch_attn_fwd(const AttnParams& p, hipStream_t st) {
  if (p.splits > 0) {
    const dim3 grid((unsigned)((int64_t)p.B * p.G * p.splits * ((p.R * p.S + 31) / 32)));
#define AMOE_LAUNCH(TYPE, DP, EDGE) hipLaunchKernelGGL((&attn_fwd_split_kernel<TYPE, DP, EDGE>), grid, dim3(kAttnThreads), 0, st, p)
    AMOE_ATTN_SIZES(AMOE_LAUNCH, T, p);
#undef AMOE_LAUNCH
    if (p.splits > 1) {
      const dim3 join((unsigned)((int64_t)p.B * p.H * p.S)), block(kAttnThreads);
      hipLaunchKernelGGL((&attn_join_kernel<T>), join, block, 0, st, p);
    }
    return launch_rc();
  }
  const dim3 grid((unsigned)((int64_t)p.B * p.H * ((p.S + kAttnRows - 1) / kAttnRows)));
#define AMOE_LAUNCH(TYPE, DP, EDGE) hipLaunchKernelGGL((&attn_fwd_rows_kernel<TYPE, DP, EDGE>), grid, dim3(kAttnThreads), 0, st, p)
  AMOE_ATTN_SIZES(AMOE_LAUNCH, T, p);
#undef AMOE_LAUNCH
  return launch_rc();
}

template <typename T>
int launch_attn_bwd(const AttnParams& p, hipStream_t st) {
  if (p.S > 0) {
    const dim3 grid((unsigned)((int64_t)p.B * p.H * ((p.S + kAttnRows - 1) / kAttnRows)));
#define AMOE_LAUNCH(TYPE, DP, EDGE) hipLaunchKernelGGL((&attn_bwd_q_kernel<TYPE, DP, EDGE>), grid, dim3(kAttnThreads), 0, st, p)
    AMOE_ATTN_SIZES(AMOE_LAUNCH, T, p);          // (leaves delta for the next)
#undef AMOE_LAUNCH
  }
  if (p.T > 0 && p.dk) {
#define AMOE_LAUNCH(TYPE, DP, EDGE)                                                                             \
  do {                                                                                                          \
    using Shape = AttnKvShape<TYPE, DP, EDGE>;                                                                  \
    const dim3 grid((unsigned)((int64_t)p.B * p.G * ((p.T + 32 * Shape::KW - 1) / (32 * Shape::KW))));          \
    hipLaunchKernelGGL((&attn_bwd_kv_kernel<TYPE, DP, EDGE>), grid, dim3(Shape::kThreads), 0, st, p); \
  } while (0)
    AMOE_ATTN_SIZES(AMOE_LAUNCH, T, p);
#undef AMOE_LAUNCH
  }
  return launch_rc();
}

}  // namespace amoe

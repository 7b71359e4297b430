// Instantiations of the attention kernels for one element type, a translation unit each.
#pragma once
#include "attn_bwd.h"
#include "attn_host.h"

namespace amoe {

// Heads are padded to 64, 96 or 128 elements in LDS and registers (zeros that no memory is read for).  Operands that are not
// in whole aligned 16-byte chunks take the 128 form with element-wise edges, whatever their size.
#define AMOE_ATTN_SIZES(KERNEL, TYPE, GRID, ST, P)                                                                  \
  do {                                                                                                              \
    const dim3 block(kAttnThreads);                                                                                 \
    if (!attn_whole_chunks(P, sizeof(TYPE))) hipLaunchKernelGGL((&KERNEL<TYPE, 128, true>), GRID, block, 0, ST, P);  \
    else if ((P).d <= 64) hipLaunchKernelGGL((&KERNEL<TYPE, 64, false>), GRID, block, 0, ST, P);                    \
    else if ((P).d <= 96) hipLaunchKernelGGL((&KERNEL<TYPE, 96, false>), GRID, block, 0, ST, P);                    \
    else hipLaunchKernelGGL((&KERNEL<TYPE, 128, false>), GRID, block, 0, ST, P);                                    \
  } while (0)

template <typename T>
int launch_attn_fwd(const AttnParams& p, hipStream_t st) {
  if (p.splits > 0) {
    const dim3 grid((unsigned)((int64_t)p.B * p.G * p.splits * ((p.R * p.S + 31) / 32)));
    AMOE_ATTN_SIZES(attn_fwd_split_kernel, T, grid, st, p);
    if (p.splits > 1) {
      const dim3 join((unsigned)(((int64_t)p.B * p.H * p.S + 3) / 4)), block(kAttnThreads);
      hipLaunchKernelGGL((&attn_join_kernel<T>), join, block, 0, st, p);
    }
    return launch_rc();
  }
  const dim3 grid((unsigned)((int64_t)p.B * p.H * ((p.S + kAttnRows - 1) / kAttnRows)));
  AMOE_ATTN_SIZES(attn_fwd_rows_kernel, T, grid, st, p);
  return launch_rc();
}

template <typename T>
int launch_attn_bwd(const AttnParams& p, hipStream_t st) {
  if (p.S > 0) {
    const dim3 grid_q((unsigned)((int64_t)p.B * p.H * ((p.S + kAttnRows - 1) / kAttnRows)));
    AMOE_ATTN_SIZES(attn_bwd_q_kernel, T, grid_q, st, p);          // (leaves delta for the next)
  }
  if (p.T > 0 && p.dk) {
    const dim3 grid_kv((unsigned)((int64_t)p.B * p.G * ((p.T + kAttnRows - 1) / kAttnRows)));
    AMOE_ATTN_SIZES(attn_bwd_kv_kernel, T, grid_kv, st, p);
  }
  return launch_rc();
}

}  // namespace amoe

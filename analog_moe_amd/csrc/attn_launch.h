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

// Waves over the rows of a workgroup (AttnShape) by how many workgroups there are: four where two can be on every CU, else two,
// and one where those would not give every CU a workgroup; the tiles' room allowing.  Measured, forward pass: 256 workgroups of
// 128 rows (2 sequences of 1024, 16 heads of 64, fp32) 87 us, 512 of 64 62 us, 1024 of 32 75 us; 256 of 128 (2 x 1003 queries over
// 5003 keys, 16 heads of 128, bf16) 100 us, 512 of 64 75 us, 1024 of 32 168 us; 8 of 128 (2 x 100, 4 heads of 32, fp32) 14 us, 16 of
// 64 10 us, 32 of 32 8 us; 2048 of 128 (16 x 1024, 16 heads of 64, bf16) 70 us, 4096 of 64 88 us.
template <template <int> class Launch, bool FITS2, bool FITS1>
int launch_attn_rows(const AttnParams& p, hipStream_t st) {
  const int64_t heads = (int64_t)p.B * p.H, want = 2 * num_compute_units();
  if constexpr (FITS2) {
    if (heads * ((p.S + 127) / 128) < want) {
      if constexpr (FITS1) {
        if (heads * ((p.S + 63) / 64) < want / 2) return Launch<1>::run(p, st);
      }
      return Launch<2>::run(p, st);
    }
  }
  return Launch<4>::run(p, st);
}

template <typename T, int DP, bool EDGE> struct AttnFwdRows {
  template <int RW> struct Launch {
    static int run(const AttnParams& p, hipStream_t st) {
      const dim3 grid((unsigned)((int64_t)p.B * p.H * ((p.S + 32 * RW - 1) / (32 * RW))));
      hipLaunchKernelGGL((&attn_fwd_rows_kernel<T, DP, EDGE, RW>), grid, dim3(kAttnThreads), 0, st, p);
      return launch_rc();
    }
  };
};
template <typename T, int DP, bool EDGE> struct AttnBwdRows {
  template <int RW> struct Launch {
    static int run(const AttnParams& p, hipStream_t st) {
      const dim3 grid((unsigned)((int64_t)p.B * p.H * ((p.S + 32 * RW - 1) / (32 * RW))));
      hipLaunchKernelGGL((&attn_bwd_q_kernel<T, DP, EDGE, RW>), grid, dim3(kAttnThreads), 0, st, p);
      return launch_rc();
    }
  };
};

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
  int rc = AMOE_OK;
#define AMOE_LAUNCH(TYPE, DP, EDGE)                                                                             \
  rc = launch_attn_rows<AttnFwdRows<TYPE, DP, EDGE>::template Launch, !EDGE && AttnShape<TYPE, DP, EDGE, 2>::kFits, \
                        !EDGE && AttnShape<TYPE, DP, EDGE, 1>::kFits>(p, st)
  AMOE_ATTN_SIZES(AMOE_LAUNCH, T, p);
#undef AMOE_LAUNCH
  return rc;
}

// Copies of the waves over the queries: two where there are two workgroups for every CU, else four.  Measured: 324 workgroups
// (6 padded sequences of 1717, 2 key heads of 80, fp16) 141 us with two, 108 us with four; 512 (2 x 1024, 16 heads of 64, fp32) 119
// and 104 us; 4096 (16 x 1024, 16 heads of 64, bf16) 125 and 214 us.
template <typename T, int DP, bool EDGE, int QW>
int launch_attn_kv_of(const AttnParams& p, int64_t groups, hipStream_t st) {
  hipLaunchKernelGGL((&attn_bwd_kv_kernel<T, DP, EDGE, QW>), dim3((unsigned)groups), dim3(AttnKvShape<T, DP, EDGE, QW>::kThreads), 0, st, p);
  return launch_rc();
}
template <typename T, int DP, bool EDGE>
int launch_attn_kv(const AttnParams& p, hipStream_t st) {
  constexpr bool kTwo = AttnKvShape<T, DP, EDGE, 2>::kFits, kFour = !EDGE && AttnKvShape<T, DP, EDGE, 4>::kFits;
  static_assert(kTwo || kFour, "one of them");
  const int64_t groups = (int64_t)p.B * p.G * ((p.T + 63) / 64);
  if constexpr (kFour) {
    if (!kTwo || groups <= 2 * num_compute_units()) return launch_attn_kv_of<T, DP, EDGE, 4>(p, groups, st);
  }
  if constexpr (kTwo) return launch_attn_kv_of<T, DP, EDGE, 2>(p, groups, st);
  return AMOE_EUNSUPPORTED;
}

template <typename T>
int launch_attn_bwd(const AttnParams& p, hipStream_t st) {
  int rc = AMOE_OK;
  if (p.S > 0) {
#define AMOE_LAUNCH(TYPE, DP, EDGE)                                                                             \
  rc = launch_attn_rows<AttnBwdRows<TYPE, DP, EDGE>::template Launch, !EDGE && AttnShape<TYPE, DP, EDGE, 2>::kFits, \
                        !EDGE && AttnShape<TYPE, DP, EDGE, 1>::kFits>(p, st)
    AMOE_ATTN_SIZES(AMOE_LAUNCH, T, p);          // (leaves rows for the next)
#undef AMOE_LAUNCH
    if (rc) return rc;
  }
  if (p.T > 0 && p.dk) {
#define AMOE_LAUNCH(TYPE, DP, EDGE) rc = launch_attn_kv<TYPE, DP, EDGE>(p, st)
    AMOE_ATTN_SIZES(AMOE_LAUNCH, T, p);
#undef AMOE_LAUNCH
  }
  return rc;
}

}  // namespace amoe

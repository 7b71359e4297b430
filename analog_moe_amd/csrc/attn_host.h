// Host side of the attention entry points, shared by the translation units of the element types.
#pragma once
#include <amoe.h>
#include "attn_tile.h"
#include "host_util.h"

namespace amoe {

// Whole aligned 16-byte chunks everywhere: the kernels without edges.
inline bool attn_whole_chunks(const AttnParams& p, size_t es) { return p.vec == 2 && (p.d * es) % 16 == 0; }

int launch_attn_fwd_f32(const AttnParams& p, hipStream_t st);
int launch_attn_fwd_bf16(const AttnParams& p, hipStream_t st);
int launch_attn_fwd_f16(const AttnParams& p, hipStream_t st);
// rows that share `prefix` and have keys of their own in `own`: parts of both, and all of them joined
struct AttnShared {
  AttnParams prefix, own, join;
  int prefix_rw, own_rw;             // waves over the rows of a workgroup (prefix 4, 2; own 4, then prefix 4 too); 0: attn_split_body
};
int launch_attn_shared_f32(const AttnShared& s, hipStream_t st);
int launch_attn_shared_bf16(const AttnShared& s, hipStream_t st);
int launch_attn_shared_f16(const AttnShared& s, hipStream_t st);
int launch_attn_bwd_f32(const AttnParams& p, hipStream_t st);
int launch_attn_bwd_bf16(const AttnParams& p, hipStream_t st);
int launch_attn_bwd_f16(const AttnParams& p, hipStream_t st);

}  // namespace amoe

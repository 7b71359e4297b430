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
int launch_attn_bwd_f32(const AttnParams& p, hipStream_t st);
int launch_attn_bwd_bf16(const AttnParams& p, hipStream_t st);
int launch_attn_bwd_f16(const AttnParams& p, hipStream_t st);

}  // namespace amoe

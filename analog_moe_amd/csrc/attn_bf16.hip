// The attention kernels, bf16 elements.
#include "attn_launch.h"

namespace amoe {

int launch_attn_fwd_bf16(const AttnParams& p, hipStream_t st) { return launch_attn_fwd<uint16_t>(p, st); }
int launch_attn_bwd_bf16(const AttnParams& p, hipStream_t st) { return launch_attn_bwd<uint16_t>(p, st); }
int launch_attn_shared_bf16(const AttnShared& s, hipStream_t st) { return launch_attn_shared<uint16_t>(s, st); }

}  // namespace amoe

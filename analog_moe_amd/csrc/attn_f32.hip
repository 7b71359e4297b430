// The attention kernels, fp32 elements.
#include "attn_launch.h"

namespace amoe {

int launch_attn_fwd_f32(const AttnParams& p, hipStream_t st) { return launch_attn_fwd<float>(p, st); }
int launch_attn_bwd_f32(const AttnParams& p, hipStream_t st) { return launch_attn_bwd<float>(p, st); }
int launch_attn_shared_f32(const AttnShared& s, hipStream_t st) { return launch_attn_shared<float>(s, st); }

}  // namespace amoe

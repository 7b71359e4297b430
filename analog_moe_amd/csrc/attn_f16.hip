// The attention kernels, fp16 elements.
#include "attn_launch.h"

namespace amoe {

int launch_attn_fwd_f16(const AttnParams& p, hipStream_t st) { return launch_attn_fwd<f16_t>(p, st); }
int launch_attn_bwd_f16(const AttnParams& p, hipStream_t st) { return launch_attn_bwd<f16_t>(p, st); }
int launch_attn_shared_f16(const AttnShared& s, hipStream_t st) { return launch_attn_shared<f16_t>(s, st); }

}  // namespace amoe

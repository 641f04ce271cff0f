// Attention forward (attention_fwd_kernels.h) within a sliding window whose first tokens stay visible.
#include "attention_fwd_kernels.h"

namespace lwl {

int64_t attention_window_fwd_work(const AttnArgs& a) { return fwd_work<kWindow>(a); }

bool attention_window_fwd_fits(const AttnArgs& a) { return fwd_fits<kWindow>(a); }

hipError_t launch_attention_window_fwd(AttnArgs a, hipStream_t s) { return launch_fwd<kWindow>(a, s); }

}  // namespace lwl

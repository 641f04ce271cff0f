// Attention backward (attention_bwd_kernels.h) within a sliding window whose first tokens stay visible.
#include "attention_bwd_kernels.h"

namespace lwl {

int64_t attention_window_bwd_work(const AttnArgs& a) { return bwd_work<kWindow>(a); }

bool attention_window_bwd_fits(const AttnArgs& a) { return bwd_fits<kWindow>(a); }

hipError_t launch_attention_window_bwd(AttnArgs a, hipStream_t s) { return launch_bwd<kWindow>(a, s); }

}  // namespace lwl

// Attention backward (attention_bwd_kernels.h) over all keys that lengths and causal order leave.
#include "attention_bwd_kernels.h"

namespace lwl {

int64_t attention_bwd_work(const AttnArgs& a) { return bwd_work<kAll>(a); }

bool attention_bwd_fits(const AttnArgs& a) { return bwd_fits<kAll>(a); }

hipError_t launch_attention_bwd(AttnArgs a, hipStream_t s) { return launch_bwd<kAll>(a, s); }

}  // namespace lwl

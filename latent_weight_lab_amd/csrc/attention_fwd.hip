// Attention forward (attention_fwd_kernels.h) over all keys that lengths and causal order leave.
#include "attention_fwd_kernels.h"

namespace lwl {

int64_t attention_fwd_work(const AttnArgs& a) { return fwd_work<kAll>(a); }

bool attention_fwd_fits(const AttnArgs& a) { return fwd_fits<kAll>(a); }

hipError_t launch_attention_fwd(AttnArgs a, hipStream_t s) { return launch_fwd<kAll>(a, s); }

}  // namespace lwl

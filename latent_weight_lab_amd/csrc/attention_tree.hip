// Attention (attention_fwd_kernels.h) of a tree of drafted tokens over a cache.
#include "attention_fwd_kernels.h"

namespace lwl {

int64_t attention_tree_work(const AttnArgs& a) { return fwd_work<kTree>(a); }

bool attention_tree_fits(const AttnArgs& a) { return fwd_fits<kTree>(a); }

hipError_t launch_attention_tree(AttnArgs a, hipStream_t s) { return launch_fwd<kTree>(a, s); }

}  // namespace lwl

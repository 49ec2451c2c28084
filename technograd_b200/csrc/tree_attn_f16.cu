// tree_attn_f16.cu -- attention of drafted tokens, f16 caches.
#include "tree_attn_run.cuh"

namespace tgc {
template int attn_type<__half>(const AttnArgs &, const AttnPlan &, cudaStream_t);
} // namespace tgc

// tree_attn_f32.cu -- attention of drafted tokens, f32 caches.
#include "tree_attn_run.cuh"

namespace tgc {
template int attn_type<float>(const AttnArgs &, const AttnPlan &, cudaStream_t);
} // namespace tgc

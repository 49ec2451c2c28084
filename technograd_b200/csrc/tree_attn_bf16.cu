// tree_attn_bf16.cu -- attention of drafted tokens, bf16 caches.
#include "tree_attn_run.cuh"

namespace tgc {
template int attn_type<__nv_bfloat16>(const AttnArgs &, const AttnPlan &, cudaStream_t);
} // namespace tgc

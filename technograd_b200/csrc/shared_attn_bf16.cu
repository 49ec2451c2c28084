// shared_attn_bf16.cu -- attention below shared prefixes, bf16 caches.
#include "shared_attn.cuh"

namespace tgc {
template int shared_type<__nv_bfloat16>(const JoinArgs &, const SharedPlan &, const CUtensorMap *, cudaStream_t);
} // namespace tgc

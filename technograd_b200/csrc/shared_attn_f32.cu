// shared_attn_f32.cu -- attention below shared prefixes, f32 caches.
#include "shared_attn.cuh"

namespace tgc {
template int shared_type<float>(const JoinArgs &, const SharedPlan &, const CUtensorMap *, cudaStream_t);
} // namespace tgc

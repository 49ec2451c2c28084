// shared_attn_f16.cu -- attention below shared prefixes, f16 caches.
#include "shared_attn.cuh"

namespace tgc {
template int shared_type<__half>(const JoinArgs &, const SharedPlan &, const CUtensorMap *, cudaStream_t);
} // namespace tgc

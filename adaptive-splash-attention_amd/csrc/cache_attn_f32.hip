// Attention over the 4-bit cache (cache_attn_kernel.hpp) for fp32 queries.
#include "cache_attn_kernel.hpp"

namespace asa {

hipError_t launch_cache_attn_f32(const CacheAttnParams& p, hipStream_t s) { return launch_cache_attn_t<float>(p, s); }

}  // namespace asa

// Attention over the 4-bit cache (cache_attn_kernel.hpp) for fp16 queries.
#include "cache_attn_kernel.hpp"

namespace asa {

hipError_t launch_cache_attn_f16(const CacheAttnParams& p, hipStream_t s) { return launch_cache_attn_t<h16>(p, s); }

}  // namespace asa

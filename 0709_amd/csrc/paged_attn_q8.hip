// Paged attention over 8-bit caches.
#include "paged_launch.hpp"

namespace atlas {

int launch_paged_attn_q8(const PagedAttnArgs& a, hipStream_t stream) {
  return a.p.cache == ATLAS_CACHE_E4M3 ? launch_paged_attn_kind<kCacheE4M3>(a, stream)
                                       : launch_paged_attn_kind<kCacheInt8>(a, stream);
}

}  // namespace atlas

// Paged attention over 8-bit caches (kernel in paged_attn.hpp).
#include "paged_attn.hpp"

namespace atlas {

int launch_paged_attn_q8(const PagedAttnArgs& a, hipStream_t stream) {
  return a.p.cache == ATLAS_CACHE_E4M3 ? launch_paged_attn_kind<kCacheE4M3>(a, stream)
                                       : launch_paged_attn_kind<kCacheInt8>(a, stream);
}

}  // namespace atlas

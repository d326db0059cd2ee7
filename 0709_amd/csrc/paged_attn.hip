// Paged attention from device-side metadata: argument checks, and the kernels
// over 16-bit caches.
#include "paged_launch.hpp"

namespace atlas {

int launch_paged_attn_16bit(const PagedAttnArgs& a, hipStream_t stream) {
  return a.p.dtype == ATLAS_DTYPE_BF16 ? launch_paged_attn_kind<kCacheBf16>(a, stream)
                                       : launch_paged_attn_kind<kCacheF16>(a, stream);
}

}  // namespace atlas

using namespace atlas;

extern "C" int atlas_paged_attn(const atlas_paged_attn_t* args, void* stream) {
  ATLAS_REQUIRE(args != nullptr, "args must not be NULL");
  PagedAttnArgs a{};
  a.p = *args;
  const atlas_paged_attn_t& p = a.p;
  ATLAS_REQUIRE(p.q && p.kv && p.out, "q, kv and out must not be NULL");
  ATLAS_REQUIRE(p.qo_indptr && p.kv_indptr && p.kv_last_page_len && (p.kv_indices || p.num_indices == 0),
                "indptr / indices / last_page_len arrays must not be NULL");
  ATLAS_REQUIRE(p.batch > 0 && p.nnz >= 0, "batch must be positive and nnz non-negative");
  ATLAS_REQUIRE(p.num_kv_heads > 0 && p.num_qo_heads > 0 && p.num_qo_heads % p.num_kv_heads == 0,
                "num_qo_heads must be a positive multiple of num_kv_heads");
  if (p.head_dim != 64 && p.head_dim != 128) {
    set_error("head_dim %d is not supported (64 or 128)", p.head_dim);
    return ATLAS_EUNSUPPORTED;
  }
  ATLAS_REQUIRE(p.page_size > 0 && p.num_pages > 0 && p.num_indices >= 0, "page_size and num_pages must be positive");
  ATLAS_REQUIRE(p.dtype == ATLAS_DTYPE_F16 || p.dtype == ATLAS_DTYPE_BF16, "unknown dtype %d", p.dtype);
  ATLAS_REQUIRE(p.cache >= ATLAS_CACHE_16BIT && p.cache <= ATLAS_CACHE_INT8, "unknown cache type %d", p.cache);
  ATLAS_REQUIRE(p.cache == ATLAS_CACHE_16BIT || p.kv_scales != nullptr, "an 8-bit cache needs kv_scales");
  ATLAS_REQUIRE(p.mask_mode >= 0 && p.mask_mode <= 2, "unknown mask mode %d", p.mask_mode);
  ATLAS_REQUIRE(p.mask_mode != 1 || (p.tree_mask && p.mask_col_start && p.mask_words >= 1),
                "a tree mask needs its words and column starts");
  ATLAS_REQUIRE(p.mask_mode == 2 || (p.window_left < 0 && p.prefix_lens == nullptr),
                "windows and prefixes go with the causal mask");
  ATLAS_REQUIRE(p.mask_mode != 1 || p.alibi_slopes == nullptr, "a distance bias does not go with a tree mask");
  ATLAS_REQUIRE(p.block_rows > 0 && p.block_rows % 16 == 0 && p.block_rows <= (p.single_token ? 16 : 256),
                "block_rows must be a multiple of 16, up to 256 (16 for single tokens), got %d", p.block_rows);
  ATLAS_REQUIRE(!p.single_token || p.mask_mode != 1, "single_token does not go with a tree mask");
  ATLAS_REQUIRE(p.row_blocks > 0 && p.num_splits > 0 && p.split_keys > 0 && p.split_keys % 64 == 0,
                "row_blocks, num_splits and split_keys (a multiple of 64) must be positive");
  ATLAS_REQUIRE(p.soft_cap == 0.f || (p.soft_cap >= 1e-37f && p.soft_cap <= ATLAS_PAGED_ATTN_MAX_SOFT_CAP),
                "soft_cap must be 0 (none) or lie in [1e-37, %d]", ATLAS_PAGED_ATTN_MAX_SOFT_CAP);
  ATLAS_REQUIRE(p.sm_scale >= -1e37f && p.sm_scale <= 1e37f, "sm_scale must lie in [-1e37, 1e37]");
  // rows and lanes load 16 bytes (V of an 8-bit cache or head_dim 64: less)
  const int es = p.cache == ATLAS_CACHE_16BIT ? 2 : 1;
  ATLAS_REQUIRE((reinterpret_cast<uintptr_t>(p.q) & 15) == 0 && p.q_stride_token % 8 == 0 && p.q_stride_head % 8 == 0,
                "q must be 16-byte aligned with strides of 8 elements");
  ATLAS_REQUIRE((reinterpret_cast<uintptr_t>(p.out) & 15) == 0 && p.out_stride_token % 8 == 0 &&
                    p.out_stride_head % 8 == 0,
                "out must be 16-byte aligned with strides of 8 elements");
  ATLAS_REQUIRE((reinterpret_cast<uintptr_t>(p.kv) & 15) == 0 && p.page_stride % 16 == 0 && p.v_offset % 16 == 0 &&
                    p.token_stride % 16 == 0 && p.head_stride % 16 == 0,
                "the cache must be 16-byte aligned with strides of 16 bytes");
  ATLAS_REQUIRE(p.token_stride >= p.head_dim * es, "token_stride does not cover a head's row");
  // (a tile past the last key still has positions below 2^31)
  if (p.num_indices >= (int64_t(1) << 31) || p.num_indices * p.page_size >= (int64_t(1) << 31) - 4096 || p.nnz >= (int64_t(1) << 31) / p.num_qo_heads ||
      p.token_stride * p.page_size >= (int64_t(1) << 31)) {
    set_error("page tables of 2^31 - 4096 tokens or more, and pages of 2^31 bytes or more, are not supported");
    return ATLAS_EUNSUPPORTED;
  }
  const int64_t blocks = int64_t(p.batch) * p.num_kv_heads * p.row_blocks;
  const int64_t rows = blocks * p.num_splits * p.block_rows;
  if (blocks * p.num_splits >= (int64_t(1) << 23)) {
    set_error("%lld workgroups are too many", static_cast<long long>(blocks * p.num_splits));
    return ATLAS_EUNSUPPORTED;
  }
  if (p.num_splits > 1) {
    ATLAS_REQUIRE(p.workspace != nullptr && (reinterpret_cast<uintptr_t>(p.workspace) & 15) == 0 &&
                      p.workspace_bytes >= rows * ATLAS_PAGED_ATTN_ROW_BYTES(p.head_dim),
                  "the split states need %lld workspace bytes, 16-byte aligned, got %lld",
                  static_cast<long long>(rows * ATLAS_PAGED_ATTN_ROW_BYTES(p.head_dim)),
                  static_cast<long long>(p.workspace_bytes));
  }
  if (p.nnz == 0) return ATLAS_OK;
  a.scale_log2 = p.sm_scale * kPaLog2e;
  // (scores reach the cap multiplied by log2(e) already)
  a.cap_in = p.soft_cap > 0.f ? 2.f / p.soft_cap : 0.f;
  a.cap_out = p.soft_cap * kPaLog2e;
  a.group = p.num_qo_heads / p.num_kv_heads;
  int bits = 0;
  while ((int64_t(1) << bits) < p.page_size) ++bits;
  a.page_magic = uint32_t(((uint64_t(1) << (31 + bits)) + p.page_size - 1) / p.page_size);
  a.page_bits = 31 + bits;
  return p.cache == ATLAS_CACHE_16BIT ? launch_paged_attn_16bit(a, static_cast<hipStream_t>(stream))
                                      : launch_paged_attn_q8(a, static_cast<hipStream_t>(stream));
}

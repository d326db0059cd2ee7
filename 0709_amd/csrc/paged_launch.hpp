// Launches of the paged attention kernels over one kind of cache.
#pragma once

#include "paged_rows.hpp"
#include "paged_stream.hpp"

namespace atlas {
namespace {

// Few rows stream: as many row tiles as the registers hold beside a step's K and V (page
// sizes that look every key up: one; 16-bit rows: two; codes: three).
template <int KIND, int D, bool PAGE16, bool SCORED>
void launch_paged_kernel(const PagedAttnArgs& a, hipStream_t stream) {
  const atlas_paged_attn_t& p = a.p;
  const int64_t units = int64_t(p.batch) * p.num_kv_heads * p.num_splits;
  const dim3 grid(static_cast<unsigned>(p.row_blocks == 1 ? units : (units + 7) / 8 * 8 * p.row_blocks));
  const dim3 block(kPaThreads);
  if (p.single_token) {
    hipLaunchKernelGGL((paged_stream_kernel<KIND, D, 1, PAGE16, SCORED, false>), grid, block, 0, stream, a);
    return;
  }
  if (p.block_rows <= 16) {
    hipLaunchKernelGGL((paged_stream_kernel<KIND, D, 1, PAGE16, SCORED, true>), grid, block, 0, stream, a);
    return;
  }
  if constexpr (PAGE16) {
    if (p.block_rows <= 32) {
      hipLaunchKernelGGL((paged_stream_kernel<KIND, D, 2, PAGE16, SCORED, true>), grid, block, 0, stream, a);
      return;
    }
    if constexpr (Cache<KIND>::kQuant) {
      if (p.block_rows <= 48) {
        hipLaunchKernelGGL((paged_stream_kernel<KIND, D, 3, PAGE16, SCORED, true>), grid, block, 0, stream, a);
        return;
      }
    }
  }
  hipLaunchKernelGGL((paged_rows_kernel<KIND, D, PAGE16, SCORED>), grid, dim3(kRowThreads), 0, stream, a);
}

template <int KIND, int D>
int launch_paged_attn(const PagedAttnArgs& a, hipStream_t stream) {
  const atlas_paged_attn_t& p = a.p;
  const bool scored = p.soft_cap > 0.f || p.alibi_slopes != nullptr || p.sm_scale < 0.f;
  // (page sizes that are no multiple of 16 are bound by looking keys up; they take the general
  // scores: 48 bf16 rows over 8 x 4096 keys take 47.7 us in pages of 24, 43.6 in pages of 16)
  if (p.page_size % 16 != 0) launch_paged_kernel<KIND, D, false, true>(a, stream);
  else if (scored) launch_paged_kernel<KIND, D, true, true>(a, stream);
  else launch_paged_kernel<KIND, D, true, false>(a, stream);
  int rc = launch_status("paged attention kernel");
  if (rc || p.num_splits == 1) return rc;
  const dim3 mgrid(static_cast<unsigned>(p.batch * p.num_kv_heads * p.row_blocks), p.block_rows / 16);
  hipLaunchKernelGGL((paged_attn_merge_kernel<D>), mgrid, dim3(256), 0, stream, a);
  return launch_status("paged_attn_merge_kernel");
}

template <int KIND>
int launch_paged_attn_kind(const PagedAttnArgs& a, hipStream_t stream) {
  return a.p.head_dim == 128 ? launch_paged_attn<KIND, 128>(a, stream) : launch_paged_attn<KIND, 64>(a, stream);
}

}  // namespace
}  // namespace atlas

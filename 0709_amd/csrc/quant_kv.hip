// Writes into 8-bit caches: the quantising append and the commit of a route.
//
// A block is one page's rows of one KV head and of K or V; its scale is a power
// of two, so changing it shifts the values by whole binary places: an e4m3 value stays
// as it is unless it falls below the format's normal range, an int8 value is
// rounded once more, and since the shifts only go one way, all the roundings of a row
// together are off by less than one step of the last scale.
#include "quant8.hpp"

namespace atlas {
namespace {

typedef uint32_t w4 __attribute__((ext_vector_type(4)));
typedef uint32_t w2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));

constexpr int kAppendThreads = 256;

struct QuantTables {
  char* kv[ATLAS_MAX_LAYERS_PER_LAUNCH];
  float* scales[ATLAS_MAX_LAYERS_PER_LAUNCH];
};
struct RowTables {
  const char* k[ATLAS_MAX_LAYERS_PER_LAUNCH];
  const char* v[ATLAS_MAX_LAYERS_PER_LAUNCH];
};

struct QuantGeom {
  int64_t page_stride, v_offset, token_stride, head_stride;  // bytes
  int64_t scale_page, scale_kv, scale_head;                  // elements
  int64_t num_pages, num_indices;
  int page_size, page_shift, heads, head_dim;
};

struct Appends {
  const int32_t* indptr;
  const int32_t* kv_indptr;
  const int32_t* kv_indices;
  const int32_t* last_page_len;
  int64_t nnz, src_stride;  // src_stride: elements between tokens
  int64_t max_append;
  int batch, pages;  // pages: most pages a request's rows touch
  int layers;
};

template <bool BF16>
__device__ __forceinline__ void to_floats(w4 v, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF16) {
      f[2 * i] = __uint_as_float(v[i] << 16);
      f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    } else {
      const h2 h = __builtin_bit_cast(h2, uint32_t(v[i]));
      f[2 * i] = float(h[0]);
      f[2 * i + 1] = float(h[1]);
    }
  }
}

// One unit (a touched page's rows of one head, K or V, of one layer) per UNIT
// threads.  Two passes over the unit's new rows: their largest value, then the codes.
template <int CACHE, bool BF16, int UNIT>
__global__ __launch_bounds__(kAppendThreads) void kv_append_quantized_kernel(QuantTables qt, RowTables st, QuantGeom g,
                                                                             Appends a) {
  typedef Quant8<CACHE> Q;
  __shared__ float top_lds[kAppendThreads / 64];
  const int per_block = kAppendThreads / UNIT;
  const int t = threadIdx.x % UNIT;
  // units: head fastest, then K / V, page, request, layer
  int64_t u = int64_t(blockIdx.x) * per_block + threadIdx.x / UNIT;
  const int64_t units = int64_t(a.layers) * a.batch * a.pages * 2 * g.heads;
  bool live = u < units;
  if (!live) u = 0;
  const int head = int(u % g.heads);
  u /= g.heads;
  const int kv = int(u & 1);
  u >>= 1;
  const int touched = int(u % a.pages);
  u /= a.pages;
  const int b = int(u % a.batch);
  const int layer = int(u / a.batch);

  const int64_t r0 = min(max(int64_t(a.indptr[b]), int64_t(0)), a.nnz);
  const int64_t r1 = min(max(int64_t(a.indptr[b + 1]), r0), a.nnz);
  const int64_t pt = min(max(int64_t(a.kv_indptr[b]), int64_t(0)), g.num_indices);
  const int64_t np = min(max(int64_t(a.kv_indptr[b + 1]), pt), g.num_indices) - pt;
  const int last = min(max(a.last_page_len[b], 0), g.page_size);
  const int64_t len = np > 0 ? (np - 1) * g.page_size + last : 0;
  const int64_t lo = len - (r1 - r0);                      // position of the first new row
  const int64_t hi = min(len, lo + a.max_append);          // end of the new rows
  const int64_t first = max(lo, int64_t(0));
  const int64_t lp = (g.page_shift >= 0 ? first >> g.page_shift : first / g.page_size) + touched;
  const int64_t p0 = lp * g.page_size;
  live = live && p0 < hi && lp < np;
  const int64_t page = live ? a.kv_indices[pt + lp] : 0;
  live = live && page >= 0 && page < g.num_pages;
  const int o0 = int(max(first, p0) - p0);                       // first new row's place in the page
  const int o1 = live ? int(min(hi - p0, int64_t(g.page_size))) : o0;  // behind the last
  const int vpr = g.head_dim / 8;  // vectors of 8 values per row
  const int nvec = (o1 - o0) * vpr;

  const char* src = (kv ? st.v[layer] : st.k[layer]) + ((r0 + p0 + o0 - lo) * a.src_stride + int64_t(head) * g.head_dim) * 2;
  char* dst = qt.kv[layer] + page * g.page_stride + kv * g.v_offset + int64_t(head) * g.head_stride;
  float* scale = qt.scales[layer] + page * g.scale_page + kv * g.scale_kv + head * g.scale_head;
  const float before = live ? *scale : 0.f;

  float top = 0.f;
  for (int i = t; i < nvec; i += UNIT) {
    const int row = i / vpr, v = i - row * vpr;
    float f[8];
    to_floats<BF16>(*reinterpret_cast<const w4*>(src + (row * a.src_stride + v * 8) * 2), f);
#pragma unroll
    for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(f[j]) < INFINITY ? fabsf(f[j]) : 0.f);
  }
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor(top, s));
  if (UNIT > 64) {
    if ((threadIdx.x & 63) == 0) top_lds[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < UNIT / 64; ++w) top = fmaxf(top, top_lds[w]);
  }
  float now = exp2_int(scale_exponent<CACHE>(top));
  if (o0 > 0 && before > now) now = before;
  const float up = 1.0f / now;
  // older rows, when the scale grew
  if (live && o0 > 0 && now != before) {
    const float ratio = before * up;
    for (int i = t; i < o0 * vpr; i += UNIT) {
      const int row = i / vpr, v = i - row * vpr;
      w2* at = reinterpret_cast<w2*>(dst + row * g.token_stride + v * 8);
      w2 w = *at;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float f[4];
        Q::decode4(w[j], f);
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] *= ratio;
        w[j] = Q::encode4(f);
      }
      *at = w;
    }
  }
  for (int i = t; i < nvec; i += UNIT) {
    const int row = i / vpr, v = i - row * vpr;
    float f[8];
    to_floats<BF16>(*reinterpret_cast<const w4*>(src + (row * a.src_stride + v * 8) * 2), f);
    w2 w;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = f[4 * j + e] * up;
      w[j] = Q::encode4(x);
    }
    *reinterpret_cast<w2*>(dst + (o0 + row) * g.token_stride + v * 8) = w;
  }
  if (live && t == 0) *scale = now;
}

struct Commits {
  const int64_t* src_pos;
  const int64_t* dst_pos;
  const int32_t* indptr;
  const int32_t* kv_indptr;
  const int32_t* kv_indices;
  int64_t num_items;
  int batch, max_items, layers;
};

// One wave per (layer, request, K or V, head): all of a request's rows of a head are
// read into LDS before any is written, so sources and destinations may overlap.
// Lane i prepares item i: its rows' offsets, its destination block's scales, and
// whether it is the first item of that block.
template <int CACHE>
__global__ __launch_bounds__(64) void kv_commit_quantized_kernel(QuantTables qt, QuantGeom g, Commits c) {
  typedef Quant8<CACHE> Q;
  constexpr int kMax = ATLAS_QUANT_COMMIT_MAX_ITEMS;
  __shared__ __attribute__((aligned(16))) uint32_t rows[kMax * 32];
  __shared__ int64_t page_of[kMax], src_off[kMax], dst_off[kMax];
  __shared__ float old_scale[kMax], src_scale[kMax], new_scale[kMax];
  __shared__ int state[kMax];  // 0: skipped, 1: moved, 2: moved and first of its block
  int u = blockIdx.x;
  const int head = u % g.heads;
  u /= g.heads;
  const int kv = u & 1;
  u >>= 1;
  const int b = u % c.batch;
  const int layer = u / c.batch;
  const int lane = threadIdx.x;

  const int64_t i0 = min(max(int64_t(c.indptr[b]), int64_t(0)), c.num_items);
  const int64_t i1 = min(max(int64_t(c.indptr[b + 1]), i0), c.num_items);
  const int n = int(min(i1 - i0, int64_t(c.max_items)));
  if (n == 0) return;
  const int64_t pt = min(max(int64_t(c.kv_indptr[b]), int64_t(0)), g.num_indices);
  const int64_t np = min(max(int64_t(c.kv_indptr[b + 1]), pt), g.num_indices) - pt;

  char* base = qt.kv[layer] + kv * g.v_offset + int64_t(head) * g.head_stride;
  float* sbase = qt.scales[layer] + kv * g.scale_kv + head * g.scale_head;
  auto place = [&](int64_t pos, int64_t& page, int64_t& off) {
    const int64_t lp = g.page_shift >= 0 ? pos >> g.page_shift : pos / g.page_size;
    if (pos < 0 || lp >= np) return false;
    page = c.kv_indices[pt + lp];
    off = page * g.page_stride + (pos - lp * g.page_size) * g.token_stride;
    return page >= 0 && page < g.num_pages;
  };
  if (lane < n) {
    int64_t sp = 0, dp = 0, so = 0, dof = 0;
    const bool ok = place(c.src_pos[i0 + lane], sp, so) && place(c.dst_pos[i0 + lane], dp, dof);
    page_of[lane] = ok ? dp : -1;
    src_off[lane] = so;
    dst_off[lane] = dof;
    src_scale[lane] = ok ? sbase[sp * g.scale_page] : 0.f;
    old_scale[lane] = ok ? sbase[dp * g.scale_page] : 0.f;
    state[lane] = ok;
  }
  __syncthreads();
  if (lane < n && state[lane]) {
    float now = old_scale[lane];
    bool leads = true;
    for (int j = 0; j < n; ++j) {
      if (page_of[j] != page_of[lane]) continue;
      now = fmaxf(now, src_scale[j]);
      if (j < lane) leads = false;
    }
    new_scale[lane] = now;
    if (leads) state[lane] = 2;
  }
  __syncthreads();
  const int wpr = g.head_dim / 4;  // words per row
  for (int i = lane; i < n * wpr; i += 64) {
    const int item = i / wpr, w = i - item * wpr;
    if (state[item]) rows[i] = *reinterpret_cast<const uint32_t*>(base + src_off[item] + w * 4);
  }
  __syncthreads();
  for (int j = 0; j < n; ++j) {
    if (state[j] != 2 || new_scale[j] == old_scale[j]) continue;
    const float ratio = old_scale[j] / new_scale[j];
    char* page = base + page_of[j] * g.page_stride;
    for (int i = lane; i < g.page_size * wpr; i += 64) {
      const int row = i / wpr, w = i - row * wpr;
      uint32_t* at = reinterpret_cast<uint32_t*>(page + row * g.token_stride + w * 4);
      float f[4];
      Q::decode4(*at, f);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] *= ratio;
      *at = Q::encode4(f);
    }
    if (lane == 0) sbase[page_of[j] * g.scale_page] = new_scale[j];
  }
  __syncthreads();  // (the rounded rows are in memory before rows are moved over them)
  for (int i = lane; i < n * wpr; i += 64) {
    const int item = i / wpr, w = i - item * wpr;
    if (!state[item]) continue;
    const float ratio = src_scale[item] / new_scale[item];
    float f[4];
    Q::decode4(rows[i], f);
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] *= ratio;
    *reinterpret_cast<uint32_t*>(base + dst_off[item] + w * 4) = Q::encode4(f);
  }
}

int make_quant_geom(const void* const* layers, const void* const* scales, int num_layers, int cache, int64_t page_size,
                    int64_t page_stride, int64_t v_offset, int64_t token_stride, int64_t head_stride,
                    int64_t scale_page, int64_t scale_kv, int64_t scale_head, int heads, int head_dim,
                    int64_t num_pages, int64_t num_indices, QuantGeom& g) {
  ATLAS_REQUIRE(num_layers > 0 && layers != nullptr && scales != nullptr, "layer and scale tables must not be NULL");
  for (int i = 0; i < num_layers; ++i)
    ATLAS_REQUIRE(layers[i] != nullptr && scales[i] != nullptr &&
                      (reinterpret_cast<uintptr_t>(layers[i]) & 15) == 0,
                  "layer %d: the cache must be 16-byte aligned and its scales not NULL", i);
  ATLAS_REQUIRE(cache == ATLAS_CACHE_E4M3 || cache == ATLAS_CACHE_INT8, "cache type %d has no codes", cache);
  ATLAS_REQUIRE(page_size > 0 && page_size < (1 << 30) && num_pages > 0 && num_indices >= 0,
                "page_size and num_pages must be positive");
  ATLAS_REQUIRE(heads > 0, "num_kv_heads must be positive");
  if (head_dim != 64 && head_dim != 128) {
    set_error("head_dim %d is not supported (64 or 128)", head_dim);
    return ATLAS_EUNSUPPORTED;
  }
  ATLAS_REQUIRE(page_stride % 16 == 0 && v_offset % 16 == 0 && token_stride % 16 == 0 && head_stride % 16 == 0,
                "cache strides must be multiples of 16 bytes");
  g = QuantGeom{page_stride, v_offset, token_stride, head_stride, scale_page, scale_kv, scale_head, num_pages,
                num_indices, int(page_size), ilog2_exact(page_size), heads, head_dim};
  return ATLAS_OK;
}

void fill_quant_tables(QuantTables& qt, const void* const* layers, const void* const* scales, int l0, int nl) {
  for (int i = 0; i < ATLAS_MAX_LAYERS_PER_LAUNCH; ++i) {
    qt.kv[i] = i < nl ? const_cast<char*>(static_cast<const char*>(layers[l0 + i])) : nullptr;
    qt.scales[i] = i < nl ? const_cast<float*>(static_cast<const float*>(scales[l0 + i])) : nullptr;
  }
}

template <int CACHE, bool BF16>
void launch_append(int64_t units, int unit, hipStream_t stream, const QuantTables& qt, const RowTables& st,
                   const QuantGeom& g, const Appends& a) {
  const int per_block = kAppendThreads / unit;
  const dim3 grid(static_cast<unsigned>((units + per_block - 1) / per_block));
  if (unit == 64)
    hipLaunchKernelGGL((kv_append_quantized_kernel<CACHE, BF16, 64>), grid, dim3(kAppendThreads), 0, stream, qt, st, g, a);
  else
    hipLaunchKernelGGL((kv_append_quantized_kernel<CACHE, BF16, 256>), grid, dim3(kAppendThreads), 0, stream, qt, st, g, a);
}

}  // namespace
}  // namespace atlas

using namespace atlas;

extern "C" int atlas_kv_append_quantized(
    const void* const* layers, const void* const* scales, int num_layers, int cache, int64_t page_size,
    int64_t page_stride, int64_t v_offset, int64_t token_stride, int64_t head_stride, int64_t scale_stride_page,
    int64_t scale_stride_kv, int64_t scale_stride_head, const void* const* k_src, const void* const* v_src,
    int64_t src_token_stride, int dtype, int num_kv_heads, int head_dim, const int32_t* append_indptr_dev,
    const int32_t* kv_indptr_dev, const int32_t* kv_indices_dev, const int32_t* kv_last_page_len_dev, int batch,
    int64_t max_append, int64_t nnz, int64_t num_pages, int64_t num_indices, void* stream) {
  QuantGeom g;
  int rc = make_quant_geom(layers, scales, num_layers, cache, page_size, page_stride, v_offset, token_stride, head_stride,
                           scale_stride_page, scale_stride_kv, scale_stride_head, num_kv_heads, head_dim, num_pages,
                           num_indices, g);
  if (rc) return rc;
  ATLAS_REQUIRE(k_src != nullptr && v_src != nullptr, "source tables must not be NULL");
  for (int i = 0; i < num_layers; ++i)
    ATLAS_REQUIRE(k_src[i] != nullptr && v_src[i] != nullptr && (reinterpret_cast<uintptr_t>(k_src[i]) & 15) == 0 &&
                      (reinterpret_cast<uintptr_t>(v_src[i]) & 15) == 0,
                  "source %d is NULL or not 16-byte aligned", i);
  ATLAS_REQUIRE(dtype == ATLAS_DTYPE_F16 || dtype == ATLAS_DTYPE_BF16, "unknown source dtype %d", dtype);
  ATLAS_REQUIRE(src_token_stride % 8 == 0 && src_token_stride >= int64_t(num_kv_heads) * head_dim,
                "source token stride must be a multiple of 8 elements and cover a row");
  ATLAS_REQUIRE(append_indptr_dev && kv_indptr_dev && kv_last_page_len_dev && kv_indices_dev,
                "indptr / indices / last_page_len arrays must not be NULL");
  ATLAS_REQUIRE(batch > 0 && nnz >= 0 && max_append >= 0, "batch must be positive, nnz and max_append non-negative");
  if (nnz == 0 || max_append == 0) return ATLAS_OK;
  max_append = std::min(max_append, nnz);
  const int64_t pages = (max_append + page_size - 2) / page_size + 1;
  Appends a{append_indptr_dev, kv_indptr_dev, kv_indices_dev, kv_last_page_len_dev, nnz, src_token_stride,
            max_append, batch, int(pages), 0};
  for (int l0 = 0; l0 < num_layers; l0 += ATLAS_MAX_LAYERS_PER_LAUNCH) {
    const int nl = std::min(ATLAS_MAX_LAYERS_PER_LAUNCH, num_layers - l0);
    QuantTables qt;
    fill_quant_tables(qt, layers, scales, l0, nl);
    RowTables st;
    for (int i = 0; i < ATLAS_MAX_LAYERS_PER_LAUNCH; ++i) {
      st.k[i] = i < nl ? static_cast<const char*>(k_src[l0 + i]) : nullptr;
      st.v[i] = i < nl ? static_cast<const char*>(v_src[l0 + i]) : nullptr;
    }
    a.layers = nl;
    const int64_t units = int64_t(nl) * batch * pages * 2 * num_kv_heads;
    const int unit = std::min(page_size, max_append) * head_dim > 4096 ? 256 : 64;
    if (units >= (int64_t(1) << 24)) {
      set_error("%lld blocks are too many for one append", static_cast<long long>(units));
      return ATLAS_EUNSUPPORTED;
    }
    const hipStream_t hs = static_cast<hipStream_t>(stream);
    if (cache == ATLAS_CACHE_E4M3) {
      if (dtype == ATLAS_DTYPE_BF16) launch_append<ATLAS_CACHE_E4M3, true>(units, unit, hs, qt, st, g, a);
      else launch_append<ATLAS_CACHE_E4M3, false>(units, unit, hs, qt, st, g, a);
    } else {
      if (dtype == ATLAS_DTYPE_BF16) launch_append<ATLAS_CACHE_INT8, true>(units, unit, hs, qt, st, g, a);
      else launch_append<ATLAS_CACHE_INT8, false>(units, unit, hs, qt, st, g, a);
    }
    if ((rc = launch_status("kv_append_quantized_kernel"))) return rc;
  }
  return ATLAS_OK;
}

extern "C" int atlas_kv_commit_quantized(
    const void* const* layers, const void* const* scales, int num_layers, int cache, int64_t page_size,
    int64_t page_stride, int64_t v_offset, int64_t token_stride, int64_t head_stride, int64_t scale_stride_page,
    int64_t scale_stride_kv, int64_t scale_stride_head, int num_kv_heads, int head_dim, const int64_t* src_pos_dev,
    const int64_t* dst_pos_dev, const int32_t* item_indptr_dev, const int32_t* kv_indptr_dev,
    const int32_t* kv_indices_dev, int batch, int max_items, int64_t num_items, int64_t num_pages, int64_t num_indices,
    void* stream) {
  QuantGeom g;
  int rc = make_quant_geom(layers, scales, num_layers, cache, page_size, page_stride, v_offset, token_stride, head_stride,
                           scale_stride_page, scale_stride_kv, scale_stride_head, num_kv_heads, head_dim, num_pages,
                           num_indices, g);
  if (rc) return rc;
  ATLAS_REQUIRE(src_pos_dev && dst_pos_dev && item_indptr_dev && kv_indptr_dev && kv_indices_dev,
                "position and table arrays must not be NULL");
  ATLAS_REQUIRE(batch > 0 && num_items >= 0 && max_items >= 0, "batch must be positive, item counts non-negative");
  if (max_items > ATLAS_QUANT_COMMIT_MAX_ITEMS) {
    set_error("a request commits at most %d rows, got %d", ATLAS_QUANT_COMMIT_MAX_ITEMS, max_items);
    return ATLAS_EUNSUPPORTED;
  }
  if (num_items == 0 || max_items == 0) return ATLAS_OK;
  Commits c{src_pos_dev, dst_pos_dev, item_indptr_dev, kv_indptr_dev, kv_indices_dev, num_items, batch, max_items, 0};
  for (int l0 = 0; l0 < num_layers; l0 += ATLAS_MAX_LAYERS_PER_LAUNCH) {
    const int nl = std::min(ATLAS_MAX_LAYERS_PER_LAUNCH, num_layers - l0);
    QuantTables qt;
    fill_quant_tables(qt, layers, scales, l0, nl);
    c.layers = nl;
    const int64_t units = int64_t(nl) * batch * 2 * num_kv_heads;
    if (units >= (int64_t(1) << 26)) {
      set_error("%lld blocks are too many for one commit", static_cast<long long>(units));
      return ATLAS_EUNSUPPORTED;
    }
    const dim3 grid(static_cast<unsigned>(units));
    if (cache == ATLAS_CACHE_E4M3)
      hipLaunchKernelGGL((kv_commit_quantized_kernel<ATLAS_CACHE_E4M3>), grid, dim3(64), 0,
                         static_cast<hipStream_t>(stream), qt, g, c);
    else
      hipLaunchKernelGGL((kv_commit_quantized_kernel<ATLAS_CACHE_INT8>), grid, dim3(64), 0,
                         static_cast<hipStream_t>(stream), qt, g, c);
    if ((rc = launch_status("kv_commit_quantized_kernel"))) return rc;
  }
  return ATLAS_OK;
}

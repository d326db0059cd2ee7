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
typedef uint16_t u2 __attribute__((ext_vector_type(2)));

constexpr int kAppendThreads = 256;
constexpr int kHeld = 8;  // vectors of a thread's rows in registers
constexpr int kCommitWaves = 4;

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

// Largest magnitude so far, as bits, of the even and the odd values: those of finite
// 16-bit values are in their order.  (In fp32 the compiler keeps the values for the codes
// as well, and half as many waves fit.)
template <bool BF16>
__device__ __forceinline__ u2 largest(u2 most, w4 v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t bad = ((v[i] & (BF16 ? 0x7f807f80u : 0x7c007c00u)) + (BF16 ? 0x00800080u : 0x04000400u)) & 0x80008000u;
    const uint32_t x = v[i] & 0x7fff7fffu & ~((bad << 1) - (bad >> 15));
    most = __builtin_elementwise_max(most, __builtin_bit_cast(u2, x));
  }
  return most;
}

// Four codes under a scale that is 1 / ratio times theirs.
template <int CACHE>
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float ratio) {
  float f[4];
  Quant8<CACHE>::decode4(w, f);
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] *= ratio;
  return Quant8<CACHE>::encode4(f);
}

// One unit (a touched page's rows of one head, K or V, of one layer) per UNIT
// threads: the rows are read once, into registers (kHeld vectors of 8 values a
// thread; what a large page holds beyond that is read twice), their largest value
// gives the scale, and the codes follow.  Bound by the bytes: 2 read and 1 written
// per value: 128 us for 647 MB, 5.1 TB/s, for 8 prompts of 2048 tokens into 16 layers.  In
// replays of a graph 133; reading the rows a second time, for the codes, took 150 there, the
// largest value in fp32 146.  A decode step's rows are one chain of loads, about 5 us.
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
  const int vs = g.head_dim == 64 ? 3 : 4, vmask = (1 << vs) - 1;  // vectors of 8 values per row
  const int nvec = (o1 - o0) << vs;

  const char* src = (kv ? st.v[layer] : st.k[layer]) + ((r0 + p0 + o0 - lo) * a.src_stride + int64_t(head) * g.head_dim) * 2;
  char* dst = qt.kv[layer] + page * g.page_stride + kv * g.v_offset + int64_t(head) * g.head_stride;
  float* scale = qt.scales[layer] + page * g.scale_page + kv * g.scale_kv + head * g.scale_head;
  const float before = live ? *scale : 0.f;

  auto read = [&](int i) __attribute__((always_inline)) {
    return *reinterpret_cast<const w4*>(src + ((i >> vs) * a.src_stride + (i & vmask) * 8) * 2);
  };
  u2 most = u2{0, 0};
  w4 held[kHeld];
#pragma unroll
  for (int k = 0; k < kHeld; ++k) {
    held[k] = w4{0, 0, 0, 0};
    if (t + k * UNIT < nvec) held[k] = read(t + k * UNIT);
  }
#pragma unroll
  for (int k = 0; k < kHeld; ++k) most = largest<BF16>(most, held[k]);
  for (int i = t + kHeld * UNIT; i < nvec; i += UNIT) most = largest<BF16>(most, read(i));
  const uint32_t bits = max(most[0], most[1]);
  float top = BF16 ? __uint_as_float(bits << 16) : float(__builtin_bit_cast(_Float16, uint16_t(bits)));
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
    for (int i = t; i < o0 << vs; i += UNIT) {
      w2* at = reinterpret_cast<w2*>(dst + (i >> vs) * g.token_stride + (i & vmask) * 8);
      w2 w = *at;
      w[0] = rescale4<CACHE>(w[0], ratio);
      w[1] = rescale4<CACHE>(w[1], ratio);
      *at = w;
    }
  }
  auto write = [&](int i, w4 v) __attribute__((always_inline)) {
    float f[8];
    to_floats<BF16>(v, f);
    w2 w;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = f[4 * j + e] * up;
      w[j] = Q::encode4(x);
    }
    *reinterpret_cast<w2*>(dst + (o0 + (i >> vs)) * g.token_stride + (i & vmask) * 8) = w;
  };
#pragma unroll
  for (int k = 0; k < kHeld; ++k)
    if (t + k * UNIT < nvec) write(t + k * UNIT, held[k]);
  for (int i = t + kHeld * UNIT; i < nvec; i += UNIT) write(i, read(i));
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

__device__ __forceinline__ int64_t shuffle64(int64_t v, int lane) {
  const uint32_t low = __shfl(uint32_t(v), lane), high = __shfl(uint32_t(v >> 32), lane);
  return int64_t(uint64_t(high) << 32 | low);
}

// One wave per (layer, request, K or V, head).  All of a request's rows of a head are
// read into registers before any is written, so sources and destinations may overlap.
// Lane i holds item i: its rows' offsets, its blocks' scales, whether it is the first
// item of its destination block; what the others need of it goes through readlane and
// shuffles.  A few hundred bytes per wave: bound by the chain of loads from the
// positions to the rows, so every wave of a call should be in flight at once: 4.4 us for one
// request, 17 us for 32 requests and 32 layers (16384 waves).  With the rows and tables in LDS, one
// wave a workgroup, those took 7.5 and 29 us.
template <int CACHE, int D>
__global__ __launch_bounds__(64 * kCommitWaves) void kv_commit_quantized_kernel(QuantTables qt, QuantGeom g, Commits c) {
  constexpr int kLanes = D / 16;        // lanes of 16 codes per row
  constexpr int kRows = 64 / kLanes;    // rows per pass
  constexpr int kPasses = ATLAS_QUANT_COMMIT_MAX_ITEMS / kRows;
  const int units = 2 * g.heads, groups = (units + kCommitWaves - 1) / kCommitWaves;
  int u = blockIdx.x;
  const int unit = (u % groups) * kCommitWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  u /= groups;
  const int b = u % c.batch;
  const int layer = u / c.batch;
  const int kv = unit >= g.heads, head = unit - kv * g.heads;
  const int lane = threadIdx.x & 63;

  const int64_t i0 = min(max(int64_t(c.indptr[b]), int64_t(0)), c.num_items);
  const int64_t i1 = min(max(int64_t(c.indptr[b + 1]), i0), c.num_items);
  // (a wave past the last unit moves nothing, but meets the others at the barriers)
  const int n = unit < units ? int(min(i1 - i0, int64_t(c.max_items))) : 0;
  const int64_t pt = min(max(int64_t(c.kv_indptr[b]), int64_t(0)), g.num_indices);
  const int64_t np = min(max(int64_t(c.kv_indptr[b + 1]), pt), g.num_indices) - pt;

  char* base = qt.kv[layer] + kv * g.v_offset + int64_t(head) * g.head_stride;
  float* sbase = qt.scales[layer] + kv * g.scale_kv + head * g.scale_head;
  auto place = [&](int64_t pos, int& page, int64_t& off) __attribute__((always_inline)) {
    const int64_t lp = g.page_shift >= 0 ? pos >> g.page_shift : pos / g.page_size;
    if (pos < 0 || lp >= np) return false;
    page = c.kv_indices[pt + lp];
    off = page * g.page_stride + (pos - lp * g.page_size) * g.token_stride;
    return page >= 0 && page < g.num_pages;
  };
  int src_page = -1, page = -1;
  int64_t src = 0, dst = 0;
  float src_scale = 0.f, before = 0.f;
  bool moves = false;
  if (lane < n) {
    const int64_t from = c.src_pos[i0 + lane], to = c.dst_pos[i0 + lane];
    const bool from_ok = place(from, src_page, src), to_ok = place(to, page, dst);
    moves = from_ok && to_ok;
    if (moves) {
      src_scale = sbase[src_page * g.scale_page];
      before = sbase[page * g.scale_page];
    }
  }
  if (!moves) page = -1;

  w4 rows[kPasses];
  const int word = (lane % kLanes) * 16;
#pragma unroll
  for (int k = 0; k < kPasses; ++k) {
    if (k * kRows >= n) break;  // (the same for the wave: every lane takes part in the shuffles)
    const int item = k * kRows + lane / kLanes;
    const int64_t off = shuffle64(src, item);
    if (__shfl(page, item) >= 0) rows[k] = *reinterpret_cast<const w4*>(base + off + word);
  }
  // the block's new scale, its first item, and items whose row a later one writes again
  float now = before;
  bool leads = moves, stays = false;
  for (int j = 0; j < n; ++j) {
    const int pj = __builtin_amdgcn_readlane(page, j);
    const float sj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(src_scale), j));
    if (pj < 0 || pj != page) continue;
    now = fmaxf(now, sj);
    if (j < lane) leads = false;
    const int64_t dj = int64_t(uint64_t(uint32_t(__builtin_amdgcn_readlane(int(dst >> 32), j))) << 32 |
                               uint32_t(__builtin_amdgcn_readlane(int(dst), j)));
    if (j > lane && dj == dst) stays = true;
  }
  __syncthreads();  // (every row has been read)
  for (uint64_t grown = __ballot(leads && now != before); grown; grown &= grown - 1) {
    const int j = __builtin_ctzll(grown);
    const float ratio = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(before), j)) /
                        __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(now), j));
    char* at = base + int64_t(__builtin_amdgcn_readlane(page, j)) * g.page_stride + word;
    for (int row = lane / kLanes; row < g.page_size; row += kRows) {
      w4* p = reinterpret_cast<w4*>(at + row * g.token_stride);
      w4 w = *p;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = rescale4<CACHE>(w[e], ratio);
      *p = w;
    }
  }
  if (leads && now != before) sbase[page * g.scale_page] = now;
  __syncthreads();  // (the rounded rows are in memory before rows are moved over them)
  const float ratio = src_scale / now;
#pragma unroll
  for (int k = 0; k < kPasses; ++k) {
    if (k * kRows >= n) break;
    const int item = k * kRows + lane / kLanes;
    const int64_t off = shuffle64(dst, item);
    const float r = __shfl(ratio, item);
    if (!__shfl(int(moves && !stays), item)) continue;
    w4 w = rows[k];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = rescale4<CACHE>(w[e], r);
    *reinterpret_cast<w4*>(base + off + word) = w;
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

template <int CACHE, int D>
void launch_commit(int64_t blocks, hipStream_t stream, const QuantTables& qt, const QuantGeom& g, const Commits& c) {
  hipLaunchKernelGGL((kv_commit_quantized_kernel<CACHE, D>), dim3(static_cast<unsigned>(blocks)), dim3(64 * kCommitWaves),
                     0, stream, qt, g, c);
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
    const int64_t units = int64_t(nl) * batch * ((2 * int64_t(num_kv_heads) + kCommitWaves - 1) / kCommitWaves);
    if (units >= (int64_t(1) << 24)) {
      set_error("%lld blocks are too many for one commit", static_cast<long long>(units));
      return ATLAS_EUNSUPPORTED;
    }
    const hipStream_t hs = static_cast<hipStream_t>(stream);
    if (cache == ATLAS_CACHE_E4M3) {
      if (head_dim == 128) launch_commit<ATLAS_CACHE_E4M3, 128>(units, hs, qt, g, c);
      else launch_commit<ATLAS_CACHE_E4M3, 64>(units, hs, qt, g, c);
    } else {
      if (head_dim == 128) launch_commit<ATLAS_CACHE_INT8, 128>(units, hs, qt, g, c);
      else launch_commit<ATLAS_CACHE_INT8, 64>(units, hs, qt, g, c);
    }
    if ((rc = launch_status("kv_commit_quantized_kernel"))) return rc;
  }
  return ATLAS_OK;
}

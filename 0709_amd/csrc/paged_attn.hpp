// Paged attention from device-side metadata, over 16-bit caches and over 8-bit
// caches with one scale for each page, K or V, and KV head; scores may be
// capped, biased by distance, windowed or masked by a draft tree's words.
// This file: what the two kernels share, and the join of key splits.
//
//   paged_stream.hpp  few packed rows: one query token per request, or short blocks;
//   paged_rows.hpp    many rows.
//
// Rows are packed: row = query token * group + head of the group, for one KV head.
//
//   S^T[key, row] = K[key, :] . Q[row, :]     A = K, B = Q
//   O^T[dim, row] += V^T[dim, key] P^T[key, row]
//
// The C layout of a 16x16 product gives lane l = 16 g + c the column (row of Q) c
// and rows (keys, dims) 4g .. 4g + 3, so a lane's scores belong to one query row and
// P^T is the second product's operand as it stands, when V^T brings its keys in the
// order 4g .. 4g + 3 of one 16-key tile, then of the next.
//
// 8-bit codes are exact in fp16, so both products run in fp16 there: Q is scaled by a
// power of two per row (largest element in [2^14, 2^15); what falls below fp16's
// normal range is 2^-29 of it, an absolute error below fp32's own), K's scale goes
// into the score's factor, and V's scale into P relative to the largest V scale met
// so far, which keeps P within fp16.
//
// Scores, running maxima and sums, and O are fp32.  P is rounded to 16 bits, to
// nearest, for the matrix product; the sum of the softmax adds the values before
// that rounding, so the LSE does not see it.
#pragma once

#include "common.hpp"

namespace atlas {

struct PagedAttnArgs {
  atlas_paged_attn_t p;
  float scale_log2;  // sm_scale * log2(e)
  float cap_in;      // soft cap: 2 * log2(e) * sm_scale / cap
  float cap_out;     // cap * log2(e)
  int group;
  // key / page_size = key * page_magic >> page_bits for keys below 2^31
  uint32_t page_magic;
  int page_bits;
};

int launch_paged_attn_16bit(const PagedAttnArgs& a, hipStream_t stream);
int launch_paged_attn_q8(const PagedAttnArgs& a, hipStream_t stream);

namespace {

constexpr int kPaWaves = 4;
constexpr int kPaThreads = kPaWaves * 64;
constexpr float kPaLog2e = 1.4426950408889634f;
constexpr float kPaLn2 = 0.6931471805599453f;
// The running maximum is raised only when a score exceeds it by this much (in
// powers of two): P then stays below 2^8.
constexpr float kPaLazyLog2 = 8.0f;

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef uint32_t w4 __attribute__((ext_vector_type(4)));
typedef uint32_t w2 __attribute__((ext_vector_type(2)));

// A request's lengths, clamped so that no metadata leads outside the arrays.
struct Request {
  int q0, q_len, pt, kv_len;
};

__device__ __forceinline__ Request read_request(const atlas_paged_attn_t& p, int b) {
  Request r;
  const int nnz = int(p.nnz), ni = int(p.num_indices);
  r.q0 = min(max(p.qo_indptr[b], 0), nnz);
  r.q_len = min(max(p.qo_indptr[b + 1], r.q0), nnz) - r.q0;
  r.pt = min(max(p.kv_indptr[b], 0), ni);
  const int pages = min(max(p.kv_indptr[b + 1], r.pt), ni) - r.pt;
  const int last = min(max(p.kv_last_page_len[b], 0), p.page_size);
  r.kv_len = pages > 0 ? (pages - 1) * p.page_size + last : 0;
  return r;
}

// Rows of a block that starts at packed row row_start (none: not positive).
__device__ __forceinline__ int block_of(const PagedAttnArgs& a, const Request& r, int row_start) {
  const int tokens = a.p.single_token ? min(r.q_len, 1) : r.q_len;
  return min(a.p.block_rows, tokens * a.group - row_start);
}

// What a row block has to stream: the key chunks that some row of it may see, as
// chunks of 64 keys 0 .. ca - 1 (the visible prefix) and cb .. ce - 1, and its splits.
constexpr int kChunk = 64;
struct Block {
  int n0, n1;      // first and last query token
  int prefix;      // keys below it are visible to every row (causal)
  int lo, hi;      // keys of the second part
  int ca, cb;      // chunks of the first part; first chunk of the second
  int chunks;      // chunks in all
  int per, splits; // chunks of a split, splits
};

__device__ __forceinline__ Block plan_block(const PagedAttnArgs& a, const Request& r, int b, int row_start, int rows) {
  const atlas_paged_attn_t& p = a.p;
  Block k;
  k.n0 = row_start / a.group;
  k.n1 = (row_start + rows - 1) / a.group;
  k.prefix = 0;
  k.lo = 0;
  k.hi = r.kv_len;
  if (p.mask_mode == 2) {
    const int shift = r.kv_len - r.q_len;
    if (p.prefix_lens) k.prefix = min(max(p.prefix_lens[b], 0), r.kv_len);
    k.hi = max(min(r.kv_len, shift + k.n1 + 1), 0);
    if (p.window_left >= 0) k.lo = max(0, shift + k.n0 - p.window_left);
    if (k.hi <= k.prefix) {
      k.hi = k.prefix;
      k.lo = 0;
    }
    k.lo = min(k.lo, k.hi);
  }
  k.ca = (k.prefix + kChunk - 1) / kChunk;
  k.cb = k.lo / kChunk;
  if (k.ca >= k.cb) {
    k.ca = k.cb = 0;
    k.lo = 0;
  }
  k.chunks = k.ca + (k.hi + kChunk - 1) / kChunk - k.cb;
  k.per = max(p.split_keys / kChunk, (k.chunks + p.num_splits - 1) / p.num_splits);
  k.splits = max(1, (k.chunks + k.per - 1) / k.per);
  k.per = (k.chunks + k.splits - 1) / k.splits;  // (as equal as they come)
  return k;
}

__device__ __forceinline__ float pa_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float groups_max(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = pa_max(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return pa_max(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float groups_sum(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Bits of the four keys key0 .. key0 + 3 below `end`.
__device__ __forceinline__ uint32_t below4(int key0, int end) {
  return (1u << min(max(end - key0, 0), 4)) - 1u;
}
// Those that a word of tree columns shows, the first of them `off` columns behind the
// word's start (columns before it are the prefix, those past its end are hidden).
__device__ __forceinline__ uint32_t tree4(uint64_t w, int off) {
  const int pre = min(max(-off, 0), 4);
  const uint32_t up = off >= 0 && off < 64 ? uint32_t(w >> (off & 63)) : 0u;
  const uint32_t down = uint32_t(w << pre) | ((1u << pre) - 1u);
  return off >= 0 ? up : down;
}

// Two 16-bit values at a time: the exponent's carry (bits 15 and 31) marks what is
// not finite, the mantissa's carry NaN.
template <bool BF16>
__device__ __forceinline__ uint32_t not_finite2(uint32_t x) {
  return ((x & (BF16 ? 0x7f807f80u : 0x7c007c00u)) + (BF16 ? 0x00800080u : 0x04000400u)) & 0x80008000u;
}
// The values with zeros for what is not finite; u marks +inf and NaN, d -inf and NaN.
template <bool BF16>
__device__ __forceinline__ uint32_t take_out2(uint32_t x, uint32_t& u, uint32_t& d) {
  const uint32_t bad = not_finite2<BF16>(x), nan = (x & (BF16 ? 0x007f007fu : 0x03ff03ffu)) + 0x7fff7fffu;
  u = bad & (nan | ~x);
  d = bad & (nan | x);
  return x & ~((bad << 1) - (bad >> 15));
}

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  return __builtin_bit_cast(uint32_t, h2{static_cast<_Float16>(a), static_cast<_Float16>(b)});
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  return __builtin_bit_cast(uint32_t, b2{static_cast<__bf16>(a), static_cast<__bf16>(b)});
}

// Kinds of cache: kCacheF16 / kCacheBf16 hold q's type, the others codes.
enum CacheKind { kCacheF16, kCacheBf16, kCacheE4M3, kCacheInt8 };

template <int KIND>
struct Cache {
  static constexpr bool kQuant = KIND == kCacheE4M3 || KIND == kCacheInt8;
  static constexpr int kBytes = kQuant ? 1 : 2;
  static constexpr bool kBf16 = KIND == kCacheBf16;  // type of the products
  typedef uint32_t frag __attribute__((ext_vector_type(4)));

  static __device__ __forceinline__ f32x4 mfma(frag a, frag b, f32x4 c) {
    if constexpr (kBf16)
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c,
                                                     0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0,
                                                    0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return kBf16 ? pack_bf16(a, b) : pack_f16(a, b); }

  // Two int8 codes (bytes sel of hi:lo, biased by 128) as fp16: the byte under
  // fp16's 1024 is 1024 + code + 128.
  static __device__ __forceinline__ uint32_t int8_pair(uint32_t hi, uint32_t lo, uint32_t sel) {
    const uint32_t u = __builtin_amdgcn_perm(hi, lo, sel) | 0x64006400u;
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, u) - h2{(_Float16)1152.f, (_Float16)1152.f});
  }

  // Eight codes of one key (two words) as an operand.
  static __device__ __forceinline__ frag keys8(uint32_t x, uint32_t y) {
    if constexpr (KIND == kCacheE4M3) {
      return frag{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, false)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, true)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(y, 1.0f, false)),
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(y, 1.0f, true))};
    } else {
      x ^= 0x80808080u;
      y ^= 0x80808080u;
      return frag{int8_pair(0, x, 0x0c010c00u), int8_pair(0, x, 0x0c030c02u), int8_pair(0, y, 0x0c010c00u),
                  int8_pair(0, y, 0x0c030c02u)};
    }
  }
};

// The NW words that a lane loads of its dims of one V row, for eight keys, as
// operands of the lane's dims.
template <int KIND, int NW, int NDIM>
__device__ __forceinline__ void transpose_v(const uint32_t (&v)[8][NW], typename Cache<KIND>::frag (&out)[NDIM]) {
  constexpr uint32_t kLoLo = 0x05040100u, kHiHi = 0x07060302u;
  if constexpr (!Cache<KIND>::kQuant) {
    static_assert(NDIM == 2 * NW, "two dims a word");
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        out[2 * w][j] = __builtin_amdgcn_perm(v[2 * j + 1][w], v[2 * j][w], kLoLo);
        out[2 * w + 1][j] = __builtin_amdgcn_perm(v[2 * j + 1][w], v[2 * j][w], kHiHi);
      }
  } else if constexpr (KIND == kCacheE4M3) {
    static_assert(NDIM == 4 * NW, "four dims a word");
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t a0 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[2 * j][w], 1.0f, false));
        const uint32_t a1 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[2 * j][w], 1.0f, true));
        const uint32_t b0 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[2 * j + 1][w], 1.0f, false));
        const uint32_t b1 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v[2 * j + 1][w], 1.0f, true));
        out[4 * w][j] = __builtin_amdgcn_perm(b0, a0, kLoLo);
        out[4 * w + 1][j] = __builtin_amdgcn_perm(b0, a0, kHiHi);
        out[4 * w + 2][j] = __builtin_amdgcn_perm(b1, a1, kLoLo);
        out[4 * w + 3][j] = __builtin_amdgcn_perm(b1, a1, kHiHi);
      }
  } else {
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t a = v[2 * j][w] ^ 0x80808080u, b = v[2 * j + 1][w] ^ 0x80808080u;
        out[4 * w][j] = Cache<KIND>::int8_pair(b, a, 0x0c040c00u);
        out[4 * w + 1][j] = Cache<KIND>::int8_pair(b, a, 0x0c050c01u);
        out[4 * w + 2][j] = Cache<KIND>::int8_pair(b, a, 0x0c060c02u);
        out[4 * w + 3][j] = Cache<KIND>::int8_pair(b, a, 0x0c070c03u);
      }
  }
}

// Eight 16-bit values of q (fp16 or bf16) as floats.
__device__ __forceinline__ void q_floats(w4 v, bool bf16, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = bf16 ? __uint_as_float(v[i] << 16) : float(__builtin_bit_cast(h2, uint32_t(v[i]))[0]);
    f[2 * i + 1] = bf16 ? __uint_as_float(v[i] & 0xffff0000u) : float(__builtin_bit_cast(h2, uint32_t(v[i]))[1]);
  }
}

// A row of Q as fp16 operands for an 8-bit cache: scaled by 2^-e so that its largest
// element lies in [2^14, 2^15); returns 2^e.  A row of zeros, or one below 2^-111, takes
// the largest power; a row with infinities gets no meaningful one.
template <int KS>
__device__ __forceinline__ float q_to_f16(const float (&f)[KS][8], w4 (&q)[KS]) {
  float top = 0.f;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(f[ks][i]));
  top = groups_max(top);
  const int e = min(max(int(__float_as_uint(top) >> 23) - 127 - 14, -126), 126);
  const float down = __uint_as_float(uint32_t(127 - e) << 23);
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
#pragma unroll
    for (int i = 0; i < 4; ++i) q[ks][i] = pack_f16(f[ks][2 * i] * down, f[ks][2 * i + 1] * down);
  return __uint_as_float(uint32_t(127 + e) << 23);
}

__device__ __forceinline__ int slot_of(const PagedAttnArgs& a, int key) {
  return int((uint64_t(uint32_t(key)) * a.page_magic) >> a.page_bits);
}

// A request's page ids.  For page sizes that are multiples of 16 the kernels read
// what a run of 16-key tiles needs by lane, once for many steps, and take a tile's by
// readlane: no memory access of the key loop waits for another.
struct Pages {
  const int32_t* ids;
  int64_t page_stride;
  int64_t last_id;  // ids are clamped to [0, last_id]
  int page_size, ts;

  __device__ __forceinline__ void begin(const PagedAttnArgs& a, const Request& r) {
    ids = a.p.kv_indices + r.pt;
    page_stride = a.p.page_stride;
    last_id = a.p.num_pages - 1;
    page_size = a.p.page_size;
    ts = int(a.p.token_stride);
  }
  // First key of tile kt of the step at kb, on a tile that holds a key of [lo, hi]
  static __device__ __forceinline__ int tile_key(int kb, int kt, int lo, int hi) {
    return min(max(kb + kt * 16, lo & ~15), hi & ~15);
  }
  __device__ __forceinline__ int64_t valid(int id) const {
    const int64_t x = id;
    return x < 0 ? 0 : (x > last_id ? last_id : x);
  }
  // Of the lane's tile (first key `tile`):
  __device__ __forceinline__ int read_id(const PagedAttnArgs& a, int tile) const { return ids[slot_of(a, tile)]; }
  __device__ __forceinline__ int64_t row_offset(const PagedAttnArgs& a, int id, int tile) const {
    return valid(id) * page_stride + int64_t((tile - slot_of(a, tile) * page_size) * ts);
  }
  static __device__ __forceinline__ int64_t tile_row(int64_t v, int kt) {
    const uint32_t lo = __builtin_amdgcn_readlane(uint32_t(v), kt);
    const uint32_t hi = __builtin_amdgcn_readlane(uint32_t(uint64_t(v) >> 32), kt);
    return int64_t((uint64_t(hi) << 32) | lo);
  }
};

// Joins the splits of a row block: 16 lanes per row, each over D / 16 dims, four rows a
// wave.  Bound by the chain from the metadata to the partial states, which is walked once a
// wave: 9.3 us over two chunks of 512 tokens and 32 heads in two splits (24.6 us with one row a
// wave), 4 to 6 us over one token's rows.
template <int D>
__global__ __launch_bounds__(256) void paged_attn_merge_kernel(PagedAttnArgs a) {
  constexpr int DL = D / 16;
  const atlas_paged_attn_t& p = a.p;
  const int item = blockIdx.x;
  const int rb = item % p.row_blocks;
  const int h = item / p.row_blocks % p.num_kv_heads;
  const int b = item / p.row_blocks / p.num_kv_heads;
  const Request r = read_request(p, b);
  const int block_rows = p.block_rows, row_start = rb * block_rows;
  const int rows = block_of(a, r, row_start);
  const int lr = blockIdx.y * 16 + (threadIdx.x >> 4), lane = threadIdx.x & 15;
  if (lr >= rows) return;  // (whole rows: a row's lanes stay together)
  const Block k = plan_block(a, r, b, row_start, rows);
  if (k.splits <= 1) return;
  const float* ws = static_cast<const float*>(p.workspace);
  const int64_t nrows = int64_t(p.batch) * p.num_kv_heads * p.row_blocks * p.num_splits * block_rows;
  const int64_t row0 = int64_t(item) * p.num_splits * block_rows + lr;
  const float* lse_of = ws + nrows * D + row0;
  const float* o_of = ws + row0 * D + lane * DL;
  float m = -INFINITY;
  for (int s = lane; s < k.splits; s += 16) m = fmaxf(m, lse_of[int64_t(s) * block_rows]);
#pragma unroll
  for (int x = 8; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
  float sum = 0.f;
  f32x4 acc[DL / 4];
#pragma unroll
  for (int t = 0; t < DL / 4; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < k.splits; ++s) {
    const float lse2 = lse_of[int64_t(s) * block_rows];
    const float f = lse2 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(lse2 - m);
    sum += f;
#pragma unroll
    for (int t = 0; t < DL / 4; ++t)
      acc[t] += f * *reinterpret_cast<const f32x4*>(o_of + int64_t(s) * block_rows * D + 4 * t);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int prow = row_start + lr, node = prow / a.group;
  const int head = h * a.group + (prow - node * a.group);
  uint16_t* out = static_cast<uint16_t*>(p.out) + int64_t(r.q0 + node) * p.out_stride_token +
                  int64_t(head) * p.out_stride_head + lane * DL;
  const bool bf16 = p.dtype == ATLAS_DTYPE_BF16;
#pragma unroll
  for (int t = 0; t < DL / 4; ++t) {
    const f32x4 x = acc[t] * inv;
    *reinterpret_cast<w2*>(out + 4 * t) =
        bf16 ? w2{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])} : w2{pack_f16(x[0], x[1]), pack_f16(x[2], x[3])};
  }
  if (p.lse != nullptr && lane == 0)
    p.lse[int64_t(r.q0 + node) * p.num_qo_heads + head] = sum == 0.f ? -INFINITY : (m + __builtin_log2f(sum)) * kPaLn2;
}

}  // namespace
}  // namespace atlas

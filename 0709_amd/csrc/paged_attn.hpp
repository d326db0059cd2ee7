// Paged attention from device-side metadata, over 16-bit caches and over 8-bit
// caches with one scale for each page, K or V, and KV head; scores may be
// capped, biased by distance, windowed or masked by a draft tree's words.
//
// A workgroup takes a block of packed query rows (row = token * group + head of
// the group) of one KV head and one split of the request's keys; its four waves
// take that split's key chunks in turn and join their states at the end.  A
// wave works alone: K and V go from HBM to registers and from there into the
// matrix instructions, with no LDS and no barrier in the key loop.
//
//   S^T[key, row] = K[key, :] . Q[row, :]     A = K, B = Q
//   O^T[dim, row] += V^T[dim, key] P^T[key, row]
//
// K's A operand wants eight dims of one key per lane, in any order that Q shares,
// so a lane loads 16 bytes of a key's row and that is its operand (16-bit), or two
// of them (8-bit).  V's A operand wants eight keys of one dim per lane.  Which dim a
// lane's row of the tile stands for is free, so lane r of 16 owns the dims
// r * D/16 .. + D/16 - 1, loads that piece of the row for each of its keys, and
// pairs of keys are put together with byte permutes.  The keys a lane needs
// there are those whose scores it holds (rows 4g .. 4g+3 of each 16-key tile), so P^T
// goes from the score tile into the second product as it is.
//
// 8-bit codes are exact in fp16, so both products run in fp16: Q is scaled by a power
// of two per row (largest element in [2^14, 2^15); what falls below fp16's
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
  int page_shift;  // log2(page_size), or -1
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

// What a row block has to stream: the key chunks that some row of it may see, as
// chunks 0 .. ca - 1 (the visible prefix) and cb .. ce - 1, and its splits.
struct Block {
  int n0, n1;      // first and last query token
  int prefix;      // keys below it are visible to every row (causal)
  int lo, hi;      // keys of the second part
  int ca, cb;      // chunks of the first part; first chunk of the second
  int chunks;      // chunks in all
  int per, splits; // chunks of a split, splits
};

template <int CK>
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
  k.ca = (k.prefix + CK - 1) / CK;
  k.cb = k.lo / CK;
  if (k.ca >= k.cb) {
    k.ca = k.cb = 0;
    k.lo = 0;
  }
  k.chunks = k.ca + (k.hi + CK - 1) / CK - k.cb;
  k.per = max(p.split_keys / CK, (k.chunks + p.num_splits - 1) / p.num_splits);
  k.splits = max(1, (k.chunks + k.per - 1) / k.per);
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

template <int NB>
__device__ __forceinline__ void load_words(const char* p, uint32_t* out) {
  if constexpr (NB == 16) {
    const w4 v = *reinterpret_cast<const w4*>(p);
    out[0] = v[0];
    out[1] = v[1];
    out[2] = v[2];
    out[3] = v[3];
  } else if constexpr (NB == 8) {
    const w2 v = *reinterpret_cast<const w2*>(p);
    out[0] = v[0];
    out[1] = v[1];
  } else {
    out[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// Whether any 16-bit value of the operands is infinite or NaN.
template <bool BF16, int N>
__device__ __forceinline__ bool any_not_finite(const w4 (&f)[N]) {
  constexpr uint32_t kExp = BF16 ? 0x7f80u : 0x7c00u;
  bool any = false;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      any |= ((f[i][j] & kExp) == kExp) | (((f[i][j] >> 16) & kExp) == kExp);
  return __builtin_amdgcn_ballot_w64(any) != 0;
}

// KIND: what the cache holds.  D: head_dim.  RT: row tiles of 16 in a row block.
// PAGE16: page_size is a multiple of 16, so a 16-key tile lies in one page and its
// page id and scales are wave-uniform; other page sizes look every key up.
template <int KIND, int D, int RT, bool PAGE16>
__global__ __launch_bounds__(kPaThreads, RT == 1 ? 2 : 1) void paged_attn_kernel(PagedAttnArgs a) {
  typedef Cache<KIND> C;
  typedef typename C::frag frag;
  constexpr bool Q8 = C::kQuant;
  constexpr int KT = D == 128 ? 2 : 4;       // 16-key tiles of a chunk
  constexpr int CK = KT * 16;                // keys of a chunk
  constexpr int KS = D / 32;                 // steps of the score product
  constexpr int KL = D * C::kBytes / 64;     // 16-byte loads of a lane per key row
  constexpr int DL = D / 16;                 // dims of V a lane owns
  constexpr int VB = DL * C::kBytes;         // their bytes
  constexpr int VW = VB / 4;
  constexpr int ROWS = RT * 16;
  constexpr int OS = D + 4;  // LDS row stride (floats)
  const atlas_paged_attn_t& p = a.p;

  __shared__ __attribute__((aligned(16))) float o_lds[kPaWaves][16 * OS];
  __shared__ float ml_lds[kPaWaves][16][2];

  // Row blocks of one (request, head, split) stream the same keys: they run next to
  // each other on one XCD (workgroups go round the 8 XCDs).
  int unit, rb;
  if (p.row_blocks == 1) {
    unit = blockIdx.x;
    rb = 0;
  } else {
    const int j = blockIdx.x >> 3;
    rb = j % p.row_blocks;
    unit = (j / p.row_blocks) * 8 + (blockIdx.x & 7);
  }
  const int h = unit % p.num_kv_heads;
  const int split = (unit / p.num_kv_heads) % p.num_splits;
  const int b = unit / p.num_kv_heads / p.num_splits;
  if (b >= p.batch) return;
  const Request r = read_request(p, b);
  const int row_start = rb * ROWS;
  const int rows = min(ROWS, r.q_len * a.group - row_start);
  if (rows <= 0) return;
  const Block k = plan_block<CK>(a, r, b, row_start, rows);
  if (split >= k.splits) return;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, r16 = lane & 15;
  const bool bf16 = p.dtype == ATLAS_DTYPE_BF16;
  const int shift = r.kv_len - r.q_len;  // position of query token 0

  // ---- queries ----
  frag qf[RT][KS];
  float qscale[RT];  // factor of a row's scores, to powers of two (8-bit: without K's scale)
  float m_run[RT], l_run[RT], slope[RT];
  f32x4 o[RT][DL];
  int node_of[RT];
  uint64_t word[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row = rt * 16 + r16;
    const bool ok = row < rows;
    const int prow = row_start + (ok ? row : 0);
    node_of[rt] = prow / a.group;
    const int head = h * a.group + (prow - node_of[rt] * a.group);
    const char* qrow = static_cast<const char*>(p.q) +
                       (int64_t(r.q0 + node_of[rt]) * p.q_stride_token + int64_t(head) * p.q_stride_head) * 2;
    qscale[rt] = a.scale_log2;
    if constexpr (!Q8) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        qf[rt][ks] = *reinterpret_cast<const frag*>(qrow + (ks * 32 + g * 8) * 2);
        if (!ok) qf[rt][ks] = frag{0, 0, 0, 0};
      }
    } else {
      // k-step 2j + e of group g holds dims 64 j + 16 g + 8 e ..: those of 16 codes
      float f[KS][8];
      float top = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const w4 v = *reinterpret_cast<const w4*>(qrow + ((ks >> 1) * 64 + g * 16 + (ks & 1) * 8) * 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t u = ok ? v[i] : 0;
          f[ks][2 * i] = bf16 ? __uint_as_float(u << 16) : float(__builtin_bit_cast(h2, u)[0]);
          f[ks][2 * i + 1] = bf16 ? __uint_as_float(u & 0xffff0000u) : float(__builtin_bit_cast(h2, u)[1]);
          top = fmaxf(top, fmaxf(fabsf(f[ks][2 * i]), fabsf(f[ks][2 * i + 1])));
        }
      }
      top = groups_max(top);
      // 2^-e with the largest element in [2^14, 2^15) (a row of zeros or below
      // 2^-111 takes the largest power, an infinite one whatever comes)
      const int e = min(max(int(__float_as_uint(top) >> 23) - 127 - 14, -126), 126);
      const float down = __uint_as_float(uint32_t(127 - e) << 23);
      qscale[rt] *= __uint_as_float(uint32_t(127 + e) << 23);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int i = 0; i < 4; ++i) qf[rt][ks][i] = pack_f16(f[ks][2 * i] * down, f[ks][2 * i + 1] * down);
    }
    m_run[rt] = -INFINITY;
    l_run[rt] = 0.f;
    slope[rt] = p.alibi_slopes ? p.alibi_slopes[head] * kPaLog2e : 0.f;
    word[rt] = (p.mask_mode == 1 && p.mask_words == 1 && ok) ? p.tree_mask[r.q0 + node_of[rt]] : 0ull;
#pragma unroll
    for (int t = 0; t < DL; ++t) o[rt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int col0 = p.mask_mode == 1 ? p.mask_col_start[b] : 0;

  // ---- keys ----
  const char* kbase = static_cast<const char*>(p.kv) + int64_t(h) * p.head_stride;
  const float* sbase = Q8 ? p.kv_scales + int64_t(h) * p.scale_stride_head : nullptr;
  const int64_t last_page = p.num_pages - 1;
  const int ts = int(p.token_stride);

  struct Raw {
    uint32_t k[KT][KL * 4];
    uint32_t v[KT][4][VW];
    float ks[PAGE16 ? KT : KT * 4];  // 8-bit: scales by tile, or by key
    float vs[PAGE16 ? KT : KT * 4];
  };
  auto page_slot = [&](int key) { return a.page_shift >= 0 ? key >> a.page_shift : key / p.page_size; };
  auto page_of = [&](int slot) -> int64_t {
    const int64_t id = p.kv_indices[r.pt + slot];
    return id < 0 ? 0 : (id > last_page ? last_page : id);
  };
  auto chunk_at = [&](int c) { return c < k.ca ? c : c - k.ca + k.cb; };
  // Keys outside [lo, hi) of the chunk's part repeat its nearest key.
  auto load = [&](Raw& x, int c) {
    const int kb = chunk_at(c) * CK;
    const int lo = c < k.ca ? 0 : k.lo;
    const int hi = (c < k.ca ? k.prefix : k.hi) - 1;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const int t0 = kb + kt * 16;
      if constexpr (PAGE16) {
        const int tile = min(max(t0, lo & ~15), hi & ~15);
        const int slot = page_slot(tile);
        const int64_t page = page_of(slot);
        const char* base = kbase + page * p.page_stride;
        const int first = slot * p.page_size;
        const int key = min(max(t0 + r16, lo), hi) - first;
#pragma unroll
        for (int j = 0; j < KL; ++j) load_words<16>(base + uint32_t(key * ts + j * 64 + g * 16), &x.k[kt][4 * j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int vk = min(max(t0 + 4 * g + i, lo), hi) - first;
          load_words<VB>(base + p.v_offset + uint32_t(vk * ts + r16 * VB), x.v[kt][i]);
        }
        if constexpr (Q8) {
          const float* s = sbase + page * p.scale_stride_page;
          x.ks[kt] = s[0];
          x.vs[kt] = s[p.scale_stride_kv];
        }
      } else {
        const int key = min(max(t0 + r16, lo), hi);
        const int slot = page_slot(key);
        const char* base = kbase + page_of(slot) * p.page_stride + int64_t(key - slot * p.page_size) * p.token_stride;
#pragma unroll
        for (int j = 0; j < KL; ++j) load_words<16>(base + j * 64 + g * 16, &x.k[kt][4 * j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int vk = min(max(t0 + 4 * g + i, lo), hi);
          const int vslot = page_slot(vk);
          const int64_t page = page_of(vslot);
          load_words<VB>(kbase + p.v_offset + page * p.page_stride +
                             int64_t(vk - vslot * p.page_size) * p.token_stride + r16 * VB, x.v[kt][i]);
          if constexpr (Q8) {
            const float* s = sbase + page * p.scale_stride_page;
            x.ks[kt * 4 + i] = s[0];
            x.vs[kt * 4 + i] = s[p.scale_stride_kv];
          }
        }
      }
    }
  };

  // Largest V scale so far: O holds sums of p * v * (scale / vref).
  float vref = 1.17549435e-38f, vinv = 8.5070592e37f;

  auto compute = [&](const Raw& x, int c) {
    const int kb = chunk_at(c) * CK;
    // does some key of the chunk hide from some row?
    bool masked;
    if (p.mask_mode == 2) {
      masked = !(kb + CK <= k.prefix ||
                 (kb + CK <= shift + k.n0 + 1 && (p.window_left < 0 || kb >= shift + k.n1 - p.window_left)));
    } else {
      masked = kb + CK > (p.mask_mode == 1 ? min(r.kv_len, col0) : r.kv_len);
    }
    frag kf[KT][KS];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if constexpr (Q8) kf[kt][ks] = C::keys8(x.k[kt][2 * ks], x.k[kt][2 * ks + 1]);
        else kf[kt][ks] = frag{x.k[kt][4 * ks], x.k[kt][4 * ks + 1], x.k[kt][4 * ks + 2], x.k[kt][4 * ks + 3]};
      }
    frag vf[KT / 2][DL];
#pragma unroll
    for (int tp = 0; tp < KT / 2; ++tp) {
      uint32_t raw[8][VW];
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int w = 0; w < VW; ++w) raw[i][w] = x.v[2 * tp + (i >> 2)][i & 3][w];
      transpose_v<KIND, VW, DL>(raw, vf[tp]);
    }
    // Infinities and NaN in V rows that a row does not see must not reach it
    // (0 * inf): in chunks with hidden keys they are taken out of the product and
    // added to the rows that see them.
    bool strange = false;
    if (masked && KIND != kCacheInt8) {
#pragma unroll
      for (int tp = 0; tp < KT / 2; ++tp) strange |= any_not_finite<C::kBf16>(vf[tp]);
    }
    if constexpr (Q8) {
      float top = x.vs[0];
#pragma unroll
      for (int i = 1; i < (PAGE16 ? KT : KT * 4); ++i) top = fmaxf(top, x.vs[i]);
      if (__builtin_amdgcn_ballot_w64(top > vref) != 0) {
        if constexpr (!PAGE16) top = groups_max(top);
        const float now = fmaxf(vref, top);
        const float down = vref / now;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int t = 0; t < DL; ++t) o[rt][t] *= down;
        vref = now;
        vinv = 1.0f / now;
      }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float s[KT * 4];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) acc = C::mfma(kf[kt][ks], qf[rt][ks], acc);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (Q8) s[kt * 4 + i] = acc[i] * (qscale[rt] * x.ks[PAGE16 ? kt : kt * 4 + i]);
          else s[kt * 4 + i] = acc[i] * qscale[rt];
        }
      }
      if (p.soft_cap > 0.f) {
        // cap * tanh(y / cap) = cap * (1 - 2 / (1 + e^(2 y / cap))), to powers of two
#pragma unroll
        for (int i = 0; i < KT * 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(s[i] * a.cap_in);
          s[i] = __builtin_fmaf(-2.f * a.cap_out, __builtin_amdgcn_rcpf(1.f + e), a.cap_out);
        }
      }
      const int qpos = shift + node_of[rt];
      if (p.alibi_slopes != nullptr) {
#pragma unroll
        for (int i = 0; i < KT * 4; ++i) {
          const int key = kb + (i >> 2) * 16 + 4 * g + (i & 3);
          s[i] = __builtin_fmaf(-slope[rt], fabsf(float(qpos - key)), s[i]);
        }
      }
      if (masked) {
        uint64_t w = word[rt];
        int w0 = col0;
        if (p.mask_mode == 1 && p.mask_words > 1) {
          // one word for each 64 keys; a chunk lies in one of them
          const int idx = (kb >> 6) - (col0 >> 6);
          w = idx < 0 ? ~0ull
                      : (idx < p.mask_words && rt * 16 + r16 < rows
                             ? p.tree_mask[int64_t(r.q0 + node_of[rt]) * p.mask_words + idx] : 0ull);
          w0 = kb & ~63;
        }
#pragma unroll
        for (int i = 0; i < KT * 4; ++i) {
          const int key = kb + (i >> 2) * 16 + 4 * g + (i & 3);
          bool vis = key < r.kv_len;
          if (p.mask_mode == 2) {
            const bool near = key <= qpos && (p.window_left < 0 || key >= qpos - p.window_left);
            vis = vis && (near || key < k.prefix);
          } else if (p.mask_mode == 1) {
            const int off = key - w0;
            vis = vis && (off < 0 || (off < 64 && ((w >> (off & 63)) & 1)));
          }
          s[i] = vis ? s[i] : -INFINITY;
        }
      }
      float mx = s[0];
#pragma unroll
      for (int i = 1; i < KT * 4; ++i) mx = pa_max(mx, s[i]);
      if (__builtin_amdgcn_ballot_w64(mx > m_run[rt] + kPaLazyLog2) != 0) {
        const float m_new = fmaxf(m_run[rt], groups_max(mx));
        const float alpha = m_run[rt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m_run[rt] - m_new);
        l_run[rt] *= alpha;
#pragma unroll
        for (int t = 0; t < DL; ++t) o[rt][t] *= alpha;
        m_run[rt] = m_new;
      }
      const float m = m_run[rt] == -INFINITY ? 0.f : m_run[rt];
      frag pf[KT / 2];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[i] = __builtin_amdgcn_exp2f(s[kt * 4 + i] - m);
          l_run[rt] += e[i];
          if constexpr (Q8) e[i] *= x.vs[PAGE16 ? kt : kt * 4 + i] * vinv;
        }
        pf[kt >> 1][(kt & 1) * 2] = C::pack(e[0], e[1]);
        pf[kt >> 1][(kt & 1) * 2 + 1] = C::pack(e[2], e[3]);
      }
      if (!strange) {
#pragma unroll
        for (int t = 0; t < DL; ++t)
#pragma unroll
          for (int tp = 0; tp < KT / 2; ++tp) o[rt][t] = C::mfma(vf[tp][t], pf[tp], o[rt][t]);
      } else {
        constexpr uint32_t kExp = C::kBf16 ? 0x7f80u : 0x7c00u, kOne = C::kBf16 ? 0x3f80u : 0x3c00u;
#pragma unroll
        for (int t = 0; t < DL; ++t) {
          f32x4 plus = f32x4{0.f, 0.f, 0.f, 0.f}, minus = plus;
#pragma unroll
          for (int tp = 0; tp < KT / 2; ++tp) {
            frag fine, up, dn;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              fine[j] = up[j] = dn[j] = 0;
#pragma unroll
              for (int hw = 0; hw < 2; ++hw) {
                const uint32_t v = (vf[tp][t][j] >> (16 * hw)) & 0xffffu;
                const bool odd = (v & kExp) == kExp, nan = (v & 0x7fffu) > kExp;
                fine[j] |= (odd ? 0u : v) << (16 * hw);
                up[j] |= (odd && (nan || v == kExp) ? kOne : 0u) << (16 * hw);
                dn[j] |= (odd && (nan || v != kExp) ? kOne : 0u) << (16 * hw);
              }
            }
            o[rt][t] = C::mfma(fine, pf[tp], o[rt][t]);
            plus = C::mfma(up, pf[tp], plus);
            minus = C::mfma(dn, pf[tp], minus);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (plus[i] > 0.f) o[rt][t][i] += INFINITY;
            if (minus[i] > 0.f) o[rt][t][i] -= INFINITY;
          }
        }
      }
    }
  };

  const int c_end = min(k.chunks, (split + 1) * k.per);
  int c = split * k.per + wave;
  if (c < c_end) {
    // The next chunk of the wave is in flight while this one is computed; the last
    // one is asked for again rather than branched around, so the waits stay exact.
    Raw x, y;
    load(x, c);
    while (true) {
      load(y, c + kPaWaves < c_end ? c + kPaWaves : c);
      compute(x, c);
      c += kPaWaves;
      if (c >= c_end) break;
      load(x, c + kPaWaves < c_end ? c + kPaWaves : c);
      compute(y, c);
      c += kPaWaves;
      if (c >= c_end) break;
    }
  }

  // ---- the waves' states into one ----
  const int item = (b * p.num_kv_heads + h) * p.row_blocks + rb;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const float l = groups_sum(l_run[rt]);
    if (rt > 0) __syncthreads();
    if (g == 0) {
      ml_lds[wave][r16][0] = m_run[rt];
      ml_lds[wave][r16][1] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int t = 0; t < DL; ++t)
        o_lds[wave][r16 * OS + (4 * g + i) * DL + t] = Q8 ? o[rt][t][i] * vref : o[rt][t][i];
    __syncthreads();
    const int row = tid >> 4, d0 = (tid & 15) * DL;
    float m = ml_lds[0][row][0];
#pragma unroll
    for (int w = 1; w < kPaWaves; ++w) m = fmaxf(m, ml_lds[w][row][0]);
    float sum = 0.f, acc[DL];
#pragma unroll
    for (int t = 0; t < DL; ++t) acc[t] = 0.f;
#pragma unroll
    for (int w = 0; w < kPaWaves; ++w) {
      const float mw = ml_lds[w][row][0];
      const float f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - m);
      sum += f * ml_lds[w][row][1];
      if (mw == -INFINITY) continue;
#pragma unroll
      for (int t = 0; t < DL; ++t) acc[t] += f * o_lds[w][row * OS + d0 + t];
    }
    const int lr = rt * 16 + row;
    if (lr >= rows) continue;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const float lse2 = sum == 0.f ? -INFINITY : m + __builtin_log2f(sum);
    if (k.splits > 1) {
      float* ws = static_cast<float*>(p.workspace);
      const int64_t prow = (int64_t(item) * p.num_splits + split) * ROWS + lr;
      const int64_t nrows = int64_t(p.batch) * p.num_kv_heads * p.row_blocks * p.num_splits * ROWS;
#pragma unroll
      for (int t = 0; t < DL; t += 4)
        *reinterpret_cast<f32x4*>(ws + prow * D + d0 + t) =
            f32x4{acc[t] * inv, acc[t + 1] * inv, acc[t + 2] * inv, acc[t + 3] * inv};
      if ((tid & 15) == 0) ws[nrows * D + prow] = lse2;
    } else {
      const int prow = row_start + lr, node = prow / a.group;
      const int head = h * a.group + (prow - node * a.group);
      char* out = static_cast<char*>(p.out) +
                  (int64_t(r.q0 + node) * p.out_stride_token + int64_t(head) * p.out_stride_head + d0) * 2;
      uint32_t packed[DL / 2];
#pragma unroll
      for (int t = 0; t < DL / 2; ++t)
        packed[t] = bf16 ? pack_bf16(acc[2 * t] * inv, acc[2 * t + 1] * inv)
                         : pack_f16(acc[2 * t] * inv, acc[2 * t + 1] * inv);
      if constexpr (DL == 8) *reinterpret_cast<w4*>(out) = w4{packed[0], packed[1], packed[2], packed[3]};
      else *reinterpret_cast<w2*>(out) = w2{packed[0], packed[1]};
      if (p.lse != nullptr && (tid & 15) == 0)
        p.lse[int64_t(r.q0 + node) * p.num_qo_heads + head] = lse2 * kPaLn2;
    }
  }
}

// Joins the splits of a row block: one wave per row, its lanes over the dims.
template <int D, int RT>
__global__ __launch_bounds__(256) void paged_attn_merge_kernel(PagedAttnArgs a) {
  constexpr int CK = D == 128 ? 32 : 64;
  constexpr int ROWS = RT * 16, PL = D / 64;
  const atlas_paged_attn_t& p = a.p;
  const int item = blockIdx.x;
  const int rb = item % p.row_blocks;
  const int h = item / p.row_blocks % p.num_kv_heads;
  const int b = item / p.row_blocks / p.num_kv_heads;
  const Request r = read_request(p, b);
  const int row_start = rb * ROWS;
  const int rows = min(ROWS, r.q_len * a.group - row_start);
  const int lr = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (lr >= rows) return;
  const Block k = plan_block<CK>(a, r, b, row_start, rows);
  if (k.splits <= 1) return;
  const int lane = threadIdx.x & 63;
  const float* ws = static_cast<const float*>(p.workspace);
  const int64_t nrows = int64_t(p.batch) * p.num_kv_heads * p.row_blocks * p.num_splits * ROWS;
  const int64_t row0 = int64_t(item) * p.num_splits * ROWS + lr;
  float m = -INFINITY;
  for (int s = 0; s < k.splits; ++s) m = fmaxf(m, ws[nrows * D + row0 + int64_t(s) * ROWS]);
  float sum = 0.f, acc[PL];
#pragma unroll
  for (int t = 0; t < PL; ++t) acc[t] = 0.f;
  for (int s = 0; s < k.splits; ++s) {
    const int64_t prow = row0 + int64_t(s) * ROWS;
    const float lse2 = ws[nrows * D + prow];
    if (lse2 == -INFINITY) continue;
    const float f = __builtin_amdgcn_exp2f(lse2 - m);
    sum += f;
#pragma unroll
    for (int t = 0; t < PL; ++t) acc[t] += f * ws[prow * D + lane * PL + t];
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int prow = row_start + lr, node = prow / a.group;
  const int head = h * a.group + (prow - node * a.group);
  uint16_t* out = static_cast<uint16_t*>(p.out) + int64_t(r.q0 + node) * p.out_stride_token +
                  int64_t(head) * p.out_stride_head + lane * PL;
  const bool bf16 = p.dtype == ATLAS_DTYPE_BF16;
  if constexpr (PL == 2)
    *reinterpret_cast<uint32_t*>(out) = bf16 ? pack_bf16(acc[0] * inv, acc[1] * inv) : pack_f16(acc[0] * inv, acc[1] * inv);
  else
    *out = uint16_t(bf16 ? pack_bf16(acc[0] * inv, 0.f) : pack_f16(acc[0] * inv, 0.f));
  if (p.lse != nullptr && lane == 0)
    p.lse[int64_t(r.q0 + node) * p.num_qo_heads + head] = sum == 0.f ? -INFINITY : (m + __builtin_log2f(sum)) * kPaLn2;
}

template <int KIND, int D, int RT>
int launch_paged_attn(const PagedAttnArgs& a, hipStream_t stream) {
  const atlas_paged_attn_t& p = a.p;
  const int64_t units = int64_t(p.batch) * p.num_kv_heads * p.num_splits;
  const int64_t blocks = p.row_blocks == 1 ? units : (units + 7) / 8 * 8 * p.row_blocks;
  const dim3 grid(static_cast<unsigned>(blocks));
  if (p.page_size % 16 == 0)
    hipLaunchKernelGGL((paged_attn_kernel<KIND, D, RT, true>), grid, dim3(kPaThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((paged_attn_kernel<KIND, D, RT, false>), grid, dim3(kPaThreads), 0, stream, a);
  int rc = launch_status("paged_attn_kernel");
  if (rc || p.num_splits == 1) return rc;
  const dim3 mgrid(static_cast<unsigned>(p.batch * p.num_kv_heads * p.row_blocks), RT * 4);
  hipLaunchKernelGGL((paged_attn_merge_kernel<D, RT>), mgrid, dim3(256), 0, stream, a);
  return launch_status("paged_attn_merge_kernel");
}

template <int KIND>
int launch_paged_attn_kind(const PagedAttnArgs& a, hipStream_t stream) {
  const bool one = a.p.row_tiles == 1;
  if (a.p.head_dim == 128) return one ? launch_paged_attn<KIND, 128, 1>(a, stream) : launch_paged_attn<KIND, 128, 4>(a, stream);
  return one ? launch_paged_attn<KIND, 64, 1>(a, stream) : launch_paged_attn<KIND, 64, 4>(a, stream);
}

}  // namespace
}  // namespace atlas

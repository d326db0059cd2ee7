// Paged attention for many packed rows: prompts' chunks and wide draft trees.
//
// A workgroup of eight waves takes up to 256 packed rows of one KV head and one split
// of the request's keys.  Tiles of 64 keys go from HBM through registers into LDS as
// 16-bit rows (8-bit codes are converted on the way, once for all rows): one tile is
// computed from one of two stages, the next is written to the other, and one more (two
// at head_dim 64) is on its way.  Row tiles of 16 go round the waves, two for each; K's
// operand is a 16-byte LDS read, V's two transposing reads.  A row's 16-byte granules
// are swapped by the key so that neither the writes nor either kind of read meets in a
// bank.
//
// Bound by the vector instructions of the softmax (per score of a lane about ten, the
// exponential counting for four) beside the matrix instructions, which two waves of a SIMD
// overlap in part.  Four waves on 128 rows, two such workgroups to a CU, or tiles of 32 keys
// took 3 to 10 % longer: each wave then has more of the staging to do, or meets more barriers.
// 146 us (450 TFLOP/s) for two chunks of 512 tokens over up to 5464 keys with a distance
// bias; 75 us (320 TFLOP/s) for four trees of 200 nodes over an int8 cache.
#pragma once

#include "paged_attn.hpp"

namespace atlas {
namespace {

typedef short s4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ w2 read_tr16(const char* p) {
  return __builtin_bit_cast(w2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                    (__attribute__((address_space(3))) s4*)(p)));
}

// LDS writes of every wave are visible behind it; loads from memory stay in flight.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

constexpr int kRowWaves = 8;
constexpr int kRowThreads = 64 * kRowWaves;

template <int N>
using Stage = std::integral_constant<int, N>;

// KIND: what the cache holds.  D: head_dim.  PAGE16: page_size is a multiple of 16, so a 16-key tile lies in one page and its id and scales are
// wave-uniform; other page sizes look every key up.  SCORED: scores may be capped or
// biased, or their factor negative.
template <int KIND, int D, bool PAGE16, bool SCORED>
__global__ __launch_bounds__(kRowThreads, 2) void paged_rows_kernel(PagedAttnArgs a) {
  typedef Cache<KIND> C;
  typedef typename C::frag frag;
  constexpr bool Q8 = C::kQuant;
  constexpr int RT = 2;                    // row tiles of a wave
  constexpr int TK = 64;                   // keys of a tile
  constexpr int SUB = kChunk / TK;         // tiles of a chunk
  constexpr int NT = TK / 16;              // its 16-key tiles
  constexpr int KS = D / 32;               // steps of the score product
  constexpr int DT = D / 16;               // 16-dim tiles of O
  constexpr int RB = D * 2;                // bytes of an LDS row
  constexpr int GR = RB / 16;              // its granules
  constexpr int HALF = TK * RB;            // K's or V's half of a stage
  constexpr int PB = 8 * C::kBytes;        // bytes of eight values in the cache, a granule in LDS
  constexpr int KSW = GR - 1;              // granule swaps: K by key, V by key pairs
  constexpr int VSW = GR / 2 - 1;
  const atlas_paged_attn_t& p = a.p;

  __shared__ __attribute__((aligned(16))) char lds[2][2 * HALF];
  constexpr int NSC = PAGE16 ? NT : TK;     // scales of a tile: by 16 keys, or by key
  __shared__ __attribute__((aligned(16))) float scale_lds[2][2][NSC];
  __shared__ int strange_lds[2];             // tile (+ 1) of the stage that holds such values
  __shared__ uint8_t up_lds[2][TK * D / 8];  // bits of V values that are +inf or NaN, by key and dim
  __shared__ uint8_t dn_lds[2][TK * D / 8];  // -inf or NaN

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
  const int row_start = rb * p.block_rows;
  const int rows = block_of(a, r, row_start);
  if (rows <= 0) return;
  const int tid = threadIdx.x, lane = tid & 63;
  const Block k = plan_block(a, r, b, row_start, rows);
  if (split >= k.splits) return;

  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, r16 = lane & 15;
  const bool bf16 = p.dtype == ATLAS_DTYPE_BF16;
  const int shift = r.kv_len - r.q_len;  // position of query token 0
  const int col0 = p.mask_mode == 1 ? p.mask_col_start[b] : 0;
  // this wave's row tiles are wave, wave + 4 (one without rows computes with queries of zeros)
  const bool computes = wave * 16 < rows;

  // ---- queries ----
  frag qf[RT][KS];
  float qscale[RT], m_run[RT], l_run[RT], slope[RT];
  f32x4 o[RT][DT];
  int node_of[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row = (wave + kRowWaves * rt) * 16 + r16;
    const bool ok = row < rows;
    const int prow = row_start + (ok ? row : 0);
    node_of[rt] = prow / a.group;
    const int head = h * a.group + (prow - node_of[rt] * a.group);
    const char* qrow = static_cast<const char*>(p.q) +
                       (int64_t(r.q0 + node_of[rt]) * p.q_stride_token + int64_t(head) * p.q_stride_head) * 2;
    qscale[rt] = a.scale_log2;
    w4 v[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      v[ks] = *reinterpret_cast<const w4*>(qrow + (ks * 32 + g * 8) * 2);
      if (!ok) v[ks] = w4{0, 0, 0, 0};
    }
    if constexpr (Q8) {
      float f[KS][8];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) q_floats(v[ks], bf16, f[ks]);
      qscale[rt] *= q_to_f16<KS>(f, qf[rt]);
    } else {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qf[rt][ks] = v[ks];
    }
    m_run[rt] = -INFINITY;
    l_run[rt] = 0.f;
    slope[rt] = SCORED && p.alibi_slopes ? p.alibi_slopes[head] * kPaLog2e : 0.f;
#pragma unroll
    for (int t = 0; t < DT; ++t) o[rt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // ---- keys ----
  const char* kbase = static_cast<const char*>(p.kv) + int64_t(h) * p.head_stride;
  const char* vbase = kbase + p.v_offset;
  const int ts = int(p.token_stride);
  const int page_size = p.page_size;
  Pages pages;
  pages.begin(a, r);

  auto key_of = [&](int c) __attribute__((always_inline)) {
    return (c < k.ca * SUB ? c : c - k.ca * SUB + k.cb * SUB) * TK;
  };
  auto bounds = [&](int c, int& lo, int& hi) __attribute__((always_inline)) {
    lo = c < k.ca * SUB ? 0 : k.lo;
    hi = (c < k.ca * SUB ? k.prefix : k.hi) - 1;
  };
  // 64 / NT tiles make a window: lane l holds the offset of the first row of 16-key tile
  // l % NT of its tile l / NT, and that page's scales.  A window is read at once, when
  // its first tile is asked for, so that the loads of the key loop are all alike and
  // a wait for one tile's rows is not a wait for the next one's page ids.
  constexpr int WIN = 64 / NT;
  int64_t win_rows = 0;
  float win_ks = 0.f, win_vs = 0.f;
  int win0 = 0, win1 = 0;
  auto open_window = [&](int c, int end) __attribute__((always_inline)) {
    win0 = c;
    win1 = min(end, c + WIN);
    const int mine = min(c + lane / NT, win1 - 1);
    int lo, hi;
    bounds(mine, lo, hi);
    const int tile = Pages::tile_key(key_of(mine), lane & (NT - 1), lo, hi);
    const int id = pages.read_id(a, tile);
    win_rows = pages.row_offset(a, id, tile);
    if constexpr (Q8) {
      const float* sc = p.kv_scales + int64_t(h) * p.scale_stride_head + pages.valid(id) * p.scale_stride_page;
      win_ks = sc[0];
      win_vs = sc[p.scale_stride_kv];
    }
  };
  // A thread carries eight values of NL K rows and of as many V rows of a tile: those of
  // granule `gr` of rows `row`, `row` + RSTEP ..
  constexpr int NL = TK * GR / kRowThreads, RSTEP = kRowThreads / GR;
  static_assert(RSTEP % 16 == 0, "a thread's rows have the same place in their 16-key tiles");
  typedef std::conditional_t<Q8, w2, w4> Piece;
  const int gr = tid % GR, row = tid / GR;
  const int kt_of = wave * (64 / GR) >> 4;  // (a wave's rows lie in one 16-key tile)
  const uint32_t piece_at = uint32_t((row & 15) * ts + gr * PB);
  constexpr int KTH = kRowThreads / TK;  // threads per key
  constexpr int SETS = 2 / NL;           // tiles in flight in registers
  struct Raw {
    Piece k[NL], v[NL];
    float ks, vs;  // scales of 16-key tile lane % NT; other page sizes: of key tid / KTH
  };
  // Keys outside [lo, hi) of the tile's part repeat its nearest key.
  auto load = [&](Raw& x, int c) __attribute__((always_inline)) {
    const int kb = key_of(c);
    int lo, hi;
    bounds(c, lo, hi);
    const bool whole = (kb >= lo) & (kb + TK <= hi + 1);
#pragma unroll
    for (int j = 0; j < NL; ++j) {
      if constexpr (PAGE16) {
        const int kt = kt_of + j * RSTEP / 16;
        const int64_t row0 = Pages::tile_row(win_rows, (c - win0) * NT + kt);
        uint32_t off = piece_at;
        if (!whole)
          off = uint32_t((min(max(kb + row + j * RSTEP, lo), hi) - Pages::tile_key(kb, kt, lo, hi)) * ts + gr * PB);
        x.k[j] = *reinterpret_cast<const Piece*>(kbase + row0 + off);
        x.v[j] = *reinterpret_cast<const Piece*>(vbase + row0 + off);
      } else {
        const int key = min(max(kb + row + j * RSTEP, lo), hi);
        const int slot = slot_of(a, key);
        const int64_t at = pages.valid(pages.ids[slot]) * p.page_stride + int64_t(key - slot * page_size) * ts + gr * PB;
        x.k[j] = *reinterpret_cast<const Piece*>(kbase + at);
        x.v[j] = *reinterpret_cast<const Piece*>(vbase + at);
      }
    }
    if constexpr (Q8 && PAGE16) {
      const int from = ((c - win0) * NT + (lane & (NT - 1))) * 4;
      x.ks = __uint_as_float(__builtin_amdgcn_ds_bpermute(from, __float_as_uint(win_ks)));
      x.vs = __uint_as_float(__builtin_amdgcn_ds_bpermute(from, __float_as_uint(win_vs)));
    } else if constexpr (Q8) {
      const int slot = slot_of(a, min(max(kb + tid / KTH, lo), hi));
      const float* s = p.kv_scales + int64_t(h) * p.scale_stride_head + pages.valid(pages.ids[slot]) * p.scale_stride_page;
      x.ks = s[0];
      x.vs = s[p.scale_stride_kv];
    }
  };
  // Does some key of tile c hide from some row?
  const int plain_hi = p.mask_mode == 2 ? shift + k.n0 + 1 : (p.mask_mode == 1 ? min(r.kv_len, col0) : r.kv_len);
  const int plain_lo = p.mask_mode == 2 && p.window_left >= 0 ? shift + k.n1 - p.window_left : 0;
  auto masked_tile = [&](int kb) __attribute__((always_inline)) {
    return ((kb + TK > plain_hi) | (kb < plain_lo)) & (kb + TK > k.prefix);
  };
  // Infinities and NaN in V rows that a row does not see must not reach it (0 * inf):
  // in tiles with hidden keys they are stored as zeros and marked, and the rows
  // that see them get them from the marks.
  auto take_out = [&](frag v, int st, int at, uint32_t& odd) __attribute__((always_inline)) {
    uint32_t up = 0, dn = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t u, d;
      v[w] = take_out2<C::kBf16>(v[w], u, d);
      up |= ((u >> 15 & 1u) | (u >> 30 & 2u)) << (2 * w);
      dn |= ((d >> 15 & 1u) | (d >> 30 & 2u)) << (2 * w);
      odd |= u | d;
    }
    up_lds[st][at * GR + gr] = uint8_t(up);
    dn_lds[st][at * GR + gr] = uint8_t(dn);
    return v;
  };
  const int k_to = row * RB + ((gr ^ (row & KSW)) << 4), v_to = row * RB + ((gr ^ ((row & VSW) << 1)) << 4);
  auto store = [&](const Raw& x, auto st_tag, int c) __attribute__((always_inline)) {
    constexpr int st = decltype(st_tag)::value;
    frag vv[NL];
#pragma unroll
    for (int j = 0; j < NL; ++j) {
      frag kk;
      if constexpr (Q8) {
        kk = C::keys8(x.k[j][0], x.k[j][1]);
        vv[j] = C::keys8(x.v[j][0], x.v[j][1]);
      } else {
        kk = x.k[j];
        vv[j] = x.v[j];
      }
      *reinterpret_cast<frag*>(lds[st] + k_to + j * RSTEP * RB) = kk;
    }
    if (KIND != kCacheInt8 && masked_tile(key_of(c))) {
      // (the marks of a tile are whole: every thread writes its part, whether it has some or not)
      uint32_t odd = 0;
#pragma unroll
      for (int j = 0; j < NL; ++j) vv[j] = take_out(vv[j], st, row + j * RSTEP, odd);
      if (odd) strange_lds[st] = c + 1;
    }
#pragma unroll
    for (int j = 0; j < NL; ++j) *reinterpret_cast<frag*>(lds[st] + HALF + v_to + j * RSTEP * RB) = vv[j];
    if constexpr (Q8 && PAGE16) {
      if (tid < NT) {
        scale_lds[st][0][tid] = x.ks;
        scale_lds[st][1][tid] = x.vs;
      }
    } else if constexpr (Q8) {
      if (tid % KTH == 0) {
        scale_lds[st][0][tid / KTH] = x.ks;
        scale_lds[st][1][tid / KTH] = x.vs;
      }
    }
  };

  // Largest V scale so far: O holds sums of p * v * (scale / vref).
  float vref = 1.17549435e-38f, vinv = 8.5070592e37f;

  // Lane parts of the LDS addresses: K row r16 of a 16-key tile, V rows 4g + r16 / 4.
  const int e4 = r16 >> 2, q4 = r16 & 3;
  const int vkey = 4 * g + e4;

  // One tile for this wave's row tiles, 32 keys at a time.
  auto compute = [&](auto masked_tag, auto st_tag, int c) __attribute__((always_inline)) {
    constexpr bool masked = decltype(masked_tag)::value;
    constexpr int st = decltype(st_tag)::value;
    const int kb = key_of(c);
    const char* kd = lds[st];
    const char* vd = lds[st] + HALF;
    const bool strange = masked && KIND != kCacheInt8 && strange_lds[st] == c + 1;
#pragma unroll
    for (int hh = 0; hh < TK / 32; ++hh) {
      f32x4 acc[RT][2];
      // The reads of an operand run ahead of the products before it, in this order: the
      // compiler would put each next to its use, and every product would wait for its read.
      frag kf[2][KS];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
          kf[kt][ks] = *reinterpret_cast<const frag*>(kd + (hh * 32 + kt * 16 + r16) * RB + (((ks * 4 + g) ^ (r16 & KSW)) << 4));
      f32x4 ksk[2], vsk[2];  // scales of the lane's keys (by 16-key tile: the first element)
      if constexpr (Q8) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          if constexpr (PAGE16) {
            ksk[kt][0] = scale_lds[st][0][hh * 2 + kt];
            vsk[kt][0] = scale_lds[st][1][hh * 2 + kt];
          } else {
            ksk[kt] = *reinterpret_cast<const f32x4*>(&scale_lds[st][0][hh * 32 + kt * 16 + 4 * g]);
            vsk[kt] = *reinterpret_cast<const f32x4*>(&scale_lds[st][1][hh * 32 + kt * 16 + 4 * g]);
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) acc[rt][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int kt = 0; kt < 2; ++kt) acc[rt][kt] = C::mfma(kf[kt][ks], qf[rt][ks], acc[rt][kt]);
      __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
      frag vf[DT];  // V^T's operands by dim tile
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        const char* at = vd + (32 * hh + vkey) * RB + (((2 * t + (q4 >> 1)) ^ ((vkey & VSW) << 1)) << 4) + ((q4 & 1) << 3);
        const w2 lo = read_tr16(at), hi = read_tr16(at + 16 * RB);
        vf[t] = frag{lo[0], lo[1], hi[0], hi[1]};
      }
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (Q8) {
        float top = pa_max(vsk[0][0], vsk[1][0]);
        if constexpr (!PAGE16) {
#pragma unroll
          for (int i = 1; i < 4; ++i) top = pa_max(top, pa_max(vsk[0][i], vsk[1][i]));
          top = groups_max(top);
        }
        if (__builtin_amdgcn_ballot_w64(top > vref) != 0) {
          const float down = vref / top;
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int t = 0; t < DT; ++t) o[rt][t] *= down;
          vref = top;
          vinv = 1.0f / top;
        }
      }
      frag pf[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int qpos = shift + node_of[rt];
        const int key0 = kb + hh * 32 + 4 * g;
        // x: scores to powers of two; without a cap, a bias or hidden keys the factor (not
        // negative there) is left to the exponent
        float x[8], f[PAGE16 || !Q8 ? 2 : 8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = acc[rt][i >> 2][i & 3];
#pragma unroll
        for (int i = 0; i < (PAGE16 || !Q8 ? 2 : 8); ++i)
          f[i] = !Q8 ? qscale[rt] : qscale[rt] * (PAGE16 ? ksk[i][0] : ksk[i >> 2][i & 3]);
        if constexpr (SCORED || masked) {
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] *= f[PAGE16 || !Q8 ? i >> 2 : i];
#pragma unroll
          for (int i = 0; i < (PAGE16 || !Q8 ? 2 : 8); ++i) f[i] = 1.f;
        }
        if constexpr (SCORED) {
          if (p.soft_cap > 0.f) {
            // cap * tanh(y / cap) = cap * (1 - 2 / (1 + e^(2 y / cap))), to powers of two
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float e = __builtin_amdgcn_exp2f(x[i] * a.cap_in);
              x[i] = __builtin_fmaf(-2.f * a.cap_out, __builtin_amdgcn_rcpf(1.f + e), a.cap_out);
            }
          }
          if (p.alibi_slopes != nullptr) {
            const float away = float(qpos - key0);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              x[i] = __builtin_fmaf(-slope[rt], fabsf(away - float((i >> 2) * 16 + (i & 3))), x[i]);
          }
        }
        if constexpr (masked) {
          uint64_t w = 0;
          int w0 = col0;
          if (p.mask_mode == 1) {
            // one word of the tree's columns, or one for each 64 keys (a tile lies in one of them)
            const int idx = p.mask_words > 1 ? (kb >> 6) - (col0 >> 6) : 0;
            if (idx >= 0 && idx < p.mask_words) w = p.tree_mask[int64_t(r.q0 + node_of[rt]) * p.mask_words + idx];
            if (idx < 0) w = ~0ull;
            if (p.mask_words > 1) w0 = kb & ~63;
          }
          const int wlo = p.window_left >= 0 ? qpos - p.window_left : 0;
#pragma unroll
          for (int kt = 0; kt < 2; ++kt) {
            const int at = key0 + kt * 16;
            uint32_t vis = below4(at, r.kv_len);
            if (p.mask_mode == 2) {
              vis &= (below4(at, qpos + 1) & ~below4(at, wlo)) | below4(at, k.prefix);
            } else if (p.mask_mode == 1) {
              vis &= tree4(w, at - w0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) x[kt * 4 + i] = (vis >> i) & 1u ? x[kt * 4 + i] : -INFINITY;
          }
        }
        float mx;
        if constexpr (PAGE16 || !Q8) {
          mx = pa_max(pa_max(pa_max(x[0], x[1]), pa_max(x[2], x[3])) * f[0],
                      pa_max(pa_max(x[4], x[5]), pa_max(x[6], x[7])) * f[1]);
        } else {
          mx = x[0] * f[0];
#pragma unroll
          for (int i = 1; i < 8; ++i) mx = pa_max(mx, x[i] * f[i]);
        }
        if (__builtin_amdgcn_ballot_w64(mx > m_run[rt] + kPaLazyLog2) != 0) {
          const float top = groups_max(mx);
          const bool grow = top > m_run[rt] + kPaLazyLog2;  // (a row's results do not depend on its neighbours)
          const float m_new = grow ? top : m_run[rt];
          const float alpha = grow ? __builtin_amdgcn_exp2f(m_run[rt] - m_new) : 1.f;
          l_run[rt] *= alpha;
#pragma unroll
          for (int t = 0; t < DT; ++t) o[rt][t] *= alpha;
          m_run[rt] = m_new;
        }
        const float m = m_run[rt] == -INFINITY ? 0.f : m_run[rt];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          float e[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[kt * 4 + i], f[PAGE16 || !Q8 ? kt : kt * 4 + i], -m));
            l_run[rt] += e[i];
            if constexpr (Q8) e[i] *= vsk[kt][PAGE16 ? 0 : i] * vinv;
          }
          pf[rt][kt * 2] = C::pack(e[0], e[1]);
          pf[rt][kt * 2 + 1] = C::pack(e[2], e[3]);
        }
      }
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) o[rt][t] = C::mfma(vf[t], pf[rt], o[rt][t]);
      __builtin_amdgcn_s_setprio(0);
      if (masked && strange) {
        // Where a row sees an infinity or NaN, its sum becomes one: a product with the
        // marks is zero for the rows that do not.
        constexpr uint32_t kOne = C::kBf16 ? 0x3f80u : 0x3c00u;
        constexpr float kHuge = 3e38f;
#pragma unroll
        for (int t = 0; t < DT; ++t) {
          frag up = frag{0, 0, 0, 0}, dn = up;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int byte = (32 * hh + 16 * (j >> 2) + 4 * g + (j & 3)) * (D / 8) + 2 * t + (r16 >> 3);
            up[j >> 1] |= ((uint32_t(up_lds[st][byte]) >> (r16 & 7)) & 1u) * (kOne << (16 * (j & 1)));
            dn[j >> 1] |= ((uint32_t(dn_lds[st][byte]) >> (r16 & 7)) & 1u) * (kOne << (16 * (j & 1)));
          }
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            const f32x4 zero = f32x4{0.f, 0.f, 0.f, 0.f};
            const f32x4 plus = C::mfma(up, pf[rt], zero), minus = C::mfma(dn, pf[rt], zero);
            o[rt][t] += plus * kHuge * kHuge - minus * kHuge * kHuge;
          }
        }
      }
    }
  };

  const int c0 = split * k.per * SUB, c1 = min(k.chunks, (split + 1) * k.per) * SUB;
  if (c0 < c1) {
    if (tid < 2) strange_lds[tid] = 0;
    // Ahead of the tile that is computed: one in LDS, SETS in registers.
    Raw x[SETS];
    auto ask = [&](Raw& y, int c) __attribute__((always_inline)) {
      if (c >= c1) return;
      if constexpr (PAGE16) {
        if (c >= win1) open_window(c, c1);
      }
      load(y, c);
    };
    if constexpr (PAGE16) open_window(c0, c1);
    load(x[0], c0);
    lds_barrier();  // (the marks are cleared)
    store(x[0], Stage<0>{}, c0);
#pragma unroll
    for (int i = 1; i <= SETS; ++i) ask(x[i % SETS], c0 + i);
    lds_barrier();
    auto step = [&](auto masked_tag, auto st_tag, Raw& y, int c) __attribute__((always_inline)) {
      // the next tile's registers go to the other stage, which every wave left
      // before the last barrier; then the one SETS behind it is asked for
      if (c + 1 < c1) store(y, Stage<1 - decltype(st_tag)::value>{}, c + 1);
      ask(y, c + 1 + SETS);
      if (computes) compute(masked_tag, st_tag, c);
      lds_barrier();
    };
    // Runs of tiles without hidden keys take the shorter form.  (A choice at every tile
    // would keep both forms' registers alive.)  Stages and sets alternate, so tiles come in
    // pairs and their addresses are constants.
    auto masked_pair = [&](int c) { return masked_tile(key_of(c)) || (c + 1 < c1 && masked_tile(key_of(c + 1))); };
    int c = c0;
    while (c < c1) {
      for (; c < c1 && masked_pair(c); c += 2) {
        step(std::true_type{}, Stage<0>{}, x[SETS - 1], c);
        if (c + 1 < c1) step(std::true_type{}, Stage<1>{}, x[0], c + 1);
      }
      for (; c < c1 && !masked_pair(c); c += 2) {
        step(std::false_type{}, Stage<0>{}, x[SETS - 1], c);
        if (c + 1 < c1) step(std::false_type{}, Stage<1>{}, x[0], c + 1);
      }
    }
  }

  // ---- results ----
  const int64_t item = (int64_t(b) * p.num_kv_heads + h) * p.row_blocks + rb;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int lr = (wave + kRowWaves * rt) * 16 + r16;
    const float sum = groups_sum(l_run[rt]);
    if (lr >= rows) continue;
    const float inv = (sum == 0.f ? 0.f : 1.f / sum) * (Q8 ? vref : 1.f);
    const float lse2 = sum == 0.f ? -INFINITY : m_run[rt] + __builtin_log2f(sum);
    if (k.splits > 1) {
      float* ws = static_cast<float*>(p.workspace);
      const int64_t prow = (item * p.num_splits + split) * p.block_rows + lr;
      const int64_t nrows = int64_t(p.batch) * p.num_kv_heads * p.row_blocks * p.num_splits * p.block_rows;
#pragma unroll
      for (int t = 0; t < DT; ++t) *reinterpret_cast<f32x4*>(ws + prow * D + t * 16 + 4 * g) = o[rt][t] * inv;
      if (g == 0) ws[nrows * D + prow] = lse2;
    } else {
      const int head = h * a.group + (row_start + lr - node_of[rt] * a.group);
      char* out = static_cast<char*>(p.out) + (int64_t(r.q0 + node_of[rt]) * p.out_stride_token +
                                               int64_t(head) * p.out_stride_head) * 2;
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        const f32x4 x = o[rt][t] * inv;
        *reinterpret_cast<w2*>(out + (t * 16 + 4 * g) * 2) =
            bf16 ? w2{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])} : w2{pack_f16(x[0], x[1]), pack_f16(x[2], x[3])};
      }
      if (p.lse != nullptr && g == 0)
        p.lse[int64_t(r.q0 + node_of[rt]) * p.num_qo_heads + head] = lse2 * kPaLn2;
    }
  }
}

}  // namespace
}  // namespace atlas

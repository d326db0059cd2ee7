// Paged attention for few packed rows: one query token per request, or several
// with up to 16 * RT rows a block.
//
// The time goes into reading the cache once.  Four waves take contiguous parts of the
// split, each for all rows, and work alone until their states are joined: K and V go
// from HBM to registers and from there into the matrix instructions, with no LDS for
// them and no barrier in the key loop.  K's operand wants eight dims of one key per
// lane, in any order that Q shares: a lane loads 16 bytes of a key's row and that is one
// operand (16-bit) or two (8-bit).  V's operand wants eight keys of one dim per lane.
// Which dims a lane's row of the tile stands for is free, so lane c of 16 owns the dims
// c * D/16 .., loads that piece of the rows of its keys, and byte permutes put pairs of
// keys together.
//
// One token: bound by HBM, 98 us for 497 MB (5.1 TB/s) over 32 requests of up to 16384 keys
// in e4m3; 52 us for 226 MB (4.3 TB/s) over 24 capped requests in bf16 at head_dim 64.  A CU
// takes in about 50 bytes a ns however many of its waves ask, so few requests want their
// keys on more CUs: 1024 bf16 keys of 8 heads take 14.0 us whole and 10.1 in six splits.
// Eight waves a workgroup were 2 % slower there and 20 % where requests are many (their
// starts and ends overlap less).  Several rows: 30 us for a tree of 36 nodes over 16384 keys
// (144 rows, three blocks), 1.6 to 2.5 us a step of 32 keys, bound by the conversions,
// permutes and softmax of one wave a SIMD in turn with its matrix instructions; eight waves
// did not help there either (34.7 against 34.0 us with the join).
#pragma once

#include "paged_attn.hpp"

namespace atlas {
namespace {

template <int BYTES>
__device__ __forceinline__ void load_words(const char* p, uint32_t* out) {
  if constexpr (BYTES == 16) {
    const w4 v = *reinterpret_cast<const w4*>(p);
    out[0] = v[0];
    out[1] = v[1];
    out[2] = v[2];
    out[3] = v[3];
  } else if constexpr (BYTES == 8) {
    const w2 v = *reinterpret_cast<const w2*>(p);
    out[0] = v[0];
    out[1] = v[1];
  } else {
    out[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// KIND: what the cache holds.  D: head_dim.  RT: row tiles of 16 in a block.  PAGE16:
// page_size is a multiple of 16, so a 16-key tile lies in one page and its id and
// scales are wave-uniform; other page sizes look every key up.  SCORED: scores may be
// capped or biased.  MULTI: several query tokens per request (their masks differ).
template <int KIND, int D, int RT, bool PAGE16, bool SCORED, bool MULTI>
__global__ __launch_bounds__(kPaThreads, 2) void paged_stream_kernel(PagedAttnArgs a) {
  typedef Cache<KIND> C;
  typedef typename C::frag frag;
  static_assert(MULTI || RT == 1, "one token has one row tile a block");
  constexpr bool Q8 = C::kQuant;
  constexpr int KT = D == 128 ? 2 : 4;    // 16-key tiles of a step
  constexpr int CK = KT * 16;             // keys of a step
  constexpr int SUB = kChunk / CK;        // steps of a chunk
  constexpr int KS = D / 32;              // steps of the score product
  constexpr int KL = D * C::kBytes / 64;  // 16-byte loads of a lane per key row
  constexpr int DL = D / 16;              // dims of V a lane owns
  constexpr int VB = DL * C::kBytes;      // their bytes
  constexpr int VW = VB / 4;
  constexpr int OS = D + 4;               // LDS row stride (floats)
  constexpr int NS = PAGE16 ? KT : KT * 4;  // scales of a step: by tile or by key
  constexpr bool QLDS = RT > 1;           // more than one tile of queries stays in LDS
  const atlas_paged_attn_t& p = a.p;

  __shared__ __attribute__((aligned(16))) float o_lds[kPaWaves][16 * OS];
  __shared__ float ml_lds[kPaWaves][16][2];
  __shared__ __attribute__((aligned(16))) frag q_lds[QLDS ? RT * KS * 64 : 1];
  __shared__ float qscale_lds[QLDS ? RT * 16 : 1];

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
  unit /= p.num_kv_heads;
  const int split = unit % p.num_splits;
  const int b = unit / p.num_splits;
  if (b >= p.batch) return;
  const Request r = read_request(p, b);
  const int row_start = rb * p.block_rows;
  const int rows = block_of(a, r, row_start);
  if (rows <= 0) return;
  const Block k = plan_block(a, r, b, row_start, rows);
  if (split >= k.splits) return;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, r16 = lane & 15;
  const bool bf16 = p.dtype == ATLAS_DTYPE_BF16;
  const int shift = r.kv_len - r.q_len;  // position of query token 0
  const int col0 = MULTI && p.mask_mode == 1 ? p.mask_col_start[b] : 0;

  // ---- queries ----
  // The operands of row tile rt; returns 2^e of the lane's row.
  auto read_q = [&](int rt, frag (&out)[KS]) __attribute__((always_inline)) {
    const bool ok = rt * 16 + r16 < rows;
    const int prow = row_start + (ok ? rt * 16 + r16 : 0);
    const int node = MULTI ? prow / a.group : 0;
    const char* qrow = static_cast<const char*>(p.q) + (int64_t(r.q0 + node) * p.q_stride_token +
                                                        int64_t(h * a.group + prow - node * a.group) * p.q_stride_head) * 2;
    // (8-bit: step 2j + e of group g holds dims 64 j + 16 g + 8 e ..: those of its 16 codes)
    float f[KS][8];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      w4 v = *reinterpret_cast<const w4*>(qrow + (Q8 ? (ks >> 1) * 64 + g * 16 + (ks & 1) * 8 : ks * 32 + g * 8) * 2);
      if (!ok) v = w4{0, 0, 0, 0};
      if constexpr (Q8) q_floats(v, bf16, f[ks]);
      else out[ks] = v;
    }
    if constexpr (Q8) return q_to_f16<KS>(f, out);
    else return 1.f;
  };
  frag qf[KS];
  float qscale[RT], m_run[RT], l_run[RT], slope[RT];
  int qpos[RT];
  if constexpr (QLDS) {
    static_assert(RT <= kPaWaves, "a wave reads at most one tile of queries");
    if (wave < RT) {
      const float s = read_q(wave, qf);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) q_lds[(wave * KS + ks) * 64 + lane] = qf[ks];
      if (g == 0) qscale_lds[wave * 16 + r16] = s;
    }
    __syncthreads();
  } else {
    qscale[0] = a.scale_log2 * read_q(0, qf);
  }
  f32x4 o[RT][DL];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    if constexpr (QLDS) qscale[rt] = a.scale_log2 * qscale_lds[rt * 16 + r16];
    const int prow = row_start + (rt * 16 + r16 < rows ? rt * 16 + r16 : 0);
    const int node = MULTI ? prow / a.group : 0;
    qpos[rt] = shift + node;
    slope[rt] = SCORED && p.alibi_slopes ? p.alibi_slopes[h * a.group + prow - node * a.group] * kPaLog2e : 0.f;
    m_run[rt] = -INFINITY;
    l_run[rt] = 0.f;
#pragma unroll
    for (int t = 0; t < DL; ++t) o[rt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // Steps that hide no key from any row end by plain_hi and start at plain_lo, or end
  // by the prefix.
  const int plain_hi = p.mask_mode == 2 ? shift + k.n0 + 1 : (MULTI && p.mask_mode == 1 ? min(r.kv_len, col0) : r.kv_len);
  const int plain_lo = p.mask_mode == 2 && p.window_left >= 0 ? shift + k.n1 - p.window_left : 0;

  // ---- this wave's steps ----
  const int chunk0 = split * k.per;
  const int steps = (min(k.chunks, chunk0 + k.per) - chunk0) * SUB;
  const int mine = (steps + kPaWaves - 1) / kPaWaves;
  const int s0 = chunk0 * SUB + wave * mine;
  const int s1 = min(chunk0 * SUB + steps, s0 + mine);

  const char* kbase = static_cast<const char*>(p.kv) + int64_t(h) * p.head_stride;
  const char* vbase = kbase + p.v_offset;
  const int ts = int(p.token_stride);
  const int page_size = p.page_size;
  Pages pages;
  pages.begin(a, r);

  struct RawK {
    uint32_t k[KT][KL * 4];
    float ks[NS], vs[NS];
  };
  struct RawV {
    uint32_t v[KT][4][VW];
  };
  // first key of step s
  auto key_of = [&](int s) __attribute__((always_inline)) {
    const int c = s / SUB;
    return (c < k.ca ? c : c - k.ca + k.cb) * kChunk + (s % SUB) * CK;
  };
  auto bounds = [&](int s, int& lo, int& hi) __attribute__((always_inline)) {
    const bool first = s < k.ca * SUB;
    lo = first ? 0 : k.lo;
    hi = (first ? k.prefix : k.hi) - 1;
  };
  // Up to 64 / KT steps make a window: lane l holds the offset of the first row of
  // tile l % KT of its step l / KT, and that page's scales, read together before the
  // window's first step.
  constexpr int WIN = 64 / KT;
  int64_t win_rows = 0;
  float win_ks = 0.f, win_vs = 0.f;
  int win0 = 0;
  auto open_window = [&](int s, int end) __attribute__((always_inline)) {
    win0 = s;
    const int mine = min(s + lane / KT, end - 1);
    int lo, hi;
    bounds(mine, lo, hi);
    const int tile = Pages::tile_key(key_of(mine), lane & (KT - 1), lo, hi);
    const int id = pages.read_id(a, tile);
    win_rows = pages.row_offset(a, id, tile);
    if constexpr (Q8) {
      const float* sc = p.kv_scales + int64_t(h) * p.scale_stride_head + pages.valid(id) * p.scale_stride_page;
      win_ks = sc[0];
      win_vs = sc[p.scale_stride_kv];
    }
  };
  // lane offsets of a tile's rows
  const uint32_t k_lane = uint32_t(r16 * ts + g * 16), v_lane = uint32_t(4 * g * ts + r16 * VB);
  // Keys outside [lo, hi) of the step's part repeat its nearest key, so that
  // every load falls on a row that is there.
  auto load_k = [&](RawK& x, int s) __attribute__((always_inline)) {
    const int kb = key_of(s);
    int lo, hi;
    bounds(s, lo, hi);
    const bool whole = (kb >= lo) & (kb + CK <= hi + 1);
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const int t0 = kb + kt * 16;
      if constexpr (PAGE16) {
        const char* kp = kbase + Pages::tile_row(win_rows, (s - win0) * KT + kt);
        uint32_t ko = k_lane;
        if (!whole) ko = uint32_t((min(max(t0 + r16, lo), hi) - Pages::tile_key(kb, kt, lo, hi)) * ts + g * 16);
#pragma unroll
        for (int j = 0; j < KL; ++j) load_words<16>(kp + (ko + j * 64), &x.k[kt][4 * j]);
        if constexpr (Q8) {
          x.ks[kt] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(win_ks), (s - win0) * KT + kt));
          x.vs[kt] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(win_vs), (s - win0) * KT + kt));
        }
      } else {
        const int key = min(max(t0 + r16, lo), hi);
        const int slot = slot_of(a, key);
        const char* kp = kbase + pages.valid(pages.ids[slot]) * p.page_stride + int64_t(key - slot * page_size) * ts;
#pragma unroll
        for (int j = 0; j < KL; ++j) load_words<16>(kp + j * 64 + g * 16, &x.k[kt][4 * j]);
        if constexpr (Q8) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int64_t page = pages.valid(pages.ids[slot_of(a, min(max(t0 + 4 * g + i, lo), hi))]);
            const float* sc = p.kv_scales + int64_t(h) * p.scale_stride_head + page * p.scale_stride_page;
            x.ks[kt * 4 + i] = sc[0];
            x.vs[kt * 4 + i] = sc[p.scale_stride_kv];
          }
        }
      }
    }
  };
  auto load_v = [&](RawV& x, int s) __attribute__((always_inline)) {
    const int kb = key_of(s);
    int lo, hi;
    bounds(s, lo, hi);
    const bool whole = (kb >= lo) & (kb + CK <= hi + 1);
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const int t0 = kb + kt * 16;
      if constexpr (PAGE16) {
        const char* vp = vbase + Pages::tile_row(win_rows, (s - win0) * KT + kt);
        uint32_t vo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) vo[i] = v_lane + uint32_t(i * ts);
        if (!whole) {
          const int tile = Pages::tile_key(kb, kt, lo, hi);
#pragma unroll
          for (int i = 0; i < 4; ++i) vo[i] = uint32_t((min(max(t0 + 4 * g + i, lo), hi) - tile) * ts + r16 * VB);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) load_words<VB>(vp + vo[i], x.v[kt][i]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = min(max(t0 + 4 * g + i, lo), hi);
          const int slot = slot_of(a, key);
          load_words<VB>(vbase + pages.valid(pages.ids[slot]) * p.page_stride + int64_t(key - slot * page_size) * ts + r16 * VB,
                         x.v[kt][i]);
        }
      }
    }
  };

  // Largest V scale so far: O holds sums of p * v * (scale / vref).
  float vref = 1.17549435e-38f, vinv = 8.5070592e37f;

  auto masked_step = [&](int s) __attribute__((always_inline)) {
    const int kb = key_of(s);
    return ((kb + CK > plain_hi) | (kb < plain_lo)) & (kb + CK > k.prefix);
  };
  f32x4 acc[RT][KT];
  auto scores = [&](const RawK& x) __attribute__((always_inline)) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) acc[rt][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      frag kf[KT];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        if constexpr (Q8) kf[kt] = C::keys8(x.k[kt][2 * ks], x.k[kt][2 * ks + 1]);
        else kf[kt] = frag{x.k[kt][4 * ks], x.k[kt][4 * ks + 1], x.k[kt][4 * ks + 2], x.k[kt][4 * ks + 3]};
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const frag q = QLDS ? q_lds[(rt * KS + ks) * 64 + lane] : qf[ks];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) acc[rt][kt] = C::mfma(kf[kt], q, acc[rt][kt]);
      }
    }
  };
  // The softmax's part: weights pf of the step's scores (ks, vs: its scales).
  frag pf[RT][KT / 2];
  auto weights = [&](auto masked_tag, int s, const float (&ks_of)[NS], const float (&vs_of)[NS]) __attribute__((always_inline)) {
    constexpr bool masked = decltype(masked_tag)::value;
    const int kb = key_of(s);
    if constexpr (Q8) {
      float top = vs_of[0];
#pragma unroll
      for (int i = 1; i < NS; ++i) top = pa_max(top, vs_of[i]);
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
    const int key0 = kb + 4 * g;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float sc[KT * 4];
#pragma unroll
      for (int i = 0; i < KT * 4; ++i)
        sc[i] = acc[rt][i >> 2][i & 3] * (Q8 ? qscale[rt] * ks_of[PAGE16 ? i >> 2 : i] : qscale[rt]);
      if (SCORED && p.soft_cap > 0.f) {
        // cap * tanh(y / cap) = cap * (1 - 2 / (1 + e^(2 y / cap))), to powers of two
#pragma unroll
        for (int i = 0; i < KT * 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(sc[i] * a.cap_in);
          sc[i] = __builtin_fmaf(-2.f * a.cap_out, __builtin_amdgcn_rcpf(1.f + e), a.cap_out);
        }
      }
      if (SCORED && p.alibi_slopes != nullptr) {
        const float away = float(qpos[rt] - key0);
#pragma unroll
        for (int i = 0; i < KT * 4; ++i)
          sc[i] = __builtin_fmaf(-slope[rt], fabsf(away - float((i >> 2) * 16 + (i & 3))), sc[i]);
      }
      if constexpr (masked) {
        uint64_t w = 0;
        int w0 = col0;
        if (MULTI && p.mask_mode == 1) {
          // one word of the tree's columns, or one for each 64 keys (a step lies in one of them)
          const int idx = p.mask_words > 1 ? (kb >> 6) - (col0 >> 6) : 0;
          if (idx >= 0 && idx < p.mask_words) w = p.tree_mask[int64_t(r.q0 + qpos[rt] - shift) * p.mask_words + idx];
          if (idx < 0) w = ~0ull;
          if (p.mask_words > 1) w0 = kb & ~63;
        }
        const int wlo = p.window_left >= 0 ? qpos[rt] - p.window_left : 0;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          const int at = key0 + kt * 16;
          uint32_t vis = below4(at, r.kv_len);
          if (p.mask_mode == 2) {
            vis &= (below4(at, qpos[rt] + 1) & ~below4(at, wlo)) | below4(at, k.prefix);
          } else if (MULTI && p.mask_mode == 1) {
            vis &= tree4(w, at - w0);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[kt * 4 + i] = (vis >> i) & 1u ? sc[kt * 4 + i] : -INFINITY;
        }
      }
      float mx = sc[0];
#pragma unroll
      for (int i = 1; i < KT * 4; ++i) mx = pa_max(mx, sc[i]);
      if (__builtin_amdgcn_ballot_w64(mx > m_run[rt] + kPaLazyLog2) != 0) {
        const float top = groups_max(mx);
        const bool grow = top > m_run[rt] + kPaLazyLog2;  // (a row's results do not depend on its neighbours)
        const float m_new = grow ? top : m_run[rt];
        const float alpha = grow ? __builtin_amdgcn_exp2f(m_run[rt] - m_new) : 1.f;
        l_run[rt] *= alpha;
#pragma unroll
        for (int t = 0; t < DL; ++t) o[rt][t] *= alpha;
        m_run[rt] = m_new;
      }
      const float m = m_run[rt] == -INFINITY ? 0.f : m_run[rt];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[i] = __builtin_amdgcn_exp2f(sc[kt * 4 + i] - m);
          l_run[rt] += e[i];
          if constexpr (Q8) e[i] *= vs_of[PAGE16 ? kt : kt * 4 + i] * vinv;
        }
        pf[rt][kt >> 1][(kt & 1) * 2] = C::pack(e[0], e[1]);
        pf[rt][kt >> 1][(kt & 1) * 2 + 1] = C::pack(e[2], e[3]);
      }
    }
  };
  auto values = [&](auto masked_tag, const RawV& x) __attribute__((always_inline)) {
    constexpr bool masked = decltype(masked_tag)::value;
#pragma unroll
    for (int tp = 0; tp < KT / 2; ++tp)
      // (a word of each row at a time: its dims' operands are all that is alive)
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        constexpr int DW = DL / VW;
        uint32_t raw[8][1];
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[i][0] = x.v[2 * tp + (i >> 2)][i & 3][w];
        frag vf[DW];
        transpose_v<KIND, 1, DW>(raw, vf);
        if constexpr (MULTI && masked && KIND != kCacheInt8) {
          // Infinities and NaN in V rows that a row does not see must not reach it
          // (0 * inf): where keys are hidden they are taken out of the product, and the
          // rows that see them get them from a product with their marks.
          uint32_t odd = 0;
#pragma unroll
          for (int t = 0; t < DW; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) odd |= not_finite2<C::kBf16>(vf[t][j]);
          if (__builtin_amdgcn_ballot_w64(odd != 0) != 0) {
            constexpr uint32_t kOne = C::kBf16 ? 0x3f80u : 0x3c00u;
            constexpr float kHuge = 3e38f;
#pragma unroll
            for (int t = 0; t < DW; ++t) {
              frag up, dn;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                uint32_t u, d;
                vf[t][j] = take_out2<C::kBf16>(vf[t][j], u, d);
                up[j] = (u >> 15) * kOne;
                dn[j] = (d >> 15) * kOne;
              }
#pragma unroll
              for (int rt = 0; rt < RT; ++rt) {
                const f32x4 zero = f32x4{0.f, 0.f, 0.f, 0.f};
                const f32x4 plus = C::mfma(up, pf[rt][tp], zero), minus = C::mfma(dn, pf[rt][tp], zero);
                o[rt][w * DW + t] += plus * kHuge * kHuge - minus * kHuge * kHuge;
              }
            }
          }
        }
#pragma unroll
        for (int t = 0; t < DW; ++t)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) o[rt][w * DW + t] = C::mfma(vf[t], pf[rt][tp], o[rt][w * DW + t]);
      }
  };

  for (int s = s0; s < s1;) {
    const int end = PAGE16 ? min(s1, s + WIN) : s1;
    if constexpr (PAGE16) open_window(s, end);
    auto at = [&](int t) { return min(t, end - 1); };
    if constexpr (RT == 1) {
      // One step is in flight while another is computed; past the window's last step it
      // is asked for again rather than branched around, so the waits stay exact.
      RawK xk[2];
      RawV xv[2];
      load_k(xk[0], s);
      load_v(xv[0], s);
      auto step = [&](int cur) __attribute__((always_inline)) {
        load_k(xk[1 - cur], at(s + 1));
        load_v(xv[1 - cur], at(s + 1));
        scores(xk[cur]);
        if (masked_step(s)) {
          weights(std::true_type{}, s, xk[cur].ks, xk[cur].vs);
          values(std::true_type{}, xv[cur]);
        } else {
          weights(std::false_type{}, s, xk[cur].ks, xk[cur].vs);
          values(std::false_type{}, xv[cur]);
        }
        return ++s < end;
      };
      while (step(0) && step(1)) {
      }
    } else {
      // The rows of O leave room for one step: the next step's K is asked for when the
      // scores are done with this one's, its V when the second product is.
      RawK xk;
      RawV xv;
      load_k(xk, s);
      load_v(xv, s);
      auto step = [&](auto masked_tag) __attribute__((always_inline)) {
        scores(xk);
        float ks_of[NS], vs_of[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) {
          ks_of[i] = xk.ks[i];
          vs_of[i] = xk.vs[i];
        }
        load_k(xk, at(s + 1));
        weights(masked_tag, s, ks_of, vs_of);
        values(masked_tag, xv);
        load_v(xv, at(s + 1));
        ++s;
      };
      while (s < end) {
        while (s < end && masked_step(s)) step(std::true_type{});
        while (s < end && !masked_step(s)) step(std::false_type{});
      }
    }
  }

  // ---- the waves' states into one ----
  const int row = tid >> 4, d0 = (tid & 15) * DL;
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
    const int lr = rt * 16 + row;
    if (lr >= rows) continue;
    float m = ml_lds[0][row][0];
#pragma unroll
    for (int w = 1; w < kPaWaves; ++w) m = fmaxf(m, ml_lds[w][row][0]);
    float sum = 0.f, acc[DL];
#pragma unroll
    for (int t = 0; t < DL; ++t) acc[t] = 0.f;
#pragma unroll
    for (int w = 0; w < kPaWaves; ++w) {
      const float mw = ml_lds[w][row][0];
      if (mw == -INFINITY && ml_lds[w][row][1] == 0.f) continue;  // (no key; a NaN score leaves a sum)
      const float f = __builtin_amdgcn_exp2f(mw - m);
      sum += f * ml_lds[w][row][1];
#pragma unroll
      for (int t = 0; t < DL; ++t) acc[t] += f * o_lds[w][row * OS + d0 + t];
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const float lse2 = sum == 0.f ? -INFINITY : m + __builtin_log2f(sum);
    if (k.splits > 1) {
      const int64_t item = (int64_t(b) * p.num_kv_heads + h) * p.row_blocks + rb;
      float* ws = static_cast<float*>(p.workspace);
      const int64_t prow = (item * p.num_splits + split) * p.block_rows + lr;
      const int64_t nrows = int64_t(p.batch) * p.num_kv_heads * p.row_blocks * p.num_splits * p.block_rows;
#pragma unroll
      for (int t = 0; t < DL; t += 4)
        *reinterpret_cast<f32x4*>(ws + prow * D + d0 + t) =
            f32x4{acc[t] * inv, acc[t + 1] * inv, acc[t + 2] * inv, acc[t + 3] * inv};
      if ((tid & 15) == 0) ws[nrows * D + prow] = lse2;
    } else {
      const int prow = row_start + lr, node = MULTI ? prow / a.group : 0;
      const int hd = h * a.group + prow - node * a.group;
      char* out = static_cast<char*>(p.out) +
                  (int64_t(r.q0 + node) * p.out_stride_token + int64_t(hd) * p.out_stride_head + d0) * 2;
      uint32_t packed[DL / 2];
#pragma unroll
      for (int t = 0; t < DL / 2; ++t)
        packed[t] = bf16 ? pack_bf16(acc[2 * t] * inv, acc[2 * t + 1] * inv)
                         : pack_f16(acc[2 * t] * inv, acc[2 * t + 1] * inv);
      if constexpr (DL == 8) *reinterpret_cast<w4*>(out) = w4{packed[0], packed[1], packed[2], packed[3]};
      else *reinterpret_cast<w2*>(out) = w2{packed[0], packed[1]};
      if (p.lse != nullptr && (tid & 15) == 0) p.lse[int64_t(r.q0 + node) * p.num_qo_heads + hd] = lse2 * kPaLn2;
    }
  }
}

}  // namespace
}  // namespace atlas

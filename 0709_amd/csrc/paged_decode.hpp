// Paged attention for one query token per request: up to 16 packed rows (the heads
// of a KV head's group) against one split of the request's keys.
//
// The time goes into reading the cache once.  Four waves take contiguous parts of the
// split and work alone until their states are joined: K and V go from HBM to
// registers and from there into the matrix instructions, with no LDS and no barrier in
// the key loop.  K's operand wants eight dims of one key per lane, in any order that Q
// shares: a lane loads 16 bytes of a key's row and that is one operand (16-bit) or
// two (8-bit).  V's operand wants eight keys of one dim per lane.  Which dims a lane's
// row of the tile stands for is free, so lane c of 16 owns the dims c * D/16 ..,
// loads that piece of the rows of its keys, and byte permutes put pairs of keys
// together.
#pragma once

#include "paged_attn.hpp"

namespace atlas {
namespace {

template <int NB>
__device__ __forceinline__ void load_words(const char* p, uint32_t* out) {
  if constexpr (NB == 16) {
    const w4 v = __builtin_nontemporal_load(reinterpret_cast<const w4*>(p));
    out[0] = v[0];
    out[1] = v[1];
    out[2] = v[2];
    out[3] = v[3];
  } else if constexpr (NB == 8) {
    const w2 v = __builtin_nontemporal_load(reinterpret_cast<const w2*>(p));
    out[0] = v[0];
    out[1] = v[1];
  } else {
    out[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
  }
}

// KIND: what the cache holds.  D: head_dim.  PAGE16: page_size is a multiple of 16,
// so a 16-key tile lies in one page and its id and scales are wave-uniform;
// other page sizes look every key up.  SCORED: scores may be capped or biased.
template <int KIND, int D, bool PAGE16, bool SCORED>
__global__ __launch_bounds__(kPaThreads, 2) void paged_decode_kernel(PagedAttnArgs a) {
  typedef Cache<KIND> C;
  typedef typename C::frag frag;
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
  const atlas_paged_attn_t& p = a.p;

  __shared__ __attribute__((aligned(16))) float o_lds[kPaWaves][16 * OS];
  __shared__ float ml_lds[kPaWaves][16][2];

  int unit = blockIdx.x;
  const int rb = unit % p.row_blocks;
  unit /= p.row_blocks;
  const int h = unit % p.num_kv_heads;
  unit /= p.num_kv_heads;
  const int split = unit % p.num_splits;
  const int b = unit / p.num_splits;
  Request r = read_request(p, b);
  r.q_len = min(r.q_len, 1);
  const int row_start = rb * 16;
  const int rows = min(16, r.q_len * a.group - row_start);
  if (rows <= 0) return;
  const Block k = plan_block(a, r, b, row_start, rows);
  if (split >= k.splits) return;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, r16 = lane & 15;
  const bool bf16 = p.dtype == ATLAS_DTYPE_BF16;
  const bool ok = r16 < rows;
  const int head = h * a.group + row_start + (ok ? r16 : 0);
  const int qpos = r.kv_len - 1;
  // keys below it are hidden unless they belong to the prefix
  const int wlo = p.mask_mode == 2 && p.window_left >= 0 ? qpos - p.window_left : 0;

  // ---- query ----
  frag qf[KS];
  float qscale = a.scale_log2;
  {
    const char* qrow = static_cast<const char*>(p.q) + (int64_t(r.q0) * p.q_stride_token + int64_t(head) * p.q_stride_head) * 2;
    if constexpr (!Q8) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        qf[ks] = *reinterpret_cast<const frag*>(qrow + (ks * 32 + g * 8) * 2);
        if (!ok) qf[ks] = frag{0, 0, 0, 0};
      }
    } else {
      // step 2j + e of group g holds dims 64 j + 16 g + 8 e ..: those of its 16 codes
      float f[KS][8];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        w4 v = *reinterpret_cast<const w4*>(qrow + ((ks >> 1) * 64 + g * 16 + (ks & 1) * 8) * 2);
        if (!ok) v = w4{0, 0, 0, 0};
        q_floats(v, bf16, f[ks]);
      }
      qscale *= q_to_f16<KS>(f, qf);
    }
  }
  const float slope = SCORED && p.alibi_slopes ? p.alibi_slopes[head] * kPaLog2e : 0.f;
  float m_run = -INFINITY, l_run = 0.f;
  f32x4 o[DL];
#pragma unroll
  for (int t = 0; t < DL; ++t) o[t] = f32x4{0.f, 0.f, 0.f, 0.f};

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
  TilePages<Q8, KT> pages;
  pages.begin(a, r, h, lane);

  struct Raw {
    uint32_t k[KT][KL * 4];
    uint32_t v[KT][4][VW];
    float ks[NS], vs[NS];
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
  typedef TilePages<Q8, KT> Tiles;
  // first key of the lane's tile of step s
  auto lane_tile = [&](int s) __attribute__((always_inline)) {
    int lo, hi;
    bounds(s, lo, hi);
    return Tiles::tile_key(key_of(s), lane & (KT - 1), lo, hi);
  };
  // lane offsets of a tile's rows
  const uint32_t k_lane = uint32_t(r16 * ts + g * 16), v_lane = uint32_t(4 * g * ts + r16 * VB);
  // Keys outside [lo, hi) of the step's part repeat its nearest key, so that
  // every load falls on a row that is there.
  auto load = [&](Raw& x, int s, int64_t rows_at, float scale) __attribute__((always_inline)) {
    const int kb = key_of(s);
    int lo, hi;
    bounds(s, lo, hi);
    if constexpr (PAGE16) {
      const bool whole = kb >= lo && kb + CK <= hi + 1;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        // the tile's first row; then lane offsets from it
        const int64_t row0 = Tiles::tile_row(rows_at, kt);
        const char* kp = kbase + row0;
        const char* vp = vbase + row0;
        uint32_t ko = k_lane, vo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) vo[i] = v_lane + uint32_t(i * ts);
        if (!whole) {
          const int t0 = kb + kt * 16, tile = Tiles::tile_key(kb, kt, lo, hi);
          ko = uint32_t((min(max(t0 + r16, lo), hi) - tile) * ts + g * 16);
#pragma unroll
          for (int i = 0; i < 4; ++i) vo[i] = uint32_t((min(max(t0 + 4 * g + i, lo), hi) - tile) * ts + r16 * VB);
        }
#pragma unroll
        for (int j = 0; j < KL; ++j) load_words<16>(kp + (ko + j * 64), &x.k[kt][4 * j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) load_words<VB>(vp + vo[i], x.v[kt][i]);
        if constexpr (Q8) {
          x.ks[kt] = Tiles::tile_scale(scale, 0, kt);
          x.vs[kt] = Tiles::tile_scale(scale, 1, kt);
        }
      }
    } else {
      auto page_of = [&](int slot) __attribute__((always_inline)) { return pages.valid(pages.ids[slot]); };
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        const int t0 = kb + kt * 16;
        const int key = min(max(t0 + r16, lo), hi);
        const int slot = slot_of(a, key);
        const char* kp = kbase + page_of(slot) * p.page_stride + int64_t(key - slot * page_size) * ts;
#pragma unroll
        for (int j = 0; j < KL; ++j) load_words<16>(kp + j * 64 + g * 16, &x.k[kt][4 * j]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int vk = min(max(t0 + 4 * g + i, lo), hi);
          const int vslot = slot_of(a, vk);
          const int64_t page = page_of(vslot);
          load_words<VB>(vbase + page * p.page_stride + int64_t(vk - vslot * page_size) * ts + r16 * VB, x.v[kt][i]);
          if constexpr (Q8) {
            const float* sc = p.kv_scales + int64_t(h) * p.scale_stride_head + page * p.scale_stride_page;
            x.ks[kt * 4 + i] = sc[0];
            x.vs[kt * 4 + i] = sc[p.scale_stride_kv];
          }
        }
      }
    }
  };

  // Largest V scale so far: O holds sums of p * v * (scale / vref).
  float vref = 1.17549435e-38f, vinv = 8.5070592e37f;

  auto compute = [&](const Raw& x, int s) __attribute__((always_inline)) {
    const int kb = key_of(s);
    f32x4 acc[KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      acc[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        frag kf;
        if constexpr (Q8) kf = C::keys8(x.k[kt][2 * ks], x.k[kt][2 * ks + 1]);
        else kf = frag{x.k[kt][4 * ks], x.k[kt][4 * ks + 1], x.k[kt][4 * ks + 2], x.k[kt][4 * ks + 3]};
        acc[kt] = C::mfma(kf, qf[ks], acc[kt]);
      }
    }
    float sc[KT * 4];
#pragma unroll
    for (int i = 0; i < KT * 4; ++i)
      sc[i] = acc[i >> 2][i & 3] * (Q8 ? qscale * x.ks[PAGE16 ? i >> 2 : i] : qscale);
    if (SCORED && p.soft_cap > 0.f) {
      // cap * tanh(y / cap) = cap * (1 - 2 / (1 + e^(2 y / cap))), to powers of two
#pragma unroll
      for (int i = 0; i < KT * 4; ++i) {
        const float e = __builtin_amdgcn_exp2f(sc[i] * a.cap_in);
        sc[i] = __builtin_fmaf(-2.f * a.cap_out, __builtin_amdgcn_rcpf(1.f + e), a.cap_out);
      }
    }
    const int key0 = kb + 4 * g;
    if (SCORED && p.alibi_slopes != nullptr) {
#pragma unroll
      for (int i = 0; i < KT * 4; ++i)
        sc[i] = __builtin_fmaf(-slope, fabsf(float(qpos - key0 - ((i >> 2) * 16 + (i & 3)))), sc[i]);
    }
    if (kb + CK > r.kv_len || (kb < wlo && kb + CK > k.prefix)) {
#pragma unroll
      for (int i = 0; i < KT * 4; ++i) {
        const int key = key0 + (i >> 2) * 16 + (i & 3);
        sc[i] = key <= qpos && (key >= wlo || key < k.prefix) ? sc[i] : -INFINITY;
      }
    }
    float mx = sc[0];
#pragma unroll
    for (int i = 1; i < KT * 4; ++i) mx = pa_max(mx, sc[i]);
    if (__builtin_amdgcn_ballot_w64(mx > m_run + kPaLazyLog2) != 0) {
      const float top = groups_max(mx);
      const bool grow = top > m_run + kPaLazyLog2;  // (a row's results do not depend on its neighbours)
      const float m_new = grow ? top : m_run;
      const float alpha = grow ? __builtin_amdgcn_exp2f(m_run - m_new) : 1.f;
      l_run *= alpha;
#pragma unroll
      for (int t = 0; t < DL; ++t) o[t] *= alpha;
      m_run = m_new;
    }
    if constexpr (Q8) {
      float top = x.vs[0];
#pragma unroll
      for (int i = 1; i < NS; ++i) top = fmaxf(top, x.vs[i]);
      if (__builtin_amdgcn_ballot_w64(top > vref) != 0) {
        if constexpr (!PAGE16) top = groups_max(top);
        const float now = fmaxf(vref, top);
        const float down = vref / now;
#pragma unroll
        for (int t = 0; t < DL; ++t) o[t] *= down;
        vref = now;
        vinv = 1.0f / now;
      }
    }
    const float m = m_run == -INFINITY ? 0.f : m_run;
    frag pf[KT / 2];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      float e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e[i] = __builtin_amdgcn_exp2f(sc[kt * 4 + i] - m);
        l_run += e[i];
        if constexpr (Q8) e[i] *= x.vs[PAGE16 ? kt : kt * 4 + i] * vinv;
      }
      pf[kt >> 1][(kt & 1) * 2] = C::pack(e[0], e[1]);
      pf[kt >> 1][(kt & 1) * 2 + 1] = C::pack(e[2], e[3]);
    }
#pragma unroll
    for (int tp = 0; tp < KT / 2; ++tp) {
      uint32_t raw[8][VW];
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int w = 0; w < VW; ++w) raw[i][w] = x.v[2 * tp + (i >> 2)][i & 3][w];
      frag vf[DL];
      transpose_v<KIND, VW, DL>(raw, vf);
#pragma unroll
      for (int t = 0; t < DL; ++t) o[t] = C::mfma(vf[t], pf[tp], o[t]);
    }
  };

  if (s0 < s1) {
    // The next step's rows, the scales of the one behind it and the page ids of the
    // third are in flight while a step is computed; past the last step it is asked
    // for again rather than branched around, so the waits stay exact.
    auto at = [&](int s) __attribute__((always_inline)) { return min(s, s1 - 1); };
    int64_t row0 = 0, row1 = 0;
    int id2 = 0;
    float sc0 = 0.f, sc1 = 0.f;
    if constexpr (PAGE16) {
      const int t0 = lane_tile(s0), t1 = lane_tile(at(s0 + 1));
      const int id0 = pages.read_id(a, t0), id1 = pages.read_id(a, t1);
      id2 = pages.read_id(a, lane_tile(at(s0 + 2)));
      sc0 = pages.read_scale(id0);
      row0 = pages.row_offset(a, id0, t0);
      sc1 = pages.read_scale(id1);
      row1 = pages.row_offset(a, id1, t1);
    }
    Raw x, y;
    load(x, s0, row0, sc0);
    int s = s0;
    auto step = [&](Raw& cur, Raw& next) __attribute__((always_inline)) {
      int id3 = 0;
      int64_t row2 = 0;
      float sc2 = 0.f;
      if constexpr (PAGE16) {
        id3 = pages.read_id(a, lane_tile(at(s + 3)));
        sc2 = pages.read_scale(id2);
        row2 = pages.row_offset(a, id2, lane_tile(at(s + 2)));
      }
      load(next, at(s + 1), row1, sc1);
      compute(cur, s);
      id2 = id3;
      row1 = row2;
      sc1 = sc2;
      return ++s < s1;
    };
    while (step(x, y) && step(y, x)) {
    }
  }

  // ---- the waves' states into one ----
  const float l = groups_sum(l_run);
  if (g == 0) {
    ml_lds[wave][r16][0] = m_run;
    ml_lds[wave][r16][1] = l;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int t = 0; t < DL; ++t) o_lds[wave][r16 * OS + (4 * g + i) * DL + t] = Q8 ? o[t][i] * vref : o[t][i];
  __syncthreads();
  const int row = tid >> 4, d0 = (tid & 15) * DL;
  if (row >= rows) return;
  float m = ml_lds[0][row][0];
#pragma unroll
  for (int w = 1; w < kPaWaves; ++w) m = fmaxf(m, ml_lds[w][row][0]);
  float sum = 0.f, acc[DL];
#pragma unroll
  for (int t = 0; t < DL; ++t) acc[t] = 0.f;
#pragma unroll
  for (int w = 0; w < kPaWaves; ++w) {
    const float mw = ml_lds[w][row][0];
    if (mw == -INFINITY) continue;
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
    const int64_t prow = (item * p.num_splits + split) * 16 + row;
    const int64_t nrows = int64_t(p.batch) * p.num_kv_heads * p.row_blocks * p.num_splits * 16;
#pragma unroll
    for (int t = 0; t < DL; t += 4)
      *reinterpret_cast<f32x4*>(ws + prow * D + d0 + t) =
          f32x4{acc[t] * inv, acc[t + 1] * inv, acc[t + 2] * inv, acc[t + 3] * inv};
    if ((tid & 15) == 0) ws[nrows * D + prow] = lse2;
  } else {
    const int hd = h * a.group + row_start + row;
    char* out = static_cast<char*>(p.out) +
                (int64_t(r.q0) * p.out_stride_token + int64_t(hd) * p.out_stride_head + d0) * 2;
    uint32_t packed[DL / 2];
#pragma unroll
    for (int t = 0; t < DL / 2; ++t)
      packed[t] = bf16 ? pack_bf16(acc[2 * t] * inv, acc[2 * t + 1] * inv)
                       : pack_f16(acc[2 * t] * inv, acc[2 * t + 1] * inv);
    if constexpr (DL == 8) *reinterpret_cast<w4*>(out) = w4{packed[0], packed[1], packed[2], packed[3]};
    else *reinterpret_cast<w2*>(out) = w2{packed[0], packed[1]};
    if (p.lse != nullptr && (tid & 15) == 0) p.lse[int64_t(r.q0) * p.num_qo_heads + hd] = lse2 * kPaLn2;
  }
}

}  // namespace
}  // namespace atlas

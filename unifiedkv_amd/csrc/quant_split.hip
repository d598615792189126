// Attention over the 8-bit paged cache where keys, not queries, are many (gfx950): a decode batch's single tokens, and
// chunks of a few (drafted) tokens a sequence.
//
// Work cut, partials and merge are page16_decode.hip's: the batch's pages in sequence order are cut into equal shares,
// one workgroup each, a wave for each KV head (or several where there are few heads), and a partial (m, l, O) for
// each sequence a share touches. What differs is what a wave does with a page:
//   * an MFMA column is a (query, q head) pair of the KV head: n_rep of them a query, 16 a column block, CB blocks a wave;
//   * K comes from HBM in whole rows, as codes through a wave-private LDS buffer, and out of it in the layout of the
//     score product's A operand: lane (i16, kg) reads the sixteen dims 16 (kg + 4 j) .. of token i16, its operands of
//     steps 2 j and 2 j + 1 (the queries are loaded in the same order of dims), and widens them. (Loaded from HBM in
//     that layout, 64 bytes of sixteen rows at a time, 16 x 32K took 181 us against 170.)
//   * V: lane (i16, kg) loads dims DPL * i16 .. of tokens 4 kg .. + 3, and permutes make the B operands of P.V;
//   * queries become fp16 under a power of two for each row (query_to_f16), the values are exact in fp16: scores have
//     fp32's precision whatever the model's type;
//   * the page after the one being reduced is in flight, across the border to a share's next sequence too.
// A page's codes take half of an fp16 page's time on HBM and as many instructions to reduce, and some 110 more to
// widen: with two waves a SIMD the long calls run at HBM's rate for e4m3, whose conversions are one instruction for two
// codes, and within 10 % of it for int8 (five for four).
#include <type_traits>

#include "page16_split.h"
#include "quant_common.h"
#include "quant_rows.h"

namespace ukv {

struct QuantSplitArgs : DecodeArgs {
  const uint8_t* ks;
  const uint8_t* vs;
  int64_t ks_sp, ks_sh, ks_sb, vs_sp, vs_sh, vs_sb;
  const int32_t* cu;  // chunks: [B + 1] first query row of each sequence
  int max_chunk;      // queries a sequence at most (decode: 1)
};

typedef const __attribute__((address_space(1))) uint8_t global_u8;
template <class T> __device__ __forceinline__ T load_global(global_u8* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const __attribute__((address_space(1))) T*>(p));
}

// One lane's part of a page.
template <int D> struct CodePage {
  u32x4 k[D / 64];         // sixteen codes of each of D / 64 rows, D / 16 lanes a row
  uint32_t ke[D / 64];     // exponent bytes of token i16, dims 16 (kg + 4 j) ..
  uint32_t v[4][D / 64];   // tokens 4 kg + t, dims D / 16 * i16 ..
  uint32_t ve;             // the four tokens' exponent bytes
  int nv, key0;            // (uniform) tokens of the sequence on the page, 0 where its id is no page; its first key
};

// The exponent byte of token t as 2^(s - 127). 255 is 2^128, infinity: zero codes make NaN of it, e4m3's are NaN.
__device__ __forceinline__ float exps_scale(uint32_t exps, int t) {
  return __uint_as_float((exps >> (8 * t) & 255u) << 23);
}

// Codes of four dims (word c of the rows) of a lane's four tokens -> its part of four B operands of P.V, one for each
// dim: fp16 values of tokens 01 and 23. int8: the tokens are paired as bytes (half the permutes that pairing fp16 values
// would take), and the pair's two scales are one packed factor. e4m3's conversion takes one scale along, so the fp16
// values are paired.
template <int QF, class P>
__device__ __forceinline__ void v_operands(const P& pg, int c, const f16x2 (&scales)[2], u32x2 (&out)[4]) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if constexpr (QF == UKV_CACHE_INT8) {
      const f16x2 off = {(_Float16)1152.f, (_Float16)1152.f};
      const uint32_t x = pg.v[2 * j][c] ^ 0x80808080u, y = pg.v[2 * j + 1][c] ^ 0x80808080u;
      const uint32_t lo = __builtin_amdgcn_perm(y, x, 0x05010400u), hi = __builtin_amdgcn_perm(y, x, 0x07030602u);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t w = __builtin_amdgcn_perm(0x64646464u, e < 2 ? lo : hi, e & 1 ? 0x04030402u : 0x04010400u);
        out[e][j] = __builtin_bit_cast(uint32_t, (__builtin_bit_cast(f16x2, w) - off) * scales[j]);
      }
    } else {
      const u32x2 x = quant_f16x4<QF>(pg.v[2 * j][c], exps_scale(pg.ve, 2 * j));
      const u32x2 y = quant_f16x4<QF>(pg.v[2 * j + 1][c], exps_scale(pg.ve, 2 * j + 1));
#pragma unroll
      for (int e = 0; e < 4; ++e)
        out[e][j] = __builtin_amdgcn_perm(y[e / 2], x[e / 2], e & 1 ? 0x07060302u : 0x05040100u);
    }
  }
}

// MODE as in page16_decode.hip. CHUNK: several queries a sequence, causal, the weights of P.V as one fp16 number (off
// by 2^-12 of themselves on average; two parts, as the single-token form has them, would make P.V the bound);
// not with kDirect.
template <int DT, int D, int CB, bool CHUNK, int MODE, int QF>
__global__ void __launch_bounds__(64 * UKV_PAGE16_WAVES, 1) quant_split_kernel(const QuantSplitArgs a) {
  constexpr int DPL = D / 16, STEPS = D / 32, KJ = D / 64, VW = D / 64;
  constexpr float kTau = 8.f;
  constexpr bool SHARED = MODE != kSplit, DIRECT = MODE == kDirect;
  static_assert(CHUNK || CB == 1, "one query's heads are one column block");
  typedef PSplit<UKV_DTYPE_F16> Weights;

  const int lane = threadIdx.x & 63;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wg_heads = DIRECT ? 1 : a.n_groups;  // SHARED: KV heads of this workgroup
  const int sub = SHARED ? wv / wg_heads : 0;
  const int subs = DIRECT ? UKV_PAGE16_WAVES : SHARED ? a.subs : 1;
  const int g = DIRECT ? (int)blockIdx.y : SHARED ? wv - sub * a.n_groups : blockIdx.z * (blockDim.x >> 6) + wv;
  if (!SHARED && g >= a.n_groups) return;  // whole wave leaves; only SHARED has barriers below
  const bool writer = blockIdx.x == 0 && blockIdx.z == 0 && wv == 0;

  // This workgroup's share of the pages: pages x0 .. x1 - 1 of the batch's list, from page x0 - s_first of sequence
  // b_first on (page16_decode.hip has the reasons). w: the share's number.
  const bool one = a.B <= 64;  // (uniform)
  int len_reg = 0, w = 0, G = 0, x0 = 0, x1 = 0, b_first = -1, s_first = 0;
  uint64_t nonempty = 0;
  auto share = [&](int P) {
    w = (G & 7) == 0 ? (int)(blockIdx.x & 7) * (G >> 3) + (int)(blockIdx.x >> 3) : (int)blockIdx.x;
    x0 = __builtin_amdgcn_readfirstlane(mul_div(w, P, G));
    x1 = __builtin_amdgcn_readfirstlane(mul_div(w + 1, P, G));
  };
  if constexpr (DIRECT) {
    b_first = blockIdx.x;
    x1 = pages_of(a.lens[b_first], a.max_blocks);
  } else if (one) {
    len_reg = lane < a.B ? clamp_len(a.lens[lane], a.max_blocks) : 0;
    const int n = (len_reg + 15) >> 4;
    const int incl = wave_inclusive_scan_i32(n);
    const int P = __builtin_amdgcn_readlane(incl, 63);
    nonempty = __ballot(n > 0);
    G = shares_for(a, P, [&]() { return wave_max_i32(n); });
    if (writer && lane < a.B) {
      a.seq_start[lane] = lane == 0 ? G : incl - n;
      a.seq_pages[lane] = n;
    }
    if ((int)blockIdx.x >= G) return;
    share(P);
    if (x0 >= x1) return;
    b_first = __builtin_ctzll(__ballot(n > 0 && incl > x0));
    s_first = __builtin_amdgcn_readlane(incl - n, b_first);
  } else {
    int P = 0, longest = 0;
    for (int c0 = 0; c0 < a.B; c0 += 64) {
      const int n = c0 + lane < a.B ? pages_of(a.lens[c0 + lane], a.max_blocks) : 0;
      P += __builtin_amdgcn_readlane(wave_inclusive_scan_i32(n), 63);
      longest = max(longest, wave_max_i32(n));
    }
    G = shares_for(a, P, [&]() { return longest; });
    if ((int)blockIdx.x >= G) return;
    share(P);
    if (x0 >= x1 && !writer) return;
    int carry = 0;
    for (int c0 = 0; c0 < a.B; c0 += 64) {
      const int bb = c0 + lane;
      const int n = bb < a.B ? pages_of(a.lens[bb], a.max_blocks) : 0;
      const int incl = wave_inclusive_scan_i32(n);
      const int start = carry + incl - n;
      if (writer && bb < a.B) {
        a.seq_start[bb] = bb == 0 ? G : start;
        a.seq_pages[bb] = n;
      }
      if (b_first < 0) {
        const uint64_t hit = __ballot(n > 0 && start + n > x0);
        if (hit) {
          const int l = __builtin_ctzll(hit);
          b_first = c0 + l;
          s_first = __builtin_amdgcn_readlane(start, l);
          if (!writer) break;
        }
      }
      carry += __builtin_amdgcn_readlane(incl, 63);
    }
    if (x0 >= x1) return;
  }

  const int i16 = lane & 15, kg = lane >> 4;
  // A lane's byte offsets within a page (32 bits, checked on the host), on top of wave-uniform addresses: the loads
  // take the two as a scalar base and a vector offset. (64-bit vector addresses cost a fifth of the loop.)
  constexpr int kRowLanes = D / 16, kRows = 64 / kRowLanes;  // K: lanes a row, rows a load
  const int k_row = lane / kRowLanes, k_chunk = lane % kRowLanes;
  const uint32_t koff = k_row * (uint32_t)a.k_st + 16 * k_chunk, voff = 4 * kg * (uint32_t)a.v_st + DPL * i16;
  const uint32_t keoff = (kg >> 1) * (uint32_t)a.ks_sb + i16;
  const uint32_t veoff = DPL * i16 / kQuantBlock * (uint32_t)a.vs_sb + 4 * kg;
  constexpr int KP = D + 16;  // bytes from row to row of the codes in LDS: the sixteen rows' reads meet no bank twice
  __shared__ __attribute__((aligned(16))) uint8_t k_lds[UKV_PAGE16_WAVES][16 * KP];
  uint8_t* ks = k_lds[wv];
  __shared__ __attribute__((aligned(16))) float part_lds[SHARED ? UKV_PAGE16_WAVES * 16 * D : 4];
  __shared__ float2 ml_lds[SHARED ? UKV_PAGE16_WAVES * 16 : 1];

  // A sequence's part of the share.
  struct Segment {
    int b, L, pa, n_pages, n_mine;  // its keys, first page, pages, and those this wave takes: pa + sub + i * subs
  };
  auto seq_len = [&](int b) -> int {
    return one && !DIRECT ? __builtin_amdgcn_readlane(len_reg, b)
                          : __builtin_amdgcn_readfirstlane(clamp_len(a.lens[b], a.max_blocks));
  };
  auto segment = [&](int b, int pa, int most) -> Segment {
    Segment s;
    s.b = __builtin_amdgcn_readfirstlane(b);
    s.L = seq_len(s.b);
    s.pa = __builtin_amdgcn_readfirstlane(pa);
    s.n_pages = __builtin_amdgcn_readfirstlane(min(((s.L + 15) >> 4) - pa, most));
    s.n_mine = SHARED ? __builtin_amdgcn_readfirstlane(max(0, s.n_pages - sub + subs - 1) / subs) : s.n_pages;
    if constexpr (CHUNK)
      if (a.cu[s.b + 1] <= a.cu[s.b]) s.n_mine = 0;  // no query: the pages are not read
    return s;
  };
  auto page_at = [&](const Segment& s, int i) -> int { return SHARED ? s.pa + sub + i * subs : s.pa + i; };
  auto window_ids = [&](const Segment& s, int i0) -> int {  // ids of the wave's pages i0 + lane
    return i0 + lane < s.n_mine ? a.bt[(int64_t)s.b * a.max_blocks + page_at(s, i0 + lane)] : 0;
  };

  u32x4 qb[CB][STEPS];  // B operands of the scores: column i16 of each block (zero where there is none)
  float q_scale[CB];    // the column's scale (log2 units), its row's power of two included
  float m_ref[CB];      // running max of the column (log2 units)
  float lsum[CB];       // this lane's share of the column's sum of weights
  int limit[CHUNK ? CB : 1];  // keys the column sees
  int all_see = 0;            // keys that every query of the sequence sees
  f32x4 acc[CB][DPL];

  auto load_page = [&](CodePage<D>& pg, int bid, int key0, int L) {
    bid = __builtin_amdgcn_readfirstlane(bid);
    const bool ok = (unsigned)bid < (unsigned)a.num_pages;
    const uint32_t page = ok ? (uint32_t)bid : 0u;
    pg.nv = ok ? min(16, L - key0) : 0;
    pg.key0 = key0;
    auto at = [&](const void* base, int64_t sp, int64_t sh) -> global_u8* {
      auto p = (global_u8*)base + (uint64_t)page * (uint32_t)sp + (int64_t)g * sh;
      asm("" : "+s"(p));
      return p;
    };
    global_u8* kp = at(a.k, a.k_sp, a.k_sh);
    global_u8* ke = at(a.ks, a.ks_sp, a.ks_sh);
    global_u8* vp = at(a.v, a.v_sp, a.v_sh);
    global_u8* ve = at(a.vs, a.vs_sp, a.vs_sh);
#pragma unroll
    for (int j = 0; j < KJ; ++j) pg.k[j] = load_global<u32x4>(kp + (koff + j * kRows * (uint32_t)a.k_st));
#pragma unroll
    for (int j = 0; j < KJ; ++j) pg.ke[j] = load_global<uint8_t>(ke + (keoff + 2 * j * (uint32_t)a.ks_sb));
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      global_u8* p = vp + (voff + t * (uint32_t)a.v_st);
      if constexpr (VW == 1) {
        pg.v[t][0] = load_global<uint32_t>(p);
      } else if constexpr (VW == 2) {
        const u32x2 x = load_global<u32x2>(p);
        pg.v[t][0] = x[0];
        pg.v[t][1] = x[1];
      } else {
        const u32x4 x = load_global<u32x4>(p);
#pragma unroll
        for (int c = 0; c < 4; ++c) pg.v[t][c] = x[c];
      }
    }
    pg.ve = load_global<uint32_t>(ve + veoff);
  };

  // Weights of a block's column in the order of P.V's A operand, and the keys' and values' part of the masks.
  auto process = [&](CodePage<D>& pg) {
    f32x4 sacc[CB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) sacc[cb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < KJ; ++j) *reinterpret_cast<u32x4*>(ks + (k_row + j * kRows) * KP + 16 * k_chunk) = pg.k[j];
#pragma unroll
    for (int j = 0; j < KJ; ++j) {
      const float scale = __uint_as_float(pg.ke[j] << 23);
      const u32x4 codes = *reinterpret_cast<const u32x4*>(ks + i16 * KP + 16 * (kg + 4 * j));
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t w0 = codes[2 * half], w1 = codes[2 * half + 1];
        const u32x2 x = quant_f16x4<QF>(w0, scale), y = quant_f16x4<QF>(w1, scale);
#pragma unroll
        for (int cb = 0; cb < CB; ++cb)
          sacc[cb] = mfma16x16x32<UKV_DTYPE_F16>(u32x4{x[0], x[1], y[0], y[1]}, qb[cb][2 * j + half], sacc[cb]);
      }
    }
    float s2[CB][4];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
#pragma unroll
      for (int r = 0; r < 4; ++r) s2[cb][r] = sacc[cb][r] * q_scale[cb];
    if (pg.nv < 16 || (CHUNK && pg.key0 + 16 > all_see)) {  // the sequence's end, a bad page id, the diagonal
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (4 * kg + r >= pg.nv) {
          pg.ve &= ~(255u << (8 * r));  // junk rows may read as NaN
#pragma unroll
          for (int c = 0; c < VW; ++c) pg.v[r][c] = 0u;
        }
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        const int vis = min(CHUNK ? limit[CHUNK ? cb : 0] - pg.key0 : 16, pg.nv) - 4 * kg;
#pragma unroll
        for (int r = 0; r < 4; ++r) s2[cb][r] = r < vis ? s2[cb][r] : -INFINITY;
      }
      if constexpr (CHUNK) {
        // A block of NaN among keys that some columns do not see (zero weights make NaN of it): its values count as
        // zeros below, and the columns that do see it get their NaN here. cnt: NaN tokens of the lane's dims that
        // column 4 kg + r sees.
        uint32_t bad = 0;
#pragma unroll
        for (int t = 0; t < 4; ++t) bad |= (pg.ve >> (8 * t) & 255u) == 255u ? 1u << t : 0u;
        if (__any(bad != 0)) {
          const uint32_t h1 = 0x3C00u;  // 1 in fp16
          const u32x2 marks = {(bad & 1u ? h1 : 0u) | (bad & 2u ? h1 << 16 : 0u),
                               (bad & 4u ? h1 : 0u) | (bad & 8u ? h1 << 16 : 0u)};
#pragma unroll
          for (int cb = 0; cb < CB; ++cb) {
            const int vis = min(limit[CHUNK ? cb : 0] - pg.key0, pg.nv) - 4 * kg;
            const u32x2 seen = {(vis > 0 ? h1 : 0u) | (vis > 1 ? h1 << 16 : 0u),
                                (vis > 2 ? h1 : 0u) | (vis > 3 ? h1 << 16 : 0u)};
            const f32x4 cnt = mfma16x16x16<UKV_DTYPE_F16>(seen, marks, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
              for (int e = 0; e < DPL; ++e) acc[cb][e][r] = cnt[r] > 0.f ? NAN : acc[cb][e][r];
          }
#pragma unroll
          for (int t = 0; t < 4; ++t)
            if (bad >> t & 1u) {
              pg.ve &= ~(255u << (8 * t));
#pragma unroll
              for (int c = 0; c < VW; ++c) pg.v[t][c] = 0u;
            }
        }
      }
    }
    bool move = false;
#pragma unroll
    for (int cb = 0; cb < CB; ++cb)
      move |= fmaxf(fmaxf(s2[cb][0], s2[cb][1]), fmaxf(s2[cb][2], s2[cb][3])) > m_ref[cb] + kTau;
    if (__any(move)) {
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        float mcol = fmaxf(fmaxf(s2[cb][0], s2[cb][1]), fmaxf(s2[cb][2], s2[cb][3]));
        mcol = fmaxf(mcol, __shfl_xor(mcol, 16));
        mcol = fmaxf(mcol, __shfl_xor(mcol, 32));
        const float m_new = fmaxf(m_ref[cb], mcol);
        const float alpha = fast_exp2(m_ref[cb] - m_new);
        lsum[cb] *= alpha;
        m_ref[cb] = m_new;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float ar = __shfl(alpha, 4 * kg + r);
#pragma unroll
          for (int e = 0; e < DPL; ++e) acc[cb][e][r] *= ar;
        }
      }
    }
    u32x2 phi[CB], plo[CB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      float p[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[r] = fast_exp2(s2[cb][r] - m_ref[cb]);
        lsum[cb] += p[r];
      }
      if constexpr (CHUNK) {
        constexpr float k = Weights::kScale;
        phi[cb] = u32x2{pack_f16(p[0] * k, p[1] * k), pack_f16(p[2] * k, p[3] * k)};
      } else {
        Weights::split(p, phi[cb], plo[cb]);
      }
    }
    f16x2 scales[2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
      scales[j] = f16x2{(_Float16)exps_scale(pg.ve, 2 * j), (_Float16)exps_scale(pg.ve, 2 * j + 1)};
#pragma unroll
    for (int c = 0; c < VW; ++c) {
      u32x2 bv[4];
      v_operands<QF>(pg, c, scales, bv);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
          f32x4& o = acc[cb][4 * c + e];
          o = mfma16x16x16<UKV_DTYPE_F16>(phi[cb], bv[e], o);
          if constexpr (!CHUNK) o = mfma16x16x16<UKV_DTYPE_F16>(plo[cb], bv[e], o);
        }
    }
  };

  CodePage<D> page;
  bool primed = false;  // it is the segment's first page, loaded at the end of the one before
  Segment s = segment(b_first, x0 - s_first, x1 - x0);
  int x = x0;  // global index of the segment's first page
  int bid_win = window_ids(s, 0);
  while (true) {
    // The next segment, and the first ids of its pages.
    x += s.n_pages;
    Segment nx = {};
    int bid_after = 0;
    if (!DIRECT && x < x1) {
      int b = s.b + 1;
      if (one) {
        b += __builtin_ctzll(nonempty >> b);  // (there is one: pages are left)
      } else {
        while (b < a.B - 1 && pages_of(a.lens[b], a.max_blocks) == 0) ++b;
      }
      nx = segment(b, 0, x1 - x);
      bid_after = window_ids(nx, 0);
    }
    int bid_next = window_ids(s, 64), w_begin = 0;

    int q0 = s.b, C = 1;  // the sequence's first query row, and its queries
    if constexpr (CHUNK) {
      q0 = __builtin_amdgcn_readfirstlane(a.cu[s.b]);
      C = __builtin_amdgcn_readfirstlane(a.cu[s.b + 1]) - q0;
      all_see = s.L - C + 1;
    }
    // Column x of block cb: its query and q head.
    auto col_query = [&](int cb, int x) -> int { return CHUNK ? (cb * 16 + x) / a.n_rep : 0; };
    auto col_head = [&](int cb, int x) -> int {
      return g * a.n_rep + (CHUNK ? (cb * 16 + x) % a.n_rep : x);
    };
    auto col_live = [&](int cb, int x) -> bool {
      return (CHUNK ? col_query(cb, x) < min(C, a.max_chunk) : x < a.n_rep) && col_head(cb, x) < a.Hq;
    };
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      const bool live = col_live(cb, i16);
      const uint16_t* qp =
          a.q + (live ? (int64_t)(q0 + col_query(cb, i16)) * a.q_sb + (int64_t)col_head(cb, i16) * a.q_sh : 0);
#pragma unroll
      for (int j = 0; j < KJ; ++j)
#pragma unroll
        for (int half = 0; half < 2; ++half)
          qb[cb][2 * j + half] = live ? ld16(qp + 16 * (kg + 4 * j) + 8 * half) : u32x4{0u, 0u, 0u, 0u};
      if constexpr (CHUNK) limit[cb] = live ? s.L - C + col_query(cb, i16) + 1 : 0;
      m_ref[cb] = kNegFltMax;
      lsum[cb] = 0.f;
#pragma unroll
      for (int e = 0; e < DPL; ++e) acc[cb][e] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    if (s.n_mine > 0) {
      // Page i of the wave; past its last page the next segment's first, or, where there is none, the last again (a load
      // of known age, which the compiler's waits count).
      auto load = [&](CodePage<D>& pg, int i) {
        int bid, key0, L = s.L;
        if (i >= s.n_mine && nx.n_mine > 0) {
          bid = __builtin_amdgcn_readlane(bid_after, 0);
          key0 = 16 * page_at(nx, 0);
          L = nx.L;
        } else {
          i = min(i, s.n_mine - 1);
          const int l = i - w_begin;
          bid = __builtin_amdgcn_readlane(bid_win, l & 63);
          if (l >= 64) bid = __builtin_amdgcn_readlane(bid_next, l - 64);
          key0 = 16 * page_at(s, i);
        }
        load_page(pg, bid, key0, L);
      };
      if (!primed) load(page, 0);
#pragma unroll
      for (int cb = 0; cb < CB; ++cb) {
        q_scale[cb] = a.scale_log2;
        if constexpr (DT == UKV_DTYPE_BF16) {
          const int top = query_top<STEPS>(qb[cb]);
          query_to_f16<STEPS>(qb[cb], top);
          q_scale[cb] *= query_scale(top);
        }
      }
      // One copy of the loop's body, the page in flight handed on by register moves: 19 of them against a body that
      // the instruction cache holds sooner and that leaves HBM more even (two copies in turn took 16.4 us against 14.8
      // for four sequences of 256-2048 tokens, 90 against 86.5 for 64 ragged ones and 176 against 172 for 16 x 32K; at
      // 64 dims, whose pages are short, 117 against 113 for the last, but 57 against 62 for the ragged ones. More pages
      // in flight only lost).
      while (true) {
        const int end = min(s.n_mine, w_begin + 64);
#pragma unroll 1
        for (int i = w_begin; i < end; ++i) {
          if constexpr (D > 128) {  // (no registers for a second page)
            process(page);
            load(page, i + 1);
          } else {
            CodePage<D> ahead;
            load(ahead, i + 1);
            process(page);
            page = ahead;
          }
        }
        w_begin += 64;
        if (w_begin >= s.n_mine) break;
        bid_win = bid_next;
        bid_next = window_ids(s, w_begin + 64);
      }
    }
    primed = s.n_mine > 0 && nx.n_mine > 0;

    // Partial slot w + b is unique: a workgroup's sequences are consecutive and a sequence's workgroups are consecutive.
    constexpr float kUnscale = 1.f / Weights::kScale;
    const int64_t slot = (int64_t)(w + s.b) * a.max_chunk * a.Hq;
    auto part_row = [&](int cb, int x) -> int64_t { return slot + (int64_t)col_query(cb, x) * a.Hq + col_head(cb, x); };
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
      // Column sums of the weights over the four token groups.
      float lcol = lsum[cb] + __shfl_xor(lsum[cb], 16);
      lcol += __shfl_xor(lcol, 32);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int x = 4 * kg + r;
        if (!col_live(cb, x)) continue;
        f32x4* dst = reinterpret_cast<f32x4*>(SHARED ? part_lds + (wv * 16 + x) * D + DPL * i16
                                                     : a.part_o + part_row(cb, x) * D + DPL * i16);
#pragma unroll
        for (int c = 0; c < DPL / 4; ++c)
          dst[c] = f32x4{acc[cb][4 * c][r], acc[cb][4 * c + 1][r], acc[cb][4 * c + 2][r], acc[cb][4 * c + 3][r]} * kUnscale;
      }
      if (kg == 0 && col_live(cb, i16)) {
        if (SHARED) ml_lds[wv * 16 + i16] = make_float2(m_ref[cb], lcol);
        else a.part_ml[part_row(cb, i16)] = make_float2(m_ref[cb], lcol);
      }
      if constexpr (SHARED) {
        // The head's waves add their rows up, each 64 * subs-th float4 of the sixteen, and write the segment's
        // partial. (Every wave of the workgroup walks the same segments.)
        __syncthreads();
        for (int it = sub * 64 + lane; it < 16 * (D / 4); it += 64 * subs) {
          const int h = it / (D / 4), dq = it % (D / 4);
          if (!col_live(cb, h)) continue;
          float M = kNegFltMax;
          const int gl = DIRECT ? 0 : g;
          for (int u = 0; u < subs; ++u) M = fmaxf(M, ml_lds[(u * wg_heads + gl) * 16 + h].x);
          f32x4 sum = {0.f, 0.f, 0.f, 0.f};
          float l = 0.f;
          for (int u = 0; u < subs; ++u) {
            const int sw = u * wg_heads + gl;
            const float2 ml = ml_lds[sw * 16 + h];
            const float f = fast_exp2(ml.x - M);
            sum += f * *reinterpret_cast<const f32x4*>(part_lds + (sw * 16 + h) * D + 4 * dq);
            l += f * ml.y;
          }
          if constexpr (DIRECT) {  // (a sequence without keys: 0 / 0)
            const uint32_t o01 = Elem<DT>::from_float(sum[0] / l) | (uint32_t)Elem<DT>::from_float(sum[1] / l) << 16;
            const uint32_t o23 = Elem<DT>::from_float(sum[2] / l) | (uint32_t)Elem<DT>::from_float(sum[3] / l) << 16;
            *reinterpret_cast<u32x2*>(a.out + ((int64_t)s.b * a.Hq + col_head(cb, h)) * D + 4 * dq) = u32x2{o01, o23};
          } else {
            *reinterpret_cast<f32x4*>(a.part_o + part_row(cb, h) * D + 4 * dq) = sum;
            if (dq == 0) a.part_ml[part_row(cb, h)] = make_float2(M, l);
          }
        }
        if (DIRECT && cb == CB - 1) break;
        __syncthreads();  // read before the next block's or segment's rows
      }
    }
    if (DIRECT || x >= x1) break;
    s = nx;
    bid_win = bid_after;
  }
}

// Merges the partials of one chunk query's q head (blockIdx.x = query * Hq + head) of sequence blockIdx.y. A chunk
// longer than declared gets NaN in every row.
template <int DT, int D> __global__ void __launch_bounds__(256) quant_chunk_combine_kernel(const QuantSplitArgs a) {
  const int qi = blockIdx.x / a.Hq, h = blockIdx.x % a.Hq, b = blockIdx.y;
  const int q0 = a.cu[b], C = a.cu[b + 1] - q0;
  if (qi >= C) return;
  if (C > a.max_chunk) {
    for (int i = qi; i < C; i += a.max_chunk)
      for (int d = threadIdx.x; d < D; d += 256) a.out[((int64_t)(q0 + i) * a.Hq + h) * D + d] = 0x7FFFu;
    return;
  }
  combine_row<DT, D>(a, b, (int64_t)a.max_chunk * a.Hq, (int64_t)qi * a.Hq + h,
                     a.out + ((int64_t)(q0 + qi) * a.Hq + h) * D);
}

namespace {

template <int DT, int D, int QF> void launch_decode(const QuantSplitArgs& a, hipStream_t stream) {
  const int waves = std::min(UKV_PAGE16_WAVES, a.n_groups);
  if (D <= 128 && direct_shape(a.B, a.n_groups, a.n_rep, a.D, a.max_blocks)) {
    if constexpr (D <= 128)
      hipLaunchKernelGGL((quant_split_kernel<DT, D, 1, false, kDirect, QF>), dim3(a.B, a.n_groups),
                         dim3(64 * UKV_PAGE16_WAVES), 0, stream, a);
  } else if (D <= 128 && a.n_groups <= UKV_PAGE16_WAVES / 2) {
    if constexpr (D <= 128)
      hipLaunchKernelGGL((quant_split_kernel<DT, D, 1, false, kShared, QF>), dim3(a.grid_wgs),
                         dim3(64 * a.subs * a.n_groups), 0, stream, a);
  } else {
    hipLaunchKernelGGL((quant_split_kernel<DT, D, 1, false, kSplit, QF>),
                       dim3(a.grid_wgs, 1, (a.n_groups + waves - 1) / waves), dim3(64 * waves), 0, stream, a);
  }
}

template <int DT, int D, int CB, int QF> void launch_chunk(const QuantSplitArgs& a, hipStream_t stream) {
  const int waves = std::min(UKV_PAGE16_WAVES, a.n_groups);
  if (a.n_groups <= UKV_PAGE16_WAVES / 2)
    hipLaunchKernelGGL((quant_split_kernel<DT, D, CB, true, kShared, QF>), dim3(a.grid_wgs),
                       dim3(64 * a.subs * a.n_groups), 0, stream, a);
  else
    hipLaunchKernelGGL((quant_split_kernel<DT, D, CB, true, kSplit, QF>),
                       dim3(a.grid_wgs, 1, (a.n_groups + waves - 1) / waves), dim3(64 * waves), 0, stream, a);
  const size_t lds = (size_t)(a.grid_wgs + 256 * 4) * sizeof(float);
  hipLaunchKernelGGL((quant_chunk_combine_kernel<DT, D>), dim3(a.max_chunk * a.Hq, a.B), dim3(256), lds, stream, a);
}

template <int DT, int QF> void launch_format(const QuantSplitArgs& a, bool chunk, hipStream_t stream) {
  if (chunk) {
    const bool two = a.max_chunk * a.n_rep > 16;
    if (a.D == 64)
      two ? launch_chunk<DT, 64, 2, QF>(a, stream) : launch_chunk<DT, 64, 1, QF>(a, stream);
    else
      two ? launch_chunk<DT, 128, 2, QF>(a, stream) : launch_chunk<DT, 128, 1, QF>(a, stream);
    return;
  }
  switch (a.D) {
    case 64: launch_decode<DT, 64, QF>(a, stream); break;
    case 128: launch_decode<DT, 128, QF>(a, stream); break;
    default: launch_decode<DT, 256, QF>(a, stream); break;
  }
}

// Whether the split kernel takes the cache and the queries: its loads' alignment, offsets within a page and page
// strides in 32 bits.
bool split_layout(const QuantAttnArgs& x) {
  const QuantLayer& c = x.c;
  auto aligned = [](const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  auto narrow = [](int64_t stride) { return stride >= 0 && stride < (1 << 26); };
  auto page = [](int64_t stride) { return stride >= 0 && stride <= (int64_t)UINT32_MAX; };
  const unsigned vw = (unsigned)x.D / 16;  // bytes of V a lane loads of a token
  return ((c.k_sp | c.k_st | c.k_sh) & 15) == 0 && aligned(c.k, 16) && ((c.v_sp | c.v_st | c.v_sh) & (vw - 1)) == 0 &&
         aligned(c.v, vw) && ((c.vs_sp | c.vs_sh | c.vs_sb) & 3) == 0 && aligned(c.vs, 4) && narrow(c.k_st) &&
         narrow(c.v_st) && narrow(c.ks_sb) && narrow(c.vs_sb) && page(c.k_sp) && page(c.v_sp) && page(c.ks_sp) &&
         page(c.vs_sp) && ((x.q_st | x.q_sh) & 7) == 0 && aligned16(x.q) && aligned16(x.out) && x.max_blocks > 0;
}

int launch(const QuantAttnArgs& x, bool chunk, const WorkspaceLayout& w, int dtype, int format, void* workspace,
           hipStream_t stream) {
  const QuantLayer& c = x.c;
  QuantSplitArgs a{};
  a.q = x.q;
  a.k = reinterpret_cast<const uint16_t*>(c.k);
  a.v = reinterpret_cast<const uint16_t*>(c.v);
  a.bt = x.bt;
  a.lens = x.lens;
  a.out = x.out;
  a.q_sb = x.q_st;
  a.q_sh = x.q_sh;
  a.k_sp = c.k_sp;
  a.k_st = c.k_st;
  a.k_sh = c.k_sh;
  a.v_sp = c.v_sp;
  a.v_st = c.v_st;
  a.v_sh = c.v_sh;
  a.ks = c.ks;
  a.vs = c.vs;
  a.ks_sp = c.ks_sp;
  a.ks_sh = c.ks_sh;
  a.ks_sb = c.ks_sb;
  a.vs_sp = c.vs_sp;
  a.vs_sh = c.vs_sh;
  a.vs_sb = c.vs_sb;
  a.cu = x.cu;
  a.B = x.B;
  a.Hq = x.Hq;
  a.n_rep = x.n_rep;
  a.n_groups = (x.Hq + x.n_rep - 1) / x.n_rep;
  a.D = x.D;
  a.max_blocks = x.max_blocks;
  a.num_pages = c.num_pages;
  a.max_chunk = chunk ? x.max_chunk : 1;
  a.scale = x.scale;
  a.scale_log2 = x.scale * kLog2e;
  for (a.subs = 2; 2 * a.subs * a.n_groups <= UKV_PAGE16_WAVES;) a.subs *= 2;  // (where the kernel shares heads)
  char* ws = static_cast<char*>(workspace);
  a.part_o = reinterpret_cast<float*>(ws + w.part_o_off);
  a.part_ml = reinterpret_cast<float2*>(ws + w.part_ml_off);
  a.seq_start = reinterpret_cast<int32_t*>(ws + w.seq_off);
  a.seq_pages = a.seq_start + x.B;
  a.grid_wgs = launch_wgs(w.wgs, x.B, x.max_blocks, a.n_groups);
  a.fixed_shares = env_wgs() > 0;
  if (dtype == UKV_DTYPE_BF16)
    format == UKV_CACHE_INT8 ? launch_format<UKV_DTYPE_BF16, UKV_CACHE_INT8>(a, chunk, stream)
                             : launch_format<UKV_DTYPE_BF16, UKV_CACHE_FP8>(a, chunk, stream);
  else
    format == UKV_CACHE_INT8 ? launch_format<UKV_DTYPE_F16, UKV_CACHE_INT8>(a, chunk, stream)
                             : launch_format<UKV_DTYPE_F16, UKV_CACHE_FP8>(a, chunk, stream);
  if (hipGetLastError() != hipSuccess) return UKV_ERR_LAUNCH;
  if (!chunk && !direct_shape(x.B, a.n_groups, x.n_rep, x.D, x.max_blocks)) launch_combine(a, dtype, stream);
  return hipGetLastError() == hipSuccess ? UKV_OK : UKV_ERR_LAUNCH;
}

// Chunks the split kernel takes: up to two column blocks a wave. One block always pays against the tiled kernel, whose
// workgroups hold 256 columns and more: two queries a sequence on 32/8 heads, 16 sequences of 100-600 tokens 17.8 us
// against 22.5, 32 of 1-4K 44 against 96, one of 32K 32 against 59. Two need keys enough for the shares, four pages a CU:
// eight queries 66 against 98 and 41 against 60 us behind the longer ones, but 32 against 24 behind 100-600 tokens and 27
// against 24 for four of 300-1500. (A second pass over the keys for up to 64 columns took 236 us behind sixteen sequences of
// 4-32K, where quant_shares.hip takes 204, 66 against 61 behind one of 32K and 120 against 100 behind 32 of 1-4K.)
bool chunk_shape(int batch, int max_chunk, int n_rep, int head_dim, int max_blocks) {
  const int64_t columns = (int64_t)max_chunk * n_rep;
  return (head_dim == 64 || head_dim == 128) &&
         (columns <= 16 || (columns <= 32 && (int64_t)batch * max_blocks >= 4 * device_cu_count()));
}

WorkspaceLayout chunk_layout(int batch, int hq, int d, int max_chunk, int max_blocks) {
  return workspace_layout(batch, hq * max_chunk, d, max_blocks);
}

}  // namespace

// The decode over the 8-bit cache (arguments checked by the caller).
int quant_decode(const QuantAttnArgs& x, int dtype, int format, void* workspace, size_t workspace_bytes,
                 hipStream_t stream) {
  if (!((x.D == 64 || x.D == 128 || x.D == 256) && x.n_rep <= 16 && split_layout(x)))
    return quant_rows_attention(x, x.B, dtype, format, stream);
  if (x.B > 65535) return UKV_ERR_INVALID_ARGUMENT;  // (the merge's grid)
  const WorkspaceLayout w = workspace_layout(x.B, x.Hq, x.D, x.max_blocks);
  if (!workspace || workspace_bytes < w.total || !aligned16(workspace)) return UKV_ERR_WORKSPACE;
  return launch(x, false, w, dtype, format, workspace, stream);
}

size_t quant_chunk_workspace(int batch, int hq, int n_rep, int d, int max_chunk, int max_blocks) {
  if (!chunk_shape(batch, max_chunk, n_rep, d, max_blocks)) return 0;
  return chunk_layout(batch, hq, d, max_chunk, max_blocks).total;
}

bool quant_chunk(const QuantAttnArgs& x, int dtype, int format, void* workspace, size_t workspace_bytes,
                 hipStream_t stream, int& status) {
  if (!chunk_shape(x.B, x.max_chunk, x.n_rep, x.D, x.max_blocks) || !split_layout(x)) return false;
  const WorkspaceLayout w = chunk_layout(x.B, x.Hq, x.D, x.max_chunk, x.max_blocks);
  if (!workspace || workspace_bytes < w.total || !aligned16(workspace) || x.B > 65535) return false;
  status = launch(x, true, w, dtype, format, workspace, stream);
  return true;
}

}  // namespace ukv

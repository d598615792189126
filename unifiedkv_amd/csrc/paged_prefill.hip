// Chunked prefill attention over the paged pool (gfx950, bf16/fp16 MFMA).
//
// Semantics: for sequence b with kv_lens[b] keys resident in pages (the
// prefix plus this chunk) and C_b = cu_q[b+1] - cu_q[b] chunk queries, query i
// sits at absolute position P_b + i, P_b = kv_lens[b] - C_b, and attends to
// keys 0 .. P_b + i (causal, aligned to the bottom right) - what the
// reference's chunked prefill computes through HF attention over the past KV
// (core/engine.py:1826-1854, core/chunked_prefill.py:9-33) and what
// flash_attn_varlen_func(causal=True) computes for a single chunk
// (core/varlen.py:19-42). The reference has no paged prefill; here the keys
// are read from 16-token pages through the block table, and
// ukv_kv_write_varlen first writes the chunk's own K/V into its pages.
//
// Kernel: one workgroup of W waves (W = 8, two per SIMD) takes QW = W * CB *
// (16 / n_rep) consecutive queries of one KV group. Within a wave, an MFMA
// column is a (query, q head) pair: 16 / n_rep queries times the n_rep q heads
// of the group, so one K/V read serves the whole GQA group; a wave holds CB
// 16-column blocks, three or two.
//   * block plan: the chunk of each (sequence, group) is cut from its end down
//     into three-column blocks and then two-column ones (three are cheaper per
//     query, two fill the last round of the launch: the host picks the mix that
//     its model of the dispatch finishes first); each XCD (dispatch is
//     round-robin over the 8 XCDs) runs a contiguous range of (sequence, group)
//     pairs, three-column blocks first: the query blocks of one pair share that
//     XCD's L2 while they stream the same pages;
//   * key tiles of 32 keys (two pages) pass through registers into a 4-slot
//     LDS ring (rows padded to 288 B), written two tiles ahead of their use,
//     with a barrier after every second tile; the loads of tiles t+3 and t+4
//     are in flight while tile t is computed;
//   * S^T = K Q^T on v_mfma_f32_16x16x32 in the input type (A = 16 keys x 32
//     dims from LDS, B = the wave's q columns in registers); lane l ends with
//     keys 4*(l/16) + r of column l % 16;
//   * online softmax per column in log2 units; masks only on tiles that touch
//     the sequence end, an invalid page or the causal diagonal; the running max
//     moves only when a weight reaches 2^8 (wave vote on the packed weights);
//   * P.V on v_mfma_f32_16x16x32_f16: P is rounded to fp16 (11 significant
//     bits, 4x finer than a bf16 P) and, for bf16 pools, the loader converts
//     the V tile to fp16, which is exact for |v| < 65520; a workgroup whose
//     keys hold a larger or non-finite bf16 V recomputes its columns on an
//     fp32 path. The S^T layout is already P's A-operand layout; V's B
//     operands come from ds_read_b64_tr_b16 transpose reads; the softmax
//     denominators come from one more MFMA against a ones operand, so they sum
//     exactly the rounded P;
//   * shapes whose n_rep does not divide 16, and 64-dim heads, run FINE instances: columns are
//     (query, head) pairs laid end to end, so every column of the matrix cores is used, V keeps its
//     type and P goes in as two 16-bit parts (fp32-grade weights, as the scalar kernel they ran on
//     before had): 28 q heads on 4 KV heads, 4 x 512 queries over 5-8K keys in 0.314 ms against
//     72.7 ms; twelve 64-dim prompts of 16-700 tokens in 0.055 ms against 6.4 ms (0.10 ms with one
//     workgroup per CU, three column blocks, 64-key tiles and the pairs' blocks in turn);
//   * key parts: a launch of few query blocks leaves CUs idle however long its prefix. Its keys are
//     then cut into equal parts, each (block, part) a workgroup, and a merge kernel adds the parts
//     up: one 389-query chunk behind 32256 keys (40 blocks) in 0.22 ms against 0.86 ms;
//   * SnapKV row statistics: the blocks holding each sequence's last obs queries
//     also write those rows' running max and denominator; obs_rows_finish_kernel
//     then sums the sink and window keys' weights again from the same scores and
//     takes them off, leaving the middle keys' sum.
#include "paged_prefill.h"

namespace ukv {

// SnapKV row statistics from the (m, l) pairs paged_prefill_kernel left in obs_stats.
// l sums the weights 2^(s * scale * log2e - m) of every key the query sees, each rounded to fp16;
// the sink keys [0, sink) and the window keys [max(L - obs, sink), the query's own position] are
// summed again here from the same scores (v_mfma_f32_16x16x32 on the same operands, in the same
// order), exp2 and fp16 rounding, and taken off, which leaves the middle keys [sink, L - obs).
// Where the prefill computed those weights against the final m (m moves only when a weight would
// reach 2^8), they cancel exactly and the sum carries only the middle weights' own fp16 rounding;
// weights taken before a later move of m were rescaled in fp32 and leave a residue of at most
// 2^-11 of their share. The row becomes (log2 of that sum and of
// the zero rows padding the middle keys to a multiple of 16, 0) in the units of s * scale * log2e;
// it is flagged (y = 1) for the scoring pass to recompute from the keys where the prefill flagged
// it, where the sink and window hold half of its weight or more (the difference would lose bits),
// or where the middle sum falls below 2^-100 of its max (m is the max over every key the query
// sees: middle weights below 2^-126 of it lose bits). One workgroup per 16 columns (observation query,
// q head of the group) of a (sequence, KV group), its four waves taking every fourth page: a 64-key
// sink and a 128-key window are one round of loads (one wave took them in four, 13.5 us a layer at 2
// x 8 x 32 column blocks). Lane (i16, kg) holds column i16 and keys 4kg .. 4kg + 3 of each 16-key
// page. (The (m, l) pairs exist only where the tiled kernel ran.)
// FINE: the weights as the FINE instances sum them, in two parts.
template <int DT, bool FINE>
__global__ void __launch_bounds__(256) obs_rows_finish_kernel(const PrefillArgs a) {
  __shared__ float wave_part[4][16];
  const int lane = threadIdx.x & 63, i16 = lane & 15, kg = lane >> 4;
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int cols = a.obs * a.n_rep;
  const int nblk = (cols + 15) >> 4;
  const int blk = (int)(blockIdx.x % nblk);
  const int64_t pair = blockIdx.x / nblk;
  const int g = (int)(pair % a.n_groups), b = (int)(pair / a.n_groups);
  const int q_begin = a.cu_q[b], C = a.cu_q[b + 1] - q_begin;
  const int L = kv_len_of(a, b);
  const int col = blk * 16 + i16;
  const int i = col / a.n_rep, h = g * a.n_rep + col % a.n_rep;
  const int qi = C - a.obs + i;
  const bool live = col < cols && h < a.Hq && qi >= 0 && C <= a.max_chunk;
  if (!__any(live)) return;  // (workgroup-uniform: a chunk shorter than the window, or too long)
  float2* slot = a.obs_stats + (int64_t)b * a.stats_seq_stride + (int64_t)h * a.obs + i;
  const float2 ml = live ? *slot : make_float2(0.f, 0.f);
  const bool ok = live && __builtin_isfinite(ml.x) && ml.y > 0.f && __builtin_isfinite(ml.y);
  const float m = ok ? ml.x : 0.f;
  // B operand: dims 32s + 8kg .. 32s + 8kg + 7 of column i16's query row
  const uint16_t* qp = a.q + (live ? (int64_t)(q_begin + qi) * a.q_st + (int64_t)h * a.q_sh : 0) + 8 * kg;
  u32x4 qv[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) qv[s] = live ? ld16(qp + 32 * s) : u32x4{0u, 0u, 0u, 0u};
  const int pos = L - C + qi;  // the query's position: it sees keys 0 .. pos
  const float sl2 = a.scale_log2;
  const int32_t* btrow = a.bt + (int64_t)b * a.max_blocks;
  float part = 0.f;
  // The sink's keys [0, s_end) and the window's [w_beg, L), page by page (page pg holds keys 16 pg ..
  // 16 pg + 15): this wave's pages four at a time, their loads issued together. A operand: dims
  // 32s + 8kg .. of key 16 pg + i16.
  const int s_end = min(a.sink, L), w_beg = max(L - a.obs, a.sink);
  const int n_sink = (s_end + 15) >> 4, w_page = w_beg >> 4;
  const int n_all = n_sink + max(0, ((L + 15) >> 4) - w_page);
  for (int t0 = wv; t0 < n_all; t0 += 16) {
    u32x4 ka[4][4];
    int pg[4];
    bool pok[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int t = t0 + 4 * u;
      pg[u] = t < n_sink ? t : w_page + t - n_sink;
      const int id = t < n_all ? btrow[pg[u]] : -1;
      pok[u] = (unsigned)id < (unsigned)a.num_pages;
      const uint16_t* kp =
          a.k + (int64_t)(pok[u] ? id : 0) * a.k_sp + (int64_t)i16 * a.k_st + (int64_t)g * a.k_sh + 8 * kg;
#pragma unroll
      for (int s = 0; s < 4; ++s) ka[u][s] = pok[u] ? ld16(kp + 32 * s) : u32x4{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool in_sink = t0 + 4 * u < n_sink;
      const int lo = in_sink ? 0 : w_beg, hi = in_sink ? s_end : L;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < 4; ++s) acc = mfma16x16x32<DT>(ka[u][s], qv[s], acc);
      // the weights rounded as the prefill kernel summed them (see above)
      float p[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) p[r] = fast_exp2(__builtin_fmaf(acc[r], sl2, -m));
      if constexpr (FINE) {
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
          uint32_t h, l;
          PrefillSplit<DT>::split(p[r], p[r + 1], h, l);
          p[r] = Elem<DT>::lo(h) + Elem<DT>::lo(l);
          p[r + 1] = Elem<DT>::hi(h) + Elem<DT>::hi(l);
        }
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) p[r] = (float)(_Float16)p[r];
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int key = 16 * pg[u] + 4 * kg + r;
        part += (pok[u] && key >= lo && key < hi && key <= pos) ? p[r] : 0.f;
      }
    }
  }
  part += __shfl_xor(part, 16);
  part += __shfl_xor(part, 32);
  if (kg == 0) wave_part[wv][i16] = part;
  __syncthreads();
  if (wv > 0) return;
  part = (wave_part[0][i16] + wave_part[1][i16]) + (wave_part[2][i16] + wave_part[3][i16]);
  if (kg == 0 && live) {
    float2 res = make_float2(0.f, 1.f);
    if (ok) {
      const float l = ml.y - part;
      const int L_mid = L - a.sink - a.obs;
      const int n_pad = ((L_mid + 15) & ~15) - L_mid;
      const float top = n_pad > 0 ? fmaxf(m, 0.f) : m;
      const float lse = top + __log2f(l * exp2f(m - top) + (float)n_pad * exp2f(-top));
      if (l >= 0.5f * ml.y && l >= 0x1p-100f && __builtin_isfinite(lse)) res = make_float2(lse, 0.f);
    }
    *slot = res;
  }
}

// Marks every observation row of the call as recomputed-by-the-scorer: (0, 1) at row
// obs_stats[b * stats_seq_stride + h * obs + i] for b < B, h < Hq, i < obs.
__global__ void __launch_bounds__(256) obs_flag_kernel(const PrefillArgs a, const int64_t rows) {
  const int64_t idx = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (idx >= rows) return;
  const int64_t per = (int64_t)a.Hq * a.obs;
  a.obs_stats[(idx / per) * a.stats_seq_stride + idx % per] = make_float2(0.f, 1.f);
}

// Reference-order scalar prefill for shapes the MFMA kernel does not cover: one
// workgroup per (q head, query row); natural exp; keys 0 .. P + i in page order.
template <int DT>
__global__ void __launch_bounds__(256) paged_prefill_scalar_kernel(const PrefillArgs a) {
  const int row = blockIdx.x;
  const int h = blockIdx.y;
  // sequence of this query row
  int b = 0;
  while (b + 1 < a.B && a.cu_q[b + 1] <= row) ++b;
  const int C = a.cu_q[b + 1] - a.cu_q[b];
  const int i = row - a.cu_q[b];
  if (i < 0 || i >= C) return;
  if (C > a.max_chunk) {  // longer than declared: its K/V were not all written (see prefill_nan_rows)
    for (int d = threadIdx.x; d < a.D; d += blockDim.x) a.out[((int64_t)row * a.Hq + h) * a.D + d] = 0x7FFFu;
    return;
  }
  const int Lk = kv_len_of(a, b);
  const int L = max(0, min(Lk, Lk - C + i + 1));
  const int g = h / a.n_rep;
  const int tid = threadIdx.x, t = tid >> 4, sub = tid & 15;
  __shared__ float qs[256];
  __shared__ float ss[16];
  const uint16_t* qrow = a.q + (int64_t)row * a.q_st + (int64_t)h * a.q_sh;
  for (int d = tid; d < a.D; d += blockDim.x) qs[d] = Elem<DT>::one(qrow[d]);
  __syncthreads();
  const int n_pages = (L + 15) >> 4;
  const int d = tid;
  float m = kNegFltMax, l = 0.f, acc = 0.f;
  for (int pg = 0; pg < n_pages; ++pg) {
    int bid = a.bt[(int64_t)b * a.max_blocks + pg];
    const bool ok = (unsigned)bid < (unsigned)a.num_pages;
    bid = ok ? bid : 0;
    const int nv = ok ? min(16, L - 16 * pg) : 0;
    float part = 0.f;
    if (t < nv) {
      const uint16_t* krow = a.k + (int64_t)bid * a.k_sp + (int64_t)t * a.k_st + (int64_t)g * a.k_sh;
      for (int dd = sub; dd < a.D; dd += 16) part += Elem<DT>::one(krow[dd]) * qs[dd];
    }
    part = row_sum16(part);
    if (sub == 0) ss[t] = (t < nv) ? part * a.scale : kNegFltMax;
    __syncthreads();
    float mx = kNegFltMax;
    for (int tt = 0; tt < 16; ++tt) mx = fmaxf(mx, ss[tt]);
    const float mn = fmaxf(m, mx);
    const float alpha = expf(m - mn);
    float psum = 0.f, pv = 0.f;
    for (int tt = 0; tt < 16; ++tt) {
      const float pt = (tt < nv) ? expf(ss[tt] - mn) : 0.f;
      psum += pt;
      if (d < a.D && tt < nv)
        pv += pt * Elem<DT>::one(a.v[(int64_t)bid * a.v_sp + (int64_t)tt * a.v_st + (int64_t)g * a.v_sh + d]);
    }
    l = l * alpha + psum;
    acc = acc * alpha + pv;
    m = mn;
    __syncthreads();
  }
  if (d < a.D) a.out[((int64_t)row * a.Hq + h) * a.D + d] = Elem<DT>::from_float(acc / l);
}

// Chunk K/V rows into their pages: row cu_q[b] + i goes to position P_b + i.
struct VarlenWriteArgs {
  uint16_t* k_pool;
  uint16_t* v_pool;
  int64_t k_sp, k_st, k_sh, v_sp, v_st, v_sh;
  const uint16_t* k_new;
  const uint16_t* v_new;
  int64_t n_st, n_sh;  // [total][H][D] strides shared by k_new and v_new
  const int32_t* bt;
  const int32_t* cu_q;
  const int32_t* kv_lens;
  int B, H, D, max_blocks, num_pages, vec;
  int per_shift, h_shift;  // log2(D / 8), log2(H) for the 16-byte path (-1: not powers of two)
};

// 16-byte path for power-of-two heads and D / 8: block (tb, b) writes 16 chunk tokens of
// sequence b; 16-byte chunk `it` = (token, head, chunk) by shifts. The two pages the 16
// positions can touch are read once; each pass issues 8 K and 8 V loads before its stores.
__global__ void __launch_bounds__(256) kv_write_varlen_vec_kernel(const VarlenWriteArgs a) {
  constexpr int J = 8;
  const int b = blockIdx.y;
  const int q_begin = a.cu_q[b];
  const int C = a.cu_q[b + 1] - q_begin;
  const int i0 = blockIdx.x * 16;
  if (i0 >= C) return;
  const int cap = a.max_blocks * 16;
  const int Lk = min(max(a.kv_lens[b], 0), cap);
  const int P0 = Lk - C;
  const int blk0 = (P0 + i0) >> 4;  // first page index these 16 positions touch (P0 + i0 >= 0 when valid)
  const int32_t* btrow = a.bt + (int64_t)b * a.max_blocks;
  const int pg0 = (blk0 >= 0 && blk0 < a.max_blocks) ? btrow[blk0] : -1;
  const int pg1 = (blk0 + 1 >= 0 && blk0 + 1 < a.max_blocks) ? btrow[blk0 + 1] : -1;
  const int per_mask = (1 << a.per_shift) - 1, h_mask = (1 << a.h_shift) - 1;
  const int items = 16 << (a.per_shift + a.h_shift);
  for (int base = 0; base < items; base += J * 256) {
    u32x4 kx[J], vx[J];
    uint16_t* kd[J];
    uint16_t* vd[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int it = base + j * 256 + threadIdx.x;
      const int c = it & per_mask;
      const int h = (it >> a.per_shift) & h_mask;
      const int i = i0 + (it >> (a.per_shift + a.h_shift));
      const int pos = P0 + i;
      const int page = ((pos >> 4) == blk0) ? pg0 : pg1;
      const bool ok = it < items && i < C && pos >= 0 && pos < cap && (unsigned)page < (unsigned)a.num_pages;
      kd[j] = ok ? a.k_pool + (int64_t)page * a.k_sp + (int64_t)(pos & 15) * a.k_st + (int64_t)h * a.k_sh + 8 * c
                 : nullptr;
      vd[j] = ok ? a.v_pool + (int64_t)page * a.v_sp + (int64_t)(pos & 15) * a.v_st + (int64_t)h * a.v_sh + 8 * c
                 : nullptr;
      const int64_t src = (int64_t)(q_begin + (ok ? i : i0)) * a.n_st + (int64_t)h * a.n_sh + 8 * c;
      kx[j] = ok ? *reinterpret_cast<const u32x4*>(a.k_new + src) : u32x4{0u, 0u, 0u, 0u};
      vx[j] = ok ? *reinterpret_cast<const u32x4*>(a.v_new + src) : u32x4{0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (kd[j]) {
        *reinterpret_cast<u32x4*>(kd[j]) = kx[j];
        *reinterpret_cast<u32x4*>(vd[j]) = vx[j];
      }
    }
  }
}

// grid (token blocks of 16, B): block (tb, b) writes 16 chunk tokens of sequence b.
__global__ void __launch_bounds__(256) kv_write_varlen_kernel(const VarlenWriteArgs a) {
  const int b = blockIdx.y;
  const int q_begin = a.cu_q[b];
  const int C = a.cu_q[b + 1] - q_begin;
  const int cap = a.max_blocks * 16;
  const int Lk = min(max(a.kv_lens[b], 0), cap);
  const int P0 = Lk - C;
  const int per = a.vec ? a.D / 8 : a.D;
  const int items = 16 * a.H * per;
  for (int it = threadIdx.x; it < items; it += blockDim.x) {
    const int c = it % per;
    const int h = (it / per) % a.H;
    const int i = blockIdx.x * 16 + it / (per * a.H);
    if (i >= C) continue;
    const int pos = P0 + i;
    if (pos < 0 || pos >= cap) continue;
    const int page = a.bt[(int64_t)b * a.max_blocks + (pos >> 4)];
    if ((unsigned)page >= (unsigned)a.num_pages) continue;
    const int64_t e = a.vec ? 8 * c : c;
    const int64_t src = (int64_t)(q_begin + i) * a.n_st + (int64_t)h * a.n_sh + e;
    uint16_t* kd = a.k_pool + (int64_t)page * a.k_sp + (int64_t)(pos & 15) * a.k_st + (int64_t)h * a.k_sh + e;
    uint16_t* vd = a.v_pool + (int64_t)page * a.v_sp + (int64_t)(pos & 15) * a.v_st + (int64_t)h * a.v_sh + e;
    if (a.vec) {
      *reinterpret_cast<u32x4*>(kd) = *reinterpret_cast<const u32x4*>(a.k_new + src);
      *reinterpret_cast<u32x4*>(vd) = *reinterpret_cast<const u32x4*>(a.v_new + src);
    } else {
      *kd = a.k_new[src];
      *vd = a.v_new[src];
    }
  }
}

}  // namespace ukv

using namespace ukv;

extern "C" int ukv_kv_write_varlen(void* k_pool_layer, void* v_pool_layer, const int64_t* k_strides,
                                   const int64_t* v_strides, const void* k_new, const void* v_new,
                                   const int64_t* new_strides, const int32_t* block_table, int max_blocks,
                                   const int32_t* cu_seqlens_q, const int32_t* kv_lens, int batch, int max_chunk,
                                   int num_heads, int head_dim, int num_pages, ukv_stream_t stream) {
  if (batch < 0 || max_chunk < 0 || num_heads <= 0 || head_dim <= 0 || max_blocks < 0) return UKV_ERR_INVALID_ARGUMENT;
  if (batch == 0 || max_chunk == 0) return UKV_OK;
  if (!k_pool_layer || !v_pool_layer || !k_strides || !v_strides || !k_new || !v_new || !new_strides ||
      !block_table || !cu_seqlens_q || !kv_lens)
    return UKV_ERR_INVALID_ARGUMENT;
  VarlenWriteArgs a{};
  a.k_pool = static_cast<uint16_t*>(k_pool_layer);
  a.v_pool = static_cast<uint16_t*>(v_pool_layer);
  a.k_sp = k_strides[0];
  a.k_st = k_strides[1];
  a.k_sh = k_strides[2];
  a.v_sp = v_strides[0];
  a.v_st = v_strides[1];
  a.v_sh = v_strides[2];
  a.k_new = static_cast<const uint16_t*>(k_new);
  a.v_new = static_cast<const uint16_t*>(v_new);
  a.n_st = new_strides[0];
  a.n_sh = new_strides[1];
  a.bt = block_table;
  a.cu_q = cu_seqlens_q;
  a.kv_lens = kv_lens;
  a.B = batch;
  a.H = num_heads;
  a.D = head_dim;
  a.max_blocks = max_blocks;
  a.num_pages = num_pages;
  a.vec = head_dim % 8 == 0 && al16(k_pool_layer) && al16(v_pool_layer) && al16(k_new) && al16(v_new) &&
          mul8(a.k_sp) && mul8(a.k_st) && mul8(a.k_sh) && mul8(a.v_sp) && mul8(a.v_st) && mul8(a.v_sh) &&
          mul8(a.n_st) && mul8(a.n_sh);
  auto log2_exact = [](int x) {
    int s = 0;
    while ((1 << s) < x) ++s;
    return (1 << s) == x ? s : -1;
  };
  a.per_shift = a.vec ? log2_exact(head_dim / 8) : -1;
  a.h_shift = log2_exact(num_heads);
  const dim3 grid((max_chunk + 15) / 16, batch);
  if (a.vec && a.per_shift >= 0 && a.h_shift >= 0)
    hipLaunchKernelGGL(kv_write_varlen_vec_kernel, grid, dim3(256), 0, reinterpret_cast<hipStream_t>(stream), a);
  else
    hipLaunchKernelGGL(kv_write_varlen_kernel, grid, dim3(256), 0, reinterpret_cast<hipStream_t>(stream), a);
  return hipGetLastError() == hipSuccess ? UKV_OK : UKV_ERR_LAUNCH;
}

namespace {

struct ObsStats {
  void* stats;
  int64_t seq_stride;
  int sink, obs;
};

template <int DT>
void launch_finish(const PrefillArgs& a, bool fine, dim3 grid, hipStream_t stream) {
  if (fine)
    hipLaunchKernelGGL((obs_rows_finish_kernel<DT, true>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((obs_rows_finish_kernel<DT, false>), grid, dim3(256), 0, stream, a);
}

void launch_tiled_any(const PrefillArgs& a, int dtype, bool fine, unsigned wgs, hipStream_t stream) {
  const bool parts = a.n_parts > 1;
  if (dtype == UKV_DTYPE_BF16)
    parts ? launch_tiled_dt<UKV_DTYPE_BF16, true>(a, fine, wgs, stream)
          : launch_tiled_dt<UKV_DTYPE_BF16, false>(a, fine, wgs, stream);
  else
    parts ? launch_tiled_dt<UKV_DTYPE_F16, true>(a, fine, wgs, stream)
          : launch_tiled_dt<UKV_DTYPE_F16, false>(a, fine, wgs, stream);
}

int prefill_impl(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table,
                 const int32_t* cu_seqlens_q, const int32_t* kv_lens, void* out, int batch, int total_q, int max_chunk,
                 int num_q_heads, int num_kv_heads, int head_dim, int n_rep, int max_blocks, int num_pages,
                 const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides, float softmax_scale,
                 int dtype, void* workspace, size_t workspace_bytes, ukv_stream_t stream_handle, const ObsStats* obs) {
  if (batch <= 0 || num_q_heads <= 0 || head_dim <= 0) return UKV_ERR_EMPTY;
  if (head_dim > 256) return UKV_ERR_HEAD_DIM;
  if (dtype != UKV_DTYPE_F16 && dtype != UKV_DTYPE_BF16) return UKV_ERR_DTYPE;
  if (num_kv_heads <= 0 || n_rep < 1) return UKV_ERR_GQA;
  const int n_groups = (num_q_heads + n_rep - 1) / n_rep;
  if (n_groups > num_kv_heads) return UKV_ERR_GQA;
  if (total_q < 0 || max_chunk < 0 || max_blocks < 0 || num_pages < 0) return UKV_ERR_INVALID_ARGUMENT;
  if (total_q == 0) return UKV_OK;
  // The chunks hold total_q queries, so the longest holds at least total_q / batch of them.
  if ((int64_t)max_chunk * batch < total_q) return UKV_ERR_INVALID_ARGUMENT;
  if (!q || !out || !cu_seqlens_q || !kv_lens || !q_strides || !k_strides || !v_strides)
    return UKV_ERR_INVALID_ARGUMENT;
  if (max_blocks > 0 && (!block_table || !k_cache || !v_cache || num_pages <= 0)) return UKV_ERR_INVALID_ARGUMENT;
  PrefillArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.out = static_cast<uint16_t*>(out);
  a.k = static_cast<const uint16_t*>(k_cache);
  a.v = static_cast<const uint16_t*>(v_cache);
  a.q_st = q_strides[0];
  a.q_sh = q_strides[1];
  a.k_sp = k_strides[0];
  a.k_st = k_strides[1];
  a.k_sh = k_strides[2];
  a.v_sp = v_strides[0];
  a.v_st = v_strides[1];
  a.v_sh = v_strides[2];
  a.bt = block_table;
  a.cu_q = cu_seqlens_q;
  a.kv_lens = kv_lens;
  a.B = batch;
  a.Hq = num_q_heads;
  a.n_rep = n_rep;
  a.n_groups = n_groups;
  a.D = head_dim;
  a.max_blocks = max_blocks;
  a.num_pages = num_pages;
  a.max_chunk = max_chunk;
  a.scale = softmax_scale;
  a.scale_log2 = softmax_scale * kLog2e;
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_handle);
  // The tiled kernel keeps a row's offset within its page in 32 bits.
  auto in_page_ok = [&](int64_t st, int64_t sh) {
    return st >= 0 && sh >= 0 && 15 * st + (int64_t)(num_kv_heads - 1) * sh + head_dim <= (int64_t)UINT32_MAX;
  };
  auto page_stride_ok = [](int64_t sp) { return sp >= 0 && sp <= (int64_t)UINT32_MAX; };
  const bool strides_ok = mul8(a.q_st) && mul8(a.q_sh) && mul8(a.k_sp) && mul8(a.k_st) && mul8(a.k_sh) &&
                          mul8(a.v_sp) && mul8(a.v_st) && mul8(a.v_sh) && in_page_ok(a.k_st, a.k_sh) &&
                          in_page_ok(a.v_st, a.v_sh) && page_stride_ok(a.k_sp) && page_stride_ok(a.v_sp);
  const bool fast = tiled_shape(head_dim, n_rep) && softmax_scale > 0.f && std::isfinite(softmax_scale) && strides_ok &&
                    al16(q) && al16(out) && al16(k_cache) && al16(v_cache) && max_blocks > 0;
  if (obs) {
    a.obs_stats = static_cast<float2*>(obs->stats);
    a.stats_seq_stride = obs->seq_stride;
    a.sink = obs->sink;
    a.obs = obs->obs;
  }
  if (fast) {
    const bool fine = fine_shape(head_dim, n_rep);
    const int64_t wgs = plan_launch(a, total_q, false, workspace, workspace_bytes);
    // The 64-dim instances write no statistics: every row is flagged, and the scoring pass recomputes
    // them from the keys.
    const int obs_rows = obs && head_dim == 64 ? a.obs : 0;
    if (obs_rows > 0) a.obs = 0;
    const int64_t finish_wgs = obs && obs_rows == 0 ? (int64_t)batch * n_groups * ((a.obs * n_rep + 15) / 16) : 0;
    if (wgs > INT32_MAX || finish_wgs > INT32_MAX) return UKV_ERR_INVALID_ARGUMENT;
    if (wgs > 0) {
      // With statistics, the prefill kernel writes the observation rows' (m, l) pairs and
      // obs_rows_finish_kernel, next on the same stream, turns them into the rows.
      launch_tiled_any(a, dtype, fine, (unsigned)wgs, stream);
    }
    if (obs_rows > 0) {
      a.obs = obs_rows;
      const int64_t flags = (int64_t)batch * num_q_heads * a.obs;
      hipLaunchKernelGGL(obs_flag_kernel, dim3((unsigned)((flags + 255) / 256)), dim3(256), 0, stream, a, flags);
    }
    if (finish_wgs > 0) {
      const dim3 fgrid((unsigned)finish_wgs);
      if (dtype == UKV_DTYPE_BF16)
        launch_finish<UKV_DTYPE_BF16>(a, fine, fgrid, stream);
      else
        launch_finish<UKV_DTYPE_F16>(a, fine, fgrid, stream);
    }
  } else {
    const dim3 grid(total_q, num_q_heads);
    if (dtype == UKV_DTYPE_BF16)
      hipLaunchKernelGGL(paged_prefill_scalar_kernel<UKV_DTYPE_BF16>, grid, dim3(256), 0, stream, a);
    else
      hipLaunchKernelGGL(paged_prefill_scalar_kernel<UKV_DTYPE_F16>, grid, dim3(256), 0, stream, a);
    // The statistics come from the tiled kernel only: here every row is flagged, and the
    // scoring pass recomputes them from the keys.
    if (obs) {
      const int64_t rows = (int64_t)batch * num_q_heads * a.obs;
      if (rows > 0)
        hipLaunchKernelGGL(obs_flag_kernel, dim3((unsigned)((rows + 255) / 256)), dim3(256), 0, stream, a, rows);
    }
  }
  return hipGetLastError() == hipSuccess ? UKV_OK : UKV_ERR_LAUNCH;
}

}  // namespace

extern "C" int ukv_paged_prefill(const void* q, const void* k_cache, const void* v_cache, const int32_t* block_table,
                                 const int32_t* cu_seqlens_q, const int32_t* kv_lens, void* out, int batch,
                                 int total_q, int max_chunk, int num_q_heads, int num_kv_heads, int head_dim,
                                 int n_rep, int max_blocks, int num_pages, const int64_t* q_strides,
                                 const int64_t* k_strides, const int64_t* v_strides, float softmax_scale,
                                 int dtype, ukv_stream_t stream_handle) {
  return prefill_impl(q, k_cache, v_cache, block_table, cu_seqlens_q, kv_lens, out, batch, total_q, max_chunk,
                      num_q_heads, num_kv_heads, head_dim, n_rep, max_blocks, num_pages, q_strides, k_strides,
                      v_strides, softmax_scale, dtype, nullptr, 0, stream_handle, nullptr);
}

extern "C" int ukv_paged_prefill_obs_stats(const void* q, const void* k_cache, const void* v_cache,
                                           const int32_t* block_table, const int32_t* cu_seqlens_q,
                                           const int32_t* kv_lens, void* out, int batch, int total_q, int max_chunk,
                                           int num_q_heads, int num_kv_heads, int head_dim, int n_rep,
                                           int max_blocks, int num_pages, const int64_t* q_strides,
                                           const int64_t* k_strides, const int64_t* v_strides,
                                           float softmax_scale, int dtype, int sink_len, int obs_len,
                                           float* obs_stats, int64_t stats_seq_stride, ukv_stream_t stream_handle) {
  if (sink_len < 0 || obs_len <= 0 || !obs_stats || (reinterpret_cast<uintptr_t>(obs_stats) & 7u) ||
      stats_seq_stride < (int64_t)num_q_heads * obs_len)
    return UKV_ERR_INVALID_ARGUMENT;
  const ObsStats st{obs_stats, stats_seq_stride, sink_len, obs_len};
  return prefill_impl(q, k_cache, v_cache, block_table, cu_seqlens_q, kv_lens, out, batch, total_q, max_chunk,
                      num_q_heads, num_kv_heads, head_dim, n_rep, max_blocks, num_pages, q_strides, k_strides,
                      v_strides, softmax_scale, dtype, nullptr, 0, stream_handle, &st);
}

extern "C" size_t ukv_paged_prefill_workspace_bytes(int batch, int total_q, int max_chunk, int num_q_heads,
                                                    int num_kv_heads, int head_dim, int n_rep, int max_blocks) {
  return parts_workspace(batch, total_q, max_chunk, num_q_heads, num_kv_heads, head_dim, n_rep, max_blocks, false);
}

extern "C" int ukv_paged_prefill_parts(const void* q, const void* k_cache, const void* v_cache,
                                       const int32_t* block_table, const int32_t* cu_seqlens_q,
                                       const int32_t* kv_lens, void* out, int batch, int total_q, int max_chunk,
                                       int num_q_heads, int num_kv_heads, int head_dim, int n_rep, int max_blocks,
                                       int num_pages, const int64_t* q_strides, const int64_t* k_strides,
                                       const int64_t* v_strides, float softmax_scale, int dtype, int sink_len,
                                       int obs_len, float* obs_stats, int64_t stats_seq_stride, void* workspace,
                                       size_t workspace_bytes, ukv_stream_t stream_handle) {
  if (obs_stats && (sink_len < 0 || obs_len <= 0 || (reinterpret_cast<uintptr_t>(obs_stats) & 7u) ||
                    stats_seq_stride < (int64_t)num_q_heads * obs_len))
    return UKV_ERR_INVALID_ARGUMENT;
  const ObsStats st{obs_stats, stats_seq_stride, sink_len, obs_len};
  return prefill_impl(q, k_cache, v_cache, block_table, cu_seqlens_q, kv_lens, out, batch, total_q, max_chunk,
                      num_q_heads, num_kv_heads, head_dim, n_rep, max_blocks, num_pages, q_strides, k_strides,
                      v_strides, softmax_scale, dtype, workspace, workspace_bytes, stream_handle,
                      obs_stats ? &st : nullptr);
}

// Chunked prefill attention over the 8-bit paged cache in shares (gfx950): longer chunks, cut by the lengths that the
// device knows.
#include "quant_shares.h"

#include "quant_rows.h"

namespace ukv {

// The batch's tiles, as the lengths on the device say, in as many equal runs as the device holds workgroups.
//
// The host's plan knows the table's width, not the sequences' lengths: whole blocks of short sequences leave their CUs
// (and, each XCD taking whole pairs, their XCDs) idle while those of the longest run on. Here the list of all tiles,
// sequence after sequence, KV group after group, query block after block, each with the tiles that its last query sees,
// is cut into G shares; a workgroup runs the pieces of blocks that its share holds, one after another. A block in one
// piece is written as by a launch without shares; the pieces of the others leave their partials (m, l, O) in two slots
// of each workgroup, and quant_shares_merge_kernel adds them up. A share's first and last pieces alone can be parts of
// blocks: slot 2 w for a piece that begins the share, 2 w + 1 for one that does not. Bound, like the tiled kernel, by
// the issue of softmax and matrix instructions, then by the partials, up to two of 200 KB a workgroup at 128 dims, and
// their merge, 15-20 us at 5 TB/s where 400 of them are full.
//
// 512 queries each behind 6324, 7670, 2480 and 2057 tokens on 28/4 heads 158 us (whole blocks 249), behind 7668 each
// 242 (261); 16 sequences' 16 drafted tokens behind 4-32K on 32/8 heads 204 us (parts 343), behind 32K each 372 (371);
// 2048 each behind 0.5-16K 1445 (2035), behind 16K each 2110 (2115; e4m3 1995 against 1950), one alone 540 (590). A table
// much wider than its sequences is what this costs most: four 512-token prompts in 2048 pages 46 us (33), unless the host
// knows the lengths too.
constexpr int kMaxShareItems = 512;  // (sequence, block) pairs of a launch
constexpr int kMinShareTiles = 12;   // tiles a share is worth a workgroup for
// What beginning a block takes, in tiles, ahead of the block's own in the list: with none 178 and 1550 us in place of the
// 158 and 1445 above, with 5 164 and 1539.
constexpr int kBlockTiles = 8;
// Wide tiles of the list, by the table's width, for each workgroup: shorter calls lose more to the pieces' starts and
// partials than even shares gain (16 x 256 queries behind 1000 tokens 128 us against 114, behind 100-2000 182 against
// 165).
constexpr int kMinSlotTiles = 128;

__device__ __forceinline__ int first_lane(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int share_start(int w, int T, int G) { return (int)((uint64_t)w * T / G); }
__device__ __forceinline__ int share_of(int x, int T, int G) { return (int)(((uint64_t)(x + 1) * G - 1) / T); }
// The largest i of [lo, hi) with starts[i] * f <= x (starts[lo] * f does).
__device__ __forceinline__ int last_at(const int* starts, int f, int x, int lo, int hi, int step) {
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first_lane(starts[mid * step]) * f <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <int DT, int D, int WAVES, int CB, bool FINE, int QF>
__global__ void __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(D == 64 ? 4 : 2)))
quant_shares_kernel(const QuantPrefillArgs a) {
  constexpr int W = WAVES * CB * 16;
  __shared__ PrefillLds<D> lds;
  __shared__ int starts[kMaxShareItems + 1];  // list entries of one KV group before (sequence, block) i
  const int tid = threadIdx.x, wave = first_lane(tid >> 6), nb = a.share_blocks, n = a.B * nb;
  int tiles = 0;
  if (tid < n) {
    const int b = tid / nb, j = tid - b * nb, C = a.cu_q[b + 1] - a.cu_q[b];
    const int cols = min(C, a.max_chunk) * a.n_rep, c1 = cols - W * j;
    if (c1 > 0) {
      const int Lk = kv_len_of(a, b), kend = min(Lk, Lk - C + (c1 + a.n_rep - 1) / a.n_rep);
      // (a row without a key is written too)
      tiles = kBlockTiles + (C > a.max_chunk ? 1 : max(1, (kend + kTileKeys - 1) / kTileKeys));
    }
  }
  static_assert(64 * WAVES == kMaxShareItems, "a thread to an item");
  const int incl = wave_inclusive_scan_i32(tiles);
  starts[tid + 1] = incl;
  if (tid == 0) starts[0] = 0;
  __syncthreads();
  int before = 0;
  for (int w = 0; w < wave; ++w) before += starts[64 * (w + 1)];
  __syncthreads();
  starts[tid + 1] = incl + before;
  __syncthreads();
  const int T = a.n_groups * first_lane(starts[n]);  // (below 2^31, checked on the host)
  const int G = T < 8 ? 1 : min((int)gridDim.x, max(8, T / kMinShareTiles & ~7));  // (no share without a tile)
  if (blockIdx.x == 0) {
    for (int i = tid; i <= n; i += 64 * WAVES) a.share_map[i] = starts[i];
    if (tid == 0) a.share_map[n + 1] = G;
  }
  if ((int)blockIdx.x >= G) return;
  const int w = (int)(blockIdx.x & 7) * (G >> 3) + (int)(blockIdx.x >> 3);  // an XCD's shares next to each other
  const int x0 = first_lane(share_start(w, T, G)), x1 = first_lane(share_start(w + 1, T, G));
  int cut = -1;  // the block that the share holds the first of several pieces of (one at most, its last)
  for (int x = x0; x < x1;) {
    const int b = last_at(starts, a.n_groups, x, 0, a.B, nb);
    const int s_b = first_lane(starts[b * nb]), u_b = first_lane(starts[(b + 1) * nb]) - s_b;
    const int g = first_lane((x - a.n_groups * s_b) / u_b), r = x - a.n_groups * s_b - g * u_b + s_b;
    const int i = last_at(starts, 1, r, b * nb, (b + 1) * nb, 1), j = i - b * nb;
    const int u0 = r - first_lane(starts[i]), all = first_lane(starts[i + 1]) - first_lane(starts[i]) - kBlockTiles;
    const int u1 = min(all + kBlockTiles, u0 + x1 - x), t0 = max(0, u0 - kBlockTiles), t1 = u1 - kBlockTiles;
    const int C = a.cu_q[b + 1] - a.cu_q[b];
    if (t1 > 0 && C <= a.max_chunk)  // (a longer chunk's rows are the merge's)
      prefill_tile<DT, D, WAVES, CB, FINE, true, QF, true>(args_again<QuantPrefillArgs>(), b, g,
                                                           C * a.n_rep - W * (j + 1), 2 * w + (x > x0),
                                                           t0 == 0 && t1 == all ? 1 : 2, lds, t0, t1, wave);
    if (t1 > 0 && t0 == 0 && t1 < all) cut = i * a.n_groups + g;
    x += u1 - u0;
    __syncthreads();  // the tiles in LDS are read
  }
  int lane;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(lane));
  const QuantPrefillArgs& e = args_again<QuantPrefillArgs>();
  if (wave == 0 && lane == 0) e.share_map[e.B * e.share_blocks + 2 + w] = cut;
}

// Workgroup w * SUB + s takes part s of the rows of the block that share w holds the first piece of, a group of D / 4
// lanes a row: with M the largest of the pieces' m, out = sum(2^(m - M) O) / sum(2^(m - M) l). Bound: HBM, where the
// partials go. The last workgroups write the chunks longer than declared.
template <int D, int W> constexpr int kMergeSub = W / (2 * (256 / (D / 4)));
template <int DT, int D, int W>
__global__ void __launch_bounds__(256) quant_shares_merge_kernel(const QuantPrefillArgs a, const int wgs) {
  constexpr int LANES = D / 4, ROWS = 256 / LANES, SUB = kMergeSub<D, W>, PER = W / SUB;
  const int w0 = blockIdx.x / SUB, sub = blockIdx.x % SUB, nb = a.share_blocks, n = a.B * nb;
  if (w0 >= wgs) {
    const int pair = blockIdx.x - wgs * SUB, b = pair / a.n_groups, C = a.cu_q[b + 1] - a.cu_q[b];
    if (C > a.max_chunk) prefill_nan_rows<4>(a, b, pair % a.n_groups, 0, C);
    return;
  }
  const int32_t* starts = a.share_map;
  const int item = starts[n + 2 + w0], T = a.n_groups * starts[n], G = starts[n + 1];
  if (w0 >= G || item < 0) return;
  const int i = item / a.n_groups, g = item - i * a.n_groups, b = i / nb, j = i - b * nb;
  const int all = starts[i + 1] - starts[i] - kBlockTiles;
  const int s_b = starts[b * nb], u_b = starts[(b + 1) * nb] - s_b;
  const int begin = a.n_groups * s_b + g * u_b + starts[i] - s_b, X = begin + kBlockTiles;  // the block, its first tile
  const int q_begin = a.cu_q[b], C = a.cu_q[b + 1] - q_begin, Lk = kv_len_of(a, b);
  const int c0 = C * a.n_rep - W * (j + 1), dq = threadIdx.x % LANES;
  const int slot0 = 2 * w0 + (begin > share_start(w0, T, G));
#pragma unroll
  for (int k = 0; k < PER / ROWS; ++k) {
    const int col = sub * PER + k * ROWS + threadIdx.x / LANES;
    const int c = c0 + col, qi = c / a.n_rep, h = g * a.n_rep + c - qi * a.n_rep;
    if (c < 0 || h >= a.Hq) continue;
    const int pos = Lk - C + qi;
    // Pieces that start at or below the row's tile: of the shares up to that of its own.
    const int n_pieces = pos < 0 ? 0 : share_of(min(X + pos / kTileKeys, X + all - 1), T, G) - w0 + 1;
    float M = kNegFltMax, l = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int p0 = 0; p0 < n_pieces; p0 += 2) {  // (two in most blocks)
      float2 ml[2];
      f32x4 o[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int p = min(p0 + u, n_pieces - 1);
        const int64_t at = (int64_t)(p == 0 ? slot0 : 2 * (w0 + p)) * W + col;
        ml[u] = a.part_ml[at];
        o[u] = *reinterpret_cast<const f32x4*>(a.part_o + at * D + 4 * dq);
        if (p0 + u >= n_pieces) ml[u] = make_float2(kNegFltMax, 0.f);
      }
      const float top = fmaxf(M, fmaxf(ml[0].x, ml[1].x));
      const float f = fast_exp2(M - top);
      l *= f;
      acc *= f;
      M = top;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (p0 + u >= n_pieces) continue;
        const float wt = fast_exp2(ml[u].x - M);
        l += wt * ml[u].y;
        acc += wt * o[u];
      }
    }
    const float inv = 1.f / l;
    const uint32_t o01 = Elem<DT>::from_float(acc[0] * inv) | (uint32_t)Elem<DT>::from_float(acc[1] * inv) << 16;
    const uint32_t o23 = Elem<DT>::from_float(acc[2] * inv) | (uint32_t)Elem<DT>::from_float(acc[3] * inv) << 16;
    *reinterpret_cast<u32x2*>(a.out + ((int64_t)(q_begin + qi) * a.Hq + h) * D + 4 * dq) = u32x2{o01, o23};
  }
}

namespace {

template <int DT, int D, int CB, bool FINE, int QF>
void launch(const QuantPrefillArgs& a, int wgs, hipStream_t stream) {
  constexpr int WV = UKV_PREFILL_WAVES;
  hipLaunchKernelGGL((quant_shares_kernel<DT, D, WV, CB, FINE, QF>), dim3(wgs), dim3(64 * WV), 0, stream, a);
  constexpr int W = WV * CB * 16;
  hipLaunchKernelGGL((quant_shares_merge_kernel<DT, D, W>), dim3(wgs * kMergeSub<D, W> + a.B * a.n_groups), dim3(256), 0,
                     stream, a, wgs);
}
template <int DT, int D, bool FINE, int QF>
void launch_blocks(const QuantPrefillArgs& a, const Shares& s, hipStream_t stream) {
  constexpr int CB = wide_blocks(FINE, D, true);
  s.column_blocks == CB ? launch<DT, D, CB, FINE, QF>(a, s.wgs, stream)
                        : launch<DT, D, CB - 1, FINE, QF>(a, s.wgs, stream);
}
template <int DT, int QF> void launch_shape(const QuantPrefillArgs& a, const Shares& s, hipStream_t stream) {
  if (a.D == 64)
    launch_blocks<DT, 64, true, QF>(a, s, stream);
  else if (fine_shape(a.D, a.n_rep))
    launch_blocks<DT, 128, true, QF>(a, s, stream);
  else
    launch_blocks<DT, 128, false, QF>(a, s, stream);
}

}  // namespace

bool shares_plan(int batch, int max_chunk, int n_groups, int head_dim, int n_rep, int max_blocks, Shares& s) {
  const int wide = wide_blocks(fine_shape(head_dim, n_rep), head_dim, true);
  const int64_t columns = (int64_t)max_chunk * n_rep, tiles = ((int64_t)max_blocks + 1) / 2;
  auto blocks_of = [&](int cb) { return (columns + UKV_PREFILL_WAVES * cb * 16 - 1) / (UKV_PREFILL_WAVES * cb * 16); };
  const double narrow = wide == 2 ? kNarrowCostFine : kNarrowCost;
  s.column_blocks = narrow * blocks_of(wide - 1) < (double)blocks_of(wide) ? wide - 1 : wide;
  const int64_t blocks = blocks_of(s.column_blocks);
  s.wgs = 8 * cus_per_xcd() * (head_dim == 64 ? 2 : 1);  // (two 64-dim workgroups share a CU)
  if (s.wgs == 0 || batch * blocks > kMaxShareItems || batch * blocks * n_groups * (tiles + kBlockTiles) > INT32_MAX)
    return false;
  const double list = (double)(batch * n_groups * blocks) * (double)(tiles + kBlockTiles) *
                      (s.column_blocks == wide ? 1.0 : narrow);
  // (With no more keys than twice the chunk's the blocks differ by a factor of two and more, and the host's plan runs
  // the longest first: 4 x 4096 tokens without a prefix 553 us, 627 in shares.)
  if (list < kMinSlotTiles * s.wgs || (int64_t)max_blocks * 16 <= 2 * (int64_t)max_chunk) return false;
  s.blocks = (int)blocks;
  const size_t rows = 2 * (size_t)s.wgs * UKV_PREFILL_WAVES * s.column_blocks * 16;
  s.ml_off = up256(rows * head_dim * sizeof(float));
  s.map_off = s.ml_off + up256(rows * sizeof(float2));
  s.total = s.map_off + up256((batch * blocks + 2 + s.wgs) * sizeof(int32_t));
  return true;
}

int launch_shares(QuantPrefillArgs a, const Shares& s, int dtype, int format, void* workspace, hipStream_t stream) {
  char* ws = static_cast<char*>(workspace);
  a.part_o = reinterpret_cast<float*>(ws);
  a.part_ml = reinterpret_cast<float2*>(ws + s.ml_off);
  a.share_map = reinterpret_cast<int32_t*>(ws + s.map_off);
  a.share_blocks = s.blocks;
  if (dtype == UKV_DTYPE_BF16)
    format == UKV_CACHE_INT8 ? launch_shape<UKV_DTYPE_BF16, UKV_CACHE_INT8>(a, s, stream)
                             : launch_shape<UKV_DTYPE_BF16, UKV_CACHE_FP8>(a, s, stream);
  else
    format == UKV_CACHE_INT8 ? launch_shape<UKV_DTYPE_F16, UKV_CACHE_INT8>(a, s, stream)
                             : launch_shape<UKV_DTYPE_F16, UKV_CACHE_FP8>(a, s, stream);
  return hipGetLastError() == hipSuccess ? UKV_OK : UKV_ERR_LAUNCH;
}

}  // namespace ukv

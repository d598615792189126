// The Page16 split decode's work cut, merge and launch arithmetic (page16_decode.hip describes them), shared by the
// 16-bit pool's kernels and the 8-bit cache's (quant_split.hip).
#pragma once

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdlib>
#include <cstring>

#include "ukv_common.h"

namespace ukv {

struct DecodeArgs {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const int32_t* bt;
  const int32_t* lens;
  uint16_t* out;
  float* part_o;     // [slots][Hq][D], slots = grid_wgs + B
  float2* part_ml;   // [slots][Hq]: (running max in log2 units, sum of exp2)
  int32_t* seq_start;  // [B] first global page of each sequence (written by workgroup 0); entry 0, whose
                       // page is 0, holds the shares the pages were cut into
  int32_t* seq_pages;  // [B] pages of each sequence
  int64_t q_sb, q_sh;
  int64_t k_sp, k_st, k_sh;
  int64_t v_sp, v_st, v_sh;
  int B, Hq, n_rep, n_groups, D, max_blocks, num_pages;
  int grid_wgs;      // workgroups sharing the batch's pages (the most shares they are cut into)
  int fixed_shares;  // cut them into exactly grid_wgs shares (launch-shape sweeps)
  int subs;          // waves of a workgroup that share each KV head's pages (split kernel, SHARED)
  // Decode-token append (fused variant): k_new/v_new [B][n_groups][D] rows with
  // strides n_sb, n_sh; the token of sequence b goes to position lens[b] - 1.
  const uint16_t* k_new;
  const uint16_t* v_new;
  int64_t n_sb, n_sh;
  float scale;       // natural-log units (scalar kernel)
  float scale_log2;  // scale * log2(e) (split kernel)
};

__device__ __forceinline__ int clamp_len(int L, int max_blocks) {
  const int cap = max_blocks * 16;
  return L < 0 ? 0 : (L > cap ? cap : L);
}

__device__ __forceinline__ int pages_of(int len, int max_blocks) { return (clamp_len(len, max_blocks) + 15) >> 4; }

// floor(x * y / z) for 0 <= x, y and 0 < z: one 32-bit division where the product fits.
__device__ __forceinline__ int mul_div(int x, int y, int z) {
  const uint64_t p = (uint64_t)(uint32_t)x * (uint32_t)y;
  if ((p >> 32) == 0) return (int)((uint32_t)p / (uint32_t)z);
  return (int)(p / (uint32_t)z);
}

// Largest of the wave's 64 values (>= 0), in every lane.
__device__ __forceinline__ int wave_max_i32(int x) {
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(x, 63);
}

// Shares the batch's P pages are cut into, at most G. The host sees the table's width alone; here the
// lengths say how much there is to share: a page more in a share costs ~0.85 us, a share more of the
// longest sequence ~0.05 us in the merge, so a share takes about sqrt(longest) / 4 pages. One sequence
// of 4096 tokens beside three of 17: 16.8 us with 72 shares, 23.9 with 256, 21.2 with 32; four of 128
// pages keep their 128 shares. A multiple of 8 (G too, or it is taken whole) for the XCDs' equal runs.
// With P >= G^2 / 16 + 2 G the rule gives G whatever the longest (a share takes at most
// sqrt(P) / 4 + 1/2 pages), and neither it nor the square root is waited for.
template <class F>
__device__ __forceinline__ int shares_for(const DecodeArgs& a, int P, F longest_pages) {
  const int many = (int)min((int64_t)INT32_MAX, (int64_t)a.grid_wgs * (a.grid_wgs + 32) / 16 + 1);
  if (a.fixed_shares || P >= many) return a.grid_wgs;
  const int longest = longest_pages();
  // (the square root is vector code: its result back to a scalar register, with all that follows from it; three
  // more vector registers would leave the 64-dim split one workgroup to a CU)
  const int per = max(1, __builtin_amdgcn_readfirstlane((int)(0.25f * __builtin_sqrtf((float)longest) + 0.5f)));
  return min(a.grid_wgs, max(8, ((P + per - 1) / per + 7) & ~7));
}

// Splits fp32 softmax weights into two 16-bit parts (p ~= hi + lo, relative
// error below 2^-16) so that P.V can run on 16-bit MFMA with fp32-grade
// weights. The fp16 path scales p by 2^7 first so small weights stay normal.
template <int DT> struct PSplit;

template <> struct PSplit<UKV_DTYPE_BF16> {
  static constexpr float kScale = 1.f;
  static __device__ __forceinline__ uint32_t pack(float x0, float x1) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x0, x1}, bf16x2));
  }
  static __device__ __forceinline__ void split(const float (&p)[4], u32x2& hi, u32x2& lo) {
    hi = u32x2{pack(p[0], p[1]), pack(p[2], p[3])};
    const float r0 = p[0] - __uint_as_float(hi[0] << 16), r1 = p[1] - __uint_as_float(hi[0] & 0xffff0000u);
    const float r2 = p[2] - __uint_as_float(hi[1] << 16), r3 = p[3] - __uint_as_float(hi[1] & 0xffff0000u);
    lo = u32x2{pack(r0, r1), pack(r2, r3)};
  }
};

template <> struct PSplit<UKV_DTYPE_F16> {
  static constexpr float kScale = 128.f;
  static __device__ __forceinline__ uint32_t pack(float x0, float x1) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x0, x1));
  }
  static __device__ __forceinline__ void split(const float (&pin)[4], u32x2& hi, u32x2& lo) {
    float p[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) p[r] = pin[r] * kScale;
    hi = u32x2{pack(p[0], p[1]), pack(p[2], p[3])};
    const float r0 = p[0] - Elem<UKV_DTYPE_F16>::lo(hi[0]), r1 = p[1] - Elem<UKV_DTYPE_F16>::hi(hi[0]);
    const float r2 = p[2] - Elem<UKV_DTYPE_F16>::lo(hi[1]), r3 = p[3] - Elem<UKV_DTYPE_F16>::hi(hi[1]);
    lo = u32x2{pack(r0, r1), pack(r2, r3)};
  }
};

#ifndef UKV_PAGE16_WAVES
#define UKV_PAGE16_WAVES 8
#endif
enum SplitMode { kSplit = 0, kShared = 1, kDirect = 2 };

// Maximum / sum over the wave's 64 lanes, in every lane (the steps of wave_inclusive_scan_i32).
#define UKV_WAVE_REDUCE(x, op, old)                                                                        \
  x = op(x, __int_as_float(__builtin_amdgcn_update_dpp(old, __float_as_int(x), 0x111, 0xf, 0xf, false))); \
  x = op(x, __int_as_float(__builtin_amdgcn_update_dpp(old, __float_as_int(x), 0x112, 0xf, 0xf, false))); \
  x = op(x, __int_as_float(__builtin_amdgcn_update_dpp(old, __float_as_int(x), 0x114, 0xf, 0xf, false))); \
  x = op(x, __int_as_float(__builtin_amdgcn_update_dpp(old, __float_as_int(x), 0x118, 0xf, 0xf, false))); \
  x = op(x, __int_as_float(__builtin_amdgcn_update_dpp(old, __float_as_int(x), 0x142, 0xa, 0xf, false))); \
  x = op(x, __int_as_float(__builtin_amdgcn_update_dpp(old, __float_as_int(x), 0x143, 0xc, 0xf, false)));
__device__ __forceinline__ float wave_max(float x) {
  UKV_WAVE_REDUCE(x, fmaxf, (int)0xff800000)  // -inf
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}
__device__ __forceinline__ float add_f32(float x, float y) { return x + y; }
__device__ __forceinline__ float wave_sum(float x) {
  UKV_WAVE_REDUCE(x, add_f32, 0)
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

// Merges the partials of one (sequence, q head): log-sum-exp in log2 units.
// The sequence's pages [S, S+n) of the batch's P pages were split over
// shares w = floor(((S+1)G - 1)/P) .. floor(((S+n)G - 1)/P), whose partials
// sit in slots w + b. 256 threads: thread (cs, dq) owns float4 dims 4*dq.. of
// partials cs, cs+CS, ...; it issues the loads of its first kPre rows together
// with the (m, l) loads, so that one memory round trip serves both. Every wave computes
// all the weights itself, with register reductions, and reads back what it wrote to LDS
// (every wave writes the same values): the one barrier is the CS partial sums' meeting in LDS.
//
// A slot holds `stride` rows of partials; the merged one is `row` of each, and goes to out_row.
template <int DT, int D>
__device__ __forceinline__ void combine_row(const DecodeArgs& a, const int b, const int64_t stride, const int64_t row,
                                            uint16_t* out_row) {
  constexpr int TD = D / 4;       // threads per partial row (float4 each)
  constexpr int CS = 256 / TD;    // chunk groups
  constexpr int kPre = 4;         // partial rows per thread loaded before the weights
  extern __shared__ float sums[];  // [CS][D] sums, then [grid_wgs] weights

  const int tid = threadIdx.x;
  const int n_pages = a.seq_pages[b];
  const int P = (a.B > 1 ? a.seq_start[a.B - 1] : 0) + a.seq_pages[a.B - 1];
  const int S = b > 0 ? a.seq_start[b] : 0;
  const int G = a.seq_start[0];
  auto share_of = [&](int x) -> int {  // floor(((x + 1) G - 1) / P): the share holding page x
    const uint64_t p = (uint64_t)(uint32_t)(x + 1) * (uint32_t)G - 1;
    return (p >> 32) == 0 ? (int)((uint32_t)p / (uint32_t)P) : (int)(p / (uint32_t)P);
  };
  const int w_first = n_pages > 0 ? share_of(S) : 0;
  const int w_last = n_pages > 0 ? share_of(S + n_pages - 1) : -1;
  const int n_chunks = w_last - w_first + 1;
  const int64_t base = (int64_t)(w_first + b) * stride + row;
  // With fewer pages than workgroups (P < G) some workgroups in [w_first, w_last]
  // own no page and wrote no partial: their slots hold stale data and are skipped.
  auto owns_pages = [&](int c) {
    const int w = w_first + c;
    return P >= G || mul_div(w + 1, P, G) > mul_div(w, P, G);
  };

  const int cs = tid / TD;
  const int dq = tid % TD;
  const float* po = a.part_o + base * D + 4 * dq;
  const int64_t cstride = stride * D;
  f32x4 rows[kPre];  // partials cs + k*CS (in the workspace even when stale; skipped below)
#pragma unroll
  for (int k = 0; k < kPre; ++k) {
    const int c = cs + k * CS;
    rows[k] = c < n_chunks ? *reinterpret_cast<const f32x4*>(po + (int64_t)c * cstride) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int lane = tid & 63;
  float* w_s = sums + CS * D;
  const bool own0 = lane < n_chunks && owns_pages(lane);
  const float2 ml0 = own0 ? a.part_ml[base + (int64_t)lane * stride] : make_float2(-INFINITY, 0.f);

  float mx = ml0.x;
  for (int c = lane + 64; c < n_chunks; c += 64)
    if (owns_pages(c)) mx = fmaxf(mx, a.part_ml[base + (int64_t)c * stride].x);
  const float M = wave_max(mx);
  float dsum = 0.f;
  for (int c = lane; c < n_chunks; c += 64) {
    const bool own = c == lane ? own0 : owns_pages(c);
    if (!own) {
      w_s[c] = -1.f;  // marks an empty slot (real weights are >= 0 or NaN)
      continue;
    }
    const float2 ml = c == lane ? ml0 : a.part_ml[base + (int64_t)c * stride];
    const float w = exp2f(ml.x - M);
    w_s[c] = w;
    dsum += ml.y * w;
  }
  const float den = wave_sum(dsum);
  // the wave's own LDS writes, by other lanes, before the reads below
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();

  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < kPre; ++k) {
    const int c = cs + k * CS;
    if (c < n_chunks) {
      const float w = w_s[c];
      if (!(w < 0.f)) acc += w * rows[k];
    }
  }
#pragma unroll 4
  for (int c = cs + kPre * CS; c < n_chunks; c += CS) {
    const float w = w_s[c];
    if (!(w < 0.f)) acc += w * *reinterpret_cast<const f32x4*>(po + (int64_t)c * cstride);
  }
  *reinterpret_cast<f32x4*>(sums + cs * D + 4 * dq) = acc;
  __syncthreads();
  if (tid < D) {
    float num = 0.f;
#pragma unroll
    for (int g = 0; g < CS; ++g) num += sums[g * D + tid];
    out_row[tid] = Elem<DT>::from_float(n_chunks > 0 ? num / den : NAN);
  }
}

template <int DT, int D>
__global__ void __launch_bounds__(256) page16_combine_kernel(const DecodeArgs a) {
  const int h = blockIdx.x, b = blockIdx.y;
  combine_row<DT, D>(a, b, a.Hq, h, a.out + ((int64_t)b * a.Hq + h) * D);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
namespace {

constexpr int kMinPagesPerWg = 4;  // below this a workgroup's setup outweighs its pages

// CU count of the current device, cached per device id (0 = not yet read; a
// racing first read stores the same value twice).
int device_cu_count() {
  static std::atomic<int> cached[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0) return 256;
  if (dev < 64) {
    const int c = cached[dev].load(std::memory_order_relaxed);
    if (c > 0) return c;
  }
  int cus = 0;
  if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) cus = 256;
  if (dev < 64) cached[dev].store(cus, std::memory_order_relaxed);
  return cus;
}

// UKV_PAGE16_WGS, read once per process (0 when unset or not a positive number).
int env_wgs() {
  static const int v = [] {
    const char* env = std::getenv("UKV_PAGE16_WGS");
    const int x = (env && *env) ? std::atoi(env) : 0;
    return x > 0 ? std::min(x, 65535) : 0;
  }();
  return v;
}

// Workgroups G sharing the batch's pages: one per CU (a single round of equal
// workgroups measured fastest), fewer when even the largest possible batch
// (batch * max_blocks pages) gives each fewer than kMinPagesPerWg pages, but one per sequence (a
// workgroup takes its segments one after another); a multiple of 8 for the XCDs' equal runs. The lengths
// may lower it on the device (shares_for). Partials
// beyond kMaxPartials bytes keep the coarser rule. UKV_PAGE16_WGS overrides it for launch-shape sweeps.
constexpr size_t kMaxPartials = size_t(16) << 20;
long long coarse_wgs(int batch, int max_blocks) {  // one per eight pages the table holds
  const long long bound = (long long)batch * (long long)std::max(max_blocks, 1);
  return std::max<long long>(1, std::min<long long>(device_cu_count(), (bound + 7) / 8));
}
long long fine_wgs(int batch, int max_blocks) {
  const long long bound = (long long)batch * (long long)std::max(max_blocks, 1);
  const long long want = std::max<long long>((bound + kMinPagesPerWg - 1) / kMinPagesPerWg, batch);
  return std::max(coarse_wgs(batch, max_blocks), std::min<long long>(device_cu_count(), (want + 7) / 8 * 8));
}
int split_wgs_for(int batch, int hq, int d, int max_blocks) {
  if (const int v = env_wgs()) return v;
  const long long g = fine_wgs(batch, max_blocks);
  const bool fits = (size_t)(g + batch) * hq * (d + 2) * sizeof(float) <= kMaxPartials;
  return (int)(fits ? g : coarse_wgs(batch, max_blocks));
}

// More KV heads than a workgroup's waves take several workgroups a share: the finer split stops where these
// fill the CUs, as a second round costs more than it spreads (4 x 4096 tokens on 16 heads of 128 dims, one
// workgroup to a CU: 26.4 us with 128 shares, 37 with 256).
int launch_wgs(int wgs, int batch, int max_blocks, int n_groups) {
  const int per_share = (n_groups + UKV_PAGE16_WAVES - 1) / UKV_PAGE16_WAVES;
  if (per_share == 1 || env_wgs()) return wgs;
  const int one_round = std::max(8, (device_cu_count() / per_share) & ~7);
  return (int)std::max<long long>(coarse_wgs(batch, max_blocks), std::min(wgs, one_round));
}

// kDirect: a CU streams at most ~47 GB/s (32 KB in flight against ~0.7 us), so a sequence on one
// workgroup per KV head pays only while its pages are few: per layer of a step at 512 tokens 7-10 us
// against 9-13 (1-8 sequences) and 14.5 / 24.7 against 19.4 / 29.3 us (32 / 64 sequences, 8 KV heads). At
// 1024 it wins where the (sequence, head) pairs fill half of the CUs (17 against 21 us at 128 pairs, 24
// against 29 at 256) and loses below (15.7 against 14.3 us at 8 x 8, 11.4 against 9.4 at 8 x 1). Pairs
// beyond the workgroups the device holds (one to a CU at 128 dims, two at 64) wait ~2.9 us a round behind
// the short sequences before a long one starts: 64 sequences on 8 heads, one of 1024 tokens among 17s, took
// 20.2 us against 15.3 for the split. There the longer tables are left to the split, and with few q heads a KV
// head, whose merge is cheap, all but the shortest (as many q heads as KV heads, one long sequence: 32 x 16 in
// 24 pages 12.6 against 11.3 us, 64 x 16 in 16 pages 16.1 against 14.5; 128 x 8 at two q heads a KV head in 32
// pages 18.4 against 16.1, in 16 pages 15 against 17; 256 x 16 one-page sequences 41 against 35).
constexpr int kDirectPages = 32, kDirectPagesWide = 64;
bool direct_shape(int batch, int n_groups, int n_rep, int head_dim, int max_blocks) {
  if (head_dim > 128 || n_groups > 65535 || env_wgs()) return false;
  const long long pairs = (long long)batch * n_groups, cus = device_cu_count();
  const long long held = head_dim == 64 ? 2 * cus : cus;
  if (max_blocks > (pairs >= cus / 2 && pairs <= cus ? kDirectPagesWide : kDirectPages)) return false;
  if (pairs <= held || n_rep >= 4 || (head_dim == 64 && n_groups <= UKV_PAGE16_WAVES)) return true;
  return pairs <= 8 * held && pairs * max_blocks <= held * (head_dim == 64 ? 48 : n_rep == 1 ? 40 : 80);
}

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

struct WorkspaceLayout {
  size_t part_o_off, part_ml_off, seq_off, total;
  int wgs;
};

// [slots][Hq][D] fp32 partials, [slots][Hq] (m, l), then the per-sequence page
// starts and counts; slots = G + batch.
WorkspaceLayout layout_of(int wgs, int batch, int hq, int d) {
  WorkspaceLayout w{};
  w.wgs = wgs;
  const size_t slots = ((size_t)w.wgs + (size_t)batch) * hq;
  w.part_o_off = 0;
  w.part_ml_off = align256(slots * d * sizeof(float));
  w.seq_off = w.part_ml_off + align256(slots * sizeof(float2));
  w.total = w.seq_off + align256(2 * (size_t)batch * sizeof(int32_t));
  return w;
}
WorkspaceLayout workspace_layout(int batch, int hq, int d, int max_blocks) {
  return layout_of(split_wgs_for(batch, hq, d, max_blocks), batch, hq, d);
}

// What the size query reports: no less than workspace_layout() takes, and never less for a larger batch,
// table or head shape, so that one buffer sized for the largest serves the smaller ones (the layout itself
// shrinks where the partials pass kMaxPartials).
size_t workspace_report(int batch, int hq, int d, int max_blocks) {
  if (env_wgs()) return workspace_layout(batch, hq, d, max_blocks).total;
  const size_t fine = layout_of((int)fine_wgs(batch, max_blocks), batch, hq, d).total;
  const size_t coarse = layout_of((int)coarse_wgs(batch, max_blocks), batch, hq, d).total;
  const size_t most_fine = kMaxPartials + 2 * 256 + align256(2 * (size_t)batch * sizeof(int32_t));  // where it fits
  return std::max(coarse, std::min(fine, most_fine));
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <int DT>
void launch_combine_dt(const DecodeArgs& a, hipStream_t stream) {
  const dim3 grid(a.Hq, a.B);
  const size_t lds = (size_t)(a.grid_wgs + 256 * 4) * sizeof(float);
  switch (a.D) {
    case 64: hipLaunchKernelGGL((page16_combine_kernel<DT, 64>), grid, dim3(256), lds, stream, a); break;
    case 128: hipLaunchKernelGGL((page16_combine_kernel<DT, 128>), grid, dim3(256), lds, stream, a); break;
    default: hipLaunchKernelGGL((page16_combine_kernel<DT, 256>), grid, dim3(256), lds, stream, a); break;
  }
}

void launch_combine(const DecodeArgs& a, int dtype, hipStream_t stream) {
  if (dtype == UKV_DTYPE_BF16)
    launch_combine_dt<UKV_DTYPE_BF16>(a, stream);
  else
    launch_combine_dt<UKV_DTYPE_F16>(a, stream);
}

}  // namespace
}  // namespace ukv

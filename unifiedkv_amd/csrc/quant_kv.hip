// Writing and reading the 8-bit paged cache, and its attention for any shape (gfx950).
//
//   ukv_quant_kv_write   16-bit rows -> codes and exponents: a prefill chunk, a decode step's tokens, dense rows
//   ukv_quant_kv_read    codes and exponents -> 16-bit rows
//   quant_rows_attention the attention of one query row and head per workgroup, for the head shapes and
//                        alignments that the matrix-core kernels do not take
//
// quant_common.h has the format.
#include <algorithm>

#include "quant_common.h"
#include "quant_rows.h"

namespace ukv {

struct QuantRowsArgs {
  QuantLayer c;
  uint16_t* rows_k;  // [rows][H][D], strides r_*
  uint16_t* rows_v;
  int64_t rk_st, rk_sh, rv_st, rv_sh;
  const int32_t* bt;
  const int32_t* cu;    // [B + 1] first row of each sequence; null: max_chunk rows each
  const int32_t* lens;  // [B] tokens of each sequence with its rows, less lens_add; null: the rows alone
  int lens_add, max_chunk, H, D, max_blocks;
  int slice;        // eight-dim chunks of a row that a workgroup takes (whole blocks; blockIdx.z: which)
  float inv_head;   // 1 / those of a head
  int wide_exps;            // sixteen tokens' exponents are one 16-byte store
};

// A sequence's rows: `first`.. of the packed ones, `count` of them, at positions `before`.. (64 bits: any length
// may come in, and none is moved into the table, where it would overwrite another token).
struct RowSpan {
  int first, count, cap;
  int64_t before;
};
__device__ __forceinline__ RowSpan span_of(const QuantRowsArgs& a, int b) {
  RowSpan s;
  s.first = a.cu ? a.cu[b] : b * a.max_chunk;
  s.count = a.cu ? a.cu[b + 1] - s.first : a.max_chunk;
  s.cap = a.max_blocks * 16;
  s.before = a.lens ? (int64_t)a.lens[b] + a.lens_add - s.count : 0;
  return s;
}
// The page of a row's position, -1 where it has none.
__device__ __forceinline__ int page_of(const QuantRowsArgs& a, const RowSpan& s, int b, int64_t pos) {
  if (pos < 0 || pos >= s.cap) return -1;
  const int id = a.bt[(int64_t)b * a.max_blocks + (pos >> 4)];
  return (unsigned)id < (unsigned)a.c.num_pages ? id : -1;
}

// The largest magnitude of eight 16-bit values as their bit pattern (patterns order like magnitudes, NaN
// above infinity).
__device__ __forceinline__ uint32_t largest_bits(const u32x4& x) {
  u16x2 m = as_u16x2(x[0] & 0x7fff7fffu);
#pragma unroll
  for (int i = 1; i < 4; ++i) m = __builtin_elementwise_max(m, as_u16x2(x[i] & 0x7fff7fffu));
  return max((uint32_t)m[0], (uint32_t)m[1]);
}

template <int DT> __device__ __forceinline__ bool finite_bits(uint32_t magnitude) {
  return magnitude < (DT == UKV_DTYPE_BF16 ? 0x7F80u : 0x7C00u);
}

#define UKV_DPP_U32(x, ctrl) (uint32_t) __builtin_amdgcn_update_dpp(0, (int)(x), (ctrl), 0xf, 0xf, false)

// Four neighbouring lanes hold a block of 32 dims, eight each: its exponent byte, and this lane's eight codes.
template <int DT, int QF> __device__ __forceinline__ uint32_t quantise8(const u32x4& x, u32x2& codes) {
  uint32_t m = largest_bits(x);
  m = max(m, UKV_DPP_U32(m, 0xB1));
  m = max(m, UKV_DPP_U32(m, 0x4E));
  if (!finite_bits<DT>(m)) {
    codes = u32x2{QuantFmt<QF>::kNanCodes, QuantFmt<QF>::kNanCodes};
    return 255u;
  }
  const int e = quant_exponent<QF>(Elem<DT>::one((uint16_t)m));
  const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
  typedef Elem<DT> E;
  codes[0] = quant_codes4<QF>({E::lo(x[0]), E::hi(x[0]), E::lo(x[1]), E::hi(x[1])}, inv);
  codes[1] = quant_codes4<QF>({E::lo(x[2]), E::hi(x[2]), E::lo(x[3]), E::hi(x[3])}, inv);
  return (uint32_t)(e + 127);
}

// The pages a sequence's rows lie on, one after another for each workgroup of the sequence: rows i0 .. i0 + n - 1 are
// on page `id` from slot `slot` on.
template <class F> __device__ __forceinline__ void for_pages(const QuantRowsArgs& a, int b, F f) {
  const RowSpan s = span_of(a, b);
  const int64_t begin = max(s.before, (int64_t)0), end = min(s.before + s.count, (int64_t)s.cap);
  for (int64_t pg = (begin >> 4) + blockIdx.x; 16 * pg < end; pg += gridDim.x) {
    const int64_t lo = max(begin, 16 * pg);
    f(page_of(a, s, b, lo), s.first + (int)(lo - s.before), (int)(min(end, 16 * pg + 16) - lo), (int)(lo & 15));
  }
}
// floor(x / n) for x < 2^20 from inv = 1 / n: (x + 1/2) / n is off the next integer by 1/2n at least.
__device__ __forceinline__ int div_small(int x, float inv) { return (int)(((float)x + 0.5f) * inv); }

// Rows of whole blocks (D a multiple of 32), 16-byte aligned: a workgroup takes a page, a thread eight dims of a (row,
// head) at a time, K and V, kAtOnce loads of both before the first is used. A page's exponents, sixteen tokens
// together, meet in LDS and go out as 16-byte stores; a part of a page's go out as bytes. Bound: HBM (reads two bytes an
// element, writes one): 8192 rows of 8 x 128 dims, K and V, in 13.4 us, 3.8 TB/s.
template <int DT, int QF>
__global__ void __launch_bounds__(256) quant_write_kernel(const QuantRowsArgs a) {
  constexpr int kAtOnce = 4;
  extern __shared__ __attribute__((aligned(16))) uint8_t exps[];  // [K, V][blocks of the slice][16]
  const int per = a.D / 8, x0 = blockIdx.z * a.slice, row = min(a.slice, a.H * per - x0), blocks = row / 4;
  const float inv_row = 1.f / (float)row;
  for_pages(a, blockIdx.y, [&](int64_t page, int r0, int n, int slot0) {
    const bool together = n == 16 && a.wide_exps;  // (uniform, as is page < 0)
    uint8_t* kp = const_cast<uint8_t*>(a.c.k) + page * a.c.k_sp;
    uint8_t* vp = const_cast<uint8_t*>(a.c.v) + page * a.c.v_sp;
    uint8_t* ke = const_cast<uint8_t*>(a.c.ks) + page * a.c.ks_sp;
    uint8_t* ve = const_cast<uint8_t*>(a.c.vs) + page * a.c.vs_sp;
    for (int base = threadIdx.x; base < n * row; base += 256 * kAtOnce) {
      u32x4 kx[kAtOnce], vx[kAtOnce];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const int it = min(base + 256 * j, n * row - 1), i = div_small(it, inv_row), x = x0 + it - i * row;
        const int h = div_small(x, a.inv_head), c = x - h * per;
        const int64_t r = r0 + i;
        kx[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(a.rows_k + r * a.rk_st + h * a.rk_sh + 8 * c));
        vx[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(a.rows_v + r * a.rv_st + h * a.rv_sh + 8 * c));
      }
      if (page < 0) return;  // (after the rows are asked for, which its id would keep waiting)
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const int it = base + 256 * j;
        if (it >= n * row) break;  // (the same in a block's four lanes)
        const int i = div_small(it, inv_row), x = x0 + it - i * row, h = div_small(x, a.inv_head), c = x - h * per;
        const int64_t slot = slot0 + i;
        u32x2 kc, vc;
        const uint32_t k_exp = quantise8<DT, QF>(kx[j], kc), v_exp = quantise8<DT, QF>(vx[j], vc);
        *reinterpret_cast<u32x2*>(kp + slot * a.c.k_st + h * a.c.k_sh + 8 * c) = kc;
        *reinterpret_cast<u32x2*>(vp + slot * a.c.v_st + h * a.c.v_sh + 8 * c) = vc;
        if ((c & 3) == 0) {
          if (together) {
            exps[(x - x0) * 4 + slot] = (uint8_t)k_exp;
            exps[(4 * blocks + x - x0) * 4 + slot] = (uint8_t)v_exp;
          } else {
            ke[h * a.c.ks_sh + (c / 4) * a.c.ks_sb + slot] = (uint8_t)k_exp;
            ve[h * a.c.vs_sh + (c / 4) * a.c.vs_sb + slot] = (uint8_t)v_exp;
          }
        }
      }
    }
    if (!together || page < 0) return;  // (a small page's other threads have not met its id yet)
    __syncthreads();
    for (int y = threadIdx.x; y < 2 * blocks; y += 256) {
      const bool is_v = y >= blocks;
      const int x = x0 / 4 + (is_v ? y - blocks : y), h = div_small(4 * x, a.inv_head), blk = x - h * (per / 4);
      uint8_t* to = is_v ? ve + h * a.c.vs_sh + blk * a.c.vs_sb : ke + h * a.c.ks_sh + blk * a.c.ks_sb;
      *reinterpret_cast<u32x4*>(to) = *reinterpret_cast<const u32x4*>(exps + 16 * y);
    }
    __syncthreads();  // read before the next page's
  });
}

// Any row: a thread takes a block of one (row, head) of K or V.
template <int DT, int QF>
__global__ void __launch_bounds__(256) quant_write_any_kernel(const QuantRowsArgs a) {
  const int b = blockIdx.y;
  const bool is_v = blockIdx.z;
  const RowSpan s = span_of(a, b);
  const int blocks = (a.D + kQuantBlock - 1) / kQuantBlock;
  const int64_t total = (int64_t)max(s.count, 0) * a.H * blocks, step = (int64_t)gridDim.x * 256;
  for (int64_t it = (int64_t)blockIdx.x * 256 + threadIdx.x; it < total; it += step) {
    const int blk = (int)(it % blocks);
    const int64_t r = it / blocks;
    const int h = (int)(r % a.H), i = (int)(r / a.H);
    const int64_t pos = s.before + i;
    const int page = page_of(a, s, b, pos);
    if (page < 0) continue;
    const int64_t slot = pos & 15;
    const int d0 = kQuantBlock * blk, n = min(kQuantBlock, a.D - d0);
    const uint16_t* x = is_v ? a.rows_v + (int64_t)(s.first + i) * a.rv_st + (int64_t)h * a.rv_sh + d0
                             : a.rows_k + (int64_t)(s.first + i) * a.rk_st + (int64_t)h * a.rk_sh + d0;
    uint8_t* codes = is_v ? const_cast<uint8_t*>(a.c.v) + page * a.c.v_sp + slot * a.c.v_st + h * a.c.v_sh + d0
                          : const_cast<uint8_t*>(a.c.k) + page * a.c.k_sp + slot * a.c.k_st + h * a.c.k_sh + d0;
    uint8_t* exps = is_v ? const_cast<uint8_t*>(a.c.vs) + page * a.c.vs_sp + h * a.c.vs_sh + blk * a.c.vs_sb + slot
                         : const_cast<uint8_t*>(a.c.ks) + page * a.c.ks_sp + h * a.c.ks_sh + blk * a.c.ks_sb + slot;
    uint32_t m = 0;
    for (int d = 0; d < n; ++d) m = max(m, (uint32_t)(x[d] & 0x7fffu));
    const bool ok = finite_bits<DT>(m);
    const int e = ok ? quant_exponent<QF>(Elem<DT>::one((uint16_t)m)) : 0;
    const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
    for (int d = 0; d < n; ++d) {
      const float f = Elem<DT>::one(x[d]);
      codes[d] = (uint8_t)(ok ? quant_codes4<QF>({f, f, f, f}, inv) : QuantFmt<QF>::kNanCodes);
    }
    *exps = (uint8_t)(ok ? e + 127 : 255);
  }
}

// Rows back from the cache, cut as the write is. A row without a page reads as zeros; rows outside the table are no
// part of any page, and the workgroups share them at the end. Bound: HBM; those 8192 rows in 10 us, 5.1 TB/s, 115708 in
// 130 us, 5.5 TB/s.
template <int DT, int QF>
__global__ void __launch_bounds__(256) quant_read_kernel(const QuantRowsArgs a) {
  constexpr int kAtOnce = 4;
  const int per = a.D / 8, x0 = blockIdx.z * a.slice, row = min(a.slice, a.H * per - x0);
  const float inv_row = 1.f / (float)row;
  auto store = [&](int64_t r, int h, int c, const u32x4& k, const u32x4& v) {
    __builtin_nontemporal_store(k, reinterpret_cast<u32x4*>(a.rows_k + r * a.rk_st + h * a.rk_sh + 8 * c));
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(a.rows_v + r * a.rv_st + h * a.rv_sh + 8 * c));
  };
  for_pages(a, blockIdx.y, [&](int64_t page, int r0, int n, int slot0) {
    const bool ok = page >= 0;  // (uniform)
    const int64_t at = ok ? page : 0;
    const uint8_t *kp = a.c.k + at * a.c.k_sp, *vp = a.c.v + at * a.c.v_sp;
    const uint8_t *ke = a.c.ks + at * a.c.ks_sp, *ve = a.c.vs + at * a.c.vs_sp;
    for (int base = threadIdx.x; base < n * row; base += 256 * kAtOnce) {
      u32x2 kc[kAtOnce] = {}, vc[kAtOnce] = {};
      uint32_t k_exp[kAtOnce] = {}, v_exp[kAtOnce] = {};
      if (ok) {
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
          const int it = min(base + 256 * j, n * row - 1), i = div_small(it, inv_row), x = x0 + it - i * row;
          const int h = div_small(x, a.inv_head), c = x - h * per;
          const int64_t slot = slot0 + i;
          kc[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(kp + slot * a.c.k_st + h * a.c.k_sh + 8 * c));
          vc[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(vp + slot * a.c.v_st + h * a.c.v_sh + 8 * c));
          k_exp[j] = ke[h * a.c.ks_sh + (c >> 2) * a.c.ks_sb + slot];
          v_exp[j] = ve[h * a.c.vs_sh + (c >> 2) * a.c.vs_sb + slot];
        }
      }
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const int it = base + 256 * j;
        if (it >= n * row) break;
        const int i = div_small(it, inv_row), x = x0 + it - i * row, h = div_small(x, a.inv_head), c = x - h * per;
        u32x4 k = {0u, 0u, 0u, 0u}, v = k;
        if (ok) {
          const float ks = quant_scale(k_exp[j]), vs = quant_scale(v_exp[j]);
          const u32x2 k0 = quant_elems4<QF, DT>(kc[j][0], ks), k1 = quant_elems4<QF, DT>(kc[j][1], ks);
          const u32x2 v0 = quant_elems4<QF, DT>(vc[j][0], vs), v1 = quant_elems4<QF, DT>(vc[j][1], vs);
          k = u32x4{k0[0], k0[1], k1[0], k1[1]};
          v = u32x4{v0[0], v0[1], v1[0], v1[1]};
        }
        store(r0 + i, h, c, k, v);
      }
    }
  });
  const RowSpan s = span_of(a, blockIdx.y);
  const u32x4 zero = {0u, 0u, 0u, 0u};
  auto clear = [&](int64_t from, int64_t to) {  // the sequence's rows from .. to - 1
    for (int64_t i = from + blockIdx.x; i < to; i += gridDim.x)
      for (int x = x0 + threadIdx.x; x < x0 + row; x += 256) {
        const int h = div_small(x, a.inv_head);
        store(s.first + i, h, x - h * per, zero, zero);
      }
  };
  clear(0, min((int64_t)s.count, -s.before));                // positions below zero
  clear(max((int64_t)0, s.cap - s.before), s.count);         // positions past the table
}

// Any row: a thread takes one element of K and V.
template <int DT, int QF>
__global__ void __launch_bounds__(256) quant_read_any_kernel(const QuantRowsArgs a) {
  const int b = blockIdx.y;
  const RowSpan s = span_of(a, b);
  const int64_t total = (int64_t)max(s.count, 0) * a.H * a.D, step = (int64_t)gridDim.x * 256;
  for (int64_t it = (int64_t)blockIdx.x * 256 + threadIdx.x; it < total; it += step) {
    const int d = (int)(it % a.D);
    const int64_t r = it / a.D;
    const int h = (int)(r % a.H), i = (int)(r / a.H);
    const int64_t pos = s.before + i;
    const int page = page_of(a, s, b, pos);
    float k = 0.f, v = 0.f;
    if (page >= 0) {
      const int64_t slot = pos & 15;
      const int blk = d / kQuantBlock;
      k = quant_one<QF>(a.c.k[page * a.c.k_sp + slot * a.c.k_st + h * a.c.k_sh + d],
                        quant_scale(a.c.ks[page * a.c.ks_sp + h * a.c.ks_sh + blk * a.c.ks_sb + slot]));
      v = quant_one<QF>(a.c.v[page * a.c.v_sp + slot * a.c.v_st + h * a.c.v_sh + d],
                        quant_scale(a.c.vs[page * a.c.vs_sp + h * a.c.vs_sh + blk * a.c.vs_sb + slot]));
    }
    a.rows_k[(int64_t)(s.first + i) * a.rk_st + (int64_t)h * a.rk_sh + d] = Elem<DT>::from_float(k);
    a.rows_v[(int64_t)(s.first + i) * a.rv_st + (int64_t)h * a.rv_sh + d] = Elem<DT>::from_float(v);
  }
}

// One workgroup per (query row, q head): natural exp, the row's keys in page order, fp32 throughout.
template <int DT, int QF>
__global__ void __launch_bounds__(256) quant_rows_kernel(const QuantAttnArgs a) {
  const int row = blockIdx.x, h = blockIdx.y;
  int b = row, first = row, count = 1;
  if (a.cu) {
    b = 0;
    while (b + 1 < a.B && a.cu[b + 1] <= row) ++b;
    first = a.cu[b];
    count = a.cu[b + 1] - first;
  }
  const int i = row - first;
  if (i < 0 || i >= count) return;
  uint16_t* out = a.out + ((int64_t)row * a.Hq + h) * a.D;
  if (a.cu && count > a.max_chunk) {  // longer than declared: its keys were not all written either
    for (int d = threadIdx.x; d < a.D; d += blockDim.x) out[d] = 0x7FFFu;
    return;
  }
  const int Lk = min(max(a.lens[b], 0), a.max_blocks * 16);
  const int L = max(0, min(Lk, Lk - count + i + 1));
  const int g = h / a.n_rep, tid = threadIdx.x, t = tid >> 4, sub = tid & 15;
  __shared__ float qs[256];
  __shared__ float ss[16];
  const uint16_t* q = a.q + (int64_t)row * a.q_st + (int64_t)h * a.q_sh;
  for (int d = tid; d < a.D; d += blockDim.x) qs[d] = Elem<DT>::one(q[d]);
  __syncthreads();
  const int d = tid;
  float m = kNegFltMax, l = 0.f, acc = 0.f;
  for (int pg = 0; pg < (L + 15) >> 4; ++pg) {
    const int id = a.bt[(int64_t)b * a.max_blocks + pg];
    const bool ok = (unsigned)id < (unsigned)a.c.num_pages;
    const int64_t page = ok ? id : 0;
    const int nv = ok ? min(16, L - 16 * pg) : 0;
    float dot = 0.f;
    if (t < nv) {
      const uint8_t* kr = a.c.k + page * a.c.k_sp + t * a.c.k_st + g * a.c.k_sh;
      const uint8_t* ke = a.c.ks + page * a.c.ks_sp + g * a.c.ks_sh + t;
      for (int dd = sub; dd < a.D; dd += 16)
        dot += quant_one<QF>(kr[dd], quant_scale(ke[(dd / kQuantBlock) * a.c.ks_sb])) * qs[dd];
    }
    dot = row_sum16(dot);
    if (sub == 0) ss[t] = dot * a.scale;
    __syncthreads();
    float mx = m;
    for (int tt = 0; tt < nv; ++tt) mx = fmaxf(mx, ss[tt]);
    const float alpha = expf(m - mx);
    l *= alpha;
    acc *= alpha;
    m = mx;
    for (int tt = 0; tt < nv; ++tt) {
      const float p = expf(ss[tt] - m);
      l += p;
      if (d < a.D)
        acc += p * quant_one<QF>(a.c.v[page * a.c.v_sp + tt * a.c.v_st + g * a.c.v_sh + d],
                                 quant_scale(a.c.vs[page * a.c.vs_sp + g * a.c.vs_sh + (d / kQuantBlock) * a.c.vs_sb + tt]));
    }
    __syncthreads();
  }
  if (d < a.D) out[d] = Elem<DT>::from_float(acc / l);
}

int quant_rows_attention(const QuantAttnArgs& a, int rows, int dtype, int format, hipStream_t stream) {
  const dim3 grid(rows, a.Hq), block(256);
  if (dtype == UKV_DTYPE_BF16 && format == UKV_CACHE_INT8)
    hipLaunchKernelGGL((quant_rows_kernel<UKV_DTYPE_BF16, UKV_CACHE_INT8>), grid, block, 0, stream, a);
  else if (dtype == UKV_DTYPE_BF16)
    hipLaunchKernelGGL((quant_rows_kernel<UKV_DTYPE_BF16, UKV_CACHE_FP8>), grid, block, 0, stream, a);
  else if (format == UKV_CACHE_INT8)
    hipLaunchKernelGGL((quant_rows_kernel<UKV_DTYPE_F16, UKV_CACHE_INT8>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((quant_rows_kernel<UKV_DTYPE_F16, UKV_CACHE_FP8>), grid, block, 0, stream, a);
  return hipGetLastError() == hipSuccess ? UKV_OK : UKV_ERR_LAUNCH;
}

QuantLayer quant_layer(const void* k, const void* v, const void* ks, const void* vs, const int64_t* s, int num_pages) {
  return QuantLayer{static_cast<const uint8_t*>(k), static_cast<const uint8_t*>(v), static_cast<const uint8_t*>(ks),
                    static_cast<const uint8_t*>(vs), s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8], s[9], s[10],
                    s[11], num_pages};
}

namespace {

bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Whether a thread's eight dims are one 16-byte access of the rows and one 8-byte access of the codes, and a page's
// exponents fit LDS (32 KB).
bool wide_rows(const QuantRowsArgs& a) {
  const int64_t rows = a.rk_st | a.rk_sh | a.rv_st | a.rv_sh;
  const int64_t codes = a.c.k_sp | a.c.k_st | a.c.k_sh | a.c.v_sp | a.c.v_st | a.c.v_sh;
  return a.D % kQuantBlock == 0 && (int64_t)a.H * a.D <= 32768 && ((rows | codes) & 7) == 0 && aligned(a.rows_k, 16) &&
         aligned(a.rows_v, 16) && aligned(a.c.k, 8) && aligned(a.c.v, 8);
}

constexpr int kSlice = 64;
constexpr int64_t kMostWgs = 1 << 16;  // (longer calls: a workgroup takes several spans of its sequence)

template <int DT, int QF> void launch_rows(QuantRowsArgs a, int batch, bool write, hipStream_t stream) {
  const int blocks = (a.D + kQuantBlock - 1) / kQuantBlock;
  if (wide_rows(a)) {
    // A workgroup a page (a chunk of n rows touches (n + 14) / 16 + 1 at most), or, where these are fewer than eight a
    // CU, a few heads of one: 8192 tokens of 8 x 128 dims written and read back in 24.4 us with two slices, 26.5 with
    // one or four.
    const unsigned x = (unsigned)std::min<int64_t>(((int64_t)a.max_chunk + 14) / 16 + 1, kMostWgs);
    const int row = a.H * (a.D / 8);
    a.slice = (int64_t)x * batch < 2048 ? std::min(row, kSlice) : row;
    const dim3 grid(x, batch, (row + a.slice - 1) / a.slice);
    if (write)
      hipLaunchKernelGGL((quant_write_kernel<DT, QF>), grid, dim3(256), 8 * a.slice, stream, a);
    else
      hipLaunchKernelGGL((quant_read_kernel<DT, QF>), grid, dim3(256), 0, stream, a);
    return;
  }
  const int64_t items = (int64_t)a.max_chunk * a.H * (write ? blocks : a.D);
  const unsigned x = (unsigned)std::min<int64_t>((items + 255) / 256, kMostWgs);
  if (write)
    hipLaunchKernelGGL((quant_write_any_kernel<DT, QF>), dim3(x, batch, 2), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((quant_read_any_kernel<DT, QF>), dim3(x, batch), dim3(256), 0, stream, a);
}

int rows_call(bool write, const void* k, const void* v, const void* ks, const void* vs, const int64_t* layer_strides,
              int num_pages, const void* rows_k, const void* rows_v, const int64_t* row_strides,
              const int32_t* block_table, int max_blocks, const int32_t* cu_seqlens, const int32_t* lens, int lens_add,
              int batch, int max_chunk, int num_heads, int head_dim, int format, int dtype, ukv_stream_t stream) {
  if (dtype != UKV_DTYPE_F16 && dtype != UKV_DTYPE_BF16) return UKV_ERR_DTYPE;
  if (format != UKV_CACHE_INT8 && format != UKV_CACHE_FP8) return UKV_ERR_DTYPE;
  if (batch < 0 || max_chunk < 0 || num_heads <= 0 || head_dim <= 0 || max_blocks < 0 || num_pages < 0)
    return UKV_ERR_INVALID_ARGUMENT;
  if (batch > 65535 || max_blocks > (INT32_MAX >> 4)) return UKV_ERR_INVALID_ARGUMENT;
  if (!cu_seqlens && (int64_t)batch * max_chunk > INT32_MAX) return UKV_ERR_INVALID_ARGUMENT;  // (rows are numbered in ints)
  if (batch == 0 || max_chunk == 0) return UKV_OK;
  if (!k || !v || !ks || !vs || !layer_strides || !rows_k || !rows_v || !row_strides) return UKV_ERR_INVALID_ARGUMENT;
  if (max_blocks > 0 && !block_table) return UKV_ERR_INVALID_ARGUMENT;
  QuantRowsArgs a{};
  a.c = quant_layer(k, v, ks, vs, layer_strides, num_pages);
  a.rows_k = static_cast<uint16_t*>(const_cast<void*>(rows_k));
  a.rows_v = static_cast<uint16_t*>(const_cast<void*>(rows_v));
  a.rk_st = row_strides[0];
  a.rk_sh = row_strides[1];
  a.rv_st = row_strides[2];
  a.rv_sh = row_strides[3];
  a.bt = block_table;
  a.cu = cu_seqlens;
  a.lens = lens;
  a.lens_add = lens_add;
  a.max_chunk = max_chunk;
  a.H = num_heads;
  a.D = head_dim;
  a.max_blocks = max_blocks;
  a.inv_head = 8.f / (float)head_dim;
  const int64_t exps = a.c.ks_sp | a.c.ks_sh | a.c.ks_sb | a.c.vs_sp | a.c.vs_sh | a.c.vs_sb;
  a.wide_exps = (exps & 15) == 0 && aligned(ks, 16) && aligned(vs, 16);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == UKV_DTYPE_BF16)
    format == UKV_CACHE_INT8 ? launch_rows<UKV_DTYPE_BF16, UKV_CACHE_INT8>(a, batch, write, s)
                             : launch_rows<UKV_DTYPE_BF16, UKV_CACHE_FP8>(a, batch, write, s);
  else
    format == UKV_CACHE_INT8 ? launch_rows<UKV_DTYPE_F16, UKV_CACHE_INT8>(a, batch, write, s)
                             : launch_rows<UKV_DTYPE_F16, UKV_CACHE_FP8>(a, batch, write, s);
  return hipGetLastError() == hipSuccess ? UKV_OK : UKV_ERR_LAUNCH;
}

// Checks and arguments that the two attention calls share; cu null: one query row a sequence.
int attention_call(const void* q, const void* k, const void* v, const void* ks, const void* vs,
                   const int64_t* layer_strides, int num_pages, const int32_t* block_table, const int32_t* cu,
                   const int32_t* lens, void* out, int batch, int rows, int max_chunk, int num_q_heads, int num_kv_heads,
                   int head_dim, int n_rep, int max_blocks, const int64_t* q_strides, float softmax_scale, int format,
                   int dtype, QuantAttnArgs& a) {
  if (batch <= 0 || num_q_heads <= 0 || head_dim <= 0) return UKV_ERR_EMPTY;
  if (head_dim > 256) return UKV_ERR_HEAD_DIM;
  if (dtype != UKV_DTYPE_F16 && dtype != UKV_DTYPE_BF16) return UKV_ERR_DTYPE;
  if (format != UKV_CACHE_INT8 && format != UKV_CACHE_FP8) return UKV_ERR_DTYPE;
  if (num_kv_heads <= 0 || n_rep < 1) return UKV_ERR_GQA;
  if ((num_q_heads + n_rep - 1) / n_rep > num_kv_heads) return UKV_ERR_GQA;
  if (max_blocks < 0 || max_blocks > (INT32_MAX >> 4) || num_pages < 0 || rows < 0 || max_chunk < 0)
    return UKV_ERR_INVALID_ARGUMENT;
  if (num_q_heads > 65535) return UKV_ERR_INVALID_ARGUMENT;
  if (!q || !out || !lens || !q_strides || !layer_strides) return UKV_ERR_INVALID_ARGUMENT;
  if (max_blocks > 0 && (!block_table || !k || !v || !ks || !vs || num_pages <= 0)) return UKV_ERR_INVALID_ARGUMENT;
  a.c = quant_layer(k, v, ks, vs, layer_strides, num_pages);
  a.q = static_cast<const uint16_t*>(q);
  a.out = static_cast<uint16_t*>(out);
  a.q_st = q_strides[0];
  a.q_sh = q_strides[1];
  a.bt = block_table;
  a.cu = cu;
  a.lens = lens;
  a.B = batch;
  a.Hq = num_q_heads;
  a.n_rep = n_rep;
  a.D = head_dim;
  a.max_blocks = max_blocks;
  a.max_chunk = max_chunk;
  a.scale = softmax_scale;
  return UKV_OK;
}

}  // namespace
}  // namespace ukv

using namespace ukv;

extern "C" int ukv_quant_kv_write(void* k, void* v, void* k_scale, void* v_scale, const int64_t* layer_strides,
                                  int num_pages, const void* k_new, const void* v_new, const int64_t* new_strides,
                                  const int32_t* block_table, int max_blocks, const int32_t* cu_seqlens,
                                  const int32_t* lens, int lens_add, int batch, int max_chunk, int num_heads,
                                  int head_dim, int format, int dtype, ukv_stream_t stream) {
  return rows_call(true, k, v, k_scale, v_scale, layer_strides, num_pages, k_new, v_new, new_strides, block_table,
                   max_blocks, cu_seqlens, lens, lens_add, batch, max_chunk, num_heads, head_dim, format, dtype, stream);
}

extern "C" int ukv_quant_kv_read(const void* k, const void* v, const void* k_scale, const void* v_scale,
                                 const int64_t* layer_strides, int num_pages, void* k_out, void* v_out,
                                 const int64_t* out_strides, const int32_t* block_table, int max_blocks,
                                 const int32_t* cu_seqlens, const int32_t* lens, int batch, int max_chunk, int num_heads,
                                 int head_dim, int format, int dtype, ukv_stream_t stream) {
  return rows_call(false, k, v, k_scale, v_scale, layer_strides, num_pages, k_out, v_out, out_strides, block_table,
                   max_blocks, cu_seqlens, lens, 0, batch, max_chunk, num_heads, head_dim, format, dtype, stream);
}

extern "C" int ukv_quant_decode(const void* q, const void* k, const void* v, const void* k_scale, const void* v_scale,
                                const int64_t* layer_strides, int num_pages, const int32_t* block_table,
                                const int32_t* seqlens, void* out, int batch, int num_q_heads, int num_kv_heads,
                                int head_dim, int n_rep, int max_blocks, const int64_t* q_strides, float softmax_scale,
                                int format, int dtype, void* workspace, size_t workspace_bytes, ukv_stream_t stream) {
  QuantAttnArgs a{};
  const int rc = attention_call(q, k, v, k_scale, v_scale, layer_strides, num_pages, block_table, nullptr, seqlens, out,
                                batch, batch, 1, num_q_heads, num_kv_heads, head_dim, n_rep, max_blocks, q_strides,
                                softmax_scale, format, dtype, a);
  if (rc != UKV_OK) return rc;
  return quant_decode(a, dtype, format, workspace, workspace_bytes, reinterpret_cast<hipStream_t>(stream));
}

extern "C" int ukv_quant_prefill(const void* q, const void* k, const void* v, const void* k_scale, const void* v_scale,
                                 const int64_t* layer_strides, int num_pages, const int32_t* block_table,
                                 const int32_t* cu_seqlens_q, const int32_t* kv_lens, void* out, int batch, int total_q,
                                 int max_chunk, int num_q_heads, int num_kv_heads, int head_dim, int n_rep,
                                 int max_blocks, const int64_t* q_strides, float softmax_scale, int format, int dtype,
                                 void* workspace, size_t workspace_bytes, ukv_stream_t stream) {
  QuantAttnArgs a{};
  if (total_q == 0 && batch > 0) return UKV_OK;
  if (!cu_seqlens_q) return UKV_ERR_INVALID_ARGUMENT;
  const int rc = attention_call(q, k, v, k_scale, v_scale, layer_strides, num_pages, block_table, cu_seqlens_q, kv_lens,
                                out, batch, total_q, max_chunk, num_q_heads, num_kv_heads, head_dim, n_rep, max_blocks,
                                q_strides, softmax_scale, format, dtype, a);
  if (rc != UKV_OK) return rc;
  // The chunks hold total_q queries, so the longest holds at least total_q / batch of them.
  if ((int64_t)max_chunk * batch < total_q) return UKV_ERR_INVALID_ARGUMENT;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  int status = UKV_OK;
  if (quant_chunk(a, dtype, format, workspace, workspace_bytes, s, status)) return status;
  return quant_prefill(a, total_q, dtype, format, workspace, workspace_bytes, s);
}

extern "C" size_t ukv_quant_prefill_workspace_bytes(int batch, int total_q, int max_chunk, int num_q_heads,
                                                    int num_kv_heads, int head_dim, int n_rep, int max_blocks) {
  if (batch <= 0 || total_q <= 0 || max_chunk <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || n_rep < 1 ||
      max_blocks <= 0)
    return 0;
  return std::max(quant_chunk_workspace(batch, num_q_heads, n_rep, head_dim, max_chunk, max_blocks),
                  quant_parts_workspace(batch, total_q, max_chunk, num_q_heads, num_kv_heads, head_dim, n_rep,
                                        max_blocks));
}

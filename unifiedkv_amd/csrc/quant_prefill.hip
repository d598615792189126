// Chunked prefill attention over the 8-bit paged cache (gfx950): the tiled kernel of paged_prefill.h, whose loader
// widens codes to the 16-bit values that they are. The tile loop is the 16-bit pool's, so is its bound, the issue of
// softmax and matrix instructions; the widening adds some thirty VALU instructions a tile of 32 keys to each thread,
// a tenth of the tile's. Long calls run in shares (quant_shares.hip), cut by the lengths that the device knows.
#include "quant_rows.h"
#include "quant_shares.h"

namespace ukv {
namespace {

template <int DT> void launch_quant(const QuantPrefillArgs& a, int format, bool fine, unsigned wgs, hipStream_t stream) {
  const bool parts = a.n_parts > 1;
  if (format == UKV_CACHE_INT8)
    parts ? launch_tiled_dt<DT, true, UKV_CACHE_INT8>(a, fine, wgs, stream)
          : launch_tiled_dt<DT, false, UKV_CACHE_INT8>(a, fine, wgs, stream);
  else
    parts ? launch_tiled_dt<DT, true, UKV_CACHE_FP8>(a, fine, wgs, stream)
          : launch_tiled_dt<DT, false, UKV_CACHE_FP8>(a, fine, wgs, stream);
}

}  // namespace

size_t quant_parts_workspace(int batch, int total_q, int max_chunk, int num_q_heads, int num_kv_heads, int head_dim,
                             int n_rep, int max_blocks) {
  if (!tiled_shape(head_dim, n_rep)) return 0;
  Shares s;
  if (shares_plan(batch, max_chunk, (num_q_heads + n_rep - 1) / n_rep, head_dim, n_rep, max_blocks, s)) return s.total;
  return parts_workspace(batch, total_q, max_chunk, num_q_heads, num_kv_heads, head_dim, n_rep, max_blocks, true);
}

// (arguments checked by the caller)
int quant_prefill(const QuantAttnArgs& x, int total_q, int dtype, int format, void* workspace, size_t workspace_bytes,
                  hipStream_t stream) {
  const QuantLayer& c = x.c;
  const int n_groups = (x.Hq + x.n_rep - 1) / x.n_rep;
  // A row's offset within its page, and the page strides, in 32 bits.
  auto in_page = [&](int64_t st, int64_t sh, int64_t rows, int64_t width) {
    return st >= 0 && sh >= 0 && (rows - 1) * st + (int64_t)(n_groups - 1) * sh + width <= (int64_t)UINT32_MAX;
  };
  auto page = [](int64_t sp) { return sp >= 0 && sp <= (int64_t)UINT32_MAX; };
  const int blocks = (x.D + kQuantBlock - 1) / kQuantBlock;
  const int64_t codes = c.k_sp | c.k_st | c.k_sh | c.v_sp | c.v_st | c.v_sh;
  auto al8 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; };
  const bool tiled = tiled_shape(x.D, x.n_rep) && x.scale > 0.f && std::isfinite(x.scale) && x.max_blocks > 0 &&
                     mul8(x.q_st) && mul8(x.q_sh) && al16(x.q) && al16(x.out) && mul8(codes) && al8(c.k) && al8(c.v) &&
                     in_page(c.k_st, c.k_sh, 16, x.D) && in_page(c.v_st, c.v_sh, 16, x.D) &&
                     in_page(c.ks_sb, c.ks_sh, blocks, 16) && in_page(c.vs_sb, c.vs_sh, blocks, 16) && page(c.k_sp) &&
                     page(c.v_sp) && page(c.ks_sp) && page(c.vs_sp);
  if (!tiled) return quant_rows_attention(x, total_q, dtype, format, stream);
  QuantPrefillArgs a{};
  a.q = x.q;
  a.out = x.out;
  a.k = reinterpret_cast<const uint16_t*>(c.k);
  a.v = reinterpret_cast<const uint16_t*>(c.v);
  a.q_st = x.q_st;
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
  a.bt = x.bt;
  a.cu_q = x.cu;
  a.kv_lens = x.lens;
  a.B = x.B;
  a.Hq = x.Hq;
  a.n_rep = x.n_rep;
  a.n_groups = n_groups;
  a.D = x.D;
  a.max_blocks = x.max_blocks;
  a.num_pages = c.num_pages;
  a.max_chunk = x.max_chunk;
  a.scale = x.scale;
  a.scale_log2 = x.scale * kLog2e;
  Shares shares;
  if (shares_plan(x.B, x.max_chunk, n_groups, x.D, x.n_rep, x.max_blocks, shares) && workspace &&
      workspace_bytes >= shares.total && al16(workspace))
    return launch_shares(a, shares, dtype, format, workspace, stream);
  const bool fine = fine_shape(x.D, x.n_rep);
  const int64_t wgs = plan_launch(a, total_q, true, workspace, workspace_bytes);
  if (wgs > INT32_MAX) return UKV_ERR_INVALID_ARGUMENT;
  if (wgs > 0)
    dtype == UKV_DTYPE_BF16 ? launch_quant<UKV_DTYPE_BF16>(a, format, fine, (unsigned)wgs, stream)
                            : launch_quant<UKV_DTYPE_F16>(a, format, fine, (unsigned)wgs, stream);
  return hipGetLastError() == hipSuccess ? UKV_OK : UKV_ERR_LAUNCH;
}

}  // namespace ukv

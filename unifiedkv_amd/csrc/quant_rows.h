// The attention over the 8-bit cache for any head shape and alignment (quant_kv.hip), which the matrix-core
// kernels' calls fall back on.
#pragma once

#include "quant_common.h"

namespace ukv {

struct QuantAttnArgs {
  QuantLayer c;
  const uint16_t* q;  // [rows][Hq][D], element strides q_st, q_sh
  uint16_t* out;      // [rows][Hq][D] contiguous
  int64_t q_st, q_sh;
  const int32_t* bt;
  const int32_t* cu;    // [B + 1] first query row of each sequence; null: row b is sequence b's one query
  const int32_t* lens;  // [B] keys of each sequence, its queries' own included
  int B, Hq, n_rep, D, max_blocks, max_chunk;
  float scale;
};

// quant_split.hip; the workspace is ukv_page16_workspace_bytes().
int quant_decode(const QuantAttnArgs& a, int dtype, int format, void* workspace, size_t workspace_bytes,
                 hipStream_t stream);

// quant_prefill.hip; the workspace (null: none) is of quant_parts_workspace() bytes.
int quant_prefill(const QuantAttnArgs& a, int total_q, int dtype, int format, void* workspace, size_t workspace_bytes,
                  hipStream_t stream);

size_t quant_parts_workspace(int batch, int total_q, int max_chunk, int num_q_heads, int num_kv_heads, int head_dim,
                             int n_rep, int max_blocks);

// quant_split.hip: chunks of a few queries. Returns whether the split kernel takes them (with this workspace, of
// quant_chunk_workspace() bytes), and then the status.
bool quant_chunk(const QuantAttnArgs& a, int dtype, int format, void* workspace, size_t workspace_bytes,
                 hipStream_t stream, int& status);
size_t quant_chunk_workspace(int batch, int hq, int n_rep, int d, int max_chunk, int max_blocks);

int quant_rows_attention(const QuantAttnArgs& a, int rows, int dtype, int format, hipStream_t stream);

}  // namespace ukv

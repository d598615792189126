// Longer chunks over the 8-bit cache in shares (quant_shares.hip).
#pragma once

#include "paged_prefill.h"

namespace ukv {

// A launch in shares: its workgroups, query blocks of a pair at most and their column blocks a wave, and where in the
// workspace the partials' (m, l) and the map of the list are.
struct Shares {
  int wgs, blocks, column_blocks;
  size_t ml_off, map_off, total;
};
// Whether a call runs in shares, and how.
bool shares_plan(int batch, int max_chunk, int n_groups, int head_dim, int n_rep, int max_blocks, Shares& s);
// `a` but for the shares' own fields; a workspace of s.total bytes, 16-byte aligned.
int launch_shares(QuantPrefillArgs a, const Shares& s, int dtype, int format, void* workspace, hipStream_t stream);

}  // namespace ukv

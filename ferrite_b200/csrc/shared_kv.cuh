// A step over a paged cache whose streams may share pages: which slot a row's keys are read through.
#pragma once
#include "api_shared.h"
#include "common.cuh"

namespace fb {

// Row of the cache that holds token j of a slot, or -1 (with a status) where the table has none.
__device__ __forceinline__ long cache_row(const FbSharedStep& st, int slot, int j, int* status) {
  const int blk = slot < 0 || slot >= st.slots || j / st.kv_block >= st.max_blocks ? -1 : st.table[(size_t)slot * st.max_blocks + j / st.kv_block];
  if (blk < 0 || blk >= st.pages) {
    set_status(status, ST_BOUNDS);
    return -1;
  }
  return (long)blk * st.kv_block + j % st.kv_block;
}
// Segment of a row, or -1; group of a segment, or -1.
__device__ __forceinline__ int segment_of_row(const FbSharedStep& st, int row) {
  for (int s = 0; s < st.nseg; ++s)
    if (row >= st.seg_row0[s] && row < st.seg_row0[s] + st.seg_nrows[s]) return s;
  return -1;
}
__device__ __forceinline__ bool group_fits(const FbSharedStep& st, int g, int* status) {
  if (st.grp_seg0[g] >= 0 && st.grp_nsegs[g] >= 0 && st.grp_nsegs[g] <= st.nseg - st.grp_seg0[g]) return true;
  set_status(status, ST_BOUNDS);
  return false;
}
__device__ __forceinline__ int group_of_segment(const FbSharedStep& st, int seg, int* status) {
  for (int g = 0; g < st.ngrp; ++g)
    if (group_fits(st, g, status) && seg >= st.grp_seg0[g] && seg < st.grp_seg0[g] + st.grp_nsegs[g]) return g;
  return -1;
}

}  // namespace fb

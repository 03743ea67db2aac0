// C launch API, fourth part: page pools that streams share (attention over a common prefix, weight of cached keys, eviction).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

// A step over a paged cache. Segments: rows row0 .. row0 + nrows of one slot. Groups: nsegs consecutive segments from seg0 on, whose rows lie side by side
// and read their first `len` tokens through the table of the first of them. Row i sees the first kvlen[i] tokens. max_rows: rows of the longest segment.
typedef struct {
  const int *seg_slot, *seg_row0, *seg_nrows;
  int nseg, max_rows;
  const int *grp_seg0, *grp_nsegs, *grp_len;
  int ngrp;
  const int* kvlen;
  int rows;
  const int* table;
  int slots, max_blocks, kv_block;
  long pages;
} FbSharedStep;

// ---- shared_attn.cu ----
// out [rows, nq * hd] bf16 and lse [rows, nq] (natural logarithm of the softmax's sum; -inf where a row sees nothing), either may be null; q: rows of nq * hd,
// q_stride elements apart; proj: gate of head h in columns h * 2 hd + hd on, or null; ws: as many floats as fb_attention_shared_floats says
long fb_attention_shared_floats(int rows, int nseg, int max_rows, int ngrp, int nq, int nkv, int hd, int ctas, int want_out);
int fb_attention_shared(void* out, float* lse, float* ws, long ws_floats, const void* q, long q_stride, const void* k, const void* v, const void* proj,
                        long proj_stride, FbSharedStep st, int nq, int nkv, int hd, int ctas, int* status, cudaStream_t s);

// ---- kv_mass.cu ----
// out[page, kv head, place] = carry * mass[..] + sum over rows and heads of exp(score - lse), for the keys of the step's contexts
// (lse null: computed); one that two spans hold sets the status. room: tokens that a table has room for; keys: tokens of the pool
long fb_attention_mass_floats(int rows, int nseg, int max_rows, int ngrp, int nq, int nkv, int hd, long room, long keys, int want_lse, int ctas);
int fb_attention_mass_launches(int rows, int nseg, int max_rows, int ngrp, int nq, int nkv, int hd, int want_lse);
int fb_attention_mass(float* out, const float* mass, float carry, const float* lse, float* ws, long ws_floats, const void* q, long q_stride, const void* k,
                      FbSharedStep st, int nq, int nkv, int hd, int ctas, int* status, cudaStream_t s);

// ---- kv_evict.cu ----
// kept [segs, nkv, keep]; k, v: rows of nkv * row_bytes bytes; scale: nkv * ns floats a row, or null; mass [pages, nkv, kv_block]; ctas: SMs
int fb_kv_evict(int* kept, void* k, void* v, float* scale, float* mass, const int* seg_slot, const int* seg_len, int segs, const int* table, int slots,
                int max_blocks, const int* dst, int dst_blocks, long pages, int kv_block, int nkv, int row_bytes, int ns, int keep, int first, int recent,
                int ctas, int* status, cudaStream_t s);

#ifdef __cplusplus
}
#endif

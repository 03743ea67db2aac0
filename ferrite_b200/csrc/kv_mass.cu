// Weight that a step's queries gave to every cached key, added up beside the cache.
#include <algorithm>

#include "shared_kv.cuh"

namespace fb {

// One CTA per (64 tokens of a group's prefix or of a segment, kv head): a warp has a key at a time and walks the rows that see it.
template <int HD>
__global__ void __launch_bounds__(256) kv_mass_kernel(float* out, const float* mass, float carry, const float* lse, const __nv_bfloat16* q, long q_stride,
                                                      const __nv_bfloat16* k, FbSharedStep st, int nq, int nkv, float scale, int* status) {
  constexpr int E = HD / 32;
  const int kvh = blockIdx.y, warp = threadIdx.x / 32, lane = threadIdx.x % 32, share = nq / nkv;
  pdl_launch_dependents();
  pdl_wait();
  const int part = blockIdx.z;
  int slot, seg0, seg1, lo, hi = 0;
  if (part < st.ngrp) {
    if (!group_fits(st, part, status) || st.grp_nsegs[part] == 0) return;
    seg0 = st.grp_seg0[part];
    seg1 = seg0 + st.grp_nsegs[part];
    slot = st.seg_slot[seg0];
    lo = 0;
    hi = st.grp_len[part];
  } else {
    seg0 = part - st.ngrp;
    seg1 = seg0 + 1;
    slot = st.seg_slot[seg0];
    const int grp = group_of_segment(st, seg0, status);
    lo = grp < 0 ? 0 : st.grp_len[grp];
    for (int r = st.seg_row0[seg0]; r < st.seg_row0[seg0] + st.seg_nrows[seg0]; ++r) hi = max(hi, st.kvlen[r]);
  }
  if (hi > (long)st.max_blocks * st.kv_block) set_status(status, ST_BOUNDS);
  hi = min((long)hi, (long)st.max_blocks * st.kv_block);
  for (int j = lo + blockIdx.x * 8 + warp; j < hi; j += gridDim.x * 8) {
    const long at = cache_row(st, slot, j, status);
    if (at < 0) continue;
    float kr[E], sum = 0.f;
    for (int e = 0; e < E; ++e) kr[e] = bf2f(k[(at * nkv + kvh) * HD + e * 32 + lane]);
    for (int s = seg0; s < seg1; ++s)
      for (int r = st.seg_row0[s]; r < st.seg_row0[s] + st.seg_nrows[s]; ++r) {
        if (st.kvlen[r] <= j) continue;
        for (int h = kvh * share; h < (kvh + 1) * share; ++h) {
          float x = 0.f;
          for (int e = 0; e < E; ++e) x += kr[e] * bf2f(q[r * q_stride + (long)h * HD + e * 32 + lane]);
          sum += expf(warp_sum(x) * scale - lse[(long)r * nq + h]);
        }
      }
    const size_t o = ((size_t)(at / st.kv_block) * nkv + kvh) * st.kv_block + at % st.kv_block;
    if (lane == 0) out[o] = (carry == 0.f ? 0.f : carry * mass[o]) + sum;
  }
}

}  // namespace fb

using namespace fb;

extern "C" long fb_attention_mass_floats(int rows, int nseg, int max_rows, int ngrp, int nq, int nkv, int ctas) {
  return ((long)rows * nq + 3) / 4 * 4 + fb_attention_shared_floats(rows, nseg, max_rows, ngrp, nq, nkv, 64, ctas, 0);
}

extern "C" int fb_attention_mass(float* out, const float* mass, float carry, const float* lse, float* ws, long ws_floats, const void* q, long q_stride,
                                 const void* k, FbSharedStep st, int nq, int nkv, int hd, int ctas, int* status, cudaStream_t s) {
  if (st.rows <= 0 || st.nseg <= 0) return 0;
  if (!lse) {
    const long used = ((long)st.rows * nq + 3) / 4 * 4;
    const int rc = fb_attention_shared(nullptr, ws, ws + used, ws_floats - used, q, q_stride, k, k, nullptr, 0, st, nq, nkv, hd, ctas, status, s);
    if (rc) return rc;
    lse = ws;
  }
  const dim3 grid(std::min(256, (st.max_blocks * st.kv_block + 7) / 8), nkv, st.ngrp + st.nseg);
  const float scale = 1.f / sqrtf((float)hd);
#define FB_KM(H)                                                                                                                                  \
  if (hd == H)                                                                                                                                    \
    return (int)launch_pdl(kv_mass_kernel<H>, grid, dim3(256), 0, s, out, mass, carry, lse, (const __nv_bfloat16*)q, q_stride,                    \
                           (const __nv_bfloat16*)k, st, nq, nkv, scale, status);
  FB_KM(64) FB_KM(128) FB_KM(256)
#undef FB_KM
  return -2;
}

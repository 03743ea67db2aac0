// Attention of a step's rows over a paged cache in which streams share the pages of a prefix.
#include "shared_kv.cuh"

namespace fb {

// One CTA per (query head, row): its warps take the keys in turn, each with a running maximum and sum.
template <int HD>
__global__ void __launch_bounds__(256) shared_attn_kernel(__nv_bfloat16* out, float* lse, const __nv_bfloat16* q, long q_stride, const __nv_bfloat16* k,
                                                          const __nv_bfloat16* v, const __nv_bfloat16* proj, long proj_stride, FbSharedStep st, int nq,
                                                          int nkv, float scale, int* status) {
  constexpr int E = HD / 32;
  __shared__ float m_s[8], l_s[8], o_s[8][HD];
  const int h = blockIdx.x, row = blockIdx.y, warp = threadIdx.x / 32, lane = threadIdx.x % 32, kvh = h / (nq / nkv);
  pdl_launch_dependents();
  pdl_wait();
  const int seg = segment_of_row(st, row);
  if (seg < 0) return;
  const int grp = group_of_segment(st, seg, status), slot = st.seg_slot[seg], shared = grp < 0 ? 0 : st.grp_len[grp];
  const int gslot = grp < 0 ? slot : st.seg_slot[st.grp_seg0[grp]];
  int n = st.kvlen[row];
  if (n > (long)st.max_blocks * st.kv_block) {
    if (threadIdx.x == 0) set_status(status, ST_BOUNDS);
    n = st.max_blocks * st.kv_block;
  }
  float qr[E], o[E], m = -INFINITY, l = 0.f;
  for (int e = 0; e < E; ++e) {
    qr[e] = bf2f(q[row * q_stride + (long)h * HD + e * 32 + lane]);
    o[e] = 0.f;
  }
  for (int j = warp; j < n; j += 8) {
    const long at = cache_row(st, j < shared ? gslot : slot, j, status);
    if (at < 0) continue;
    float x = 0.f;
    for (int e = 0; e < E; ++e) x += qr[e] * bf2f(k[(at * nkv + kvh) * HD + e * 32 + lane]);
    x = warp_sum(x) * scale;
    const float top = fmaxf(m, x), f = m == -INFINITY ? 0.f : expf(m - top), p = expf(x - top);
    for (int e = 0; e < E; ++e) o[e] = o[e] * f + p * bf2f(v[(at * nkv + kvh) * HD + e * 32 + lane]);
    l = l * f + p;
    m = top;
  }
  if (lane == 0) {
    m_s[warp] = m;
    l_s[warp] = l;
  }
  for (int e = 0; e < E; ++e) o_s[warp][e * 32 + lane] = o[e];
  __syncthreads();
  float top = -INFINITY, total = 0.f;
  for (int w = 0; w < 8; ++w) top = fmaxf(top, m_s[w]);
  for (int w = 0; w < 8; ++w) total += l_s[w] == 0.f ? 0.f : l_s[w] * expf(m_s[w] - top);
  if (out)
    for (int d = threadIdx.x; d < HD; d += 256) {
      float x = 0.f;
      for (int w = 0; w < 8; ++w) x += l_s[w] == 0.f ? 0.f : o_s[w][d] * expf(m_s[w] - top);
      x = n > 0 ? x / total : 0.f;
      if (proj) x *= sigmoidf_(bf2f(proj[row * proj_stride + (long)h * 2 * HD + HD + d]));
      out[((long)row * nq + h) * HD + d] = f2bf(x);
    }
  if (lse && threadIdx.x == 0) lse[(long)row * nq + h] = n > 0 ? top + logf(total) : -INFINITY;
}

}  // namespace fb

using namespace fb;

extern "C" long fb_attention_shared_floats(int, int, int, int, int, int, int, int, int) { return 0; }

extern "C" int fb_attention_shared(void* out, float* lse, float* ws, long ws_floats, const void* q, long q_stride, const void* k, const void* v,
                                   const void* proj, long proj_stride, FbSharedStep st, int nq, int nkv, int hd, int ctas, int* status, cudaStream_t s) {
  if (st.rows <= 0 || st.nseg <= 0) return 0;
  const float scale = 1.f / sqrtf((float)hd);
#define FB_SA(H)                                                                                                                                         \
  if (hd == H)                                                                                                                                           \
    return (int)launch_pdl(shared_attn_kernel<H>, dim3(nq, st.rows), dim3(256), 0, s, (__nv_bfloat16*)out, lse, (const __nv_bfloat16*)q, q_stride,       \
                           (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, (const __nv_bfloat16*)proj, proj_stride, st, nq, nkv, scale, status);
  FB_SA(64) FB_SA(128) FB_SA(256)
#undef FB_SA
  return -2;
}

// Attention over a latent cache in 4 or 8 bits (rows as in mla_cache.cuh), absorbed form: o = softmax(q . [value | key part] * scale) value.
// One CTA per (row, head), keys over its warps, online softmax; 32-bit arithmetic throughout.
#include "api_ext.h"
#include "mla_cache.cuh"

namespace fb {

template <int BITS, int NC>
__global__ void __launch_bounds__(128) mla_attn_q_kernel(__nv_bfloat16* __restrict__ out, const __nv_bfloat16* __restrict__ qabs,
                                                         const uint8_t* __restrict__ cache, const int* __restrict__ row_slot,
                                                         const int* __restrict__ row_kvlen, const int* __restrict__ block_table, int max_blocks,
                                                         long pages, int kv_block, int nq, float scale_log2, int* status) {
  using Row = LatentRow<BITS>;
  constexpr int L = NC * 64, D = L + LC_R;
  __shared__ float so[4][L];
  __shared__ float sml[4][2];
  const int row = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kvlen = row_kvlen[row], slot = row_slot[row];
  float qf[NC + 1][2];
  const __nv_bfloat16* qr = qabs + ((size_t)row * nq + h) * D;
#pragma unroll
  for (int j = 0; j <= NC; ++j) {
    const uint32_t u = *reinterpret_cast<const uint32_t*>(qr + 64 * j + 2 * lane);
    qf[j][0] = bf_lo(u) * scale_log2; qf[j][1] = bf_hi(u) * scale_log2;
  }
  float m = -INFINITY, l = 0.f, o[NC][2];
#pragma unroll
  for (int j = 0; j < NC; ++j) o[j][0] = o[j][1] = 0.f;
  for (int t = warp; t < kvlen; t += 4) {
    const int blk = t / kv_block < max_blocks ? block_table[(size_t)slot * max_blocks + t / kv_block] : -1;
    if (blk < 0 || blk >= pages) { set_status(status, ST_BOUNDS); continue; }
    const uint8_t* p = cache + ((size_t)blk * kv_block + t % kv_block) * Row::bytes(L);
    float v[NC][2], s;
    const uint32_t rp = *reinterpret_cast<const uint32_t*>(p + Row::rope_at(L) + 4 * lane);
    s = fmaf(qf[NC][0], bf_lo(rp), qf[NC][1] * bf_hi(rp));
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      const int e = 64 * j + 2 * lane;
      const uint32_t byte = p[Row::scale_of(L, e)];
      const float sc = latent_scale_nan<BITS>(byte) ? __uint_as_float(0x7fc00000u) : latent_scale<BITS>(byte);
      if constexpr (BITS == 4) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(p + e / 8 * 4);
        v[j][0] = sc * (float)((int)(w >> (4 * (lane % 4)) & 15u) - 8);
        v[j][1] = sc * (float)((int)(w >> (16 + 4 * (lane % 4)) & 15u) - 8);
      } else {
        const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2(*reinterpret_cast<const uint16_t*>(p + e), __NV_E4M3);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hr));
        v[j][0] = sc * f.x; v[j][1] = sc * f.y;
      }
      s = fmaf(qf[j][0], v[j][0], fmaf(qf[j][1], v[j][1], s));
    }
    s = warp_sum(s);
    const float mn = fmaxf(m, s), a = exp2f(m - mn), w = exp2f(s - mn);
    l = l * a + w;
#pragma unroll
    for (int j = 0; j < NC; ++j) {
      o[j][0] = fmaf(w, v[j][0], o[j][0] * a);
      o[j][1] = fmaf(w, v[j][1], o[j][1] * a);
    }
    m = mn;
  }
#pragma unroll
  for (int j = 0; j < NC; ++j) { so[warp][64 * j + 2 * lane] = o[j][0]; so[warp][64 * j + 2 * lane + 1] = o[j][1]; }
  if (lane == 0) { sml[warp][0] = m; sml[warp][1] = l; }
  __syncthreads();
  float M = -INFINITY, sum = 0.f;
  for (int w = 0; w < 4; ++w) M = fmaxf(M, sml[w][0]);
  float f[4];
  for (int w = 0; w < 4; ++w) {
    f[w] = sml[w][0] == -INFINITY ? (sml[w][1] == 0.f ? 0.f : __uint_as_float(0x7fc00000u)) : exp2f(sml[w][0] - M);
    sum += sml[w][1] * f[w];
  }
  for (int d = threadIdx.x; d < L; d += 128) {
    const float acc = so[0][d] * f[0] + so[1][d] * f[1] + so[2][d] * f[2] + so[3][d] * f[3];
    out[((size_t)row * nq + h) * L + d] = f2bf(kvlen > 0 ? acc / sum : 0.f);
  }
}

}  // namespace fb

using namespace fb;

extern "C" int fb_mla_attn_q(void* out, const void* qabs, const void* cache, long pages, int bits, const int* row_slot, const int* row_kvlen,
                             const int* block_table, int max_blocks, int kv_block, int rows, int nq, int L, int R, float scale, int* status,
                             cudaStream_t s) {
  if (R != LC_R || (bits != 4 && bits != 8) || nq < 1 || kv_block < 1) return -1;
  if (rows <= 0) return 0;
#define FB_LA(B, N)                                                                                                                        \
  if (bits == B && L == N * 64) {                                                                                                          \
    mla_attn_q_kernel<B, N><<<dim3(rows, nq), 128, 0, s>>>((__nv_bfloat16*)out, (const __nv_bfloat16*)qabs, (const uint8_t*)cache, row_slot, \
                                                           row_kvlen, block_table, max_blocks, pages, kv_block, nq, scale * 1.4426950408889634f, status); \
    return (int)cudaGetLastError();                                                                                                        \
  }
  FB_LA(4, 8) FB_LA(4, 4) FB_LA(4, 2) FB_LA(4, 1) FB_LA(8, 8) FB_LA(8, 4) FB_LA(8, 2) FB_LA(8, 1)
#undef FB_LA
  return -2;
}

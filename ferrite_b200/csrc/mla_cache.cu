// The latent cache of the MLA models in 4 and 8 bits (rows as in mla_cache.cuh): the step that writes it, and its rows read back in bf16.
//
//   mla_prep_q   per token: y = x / sqrt(mean x^2 + eps) * (1 + w) of the latent, quantised into the paged cache; the key part and every head's
//                query part rotated by pos * inv_freq. Norm, scale and angles are taken in 64 bits, so that a code is decided by ONE rounding, that of
//                the exact y to the code: two builds, or two ways to sum, give the same codes. (Angles in 32 bits are off by 2^-24 of themselves, which at
//                position 100000 is more than a bf16 rounding of the result.)
//   mla_rows     rows of segments (or their whole contexts) as bf16 rows [latent | key part], for the expanded form that prompts run. Values are exact.
#include "api_ext.h"
#include "mla_cache.cuh"

namespace fb {

// sine and cosine of pos * f: turns are counted and dropped in 64 bits
__device__ __forceinline__ void turn(int pos, float f, float& s, float& c) {
  double t = (double)pos * (double)f * 0.15915494309189535;
  t -= rint(t);
  sincospif((float)(2.0 * t), &s, &c);
}

// x rounded to `x` = q / 8 * 2^e, q in 8..15, halves to the even q. x > 0 and finite.
__device__ __forceinline__ void four_digits(double x, int& q, int& e) {
  const long long b = __double_as_longlong(x);
  e = (int)(b >> 52) - 1023;                                             // (a subnormal comes out as 2^-1023: the caller's range ends long before)
  q = (int)rint(__longlong_as_double((b & 0xfffffffffffffll) | 0x3ff0000000000000ll) * 8.0);
  if (q == 16) { q = 8; ++e; }
}

__device__ __forceinline__ double block_sum_f64(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double r = 0.0;
#pragma unroll
  for (int i = 0; i < 8; ++i) r += red[i];
  return r;
}

// grid (rows, 1 + groups of `per` heads), 256 threads. y = 0: the cache row, two values a thread; else the heads' query parts, four rotated pairs a thread
// (8-byte accesses), whose angles serve all of its heads.
template <int BITS>
__global__ void __launch_bounds__(256) mla_prep_q_kernel(uint8_t* __restrict__ cache, __nv_bfloat16* __restrict__ qabs, const __nv_bfloat16* kva,
                                                         long kva_stride, const __nv_bfloat16* q, long q_stride,
                                                         const __nv_bfloat16* __restrict__ norm_w, const float* __restrict__ inv_freq,
                                                         const int* row_slot, const int* row_pos, const int* block_table, int max_blocks, long pages,
                                                         int kv_block, int nq, int dn, int L, float eps, int* status, int per) {
  using Row = LatentRow<BITS>;
  constexpr int R = LC_R, half = R / 2;
  __shared__ double red[8];
  const int row = blockIdx.x, tid = threadIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  kva = after_wait(kva); q = after_wait(q);
  const int pos = after_wait(row_pos)[row];
  if (blockIdx.y > 0) {
    const int h_end = min((int)blockIdx.y * per, nq), i = tid % 8 * 4;
    float s[4], c[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) turn(pos, inv_freq[i + j], s[j], c[j]);
    for (int h = (blockIdx.y - 1) * per + tid / 8; h < h_end; h += 32) {
      const __nv_bfloat16* from = q + (size_t)row * q_stride + (size_t)h * (dn + R) + dn + i;
      __nv_bfloat16* to = qabs + ((size_t)row * nq + h) * (L + R) + L + i;
      const uint2 u = *reinterpret_cast<const uint2*>(from), v = *reinterpret_cast<const uint2*>(from + half);
      const float a[4] = {bf_lo(u.x), bf_hi(u.x), bf_lo(u.y), bf_hi(u.y)}, b[4] = {bf_lo(v.x), bf_hi(v.x), bf_lo(v.y), bf_hi(v.y)};
      float x[4], y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = fmaf(a[j], c[j], -__fmul_rn(b[j], s[j]));
        y[j] = fmaf(b[j], c[j], __fmul_rn(a[j], s[j]));
      }
      *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf2(x[0], x[1]), pack_bf2(x[2], x[3]));
      *reinterpret_cast<uint2*>(to + half) = make_uint2(pack_bf2(y[0], y[1]), pack_bf2(y[2], y[3]));
    }
    return;
  }
  const int slot = after_wait(row_slot)[row], page = pos / kv_block;
  const int blk = pos < 0 || page >= max_blocks ? -1 : after_wait(block_table)[(size_t)slot * max_blocks + page];
  if (blk < 0 || blk >= pages) {                                         // (the same for all threads)
    if (tid == 0) set_status(status, ST_BOUNDS);
    return;
  }
  uint8_t* crow = cache + ((size_t)blk * kv_block + pos % kv_block) * Row::bytes(L);
  const __nv_bfloat16* kr = kva + (size_t)row * kva_stride;
  const int e0 = tid * 2;
  const bool in = e0 < L;
  double x[2] = {0.0, 0.0};
  if (in) { x[0] = bf2f(kr[e0]); x[1] = bf2f(kr[e0 + 1]); }
  const double ss = block_sum_f64(x[0] * x[0] + x[1] * x[1], red);
  const double r = 1.0 / sqrt(ss / L + (double)eps);
  if (in) {
    double y[2], top = 0.0;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      y[j] = x[j] * r * (1.0 + (double)bf2f(norm_w[e0 + j]));
      bad |= !isfinite(y[j]);
      top = fmax(top, fabs(y[j]));                                       // (fmax drops a NaN; `bad` has it)
    }
    const unsigned here = __activemask();                                // whole warps: L is a multiple of 64
#pragma unroll
    for (int o = Row::group / 4; o > 0; o >>= 1) {
      top = fmax(top, __shfl_xor_sync(here, top, o));
      bad |= __shfl_xor_sync(here, (int)bad, o) != 0;
    }
    int byte;
    if constexpr (BITS == 4) {
      int f = 8, e = -20;
      const double want = top / 7.0;
      if (want > 0x1p-20 && !bad) {
        four_digits(want, f, e);
        if (e > 10) { f = 15; e = 10; }
      }
      byte = (e + 20) << 3 | (f - 8);
      const double scale = ldexp((double)f, e - 3);
      uint32_t w = 0;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int code = bad ? 0 : (int)fmin(fmax(rint(y[j] / scale), -7.0), 7.0);
        w |= (uint32_t)(code + 8) << (16 * j + 4 * (tid % 4));           // value 2 (tid % 4) + j of the word
      }
      w |= __shfl_xor_sync(here, w, 1);
      w |= __shfl_xor_sync(here, w, 2);
      if (tid % 4 == 0) *reinterpret_cast<uint32_t*>(crow + e0 / 2) = w;
    } else {
      int k = -15;
      const double want = top / 448.0;
      if (want > 0x1p-15 && !bad) {
        const long long b = __double_as_longlong(want);
        k = min((int)(b >> 52) - 1023 + ((b & 0xfffffffffffffll) ? 1 : 0), 7);
      }
      byte = k + 127;
      const double inv = ldexp(1.0, -k);
      uint32_t w = 0;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        // rounded to odd on the way to 32 bits, so that the rounding to e4m3 is the only one
        const double v = bad ? 0.0 : y[j] * inv;
        float f = __double2float_rz(v);
        if ((double)f != v) f = __uint_as_float(__float_as_uint(f) | 1u);
        w |= (uint32_t)__nv_cvt_float_to_fp8(f, __NV_SATFINITE, __NV_E4M3) << (8 * j);
      }
      *reinterpret_cast<uint16_t*>(crow + e0) = (uint16_t)w;
    }
    if (e0 % Row::group == 0) crow[Row::scale_of(L, e0)] = (uint8_t)(bad ? LC_NAN : byte);
  }
  if (tid < half) {
    float s, c;
    turn(pos, inv_freq[tid], s, c);
    const float a = bf2f(kr[L + tid]), b = bf2f(kr[L + half + tid]);
    __nv_bfloat16* to = reinterpret_cast<__nv_bfloat16*>(crow + Row::rope_at(L)) + tid;
    to[0] = f2bf(fmaf(a, c, -__fmul_rn(b, s)));
    to[half] = f2bf(fmaf(b, c, __fmul_rn(a, s)));
  }
  const int end = Row::scale_at(L) + L / Row::group;
  if (tid < Row::bytes(L) - end) crow[end + tid] = 0;
}

constexpr int LR_ROWS = 16;            // output rows of a CTA

// grid ceil(rows / LR_ROWS), 288 threads: eight values of a row a thread. Output rows: segment after segment, each from a multiple of `align` on; `whole`:
// positions 0 .. pos0 + nrows of a segment, else its own rows pos0 .. pos0 + nrows. Rows between them are zeros.
template <int BITS>
__global__ void __launch_bounds__(288) mla_rows_kernel(__nv_bfloat16* __restrict__ out, long rows, const uint8_t* cache, const int* seg_slot,
                                                       const int* seg_pos0, const int* seg_nrows, int nseg, const int* block_table, int max_blocks,
                                                       long pages, int kv_block, int L, int whole, int align, int* status) {
  using Row = LatentRow<BITS>;
  __shared__ const uint8_t* from[LR_ROWS];
  const int tid = threadIdx.x;
  const long r0 = (long)blockIdx.x * LR_ROWS;
  pdl_launch_dependents();
  pdl_wait();
  cache = after_wait(cache); seg_slot = after_wait(seg_slot); seg_pos0 = after_wait(seg_pos0); seg_nrows = after_wait(seg_nrows);
  block_table = after_wait(block_table);
  if (tid < LR_ROWS) {
    long at = r0 + tid;
    const uint8_t* p = nullptr;
    for (int s = 0; s < nseg; ++s) {
      const int pos0 = seg_pos0[s], n = seg_nrows[s], count = max(whole ? pos0 + n : n, 0);
      const long room = ((long)count + align - 1) / align * align;
      if (at >= room) { at -= room; continue; }
      if (at < count) {
        const long pos = whole ? at : pos0 + at, page = pos / kv_block;
        const int blk = pos < 0 || page >= max_blocks ? -1 : block_table[(size_t)seg_slot[s] * max_blocks + page];
        if (blk < 0 || blk >= pages) set_status(status, ST_BOUNDS);
        else p = cache + ((size_t)blk * kv_block + pos % kv_block) * Row::bytes(L);
      }
      break;
    }
    from[tid] = p;
  }
  __syncthreads();
  const int units = (L + LC_R) / 8;
  for (int i = tid; i < LR_ROWS * units; i += blockDim.x) {
    const int r = i / units, u = i % units;
    if (r0 + r >= rows) break;
    const uint8_t* p = from[r];
    uint4 v = make_uint4(0, 0, 0, 0);
    if (p && u * 8 >= L) {
      v = *reinterpret_cast<const uint4*>(p + Row::rope_at(L) + (u * 8 - L) * 2);
    } else if (p) {
      const uint32_t byte = p[Row::scale_of(L, u * 8)];
      const float sc = latent_scale_nan<BITS>(byte) ? __uint_as_float(0x7fc00000u) : latent_scale<BITS>(byte);
      uint32_t* o = reinterpret_cast<uint32_t*>(&v);
      if constexpr (BITS == 4) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(p + u * 4);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          o[j] = pack_bf2(sc * (float)((int)(w >> (4 * j) & 15u) - 8), sc * (float)((int)(w >> (16 + 4 * j) & 15u) - 8));
      } else {
        const uint2 w = *reinterpret_cast<const uint2*>(p + u * 8);
        const uint32_t ww[2] = {w.x, w.y};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(ww[j / 2] >> (16 * (j % 2))), __NV_E4M3);
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
          o[j] = pack_bf2(sc * f.x, sc * f.y);
        }
      }
    }
    *reinterpret_cast<uint4*>(out + (r0 + r) * (L + LC_R) + u * 8) = v;
  }
}

}  // namespace fb

using namespace fb;

static bool latent_shape_ok(int L, int R, int bits) { return R == LC_R && L >= 64 && L <= LC_MAX_L && L % 64 == 0 && (bits == 4 || bits == 8); }

extern "C" int fb_latent_row_bytes(int L, int R, int bits) { return latent_shape_ok(L, R, bits) ? latent_row_bytes(L, bits) : -1; }

extern "C" int fb_mla_prep_q(void* cache, long pages, int bits, void* qabs, const void* kva, long kva_stride, const void* q, long q_stride,
                             const void* norm_w, const float* inv_freq, const int* row_slot, const int* row_pos, const int* block_table,
                             int max_blocks, int kv_block, int rows, int nq, int dn, int L, int R, float eps, int* status, cudaStream_t s) {
  if (!latent_shape_ok(L, R, bits) || nq < 1 || dn < 0 || kv_block < 1) return -1;
  if (dn % 4 || q_stride % 4 || ((uintptr_t)q | (uintptr_t)qabs) % 8 || (uintptr_t)cache % 16) return -2;
  if (rows <= 0) return 0;
  // heads a CTA: 32 (one pass of the threads) as long as the SMs hold all CTAs at once, else all heads of a row, whose angles are then taken once
  const int per = (long)rows * (1 + (nq + 31) / 32) <= 8 * 148 ? 32 : 128;
  auto kern = bits == 4 ? mla_prep_q_kernel<4> : mla_prep_q_kernel<8>;
  return (int)launch_pdl(kern, dim3(rows, 1 + (nq + per - 1) / per), dim3(256), (size_t)0, s, (uint8_t*)cache, (__nv_bfloat16*)qabs,
                         (const __nv_bfloat16*)kva, kva_stride, (const __nv_bfloat16*)q, q_stride, (const __nv_bfloat16*)norm_w, inv_freq, row_slot,
                         row_pos, block_table, max_blocks, pages, kv_block, nq, dn, L, eps, status, per);
}

extern "C" int fb_mla_rows(void* out, long rows, const void* cache, long pages, int bits, const int* seg_slot, const int* seg_pos0, const int* seg_nrows,
                           int nseg, const int* block_table, int max_blocks, int kv_block, int L, int R, int whole, int align, int* status,
                           cudaStream_t s) {
  if (!latent_shape_ok(L, R, bits) || kv_block < 1 || align < 1) return -1;
  if (((uintptr_t)out | (uintptr_t)cache) % 16) return -2;
  if (rows <= 0) return 0;
  auto kern = bits == 4 ? mla_rows_kernel<4> : mla_rows_kernel<8>;
  return (int)launch_pdl(kern, dim3((unsigned)((rows + LR_ROWS - 1) / LR_ROWS)), dim3(288), (size_t)0, s, (__nv_bfloat16*)out, rows,
                         (const uint8_t*)cache, seg_slot, seg_pos0, seg_nrows, nseg, block_table, max_blocks, pages, kv_block, L, whole, align, status);
}

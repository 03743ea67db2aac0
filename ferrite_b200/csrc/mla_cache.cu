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

constexpr int LP_ROWS = 8, LP_HEADS = 128;             // cache rows, heads of a CTA

// grid ceil(rows / LP_ROWS) + rows * kinds, kinds: groups of LP_HEADS heads, 256 threads. The first CTAs write cache rows, a warp each: 16 values a lane (the
// 64-bit square root and quotients of a row are then worked out once, not by eight warps: 2048 rows 36 -> 25 us with their reading back). The others turn
// the heads' query parts of a row, four pairs a thread (8-byte accesses), whose angles serve all of its heads (groups of 32 heads: 34 us); queries are on
// their way before the position is known. 2048 rows of 128 heads take 15 us by the profiler's clock (17 captured, cold caches) where the queries' 67 MB are 10
// at the copy rate. It is not the bytes (DRAM 32 % busy) but the chain of a row's CTA, four a SM and four waves of them: of a warp's 12.9 cycles between
// instructions 3.9 go to the barrier behind the 32 threads that turn the angles in 64 bits, 2.0 to loads; a quarter of the time SMs start or run dry.
template <int BITS>
__global__ void __launch_bounds__(256, 4) mla_prep_q_kernel(uint8_t* __restrict__ cache, __nv_bfloat16* __restrict__ qabs, const __nv_bfloat16* kva,
                                                         long kva_stride, const __nv_bfloat16* q, long q_stride,
                                                         const __nv_bfloat16* __restrict__ norm_w, const float* __restrict__ inv_freq,
                                                         const int* row_slot, const int* row_pos, const int* block_table, int max_blocks, long pages,
                                                         int kv_block, int nq, int dn, int L, double eps, int* status, int rows, int kinds) {
  using Row = LatentRow<BITS>;
  constexpr int R = LC_R, half = R / 2;
  const int tid = threadIdx.x, lane = tid & 31, writers = (rows + LP_ROWS - 1) / LP_ROWS, turner = (int)blockIdx.x - writers;
  pdl_launch_dependents();
  pdl_wait();
  kva = after_wait(kva); q = after_wait(q);
  if (turner >= 0) {
    const int row = turner / kinds, kind = turner % kinds, h0 = kind * LP_HEADS + tid / 8, h_end = min((kind + 1) * LP_HEADS, nq), i = tid % 8 * 4;
    const int pos = after_wait(row_pos)[row];
    const __nv_bfloat16* from = q + (size_t)row * q_stride + dn + i;
    uint2 u[4], v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (h0 + 32 * k < h_end) {
        u[k] = *reinterpret_cast<const uint2*>(from + (size_t)(h0 + 32 * k) * (dn + R));
        v[k] = *reinterpret_cast<const uint2*>(from + (size_t)(h0 + 32 * k) * (dn + R) + half);
      }
    __shared__ __align__(16) float sn[half], cs[half];
    if (tid < half) turn(pos, inv_freq[tid], sn[tid], cs[tid]);
    __syncthreads();
    const float4 s4 = *reinterpret_cast<const float4*>(sn + i), c4 = *reinterpret_cast<const float4*>(cs + i);
    const float s[4] = {s4.x, s4.y, s4.z, s4.w}, c[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int h = h0 + 32 * k;
      if (h >= h_end) break;
      __nv_bfloat16* to = qabs + ((size_t)row * nq + h) * (L + R) + L + i;
      const float a[4] = {bf_lo(u[k].x), bf_hi(u[k].x), bf_lo(u[k].y), bf_hi(u[k].y)}, b[4] = {bf_lo(v[k].x), bf_hi(v[k].x), bf_lo(v[k].y), bf_hi(v[k].y)};
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
  const int row = blockIdx.x * LP_ROWS + (tid >> 5);
  if (row >= rows) return;
  const int pos = after_wait(row_pos)[row], slot = after_wait(row_slot)[row], page = pos / kv_block;
  const __nv_bfloat16* kr = kva + (size_t)row * kva_stride;
  const int e0 = lane * 16;
  const bool in = e0 < L;
  uint4 xu[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)}, wu[2] = {xu[0], xu[0]};
  if (in) {
    auto take = [&](uint4 (&u)[2], const __nv_bfloat16* p) {             // 16 values, by 16 bytes where they lie so
      if ((uintptr_t)p % 16 == 0) {
        u[0] = reinterpret_cast<const uint4*>(p)[0];
        u[1] = reinterpret_cast<const uint4*>(p)[1];
      } else {
        const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
        uint32_t* o = reinterpret_cast<uint32_t*>(u);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = h[2 * j] | (uint32_t)h[2 * j + 1] << 16;
      }
    };
    take(xu, kr + e0);
    take(wu, norm_w + e0);
  }
  const float ka = bf2f(kr[L + lane]), kb = bf2f(kr[L + half + lane]);
  const int blk = pos < 0 || page >= max_blocks ? -1 : after_wait(block_table)[(size_t)slot * max_blocks + page];
  if (blk < 0 || blk >= pages) {                                         // (the same for the whole warp)
    if (lane == 0) set_status(status, ST_BOUNDS);
    return;
  }
  uint8_t* crow = cache + ((size_t)blk * kv_block + pos % kv_block) * Row::bytes(L);
  const uint32_t* xw = reinterpret_cast<const uint32_t*>(xu);
  const uint32_t* ww = reinterpret_cast<const uint32_t*>(wu);
  double ss = 0.0;
#pragma unroll
  for (int j = 0; j < 8; ++j) ss += (double)bf_lo(xw[j]) * bf_lo(xw[j]) + (double)bf_hi(xw[j]) * bf_hi(xw[j]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const double r = 1.0 / sqrt(ss / L + eps);
  double y[16], top = 0.0;
  bool bad = false;
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    y[j] = (double)(j % 2 ? bf_hi(xw[j / 2]) : bf_lo(xw[j / 2])) * r * (1.0 + (double)(j % 2 ? bf_hi(ww[j / 2]) : bf_lo(ww[j / 2])));
    bad |= !isfinite(y[j]);
    top = fmax(top, fabs(y[j]));                                         // (fmax drops a NaN; `bad` has it)
  }
  if constexpr (BITS == 8) {                                             // a group is two lanes'
    top = fmax(top, __shfl_xor_sync(0xffffffffu, top, 1));
    bad |= __shfl_xor_sync(0xffffffffu, (int)bad, 1) != 0;
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
    const double scale = ldexp((double)f, e - 3), inv = 1.0 / scale;
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      // the product is off by 2^-51 of itself: only next to a half does it take the quotient
      const double t = y[j] * inv;
      double c = rint(t);
      if (fabs(fabs(t - c) - 0.5) < 1e-9) c = rint(y[j] / scale);
      const int code = bad ? 0 : (int)fmin(fmax(c, -7.0), 7.0);
      w[j / 8] |= (uint32_t)(code + 8) << (16 * (j % 2) + 4 * (j % 8 / 2));
    }
    if (in) *reinterpret_cast<uint2*>(crow + lane * 8) = make_uint2(w[0], w[1]);
  } else {
    int k = -15;
    const double want = top / 448.0;
    if (want > 0x1p-15 && !bad) {
      const long long b = __double_as_longlong(want);
      k = min((int)(b >> 52) - 1023 + ((b & 0xfffffffffffffll) ? 1 : 0), 7);
    }
    byte = k + 127;
    const double inv = ldexp(1.0, -k);
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      // rounded to odd on the way to 32 bits, so that the rounding to e4m3 is the only one
      const double v = bad ? 0.0 : y[j] * inv;
      float f = __double2float_rz(v);
      if ((double)f != v) f = __uint_as_float(__float_as_uint(f) | 1u);
      w[j / 4] |= (uint32_t)__nv_cvt_float_to_fp8(f, __NV_SATFINITE, __NV_E4M3) << (8 * (j % 4));
    }
    if (in) *reinterpret_cast<uint4*>(crow + e0) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  if (in && e0 % Row::group == 0) crow[Row::scale_of(L, e0)] = (uint8_t)(bad ? LC_NAN : byte);
  float s, c;
  turn(pos, inv_freq[lane], s, c);
  __nv_bfloat16* to = reinterpret_cast<__nv_bfloat16*>(crow + Row::rope_at(L)) + lane;
  to[0] = f2bf(fmaf(ka, c, -__fmul_rn(kb, s)));
  to[half] = f2bf(fmaf(kb, c, __fmul_rn(ka, s)));
  const int end = Row::scale_at(L) + L / Row::group;
  if (lane < Row::bytes(L) - end) crow[end + lane] = 0;
}

constexpr int LR_ROWS = 16, LR_THREADS = 288;                            // output rows of a CTA at most

// grid ceil(rows / per), 288 threads: eight values of a row a thread. Output rows: segment after segment, each from a multiple of `align` on; `whole`:
// positions 0 .. pos0 + nrows of a segment, else its own rows pos0 .. pos0 + nrows. Rows between them are zeros. Bound by bytes: 13111 rows of 416 in,
// 1152 out, 20 MB, 10 us with cold caches (3 at the copy rate); few rows by four dependent loads, 5 us.
template <int BITS>
__global__ void __launch_bounds__(LR_THREADS) mla_rows_kernel(__nv_bfloat16* __restrict__ out, long rows, const uint8_t* cache, const int* seg_slot,
                                                              const int* seg_pos0, const int* seg_nrows, int nseg, const int* block_table,
                                                              int max_blocks, long pages, int kv_block, int L, int whole, int align, int* status,
                                                              int per) {
  using Row = LatentRow<BITS>;
  __shared__ const uint8_t* from[LR_ROWS];
  const int tid = threadIdx.x;
  const long r0 = (long)blockIdx.x * per;
  pdl_launch_dependents();
  pdl_wait();
  cache = after_wait(cache); seg_slot = after_wait(seg_slot); seg_pos0 = after_wait(seg_pos0); seg_nrows = after_wait(seg_nrows);
  block_table = after_wait(block_table);
  if (tid < 32) {
    // a lane a segment, 32 at a time: where each ends; then a lane a row looks its own up
    const bool mine = tid < per;
    const long at = r0 + tid;
    long base = 0;
    bool found = false;
    const uint8_t* p = nullptr;
    for (int s0 = 0; s0 < nseg; s0 += 32) {
      const bool there = s0 + tid < nseg;
      const int pos0 = there ? seg_pos0[s0 + tid] : 0, n = there ? seg_nrows[s0 + tid] : 0, slot = there ? seg_slot[s0 + tid] : 0;
      const int count = max(whole && there ? pos0 + n : n, 0);
      long end = align == 1 ? count : (long)((uint32_t)(count + align - 1) / (uint32_t)align) * align;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long v = __shfl_up_sync(0xffffffffu, end, o);
        if (tid >= o) end += v;
      }
      end += base;
      int k = 0;                                                         // the first segment that ends behind the row, if it is one of these
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        if (__shfl_sync(0xffffffffu, end, k + o - 1) <= at) k += o;
      const long stop = __shfl_sync(0xffffffffu, end, k), room_before = __shfl_up_sync(0xffffffffu, end, 1);
      const long start = __shfl_sync(0xffffffffu, tid == 0 ? base : room_before, k);
      const int c = __shfl_sync(0xffffffffu, count, k), q0 = __shfl_sync(0xffffffffu, pos0, k), sl = __shfl_sync(0xffffffffu, slot, k);
      if (mine && !found && at < stop) {
        found = true;
        if (at - start < c) {
          const int pos = (int)(at - start) + (whole ? 0 : q0), page = pos < 0 ? -1 : (int)((uint32_t)pos / (uint32_t)kv_block);
          const int blk = page < 0 || page >= max_blocks ? -1 : block_table[(size_t)sl * max_blocks + page];
          if (blk < 0 || blk >= pages) set_status(status, ST_BOUNDS);
          else p = cache + ((size_t)blk * kv_block + (pos - page * kv_block)) * Row::bytes(L);
        }
      }
      base = __shfl_sync(0xffffffffu, end, 31);
      if (base > r0 + per - 1) break;
    }
    if (mine) from[tid] = p;
  }
  __syncthreads();
  const int units = (L + LC_R) / 8, step = LR_THREADS / units, u = tid % units;
  if (tid >= step * units) return;
#pragma unroll 4
  for (int r = tid / units; r < per; r += step) {
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
                             int max_blocks, int kv_block, int rows, int nq, int dn, int L, int R, double eps, int* status, cudaStream_t s) {
  if (!latent_shape_ok(L, R, bits) || nq < 1 || dn < 0 || kv_block < 1) return -1;
  if (dn % 4 || q_stride % 4 || ((uintptr_t)q | (uintptr_t)qabs) % 8 || (uintptr_t)cache % 16) return -2;
  if (rows <= 0) return 0;
  const int kinds = (nq + LP_HEADS - 1) / LP_HEADS;
  if ((long)rows * (kinds + 1) > 0x7fffffffl) return -2;
  auto kern = bits == 4 ? mla_prep_q_kernel<4> : mla_prep_q_kernel<8>;
  return (int)launch_pdl(kern, dim3((rows + LP_ROWS - 1) / LP_ROWS + rows * kinds), dim3(256), (size_t)0, s, (uint8_t*)cache, (__nv_bfloat16*)qabs,
                         (const __nv_bfloat16*)kva, kva_stride, (const __nv_bfloat16*)q, q_stride, (const __nv_bfloat16*)norm_w, inv_freq, row_slot,
                         row_pos, block_table, max_blocks, pages, kv_block, nq, dn, L, eps, status, rows, kinds);
}

extern "C" int fb_mla_rows(void* out, long rows, const void* cache, long pages, int bits, const int* seg_slot, const int* seg_pos0, const int* seg_nrows,
                           int nseg, const int* block_table, int max_blocks, int kv_block, int L, int R, int whole, int align, int* status,
                           cudaStream_t s) {
  if (!latent_shape_ok(L, R, bits) || kv_block < 1 || align < 1) return -1;
  if (((uintptr_t)out | (uintptr_t)cache) % 16) return -2;
  if (rows <= 0) return 0;
  // rows a CTA: the fewest of 4, 8 and 16 with which the SMs hold all CTAs at once (2048 rows read back: 2 us less than with 16; 13111: 2 us less than with 4)
  int per = 4;
  while (per < LR_ROWS && (rows + per - 1) / per > 148 * (2048 / LR_THREADS)) per *= 2;
  auto kern = bits == 4 ? mla_rows_kernel<4> : mla_rows_kernel<8>;
  return (int)launch_pdl(kern, dim3((unsigned)((rows + per - 1) / per)), dim3(LR_THREADS), (size_t)0, s, (__nv_bfloat16*)out, rows,
                         (const uint8_t*)cache, seg_slot, seg_pos0, seg_nrows, nseg, block_table, max_blocks, pages, kv_block, L, whole, align, status, per);
}

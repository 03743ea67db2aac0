// Eviction from a paged cache by accumulated weight: which tokens of a (stream, kv head) stay, and their move into new pages.
#include <algorithm>

#include "api_shared.h"
#include "common.cuh"

namespace fb {

// Order of weights as whole numbers: larger first means larger number; no number counts as the largest, -0 as 0.
__device__ __forceinline__ uint32_t weight_order(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct EvictArgs {
  int* kept;
  unsigned char *k, *v;
  float *scale, *mass;
  const int *seg_slot, *seg_len, *table, *dst;
  int segs, slots, max_blocks, dst_blocks;
  long pages;
  int kv_block, nkv, row_bytes, ns, keep, first, recent;
  int* status;
};

// tokens in the slot's cache, as far as its table reaches
__device__ __forceinline__ int evict_len(const EvictArgs& a, int seg) {
  const int slot = a.seg_slot[seg];
  int n = a.seg_len[seg];
  if (slot < 0 || slot >= a.slots || n > (long)a.max_blocks * a.kv_block) {
    set_status(a.status, ST_BOUNDS);
    n = slot < 0 || slot >= a.slots ? 0 : a.max_blocks * a.kv_block;
  }
  return max(n, 0);
}
__device__ __forceinline__ int checked_page(const EvictArgs& a, int page) {
  if (page >= 0 && page < a.pages) return page;
  set_status(a.status, ST_BOUNDS);
  return -1;
}

// One CTA per (segment, kv head): the weight of the last one kept digit by digit, then the tokens in order.
__global__ void __launch_bounds__(1024) kv_select_kernel(EvictArgs a) {
  __shared__ uint32_t hist[256], scan[2][32], st_s[2];
  const int seg = blockIdx.x / a.nkv, h = blockIdx.x % a.nkv, t = threadIdx.x, warp = t / 32, lane = t % 32;
  pdl_launch_dependents();
  pdl_wait();
  const int n = evict_len(a, seg), slot = a.seg_slot[seg];
  int* kept = a.kept + (size_t)blockIdx.x * a.keep;
  const int m = min(n, a.keep);
  for (int i = m + t; i < a.keep; i += 1024) kept[i] = -1;
  if (n <= a.keep) {
    for (int i = t; i < n; i += 1024) kept[i] = i;
    return;
  }
  auto order = [&](int j) -> uint32_t {
    const int page = checked_page(a, a.table[(size_t)slot * a.max_blocks + j / a.kv_block]);
    return page < 0 ? 0u : weight_order(a.mass[((size_t)page * a.nkv + h) * a.kv_block + j % a.kv_block]);
  };
  const int lo = a.first, hi = n - a.recent;
  uint32_t need = a.keep - a.first - a.recent, prefix = 0, mask = 0;
  for (int shift = 24; shift >= 0 && need; shift -= 8) {
    if (t < 256) hist[t] = 0;
    __syncthreads();
    for (int j = lo + t; j < hi; j += 1024) {
      const uint32_t u = order(j);
      if ((u & mask) == prefix) atomicAdd(&hist[u >> shift & 255], 1u);
    }
    __syncthreads();
    if (t == 0) {
      int d = 255;
      uint32_t left = need;
      while (hist[d] < left) left -= hist[d--];
      st_s[0] = d;
      st_s[1] = left;
    }
    __syncthreads();
    prefix |= st_s[0] << shift;
    mask |= 255u << shift;
    need = st_s[1];
    __syncthreads();
  }
  // need: how many tokens of the weight `prefix` stay, the first ones
  const bool none = a.keep == a.first + a.recent;
  uint32_t equal = 0, at = 0;
  for (int j0 = 0; j0 < n; j0 += 1024) {
    const int j = j0 + t;
    const bool always = j < n && (j < lo || j >= hi);
    const uint32_t u = j < n && !always ? order(j) : 0;
    const bool eq = j < n && !always && !none && u == prefix, more = j < n && !always && !none && u > prefix;
    auto place = [&](bool p, int b) -> uint32_t {                   // set ones ahead of this thread; scan[b][31]: all of them
      const uint32_t bal = __ballot_sync(0xffffffffu, p);
      if (lane == 0) scan[b][warp] = __popc(bal);
      __syncthreads();
      if (warp == 0) {
        uint32_t x = scan[b][lane];
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        scan[b][lane] = x;
      }
      __syncthreads();
      return (warp ? scan[b][warp - 1] : 0) + __popc(bal & ((1u << lane) - 1));
    };
    const uint32_t e = equal + place(eq, 0);
    const bool stay = always || more || (eq && e < need);
    const uint32_t p = at + place(stay, 1);
    if (stay) kept[p] = j;
    equal += scan[0][31];
    at += scan[1][31];
    __syncthreads();
  }
}

// A warp per kept row: keys, values, scales and weight into the new page.
__global__ void __launch_bounds__(256) kv_compact_kernel(EvictArgs a) {
  const int lane = threadIdx.x % 32;
  pdl_launch_dependents();
  pdl_wait();
  const int* kept = a.kept;
  const long rows = (long)a.segs * a.nkv * a.keep;
  for (long i = (long)blockIdx.x * 8 + threadIdx.x / 32; i < rows; i += (long)gridDim.x * 8) {
    const int j = kept[i];
    if (j < 0) continue;
    const int to = (int)(i % a.keep), h = (int)(i / a.keep % a.nkv), seg = (int)(i / a.keep / a.nkv), slot = a.seg_slot[seg];
    const int src = checked_page(a, a.table[(size_t)slot * a.max_blocks + j / a.kv_block]);
    const int dst = checked_page(a, a.dst[(size_t)seg * a.dst_blocks + to / a.kv_block]);
    if (src < 0 || dst < 0) continue;
    const size_t r0 = ((size_t)src * a.kv_block + j % a.kv_block) * a.nkv + h, r1 = ((size_t)dst * a.kv_block + to % a.kv_block) * a.nkv + h;
    for (int b = lane * 4; b < a.row_bytes; b += 128) {
      *reinterpret_cast<uint32_t*>(a.k + r1 * a.row_bytes + b) = *reinterpret_cast<const uint32_t*>(a.k + r0 * a.row_bytes + b);
      *reinterpret_cast<uint32_t*>(a.v + r1 * a.row_bytes + b) = *reinterpret_cast<const uint32_t*>(a.v + r0 * a.row_bytes + b);
    }
    if (a.scale && lane < a.ns) a.scale[r1 * a.ns + lane] = a.scale[r0 * a.ns + lane];
    if (lane == 0)
      a.mass[((size_t)dst * a.nkv + h) * a.kv_block + to % a.kv_block] = a.mass[((size_t)src * a.nkv + h) * a.kv_block + j % a.kv_block];
  }
}

}  // namespace fb

using namespace fb;

extern "C" int fb_kv_evict(int* kept, void* k, void* v, float* scale, float* mass, const int* seg_slot, const int* seg_len, int segs, const int* table,
                           int slots, int max_blocks, const int* dst, int dst_blocks, long pages, int kv_block, int nkv, int row_bytes, int ns, int keep,
                           int first, int recent, int* status, cudaStream_t s) {
  if (segs <= 0) return 0;
  if (keep < 1 || first < 0 || recent < 0 || (long)first + recent > keep || (long)dst_blocks * kv_block < keep || row_bytes % 16 || ns > 32) return -1;
  const EvictArgs a{kept, (unsigned char*)k, (unsigned char*)v, scale, mass, seg_slot, seg_len, table, dst, segs, slots, max_blocks, dst_blocks, pages,
                    kv_block, nkv, row_bytes, ns, keep, first, recent, status};
  cudaError_t e = launch_pdl(kv_select_kernel, dim3(segs * nkv), dim3(1024), 0, s, a);
  if (e != cudaSuccess) return (int)e;
  return (int)launch_pdl(kv_compact_kernel, dim3((unsigned)std::min(148l * 8, ((long)segs * nkv * keep + 7) / 8)), dim3(256), 0, s, a);
}

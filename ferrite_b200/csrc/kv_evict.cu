// Eviction from a paged cache by accumulated weight: which tokens of a (stream, kv head) stay, and their move into new pages.
//
// A cluster of CTAs has a (segment, kv head), each CTA a run of its tokens. The weight of the last token that stays is found digit by digit, 11, 11 and 10
// bits of the weights as whole numbers in their order: a histogram per CTA in shared memory, added up over the cluster. How many heavier tokens and how
// many equal ones lie ahead of a token says whether it stays and where it goes (the earliest of equal ones stay), so the order of the tokens is kept without
// a sort, and nothing depends on the order in which threads run. Then the cluster copies the rows, 32 of them a warp at a time: the lanes look up the pages, then all of
// them copy one row after another, 16 bytes each. What bounds it is the copy: 512-byte rows from all over the pool.
#include <algorithm>
#include <cooperative_groups.h>

#include "api_shared.h"
#include "common.cuh"

namespace fb {

namespace cg = cooperative_groups;
constexpr int EV_THREADS = 512, EV_WARPS = EV_THREADS / 32, EV_BINS = 2048, EV_HELD = 44 << 10;   // weights that a CTA holds in shared memory

// Order of weights as whole numbers: a larger weight is a larger number; no number counts as the largest, -0 as 0.
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
  int held, row_lanes;                           // weights that fit; lanes that copy a row together (a power of two)
  int* status;
};

__device__ __forceinline__ int checked_page(const EvictArgs& a, int page) {
  if (page >= 0 && page < a.pages) return page;
  set_status(a.status, ST_BOUNDS);
  return -1;
}
// Sums of what lies ahead of a thread (low and high half apart), and of all; tmp: a place for each warp.
__device__ __forceinline__ uint64_t scan_pairs(uint64_t mine, uint64_t* tmp, uint64_t* all) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) tmp[warp] = x;
  __syncthreads();
  uint64_t ahead = x - mine, sum = 0;
#pragma unroll
  for (int w = 0; w < EV_WARPS; ++w) {
    if (w < warp) ahead += tmp[w];
    sum += tmp[w];
  }
  *all = sum;
  return ahead;
}

__global__ void __launch_bounds__(EV_THREADS, 2) kv_evict_kernel(EvictArgs a) {
  extern __shared__ uint32_t held_s[];
  __shared__ uint32_t hist[EV_BINS], total[EV_BINS];
  __shared__ uint64_t tmp[EV_WARPS], counts_s;
  __shared__ uint32_t digit_s[2];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks(), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int pair = blockIdx.x / ctas, seg = pair / a.nkv, h = pair % a.nkv;
  pdl_launch_dependents();
  pdl_wait();
  const int slot = a.seg_slot[seg];
  int n = max(a.seg_len[seg], 0);
  if (slot < 0 || slot >= a.slots || n > (long)a.max_blocks * a.kv_block) {
    set_status(a.status, ST_BOUNDS);
    n = slot < 0 || slot >= a.slots ? 0 : a.max_blocks * a.kv_block;
  }
  const int* table = a.table + (size_t)max(slot, 0) * a.max_blocks;
  int* kept = a.kept + (size_t)pair * a.keep;
  const int m = min(n, a.keep);
  for (int i = m + rank * EV_THREADS + tid; i < a.keep; i += ctas * EV_THREADS) kept[i] = -1;
  if (n <= a.keep) {
    for (int i = rank * EV_THREADS + tid; i < n; i += ctas * EV_THREADS) kept[i] = i;
  } else {
    // ---- this CTA's tokens
    const int per = (n + ctas - 1) / ctas, t0 = min(n, rank * per), t1 = min(n, t0 + per), lo = a.first, hi = n - a.recent;
    const bool hold = per <= a.held;
    auto order = [&](int j) -> uint32_t {
      const int page = checked_page(a, table[j / a.kv_block]);
      return page < 0 ? 0u : weight_order(a.mass[((size_t)page * a.nkv + h) * a.kv_block + j % a.kv_block]);
    };
    uint32_t need = (uint32_t)(a.keep - a.first - a.recent), prefix = 0, mask = 0;
    const bool none = need == 0;
    if (hold && !none)
#pragma unroll 4
      for (int j = max(t0, lo) + tid; j < min(t1, hi); j += EV_THREADS) held_s[j - t0] = order(j);
    for (int pass = 0; pass < 3 && !none; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const uint32_t bins = pass == 2 ? 1024u : 2048u;
      for (int i = tid; i < EV_BINS; i += EV_THREADS) hist[i] = 0;
      __syncthreads();
      for (int j = max(t0, lo) + tid; j < min(t1, hi); j += EV_THREADS) {
        const uint32_t u = hold ? held_s[j - t0] : order(j);
        if ((u & mask) == prefix) atomicAdd(&hist[u >> shift & (bins - 1)], 1u);
      }
      cluster.sync();
      for (int i = tid; i < EV_BINS; i += EV_THREADS) {
        uint32_t sum = 0;
        for (int c = 0; c < ctas; ++c) sum += cluster.map_shared_rank(hist, c)[i];
        total[i] = sum;
      }
      __syncthreads();
      // bins from the top, four a thread
      uint32_t mine = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) mine += total[EV_BINS - 1 - 4 * tid - e];
      uint64_t all;
      uint32_t ahead = (uint32_t)scan_pairs(mine, tmp, &all);
      if (ahead < need && need <= ahead + mine) {
        int d = EV_BINS - 1 - 4 * tid;
        while (ahead + total[d] < need) ahead += total[d--];
        digit_s[0] = (uint32_t)d;
        digit_s[1] = need - ahead;
      }
      cluster.sync();                                                // (also: nobody reads these histograms any more)
      prefix |= digit_s[0] << shift;
      mask |= (bins - 1) << shift;
      need = digit_s[1];
    }
    // need: how many tokens of the weight `prefix` stay. A thread has neighbouring tokens: how many stay for sure (low half) and equal ones (high half)
    const int each = (t1 - t0 + EV_THREADS - 1) / EV_THREADS, j0 = min(t1, t0 + tid * each), j1 = min(t1, j0 + each);
    auto kind = [&](int j) -> uint64_t {
      if (j < lo || j >= hi) return 1;
      if (none) return 0;
      const uint32_t u = hold ? held_s[j - t0] : order(j);
      return u > prefix ? 1ull : u == prefix ? 1ull << 32 : 0ull;
    };
    uint64_t mine = 0, all;
    for (int j = j0; j < j1; ++j) mine += kind(j);
    uint64_t ahead = scan_pairs(mine, tmp, &all);
    if (tid == 0) counts_s = all;
    cluster.sync();
    for (int c = 0; c < rank; ++c) ahead += *cluster.map_shared_rank(&counts_s, c);
    for (int j = j0; j < j1; ++j) {
      const uint64_t k = kind(j);
      const uint32_t sure = (uint32_t)ahead, equal = (uint32_t)(ahead >> 32), at = sure + min(equal, need);
      if (k == 1 || (k && equal < need)) kept[at] = j;
      ahead += k;
    }
  }
  __threadfence();
  cluster.sync();                                                    // the list is complete
  // ---- the copy
  const int rows0 = (int)((long)m * rank / ctas), rows1 = (int)((long)m * (rank + 1) / ctas), pieces = a.row_bytes / 16, L = a.row_lanes;
  for (int i0 = rows0 + warp * 32; i0 < rows1; i0 += EV_THREADS) {
    const int i = i0 + lane;
    long from = -1, to = -1;
    if (i < rows1) {
      int j = *reinterpret_cast<volatile int*>(kept + i);
      const int src = checked_page(a, table[j / a.kv_block]), dst = checked_page(a, a.dst[(size_t)seg * a.dst_blocks + i / a.kv_block]);
      if (src >= 0 && dst >= 0) {
        from = ((long)src * a.kv_block + j % a.kv_block) * a.nkv + h;
        to = ((long)dst * a.kv_block + i % a.kv_block) * a.nkv + h;
        a.mass[((size_t)dst * a.nkv + h) * a.kv_block + i % a.kv_block] = a.mass[((size_t)src * a.nkv + h) * a.kv_block + j % a.kv_block];
        if (a.scale)
          for (int e = 0; e < a.ns; ++e) a.scale[to * a.ns + e] = a.scale[from * a.ns + e];
      }
    }
    const int rows = min(32, rows1 - i0), step = 32 / L;
    for (int r0 = 0; r0 < rows; r0 += 4 * step) {
      long f[4], t[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = r0 + e * step + lane / L;
        f[e] = __shfl_sync(0xffffffffu, from, r & 31);
        t[e] = __shfl_sync(0xffffffffu, to, r & 31);
        if (r > 31) t[e] = -1;
      }
      for (int c = lane % L; c < pieces; c += L) {
        uint4 x[4], y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (t[e] >= 0) {
            x[e] = *reinterpret_cast<const uint4*>(a.k + f[e] * a.row_bytes + c * 16);
            y[e] = *reinterpret_cast<const uint4*>(a.v + f[e] * a.row_bytes + c * 16);
          }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (t[e] >= 0) {
            *reinterpret_cast<uint4*>(a.k + t[e] * a.row_bytes + c * 16) = x[e];
            *reinterpret_cast<uint4*>(a.v + t[e] * a.row_bytes + c * 16) = y[e];
          }
      }
    }
  }
}

}  // namespace fb

using namespace fb;

extern "C" int fb_kv_evict(int* kept, void* k, void* v, float* scale, float* mass, const int* seg_slot, const int* seg_len, int segs, const int* table,
                           int slots, int max_blocks, const int* dst, int dst_blocks, long pages, int kv_block, int nkv, int row_bytes, int ns, int keep,
                           int first, int recent, int* status, cudaStream_t s) {
  if (segs <= 0) return 0;
  if (keep < 1 || first < 0 || recent < 0 || (long)first + recent > keep || (long)dst_blocks * kv_block < keep || row_bytes % 16 || ns > 32) return -1;
  if ((long)segs * nkv > 0x7fffffffl / 8) return -2;
  const long room = (long)max_blocks * kv_block;
  const int cluster = 8;
  int lanes = 1;
  while (lanes < 32 && lanes * 16 < row_bytes) lanes *= 2;
  const EvictArgs a{kept, (unsigned char*)k, (unsigned char*)v, scale, mass, seg_slot, seg_len, table, dst, segs, slots, max_blocks, dst_blocks, pages,
                    kv_block, nkv, row_bytes, ns, keep, first, recent, (int)std::min((room + cluster - 1) / cluster, (long)EV_HELD), lanes, status};
  const size_t smem = (size_t)a.held * 4;
  FB_CUDA_CHECK(cudaFuncSetAttribute(kv_evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, EV_HELD * 4));
  return (int)launch_pdl_cluster(cluster, kv_evict_kernel, dim3((unsigned)(segs * nkv * cluster)), dim3(EV_THREADS), smem, s, a);
}

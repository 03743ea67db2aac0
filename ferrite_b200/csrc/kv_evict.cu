// Eviction from a paged cache by accumulated weight: which tokens of a (stream, kv head) stay, and their move into new pages.
//
// Selection: a cluster of CTAs has a (segment, kv head), each CTA a run of its tokens. The weight of the last token that stays is found digit by digit, 11, 11
// and 10 bits of the weights as whole numbers in their order: a histogram per CTA in shared memory, added up over the cluster (each CTA adds up a part of the
// bins). How many heavier tokens and how many equal ones lie ahead of a token says whether it stays and where it goes (the earliest of equal ones stay), so
// the order of the tokens is kept without a sort, and nothing depends on the order in which threads run.
//
// Copy: a warp has up to 32 rows at a time; its lanes look up the pages, then all of them copy row after row, 16 bytes each.
//
// Measured (B200, us): 24 streams of 12000 tokens, 4 heads of 256 in bf16, 2048 stay: 92, selection 22, copy 70 (408 MB read and written, 5.8 TB/s: HBM); two of 100000 in
// 8 bits, 8192 stay: 31 in all, 36 on other inputs each time, selection 23 (12500 weights a CTA, digits added up over the cluster); one of 4000, 1024 stay: 13 to 16,
// selection 12 of it.
// The same in tables of 131072 tokens: one of 4000 13, four of 4000 20 (15 in tables that fit), 24 of 12000 91. 40 of 50000, whose last 5000 weights a CTA do not fit its
// shared memory, 2048 stay: 234 (heads of 32).
// Selection is bound by its instructions (issue slots of its SMs 40 % busy between the digits' barriers); 1024 threads a CTA take 16 for 4000 tokens and 24 for 12000, and
// one lane a bin adding for its warp 15 to 20 % more than an addition a lane.
#include <algorithm>
#include <cooperative_groups.h>
#include <type_traits>

#include "api_shared.h"
#include "common.cuh"

namespace fb {

namespace cg = cooperative_groups;
constexpr int EV_THREADS = 512, EV_WARPS = EV_THREADS / 32, EV_BINS = 2048, EV_HELD = 44 << 10;   // weights that a CTA holds in shared memory
constexpr int EV_PART = 8192;                    // tokens of a CTA where another one could have an SM for itself

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
  int held, page_shift, row_lanes, run;          // weights that fit; log2 of kv_block, or -1; lanes that copy a row together (a power of two); rows of a warp
  int* status;

  __device__ __forceinline__ int page_of(int j) const { return page_shift >= 0 ? j >> page_shift : j / kv_block; }
  // tokens in the slot's cache, as far as its table reaches
  __device__ __forceinline__ int tokens(int slot, int seg) const {
    const int n = max(seg_len[seg], 0);
    if (slot >= 0 && slot < slots && n <= (long)max_blocks * kv_block) return n;
    set_status(status, ST_BOUNDS);
    return slot < 0 || slot >= slots ? 0 : max_blocks * kv_block;
  }
};

__device__ __forceinline__ int checked_page(const EvictArgs& a, int page) {
  if (page >= 0 && page < a.pages) return page;
  set_status(a.status, ST_BOUNDS);
  return -1;
}
// the weight of a token that shared memory does not hold (behind the first EV_HELD of a CTA)
__device__ __noinline__ uint32_t weight_of(const EvictArgs& a, const int* table, int h, int j) {
  const int p = a.page_of(j), page = checked_page(a, table[p]);
  return page < 0 ? 0u : weight_order(a.mass[((size_t)page * a.nkv + h) * a.kv_block + (j - p * a.kv_block)]);
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

__global__ void __launch_bounds__(EV_THREADS, 2) kv_select_kernel(EvictArgs a) {
  extern __shared__ uint32_t held_s[];
  __shared__ uint32_t hist[EV_BINS], total[EV_BINS];
  __shared__ uint64_t tmp[EV_WARPS], counts_s;
  __shared__ uint32_t digit_s[3];
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), most = (int)cluster.num_blocks(), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int pair = blockIdx.x / most, seg = pair / a.nkv, h = pair % a.nkv;
  pdl_launch_dependents();
  pdl_wait();
  const int slot = a.seg_slot[seg], n = a.tokens(slot, seg);
  // The cluster is for what the table has room for; the context says how many of its CTAs there is work for, and the others leave (its barriers wait for those that have
  // not left).
  int ctas = 1;
  while (ctas < most && n > EV_PART * ctas) ctas *= 2;
  if (rank >= ctas) return;
  const int* table = a.table + (size_t)max(slot, 0) * a.max_blocks;
  int* kept = a.kept + (size_t)pair * a.keep;
  for (int i = min(n, a.keep) + rank * EV_THREADS + tid; i < a.keep; i += ctas * EV_THREADS) kept[i] = -1;
  if (n <= a.keep) {                                                 // (the same for the cluster)
    for (int i = rank * EV_THREADS + tid; i < n; i += ctas * EV_THREADS) kept[i] = i;
    return;
  }
  // ---- this CTA's tokens
  const int per = (n + ctas - 1) / ctas, t0 = min(n, rank * per), t1 = min(n, t0 + per), lo = a.first, hi = n - a.recent;
  const int th = min(t1, t0 + a.held);                               // shared memory holds the weights of those ahead of this one
  const bool hold = th == t1;
  auto near = [&](int j) { return held_s[j - t0]; };
  auto far = [&](int j) { return j < th ? near(j) : weight_of(a, table, h, j); };
  uint32_t need = (uint32_t)(a.keep - a.first - a.recent), prefix = 0, mask = 0;
  const bool none = need == 0;
  const int m0 = max(t0, lo), m1 = min(t1, hi), mh = min(m1, max(m0, th));       // of the middle, where weights decide; held ones ahead of mh
  // N a thread: their pages first, then their weights, so that the loads of either are under way together (a page that is none is reported behind them; what counts for
  // its weight is the same for every digit).
  auto load = [&](auto at_once, auto far_ones, int from, int to, auto use) {
    constexpr int N = decltype(at_once)::value;
    bool bad = false;
#pragma unroll 1
    for (int j0 = from + tid; j0 < to; j0 += N * EV_THREADS) {
      int page[N];
      float w[N];
#pragma unroll
      for (int e = 0; e < N; ++e) page[e] = table[a.page_of(min(j0 + e * EV_THREADS, to - 1))];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int j = min(j0 + e * EV_THREADS, to - 1);
        const bool out = page[e] < 0 || page[e] >= a.pages;
        bad |= out;
        w[e] = a.mass[((size_t)(out ? 0 : page[e]) * a.nkv + h) * a.kv_block + (j - a.page_of(j) * a.kv_block)];
      }
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (j0 + e * EV_THREADS < to) use(j0 + e * EV_THREADS, far_ones.value && (page[e] < 0 || page[e] >= a.pages) ? 0u : weight_order(w[e]));
    }
    if (bad) set_status(a.status, ST_BOUNDS);
  };
  if (!none) {
    for (int i = tid; i < EV_BINS; i += EV_THREADS) hist[i] = 0;
    __syncthreads();
    load(std::integral_constant<int, 8>{}, std::false_type{}, m0, mh, [&](int j, uint32_t u) {                            // (the first digits are counted on the way)
      held_s[j - t0] = u;
      atomicAdd(&hist[u >> 21], 1u);
    });
  }
  for (int pass = 0; pass < 3 && !none; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t bins = pass == 2 ? 1024u : 2048u;
    auto count = [&](int, uint32_t u) {
      if ((u & mask) == prefix) atomicAdd(&hist[u >> shift & (bins - 1)], 1u);
    };
    if (pass > 0) {
      for (int i = tid; i < EV_BINS; i += EV_THREADS) hist[i] = 0;
      __syncthreads();
#pragma unroll 4
      for (int j = m0 + tid; j < mh; j += EV_THREADS) count(j, held_s[j - t0]);
    }
    if (mh < m1) load(std::integral_constant<int, 4>{}, std::true_type{}, mh, m1, count);
    if (ctas > 1) cluster.sync();
    else __syncthreads();
    if (ctas > 1) {
      // a part of the bins each, handed to everyone
      const int part = EV_BINS / ctas;
      for (int i = rank * part + tid; i < (rank + 1) * part; i += EV_THREADS) {
        uint32_t v[8], sum = 0;
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] = c < ctas ? cluster.map_shared_rank(hist, c)[i] : 0u;
#pragma unroll
        for (int c = 0; c < 8; ++c) sum += v[c];
#pragma unroll
        for (int c = 0; c < 8; ++c)
          if (c < ctas) cluster.map_shared_rank(total, c)[i] = sum;
      }
      cluster.sync();
    }
    const uint32_t* all_bins = ctas > 1 ? total : hist;
    // bins from the top, four a thread
    const uint4 q = *reinterpret_cast<const uint4*>(all_bins + EV_BINS - 4 - 4 * tid);
    const uint32_t mine = q.x + q.y + q.z + q.w;
    uint64_t all;
    uint32_t ahead = (uint32_t)scan_pairs(mine, tmp, &all);
    if (ahead < need && need <= ahead + mine) {
      uint32_t of = q.w, d = EV_BINS - 1 - 4 * tid;
      if (ahead + of < need) { ahead += of; of = q.z; --d; }
      if (ahead + of < need) { ahead += of; of = q.y; --d; }
      if (ahead + of < need) { ahead += of; of = q.x; --d; }
      digit_s[0] = d;
      digit_s[1] = need - ahead;
      digit_s[2] = of;                                               // tokens of this digit
    }
    __syncthreads();
    prefix |= digit_s[0] << shift;
    mask |= (bins - 1) << shift;
    need = digit_s[1];
    if (digit_s[2] == need) break;                                   // all of them stay: the digits behind say nothing
  }
  // ---- need: how many tokens whose weight starts with `prefix` stay. A warp has neighbouring tokens, 32 at a time: how many stay for sure (low half), equal ones (high)
  const int run = ((t1 - t0 + EV_WARPS - 1) / EV_WARPS + 31) / 32 * 32, w0 = min(t1, t0 + warp * run), w1 = min(t1, w0 + run);
  // (without weights to decide, mask and prefix are zero: all of the middle is equal, and none of it stays)
  auto kinds = [&](int j, uint32_t* sures, uint32_t* equals) {
    const bool there = j < w1, middle = there && j >= lo && j < hi;
    const uint32_t u = middle ? (hold ? near(j) : far(j)) & mask : 0u;
    *sures = __ballot_sync(0xffffffffu, there && (!middle || u > prefix));
    *equals = __ballot_sync(0xffffffffu, middle && u == prefix);
  };
  // (a lane keeps what its number's 32 tokens are, for the first 1024 of the warp)
  uint32_t sure_of = 0, equal_of = 0, sure_sum = 0, equal_sum = 0;
  int at = 0;
  for (int j = w0; j < w1; j += 32, ++at) {
    uint32_t sures, equals;
    kinds(j + lane, &sures, &equals);
    if (at == lane) {
      sure_of = sures;
      equal_of = equals;
    }
    sure_sum += __popc(sures);
    equal_sum += __popc(equals);
  }
  const uint64_t mine = (uint64_t)sure_sum | (uint64_t)equal_sum << 32;
  uint64_t all;
  uint64_t ahead = scan_pairs(lane == 0 ? mine : 0, tmp, &all);
  ahead = __shfl_sync(0xffffffffu, ahead, 0);
  if (ctas > 1) {
    if (tid == 0) counts_s = all;
    cluster.sync();
    for (int c = 0; c < rank; ++c) ahead += *cluster.map_shared_rank(&counts_s, c);
    cluster.sync();                                                  // (a CTA stays as long as its counts are read)
  }
  uint32_t sures_ahead = (uint32_t)ahead, equals_ahead = (uint32_t)(ahead >> 32);
  at = 0;
  for (int j = w0; j < w1; j += 32, ++at) {
    uint32_t sures = __shfl_sync(0xffffffffu, sure_of, at & 31), equals = __shfl_sync(0xffffffffu, equal_of, at & 31);
    if (at >= 32) kinds(j + lane, &sures, &equals);
    const uint32_t below = (1u << lane) - 1, e = equals_ahead + __popc(equals & below), s = sures_ahead + __popc(sures & below);
    if ((sures >> lane & 1u) || ((equals >> lane & 1u) && e < need)) kept[s + min(e, need)] = j + lane;
    sures_ahead += __popc(sures);
    equals_ahead += __popc(equals);
  }
}

__global__ void __launch_bounds__(256) kv_copy_kernel(EvictArgs a) {
  const int lane = threadIdx.x & 31, pieces = a.row_bytes / 16, L = a.row_lanes, step = 32 / L, run = a.run, runs = (a.keep + run - 1) / run;
  pdl_launch_dependents();
  pdl_wait();
  const int* kept_all = after_wait(a.kept);
  const long u = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (u < (long)a.segs * a.nkv * runs) {
    const int pair = (int)(u / runs), i0 = (int)(u % runs) * run, seg = pair / a.nkv, h = pair % a.nkv, i = i0 + lane, slot = a.seg_slot[seg];
    const int j = lane < run && i < a.keep ? kept_all[(size_t)pair * a.keep + i] : -1;
    long from = -1, to = -1;
    if (j >= 0 && slot >= 0 && slot < a.slots && a.page_of(j) < a.max_blocks) {
      const int sp = a.page_of(j), dp = a.page_of(i);
      const int src = checked_page(a, a.table[(size_t)slot * a.max_blocks + sp]), dst = checked_page(a, a.dst[(size_t)seg * a.dst_blocks + dp]);
      if (src >= 0 && dst >= 0) {
        const int so = j - sp * a.kv_block, d0 = i - dp * a.kv_block;
        from = ((long)src * a.kv_block + so) * a.nkv + h;
        to = ((long)dst * a.kv_block + d0) * a.nkv + h;
        a.mass[((size_t)dst * a.nkv + h) * a.kv_block + d0] = a.mass[((size_t)src * a.nkv + h) * a.kv_block + so];
        if (a.scale)
          for (int e = 0; e < a.ns; ++e) a.scale[to * a.ns + e] = a.scale[from * a.ns + e];
      }
    }
    if (!__any_sync(0xffffffffu, to >= 0)) return;
    for (int r0 = 0; r0 < run; r0 += 4 * step) {
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
                           int first, int recent, int ctas, int* status, cudaStream_t s) {
  if (segs <= 0) return 0;
  if (ctas < 1 || keep < 1 || first < 0 || recent < 0 || (long)first + recent > keep || (long)dst_blocks * kv_block < keep || row_bytes % 16 || ns > 32) return -1;
  if ((long)segs * nkv > 0x7fffffffl / 8) return -2;
  const long room = (long)max_blocks * kv_block;
  // CTAs of a cluster: the fewest of 1, 2, 4 and 8 that leave a CTA up to 8192 tokens, as far as each has an SM for itself. (A CTA alone takes 12 us for 4000 tokens and
  // 22 for 12000; what crosses a cluster costs 2 us a digit, and 96 clusters of two, some SMs with two CTAs, take 25 for 12000 where 96 CTAs take 22.) Tables are as
  // wide as contexts may get: a shorter one uses fewer of its CTAs. Weights of contexts past EV_HELD a CTA are partly read anew for every digit.
  int cluster = 1, lanes = 1, shift = -1;
  while (cluster < 8 && room > (long)EV_PART * cluster && (long)segs * nkv * cluster * 2 <= ctas) cluster *= 2;
  const long held = std::min(std::max((room + cluster - 1) / cluster, std::min(room, (long)EV_PART)), (long)EV_HELD);
  while (lanes < 32 && lanes * 16 < row_bytes) lanes *= 2;
  for (int b = 0; b < 31; ++b)
    if (kv_block == 1 << b) shift = b;
  // rows of a warp: 32, fewer where that leaves some of the SMs' 64 warps without any
  int run = 32;
  while (run > 4 && run > 128 / lanes && (long)segs * nkv * ((keep + run - 1) / run) < 64l * ctas) run /= 2;
  const EvictArgs a{kept, (unsigned char*)k, (unsigned char*)v, scale, mass, seg_slot, seg_len, table, dst, segs, slots, max_blocks, dst_blocks, pages,
                    kv_block, nkv, row_bytes, ns, keep, first, recent, (int)held, shift, lanes, run, status};
  const size_t smem = (size_t)a.held * 4;
  FB_CUDA_CHECK(cudaFuncSetAttribute(kv_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, EV_HELD * 4));
  cudaError_t e = launch_pdl_cluster(cluster, kv_select_kernel, dim3((unsigned)(segs * nkv * cluster)), dim3(EV_THREADS), smem, s, a);
  if (e != cudaSuccess) return (int)e;
  const long runs = (long)segs * nkv * ((keep + run - 1) / run);
  return (int)launch_pdl(kv_copy_kernel, dim3((unsigned)((runs + 7) / 8)), dim3(256), 0, s, a);
}

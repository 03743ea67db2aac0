// A step over a paged cache whose streams may share pages, as lists of equal pieces of work: what a kernel needs to find its own piece from the lengths
// on the device, so that a captured call follows its contexts.
//
// Spans: the shared tokens of a group, [0, len) through the table of its first segment, for the rows of all its segments; and what follows them of a segment,
// [len, longest context) through its own table, for its own rows. A span's rows are cut into blocks of R (what fills the 128 rows of a product, share query
// heads a row), and a (block, kv head) walks the key tiles of its span that one of its rows sees.
#pragma once
#include "api_shared.h"
#include "common.cuh"

namespace fb {

constexpr int SK_PLAN_BYTES = 160 << 10;         // shared memory that the plan may take while it is made
constexpr int SK_FEW = 128;                      // spans and blocks of a step that SK_FEW threads plan

// What a block is. kmin: keys that all of its rows see. place0: places of the blocks ahead of it (of one kv head): a unit has one for every key tile and,
// ahead of them, `extra` for what it costs besides.
struct __align__(16) SharedBlock {
  int row0, nrows, slot, k0;
  int k1, kmin, place0, nt;
};

__device__ __forceinline__ long table_limit(const FbSharedStep& st) { return (long)st.max_blocks * st.kv_block; }
// Row of the cache where a tile's first token lies; one far outside (a load from there reads zeros) where the table has none.
__device__ __forceinline__ int tile_row(const FbSharedStep& st, int slot, int token, int* status) {
  const int blk = st.table[(size_t)slot * st.max_blocks + token / st.kv_block];
  if (blk < 0 || blk >= st.pages) {
    set_status(status, ST_BOUNDS);
    return -1024;
  }
  return blk * st.kv_block + token % st.kv_block;
}
__device__ __forceinline__ bool rows_fit(const FbSharedStep& st, int row0, int nrows) { return row0 >= 0 && nrows >= 0 && nrows <= st.rows - row0; }

// a[0 .. n) -> sums of what lies ahead, in place; returns the sum of all. Every thread of the CTA calls it, with what it reads written ahead of a barrier;
// ends with a barrier. tmp: a place for each warp.
template <int THREADS>
__device__ __forceinline__ long long scan_ahead(int* a, int n, long long* tmp) {
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, per = (n + THREADS - 1) / THREADS;
  const int lo = min(n, tid * per), hi = min(n, lo + per);
  long long sum = 0;
  for (int i = lo; i < hi; ++i) sum += a[i];
  long long x = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) tmp[warp] = x;
  __syncthreads();
  const long long own = lane < THREADS / 32 ? tmp[lane] : 0;
  long long ahead = lane < warp ? own : 0, all = own;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
    all += __shfl_xor_sync(0xffffffffu, all, o);
  }
  long long at = ahead + x - sum;
  for (int i = lo; i < hi; ++i) {
    const int v = a[i];
    a[i] = (int)min(at, 0x7fffffffll);
    at += v;
  }
  __syncthreads();
  return all;
}

// Where the plan of a step lies in shared memory: the step's tables, which are read from global memory once, all at the same time, and what is made of them.
// kv: the rows' contexts too, where there is room for them.
struct SharedPlanSizes {
  int blocks, group_blocks;                      // room for: all, those of groups
  bool kv;
  bool few;                                      // SK_FEW threads make the plan
};
inline bool shared_plan_sizes(const FbSharedStep& st, long group_blocks, long seg_blocks, SharedPlanSizes* z) {
  const long words = 5l * st.nseg + 4l * st.ngrp + 2 * (group_blocks + seg_blocks), room = SK_PLAN_BYTES / 4;
  const bool kv = words + st.rows <= room;
  *z = {(int)(group_blocks + seg_blocks), (int)group_blocks, kv, 
        kv && group_blocks + seg_blocks <= SK_FEW && st.nseg + st.ngrp <= SK_FEW && (long)st.max_blocks * st.kv_block < 1l << 29};
  return words <= room;
}

template <int THREADS>
struct SharedPlan {
  int *slot, *row0, *rows, *group;               // of segments
  int *seg0, *segs, *len;                        // of groups
  int *start, *span, *place;                     // first block of every span (groups, then segments); span of every block, places ahead of it
  const int* kvlen;
  int blocks, group_blocks;
  long long places;                              // of one kv head

  // The step's tables into shared memory, by all threads; a barrier has to follow.
  __device__ __forceinline__ void load(const FbSharedStep& st, const SharedPlanSizes& z, unsigned char* smem) {
    const int tid = threadIdx.x, S = st.nseg, G = st.ngrp;
    slot = reinterpret_cast<int*>(smem); row0 = slot + S; rows = row0 + S; group = rows + S;
    seg0 = group + S; segs = seg0 + G; len = segs + G;
    start = len + G; span = start + S + G; place = span + z.blocks;
    kvlen = z.kv ? place + z.blocks : st.kvlen;
    if (z.kv) {
      int* to = place + z.blocks;
      for (int r = tid; r < st.rows; r += THREADS) to[r] = st.kvlen[r];
    }
    for (int s = tid; s < S; s += THREADS) {
      slot[s] = st.seg_slot[s];
      row0[s] = st.seg_row0[s];
      rows[s] = st.seg_nrows[s];
    }
    for (int g = tid; g < G; g += THREADS) {
      seg0[g] = st.grp_seg0[g];
      segs[g] = st.grp_nsegs[g];
      len[g] = st.grp_len[g];
    }
  }
  // rows of group g, 0 where it does not fit the step
  __device__ __forceinline__ int group_rows(const FbSharedStep& st, int g, int* status) const {
    const int s0 = seg0[g], n = segs[g];
    if (n == 0) return 0;
    if (s0 >= 0 && n > 0 && n <= st.nseg - s0) {
      const int count = row0[s0 + n - 1] + rows[s0 + n - 1] - row0[s0];
      if (slot[s0] >= 0 && slot[s0] < st.slots && rows_fit(st, row0[s0], count)) return count;
    }
    set_status(status, ST_BOUNDS);
    return 0;
  }
  // group of segment s and its own blocks (where `start` holds the groups' rows)
  __device__ __forceinline__ int segment(const FbSharedStep& st, int s, int R, int* status) {
    int own = -1;
    for (int g = 0; g < st.ngrp; ++g)
      if (start[g] > 0 && s >= seg0[g] && s - seg0[g] < segs[g]) {
        if (own >= 0 || (s > seg0[g] && row0[s] != row0[s - 1] + rows[s - 1])) set_status(status, ST_BOUNDS);   // of two groups; rows that lie apart
        own = g;
      }
    group[s] = own;
    if (rows[s] == 0) return 0;                                                  // (padding: its slot says nothing)
    if (slot[s] < 0 || slot[s] >= st.slots || !rows_fit(st, row0[s], rows[s])) {
      set_status(status, ST_BOUNDS);
      return 0;
    }
    if (rows[s] > st.max_rows) {
      set_status(status, ST_CAPACITY);
      return 0;
    }
    return (rows[s] + R - 1) / R;
  }
  __device__ __forceinline__ bool fits(const SharedPlanSizes& z) const {
    return blocks <= z.blocks && group_blocks <= z.group_blocks && blocks - group_blocks <= z.blocks - z.group_blocks;
  }

  // The plan of a step of up to SK_FEW spans and blocks from the loaded tables, by the first SK_FEW threads: each a span, then a block, which it keeps (`e`, with
  // its place). What make() does in loops and from shared memory stays in registers: code that an SM sees for the first time costs nine cycles an
  // instruction, and this comes before everything else.
  __device__ __forceinline__ bool make_by_few(const FbSharedStep& st, int R, int kt, int extra, const SharedPlanSizes& z, long long* tmp, int* status, SharedBlock* e,
                                              int* count) {
    const int me = threadIdx.x, lane = me & 31, warp = me >> 5, S = st.nseg, G = st.ngrp;
    int* sums = reinterpret_cast<int*>(tmp);
    auto sync = [] { asm volatile("bar.sync 11, %0;" ::"n"(SK_FEW) : "memory"); };
    auto scan = [&](int v, int* at, int* all) {                                  // v -> sum of what lies ahead, of all
      int x = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (lane == 31) at[warp] = x;
      sync();
      int ahead = x - v, total = 0;
#pragma unroll
      for (int w = 0; w < SK_FEW / 32; ++w) {
        const int y = at[w];
        if (w < warp) ahead += y;
        total += y;
      }
      *all = total;
      return ahead;
    };
    const int grows = me < G ? group_rows(st, me, status) : 0;
    if (me < G) start[me] = grows;
    sync();
    const int n = me < G ? (grows + R - 1) / R : me < G + S ? segment(st, me - G, R, status) : 0;
    // (the first barrier of the scan is behind every look at the groups' rows in `start`)
    const int first = scan(n, sums, &blocks);
    if (me == G) sums[8] = first;
    if (me < G) segs[me] = grows;                                                // (from here on: rows)
    if (me < G + S) start[me] = first;
    for (int b = 0; b < n && first + b < z.blocks; ++b) span[first + b] = me;
    sync();
    group_blocks = sums[8];
    if (!fits(z)) {
      if (me == 0) set_status(status, ST_CAPACITY);
      return false;
    }
    *e = SharedBlock{};
    if (me < blocks) *e = block(st, me, R, kt, status);
    *count = e->nt ? e->nt + extra : 0;
    int all;
    e->place0 = scan(*count, sums + 4, &all);                                    // (fewer than 2^31: 128 blocks of fewer than 2^23 tiles)
    places = all;
    return true;
  }

  // -> false where the step does not fit (with a status)
  __device__ __forceinline__ bool make(const FbSharedStep& st, int R, int kt, int extra, const SharedPlanSizes& z, unsigned char* smem, long long* tmp, int* status) {
    const int tid = threadIdx.x, S = st.nseg, G = st.ngrp;
    load(st, z, smem);
    __syncthreads();
    for (int g = tid; g < G; g += THREADS) start[g] = group_rows(st, g, status);
    __syncthreads();
    for (int s = tid; s < S; s += THREADS) start[G + s] = segment(st, s, R, status);
    __syncthreads();
    for (int g = tid; g < G; g += THREADS) {
      segs[g] = start[g];                                                        // (from here on: rows)
      start[g] = (start[g] + R - 1) / R;
    }
    __syncthreads();
    const long long all = scan_ahead<THREADS>(start, G + S, tmp);
    blocks = (int)min(all, 0x7fffffffll);
    group_blocks = start[G];
    if (!fits(z)) {
      if (tid == 0) set_status(status, ST_CAPACITY);
      return false;
    }
    for (int i = tid; i < G + S; i += THREADS) {
      const int end = i + 1 < G + S ? start[i + 1] : blocks;
      for (int b = start[i]; b < end; ++b) span[b] = i;
    }
    __syncthreads();
    for (int b = tid; b < blocks; b += THREADS) {
      const int nt = block(st, b, R, kt, status).nt;
      place[b] = nt ? nt + extra : 0;
    }
    __syncthreads();
    places = scan_ahead<THREADS>(place, blocks, tmp);
    if (places > 0x7fffffffll) {                                                 // (what a place's number holds)
      if (tid == 0) set_status(status, ST_CAPACITY);
      return false;
    }
    return true;
  }
  // block b (without place0)
  __device__ __forceinline__ SharedBlock block(const FbSharedStep& st, int b, int R, int kt, int* status) const {
    const int i = span[b], s = i - st.ngrp, m = b - start[i];
    SharedBlock e;
    long most;
    int count;
    if (s < 0) {
      const int s0 = seg0[i];
      e.slot = slot[s0];
      e.row0 = row0[s0];
      count = segs[i];
      e.k0 = 0;
      most = max(len[i], 0);
    } else {
      e.slot = slot[s];
      e.row0 = row0[s];
      count = rows[s];
      e.k0 = group[s] < 0 ? 0 : max(len[group[s]], 0);
      most = 0x7fffffffl;
    }
    e.row0 += m * R;
    e.nrows = min(R, count - m * R);
    int hi = 0, lo = 0x7fffffff;
#pragma unroll 8
    for (int r = 0; r < e.nrows; ++r) {
      const int n = kvlen[e.row0 + r];
      hi = max(hi, n);
      lo = min(lo, n);
    }
    if (hi > table_limit(st)) set_status(status, ST_BOUNDS);
    e.k1 = (int)min((long)hi, min(most, table_limit(st)));
    e.kmin = max(0, min(lo, e.k1));
    e.place0 = 0;
    e.nt = e.k1 > e.k0 ? (e.k1 + kt - 1) / kt - e.k0 / kt : 0;
    return e;
  }
  // block that place `at` of the list of all (block, kv head) units belongs to
  __device__ __forceinline__ int find(long long at, int heads) const {
    int lo = 0, hi = blocks - 1;                                                 // the last one that starts at or ahead of it: it has some
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if ((long long)place[mid] * heads <= at) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  }
};

// Most blocks of a step, from what the host knows.
inline long shared_group_blocks(long rows, int ngrp, int R) { return ngrp ? rows / R + ngrp : 0; }
inline long shared_seg_blocks(long rows, int nseg, int max_rows, int R) {
  const long each = (long)nseg * ((max_rows + R - 1) / R), all = rows / R + nseg;
  return each < all ? each : all;
}

// ---- what the kernels of this family use of the tensor cores and barriers ----------------------------------------------------------------------
__device__ __forceinline__ float sk_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Wait of at most 2^31 cycles (about a second) that leaves the issue slots to others; false where it ran out or another role gave up.
__device__ __forceinline__ bool sk_poll(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity), "r"(20000u) : "memory");
  return ok;
}
__device__ __forceinline__ bool sk_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
#pragma unroll 1
  while (!sk_poll(bar, parity))
    if (*abort_flag || clock64() - t0 > 1ll << 31) return false;
  return true;
}
// The same for two barriers at once: one that has come by already costs nothing beside the other.
__device__ __forceinline__ bool sk_wait2(uint64_t* a, uint32_t pa, uint64_t* b, uint32_t pb, volatile int* abort_flag) {
  if (mbar_try_wait(a, pa) & mbar_try_wait(b, pb)) return true;
  return sk_wait(a, pa, abort_flag) && sk_wait(b, pb, abort_flag);
}
// MN-major operand tile with the 128-byte swizzle: rows are K, 64 contiguous MN elements a row; lbo: bytes between chunks of 64 along MN, sbo between eight rows.
__device__ __forceinline__ uint64_t sk_desc_mn128(uint32_t smem_addr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((smem_addr & 0x3ffffu) >> 4) | (uint64_t)((lbo >> 4) & 0x3fff) << 16 | (uint64_t)((sbo >> 4) & 0x3fff) << 32 | 1ull << 46 | 2ull << 61;
}
// Tensor memory, by a warp that plans nothing, behind the wait for the kernels ahead: one of them whose CTA has yet to ask for its columns would never get them from a
// CTA that waits for it. For the same reason the kernels behind start only where this CTA has its columns. A barrier has to lie between the two.
constexpr int SK_ALLOC = 4;
__device__ __forceinline__ void sk_tmem_alloc(uint32_t* to, uint32_t cols) {
  if (threadIdx.x >> 5 == SK_ALLOC) {
    tmem_alloc(to, cols);
    tmem_relinquish();
  }
  tc_fence_before();
}
__device__ __forceinline__ uint32_t sk_tmem_ready(const uint32_t* at) {
  tc_fence_after();
  pdl_launch_dependents();
  return *at;
}
// D = A B^T over 16 NK columns of K-major operands in chunks of 64, chunk_a and chunk_b bytes apart, from the operands' first descriptors. (The issuing warp gets a
// fifth of its scheduler's slots beside four warps of arithmetic: a descriptor built anew for every product costs as much as the product.)
template <int NK>
__device__ __forceinline__ void sk_products(bool issue, uint32_t tmem_d, uint64_t a, uint64_t b, int chunk_a, int chunk_b, uint32_t idesc) {
#pragma unroll
  for (int kk = 0; kk < NK; ++kk)
    tc_mma_f16_if(issue, tmem_d, a + (uint32_t)(((kk >> 2) * chunk_a + (kk & 3) * 32) >> 4), b + (uint32_t)(((kk >> 2) * chunk_b + (kk & 3) * 32) >> 4), idesc,
                  kk > 0 ? 1u : 0u);
}
// The same with A in tensor memory: a lane a row, a column two of its values, K-major. Products of few columns are bound by what they read of shared memory, 128
// bytes a cycle: 128 x 64 x 256 takes 768 cycles with both operands there and 512, what its operations take, with B alone.
template <int NK>
__device__ __forceinline__ void sk_products_ts(bool issue, uint32_t tmem_d, uint32_t tmem_a, uint64_t b, int chunk_b, uint32_t idesc) {
#pragma unroll
  for (int kk = 0; kk < NK; ++kk)
    tc_mma_f16_ts_if(issue, tmem_d, tmem_a + kk * 8, b + (uint32_t)(((kk >> 2) * chunk_b + (kk & 3) * 32) >> 4), idesc, kk > 0 ? 1u : 0u);
}
__device__ __forceinline__ void sk_tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void sk_tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
// 16 lanes x 16 columns: registers 4 c, 4 c + 1 are columns 8 c + 2 (lane % 4) and the next of TMEM lane lane / 4; 4 c + 2, 4 c + 3 those of lane / 4 + 8.
__device__ __forceinline__ void sk_tmem_ld16x16(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}

}  // namespace fb

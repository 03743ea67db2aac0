// Attention over a latent cache in 4 or 8 bits (rows as in mla_cache.cuh) on the 5th-generation tensor cores, absorbed form: every head attends the same
// rows, o = softmax(scale * q . [value | key part]) value.
//
// Keys are the wide side of both products (M = 128), (row, head) pairs of a segment the narrow one (N = 16, 32 or 64): one unpacking of the codes serves
// N pairs and both products.
//
//   S^T [128 keys x N]  = [K | key part] Q^T     A: the tile's values, rows of keys; B: the pairs' queries
//   O^T [L x N]        += V^T P^T                A: the SAME tile in shared memory, read along its columns; B: the weights, written by the softmax
//
// Warps 0..15 unpack (four threads a key, 32 of every 128 values each): a word of eight 4-bit codes takes a shift, a mask and one fma per two values,
// fp16(16 + code + 8) * s - 24 s, exact in fp16 as the value itself is (a power of two times seven bits). The codes of the next tile are in flight in
// registers meanwhile. Warps 16..23 run the softmax: a thread has a key (its TMEM lane) and half of the pairs. Warp 24 issues the products, 25 and 26
// copy the key parts, 27 looks up the keys' pages.
// The values' products run in fp16, so that a weight keeps 11 bits; a query is brought to 2^10 by a power of two of its own, which keeps its bf16 bits down
// to 2^-27 of its largest value. The key part stays in bf16 (its products go to the same sums).
//
// Softmax along the lanes: a column's maximum would need all 128 threads, every tile. Instead a piece's first tile gives the reference r (its maximum - 4),
// and weights are 2^(x - r): exact whatever r is, as long as fp16 holds them. Only where a later score passes r by 2^15 (a vote of the 256 threads,
// every tile) is the maximum taken anew and O rescaled.
//
// Work is cut evenly, not by row: the tiles of all (segment, group of N pairs) units form one list, every CTA takes the same number of consecutive
// ones, from what the lengths on the device say (so a captured call follows its contexts). Units that span CTAs leave their sums in 32 bits,
// and a second kernel joins them in order. Where a row's keys are cut, and so how its sums round, therefore follows the other rows of the step, the
// number of SMs, and N: the most rows of a segment, the heads, and the keys that the block table has room for. The same call gives the same bits. (Cuts
// that follow a row's own context alone, as in the 16-bit cache, have to be fine enough for one stream on all SMs, and then leave 32-bit sums of 2 KB a
// head for every few tiles of a loaded step.)
//
// A key of which a group is no number gets the score NaN and a finite place in the tile, so that rows ahead of it, whose weight for it is zero, stay clean.
//
// What bounds it: the way to shared memory, 128 bytes a cycle. For a tile of 64 pairs the products read 36 * 6 KB (S) and 32 * 6 KB (O), 3260 cycles; stores
// of the unpacked tile, codes that come in sectors of 32 bytes, key parts and scores take 4300 more (the counters' wavefronts): 7560 of the tile's
// 8700. During the softmax's 2000 no product runs: the tile has to stay and none of the next has room (128 KB of tile, 72 KB of queries). 16 pairs: 6200
// cycles a tile. Measured, 512 values in 4 bits, captured, cold caches: 24 streams of up to 16000 keys with 128 heads 154 us (43: the products at the card's
// rate), 32 with 16 heads 82 us (22: the bytes), one of 100000 with 128 heads 89 us (17), one of 2048 21 to 25 us by the table's room (latent_pairs): 13 here,
// of which 7 until the first scores (code that is new to every SM comes slowly), 6 in the join, the rest between launches.
// Tried and slower: tiles of 64 keys in two places (S costs 65 cycles where 48 do for 128 keys), tiles in tensor memory for S, unpacking by two groups
// of warps in turn (32 streams of 16 heads 87 -> 93 us), the softmax in halves with the next one's load under
// way (registers: 161 -> 171 us), rows brought to L2 ahead one by one (114 us; a page's in one request costs nothing).
//
// Every wait is bounded: one that runs out sets the status word and an abort flag, all roles leave and the CTA frees its TMEM.
#include <algorithm>

#include "api_ext.h"
#include "mla_cache.cuh"

namespace fb {

constexpr int LA_KT = 128;                       // keys of a tile
constexpr int LA_CH = LA_KT * 128;               // bytes of 64 values of all of them
constexpr int LA_UNPACK = 16, LA_SOFT = LA_UNPACK + 8;             // warps up to which these roles go
constexpr int LA_THREADS = (LA_SOFT + 4) * 32;   // and one that issues the products, two that copy key parts, one that looks keys up
constexpr int LA_AHEAD = 4;                      // tiles whose keys are looked up ahead
constexpr int LA_ROWS = 64;                      // rows whose units walk the same keys; a segment of more, a prompt, is cut into blocks of so many
constexpr float LA_TOP = 4.f, LA_LIMIT = 15.f;   // log2 of a piece's first largest weight; of the largest one that a weight may be

template <int BITS, int NC, int N>
struct LatentAttn {
  static constexpr int L = NC * 64, CW = N / 2;                    // CW: pairs of a softmax thread
  static constexpr int NP = (NC + 1) / 2;                          // pairs of 64 values: rows of 128 of O^T
  static constexpr int NB = NC == 8 ? (N == 64 ? 4 : 5) : 2 * NP;  // buffers of them
  static constexpr bool SHARE = NC == 8 && N == 64;                // the weights take the place of the tile's key part
  static constexpr int PD = BITS == 8 && NP == 4 ? 2 : NP;         // pairs of codes in flight
  static constexpr int Q_BYTES = (NC + 1) * N * 128, P_BYTES = LA_KT * N * 2;
  static constexpr int K_AT = Q_BYTES, R_AT = K_AT + NB * 2 * LA_CH, P_AT = SHARE ? R_AT : R_AT + LA_CH;
  static constexpr int MISC_AT = SHARE ? R_AT + LA_CH : P_AT + P_BYTES;
  static constexpr int COLS = (NP + 1) * N;                        // of TMEM: O^T | S^T
  static constexpr int TMEM = COLS <= 32 ? 32 : COLS <= 64 ? 64 : COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
};
template <int N>
struct LatentAttnMisc {
  float c[2][N], nr[2][N];                       // by the piece's parity: what leads from a score to log2, minus the reference
  int see[2][N];                                 // keys that a pair sees
  float mx[4][N], d[N];
  uint32_t bad[4][16];                           // of the last tiles: keys that are no number, four bits a key
  int rows[LA_AHEAD][LA_KT];                     // ring of tiles: their keys' rows of the cache, -1 where there is none
  uint64_t bars[2 * 5 + 7 + 2 * LA_AHEAD];
  uint32_t tmem;
  int least[8];                                  // of the piece: keys that all pairs of a softmax warp see
  int abort, fail;
};

struct LatentSegs {
  const int *slot, *row0, *nrows, *kvlen;
  int nseg, nq;
  long limit;                                    // keys that a table has room for
};
// A place in the list of tiles: of segment s, block row0 .. row0 + nrows of its rows, `left` rows behind them, unit u of the block, tile t of the unit. A
// prompt's blocks end where their own last rows do (2048 rows of 128 heads from position 0: 1282 us; 2215 with every unit as long as the prompt). Its units
// count a place more than they have tiles (`extra`): the queries, the output and the gaps of a unit take 6 us where a tile takes 4.5, and the first rows'
// units are short (without it the CTA that has those is the last by far: 2354 us).
struct LatentWalk {
  int s, u, t, units, nt, kv, row0, nrows, slot, left, extra;
  bool over = false;                             // a row that sees more than the table has room for has come by
  // rows of a block may stand in any order: it is as long as the longest of their contexts, which a warp looks for, or (APART) a lane for itself
  template <int N, bool APART = false>
  __device__ __forceinline__ void block(const LatentSegs& g) {
    int most = 0;
    if constexpr (APART) {
#pragma unroll 4
      for (int r = 0; r < nrows; ++r) most = max(most, g.kvlen[row0 + r]);
    } else {
      const int lane = threadIdx.x & 31;
      static_assert(LA_ROWS == 64, "two rows a lane");
      if (lane < nrows) most = max(most, g.kvlen[row0 + lane]);
      if (lane + 32 < nrows) most = max(most, g.kvlen[row0 + 32 + lane]);
      most = __reduce_max_sync(0xffffffffu, most);
    }
    over |= most > g.limit;
    kv = (int)min((long)most, g.limit);
    units = (int)(((uint32_t)nrows * g.nq + N - 1) / N);               // (rows times heads are fewer than 2^30; those of a whole block fill its units)
    nt = max(1, (kv + LA_KT - 1) / LA_KT);
  }
  template <int N, bool APART = false>
  __device__ __forceinline__ void segment(const LatentSegs& g) {
    const int n = max(g.nrows[s], 0);
    row0 = g.row0[s]; slot = g.slot[s];
    nrows = min(n, LA_ROWS);
    left = n - nrows;
    extra = left > 0;
    block<N, APART>(g);
  }
  template <int N>
  __device__ __forceinline__ void next_block(const LatentSegs& g) {
    row0 += LA_ROWS;
    nrows = min(left, LA_ROWS);
    left -= nrows;
    block<N>(g);
  }
  template <int N>
  __device__ __forceinline__ void next_unit(const LatentSegs& g) {
    t = 0;
    if (++u < units) return;
    u = 0;
    units = 0;
    if (left > 0) {
      next_block<N>(g);
      return;
    }
#pragma unroll 1
    while (++s < g.nseg) {
      segment<N>(g);
      if (units) break;
    }
  }
};

__device__ __forceinline__ uint64_t umma_desc_mn(uint32_t smem_addr, uint32_t lbo, uint32_t sbo, uint32_t swizzle) {
  return (uint64_t)((smem_addr & 0x3ffffu) >> 4) | (uint64_t)(lbo >> 4) << 16 | (uint64_t)(sbo >> 4) << 32 | 1ull << 46 | (uint64_t)swizzle << 61;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Wait of at most 2^31 cycles (about a second) that leaves the issue slots to others: the hardware holds the warp for up to 20 us a poll.
__device__ __forceinline__ bool la_poll(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity), "r"(20000u) : "memory");
  return ok;
}
__device__ __forceinline__ bool la_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  if (la_poll(bar, parity)) return true;
  const long long t0 = clock64();
#pragma unroll 1
  while (!la_poll(bar, parity))
    if (*abort_flag || clock64() - t0 > 1ll << 31) return false;
  return true;
}
template <int W>
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t (&r)[W]) {
  if constexpr (W == 8) tmem_ld8(addr, r);
  else if constexpr (W == 16) tmem_ld16(addr, r);
  else tmem_ld32(addr, r);
}
template <int W>
__device__ __forceinline__ void tmem_st(uint32_t addr, const uint32_t (&r)[W]) {
  if constexpr (W == 32) {
    tmem_st32(addr, r);
  } else {
#pragma unroll
    for (int i = 0; i < W; i += 8)
      asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                   ::"r"(addr + i), "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
                   : "memory");
  }
}
// Per column of a warp's 32 rows: op over the rows. Lane `lane` ends with column lane % W. Halves change hands, so that W columns cost W - 1 exchanges.
template <int W, typename Op>
__device__ __forceinline__ float columns(const float (&v)[W], int lane, Op op) {
  float a[W / 2];
#pragma unroll
  for (int off = W / 2; off > 0; off >>= 1) {
    const bool up = lane & off;
#pragma unroll
    for (int i = 0; i < off; ++i) {
      const float lo = off == W / 2 ? v[i] : a[i], hi = off == W / 2 ? v[i + off] : a[i + off];
      a[i] = op(up ? hi : lo, __shfl_xor_sync(0xffffffffu, up ? lo : hi, off));
    }
  }
#pragma unroll
  for (int off = W; off < 32; off <<= 1) a[0] = op(a[0], __shfl_xor_sync(0xffffffffu, a[0], off));
  return a[0];
}
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ bool softmax_any(bool p) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred a, b;\n\tsetp.ne.b32 a, %1, 0;\n\tbar.red.or.pred b, 1, 256, a;\n\tselp.u32 %0, 1, 0, b;\n\t}"
               : "=r"(r) : "r"((uint32_t)p) : "memory");
  return r != 0;
}

__device__ __forceinline__ void st_shared_v4(uint32_t addr, const uint32_t (&v)[4]) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
// 32 values of a key: codes -> fp16 in four 16-byte places of the key's row(s) of 128 bytes. Lanes 4 r + p have key r, part p of a pair of 64 values.
// Eight lanes' stores fall on eight different places: the swizzle tells keys apart, the order within a part tells the pair's halves apart.
//   4 bits: part p is half p % 2 of 64 number p / 2; sc: the scale bytes of its two groups. Places of the words in their order (p < 2) or 2, 3, 0, 1
//   8 bits: part p is 16 values of each 64, from 16 p on; sc: the scale bytes of the two 64s. Places of the first 64, then of the second
template <int BITS>
__device__ __forceinline__ void unpack32(const uint4 (&raw)[BITS / 4], uint32_t sc, uint32_t base, const uint32_t (&at)[4], bool up, bool second) {
  if constexpr (BITS == 4) {
    const uint32_t w[4] = {up ? raw[0].z : raw[0].x, up ? raw[0].w : raw[0].y, up ? raw[0].x : raw[0].z, up ? raw[0].y : raw[0].w};
    const uint32_t sb = up ? __byte_perm(sc, 0, 0x4401) : sc;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const __half2 s = __float2half2_rn(latent_scale<4>(h ? sb >> 8 & 255u : sb & 255u)), m = __hmul2(s, __float2half2_rn(-24.f));
#pragma unroll
      for (int q = 2 * h; q < 2 * h + 2; ++q) {
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t t = ((i == 0 ? w[q] << 6 : i == 1 ? w[q] << 2 : i == 2 ? w[q] >> 2 : w[q] >> 6) & 0x03c003c0u) | 0x4c004c00u;
          const __half2 v = __hfma2(*reinterpret_cast<const __half2*>(&t), s, m);
          o[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
        st_shared_v4(base + at[q], o);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      if (e == 1 && !second) break;
      const uint32_t w[4] = {raw[e].x, raw[e].y, raw[e].z, raw[e].w};
      const __half2 s = __float2half2_rn(latent_scale<8>(sc >> (8 * e) & 255u));
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[2 * q + i / 2] >> (16 * (i % 2))), __NV_E4M3);
          const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&r), s);
          o[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
        st_shared_v4(base + at[2 * e + q], o);
      }
    }
  }
}

// grid: CTAs, one an SM. o_part [2 * CTAs][N][L], ml_part [2 * CTAs][N][2]; join [entries]: what the second kernel has to do, by unit (or, where there may
// be more units than CTAs, by the CTA that a unit starts in): first pair, pairs (0: nothing), first record, last CTA.
template <int BITS, int NC, int N>
__global__ void __launch_bounds__(LA_THREADS, 1)
mla_attn_q_kernel(__nv_bfloat16* __restrict__ out, float* __restrict__ o_part, float* __restrict__ ml_part, int4* __restrict__ join, int entries, int by_unit,
                  const __nv_bfloat16* qabs, const uint8_t* cache, LatentSegs g, const int* block_table, int max_blocks, long pages, int kv_block,
                  float scale_log2, int* status) {
  using C = LatentAttn<BITS, NC, N>;
  using Row = LatentRow<BITS>;
  constexpr int L = C::L, D = L + LC_R, CW = C::CW, NP = C::NP, NB = C::NB, RB = Row::bytes(L);
  extern __shared__ __align__(1024) unsigned char smem[];
  LatentAttnMisc<N>& ms = *reinterpret_cast<LatentAttnMisc<N>*>(smem + C::MISC_AT);
  uint64_t *kfull = ms.bars, *kempty = kfull + 5, *rfull = kempty + 5, *rempty = rfull + 1, *sfull = rempty + 1, *pfull = sfull + 1, *qfull = pfull + 1,
           *ofull = qfull + 1, *oempty = ofull + 1, *xfull = oempty + 1, *xempty = xfull + LA_AHEAD;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort_flag = &ms.abort;
  pdl_launch_dependents();
  if (smem_u32(smem) & 1023u) {                                      // the swizzled tiles need the 1024-byte base
    if (tid == 0) set_status(status, ST_BOUNDS);
    return;
  }
  if (tid == 0) {
    ms.abort = 0; ms.fail = 0;
    for (int i = 0; i < NB; ++i) { mbar_init(&kfull[i], LA_UNPACK); mbar_init(&kempty[i], 1); }
    mbar_init(rfull, 2); mbar_init(rempty, 1); mbar_init(sfull, 1); mbar_init(pfull, 8); mbar_init(qfull, LA_UNPACK); mbar_init(ofull, 1); mbar_init(oempty, 8);
    for (int i = 0; i < LA_AHEAD; ++i) { mbar_init(&xfull[i], 1); mbar_init(&xempty[i], LA_UNPACK + 2); }
    fence_mbar_init();
  }
  if (warp == LA_SOFT) {
    tmem_alloc(&ms.tmem, C::TMEM);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ms.tmem;
  pdl_wait();
  qabs = after_wait(qabs); cache = after_wait(cache); block_table = after_wait(block_table);
  g.slot = after_wait(g.slot); g.row0 = after_wait(g.row0); g.nrows = after_wait(g.nrows); g.kvlen = after_wait(g.kvlen);

  // ---- this CTA's share of the list, by every warp for itself (no barrier stands between the lengths and a role's first load): sums over the segments, a
  // lane each (a prompt's further blocks by the whole warp), of their places (low 40 bits) and units (the rest)
  constexpr long long PLACES = (1ll << 40) - 1;
  LatentWalk c;                                                      // a lane's segment, at its first block
  bool prompts = false;
  auto count = [&](int seg0) -> long long {                          // of segment seg0 + lane, where the lane's walk is then
    c.units = c.nrows = c.nt = c.left = c.extra = 0;
    if (seg0 + lane < g.nseg) {
      c.s = seg0 + lane;
      c.segment<N, true>(g);
    }
    long long sum = (long long)c.units * (c.nt + c.extra) + ((long long)c.units << 40);
#pragma unroll 1
    for (uint32_t more = __ballot_sync(0xffffffffu, c.left > 0); more; more &= more - 1) {
      const int from = __ffs(more) - 1;
      LatentWalk x;
      x.row0 = __shfl_sync(0xffffffffu, c.row0, from);
      x.left = __shfl_sync(0xffffffffu, c.left, from);
      long long rest = 0;
#pragma unroll 1
      while (x.left > 0) {
        x.next_block<N>(g);
        rest += (long long)x.units * (x.nt + 1) + ((long long)x.units << 40);
      }
      if (lane == from) sum += rest;
      c.over |= x.over;
      prompts = true;
    }
    return sum;
  };
  long long mine = 0, total = 0;
#pragma unroll 1
  for (int seg0 = 0; seg0 < g.nseg; seg0 += 32) total += mine = count(seg0);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  const int all = (int)(total & PLACES), share = max(1, (int)((uint32_t)(all + (int)gridDim.x - 1) / gridDim.x));
  const int f0 = min((int)blockIdx.x * share, all), f1 = min(f0 + share, all);
  const bool much = by_unit && (int)(total >> 40) > entries;         // segments of more rows than the caller said: nothing is written
  if (by_unit) {
    if (blockIdx.x == 0)
#pragma unroll 1
      for (int i = (much ? 0 : (int)(total >> 40)) + tid; i < entries; i += LA_THREADS) join[i] = make_int4(0, 0, 0, 0);
  } else if (tid == LA_UNPACK * 32) {                                // (the thread that may write another one there)
    join[blockIdx.x] = make_int4(0, 0, 0, 0);
  }
  if (blockIdx.x == 0 && warp == 0 && c.over) set_status(status, ST_BOUNDS);
  if (f0 == f1 || much) {                                          // the same for the whole CTA
    if (tid == 0 && much) set_status(status, ST_CAPACITY);
    if (warp == LA_SOFT) tmem_dealloc(tmem, C::TMEM);
    return;
  }
  // Where the share starts, and how many tiles it has: its places without those that a prompt's units count beside their tiles, of which `gone` lie ahead of
  // a place (of f1 first, then of f0, where the walk stays)
  LatentWalk w;
  int unit = 0, gone1 = 0, gone = 0;
#pragma unroll 1
  for (int f = prompts ? f1 : f0;; f = f0) {
    long long done = 0;
    gone = 0;
#pragma unroll 1
    for (int seg0 = 0; seg0 < g.nseg; seg0 += 32) {
      if (g.nseg > 32) mine = count(seg0);
      long long end = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, end, o);
        if (lane >= o) end += v;
      }
      end += done;
      const uint32_t hit = __ballot_sync(0xffffffffu, f < (int)(end & PLACES));
      const int from = hit ? __ffs(hit) - 1 : 32;
      if (prompts) gone += __reduce_add_sync(0xffffffffu, lane < from && c.extra ? (int)(mine >> 40) : 0);
      if (hit) {
        auto of = [&](int v) { return __shfl_sync(0xffffffffu, v, from); };
        int at = of(f - (int)(end - mine & PLACES));
        unit = of((int)(end - mine >> 40));
        w.s = seg0 + from; w.units = of(c.units); w.nt = of(c.nt); w.kv = of(c.kv); w.row0 = of(c.row0); w.nrows = of(c.nrows); w.slot = of(c.slot);
        w.left = of(c.left); w.extra = of(c.extra);
#pragma unroll 1
        while (w.left > 0 && at >= w.units * (w.nt + 1)) {
          at -= w.units * (w.nt + 1);
          unit += w.units;
          gone += w.units;
          w.next_block<N>(g);
        }
        w.u = (int)((uint32_t)at / (uint32_t)(w.nt + w.extra));
        w.t = at - w.u * (w.nt + w.extra);
        unit += w.u;
        if (w.extra) gone += w.u;
        break;
      }
      done = __shfl_sync(0xffffffffu, end, 31);
    }
    if (f == f0) break;
    gone1 = gone;
  }
  int flat = f0;
  if (w.t == w.nt) {                                                 // (a place that is no tile)
    w.next_unit<N>(g);
    ++unit;
    ++flat;
  }
  const int tiles = prompts ? f1 - f0 - (gone1 - gone) : f1 - f0;
  if (tiles <= 0) {                                                  // the same for the whole CTA
    if (warp == LA_SOFT) tmem_dealloc(tmem, C::TMEM);
    return;
  }

  // Queries of the walk's unit -> shared memory, and what belongs to each pair. Eight lanes have a pair; a thread turns the 16-byte pieces that it copied
  // itself, in their places. The first piece's are brought by the unpacking warps, while their first codes are on their way (before: copies, after: the
  // rest), the others' by the softmax. (Loops, not unrolled ones: a CTA comes by once or twice, and code that is new to the SM costs more than its instructions.)
  auto pairs_of = [&](const LatentWalk& x) { return min(N, x.nrows * g.nq - x.u * N); };
  auto place = [&](int n, int c) { return smem + (c * N + n) * 128 + (((lane & 7) ^ (n & 7)) << 4); };
  auto copy_q = [&](int n0, int step) {
    const int np = pairs_of(w);
    const __nv_bfloat16* q0 = qabs + ((size_t)w.row0 * g.nq + (size_t)w.u * N) * D + (lane & 7) * 8;
#pragma unroll 1
    for (int n = n0; n < N; n += step)
#pragma unroll 3
      for (int c = 0; c <= NC; ++c)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                     ::"r"(smem_u32(place(n, c))), "l"(q0 + (size_t)(n < np ? n : 0) * D + c * 64), "r"(n < np ? 16 : 0) : "memory");
  };
  auto turn_q = [&](int n0, int step, int par) {
    const int np = pairs_of(w);
    asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 1
    for (int n = n0; n < N; n += step) {
      __nv_bfloat162 most = __float2bfloat162_rn(0.f);
#pragma unroll 3
      for (int c = 0; c <= NC; ++c) {
        const uint4 u = *reinterpret_cast<const uint4*>(place(n, c));
        const uint32_t a[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) most = __hmax2(most, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&a[e])));
      }
      float top = fmaxf(__low2float(most), __high2float(most));
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      int ex = (int)(__float_as_uint(top) >> 23) - 127;
      ex = top == 0.f || ex > 127 ? 10 : max(ex, -110);                           // (a value that is no number stays one)
      const float mul = __uint_as_float((uint32_t)(10 - ex + 127) << 23);
#pragma unroll 3
      for (int c = 0; c <= NC; ++c) {
        uint4* at = reinterpret_cast<uint4*>(place(n, c));
        const uint4 u = *at;
        const uint32_t a[4] = {u.x, u.y, u.z, u.w};
        uint32_t o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float lo = bf_lo(a[e]) * mul, hi = bf_hi(a[e]) * mul;
          const __half2 h = __floats2half2_rn(lo, hi);
          o[e] = c < NC ? *reinterpret_cast<const uint32_t*>(&h) : pack_bf2(lo, hi);
        }
        *at = make_uint4(o[0], o[1], o[2], o[3]);
      }
      if ((lane & 7) == 0) {
        ms.c[par][n] = scale_log2 * __uint_as_float((uint32_t)(ex - 10 + 127) << 23);
        ms.nr[par][n] = 0.f;
        ms.see[par][n] = n < np ? min(max(g.kvlen[w.row0 + (int)((uint32_t)(w.u * N + n) / (uint32_t)g.nq)], 0), w.kv) : w.kv;
      }
    }
    fence_proxy_async();
    __syncwarp();
  };

  // launched with 72 registers for 896 threads (64512); sixteen warps of 56, eight of 112 and four of 56 are as many
  if (warp < LA_UNPACK) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    // ---- unpack: lanes 4 r + p of a warp have key r of its eight, part p of every pair of 64 values (unpack32), so that a load takes 64 bytes of eight
    // rows each. Codes and scales are a tile ahead in registers. A key that is not there reads row 0 in 4 bits, where any byte is some
    // number: it has no weight. (8 bits have codes that are none: zeros.)
    const int r8 = lane >> 2, p = lane & 3;
    const bool up = BITS == 4 && p >= 2;
    uint32_t at[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      at[q] = (warp * 8 + r8) * 128 + (BITS == 4 ? (p / 2) * LA_CH + ((((p & 1) * 4 + (up ? 2 : 0)) ^ r8 ^ q) << 4)
                                                  : (q / 2) * LA_CH + (((2 * p) ^ r8 ^ (q & 1)) << 4));
    const uint32_t ak = smem_u32(smem + C::K_AT);
    const uint8_t* const codes = cache + p * 16;
    const uint8_t* const bytes = cache + Row::scale_at(L) + (BITS == 4 ? (p & 1) * 2 * NC : (p >> 1) * NC);
    uint4 raw[C::PD][BITS / 4];
    auto fetch = [&](uint4 (&r)[BITS / 4], int row, int j) {
      if constexpr (BITS == 4) {
        if (2 * j + 1 < NC || p < 2) r[0] = ldg_stream(codes + (size_t)max(row, 0) * RB + j * 64);
      } else {
        const uint8_t* from = codes + (size_t)max(row, 0) * RB + j * 128;
        r[0] = row >= 0 ? ldg_stream(from) : make_uint4(0, 0, 0, 0);
        if (2 * j + 1 < NC) r[1] = row >= 0 ? ldg_stream(from + 64) : make_uint4(0, 0, 0, 0);
      }
    };
    // scale bytes of a key, as they come (arithmetic on them here would wait for them): a word has those of two pairs
    constexpr int SRW = NC == 8 && BITS == 4 ? 4 : NC == 8 ? 2 : NP, SCW = (NP + 1) / 2;
    auto scales = [&](uint32_t (&v)[SRW], int row) {
      const uint8_t* from = bytes + (size_t)max(row, 0) * RB;
      if constexpr (NC == 8 && BITS == 4) {
        const uint4 u = ldg_stream(from);
        v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
      } else if constexpr (NC == 8) {
        const uint2 u = ldg_stream8(from);
        v[0] = u.x; v[1] = u.y;
      } else {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          v[j] = 0;
          if constexpr (BITS == 4) {
            if (2 * j + 1 < NC || p < 2) asm volatile("ld.global.nc.u16 %0, [%1];" : "=r"(v[j]) : "l"(from + 4 * j + (p >> 1) * 2));
          } else if (2 * j + 1 < NC) {
            asm volatile("ld.global.nc.u16 %0, [%1];" : "=r"(v[j]) : "l"(from + 2 * j));
          } else {
            asm volatile("ld.global.nc.u8 %0, [%1];" : "=r"(v[j]) : "l"(from + 2 * j));
          }
        }
      }
    };
    auto pairs_of_bytes = [&](uint32_t (&v)[SCW], const uint32_t (&u)[SRW]) {
      if constexpr (NC == 8 && BITS == 4) {
        const uint32_t pick = p >= 2 ? 0x7632u : 0x5410u;
        v[0] = __byte_perm(u[0], u[1], pick);
        v[1] = __byte_perm(u[2], u[3], pick);
      } else if constexpr (NC == 8) {
        v[0] = u[0]; v[1] = u[1];
      } else {
#pragma unroll
        for (int j = 0; j < NP; j += 2) v[j / 2] = j + 1 < NP ? u[j] | u[j + 1] << 16 : u[j];
      }
    };
    bool ok = true;
    auto look = [&](int i) -> int {                                      // the key's row of the cache, from the warp that looks them up
      ok = ok && la_wait(&xfull[i % LA_AHEAD], i / LA_AHEAD & 1, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      const int row = ms.rows[i % LA_AHEAD][warp * 8 + r8];
      __syncwarp();
      if (lane == 0) mbar_arrive(&xempty[i % LA_AHEAD]);
      return ok ? row : -1;
    };
    if (warp * 4 < N) copy_q(warp * 4 + (lane >> 3), N);
    int row0 = look(0), row1 = -1;
    uint32_t sraw[SRW];
#pragma unroll
    for (int j = 0; j < C::PD; ++j) fetch(raw[j], row0, j);
    scales(sraw, row0);
    if (warp * 4 < N) turn_q(warp * 4 + (lane >> 3), N, 1);
    if (lane == 0) mbar_arrive(qfull);
    int buf = 0;
    uint32_t kph = 1;                                                // (a fresh barrier passes a wait for parity 1)
    for (int i = 0; i < tiles; ++i) {
      if (i + 1 < tiles) row1 = look(i + 1);
      uint32_t sc[SCW], nan = 0;
      pairs_of_bytes(sc, sraw);
      scales(sraw, row1);
#pragma unroll
      for (int j = 0; j < SCW; ++j) {
        const uint32_t m = __vcmpgeu4(sc[j], BITS == 4 ? 0xf8f8f8f8u : 0x87878787u);
        nan |= m;
        sc[j] &= ~m;
      }
      nan = __ballot_sync(0xffffffffu, nan != 0);
      if (lane == 0) ms.bad[i & 3][warp] = nan;
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        ok = ok && la_wait(&kempty[buf], kph, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        if (BITS == 8 || 2 * j + 1 < NC || p < 2)
          unpack32<BITS>(raw[j % C::PD], sc[j / 2] >> (16 * (j % 2)) & 0xffffu, ak + buf * 2 * LA_CH, at, up, 2 * j + 1 < NC);
        if (j + C::PD < NP) fetch(raw[j % C::PD], row0, j + C::PD);
        else fetch(raw[j % C::PD], row1, j + C::PD - NP);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&kfull[buf]);
        if (++buf == NB) { buf = 0; kph ^= 1; }
      }
      if (!ok) break;
      row0 = row1;
    }
    if (!ok) { set_status(status, ST_MBAR_TIMEOUT); *abort_flag = 1; }
  } else if (warp < LA_SOFT) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
    // ---- softmax: thread = (key, half of the pairs) ----------------------------------------------------------------------------------------------
    constexpr int W = CW < 16 ? CW : 16;                             // pairs in registers at a time
    const int quad = warp & 3, hc = (warp - LA_UNPACK) >> 2, st = tid - LA_UNPACK * 32, key = quad * 32 + lane;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16, ts = tmem + lanes + NP * N + hc * CW, to = tmem + lanes + hc * CW;
    auto fmx = [](float a, float b) { return fmaxf(a, b); };
    auto fad = [](float a, float b) { return a + b; };
    int i = 0;
    bool broke = false;
    la_wait(qfull, 0, abort_flag);                                   // what came with the first piece's queries (if they don't come, no score does either)
    // once round per piece: its tiles, the next one's queries (no score needs this one's any more), its end
    for (int piece = 1;; ++piece) {
      const int par = piece & 1, t0 = w.t, nt = w.nt, np = pairs_of(w), n = min(nt - t0, tiles - i), places = n + (t0 + n == nt ? w.extra : 0);
      const size_t base = (size_t)w.row0 * g.nq + (size_t)w.u * N;
      uint64_t sum[CW / 2];
      {
        softmax_sync();                                              // what came with later pieces' queries, from these warps
        if (const int m = __reduce_min_sync(0xffffffffu, ms.see[par][hc * CW + lane % CW]); lane == 0) ms.least[warp - LA_UNPACK] = m;
        __syncwarp();
        const int least = ms.least[warp - LA_UNPACK];                // (read where it is needed: a register more, and eight-bit variants spill 300 bytes)
#pragma unroll
        for (int e = 0; e < CW / 2; ++e) sum[e] = f2_pack(0.f, 0.f);
#pragma unroll 1
        for (int k = 0; k < n; ++k, ++i) {
          bool ok = la_wait(sfull, i & 1, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
          tc_fence_after();
          const int at = (t0 + k) * LA_KT + key;
          const bool edge = (t0 + k + 1) * LA_KT > least, none = ms.bad[i & 3][key >> 3] >> (4 * (key & 7)) & 15u;
          // log2 of the thread's weights, up to the reference or (`bare`) without it. The product is rounded ahead of the sum: the largest score minus itself
          // is then nothing, however large it is (in one fma the product's rounding would be left, 2^-24 of the score, as if it were a weight).
          auto scores = [&](float (&x)[CW], bool bare) {
            const uint64_t zero = f2_pack(0.f, 0.f);                 // (a product and a sum that follows may be made one; a sum of two may not)
            uint32_t r[CW];
            tmem_ld<CW>(ts, r);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < CW; e += 4) {
              const float4 c = *reinterpret_cast<const float4*>(&ms.c[par][hc * CW + e]);
              const float4 nr = bare ? make_float4(0.f, 0.f, 0.f, 0.f) : *reinterpret_cast<const float4*>(&ms.nr[par][hc * CW + e]);
              const float2 a = f2_unpack(f2_add(f2_fma(f2_pack(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), f2_pack(c.x, c.y), zero), f2_pack(nr.x, nr.y)));
              const float2 b = f2_unpack(f2_add(f2_fma(f2_pack(__uint_as_float(r[e + 2]), __uint_as_float(r[e + 3])), f2_pack(c.z, c.w), zero), f2_pack(nr.z, nr.w)));
              x[e] = a.x; x[e + 1] = a.y; x[e + 2] = b.x; x[e + 3] = b.y;
            }
            if (none) {
#pragma unroll
              for (int e = 0; e < CW; ++e) x[e] = __uint_as_float(0x7fc00000u);
            }
            if (edge) {
#pragma unroll
              for (int e = 0; e < CW; ++e)
                if (at >= ms.see[par][hc * CW + e]) x[e] = -INFINITY;
            }
          };
          unsigned char* prow = smem + C::P_AT + key * N * 2;
          const int pturn = N == 64 ? key & 7 : N == 32 ? key >> 1 & 3 : key >> 2 & 1;
          // Weights by the reference there is; a tile whose scores pass the limit (all 256 threads look) and a piece's first (load_q left zeros) get one anew
          // and go round again, once: scores so large that their difference to it is still past the limit, for rounding, weigh the limit.
          bool anew = k == 0, again = false, done = false;
#pragma unroll 1
          while (!done) {
            float x[CW];
            scores(x, anew);
            if (anew) {
              if (!ok) ms.fail = 1;
              if (k > 0) {                                           // the tile's weights leave the sums again: what they rounded off is 2^-24 of the largest
#pragma unroll
                for (int e = 0; e < CW; e += 2) {
                  const float2 nr = *reinterpret_cast<const float2*>(&ms.nr[par][hc * CW + e]), l = f2_unpack(sum[e / 2]);
                  sum[e / 2] = f2_pack(l.x - ex2(x[e] + nr.x), l.y - ex2(x[e + 1] + nr.y));
                }
              }
              const float m = columns<CW>(x, lane, fmx);
              if (lane < CW) ms.mx[quad][hc * CW + lane] = m;
              softmax_sync();
              if (ms.fail) break;
              if (st < N) {
                const float most = fmaxf(fmaxf(ms.mx[0][st], ms.mx[1][st]), fmaxf(ms.mx[2][st], ms.mx[3][st]));
                const float was = -ms.nr[par][st], to = most - LA_TOP;
                const bool up = k == 0 ? most > -INFINITY : to > was;
                ms.d[st] = up ? to - was : 0.f;
                if (up) ms.nr[par][st] = -to;
              }
              softmax_sync();
              anew = false;
              again = true;
              if (k > 0) {                                           // (the tile's scores are complete, so the products ahead of them are)
#pragma unroll
                for (int e = 0; e < CW; e += 2) {
                  const float2 d = *reinterpret_cast<const float2*>(&ms.d[hc * CW + e]), l = f2_unpack(sum[e / 2]);       // (sums of 2^-100 are none)
                  sum[e / 2] = f2_pack(d.x > 100.f ? 0.f : l.x * ex2(-d.x), d.y > 100.f ? 0.f : l.y * ex2(-d.y));
                }
#pragma unroll 1
                for (int j = 0; j < NP * CW; j += W) {
                  uint32_t o[W];
                  tmem_ld<W>(to + j / CW * N + j % CW, o);
                  tmem_ld_wait();
#pragma unroll
                  for (int e = 0; e < W; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * ex2(-ms.d[hc * CW + j % CW + e]));
                  tmem_st<W>(to + j / CW * N + j % CW, o);
                }
                tmem_st_wait();
              }
              continue;
            }
            if (again) {
#pragma unroll
              for (int e = 0; e < CW; ++e) x[e] = x[e] > LA_LIMIT ? LA_LIMIT : x[e];
            }
            float top = x[0];
#pragma unroll
            for (int h = 0; h < CW; h += 8) {
              uint32_t pw[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                top = fmaxf(top, fmaxf(x[h + 2 * e], x[h + 2 * e + 1]));
                const float a = ex2(x[h + 2 * e]), b = ex2(x[h + 2 * e + 1]);
                sum[h / 2 + e] = f2_add(sum[h / 2 + e], f2_pack(a, b));
                const __half2 p2 = __floats2half2_rn(a, b);
                pw[e] = *reinterpret_cast<const uint32_t*>(&p2);
              }
              *reinterpret_cast<uint4*>(prow + (((hc * (CW / 8) + h / 8) ^ pturn) << 4)) = make_uint4(pw[0], pw[1], pw[2], pw[3]);
            }
            anew = softmax_any(!ok || top > LA_LIMIT);
            done = !anew;
          }
          if (!done) { broke = true; break; }
          tc_fence_before();
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(pfull);
        }
        if (broke) break;
        float a[CW];
#pragma unroll
        for (int e = 0; e < CW / 2; ++e) {
          const float2 x = f2_unpack(sum[e]);
          a[2 * e] = x.x; a[2 * e + 1] = x.y;
        }
        const float l = columns<CW>(a, lane, fad);
        if (lane < CW) ms.mx[quad][hc * CW + lane] = l;
        if (t0 + n == nt) w.next_unit<N>(g);
      }
      if (i < tiles) {
        copy_q((warp - LA_UNPACK) * 4 + (lane >> 3), 32);
        turn_q((warp - LA_UNPACK) * 4 + (lane >> 3), 32, piece + 1 & 1);
        if (lane < 2) mbar_arrive(qfull);
      }
      // ---- the piece's end
      const bool whole = t0 == 0 && n == nt;
      bool ok = la_wait(ofull, piece - 1 & 1, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) ms.fail = 1;
      softmax_sync();
      if (ms.fail) { broke = true; break; }
      const int rec = 2 * (int)blockIdx.x + (t0 > 0 ? 0 : 1);
      if (st < N) {
        const float lt = ms.mx[0][st] + ms.mx[1][st] + ms.mx[2][st] + ms.mx[3][st];
        // no weight at all: nothing to see (zeros), or every score is -inf (0 / 0)
        ms.d[st] = ms.see[par][st] == 0 ? 0.f : 1.f / lt * (lt == 0.f ? 0.f : 1.f);
        if (!whole) {
          float* ml = ml_part + ((size_t)rec * N + st) * 2;
          ml[0] = lt == 0.f ? -INFINITY : -ms.nr[par][st];
          ml[1] = lt;
        }
      }
      if (st == 0 && t0 == 0 && (by_unit || !whole))
        join[by_unit ? unit : (int)blockIdx.x] = make_int4((int)base, whole ? 0 : np, rec, (int)((uint32_t)(flat + nt - 1) / (uint32_t)share));
      if (t0 + n == nt) ++unit;
      flat += places;
      softmax_sync();
      tc_fence_after();
#pragma unroll 1
      for (int j = 0; j < NP * CW; j += W) {
        uint32_t o[W];
        const int n0 = hc * CW + j % CW, e0 = j / CW * 128 + quad * 32 + lane;
        tmem_ld<W>(to + j / CW * N + j % CW, o);
        tmem_ld_wait();
        if (e0 < L) {
          if (whole) {
            __nv_bfloat16* dst = out + (base + n0) * L + e0;
#pragma unroll
            for (int e = 0; e < W; ++e)
              if (n0 + e < np) dst[(size_t)e * L] = f2bf(__uint_as_float(o[e]) * ms.d[n0 + e]);
          } else {
            float* dst = o_part + ((size_t)rec * N + n0) * L + e0;
#pragma unroll
            for (int e = 0; e < W; ++e)
              if (n0 + e < np) dst[(size_t)e * L] = __uint_as_float(o[e]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(oempty);
      if (i >= tiles) break;
    }
    if (broke && st == 0) { set_status(status, ST_MBAR_TIMEOUT); *abort_flag = 1; }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == LA_SOFT) {
      // ---- products: the whole warp, one lane of it by predicate ------------------------------------------------------------------------------------
      constexpr uint32_t id_s = umma_idesc(0, 0, 128, N), id_r = umma_idesc(1, 1, 128, N), id_o = umma_idesc(0, 0, 128, N) | 1u << 15 | 1u << 16;
      constexpr uint32_t P_ROW = N * 2, P_SW = N == 64 ? 2 : N == 32 ? 4 : 6;        // the weights' rows: swizzled over 128, 64 or 32 bytes
      const uint32_t aq = smem_u32(smem), ak = smem_u32(smem + C::K_AT), ar = smem_u32(smem + C::R_AT), ap = smem_u32(smem + C::P_AT);
      const uint32_t ts = tmem + NP * N;
      const bool issue = elect_one();
      auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, la_wait(bar, parity, abort_flag)); };
      int buf = 0, i = 0, piece = 0;
      uint32_t kph = 0;
      bool ok = true;
      while (ok && i < tiles) {
        const int n = min(w.nt - w.t, tiles - i);
        ok = wait(qfull, piece & 1);
        for (int k = 0; ok && k < n; ++k, ++i) {
          const int b0 = buf;
#pragma unroll 1
          for (int j = 0; j < NP; ++j) {
            if (!ok || !wait(&kfull[buf], kph)) { ok = false; break; }
            tc_fence_after();
            const uint64_t da = umma_desc_k128(ak + buf * 2 * LA_CH), db = umma_desc_k128(aq + j * 2 * N * 128);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)
              if (kk < 4 || 2 * j + 1 < NC)
                tc_mma_f16_if(issue, ts, da + ((kk / 4) * LA_CH + (kk & 3) * 32 >> 4), db + ((kk / 4) * N * 128 + (kk & 3) * 32 >> 4), id_s, j > 0 || kk > 0);
            if (++buf == NB) { buf = 0; kph ^= 1; }
          }
          if (!ok || !wait(rfull, i & 1)) { ok = false; break; }
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            tc_mma_f16_if(issue, ts, umma_desc_k128(ar + kk * 32), umma_desc_k128(aq + NC * N * 128 + kk * 32), id_r, 1u);
          tc_commit_if(issue, sfull);
          if (!C::SHARE) tc_commit_if(issue, rempty);
          if (!wait(pfull, i & 1) || (k == 0 && piece > 0 && !wait(oempty, (piece - 1) & 1))) { ok = false; break; }
          tc_fence_after();
          int b = b0;
          const uint64_t dp = umma_desc_mn(ap, 0, 8 * P_ROW, P_SW);
#pragma unroll 1
          for (int j = 0; j < NP; ++j) {
            const uint64_t dv = umma_desc_mn(ak + b * 2 * LA_CH, LA_CH, 1024, 2);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)
              tc_mma_f16_if(issue, tmem + j * N, dv + (kk * 2048 >> 4), dp + (kk * 16 * P_ROW >> 4), id_o, k > 0 || kk > 0);
            tc_commit_if(issue, &kempty[b]);
            if (++b == NB) b = 0;
          }
          if (C::SHARE) tc_commit_if(issue, rempty);
        }
        if (!ok) break;
        tc_commit_if(issue, ofull);
        ++piece;
        if (w.t + n == w.nt) w.next_unit<N>(g);                        // (else the list ends here)
      }
      if (!ok) {
        set_status(status, ST_MBAR_TIMEOUT);
        *abort_flag = 1;
        // products in flight end before their TMEM goes: a commit behind all of them, on a barrier that nobody else waits for any more
        tc_commit_if(issue, ofull);
        mbar_wait(ofull, piece & 1, 1u << 20);
      }
    } else if (warp == LA_SOFT + 3) {
      // ---- rows of the cache of the tiles' keys, four a lane
      bool ok = true;
      for (int i = 0; i < tiles; ++i) {
        int row[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int key = w.t * LA_KT + k * 32 + lane;
          row[k] = -1;
          if (key < w.kv) {
            const int at = key / kv_block, in = key - at * kv_block, blk = block_table[(size_t)w.slot * max_blocks + at];
            if (blk >= 0 && blk < pages) {
              row[k] = blk * kv_block + in;                            // (rows of a cache are fewer than 2^31)
              if (i > 0 && (in == 0 || k * 32 + lane == 0)) {          // the tile's rows of a page lie together: one request brings them to L2
                const int n = min(kv_block - in, min((w.t + 1) * LA_KT, w.kv) - key);
                asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(cache + (size_t)row[k] * RB), "r"(n * RB) : "memory");
              }
            } else {
              set_status(status, ST_BOUNDS);
            }
          }
        }
        ok = la_wait(&xempty[i % LA_AHEAD], (i / LA_AHEAD & 1) ^ 1, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
#pragma unroll
        for (int k = 0; k < 4; ++k) ms.rows[i % LA_AHEAD][k * 32 + lane] = row[k];
        __syncwarp();
        if (lane == 0) mbar_arrive(&xfull[i % LA_AHEAD]);
        if (++w.t == w.nt) w.next_unit<N>(g);
      }
      if (!ok) { set_status(status, ST_MBAR_TIMEOUT); *abort_flag = 1; }
    } else {
      // ---- key parts: a warp copies those of 64 keys as they are, eight lanes a row. Their place is free late and they are needed last, so they go straight
      // to shared memory.
      bool ok = true;
      for (int i = 0; i < tiles; ++i) {
        ok = la_wait(&xfull[i % LA_AHEAD], i / LA_AHEAD & 1, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        ok = la_wait(rempty, (i & 1) ^ 1, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
#pragma unroll 4
        for (int m = 0; m < 16; ++m) {
          const int key = (warp - LA_SOFT - 1) * 64 + m * 4 + (lane >> 3), r = ms.rows[i % LA_AHEAD][key];
          const uint32_t to = smem_u32(smem + C::R_AT) + key * 128 + (((lane & 7) ^ (key & 7)) << 4);
          // (no bytes, zeros in their place, where there is no row)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                       ::"r"(to), "l"(cache + (size_t)max(r, 0) * RB + Row::rope_at(L) + (lane & 7) * 16), "r"(r >= 0 ? 16 : 0) : "memory");
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&xempty[i % LA_AHEAD]);
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(rfull);
      }
      if (!ok) { set_status(status, ST_MBAR_TIMEOUT); *abort_flag = 1; }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == LA_SOFT) tmem_dealloc(tmem, C::TMEM);
}

// Units that span CTAs. grid (entries, N), 128 threads: a CTA a pair, its records in the order of their keys.
__global__ void __launch_bounds__(128) mla_attn_q_join_kernel(__nv_bfloat16* __restrict__ out, const float* o_part, const float* ml_part, const int4* join,
                                                              int N, int L, const int* row_kvlen, long pairs, int nq, int ctas) {
  const int n = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  pdl_launch_dependents();
  pdl_wait();
  o_part = after_wait(o_part); ml_part = after_wait(ml_part); row_kvlen = after_wait(row_kvlen);
  const int4 job = after_wait(join)[blockIdx.x];
  // (where a wait ran out in the kernel ahead, jobs are whatever was there)
  const int c0 = job.z >> 1, count = job.w - c0 + 1;
  if (n >= job.y || job.x < 0 || (long)job.x + n >= pairs || job.z < 0 || job.w >= ctas || count < 1 || count > ctas) return;
  auto record = [&](int i) { return (size_t)(i == 0 ? job.z : 2 * (c0 + i)) * N + n; };
  // The sums of eight records are on their way while the weights are worked out, by every warp for itself, 32 records at a time.
  constexpr int AT_ONCE = 8;
  const int e = tid * 4;
  float4 v[AT_ONCE], a = make_float4(0.f, 0.f, 0.f, 0.f);
  auto load = [&](int i0) {
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k)
      if (i0 + k < count && e < L) v[k] = *reinterpret_cast<const float4*>(o_part + record(i0 + k) * L + e);
  };
  load(0);
  float m = -INFINITY, l = 0.f, x = 0.f;
#pragma unroll 1
  for (int i = lane; i < count; i += 32) m = fmaxf(m, ml_part[record(i) * 2]);
  m = warp_max(m);
#pragma unroll 1
  for (int i0 = 0; i0 < count; i0 += AT_ONCE) {
    if (i0 % 32 == 0) {
      // a record without weight has -inf there; a reference of +inf comes with sums that are no numbers
      const float2 ml = i0 + lane < count ? *reinterpret_cast<const float2*>(ml_part + record(i0 + lane) * 2) : make_float2(-INFINITY, 0.f);
      x = ml.x == -INFINITY ? 0.f : ml.x == m ? 1.f : exp2f(ml.x - m);
      l += x == 0.f ? 0.f : x * ml.y;
    }
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      // (a record that weighs nothing is multiplied all the same: sums that are no numbers have seen a key that is none, and so has the row)
      const float y = __shfl_sync(0xffffffffu, x, (i0 + k) % 32);
      if (i0 + k < count) { a.x = fmaf(y, v[k].x, a.x); a.y = fmaf(y, v[k].y, a.y); a.z = fmaf(y, v[k].z, a.z); a.w = fmaf(y, v[k].w, a.w); }
    }
    load(i0 + AT_ONCE);
  }
  l = warp_sum(l);
  const size_t pair = (size_t)job.x + n;
  const float inv = row_kvlen[pair / nq] > 0 ? 1.f / l * (l == 0.f ? 0.f : 1.f) : 0.f;
  if (e < L) *reinterpret_cast<uint2*>(out + pair * L + e) = make_uint2(pack_bf2(a.x * inv, a.y * inv), pack_bf2(a.z * inv, a.w * inv));
}

}  // namespace fb

using namespace fb;

// Pairs of a unit: the fewest of 16, 32 and 64 that hold a segment's; more are several units (an unpacked tile serves as many as it can). Fewer where even
// then every tile that the table has room for finds a CTA of its own: its products, its softmax and the sums that it leaves are shorter, and nobody
// waits for the unpacking that is done again. It is the TABLE's room that counts, not the context, which only the device knows: one stream of 2048 with 128
// heads takes 21.0 us in a table for no more (units of 16), 21.9 in one for 4096 tokens (32), 24.6 from 8192 on (64).
static int latent_pairs(long pairs, long tiles, int ctas) {
  int N = 16;
  while (N < 64 && N < pairs && (pairs + N - 1) / N * tiles > ctas) N *= 2;
  return N;
}

extern "C" long fb_mla_attn_q_floats(int max_rows, int nq, int L, int ctas) {
  const long N = latent_pairs((long)max_rows * nq, 1l << 31, ctas);       // (the most that they can be)
  return 4l * ctas + 2l * ctas * N * (L + 2);
}

// ws: fb_mla_attn_q_floats of 32 bits
extern "C" int fb_mla_attn_q(void* out, float* ws, long ws_floats, const void* qabs, const void* cache, long pages, int bits, const int* seg_slot,
                             const int* seg_row0, const int* seg_nrows, int nseg, int max_rows, const int* row_kvlen, const int* block_table,
                             int max_blocks, int kv_block, int rows, int nq, int L, int R, float scale, int ctas, int* status, cudaStream_t s) {
  if (R != LC_R || (bits != 4 && bits != 8) || nq < 1 || kv_block < 1 || ctas < 1 || max_rows < 0) return -1;
  if (((uintptr_t)qabs | (uintptr_t)cache | (uintptr_t)ws) % 16 || (uintptr_t)out % 8) return -2;
  if (pages < 1 || pages * kv_block > 0x7fffffffl || (long)rows * nq > 0x3fffffffl) return -2;
  if (rows <= 0 || nseg <= 0 || max_rows == 0) return 0;
  if (ws_floats < fb_mla_attn_q_floats(max_rows, nq, L, ctas)) return -3;
  const int N = latent_pairs((long)max_rows * nq, nseg * std::max(1l, ((long)max_blocks * kv_block + LA_KT - 1) / LA_KT), ctas);
  const long units = (long)nseg * (((long)max_rows * nq + N - 1) / N);
  const int by_unit = units <= ctas, entries = by_unit ? (int)units : ctas;
  int4* join = reinterpret_cast<int4*>(ws);
  float *ml = ws + 4l * ctas, *op = ml + 2l * ctas * N * 2;
  const LatentSegs g{seg_slot, seg_row0, seg_nrows, row_kvlen, nseg, nq, (long)max_blocks * kv_block};
  cudaError_t e = cudaErrorInvalidValue;
  bool known = false;
#define FB_LA(B, NCV, NV)                                                                                                                        \
  if (bits == B && L == NCV * 64 && N == NV) {                                                                                                   \
    auto kern = mla_attn_q_kernel<B, NCV, NV>;                                                                                                   \
    const size_t smem = LatentAttn<B, NCV, NV>::MISC_AT + sizeof(LatentAttnMisc<NV>);                                                            \
    FB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));                                           \
    e = launch_pdl(kern, dim3(ctas), dim3(LA_THREADS), smem, s, (__nv_bfloat16*)out, op, ml, join, entries, by_unit, (const __nv_bfloat16*)qabs, \
                   (const uint8_t*)cache, g, block_table, max_blocks, pages, kv_block, scale * 1.4426950408889634f, status);                     \
    known = true;                                                                                                                                \
  }
#define FB_LA_N(B, NCV) FB_LA(B, NCV, 16) FB_LA(B, NCV, 32) FB_LA(B, NCV, 64)
  FB_LA_N(4, 8) FB_LA_N(4, 4) FB_LA_N(4, 2) FB_LA_N(4, 1) FB_LA_N(8, 8) FB_LA_N(8, 4) FB_LA_N(8, 2) FB_LA_N(8, 1)
#undef FB_LA_N
#undef FB_LA
  if (!known) return -2;
  if (e != cudaSuccess) return (int)e;
  return (int)launch_pdl(mla_attn_q_join_kernel, dim3(entries, N), dim3(128), 0, s, (__nv_bfloat16*)out, (const float*)op,
                         (const float*)ml, (const int4*)join, N, L, row_kvlen, (long)rows * nq, nq, ctas);
}

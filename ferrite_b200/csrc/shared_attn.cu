// Attention of a step's rows over a paged cache in which streams share the pages of a prefix, on the 5th-generation tensor cores: the keys and values of a
// prefix are read once for every 128 (row, head) pairs of its group.
//
//   S = Q K^T        128 (row, head) pairs of a block x 64 keys; Q and K in shared memory
//   P = exp2(S - m)  two threads a pair; P as bf16 and what that leaves, as bf16 too, back into TMEM, its sums in 32 bits. (Without the remainders a weight is off by up
//                    to 2^-8 of it, errors of either sign that add up to what rounding the output costs once more: 0.0024 instead of 0.0017 from the result
//                    in 64 bits. Their product costs 512 cycles of the tensor cores a tile of 128 pairs and 256 columns, 6 to 14 % of a long call.)
//   O += P V         A = P from TMEM, V read along its columns from shared memory, O in TMEM while the CTA stays with the pairs
//
// Work (shared_kv.cuh): every CTA takes the same number of consecutive key tiles of the list of all (block, kv head) units. A unit that a CTA leaves or ends
// is a piece: its running maximum, sum and O in 32 bits go to the workspace, and a second kernel joins a row's pieces (of its group's shared tokens, then
// of its own) in the order of the list. Where the contexts are cut follows the step's lengths, so a row may round differently beside other streams; the
// same call gives the same bits.
//
// Warp roles: 0 loads keys, 2 loads values, 1 issues the products of S, 3 those of O, 4..19 run the softmax, bring the queries and write the pieces. The
// softmax of a tile is a chain of waits, and its exponentials alone take 512 cycles of the SM: two sets of eight warps take a tile in turn, each with a
// buffer of S and P of its own, so that one set's chain hides behind the other's. They share O and the maximum that it belongs to. The maximum moves only
// when a score of some row exceeds it by 2^16 (a vote of the threads of 32 pairs, who exchange their maxima only then); sets decide in the tiles' order (`turn`), and the one
// that moves it rescales O between the two products. Every wait is bounded: one that runs out sets the status word and an abort flag; the softmax warps
// then go through their remaining barriers without work, the others leave, and the CTA frees its TMEM.
//
// Measured (B200, us a call, on the same inputs again / on others each time): 34 rows x 24 heads of 256 over 30000 shared and 2000 own tokens each 100 / 115 (bytes alone
// 48), 64 x 32 of 128 over 60000 and 500 141 / 166 (52), six over 8000 and 900 27 / 29 (7.5). The first is 45 tiles a CTA, 3040 cycles each with plan, first loads and
// pieces, of which the tensor pipe is busy for the 1536 that the operations take; the second 122 of 1830 and 768. What the sets hand over to each other for every tile
// sets the pace, and a tile of a stream's own tokens takes as long with its few pairs as one with 128. Four sets of four warps (twice the scores a thread) spill and are
// slower.
#include <algorithm>
#include <cfloat>

#include "gemm_core.cuh"
#include "shared_kv.cuh"

namespace fb {

constexpr int SA_PAIRS = 128, SA_KT = 64, SA_NEAR = 4;
constexpr int SA_EXTRA = 3;                                  // places of a unit's queries and piece, in key tiles (2 to 5 measure alike)
constexpr int SA_SET = 8;                                    // warps of a set: two threads a pair, each with half of a tile's keys
constexpr int SA_THREADS = (4 + 2 * SA_SET) * 32;
constexpr int SA_ML = 8;                                     // floats of a pair's statistics: its threads' sums, the maximum, a byte a thread (see `hidden`)

template <int HD>
struct SaCfg {
  static constexpr int NCH = HD / 64, Q_CH = SA_PAIRS * 128, KV_CH = SA_KT * 128;
  static constexpr int Q_BYTES = NCH * Q_CH, T_BYTES = NCH * KV_CH;
  static constexpr int KS = HD == 256 ? 3 : HD == 128 ? 6 : 8, VS = HD == 256 ? 2 : HD == 128 ? 5 : 8;
  static constexpr int TILES = Q_BYTES + (KS + VS) * T_BYTES;
  static constexpr int MISC_AT = TILES > SK_PLAN_BYTES ? TILES : SK_PLAN_BYTES;
  // TMEM: O | S0 S1 | P0 and its remainders, P1 and its
  static constexpr uint32_t COL_S = HD, COL_P = COL_S + 2 * SA_KT, COLS = 512;
};
// A CTA's share of the list: block that it starts in, blocks of groups, its first place, places.
struct SaShare {
  int b0, group_blocks, places;
  long long f0;
};
template <int STAGES>
struct SaMisc {
  float mx[2][SA_PAIRS], m[SA_PAIRS];            // maxima of a tile's halves (of the set whose turn it is); the maximum that O belongs to (log2)
  long long tmp[SA_THREADS / 32];
  uint64_t bars[22 + 2 * STAGES];
  uint8_t bad[2][2][8];                          // by set and turn: keys of a tile that lost values which are no finite numbers
  uint32_t tmem;
  int abort;
  SaShare share;
  SharedBlock blocks[SA_NEAR];                   // the first ones of the CTA's share; what follows is in the workspace
};

// Where things lie in the workspace. ml: sums of the pair's threads, maximum (log2); records of 128 pairs for groups, of seg_pairs for segments.
struct SaSpace {
  long long* head;                               // places a CTA, blocks of groups
  SharedBlock* table;
  int4* rows;                                    // [rows][2]: of a row's group, of its segment: place in the list of one kv head, tiles (0: none), unit, row of the block
  float *ml_grp, *ml_seg;                        // SA_ML floats a pair
  float *o_grp, *o_seg;
  float2* ml;                                    // logarithms alone: [record][half of the pairs][128][thread] maximum, sum
  SharedPlanSizes z;
  int seg_pairs;
};

// -> whether there is any (the same for the whole CTA, whose threads all call this, and which may put tiles in the place of `smem` then). kept: shared memory
template <int THREADS>
__device__ __forceinline__ bool sa_share(SaShare* mine, SaShare* kept, const FbSharedStep& st, const SaSpace& w, int R, int nkv, unsigned char* smem,
                                         long long* tmp, SharedBlock* near, int* status) {
  const int tid = threadIdx.x;
  SharedPlan<THREADS> plan{};
  // what the second kernel has to know of a row: written by every CTA that has the block's tiles (the same), or by the first one
  auto note = [&](int b, const SharedBlock& e) {
    const int s = plan.span[b] - st.ngrp, unit = (b - (s >= 0 ? plan.group_blocks : 0)) * nkv;
    for (int r = 0; r < e.nrows; ++r) {
      w.rows[2 * (e.row0 + r) + (s >= 0)] = make_int4(e.place0, e.nt, unit, r);
      if (s >= 0 && plan.group[s] < 0) w.rows[2 * (e.row0 + r)] = make_int4(0, 0, 0, 0);
    }
  };
  // the CTA's part of the plan, by `count` threads of which this is number `me`
  auto take = [&](bool fits, int me, int count) {
    const long long all = fits ? plan.places * nkv : 0, per = max(1ll, (all + gridDim.x - 1) / gridDim.x);
    const long long f0 = min(all, blockIdx.x * per), f1 = min(all, f0 + per);
    if (blockIdx.x == 0 && me == 0) {
      w.head[0] = fits && per < 1ll << 31 ? per : 0;
      w.head[1] = fits ? plan.group_blocks : 0;
    }
    if (fits && blockIdx.x == 0)
      for (int b = me; b < plan.blocks; b += count)                  // blocks that have no keys
        if ((b + 1 < plan.blocks ? (long long)plan.place[b + 1] : plan.places) == plan.place[b]) note(b, plan.block(st, b, R, SA_KT, status));
    if (f0 == f1 || per >= 1ll << 31) {
      if (me == 0 && per >= 1ll << 31) set_status(status, ST_CAPACITY);
      return SaShare{0, 0, 0, 0};
    }
    const int b0 = plan.find(f0, nkv), b1 = plan.find(f1 - 1, nkv);
    for (int b = b0 + me; b <= b1; b += count) {
      SharedBlock e = plan.block(st, b, R, SA_KT, status);
      e.place0 = plan.place[b];
      if (b - b0 < SA_NEAR) near[b - b0] = e;
      else w.table[b] = e;
      if (e.nt) note(b, e);
    }
    return SaShare{b0, plan.group_blocks, (int)(f1 - f0), f0};
  };
  if (w.z.few) {
    plan.load(st, w.z, smem);
    if (tid == 0) *kept = SaShare{0, 0, 0, 0};
    __syncthreads();
    if (tid < SK_FEW) {
      SharedBlock e;
      int count;
      const bool fits = plan.make_by_few(st, R, SA_KT, SA_EXTRA, w.z, tmp, status, &e, &count);
      const long long all = fits ? plan.places * nkv : 0, per = max(1ll, (all + gridDim.x - 1) / gridDim.x);
      const long long f0 = min(all, blockIdx.x * per), f1 = min(all, f0 + per), at = (long long)e.place0 * nkv, end = at + (long long)count * nkv;
      if (blockIdx.x == 0 && tid == 0) {
        w.head[0] = fits && per < 1ll << 31 ? per : 0;
        w.head[1] = fits ? plan.group_blocks : 0;
      }
      if (tid == 0 && per >= 1ll << 31) set_status(status, ST_CAPACITY);
      if (fits && per < 1ll << 31) {                                 // (the same for all of these threads)
        const bool here = f0 < f1 && count > 0 && at < f1 && end > f0;
        if (here && at <= f0) *kept = SaShare{tid, plan.group_blocks, (int)(f1 - f0), f0};
        asm volatile("bar.sync 11, %0;" ::"n"(SK_FEW) : "memory");
        if (here || (blockIdx.x == 0 && tid < plan.blocks && count == 0)) note(tid, e);
        const int b0 = kept->b0;
        if (f0 < f1 && tid >= b0 && tid < plan.blocks && at < f1) {  // (blocks without tiles between others too)
          if (tid - b0 < SA_NEAR) near[tid - b0] = e;
          else w.table[tid] = e;
        }
      }
    }
  } else {
    const SaShare got = take(plan.make(st, R, SA_KT, SA_EXTRA, w.z, smem, tmp, status), tid, THREADS);
    if (tid == 0) *kept = got;
  }
  fence_proxy_async();                                               // tiles take the plan's place
  __syncthreads();
  *mine = *kept;
  return mine->places > 0;
}

// A CTA's way through its share of the list: (block, kv head) after (block, kv head), as far as tiles of theirs lie in it.
struct SaWalk {
  SharedBlock e;
  int b, kvh, t, n;                              // the piece: n tiles from tile t on
  int left;                                      // places behind it
  int b0;
  const SharedBlock *near, *table;
  __device__ __forceinline__ SharedBlock block(int i) const { return i - b0 < SA_NEAR ? near[i - b0] : table[i]; }
  __device__ __forceinline__ void take(int at) {                     // from place `at` of the unit on
    const int m = min(e.nt + SA_EXTRA - at, left);
    t = max(at - SA_EXTRA, 0);
    n = max(at + m - SA_EXTRA, 0) - t;
    left -= m;
  }
  // -> whether there is a piece
  __device__ __forceinline__ bool start(const SharedBlock* close, const SharedBlock* tab, const SaShare& share, int nkv) {
    near = close;
    table = tab;
    b = b0 = share.b0;
    e = block(b);
    const int at = (int)(share.f0 - (long long)e.place0 * nkv);
    kvh = at / (e.nt + SA_EXTRA);
    left = share.places;
    take(at - kvh * (e.nt + SA_EXTRA));
    return n > 0 || next(nkv);
  }
  __device__ __forceinline__ bool next(int nkv) {
    if (left == 0) return false;
    if (++kvh == nkv) {
      kvh = 0;
      do e = block(++b);
      while (e.nt == 0);
    }
    take(0);
    return n > 0;                                // (none: the share ends in what lies ahead of the unit's tiles)
  }
  __device__ __forceinline__ int token(int j) const { return (e.k0 / SA_KT + t + j) * SA_KT; }
};

// Bits lo .. hi - 1 of 32.
__device__ __forceinline__ uint32_t key_bits(int lo, int hi) {
  const uint32_t below = hi <= 0 ? 0u : hi >= 32 ? 0xffffffffu : (1u << hi) - 1, ahead = lo <= 0 ? 0u : lo >= 32 ? 0xffffffffu : (1u << lo) - 1;
  return below & ~ahead;
}
// Two bf16 values with zeros in the place of those that are no finite numbers.
__device__ __forceinline__ uint32_t finite_or_zero(uint32_t u) {
  return ((u & 0x7f80u) == 0x7f80u ? 0u : u & 0xffffu) | ((u & 0x7f800000u) == 0x7f800000u ? 0u : u & 0xffff0000u);
}
// What meets weights of zero in a tile becomes zeros: values of keys that no row sees (outside k0 .. k1), and what is no finite number in those of a key that some row
// does not see (from kmin on). Four of a set's threads have a key. -> which of the warp's eight keys had such numbers: the second kernel looks at them for the
// rows that see them. (Out of line: a few tiles of a unit come by, and what lies between the instructions that every tile runs costs their fetches.)
template <int HD>
__device__ __noinline__ uint32_t sa_clean_values(unsigned char* base, int thread, int t0, int k0, int k1, int kmin) {
  constexpr int CH = SA_KT * 128, PER = HD / 32;                     // bytes of 64 columns; 16-byte pieces of a thread
  const int key = thread >> 2, part = thread & 3, tok = t0 + key;
  auto at = [&](int e) { return reinterpret_cast<uint4*>(base + ((part * PER + e) >> 3) * CH + key * 128 + ((part * PER + e) & 7) * 16); };
  const bool none = tok < k0 || tok >= k1;
  bool bad = false;
  if (none) {
#pragma unroll
    for (int e = 0; e < PER; ++e) *at(e) = make_uint4(0, 0, 0, 0);
  } else if (tok >= kmin) {
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const uint4 u = *at(e), c = make_uint4(finite_or_zero(u.x), finite_or_zero(u.y), finite_or_zero(u.z), finite_or_zero(u.w));
      const bool other = ((u.x ^ c.x) | (u.y ^ c.y) | (u.z ^ c.z) | (u.w ^ c.w)) != 0;
      bad |= other;
      if (other) *at(e) = c;
    }
  }
  const uint32_t bal = __ballot_sync(0xffffffffu, bad);
  uint32_t bits = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) bits |= (bal >> (4 * k) & 15u) ? 1u << k : 0u;
  return bits;
}

template <int HD>
__global__ void __launch_bounds__(SA_THREADS, 1)
shared_attn_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __nv_bfloat16* q, long q_stride, FbSharedStep st,
                   SaSpace w, int nkv, int share, float scale_log2, int* status) {
  using C = SaCfg<HD>;
  constexpr int NCH = C::NCH, KS = C::KS, VS = C::VS;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char *sQ = smem, *sK = smem + C::Q_BYTES, *sV = sK + KS * C::T_BYTES;
  SaMisc<KS + VS>& ms = *reinterpret_cast<SaMisc<KS + VS>*>(smem + C::MISC_AT);
  uint64_t *q_full = ms.bars, *o_empty = q_full + 1, *s_full = q_full + 2, *s_empty = q_full + 4, *p_full = q_full + 6, *p_empty = q_full + 10,
           *turn = q_full + 14, *k_full = q_full + 22, *k_empty = k_full + KS, *v_full = k_empty + KS, *v_empty = v_full + VS;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort_flag = &ms.abort;
  if (smem_u32(smem) & 1023u) {                                      // the swizzled tiles need the 1024-byte base
    if (tid == 0) set_status(status, ST_BOUNDS);
    return;
  }
  if (tid == 0) {
    ms.abort = 0;
    mbar_init(q_full, SA_SET);
    mbar_init(o_empty, 2 * SA_SET);
    for (int i = 0; i < 8; ++i) mbar_init(&turn[i], 2);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1); mbar_init(&s_empty[i], SA_SET);
    }
    for (int i = 0; i < 2; ++i) { mbar_init(&p_full[i], SA_SET); mbar_init(&p_empty[i], 1); }
    for (int i = 0; i < KS; ++i) { mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1); }
    for (int i = 0; i < VS; ++i) { mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 1); }
    fence_mbar_init();
  }
  pdl_wait();
  sk_tmem_alloc(&ms.tmem, C::COLS);

  SaShare mine;
  const bool any = sa_share<SA_THREADS>(&mine, &ms.share, st, w, SA_PAIRS / share, nkv, smem, ms.tmp, ms.blocks, status);
  const uint32_t tmem = sk_tmem_ready(&ms.tmem);
  if (!any) {
    if (warp == SK_ALLOC) tmem_dealloc(tmem, C::COLS);
    return;
  }
  const int group_blocks = mine.group_blocks;
  SaWalk x;
  if (!x.start(ms.blocks, w.table, mine, nkv)) goto done;            // the same for the whole CTA

  if (warp == 0 || warp == 2) {
    // ---- keys (warp 0) and values (warp 2): the lanes look up 32 tiles' pages at a time, one of them copies
    const bool keys = warp == 0;
    const CUtensorMap* tm = keys ? &tmK : &tmV;
    uint64_t *full = keys ? k_full : v_full, *empty = keys ? k_empty : v_empty;
    unsigned char* to = keys ? sK : sV;
    const int S = keys ? KS : VS;
    if (lane == 0) tma_prefetch_desc(tm);
    int i = 0, stage = 0, phase = 0;
    bool ok = true;
    do {
      int rows = 0;
      for (int j = 0; j < x.n; ++j, ++i) {
        if (j % 32 == 0) rows = j + lane < x.n ? tile_row(st, x.e.slot, x.token(j + lane), status) : 0;
        const int row = __shfl_sync(0xffffffffu, rows, j % 32);
        if (i >= S && !__all_sync(0xffffffffu, sk_wait(&empty[stage], phase ^ 1, abort_flag))) {
          ok = false;
          break;
        }
        if (lane == 0) {
          mbar_expect_tx(&full[stage], C::T_BYTES);
#pragma unroll
          for (int c = 0; c < NCH; ++c) tma_load_2d(to + stage * C::T_BYTES + c * C::KV_CH, tm, &full[stage], x.kvh * HD + c * 64, row);
        }
        if (++stage == S) {
          stage = 0;
          phase ^= 1;
        }
      }
    } while (ok && x.next(nkv));
    if (!ok && lane == 0) {
      if (!*abort_flag) set_status(status, ST_MBAR_TIMEOUT);
      *abort_flag = 1;
    }
    if (*abort_flag && lane == 0)                                    // loads may still be landing: a bounded time before the CTA's memory goes away
      for (int j = max(0, i - S); j < i; ++j) mbar_wait(&full[j % S], (j / S) & 1, 1u << 20);
  } else if (warp == 1 || warp == 3) {
    // ---- products, issued from the whole warp by one lane's predicate: S (warp 1), O (warp 3)
    const bool issue = elect_one();
    auto wait = [&](uint64_t* a, uint32_t pa, uint64_t* b, uint32_t pb, bool both) {
      return __all_sync(0xffffffffu, sk_wait2(a, pa, both ? b : a, both ? pb : pa, abort_flag));
    };
    bool ok = true;
    int i = 0, st_i = 0, phase = 0, piece = 0;
    do {
      for (int j = 0; ok && j < x.n; ++j, ++i) {
        const int s = i & 1;
        if (warp == 1) {
          constexpr uint32_t idesc = umma_idesc(1, 1, SA_PAIRS, SA_KT);
          const uint32_t aQ = smem_u32(sQ), aK = smem_u32(sK) + st_i * C::T_BYTES;
          ok = j > 0 || wait(q_full, piece & 1, q_full, 0, false);
          ok = ok && wait(&k_full[st_i], phase, &s_empty[s], ((i >> 1) - 1) & 1, i >= 2);
          if (!ok) break;
          tc_fence_after();
          sk_products<HD / 16>(issue, tmem + C::COL_S + s * SA_KT, umma_desc_k128(aQ), umma_desc_k128(aK), C::Q_CH, C::KV_CH, idesc);
          tc_commit_if(issue, &s_full[s]);
          tc_commit_if(issue, &k_empty[st_i]);
          if (++st_i == KS) {
            st_i = 0;
            phase ^= 1;
          }
        } else {
          constexpr uint32_t idesc = umma_idesc(1, 1, SA_PAIRS, HD) | (1u << 16);      // B read MN-major
          const uint32_t aV = smem_u32(sV) + st_i * C::T_BYTES;
          ok = j > 0 || piece == 0 || wait(o_empty, (piece - 1) & 1, o_empty, 0, false);
          ok = ok && wait(&v_full[st_i], phase, &p_full[s], (i >> 1) & 1, true);
          if (!ok) break;
          tc_fence_after();
          const uint64_t dV = sk_desc_mn128(aV, C::KV_CH, 1024);
#pragma unroll
          for (int kk = 0; kk < SA_KT / 8; ++kk)                      // weights, remainders
            tc_mma_f16_ts_if(issue, tmem, tmem + C::COL_P + s * SA_KT + kk * 8, dV + (uint32_t)((kk & 3) * 16 * 128 >> 4), idesc, (j > 0 || kk > 0) ? 1u : 0u);
          tc_commit_if(issue, &v_empty[st_i]);
          tc_commit_if(issue, &p_empty[s]);
          if (++st_i == VS) {
            st_i = 0;
            phase ^= 1;
          }
        }
      }
      ++piece;
    } while (ok && x.next(nkv));
    if (!ok) {
      if (lane == 0 && !*abort_flag) set_status(status, ST_MBAR_TIMEOUT);
      *abort_flag = 1;
    }
  } else {
    // ---- softmax, queries, pieces. Warps 4..11 are set 0, 12..19 set 1; of a set, four have the first 32 keys of a tile, four the others; a pair's threads
    // sit in the same lane quadrant.
    const int quad = warp & 3, set = (warp - 4) >> 3, sub = ((warp - 4) >> 2) & 1, st_tid = (tid - 128) & 255;
    const int pair = quad * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
    constexpr int HC = SA_KT / 2, OC = HD / 2;
    bool dead = false;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (!dead && !__all_sync(0xffffffffu, sk_wait(bar, parity, abort_flag))) {
        dead = true;
        if (lane == 0 && !*abort_flag) set_status(status, ST_MBAR_TIMEOUT);
        *abort_flag = 1;
      }
    };
    auto wait2 = [&](uint64_t* a, uint32_t pa, uint64_t* b, uint32_t pb) {
      if (!dead && !__all_sync(0xffffffffu, sk_wait2(a, pa, b, pb, abort_flag))) {
        dead = true;
        if (lane == 0 && !*abort_flag) set_status(status, ST_MBAR_TIMEOUT);
        *abort_flag = 1;
      }
    };
    auto copy_q = [&](const SaWalk& y) {                             // 16 bytes at a time, swizzled as the products read them
      const int pieces = y.e.nrows * share * (HD / 8);
      const __nv_bfloat16* src = q + (long)y.e.row0 * q_stride + (long)y.kvh * share * HD;
      for (int c = st_tid; c < pieces; c += SA_SET * 32) {
        const int p = c / (HD / 8), d = c % (HD / 8), r = p / share, g = p - r * share;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                     ::"r"(smem_u32(sQ + (d >> 3) * C::Q_CH + p * 128 + (((d & 7) ^ (p & 7)) << 4))), "l"(src + (long)r * q_stride + g * HD + d * 8)
                     : "memory");
      }
    };
    auto give_q = [&]() {
      asm volatile("cp.async.wait_all;" ::: "memory");
      fence_proxy_async();
      __syncwarp();
      if (lane == 0 && !dead) mbar_arrive(q_full);
    };
    if (set == 0) {
      copy_q(x);
      give_q();
    }
    int first = 0;                                                   // number of the piece's first tile
    bool more = true;
    while (more) {
      const SaWalk y = x;
      more = x.next(nkv);
      const int np = y.e.nrows * share, end = first + y.n;
      const int klen = pair < np ? min(st.kvlen[y.e.row0 + pair / share], y.e.k1) : 0;
      const bool active = quad * 32 < np;                            // (the same for all warps of a quadrant)
      float m_own = -INFINITY, l = 0.f;
      bool hidden = false;                                           // whether such a value of a key that the pair sees was taken out
      for (int i = first + ((first ^ set) & 1); i < end; i += 2) {
        const int j = i - first, t0 = y.token(j);
        const bool need_mask = t0 < y.e.k0 || t0 + SA_KT > y.e.kmin;
        wait(&s_full[set], (i >> 1) & 1);
        if (i + 1 == end && more && !dead) copy_q(x);                // every product that reads the queries is through
        if (__builtin_expect(need_mask, 0)) {
          // Values of keys that some row does not see meet weights of zero, which an infinity or NaN would not leave at that: zeros take their place, and
          // what they mean for the rows that see the key is found behind the join (sa_odd_columns).
          // (a wait tells a phase from the one ahead of it only: the values of tile i - VS have to be through)
          if (i >= 2) wait(&p_empty[set], ((i >> 1) - 1) & 1);
          wait(&v_full[i % VS], (i / VS) & 1);
          if (!dead) {
            const uint32_t bits = sa_clean_values<HD>(sV + (i % VS) * C::T_BYTES, st_tid, t0, y.e.k0, y.e.k1, y.e.kmin);
            if (lane == 0) ms.bad[set][i >> 1 & 1][st_tid >> 5] = (uint8_t)bits;
            fence_proxy_async();
          }
          asm volatile("bar.sync %0, 256;" ::"r"(9 + set) : "memory");
        }
        uint32_t sr[HC];
        float mx = -INFINITY;                                        // of the scores as they are, without the scale
        if (active && !dead) {
          tc_fence_after();
          tmem_ld32(tmem + lane_addr + C::COL_S + set * SA_KT + sub * HC, sr);
          tmem_ld_wait();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0 && !dead) mbar_arrive(&s_empty[set]);
        if (active && !dead) {
          if (__builtin_expect(need_mask, 0)) {
            const int c0 = t0 + sub * HC;
            const uint32_t bad = reinterpret_cast<const uint32_t*>(ms.bad[set][i >> 1 & 1])[sub], sees = key_bits(y.e.k0 - c0, klen - c0);
#pragma unroll
            for (int c = 0; c < HC; ++c) sr[c] = sees >> c & 1u ? sr[c] : 0xff800000u;
            hidden |= (bad & sees) != 0;
          }
#pragma unroll
          for (int c = 0; c < HC; c += 4)
            mx = fmaxf(fmaxf(mx, __uint_as_float(sr[c])), fmaxf(fmaxf(__uint_as_float(sr[c + 1]), __uint_as_float(sr[c + 2])), __uint_as_float(sr[c + 3])));
          // (what lies behind the pairs moves no maximum; of a score of infinity the largest number stands for it, so that the sum becomes infinity, and NaN only
          // where a score is)
          mx = pair < np ? fminf(mx * scale_log2, FLT_MAX) : -INFINITY;
        }
        // ---- the decision, in the order of the tiles
        if (i >= 2) wait2(&turn[2 * quad + set], ((i - 1) >> 1) & 1, &p_empty[set], ((i >> 1) - 1) & 1);      // ... and P(i - 2) has been read
        else if (i > 0) wait(&turn[2 * quad + set], ((i - 1) >> 1) & 1);
        float m_new = j > 0 ? ms.m[pair] : -INFINITY;
        const float m_old = m_new;
        uint32_t moves;
        asm volatile("{\n\t.reg .pred a, b;\n\tsetp.ne.b32 a, %1, 0;\n\tbarrier.cta.red.or.pred b, %2, 64, a;\n\tselp.u32 %0, 1, 0, b;\n\t}"
                     : "=r"(moves) : "r"((uint32_t)(!dead && mx > m_old + 16.f)), "r"(1 + 4 * set + quad) : "memory");
        if (__builtin_expect(moves, 0)) {
          ms.mx[sub][pair] = mx;
          asm volatile("bar.sync %0, 64;" ::"r"(1 + 4 * set + quad) : "memory");
          m_new = fmaxf(m_old, fmaxf(mx, ms.mx[sub ^ 1][pair]));
        }
        if (sub == 0 && (moves || j == 0)) ms.m[pair] = m_new;
        __syncwarp();
        if (lane == 0 && !dead) mbar_arrive(&turn[2 * quad + (set ^ 1)]);
        if (moves && j > 0) wait(&p_empty[set ^ 1], ((i - 1) >> 1) & 1);               // O is rescaled behind PV(i - 1)
        if (dead || !active) {
          __syncwarp();
          if (lane == 0 && !dead) mbar_arrive(&p_full[set]);
          continue;
        }
        tc_fence_after();
        if (m_new != m_own) {
          l = m_own == -INFINITY ? l : l * sk_exp2(m_own - m_new);   // (a sum that is no number stays one)
          m_own = m_new;
        }
        if (__builtin_expect(moves && j > 0, 0)) {
          const float f = m_old == -INFINITY ? 0.f : sk_exp2(m_old - m_new);
#pragma unroll 1
          for (int c0 = 0; c0 < OC; c0 += 16) {
            uint32_t o[16];
            tmem_ld16(tmem + lane_addr + sub * OC + c0, o);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * f);
            sk_tmem_st16(tmem + lane_addr + sub * OC + c0, o);
          }
          tmem_st_wait();
        }
        const float mr = m_new == -INFINITY ? 0.f : -m_new;
        const uint64_t scale2 = f2_pack(scale_log2, scale_log2), mr2 = f2_pack(mr, mr), minus = f2_pack(-1.f, -1.f);
        uint64_t sum = f2_pack(0.f, 0.f);
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          uint32_t pr[HC / 4], px[HC / 4];
#pragma unroll
          for (int c = 0; c < HC / 4; ++c) {
            const int k = part * (HC / 2) + 2 * c;
            const float2 d = f2_unpack(f2_fma(f2_pack(__uint_as_float(sr[k]), __uint_as_float(sr[k + 1])), scale2, mr2));
            const float p0 = sk_exp2(d.x), p1 = sk_exp2(d.y);
            const uint64_t pp = f2_pack(p0, p1);
            sum = f2_add(sum, pp);
            pr[c] = pack_bf2(p0, p1);
            const float2 rest = f2_unpack(f2_fma(f2_pack(__uint_as_float(pr[c] << 16), __uint_as_float(pr[c] & 0xffff0000u)), minus, pp));
            px[c] = pack_bf2(rest.x, rest.y);
          }
          const uint32_t to = tmem + lane_addr + C::COL_P + set * SA_KT + sub * (HC / 2) + part * (HC / 4);
          sk_tmem_st8(to, pr);
          sk_tmem_st8(to + SA_KT / 2, px);
        }
        const float2 both = f2_unpack(sum);
        l += both.x + both.y;
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[set]);
      }
      if (more && ((end - 1) & 1) == set) give_q();
      // ---- the piece: record number = CTA + unit, which no other piece has
      const bool grp = y.b < group_blocks;
      const long rec = (long)blockIdx.x + (long)(y.b - (grp ? 0 : group_blocks)) * nkv + y.kvh;
      const int stride = grp ? SA_PAIRS : w.seg_pairs;
      if (((end - 1) & 1) != set) {                                  // the last decision was the other set's
        wait(&turn[2 * quad + set], ((end - 1) >> 1) & 1);
        const float m = ms.m[pair];
        l = m_own == -INFINITY ? l : l * sk_exp2(m_own - m);
        m_own = m;
      }
      if (active && pair < np && !dead) {
        float* ml = (grp ? w.ml_grp : w.ml_seg) + (rec * stride + pair) * SA_ML;
        ml[2 * set + sub] = l;
        reinterpret_cast<uint8_t*>(ml + 5)[2 * set + sub] = hidden;
        if (set == 0 && sub == 0) ml[4] = m_own;
      }
      if (end >= 2) wait(&p_empty[end & 1], ((end - 2) >> 1) & 1);             // (one phase after the other)
      wait(&p_empty[(end - 1) & 1], ((end - 1) >> 1) & 1);
      if (active && !dead) {
        tc_fence_after();
        constexpr int QC = HD / 4;
        const int col = (2 * set + sub) * QC;
        float* o = (grp ? w.o_grp : w.o_seg) + (rec * stride) * HD + col + 2 * (lane & 3);
#pragma unroll 1
        for (int r0 = quad * 32; r0 < min(np, quad * 32 + 32); r0 += 16) {
          const int ra = r0 + (lane >> 2), rb = ra + 8;
#pragma unroll 1
          for (int c0 = 0; c0 < QC; c0 += 16) {
            uint32_t v[8];
            sk_tmem_ld16x16(tmem + ((uint32_t)r0 << 16) + col + c0, v);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              if (ra < np) *reinterpret_cast<float2*>(o + (long)ra * HD + c0 + 8 * k) = make_float2(__uint_as_float(v[4 * k]), __uint_as_float(v[4 * k + 1]));
              if (rb < np) *reinterpret_cast<float2*>(o + (long)rb * HD + c0 + 8 * k) = make_float2(__uint_as_float(v[4 * k + 2]), __uint_as_float(v[4 * k + 3]));
            }
          }
        }
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0 && !dead) mbar_arrive(o_empty);
      first = end;
    }
  }
done:
  tc_fence_before();
  __syncthreads();
  if (warp == SK_ALLOC) tmem_dealloc(tmem, C::COLS);
}

// ---- logarithms alone ------------------------------------------------------------------------------------------------------------------------
// Where a step's weights are wanted and its attention has been something else (a prompt's): S as above, for 256 pairs at a time, so that a key tile serves two
// products. A set of eight warps has 128 of the pairs; two threads a pair, each with half of every tile's keys and a maximum and sum of its own, which
// meet in the second kernel only: nothing passes between threads. The queries are in tensor memory, so that a product reads the keys alone from shared memory.
// Measured: 2048 rows x 24 heads of 256 over 16000 keys 300 us (340 with the queries in shared memory), tensor pipe 72 % busy under the power cap.
template <int HD>
struct SlCfg {
  static constexpr int NCH = HD / 64, KV_CH = SA_KT * 128, T_BYTES = NCH * KV_CH;
  static constexpr int KS = HD == 256 ? 6 : 8;
  static constexpr int TILES = KS * T_BYTES, MISC_AT = TILES > SK_PLAN_BYTES ? TILES : SK_PLAN_BYTES;
  // TMEM: S [tile of pairs][parity] | queries of both tiles
  static constexpr uint32_t COL_Q = 4 * SA_KT, COLS = 512;
};
template <int HD>
__global__ void __launch_bounds__(SA_THREADS, 1)
shared_lse_kernel(const __grid_constant__ CUtensorMap tmK, const __nv_bfloat16* q, long q_stride, FbSharedStep st, SaSpace w, int nkv, int share,
                  float scale_log2, int* status) {
  using C = SlCfg<HD>;
  constexpr int NCH = C::NCH, KS = C::KS;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* sK = smem;
  SaMisc<KS>& ms = *reinterpret_cast<SaMisc<KS>*>(smem + C::MISC_AT);
  uint64_t *q_full = ms.bars, *q_done = q_full + 1, *s_full = q_full + 2, *s_empty = q_full + 6, *k_full = q_full + 10, *k_empty = k_full + KS;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, Rh = SA_PAIRS / share;
  volatile int* abort_flag = &ms.abort;
  if (smem_u32(smem) & 1023u) {
    if (tid == 0) set_status(status, ST_BOUNDS);
    return;
  }
  if (tid == 0) {
    ms.abort = 0;
    mbar_init(q_full, 2 * SA_SET);
    mbar_init(q_done, 2);
    for (int i = 0; i < 4; ++i) { mbar_init(&s_full[i], 1); mbar_init(&s_empty[i], SA_SET); }        // [tile of pairs][parity]
    for (int i = 0; i < KS; ++i) { mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 2); }
    fence_mbar_init();
  }
  pdl_wait();
  sk_tmem_alloc(&ms.tmem, C::COLS);
  SaShare mine;
  const bool any = sa_share<SA_THREADS>(&mine, &ms.share, st, w, 2 * Rh, nkv, smem, ms.tmp, ms.blocks, status);
  const uint32_t tmem = sk_tmem_ready(&ms.tmem);
  if (!any) {
    if (warp == SK_ALLOC) tmem_dealloc(tmem, C::COLS);
    return;
  }
  SaWalk x;
  if (!x.start(ms.blocks, w.table, mine, nkv)) goto done;
  if (warp == 0) {
    int i = 0, stage = 0, phase = 0;
    bool ok = true;
    do {
      int rows = 0;
      for (int j = 0; j < x.n; ++j, ++i) {
        if (j % 32 == 0) rows = j + lane < x.n ? tile_row(st, x.e.slot, x.token(j + lane), status) : 0;
        const int row = __shfl_sync(0xffffffffu, rows, j % 32);
        if (i >= KS && !__all_sync(0xffffffffu, sk_wait(&k_empty[stage], phase ^ 1, abort_flag))) {
          ok = false;
          break;
        }
        if (lane == 0) {
          mbar_expect_tx(&k_full[stage], C::T_BYTES);
#pragma unroll
          for (int c = 0; c < NCH; ++c) tma_load_2d(sK + stage * C::T_BYTES + c * C::KV_CH, &tmK, &k_full[stage], x.kvh * HD + c * 64, row);
        }
        if (++stage == KS) {
          stage = 0;
          phase ^= 1;
        }
      }
    } while (ok && x.next(nkv));
    if (!ok && lane == 0) {
      if (!*abort_flag) set_status(status, ST_MBAR_TIMEOUT);
      *abort_flag = 1;
    }
    if (*abort_flag && lane == 0)
      for (int j = max(0, i - KS); j < i; ++j) mbar_wait(&k_full[j % KS], (j / KS) & 1, 1u << 20);
  } else if (warp < 3) {
    // ---- products of a tile of keys with the first 128 pairs (warp 1) and the others (warp 2)
    constexpr uint32_t idesc = umma_idesc(1, 1, SA_PAIRS, SA_KT);
    const bool issue = elect_one();
    const int a = warp - 1;
    const uint32_t tQ = tmem + C::COL_Q + a * (HD / 2);
    const uint64_t dK = umma_desc_k128(smem_u32(sK));
    int stage = 0, phase = 0, piece = 0, count = 0;
    bool ok = true;
    do {
      const bool there = a == 0 || x.e.nrows > Rh;
      ok = __all_sync(0xffffffffu, sk_wait(q_full, piece & 1, abort_flag));
      for (int j = 0; ok && j < x.n; ++j) {
        const int b = 2 * a + (count & 1);
        ok = __all_sync(0xffffffffu, sk_wait2(&k_full[stage], phase, there && count >= 2 ? &s_empty[b] : &k_full[stage],
                                              there && count >= 2 ? (count / 2 - 1) & 1 : phase, abort_flag));
        if (!ok) break;
        if (there) {
          tc_fence_after();
          sk_products_ts<HD / 16>(issue, tmem + b * SA_KT, tQ, dK + (uint32_t)(stage * C::T_BYTES >> 4), C::KV_CH, idesc);
          tc_commit_if(issue, &s_full[b]);
          ++count;
        }
        tc_commit_if(issue, &k_empty[stage]);
        if (++stage == KS) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (!ok) break;
      tc_commit_if(issue, q_done);
      ++piece;
    } while (x.next(nkv));
    if (!ok) {
      if (lane == 0 && !*abort_flag) set_status(status, ST_MBAR_TIMEOUT);
      *abort_flag = 1;
    }
  } else if (warp >= 4) {
    const int quad = warp & 3, set = (warp - 4) >> 3, sub = ((warp - 4) >> 2) & 1, pair = quad * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16), taddr = lanes + set * 2 * SA_KT + sub * (SA_KT / 2);
    const uint64_t scale2 = f2_pack(scale_log2, scale_log2);
    bool dead = false;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (!dead && !__all_sync(0xffffffffu, sk_wait(bar, parity, abort_flag))) {
        dead = true;
        if (lane == 0 && !*abort_flag) set_status(status, ST_MBAR_TIMEOUT);
        *abort_flag = 1;
      }
    };
    int piece = 0, count = 0;
    bool more = true;
    while (more) {
      const SaWalk y = x;
      const int np = min(Rh, y.e.nrows - set * Rh) * share, row0 = y.e.row0 + set * Rh;      // pairs of the set's half
      const int klen = pair < np ? min(st.kvlen[row0 + pair / share], y.e.k1) : 0;
      // half of the pair's query into its TMEM lane, 64 columns at a time (fewer registers than all at once)
      constexpr int AT_ONCE = HD == 64 ? 4 : 8;
      const int r = pair < np ? pair / share : 0;
      const uint4* src = reinterpret_cast<const uint4*>(q + (long)(row0 + r) * q_stride + (long)(y.kvh * share + pair - r * share) * HD + sub * (HD / 2));
#pragma unroll
      for (int e0 = 0; e0 < HD / 16; e0 += AT_ONCE) {
        uint4 v[AT_ONCE];
#pragma unroll
        for (int e = 0; e < AT_ONCE; ++e) v[e] = pair < np ? src[e0 + e] : make_uint4(0, 0, 0, 0);
        if (e0 == 0 && piece) wait(q_done, (piece - 1) & 1);         // the products with the queries ahead of these are through
        if (dead) continue;
        tc_fence_after();
#pragma unroll
        for (int e = 0; e < AT_ONCE; e += 4) {
          const uint32_t c[16] = {v[e].x,     v[e].y,     v[e].z,     v[e].w,     v[e + 1].x, v[e + 1].y, v[e + 1].z, v[e + 1].w,
                                  v[e + 2].x, v[e + 2].y, v[e + 2].z, v[e + 2].w, v[e + 3].x, v[e + 3].y, v[e + 3].z, v[e + 3].w};
          sk_tmem_st16(lanes + C::COL_Q + set * (HD / 2) + sub * (HD / 4) + (e0 + e) * 4, c);
        }
      }
      if (!dead) {
        tmem_st_wait();
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0 && !dead) mbar_arrive(q_full);
      more = x.next(nkv);
      float m = -INFINITY, l = 0.f;
      if (np > 0) {
        for (int j = 0; j < y.n; ++j, ++count) {
          const int t0 = y.token(j) + sub * (SA_KT / 2), b = count & 1;
          wait(&s_full[2 * set + b], count / 2 & 1);
          uint32_t sr[32];
          if (!dead) {
            tc_fence_after();
            tmem_ld32(taddr + b * SA_KT, sr);
            tmem_ld_wait();
            tc_fence_before();
          }
          __syncwarp();
          if (lane == 0 && !dead) mbar_arrive(&s_empty[2 * set + b]);
          if (dead || quad * 32 >= np) continue;
          if (__builtin_expect(t0 < y.e.k0 || t0 + SA_KT / 2 > y.e.kmin, 0)) {
            const uint32_t sees = key_bits(y.e.k0 - t0, klen - t0);
#pragma unroll
            for (int c = 0; c < 32; ++c) sr[c] = sees >> c & 1u ? sr[c] : 0xff800000u;
          }
          float mx = -INFINITY;
#pragma unroll
          for (int c = 0; c < 32; c += 4)
            mx = fmaxf(fmaxf(mx, __uint_as_float(sr[c])), fmaxf(fmaxf(__uint_as_float(sr[c + 1]), __uint_as_float(sr[c + 2])), __uint_as_float(sr[c + 3])));
          const float m_new = fmaxf(m, fminf(mx * scale_log2, FLT_MAX)), mr = m_new == -INFINITY ? 0.f : -m_new;
          const uint64_t mr2 = f2_pack(mr, mr);
          uint64_t sum[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const float2 d = f2_unpack(f2_fma(f2_pack(__uint_as_float(sr[2 * c]), __uint_as_float(sr[2 * c + 1])), scale2, mr2));
            sum[c & 1] = f2_add(sum[c & 1], f2_pack(sk_exp2(d.x), sk_exp2(d.y)));
          }
          const float2 both = f2_unpack(f2_add(sum[0], sum[1]));
          l = (m == -INFINITY ? l : l * sk_exp2(m - m_new)) + (both.x + both.y);     // (a sum that is no number stays one)
          m = m_new;
        }
      }
      const long rec = (long)blockIdx.x + (long)y.b * nkv + y.kvh;   // no other piece has this number
      if (pair < np && !dead) w.ml[((rec * 2 + set) * SA_PAIRS + pair) * 2 + sub] = make_float2(m, l);
      ++piece;
    }
  }
done:
  tc_fence_before();
  __syncthreads();
  if (warp == SK_ALLOC) tmem_dealloc(tmem, C::COLS);
}

// A thread a (row, head): its pieces' maxima and sums -> logarithm.
__global__ void __launch_bounds__(256) shared_lse_join_kernel(float* lse, FbSharedStep st, SaSpace w, int nkv, int share, int ctas) {
  pdl_launch_dependents();
  pdl_wait();
  const long id = (long)blockIdx.x * 256 + threadIdx.x, nq = (long)nkv * share;
  if (id >= st.rows * nq) return;
  const int row = (int)(id / nq), h = (int)(id % nq), kvh = h / share, g = h - kvh * share, Rh = SA_PAIRS / share;
  bool mine = false;
  for (int s = 0; s < st.nseg && !mine; ++s) mine = row >= st.seg_row0[s] && row - st.seg_row0[s] < st.seg_nrows[s];
  const long long per = w.head[0];
  if (!mine || per <= 0) return;                                     // a row of no segment; a step that did not fit
  float top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int4 info = w.rows[2 * row + k];
    const long long at = (long long)info.x * nkv + kvh * ((long long)info.y + SA_EXTRA) + SA_EXTRA;
    const long long c0 = at / per, c1 = (at + info.y - 1) / per;
    const int first = k ? (int)w.head[1] : 0, last = k ? w.z.blocks : w.z.group_blocks;
    // checked, since this is not written for rows of a segment that was refused, nor by a launch that gave up
    if (info.y <= 0 || info.x < 0 || c1 >= ctas || info.w < 0 || info.w >= 2 * Rh || info.z < 0 || info.z >= (last - (k ? w.z.group_blocks : 0)) * nkv - kvh) continue;
    const int a = info.w >= Rh, pair = (info.w - a * Rh) * share + g;
    for (long long c = c0; c <= c1; ++c) {
      const long rec = c + (long)first * nkv + info.z + kvh;
      const float4 v = *reinterpret_cast<const float4*>(&w.ml[((rec * 2 + a) * SA_PAIRS + pair) * 2]);
      const float m = fmaxf(top, fmaxf(v.x, v.z));
      auto part = [&](float mm, float l) { return mm == -INFINITY ? (l != l ? l : 0.f) : l * sk_exp2(mm - m); };
      sum = part(top, sum) + part(v.x, v.y) + part(v.z, v.w);
      top = m;
    }
  }
  lse[id] = st.kvlen[row] <= 0 ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
}

struct SaInputs {                                // what the step's kernels read besides its tables
  const __nv_bfloat16 *q, *k, *v, *proj;
  long q_stride, proj_stride;
};
// A thread's columns d .. d + 3 of a head's row in which keys that the row sees have values that are no finite numbers: an infinity, if they are alike, else NaN, into the
// output. (A weight is larger than zero, however small, but that of a score of minus infinity.) A walk over the context, out of line and the
// last thing that a thread does: the rows that come across no such values keep nothing in registers for it.
template <int HD>
__device__ __noinline__ void sa_odd_columns(__nv_bfloat16* out, const FbSharedStep& st, const SaInputs& in, int nkv, int share) {
  const int row = blockIdx.x, h = blockIdx.y, kvh = h / share, d = threadIdx.x % (HD / 4) * 4;
  const __nv_bfloat16 *q = in.q + (long)row * in.q_stride + (long)h * HD, *k = in.k, *v = in.v;
  int s = 0, shared = 0;
  while (s < st.nseg && (row < st.seg_row0[s] || row - st.seg_row0[s] >= st.seg_nrows[s])) ++s;
  if (s == st.nseg) return;
  int first = -1;
  const int slot = st.seg_slot[s];
  for (int g = 0; g < st.ngrp; ++g)
    if (st.grp_seg0[g] >= 0 && s >= st.grp_seg0[g] && s - st.grp_seg0[g] < st.grp_nsegs[g]) {
      first = st.seg_slot[st.grp_seg0[g]];
      shared = max(st.grp_len[g], 0);
    }
  const int n = (int)min((long)st.kvlen[row], table_limit(st));
  uint32_t seen = 0;                                                 // of column c: bit c an infinity above zero, bit 4 + c one below; NaN is both
#pragma unroll 1
  for (int run = 0; run < 2; ++run) {
    const int from = run ? min(shared, n) : 0, to = run ? n : min(shared, n), via = run ? slot : first;
    if (via < 0 || via >= st.slots) continue;
#pragma unroll 1
    for (int j0 = from / 8 * 8; j0 < to; j0 += 8) {                  // (eight tokens of one page)
      const int page = st.table[(size_t)via * st.max_blocks + j0 / st.kv_block];
      if (page < 0 || page >= st.pages) continue;
      const size_t r0 = ((size_t)page * st.kv_block + j0 % st.kv_block) * nkv + kvh;
      uint2 u[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e] = *reinterpret_cast<const uint2*>(v + (r0 + (size_t)e * nkv) * HD + d);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        uint32_t odd = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t x = (c & 2 ? u[e].y : u[e].x) >> (c & 1) * 16 & 0xffffu;
          if ((x & 0x7f80u) == 0x7f80u) odd |= (x & 0x7fu ? 0x11u : x & 0x8000u ? 0x10u : 0x01u) << c;
        }
        if (odd == 0 || j0 + e < from || j0 + e >= to) continue;
        float score = 0.f;
#pragma unroll 1
        for (int i = 0; i < HD; ++i) score = fmaf(bf2f(q[i]), bf2f(k[(r0 + (size_t)e * nkv) * HD + i]), score);
        seen |= score == -INFINITY ? (odd | odd >> 4 | odd << 4) & 0xffu : odd;
      }
    }
  }
  out += ((long)row * nkv * share + h) * HD + d;
  for (int c = 0; c < 4; ++c) {
    const bool above = seen >> c & 1u, below = seen >> (4 + c) & 1u;
    float x = above && below ? NAN : above ? INFINITY : -INFINITY;
    if (in.proj) x *= sigmoidf_(bf2f(in.proj[(long)row * in.proj_stride + (long)h * 2 * HD + HD + d + c]));
    if (above || below) out[c] = __float2bfloat16(x);
  }
}

// Pieces of a head's row -> output and logarithm. grid: rows x query heads; a thread has four columns and every fourth (eighth, 16th) piece. Everything that
// does not depend on the pieces is asked for at once, and the pieces' sums beside their maxima: three trips to memory.
template <int HD, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
shared_join_kernel(__nv_bfloat16* out, float* lse, const __grid_constant__ SaInputs in, const __grid_constant__ FbSharedStep st, SaSpace w, int nkv, int share,
                   int ctas) {
  constexpr int LANES = HD / 4, PARTS = THREADS / LANES;
  __shared__ float top_s[PARTS], sum_s[PARTS];
  __shared__ uint32_t hidden_s[PARTS];
  __shared__ float4 o_s[PARTS][LANES];
  const int row = blockIdx.x, h = blockIdx.y, kvh = h / share, g = h - kvh * share, tid = threadIdx.x, part = tid / LANES, d = tid % LANES * 4;
  pdl_launch_dependents();
  pdl_wait();
  bool mine = false;
  for (int s = tid; s < st.nseg; s += THREADS) mine |= row >= st.seg_row0[s] && row - st.seg_row0[s] < st.seg_nrows[s];
  const long long per = w.head[0];
  const int n = st.kvlen[row];
  const int4 info[2] = {w.rows[2 * row], w.rows[2 * row + 1]};
  float4 gate = make_float4(0.f, 0.f, 0.f, 0.f);
  if (in.proj && part == 0) {
    const __nv_bfloat16* p = in.proj + (long)row * in.proj_stride + (long)h * 2 * HD + HD + d;
    gate = make_float4(bf2f(p[0]), bf2f(p[1]), bf2f(p[2]), bf2f(p[3]));
  }
  if (!__syncthreads_or(mine) || per <= 0) return;                   // a row of no segment; a step that did not fit
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  float top = -INFINITY, sum = 0.f;
  uint32_t hidden = 0;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    // a row's run of records; checked, since this is not written for rows of a segment that was refused, nor by a launch that gave up
    const long long at = (long long)info[k].x * nkv + kvh * ((long long)info[k].y + SA_EXTRA) + SA_EXTRA;
    const long long c0 = at / per, c1 = (at + info[k].y - 1) / per;
    const int r = info[k].w, stride = k == 0 ? SA_PAIRS : w.seg_pairs, units = (k == 0 ? w.z.group_blocks : w.z.blocks - w.z.group_blocks) * nkv;
    if (info[k].y <= 0 || info[k].x < 0 || c1 >= ctas || r < 0 || r >= stride / share || info[k].z < 0 || info[k].z >= units - kvh) continue;
    const int pieces = (int)(c1 - c0) + 1;
    const long rec = (c0 + info[k].z + kvh) * stride + r * share + g;
    const float* ml = (k == 0 ? w.ml_grp : w.ml_seg) + rec * SA_ML;
    const float* o = (k == 0 ? w.o_grp : w.o_seg) + rec * HD + d;
    constexpr int AT_ONCE = 4;
    for (int i0 = part; i0 < pieces; i0 += PARTS * AT_ONCE) {
      float2 v[AT_ONCE];                                             // maximum, sum
      float4 x[AT_ONCE];
#pragma unroll
      for (int e = 0; e < AT_ONCE; ++e) {
        const long i = i0 + e * PARTS;
        v[e] = make_float2(-INFINITY, 0.f);
        if (i < pieces) {
          const float4 l = *reinterpret_cast<const float4*>(ml + i * stride * SA_ML);
          const float2 m = *reinterpret_cast<const float2*>(ml + i * stride * SA_ML + 4);
          v[e] = make_float2(m.x, l.x + l.y + (l.z + l.w));
          hidden |= __float_as_uint(m.y);
        }
        x[e] = i < pieces && out ? *reinterpret_cast<const float4*>(o + i * stride * HD) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float m = top;
#pragma unroll
      for (int e = 0; e < AT_ONCE; ++e) m = fmaxf(m, v[e].x);
      const float f0 = top == -INFINITY ? 0.f : sk_exp2(top - m);
      sum = top == -INFINITY ? sum : sum * f0;                       // (a sum that is no number stays one)
      a.x *= f0; a.y *= f0; a.z *= f0; a.w *= f0;
#pragma unroll
      for (int e = 0; e < AT_ONCE; ++e) {
        const float l = v[e].y, f = v[e].x == -INFINITY ? 0.f : sk_exp2(v[e].x - m);
        sum += v[e].x == -INFINITY ? (l != l ? l : 0.f) : l * f;
        a.x = fmaf(x[e].x, f, a.x); a.y = fmaf(x[e].y, f, a.y); a.z = fmaf(x[e].z, f, a.z); a.w = fmaf(x[e].w, f, a.w);
      }
      top = m;
    }
  }
  if (d == 0) {
    top_s[part] = top;
    sum_s[part] = sum;
    hidden_s[part] = hidden;
  }
  if (part) o_s[part][d / 4] = a;
  __syncthreads();
  if (part) return;
  float all = -INFINITY, total = 0.f;
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    all = fmaxf(all, top_s[p]);
    hidden |= hidden_s[p];
  }
#pragma unroll
  for (int p = 0; p < PARTS; ++p) {
    const float m = top_s[p], f = m == -INFINITY ? 0.f : sk_exp2(m - all), s = sum_s[p];
    const float4 x = p ? o_s[p][d / 4] : a;
    total += m == -INFINITY ? (s != s ? s : 0.f) : s * f;
    if (p == 0) a = make_float4(x.x * f, x.y * f, x.z * f, x.w * f);
    else a = make_float4(fmaf(x.x, f, a.x), fmaf(x.y, f, a.y), fmaf(x.z, f, a.z), fmaf(x.w, f, a.w));
  }
  if (lse && d == 0) lse[(long)row * nkv * share + h] = n <= 0 ? -INFINITY : (all + log2f(total)) * 0.6931471805599453f;
  if (!out) return;
  const float inv = n <= 0 ? 0.f : total == 0.f ? NAN : 1.f / total;  // (scores of minus infinity only: 0 / 0)
  a.x *= inv; a.y *= inv; a.z *= inv; a.w *= inv;
  const bool odd = (hidden || !(fabsf(a.x) + fabsf(a.y) + fabsf(a.z) + fabsf(a.w) < INFINITY)) && total > 0.f && total < INFINITY;
  if (in.proj) {
    a.x *= sigmoidf_(gate.x); a.y *= sigmoidf_(gate.y); a.z *= sigmoidf_(gate.z); a.w *= sigmoidf_(gate.w);
  }
  *reinterpret_cast<uint2*>(out + ((long)row * nkv * share + h) * HD + d) = make_uint2(pack_bf2(a.x, a.y), pack_bf2(a.z, a.w));
  if (__builtin_expect(odd, 0)) sa_odd_columns<HD>(out, st, in, nkv, share);             // weights that are numbers, of values that are none
}

}  // namespace fb

using namespace fb;

// The workspace: header | table | rows | statistics | sums. -> floats in all
static long sa_space(SaSpace* w, float* ws, int rows, int nseg, int max_rows, int ngrp, int nq, int nkv, int hd, int ctas, bool logs_only) {
  const int share = nq / nkv, R = SA_PAIRS / share * (logs_only ? 2 : 1);
  const long gb = shared_group_blocks(rows, ngrp, R), sb = shared_seg_blocks(rows, nseg, max_rows, R), pairs = std::min(R, std::max(max_rows, 1)) * (long)share;
  const long recs[2] = {gb ? (gb * nkv + ctas) * SA_PAIRS : 0, (sb * nkv + ctas) * pairs};
  float* at = ws;
  auto take = [&](long floats) {
    float* p = at;
    at += (floats + 3) / 4 * 4;
    return p;
  };
  SaSpace v{};
  v.head = (long long*)take(4);
  v.table = (SharedBlock*)take((gb + sb) * 8);
  v.rows = (int4*)take(8l * rows);
  if (logs_only) {
    v.ml = (float2*)take(((gb + sb) * nkv + ctas) * 2 * SA_PAIRS * 4);
  } else {
    v.ml_grp = take(recs[0] * SA_ML);
    v.ml_seg = take(recs[1] * SA_ML);
    v.o_grp = take(recs[0] * hd);
    v.o_seg = take(recs[1] * hd);
  }
  v.seg_pairs = (int)pairs;
  if (w) *w = v;
  return at - ws;
}
static bool sa_fits(const FbSharedStep& st, int nq, int nkv, int hd, int ctas) {
  return nkv >= 1 && nq % nkv == 0 && nq / nkv >= 1 && nq / nkv <= SA_PAIRS && st.kv_block % SA_KT == 0 && ctas >= 1 && (hd == 64 || hd == 128 || hd == 256);
}
static bool sa_sizes(const FbSharedStep& st, int R, SharedPlanSizes* z) {
  return shared_plan_sizes(st, shared_group_blocks(st.rows, st.ngrp, R), shared_seg_blocks(st.rows, st.nseg, st.max_rows, R), z);
}

extern "C" long fb_attention_shared_floats(int rows, int nseg, int max_rows, int ngrp, int nq, int nkv, int hd, int ctas, int want_out) {
  if (rows <= 0 || nseg <= 0 || nkv < 1 || nq / nkv < 1 || nq / nkv > SA_PAIRS) return 0;
  return sa_space(nullptr, nullptr, rows, nseg, max_rows, ngrp, nq, nkv, hd, ctas, !want_out);
}

// logarithms alone
static int sa_logarithms(float* lse, float* ws, const void* q, long q_stride, const void* k, FbSharedStep st, int nq, int nkv, int hd, int ctas, int* status,
                         cudaStream_t s) {
  SaSpace w;
  sa_space(&w, ws, st.rows, st.nseg, st.max_rows, st.ngrp, nq, nkv, hd, ctas, true);
  const int share = nq / nkv;
  if (!sa_sizes(st, 2 * (SA_PAIRS / share), &w.z)) return -2;
  const float scale = 1.4426950408889634f / sqrtf((float)hd);
  CUtensorMap tmK;
  const uint64_t width = (uint64_t)nkv * hd;
  if (const int rc = make_tmap_bf16_2d(&tmK, k, (uint64_t)st.pages * st.kv_block, width, width, SA_KT)) return rc;
  cudaError_t e = cudaErrorInvalidValue;
#define FB_SL(H)                                                                                                                                    \
  if (hd == H) {                                                                                                                                    \
    using C = SlCfg<H>;                                                                                                                             \
    const size_t smem = C::MISC_AT + sizeof(SaMisc<C::KS>);                                                                                         \
    static_assert(C::MISC_AT + sizeof(SaMisc<C::KS>) <= 232448, "shared memory of an SM");                                                          \
    FB_CUDA_CHECK(cudaFuncSetAttribute(shared_lse_kernel<H>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));                              \
    e = launch_pdl(shared_lse_kernel<H>, dim3(ctas), dim3(SA_THREADS), smem, s, tmK, (const __nv_bfloat16*)q, q_stride, st, w, nkv, share, scale,   \
                   status);                                                                                                                         \
  }
  FB_SL(64) FB_SL(128) FB_SL(256)
#undef FB_SL
  if (e != cudaSuccess) return (int)e;
  return (int)launch_pdl(shared_lse_join_kernel, dim3((unsigned)(((long)st.rows * nq + 255) / 256)), dim3(256), 0, s, lse, st, w, nkv, share, ctas);
}

extern "C" int fb_attention_shared(void* out, float* lse, float* ws, long ws_floats, const void* q, long q_stride, const void* k, const void* v,
                                   const void* proj, long proj_stride, FbSharedStep st, int nq, int nkv, int hd, int ctas, int* status, cudaStream_t s) {
  if (st.rows <= 0 || st.nseg <= 0 || st.max_rows <= 0) return 0;
  if (!sa_fits(st, nq, nkv, hd, ctas)) return -1;
  if (ws_floats < fb_attention_shared_floats(st.rows, st.nseg, st.max_rows, st.ngrp, nq, nkv, hd, ctas, out != nullptr)) return -3;
  if (!out) return sa_logarithms(lse, ws, q, q_stride, k, st, nq, nkv, hd, ctas, status, s);
  SaSpace w;
  sa_space(&w, ws, st.rows, st.nseg, st.max_rows, st.ngrp, nq, nkv, hd, ctas, false);
  if (!sa_sizes(st, SA_PAIRS / (nq / nkv), &w.z)) return -2;
  const int share = nq / nkv;
  const float scale = 1.4426950408889634f / sqrtf((float)hd);
  CUtensorMap tmK, tmV;
  int rc;
  const uint64_t cache_rows = (uint64_t)st.pages * st.kv_block, width = (uint64_t)nkv * hd;
  if ((rc = make_tmap_bf16_2d(&tmK, k, cache_rows, width, width, SA_KT))) return rc;
  if ((rc = make_tmap_bf16_2d(&tmV, v, cache_rows, width, width, SA_KT))) return rc;
  cudaError_t e = cudaErrorInvalidValue;
#define FB_SA(H)                                                                                                                                    \
  if (hd == H) {                                                                                                                                    \
    using C = SaCfg<H>;                                                                                                                             \
    const size_t smem = C::MISC_AT + sizeof(SaMisc<C::KS + C::VS>);                                                                                 \
    static_assert(C::MISC_AT + sizeof(SaMisc<C::KS + C::VS>) <= 232448, "shared memory of an SM");                                                  \
    FB_CUDA_CHECK(cudaFuncSetAttribute(shared_attn_kernel<H>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));                             \
    e = launch_pdl(shared_attn_kernel<H>, dim3(ctas), dim3(SA_THREADS), smem, s, tmK, tmV, (const __nv_bfloat16*)q, q_stride, st, w, nkv, share,    \
                   scale, status);                                                                                                                  \
  }
  FB_SA(64) FB_SA(128) FB_SA(256)
#undef FB_SA
  if (e != cudaSuccess) return (int)e;
  // 256 threads a head's row where all of them run at once: more pieces under way; more rows run as twice as many CTAs of 128, since each is a chain of trips to
  // memory (us, 256 / 128: 48 heads' rows 5.7 / 6.7, 144 6.8 / 8.0, 816 10.9 / 8.5, 2048 17.5 / 11.0)
  const SaInputs in{(const __nv_bfloat16*)q, (const __nv_bfloat16*)k, (const __nv_bfloat16*)v, (const __nv_bfloat16*)proj, q_stride, proj_stride};
#define FB_SJ(H, N)                                                                                                                                 \
  if (hd == H && (N == 256) == ((long)st.rows * nq <= 4l * ctas))                                                                                   \
    return (int)launch_pdl(shared_join_kernel<H, N>, dim3(st.rows, nq), dim3(N), 0, s, (__nv_bfloat16*)out, lse, in, st, w, nkv, share, ctas);
  FB_SJ(64, 256) FB_SJ(128, 256) FB_SJ(256, 256) FB_SJ(64, 128) FB_SJ(128, 128) FB_SJ(256, 128)
#undef FB_SJ
  return -1;
}

// Weight that a step's queries gave to every cached key, added up beside the cache: out = carry * mass + sum over rows and heads of exp(q k scale - lse).
//
//   S^T = K Q^T      128 keys x up to 64 (row, head) pairs on tcgen05, S^T in TMEM
//   w  += exp2(S^T scale - lse)    a thread a key: its TMEM lane; the sum over the pairs stays in a register, and nothing passes between threads
//
// Few pairs (a decode step): the queries of a group or segment stay in shared memory and its keys stream by; every key tile belongs to one CTA, which writes
// its sums. Many pairs (a prompt): 256 keys stay in tensor memory and the queries stream by; every CTA has the same number of (256 keys, 64 pairs) steps, and a
// last kernel joins the sums of a key's pieces in their order. The exponentials are 512 cycles of an SM for 128 x 64 scores, the products 512 at 256 columns
// (768 with the keys in shared memory: what the operands take from there).
// Measured (B200, us): one row of 24 heads of 256 over 100000 keys 41, 5.1 TB/s; six over 8000 shared and 900 own keys each 13; 2048 rows over 16000 keys 346, tensor
// pipe 67 % busy under the power cap, and 1111 rows of 32 heads of 128 over 5000 keys 69. Clearing the keys' bits is 1 to 2 of the first two.
// A key's sum is written once, so a key is of one span: a bit a key says that one has taken it, and a second one sets the status (idle warps ask, or those that join).
// Every wait is bounded, as in the attention.
#include <algorithm>

#include "gemm_core.cuh"
#include "shared_kv.cuh"

namespace fb {

constexpr int KM_KEYS = 128, KM_PAIRS = 64, KM_SETS = 4, KM_THREADS = (4 + 4 * KM_SETS) * 32, KM_EXTRA = 2;
constexpr int KM_NEAR = KM_PAIRS - 4;             // pairs of a full tile from which on the unmasked form takes it

template <int HD>
struct KmCfg {
  static constexpr int NCH = HD / 64, K_CH = KM_KEYS * 128, Q_CH = KM_PAIRS * 128, K_BYTES = NCH * K_CH, Q_BYTES = NCH * Q_CH;
  static constexpr int KS = HD == 256 ? 2 : HD == 128 ? 4 : 6;                    // key tiles in shared memory
  static constexpr int QS = HD == 256 ? 3 : HD == 128 ? 5 : 8;                    // tiles of queries
  static constexpr int RS = HD == 256 ? 3 : 8, AS = HD == 256 ? 5 : 8;            // ... where they stream; of what their pairs are
  static constexpr int ROWS_AT = 2 * K_BYTES + RS * Q_BYTES;                      // ... what lies behind them then
  static constexpr int TILES = KS * K_BYTES + QS * Q_BYTES, MISC_AT = TILES > SK_PLAN_BYTES ? TILES : SK_PLAN_BYTES;
};
struct KmShare {                                 // a CTA's share: first block, places, the first one
  int b0, places;
  long long f0;
};
template <int QS>
struct KmMisc {
  float nl[QS][KM_PAIRS];                        // minus a pair's logarithm (log2); minus infinity where there is no pair
  int kvl[QS][KM_PAIRS];                         // keys that it sees
  int edge[QS];                                  // keys that every pair of a full tile sees
  uint64_t bars[44];
  KmShare share;
  uint32_t tmem;
  int abort;
};

__device__ __forceinline__ void km_load_q(void* dst, const CUtensorMap* tm, uint64_t* bar, int x, int head, int row) {
  tma_load_3d(dst, tm, bar, x, head, row);
}

// Sum over a tile's pairs of the weights that they give to this thread's key. cols: 32 or 64. Columns from `pairs` on (query heads that do not divide 64) are
// scores of zeros, and NaN where a key has an infinity: they are masked as keys that a pair does not see are, up to four of them by themselves, more (shares of 11,
// 13, 14 and some above 16) with the whole tile.
template <bool MASKED>
__device__ __forceinline__ float km_weights(uint32_t taddr, int cols, int pairs, const float* nl, const int* kvl, int key, uint64_t scale2) {
  uint64_t acc[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
#pragma unroll 1
  for (int c0 = 0; c0 < cols; c0 += 32) {
    uint32_t r[32];
    tmem_ld32(taddr + c0, r);
    tmem_ld_wait();
#pragma unroll
    for (int c = 0; c < 32; c += 4) {
      const float4 n = *reinterpret_cast<const float4*>(nl + c0 + c);
      const float2 a = f2_unpack(f2_fma(f2_pack(__uint_as_float(r[c]), __uint_as_float(r[c + 1])), scale2, f2_pack(n.x, n.y)));
      const float2 b = f2_unpack(f2_fma(f2_pack(__uint_as_float(r[c + 2]), __uint_as_float(r[c + 3])), scale2, f2_pack(n.z, n.w)));
      float p[4] = {sk_exp2(a.x), sk_exp2(a.y), sk_exp2(b.x), sk_exp2(b.y)};
      if (MASKED || (c == 28 && c0 + 32 > pairs)) {
        const int4 k = *reinterpret_cast<const int4*>(kvl + c0 + c);
        if (key >= k.x) p[0] = 0.f;
        if (key >= k.y) p[1] = 0.f;
        if (key >= k.z) p[2] = 0.f;
        if (key >= k.w) p[3] = 0.f;
      }
      acc[0] = f2_add(acc[0], f2_pack(p[0], p[1]));
      acc[1] = f2_add(acc[1], f2_pack(p[2], p[3]));
    }
  }
  const float2 s = f2_unpack(f2_add(acc[0], acc[1]));
  return s.x + s.y;
}

// Words of 32 keys' bits, cleared ahead of the kernel that takes them.
__device__ __forceinline__ void km_clear(uint32_t* taken, long words) {
  for (long i = (long)blockIdx.x * blockDim.x + threadIdx.x; i < words / 4; i += (long)gridDim.x * blockDim.x) reinterpret_cast<uint4*>(taken)[i] = make_uint4(0, 0, 0, 0);
}
__global__ void __launch_bounds__(256) kv_mass_clear_kernel(uint32_t* taken, long words) {
  pdl_launch_dependents();
  pdl_wait();
  km_clear(taken, words);
}
// Takes those of k0 .. k1 of the 32 keys from `key` on (a multiple of 32; what reads the page reports one that is none).
__device__ __forceinline__ void km_take(const FbSharedStep& st, uint32_t* taken, int slot, int key, int k0, int k1, int* status) {
  const int lo = max(k0 - key, 0), hi = min(k1 - key, 32);
  if (lo >= hi) return;
  const int page = st.table[(size_t)slot * st.max_blocks + key / st.kv_block];
  if (page < 0 || page >= st.pages) return;
  const uint32_t bits = (0xffffffffu >> (32 - hi)) & (0xffffffffu << lo);
  if (atomicOr(taken + ((size_t)page * st.kv_block + key % st.kv_block) / 32, bits) & bits) set_status(status, ST_BOUNDS);
}

// What a pair of a tile is: the number that leads from its scores to weights, and the keys that it sees.
__device__ __forceinline__ void km_pair(const FbSharedStep& st, const float* lse, const SharedBlock& e, int row, int g, int head0, int nq, int share, int Rq, int c,
                                        float* nl, int* kvl) {
  const bool there = c < Rq * share && row < e.nrows;
  *nl = there ? -1.4426950408889634f * lse[(long)(e.row0 + row) * nq + head0 + g] : -INFINITY;
  *kvl = there ? st.kvlen[e.row0 + row] : 0;
}

struct KmWalk {
  SharedBlock e;
  int b, kvh, t, n, left;
  const SharedBlock* table;
  __device__ __forceinline__ void take(int at) {
    const int m = min(e.nt + KM_EXTRA - at, left);
    t = max(at - KM_EXTRA, 0);
    n = max(at + m - KM_EXTRA, 0) - t;
    left -= m;
  }
  __device__ __forceinline__ bool start(const SharedBlock* tab, int first, long long f0, int places, int nkv) {
    table = tab;
    b = first;
    e = table[b];
    const int at = (int)(f0 - (long long)e.place0 * nkv);
    kvh = at / (e.nt + KM_EXTRA);
    left = places;
    take(at - kvh * (e.nt + KM_EXTRA));
    return n > 0 || next(nkv);
  }
  __device__ __forceinline__ bool next(int nkv) {
    if (left == 0) return false;
    if (++kvh == nkv) {
      kvh = 0;
      do e = table[++b];
      while (e.nt == 0);
    }
    take(0);
    return n > 0;
  }
};

// ---- few pairs: keys stream by resident queries ---------------------------------------------------------------------------------------------
template <int HD>
__global__ void __launch_bounds__(KM_THREADS, 1)
kv_mass_keys_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmQ, float* out, const float* mass, float carry,
                    const float* lse, FbSharedStep st, SharedPlanSizes z, SharedBlock* table, uint32_t* taken, int R, int nq, int nkv, float scale_log2,
                    int* status) {
  using C = KmCfg<HD>;
  constexpr int NCH = C::NCH, KS = C::KS;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char *sK = smem, *sQ = smem + KS * C::K_BYTES;
  KmMisc<C::QS>& ms = *reinterpret_cast<KmMisc<C::QS>*>(smem + C::MISC_AT);
  uint64_t *q_full = ms.bars, *q_done = q_full + 1, *s_full = q_full + 2, *s_empty = s_full + KM_SETS, *k_full = s_empty + KM_SETS, *k_empty = k_full + KS;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, share = nq / nkv, Rq = KM_PAIRS / share;
  volatile int* abort_flag = &ms.abort;
  if (smem_u32(smem) & 1023u) {
    if (tid == 0) set_status(status, ST_BOUNDS);
    return;
  }
  if (tid == 0) {
    ms.abort = 0;
    mbar_init(q_full, 1);
    mbar_init(q_done, 1);
    for (int i = 0; i < KM_SETS; ++i) { mbar_init(&s_full[i], 1); mbar_init(&s_empty[i], 4); }
    for (int i = 0; i < KS; ++i) { mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1); }
    fence_mbar_init();
  }
  pdl_wait();
  sk_tmem_alloc(&ms.tmem, KM_SETS * KM_PAIRS);
  SharedPlan<KM_THREADS> plan{};
  // the CTA's part of the plan, by `count` threads of which this is number `me`: first block, first place, places
  auto take = [&](bool fits, int me, int count) {
    const long long all = fits ? plan.places * nkv : 0, per = max(1ll, (all + gridDim.x - 1) / gridDim.x);
    const long long f0 = min(all, blockIdx.x * per), f1 = min(all, f0 + per);
    if (f0 == f1 || per >= 1ll << 31) {
      if (me == 0 && per >= 1ll << 31) set_status(status, ST_CAPACITY);
      return KmShare{0, 0, 0};
    }
    const int b0 = plan.find(f0, nkv), b1 = plan.find(f1 - 1, nkv);
    for (int b = b0 + me; b <= b1; b += count) {                     // (other CTAs of a block write the same)
      SharedBlock e = plan.block(st, b, R, KM_KEYS, status);
      e.place0 = plan.place[b];
      table[b] = e;
    }
    return KmShare{b0, (int)(f1 - f0), f0};
  };
  if (z.few) {
    plan.load(st, z, smem);
    if (tid == 0) ms.share = KmShare{0, 0, 0};
    __syncthreads();
    if (tid < SK_FEW) {
      SharedBlock e;
      int count;
      const bool fits = plan.make_by_few(st, R, KM_KEYS, KM_EXTRA, z, reinterpret_cast<long long*>(ms.nl), status, &e, &count);
      const long long all = fits ? plan.places * nkv : 0, per = max(1ll, (all + gridDim.x - 1) / gridDim.x);
      const long long f0 = min(all, blockIdx.x * per), f1 = min(all, f0 + per), at = (long long)e.place0 * nkv, end = at + (long long)count * nkv;
      if (tid == 0 && per >= 1ll << 31) set_status(status, ST_CAPACITY);
      if (fits && per < 1ll << 31 && f0 < f1) {
        if (count > 0 && at <= f0 && end > f0) ms.share = KmShare{tid, (int)(f1 - f0), f0};
        if (tid < plan.blocks && at < f1 && end >= f0) table[tid] = e;           // (blocks without tiles between others too)
      }
    }
  } else {
    const KmShare got = take(plan.make(st, R, KM_KEYS, KM_EXTRA, z, smem, reinterpret_cast<long long*>(ms.nl), status), tid, KM_THREADS);
    if (tid == 0) ms.share = got;
  }
  __syncthreads();
  const uint32_t tmem = sk_tmem_ready(&ms.tmem);
  const KmShare share_of = ms.share;
  if (share_of.places == 0) {                                        // the same for the whole CTA
    if (warp == SK_ALLOC) tmem_dealloc(tmem, KM_SETS * KM_PAIRS);
    return;
  }
  // rows of a tile of queries that no copy writes are zeros
  for (int i = tid; i < C::QS * C::Q_BYTES / 16; i += KM_THREADS) reinterpret_cast<uint4*>(sQ)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async();
  __syncthreads();
  KmWalk x;
  if (!x.start(table, share_of.b0, share_of.f0, share_of.places, nkv)) goto done;        // the same for the whole CTA
  if (warp == 0) {
    // ---- keys
    int i = 0, stage = 0, phase = 0;
    bool ok = true;
    do {
      int rows = 0;
      for (int j = 0; j < x.n; ++j, ++i) {
        if (j % 16 == 0) {                                           // 16 tiles' pages (two halves of 64 keys each) at a time
          // (the table of a group's stream need not have what lies whole in the shared tokens)
          const int token = (x.e.k0 / KM_KEYS + x.t + j) * KM_KEYS + lane * 64;
          rows = j + lane / 2 < x.n && token + 64 > x.e.k0 && token < x.e.k1 ? tile_row(st, x.e.slot, token, status) : -1024;
        }
        const int r0 = __shfl_sync(0xffffffffu, rows, (j % 16) * 2), r1 = __shfl_sync(0xffffffffu, rows, (j % 16) * 2 + 1);
        if (i >= KS && !__all_sync(0xffffffffu, sk_wait(&k_empty[stage], phase ^ 1, abort_flag))) {
          ok = false;
          break;
        }
        if (lane == 0) {
          mbar_expect_tx(&k_full[stage], C::K_BYTES);
#pragma unroll
          for (int c = 0; c < NCH; ++c) {
            tma_load_2d(sK + stage * C::K_BYTES + c * C::K_CH, &tmK, &k_full[stage], x.kvh * HD + c * 64, r0);
            tma_load_2d(sK + stage * C::K_BYTES + c * C::K_CH + C::K_CH / 2, &tmK, &k_full[stage], x.kvh * HD + c * 64, r1);
          }
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
  } else if (warp == 2) {
    // ---- queries of a unit, where the products of the one before it are through
    int unit = 0;
    bool ok = true;
    do {
      ok = unit == 0 || __all_sync(0xffffffffu, sk_wait(q_done, (unit - 1) & 1, abort_flag));
      if (!ok) break;
      const int tiles = (x.e.nrows + Rq - 1) / Rq;
      if (lane == 0) {
        mbar_expect_tx(q_full, tiles * NCH * Rq * share * 128);
        for (int i = 0; i < tiles; ++i)
#pragma unroll
          for (int c = 0; c < NCH; ++c) km_load_q(sQ + i * C::Q_BYTES + c * C::Q_CH, &tmQ, q_full, c * 64, x.kvh * share, x.e.row0 + i * Rq);
      }
      ++unit;
    } while (x.next(nkv));
    if (!ok && lane == 0) {
      if (!*abort_flag) set_status(status, ST_MBAR_TIMEOUT);
      *abort_flag = 1;
    }
    if (*abort_flag && lane == 0 && unit) mbar_wait(q_full, (unit - 1) & 1, 1u << 20);
  } else if (warp == 1) {
    // ---- products
    const bool issue = elect_one();
    const uint64_t dK = umma_desc_k128(smem_u32(sK)), dQ = umma_desc_k128(smem_u32(sQ));
    int i = 0, stage = 0, phase = 0, unit = 0, turns[KM_SETS] = {0, 0, 0, 0};
    bool ok = true;
    do {
      const int tiles = (x.e.nrows + Rq - 1) / Rq, pairs = x.e.nrows * share;
      ok = __all_sync(0xffffffffu, sk_wait(q_full, unit & 1, abort_flag));
      for (int j = 0; ok && j < x.n; ++j, ++i) {
        const int set = i % KM_SETS;
        ok = __all_sync(0xffffffffu, sk_wait(&k_full[stage], phase, abort_flag));
        for (int t = 0; ok && t < tiles; ++t) {
          const int turn = set == 0 ? turns[0]++ : set == 1 ? turns[1]++ : set == 2 ? turns[2]++ : turns[3]++;
          ok = turn == 0 || __all_sync(0xffffffffu, sk_wait(&s_empty[set], (turn - 1) & 1, abort_flag));
          if (!ok) break;
          tc_fence_after();
          const uint32_t idesc = umma_idesc(1, 1, KM_KEYS, pairs - t * Rq * share > 32 ? 64 : 32);
          sk_products<HD / 16>(issue, tmem + set * KM_PAIRS, dK + (uint32_t)(stage * C::K_BYTES >> 4), dQ + (uint32_t)(t * C::Q_BYTES >> 4), C::K_CH, C::Q_CH, idesc);
          tc_commit_if(issue, &s_full[set]);
        }
        if (!ok) break;
        tc_commit_if(issue, &k_empty[stage]);
        if (++stage == KS) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (!ok) break;
      tc_commit_if(issue, q_done);
      ++unit;
    } while (x.next(nkv));
    if (!ok) {
      if (lane == 0 && !*abort_flag) set_status(status, ST_MBAR_TIMEOUT);
      *abort_flag = 1;
    }
  } else if (warp == 3) {
    // ---- keys of the CTA's tiles are taken
    do
      for (int w = lane; x.kvh == 0 && w < x.n * (KM_KEYS / 32); w += 32)
        km_take(st, taken, x.e.slot, (x.e.k0 / KM_KEYS + x.t) * KM_KEYS + 32 * w, x.e.k0, x.e.k1, status);
    while (x.next(nkv));
  } else if (warp >= 4) {
    // ---- weights: set i % 4 of four warps has key tile i with all of its pairs
    const int quad = warp & 3, set = (warp - 4) >> 2, st_tid = tid - 128, place = quad * 32 + lane;
    const uint32_t taddr = tmem + ((uint32_t)(quad * 32) << 16) + set * KM_PAIRS;
    const uint64_t scale2 = f2_pack(scale_log2, scale_log2);
    bool dead = false;
    int first = 0, turn = 0;
    do {
      const int tiles = (x.e.nrows + Rq - 1) / Rq, pairs = x.e.nrows * share;
      asm volatile("bar.sync 1, 512;" ::: "memory");                 // everyone is through with the pairs before these
      for (int c = st_tid; c < tiles * KM_PAIRS; c += 512) {
        const int t = c / KM_PAIRS, p = c % KM_PAIRS, r = p / share;
        km_pair(st, lse, x.e, t * Rq + r, p - r * share, x.kvh * share, nq, share, Rq, p, &ms.nl[t][p], &ms.kvl[t][p]);
      }
      asm volatile("bar.sync 1, 512;" ::: "memory");
      for (int j = (set - first) & (KM_SETS - 1); j < x.n; j += KM_SETS) {
        const int key0 = (x.e.k0 / KM_KEYS + x.t + j) * KM_KEYS, key = key0 + place;
        const bool mine = key >= x.e.k0 && key < x.e.k1, masked = key0 + KM_KEYS > x.e.kmin;
        size_t at = 0;
        float was = 0.f;
        bool write = mine;
        if (mine) {
          const int page = st.table[(size_t)x.e.slot * st.max_blocks + key / st.kv_block];
          write = page >= 0 && page < st.pages;                      // (else the loader has set the status)
          at = ((size_t)(write ? page : 0) * nkv + x.kvh) * st.kv_block + key % st.kv_block;
          if (carry != 0.f && write) was = carry * mass[at];
        }
        float sum = 0.f;
        for (int t = 0; t < tiles; ++t, ++turn) {
          if (!dead && !__all_sync(0xffffffffu, sk_wait(&s_full[set], turn & 1, abort_flag))) {
            dead = true;
            if (lane == 0 && !*abort_flag) set_status(status, ST_MBAR_TIMEOUT);
            *abort_flag = 1;
          }
          if (dead) continue;
          tc_fence_after();
          const int left = pairs - t * Rq * share, cols = left > 32 ? 64 : 32;
          sum += masked || left < Rq * share || Rq * share < KM_NEAR ? km_weights<true>(taddr, cols, Rq * share, ms.nl[t], ms.kvl[t], key, scale2)
                                                                     : km_weights<false>(taddr, cols, Rq * share, ms.nl[t], ms.kvl[t], key, scale2);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_empty[set]);
        }
        if (write && !dead) out[at] = was + sum;
      }
      first += x.n;
    } while (x.next(nkv));
  }
done:
  tc_fence_before();
  __syncthreads();
  if (warp == SK_ALLOC) tmem_dealloc(tmem, KM_SETS * KM_PAIRS);
}

// ---- many pairs: queries stream by 256 resident keys -----------------------------------------------------------------------------------------
constexpr uint32_t KP_COL_K = KM_SETS * KM_PAIRS, KP_COLS = 512;          // TMEM: S of the sets | keys of both tiles
constexpr int KP_KEYS = 2 * KM_KEYS, KP_PLAN = 1024;                      // keys of an item; threads of the plan

// The list of all steps: item after item, kv head after kv head, the blocks of queries that see it. Each CTA has the same number of consecutive steps; what it has of
// an (item, kv head) is a piece.
struct KpItem {                                  // 256 keys of a span
  int slot, key0, k0, k1;                        // its keys: key0 .. key0 + 255, those of k0 .. k1 count
  int place0, seen, first, pad;                  // steps ahead of it (of one kv head), blocks that see it, the span's first block
};
struct KpStart {                                 // of a CTA: the block and step where it starts, steps in all
  int item, kvh, block, step;
  int left, pad[3];
};
struct KpSpace {
  int* head;                                     // items, steps of a CTA
  SharedBlock* blocks;
  KpItem* items;
  KpStart* starts;
  float* sums;                                   // [pieces][sets][keys of a tile]; piece: CTA + item * kv heads + kv head
  uint32_t* taken;
  long words;
  int max_items;
  SharedPlanSizes z;
};
struct KpWalk {
  KpItem it;
  int item, kvh, block, n, left;                 // n steps from `block` on, places behind them
  __device__ __forceinline__ bool start(const KpSpace& w) {
    const KpStart s = w.starts[blockIdx.x];
    if (s.left == 0) return false;
    item = s.item;
    kvh = s.kvh;
    block = s.block;
    it = w.items[item];
    n = min(it.seen - s.step, s.left);
    left = s.left - n;
    return true;
  }
  __device__ __forceinline__ bool next(const KpSpace& w, int nkv) {
    if (left == 0) return false;
    if (++kvh == nkv) {
      kvh = 0;
      it = w.items[++item];
    }
    block = it.first;
    n = min(it.seen, left);
    left -= n;
    return true;
  }
};

// One CTA: blocks of 64 pairs, items, where the CTAs start.
__global__ void __launch_bounds__(KP_PLAN) kv_mass_plan_kernel(FbSharedStep st, KpSpace w, int Rq, int nkv, int ctas, int* status) {
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ long long tmp[32];
  const int tid = threadIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  __shared__ SharedPlan<KP_PLAN> made;
  SharedPlan<KP_PLAN> plan{};
  bool fits;
  if (w.z.few) {
    plan.load(st, w.z, smem);
    __syncthreads();
    fits = false;
    if (tid < SK_FEW) {
      SharedBlock e;
      int count;
      fits = plan.make_by_few(st, Rq, KP_KEYS, 0, w.z, tmp, status, &e, &count);
      if (fits && tid < plan.blocks) w.blocks[tid] = e;
      if (tid == 0) made = plan;
    }
    fits = __syncthreads_or(fits);
    plan = made;
  } else {
    fits = plan.make(st, Rq, KP_KEYS, 0, w.z, smem, tmp, status);
    if (fits)
      for (int b = tid; b < plan.blocks; b += KP_PLAN) w.blocks[b] = plan.block(st, b, Rq, KP_KEYS, status);
  }
  if (!fits) {
    if (tid == 0) w.head[0] = w.head[1] = 0;
    return;
  }
  __syncthreads();
  const int spans = st.ngrp + st.nseg;
  auto first = [&](int i) { return plan.start[i]; };
  auto behind = [&](int i) { return i + 1 < spans ? plan.start[i + 1] : plan.blocks; };
  // From here on: end of a span's keys in the place of its length or rows, its items (as many as its longest block has) in that of the blocks' places, the
  // blocks' tiles in that of their spans.
  auto end = [&](int i) -> int& { return i < st.ngrp ? plan.len[i] : plan.rows[i - st.ngrp]; };
  int* nts = plan.span;
  for (int i = tid; i < spans; i += KP_PLAN) {
    end(i) = 0;
    plan.place[i] = 0;
  }
  __syncthreads();
  for (int b = tid; b < plan.blocks; b += KP_PLAN) {
    const int i = plan.span[b], k1 = w.blocks[b].k1, nt = w.blocks[b].nt;
    atomicMax(&end(i), k1);
    atomicMax(&plan.place[i], nt);
    nts[b] = nt;
  }
  __syncthreads();
  const long long all = scan_ahead<KP_PLAN>(plan.place, spans, tmp);
  const int total = (int)min(all, (long long)w.max_items + 1);
  if (total > w.max_items) {
    if (tid == 0) {
      set_status(status, ST_CAPACITY);
      w.head[0] = w.head[1] = 0;
    }
    return;
  }
  const int lane = tid & 31, warp = tid >> 5;
  auto span_of = [&](int it) {                                       // the last span that starts at or ahead of the item
    int lo = 0, hi = spans - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (plan.place[mid] <= it) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  };
  // a warp an item: how many blocks see it
  for (int it = warp; it < total; it += KP_PLAN / 32) {
    const int i = span_of(it), j = it - plan.place[i];
    int n = 0;
    for (int b = first(i); b < behind(i); b += 32) n += __popc(__ballot_sync(0xffffffffu, b + lane < behind(i) && nts[min(b + lane, plan.blocks - 1)] > j));
    if (lane == 0) {
      const SharedBlock blk = w.blocks[first(i)];
      w.items[it] = KpItem{blk.slot, (blk.k0 / KP_KEYS + j) * KP_KEYS, blk.k0, end(i), 0, n, first(i), 0};
    }
  }
  __syncthreads();
  // steps ahead of the items
  int base = 0;
  for (int i0 = 0; i0 < total; i0 += KP_PLAN) {
    const int it = i0 + tid, mine = it < total ? w.items[it].seen : 0;
    int xs = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, xs, o);
      if (lane >= o) xs += y;
    }
    if (lane == 31) tmp[warp] = xs;
    __syncthreads();
    const int sum = (int)tmp[lane];
    int ahead = lane < warp ? sum : 0, all_here = sum;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
      all_here += __shfl_xor_sync(0xffffffffu, all_here, o);
    }
    if (it < total) w.items[it].place0 = base + ahead + xs - mine;
    base += all_here;
    __syncthreads();
  }
  const long long steps = (long long)base * nkv, per = max(1ll, (steps + ctas - 1) / ctas);
  if (per >= 1ll << 31) {                                            // (the same for all)
    if (tid == 0) {
      set_status(status, ST_CAPACITY);
      w.head[0] = w.head[1] = 0;
    }
    return;
  }
  for (int c = tid; c < ctas; c += KP_PLAN)
    if (c * per >= steps) w.starts[c].left = 0;
  // a warp an item: the CTAs that start in it
  for (int it = warp; it < total; it += KP_PLAN / 32) {
    const int i = span_of(it), j = it - plan.place[i], n = w.items[it].seen;
    const long long at = (long long)w.items[it].place0 * nkv, last = at + (long long)n * nkv - 1;
    for (long long c = (at + per - 1) / per; c <= last / per; ++c) {
      const long long ahead = c * per - at;
      const int kvh = (int)(ahead / n), step = (int)(ahead - (long long)kvh * n);
      int b = first(i), before = 0;                                  // the block that is number `step` of those that see the item
      for (;; b += 32) {
        const uint32_t bal = __ballot_sync(0xffffffffu, b + lane < behind(i) && nts[min(b + lane, plan.blocks - 1)] > j);
        if (before + __popc(bal) > step || b + 32 >= behind(i)) {
          b += (int)__fns(bal, 0, step - before + 1);
          break;
        }
        before += __popc(bal);
      }
      if (lane == 0) w.starts[c] = KpStart{it, kvh, b, step, (int)min(per, steps - c * per), {0, 0, 0}};
    }
  }
  if (tid == 0) {
    w.head[0] = total;
    w.head[1] = (int)per;
  }
}

template <int HD>
__global__ void __launch_bounds__(KM_THREADS, 1)
kv_mass_rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmQ, const float* lse, FbSharedStep st, KpSpace w, int nq,
                    int nkv, float scale_log2, int* status) {
  using C = KmCfg<HD>;
  constexpr int NCH = C::NCH, QS = C::RS, AS = C::AS;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char *sK = smem, *sQ = smem + 2 * C::K_BYTES;
  KmMisc<AS>& ms = *reinterpret_cast<KmMisc<AS>*>(smem + C::ROWS_AT);
  uint64_t *k_full = ms.bars, *k_empty = k_full + 1, *s_full = k_full + 2, *s_empty = s_full + KM_SETS, *q_full = s_empty + KM_SETS, *q_empty = q_full + QS,
           *a_full = q_empty + QS, *a_empty = a_full + AS, *t_full = a_empty + AS;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, share = nq / nkv, Rq = KM_PAIRS / share;
  volatile int* abort_flag = &ms.abort;
  if (smem_u32(smem) & 1023u) {
    if (tid == 0) set_status(status, ST_BOUNDS);
    return;
  }
  if (tid == 0) {
    ms.abort = 0;
    mbar_init(k_full, 1);
    mbar_init(k_empty, 4 * KM_SETS);
    mbar_init(t_full, 4 * KM_SETS);
    for (int i = 0; i < KM_SETS; ++i) { mbar_init(&s_full[i], 1); mbar_init(&s_empty[i], 4); }
    for (int i = 0; i < QS; ++i) { mbar_init(&q_full[i], 1); mbar_init(&q_empty[i], 1); }
    for (int i = 0; i < AS; ++i) { mbar_init(&a_full[i], 1); mbar_init(&a_empty[i], 8); }
    fence_mbar_init();
  }
  for (int i = tid; i < QS * C::Q_BYTES / 16; i += KM_THREADS) reinterpret_cast<uint4*>(sQ)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async();
  pdl_wait();
  sk_tmem_alloc(&ms.tmem, KP_COLS);
  __syncthreads();
  const uint32_t tmem = sk_tmem_ready(&ms.tmem);
  km_clear(w.taken, w.words);                                        // (for the kernel that joins the sums)
  const bool any = w.head[0] > 0;
  KpWalk x;
  auto sees = [&](const SharedBlock& e, const KpItem& it) { return e.nt > it.key0 / KP_KEYS - it.k0 / KP_KEYS; };
  if (warp == 0) {
    // ---- keys
    int n = 0;
    bool ok = true;
    for (bool more = any && x.start(w); ok && more; more = x.next(w, nkv), ++n) {
      const int token = x.it.key0 + lane * 64, rows = lane < 4 && token + 64 > x.it.k0 && token < x.it.k1 ? tile_row(st, x.it.slot, token, status) : -1024;
      ok = n == 0 || __all_sync(0xffffffffu, sk_wait(k_empty, (n - 1) & 1, abort_flag));
      if (!ok) break;
      if (lane == 0) mbar_expect_tx(k_full, 2 * C::K_BYTES);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int row = __shfl_sync(0xffffffffu, rows, k);
        if (lane == 0)
#pragma unroll
          for (int c = 0; c < NCH; ++c)
            tma_load_2d(sK + (k / 2) * C::K_BYTES + c * C::K_CH + (k % 2) * (C::K_CH / 2), &tmK, k_full, x.kvh * HD + c * 64, row);
      }
    }
    if (!ok && lane == 0) {
      if (!*abort_flag) set_status(status, ST_MBAR_TIMEOUT);
      *abort_flag = 1;
    }
    if (*abort_flag && lane == 0 && n) mbar_wait(k_full, (n - 1) & 1, 1u << 20);
  } else if (warp == 2 || warp == 3) {
    // ---- tiles of queries (warp 2), what their pairs are (warp 3). The lanes look at 32 blocks at a time.
    const int S = warp == 2 ? QS : AS;
    uint64_t* empty = warp == 2 ? q_empty : a_empty;
    int i = 0, stage = 0, phase = 0;
    bool ok = true;
    auto room = [&] { return ok = i < S || __all_sync(0xffffffffu, sk_wait(&empty[stage], phase ^ 1, abort_flag)); };
    auto step = [&] {
      ++i;
      if (++stage == S) {
        stage = 0;
        phase ^= 1;
      }
    };
    // warp 3: its lanes' two pairs of a tile; a tile's numbers are asked for ahead of the one before it being handed on
    const int r2[2] = {lane / share, (lane + 32) / share}, g2[2] = {lane - r2[0] * share, lane + 32 - r2[1] * share};
    float nl[2] = {0.f, 0.f};
    int kvl[2] = {0, 0}, edge = -1;
    auto give = [&] {
      if (!room()) return;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ms.nl[stage][lane + 32 * h] = nl[h] * -1.4426950408889634f;
        ms.kvl[stage][lane + 32 * h] = kvl[h];
      }
      if (lane == 0) ms.edge[stage] = edge;
      __syncwarp();
      if (lane == 0) mbar_arrive(&a_full[stage]);
      step();
    };
    for (bool more = any && x.start(w); ok && more; more = x.next(w, nkv)) {
      int b = x.block;
      SharedBlock e{};
      uint32_t bits = 0;
      for (int left = x.n; ok && left > 0;) {
        if (bits == 0) {                                             // (of the span's last blocks on, `left` says where it ends)
          e = w.blocks[min(b + lane, w.z.blocks - 1)];
          bits = __ballot_sync(0xffffffffu, b + lane < w.z.blocks && sees(e, x.it));
          b += 32;
          if (bits == 0) {
            if (b >= w.z.blocks) ok = false;
            continue;
          }
        }
        const int from = __ffs(bits) - 1, row0 = __shfl_sync(0xffffffffu, e.row0, from), nrows = __shfl_sync(0xffffffffu, e.nrows, from),
                  kmin = __shfl_sync(0xffffffffu, e.kmin, from);
        bits &= bits - 1;
        --left;
        if (warp == 2) {
          if (!room()) break;
          if (lane == 0) {
            mbar_expect_tx(&q_full[stage], NCH * Rq * share * 128);
#pragma unroll
            for (int c = 0; c < NCH; ++c) km_load_q(sQ + stage * C::Q_BYTES + c * C::Q_CH, &tmQ, &q_full[stage], c * 64, x.kvh * share, row0);
          }
          step();
        } else {
          float l[2];
          int k[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const bool there = lane + 32 * h < Rq * share && r2[h] < nrows;
            l[h] = there ? lse[(long)(row0 + r2[h]) * nq + x.kvh * share + g2[h]] : INFINITY;
            k[h] = there ? st.kvlen[row0 + r2[h]] : 0;
          }
          if (edge >= 0) give();
          nl[0] = l[0]; nl[1] = l[1];
          kvl[0] = k[0]; kvl[1] = k[1];
          edge = nrows < Rq ? 0 : kmin;
        }
      }
    }
    if (ok && warp == 3 && edge >= 0) give();
    if (!ok && lane == 0) {
      if (!*abort_flag) set_status(status, ST_MBAR_TIMEOUT);
      *abort_flag = 1;
    }
    if (warp == 2 && *abort_flag && lane == 0)
      for (int j = max(0, i - QS); j < i; ++j) mbar_wait(&q_full[j % QS], (j / QS) & 1, 1u << 20);
  } else if (warp == 1) {
    // ---- products: a tile of queries with both tiles of keys, behind one look at everything that they wait for
    const bool issue = elect_one();
    constexpr uint32_t idesc = umma_idesc(1, 1, KM_KEYS, KM_PAIRS);
    const uint64_t dQ = umma_desc_k128(smem_u32(sQ));
    int i = 0, n = 0, stage = 0, phase = 0;
    bool ok = true;
    for (bool more = any && x.start(w); ok && more; more = x.next(w, nkv), ++n) {
      ok = __all_sync(0xffffffffu, sk_wait(t_full, n & 1, abort_flag));
      for (int j = 0; ok && j < x.n; ++j, ++i) {
        const int set = 2 * (i & 1);
        bool now = mbar_try_wait(&q_full[stage], phase) & mbar_try_wait(&a_full[i % AS], i / AS & 1);
        if (i >= 2) now = now & mbar_try_wait(&s_empty[set], (i / 2 - 1) & 1) & mbar_try_wait(&s_empty[set + 1], (i / 2 - 1) & 1);
        if (!now)
          now = sk_wait2(&q_full[stage], phase, &a_full[i % AS], i / AS & 1, abort_flag) &&
                (i < 2 || sk_wait2(&s_empty[set], (i / 2 - 1) & 1, &s_empty[set + 1], (i / 2 - 1) & 1, abort_flag));
        ok = __all_sync(0xffffffffu, now);
        if (!ok) break;
        tc_fence_after();
        const uint64_t dq = dQ + (uint32_t)(stage * C::Q_BYTES >> 4);
        sk_products_ts<HD / 16>(issue, tmem + set * KM_PAIRS, tmem + KP_COL_K, dq, C::Q_CH, idesc);
        tc_commit_if(issue, &s_full[set]);
        sk_products_ts<HD / 16>(issue, tmem + (set + 1) * KM_PAIRS, tmem + KP_COL_K + HD / 2, dq, C::Q_CH, idesc);
        tc_commit_if(issue, &s_full[set + 1]);
        tc_commit_if(issue, &q_empty[stage]);
        if (++stage == QS) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (!ok) break;
    }
    if (!ok) {
      if (lane == 0 && !*abort_flag) set_status(status, ST_MBAR_TIMEOUT);
      *abort_flag = 1;
    }
  } else {
    // ---- weights: sets 0 and 2 have the first 128 keys, with every other tile of queries each, 1 and 3 the others
    const int quad = warp & 3, set = (warp - 4) >> 2, place = quad * 32 + lane;
    const uint32_t taddr = tmem + ((uint32_t)(quad * 32) << 16) + set * KM_PAIRS;
    const uint64_t scale2 = f2_pack(scale_log2, scale_log2);
    bool dead = false;
    int i = 0, n = 0;                                                // tiles of queries, units of the CTA so far
    for (bool more = any && x.start(w); more; ++n) {
      // Half of a key each from shared memory into its lane of tensor memory, where every product with the keys ahead of these is through: each set has waited
      // for its own. The next unit's keys land meanwhile.
      asm volatile("bar.sync 1, %0;" ::"n"(KM_SETS * 128) : "memory");
      if (!dead && !__all_sync(0xffffffffu, sk_wait(k_full, n & 1, abort_flag))) {
        dead = true;
        if (lane == 0 && !*abort_flag) set_status(status, ST_MBAR_TIMEOUT);
        *abort_flag = 1;
      }
      if (!dead) {
        tc_fence_after();
#pragma unroll
        for (int e = 0; e < HD / 64; ++e) {
          const int x0 = (set >> 1) * (HD / 2) + e * 32;
          const unsigned char* from = sK + (set & 1) * C::K_BYTES + (x0 >> 6) * C::K_CH + place * 128;
          uint32_t c[16];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint4 v = *reinterpret_cast<const uint4*>(from + ((((x0 & 63) >> 3) + k) ^ (place & 7)) * 16);
            c[4 * k] = v.x; c[4 * k + 1] = v.y; c[4 * k + 2] = v.z; c[4 * k + 3] = v.w;
          }
          sk_tmem_st16(tmem + ((uint32_t)(quad * 32) << 16) + KP_COL_K + (set & 1) * (HD / 2) + x0 / 2, c);
        }
        tmem_st_wait();
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0 && !dead) {
        mbar_arrive(k_empty);
        mbar_arrive(t_full);
      }

      const int key = x.it.key0 + (set & 1) * KM_KEYS + place, last = key - place + KM_KEYS;
      float sum = 0.f;
      for (int j = 0; j < x.n; ++j, ++i) {
        if ((i & 1) != set >> 1) continue;
        const int f = 2 * i + (set & 1), stage = i % AS;
        if (!dead && !__all_sync(0xffffffffu, sk_wait(&s_full[set], (f / KM_SETS) & 1, abort_flag))) {
          dead = true;
          if (lane == 0 && !*abort_flag) set_status(status, ST_MBAR_TIMEOUT);
          *abort_flag = 1;
        }
        if (dead) continue;
        tc_fence_after();
        // (the pairs' numbers came with the tile: the products have waited for both)
        sum += last > ms.edge[stage] || Rq * share < KM_NEAR ? km_weights<true>(taddr, KM_PAIRS, Rq * share, ms.nl[stage], ms.kvl[stage], key, scale2)
                                                             : km_weights<false>(taddr, KM_PAIRS, Rq * share, ms.nl[stage], ms.kvl[stage], key, scale2);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&s_empty[set]);
          mbar_arrive(&a_empty[stage]);
        }
      }
      if (!dead) w.sums[((blockIdx.x + (size_t)x.item * nkv + x.kvh) * KM_SETS + set) * KM_KEYS + place] = sum;
      more = x.next(w, nkv);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == SK_ALLOC) tmem_dealloc(tmem, KP_COLS);
}

// An item's sums of all pieces, in order, into the cache's. grid: items x kv heads, a thread a key.
__global__ void __launch_bounds__(KP_KEYS) kv_mass_join_kernel(float* out, const float* mass, float carry, FbSharedStep st, KpSpace w, int nkv, int* status) {
  pdl_launch_dependents();
  pdl_wait();
  const int items = w.head[0], per = w.head[1];
  for (int i = blockIdx.x; i < items; i += gridDim.x) {
    const KpItem it = w.items[i];
    const int kvh = blockIdx.y, key = it.key0 + threadIdx.x;
    if (kvh == 0 && threadIdx.x % 32 == 0) km_take(st, w.taken, it.slot, key, it.k0, it.k1, status);
    if (key < it.k0 || key >= it.k1) continue;
    const int page = st.table[(size_t)it.slot * st.max_blocks + key / st.kv_block];
    if (page < 0 || page >= st.pages) {
      set_status(status, ST_BOUNDS);
      continue;
    }
    const size_t at = ((size_t)page * nkv + kvh) * st.kv_block + key % st.kv_block;
    const int set = threadIdx.x / KM_KEYS, place = threadIdx.x % KM_KEYS;
    float sum = 0.f;
    const long long p0 = (long long)it.place0 * nkv + (long long)kvh * it.seen;
    const int c0 = (int)(p0 / per), c1 = (int)((p0 + it.seen - 1) / per);
#pragma unroll 4
    for (int c = c0; c <= c1; ++c) {
      const float* s = w.sums + ((c + (size_t)i * nkv + kvh) * KM_SETS + set) * KM_KEYS + place;
      sum += s[0] + s[2 * KM_KEYS];
    }
    out[at] = (carry != 0.f ? carry * mass[at] : 0.f) + sum;
  }
}

}  // namespace fb

using namespace fb;

// Tensor map of the queries [rows][heads][HD]: a copy brings 64 columns of Rq rows' heads of a kv head.
static int make_tmap_queries(CUtensorMap* out, const void* q, int rows, int nq, int hd, long stride, int share, int Rq) {
  EncodeTiledFn fn = get_encode_fn();
  if (!fn) return -10;
  if ((uintptr_t)q % 16 || stride * 2 % 16) return -11;
  cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)nq, (cuuint64_t)rows};
  cuuint64_t strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)stride * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)share, (cuuint32_t)Rq}, estr[3] = {1, 1, 1};
  const CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : -12;
}
// Rows whose queries stay in shared memory
static int km_resident_rows(int hd, int share) { return (hd == 256 ? KmCfg<256>::QS : hd == 128 ? KmCfg<128>::QS : KmCfg<64>::QS) * (KM_PAIRS / share); }
// The form for few pairs takes all that fit (us, the most rows that stay / one row more, at 500, 16000, 60000 keys: 24 heads of 256, 30 rows 11 / 23, 21 / 33, 52 / 67;
// 32 of 128, 80 rows 12 / 36, 37 / 41, 118 / 102; 4 of 64, 256 rows 14 / 23, 20 / 29, 48 / 51).
static bool km_few(int rows, int max_rows, int ngrp, int hd, int share) { return (ngrp ? rows : std::min(rows, max_rows)) <= km_resident_rows(hd, share); }
static long km_words(long keys) { return (keys / 32 + 3) / 4 * 4; }
// (A span of n keys is of up to n / 256 + 2 items, and a key of the pool is of one span.)
static long km_space(KpSpace* w, float* ws, int rows, int nseg, int max_rows, int ngrp, int nkv, int share, long room, long keys, int ctas) {
  const int Rq = KM_PAIRS / share;
  const long spans = nseg + ngrp;
  const long blocks = shared_group_blocks(rows, ngrp, Rq) + shared_seg_blocks(rows, nseg, max_rows, Rq), items = std::min(spans * ((room + KP_KEYS - 1) / KP_KEYS + 1), keys / KP_KEYS + 2 * spans);
  float* at = ws;
  auto take = [&](long floats) {
    float* p = at;
    at += (floats + 3) / 4 * 4;
    return p;
  };
  KpSpace v{};
  v.head = (int*)take(4);
  v.blocks = (SharedBlock*)take(blocks * 8);
  v.items = (KpItem*)take(items * 8);
  v.starts = (KpStart*)take(ctas * 8l);
  v.sums = take((items * nkv + ctas) * KM_SETS * KM_KEYS);
  v.words = km_words(keys);
  v.taken = (uint32_t*)take(v.words);
  v.max_items = (int)std::min(items, 0x7fffffffl);
  if (w) *w = v;
  return at - ws;
}

extern "C" long fb_attention_mass_floats(int rows, int nseg, int max_rows, int ngrp, int nq, int nkv, int hd, long room, long keys, int want_lse, int ctas) {
  if (rows <= 0 || nseg <= 0 || nkv < 1 || nq / nkv < 1 || nq / nkv > KM_PAIRS) return 0;
  const int share = nq / nkv;
  const long logs = want_lse ? ((long)rows * nq + 3) / 4 * 4 + fb_attention_shared_floats(rows, nseg, max_rows, ngrp, nq, nkv, hd, ctas, 0) : 0;
  return logs + (km_few(rows, max_rows, ngrp, hd, share) ? km_words(keys) + 8l * (nseg + ngrp) : km_space(nullptr, nullptr, rows, nseg, max_rows, ngrp, nkv, share, room, keys, ctas));
}

extern "C" int fb_attention_mass_launches(int rows, int nseg, int max_rows, int ngrp, int nq, int nkv, int hd, int want_lse) {
  return rows <= 0 || nseg <= 0 || max_rows <= 0 ? 0 : (km_few(rows, max_rows, ngrp, hd, nq / nkv) ? 2 : 3) + (want_lse ? 2 : 0);
}

extern "C" int fb_attention_mass(float* out, const float* mass, float carry, const float* lse, float* ws, long ws_floats, const void* q, long q_stride,
                                 const void* k, FbSharedStep st, int nq, int nkv, int hd, int ctas, int* status, cudaStream_t s) {
  if (st.rows <= 0 || st.nseg <= 0 || st.max_rows <= 0) return 0;
  if (nkv < 1 || nq % nkv || nq / nkv > KM_PAIRS || st.kv_block % 64 || ctas < 1 || (hd != 64 && hd != 128 && hd != 256)) return -1;
  const long room = (long)st.max_blocks * st.kv_block, keys = st.pages * st.kv_block;
  if (ws_floats < fb_attention_mass_floats(st.rows, st.nseg, st.max_rows, st.ngrp, nq, nkv, hd, room, keys, !lse, ctas)) return -3;
  const int share = nq / nkv, Rq = KM_PAIRS / share;
  int rc;
  if (!lse) {
    const long used = ((long)st.rows * nq + 3) / 4 * 4, more = fb_attention_shared_floats(st.rows, st.nseg, st.max_rows, st.ngrp, nq, nkv, hd, ctas, 0);
    if ((rc = fb_attention_shared(nullptr, ws, ws + used, more, q, q_stride, k, k, nullptr, 0, st, nq, nkv, hd, ctas, status, s))) return rc;
    lse = ws;
    ws += used + more;
  }
  const float scale = 1.4426950408889634f / sqrtf((float)hd);
  CUtensorMap tmK, tmQ;
  const uint64_t cache_rows = (uint64_t)st.pages * st.kv_block, width = (uint64_t)nkv * hd;
  if ((rc = make_tmap_bf16_2d(&tmK, k, cache_rows, width, width, 64))) return rc;
  if ((rc = make_tmap_queries(&tmQ, q, st.rows, nq, hd, st.rows > 1 ? q_stride : (long)nq * hd, share, Rq))) return rc;
  cudaError_t e = cudaErrorInvalidValue;
  if (km_few(st.rows, st.max_rows, st.ngrp, hd, share)) {
    const int R = km_resident_rows(hd, share);
    SharedPlanSizes z;
    if (!shared_plan_sizes(st, shared_group_blocks(st.rows, st.ngrp, R), shared_seg_blocks(st.rows, st.nseg, st.max_rows, R), &z)) return -2;
    const long words = km_words(keys);
    if ((e = launch_pdl(kv_mass_clear_kernel, dim3((unsigned)std::min((words + 1023) / 1024, (long)ctas)), dim3(256), 0, s, (uint32_t*)ws, words)) != cudaSuccess)
      return (int)e;
#define FB_KM(H)                                                                                                                                       \
  if (hd == H) {                                                                                                                                       \
    using C = KmCfg<H>;                                                                                                                                \
    constexpr size_t smem = C::MISC_AT + sizeof(KmMisc<C::QS>);                                                                                        \
    static_assert(smem <= 232448, "shared memory of an SM");                                                                                           \
    FB_CUDA_CHECK(cudaFuncSetAttribute(kv_mass_keys_kernel<H>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));                               \
    e = launch_pdl(kv_mass_keys_kernel<H>, dim3(ctas), dim3(KM_THREADS), smem, s, tmK, tmQ, out, mass, carry, lse, st, z, (SharedBlock*)(ws + words),  \
                   (uint32_t*)ws, R, nq, nkv, scale, status);                                                                                                                \
  }
    FB_KM(64) FB_KM(128) FB_KM(256)
#undef FB_KM
    return (int)e;
  }
  KpSpace w;
  km_space(&w, ws, st.rows, st.nseg, st.max_rows, st.ngrp, nkv, share, room, keys, ctas);
  if (!shared_plan_sizes(st, shared_group_blocks(st.rows, st.ngrp, Rq), shared_seg_blocks(st.rows, st.nseg, st.max_rows, Rq), &w.z)) return -2;
  FB_CUDA_CHECK(cudaFuncSetAttribute(kv_mass_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SK_PLAN_BYTES));
  if ((e = launch_pdl(kv_mass_plan_kernel, dim3(1), dim3(KP_PLAN), SK_PLAN_BYTES, s, st, w, Rq, nkv, ctas, status)) != cudaSuccess) return (int)e;
#define FB_KP(H)                                                                                                                                       \
  if (hd == H) {                                                                                                                                       \
    using C = KmCfg<H>;                                                                                                                                \
    using M = KmMisc<C::AS>;                                                                                                                           \
    constexpr size_t smem = C::ROWS_AT + sizeof(M);                                                                                                    \
    static_assert(smem <= 232448, "shared memory of an SM");                                                                                           \
    FB_CUDA_CHECK(cudaFuncSetAttribute(kv_mass_rows_kernel<H>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));                                \
    e = launch_pdl(kv_mass_rows_kernel<H>, dim3(ctas), dim3(KM_THREADS), smem, s, tmK, tmQ, lse, st, w, nq, nkv, scale, status);                        \
  }
  FB_KP(64) FB_KP(128) FB_KP(256)
#undef FB_KP
  if (e != cudaSuccess) return (int)e;
  return (int)launch_pdl(kv_mass_join_kernel, dim3(std::min(w.max_items, 1024), nkv), dim3(KP_KEYS), 0, s, out, mass, carry, st, w, nkv, status);
}

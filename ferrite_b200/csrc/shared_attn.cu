// Attention of a step's rows over a paged cache in which streams share the pages of a prefix, on the 5th-generation tensor cores: the keys and values of a
// prefix are read once for all rows of its group.
//
//   S = Q K^T        128 (row, head) pairs of a block x 64 keys; Q and K in shared memory
//   P = exp2(S - m)  two threads a pair; P as a bf16 value and its bf16 remainder, so that a weight keeps 16 bits, back into TMEM
//   O += P V         A = P from TMEM, V read along its columns from shared memory, O in TMEM while the CTA stays with the pairs
//
// Work (shared_kv.cuh): every CTA takes the same number of consecutive key tiles of the list of all (block, kv head) units. A unit that a CTA leaves or ends
// is a piece: its running maximum, sum and O in 32 bits go to the workspace, and a second kernel joins a row's pieces (of its group's shared tokens, then
// of its own) in the order of the list. Where the contexts are cut follows the step's lengths, so a row may round differently beside other streams; the
// same call gives the same bits.
//
// Warp roles: 0 loads keys, 10 loads values, 1 issues the products, 2..9 run the softmax, bring the queries and write the pieces. The running maximum moves only
// when a row's new one exceeds it by 2^8. Every wait is bounded: one that runs out sets the status word and an abort flag; the softmax warps then go
// through their remaining barriers without work, the others leave, and the CTA frees its TMEM.
#include <algorithm>

#include "gemm_core.cuh"
#include "shared_kv.cuh"

namespace fb {

constexpr int SA_PAIRS = 128, SA_KT = 64, SA_THREADS = 11 * 32;

template <int HD, bool OUT>
struct SaCfg {
  static constexpr int NCH = HD / 64, Q_CH = SA_PAIRS * 128, KV_CH = SA_KT * 128;
  static constexpr int Q_BYTES = NCH * Q_CH, T_BYTES = NCH * KV_CH;
  static constexpr int KS = OUT ? (HD == 256 ? 3 : HD == 128 ? 6 : 8) : (HD == 256 ? 5 : 8);
  static constexpr int VS = OUT ? (HD == 256 ? 2 : HD == 128 ? 5 : 8) : 0;
  static constexpr int TILES = Q_BYTES + (KS + VS) * T_BYTES;
  static constexpr int MISC_AT = (TILES > SK_PLAN_BYTES ? TILES : SK_PLAN_BYTES + 1023) / 1024 * 1024;
  // TMEM: O | S0 S1 | P0 P1 | remainders
  static constexpr uint32_t COL_S = OUT ? HD : 0, COL_P = COL_S + 2 * SA_KT, COL_R = COL_P + SA_KT;
  static constexpr uint32_t COLS = OUT ? 512 : 128;
};
struct SaMisc {
  float mx[2][2][SA_PAIRS];                      // by the tile's parity and half
  long long tmp[SA_THREADS / 32 + 1];
  uint64_t bars[10 + 4 * 8];
  uint8_t bad[2][8];                             // keys of a tile whose values are no numbers
  uint32_t tmem;
  int abort;
};

// Where things lie in the workspace. ml: maximum (log2), sums of the two halves of the keys; records of 128 pairs for groups, of seg_pairs for segments.
struct SaSpace {
  long long* head;                               // tiles a CTA, blocks of groups
  SharedBlock* table;
  int* rows;                                     // [rows][2]: block of a row's group, of its segment, or -1
  float4 *ml_grp, *ml_seg;
  float *o_grp, *o_seg;
  int max_blocks, max_group_blocks, seg_pairs;
};

// A CTA's way through its share of the list: (block, kv head) after (block, kv head).
struct SaWalk {
  SharedBlock e;
  int b, kvh, t, n;                              // n: tiles of the piece
  int left;                                      // ... and behind it
  const SharedBlock* table;
  __device__ __forceinline__ void take() {
    n = min(e.nt - t, left);
    left -= n;
  }
  __device__ __forceinline__ void start(const SharedBlock* tab, int b0, long long f0, int tiles, int nkv) {
    table = tab;
    b = b0;
    e = table[b];
    const int at = (int)(f0 - (long long)e.tile0 * nkv);
    kvh = at / e.nt;
    t = at - kvh * e.nt;
    left = tiles;
    take();
  }
  __device__ __forceinline__ bool next(int nkv) {
    if (left == 0) return false;
    t = 0;
    if (++kvh == nkv) {
      kvh = 0;
      do e = table[++b];
      while (e.nt == 0);
    }
    take();
    return true;
  }
  __device__ __forceinline__ int token(int j) const { return (e.k0 / SA_KT + t + j) * SA_KT; }
};

template <int HD, bool OUT>
__global__ void __launch_bounds__(SA_THREADS, 1)
shared_attn_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __nv_bfloat16* q, long q_stride, FbSharedStep st,
                   SaSpace w, int nkv, int share, float scale_log2, int* status) {
  using C = SaCfg<HD, OUT>;
  constexpr int NCH = C::NCH, KS = C::KS, VS = C::VS;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char *sQ = smem, *sK = smem + C::Q_BYTES, *sV = sK + KS * C::T_BYTES;
  SaMisc& ms = *reinterpret_cast<SaMisc*>(smem + C::MISC_AT);
  uint64_t *q_full = ms.bars, *o_empty = q_full + 1, *s_full = q_full + 2, *s_empty = q_full + 4, *p_full = q_full + 6, *p_empty = q_full + 8,
           *k_full = q_full + 10, *k_empty = k_full + KS, *v_full = k_empty + KS, *v_empty = v_full + VS;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort_flag = &ms.abort;
  pdl_launch_dependents();
  if (smem_u32(smem) & 1023u) {                                      // the swizzled tiles need the 1024-byte base
    if (tid == 0) set_status(status, ST_BOUNDS);
    return;
  }
  if (tid == 0) {
    ms.abort = 0;
    mbar_init(q_full, 8);
    mbar_init(o_empty, 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1); mbar_init(&s_empty[i], 8); mbar_init(&p_full[i], 8); mbar_init(&p_empty[i], 1);
    }
    for (int i = 0; i < KS; ++i) { mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1); }
    for (int i = 0; i < VS; ++i) { mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 1); }
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&ms.tmem, C::COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ms.tmem;
  pdl_wait();

  // ---- this CTA's share
  const int R = SA_PAIRS / share;
  SharedPlan<SA_THREADS> plan;
  const bool fits = plan.make(st, R, SA_KT, w.max_group_blocks, w.max_blocks - w.max_group_blocks, smem, ms.tmp, status);
  const long long all = fits ? plan.tiles * nkv : 0, per = max(1ll, (all + gridDim.x - 1) / gridDim.x);
  const long long f0 = min(all, blockIdx.x * per), f1 = min(all, f0 + per);
  if (blockIdx.x == 0 && tid == 0) {
    w.head[0] = fits && per < 1ll << 31 ? per : 0;
    w.head[1] = fits ? plan.group_blocks : 0;
  }
  if (fits && blockIdx.x == 0)
    for (int b = tid; b < plan.blocks; b += SA_THREADS) {            // blocks that have no keys
      if ((b + 1 < plan.blocks ? (long long)plan.tile[b + 1] : plan.tiles) > plan.tile[b]) continue;
      const SharedBlock e = plan.block(st, b, R, SA_KT, status);
      const int s = plan.span[b] - st.ngrp;
      for (int r = e.row0; r < e.row0 + e.nrows; ++r) {
        w.rows[2 * r + (s >= 0)] = -1;
        if (s >= 0 && plan.group[s] < 0) w.rows[2 * r] = -1;
      }
    }
  if (f0 == f1 || per >= 1ll << 31) {                                // the same for the whole CTA
    if (tid == 0 && per >= 1ll << 31) set_status(status, ST_CAPACITY);
    if (warp == 1) tmem_dealloc(tmem, C::COLS);
    return;
  }
  const int b0 = plan.find(f0, nkv), b1 = plan.find(f1 - 1, nkv), tiles = (int)(f1 - f0), group_blocks = plan.group_blocks;
  for (int b = b0 + tid; b <= b1; b += SA_THREADS) {                 // (other CTAs of a block write the same)
    SharedBlock e = plan.block(st, b, R, SA_KT, status);
    e.tile0 = plan.tile[b];
    w.table[b] = e;
    const int s = plan.span[b] - st.ngrp;
    for (int r = e.row0; r < e.row0 + e.nrows && e.nt; ++r) {
      w.rows[2 * r + (s >= 0)] = b;
      if (s >= 0 && plan.group[s] < 0) w.rows[2 * r] = -1;
    }
  }
  fence_proxy_async();                                               // tiles take the plan's place
  __syncthreads();
  SaWalk x;
  x.start(w.table, b0, f0, tiles, nkv);

  if (warp == 0 || warp == 10) {
    // ---- keys (warp 0) and values (warp 10): the lanes look up 32 tiles' pages at a time, one of them copies
    const bool keys = warp == 0;
    if (!keys && !OUT) goto done;
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
  } else if (warp == 1) {
    // ---- products, issued from the whole warp by one lane's predicate
    constexpr uint32_t idesc_s = umma_idesc(1, 1, SA_PAIRS, SA_KT);
    constexpr uint32_t idesc_pv = umma_idesc(1, 1, SA_PAIRS, HD) | (1u << 16);         // B read MN-major
    const uint32_t aQ = smem_u32(sQ), aK = smem_u32(sK), aV = smem_u32(sV);
    const bool issue = elect_one();
    auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, sk_wait(bar, parity, abort_flag)); };
    int kst = 0, kph = 0, vst = 0, vph = 0, i = 0, piece = 0;
    auto issue_s = [&](int at) -> bool {
      const int s = at & 1;
      if (!wait(&k_full[kst], kph)) return false;
      if (at >= 2 && !wait(&s_empty[s], ((at >> 1) - 1) & 1)) return false;
      tc_fence_after();
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        const uint32_t off = (uint32_t)(kk & 3) * 32u;
        tc_mma_f16_if(issue, tmem + C::COL_S + s * SA_KT, umma_desc_k128(aQ + (kk >> 2) * C::Q_CH + off),
                      umma_desc_k128(aK + kst * C::T_BYTES + (kk >> 2) * C::KV_CH + off), idesc_s, kk > 0 ? 1u : 0u);
      }
      tc_commit_if(issue, &s_full[s]);
      tc_commit_if(issue, &k_empty[kst]);
      if (++kst == KS) {
        kst = 0;
        kph ^= 1;
      }
      return true;
    };
    bool ok = wait(q_full, 0) && issue_s(0);
    bool more = true;
    while (ok && more) {
      for (int j = 0; ok && j < x.n; ++j, ++i) {
        if (j + 1 < x.n) ok = issue_s(i + 1);
        if constexpr (OUT) {
          const int s = i & 1;
          ok = ok && wait(&p_full[s], (i >> 1) & 1) && wait(&v_full[vst], vph) && (j > 0 || piece == 0 || wait(o_empty, (piece - 1) & 1));
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < SA_KT / 16; ++kk)
            tc_mma_f16_ts_if(issue, tmem, tmem + C::COL_P + s * (SA_KT / 2) + kk * 8,
                             sk_desc_mn128(aV + vst * C::T_BYTES + kk * 16 * 128, C::KV_CH, 1024), idesc_pv, (j > 0 || kk > 0) ? 1u : 0u);
#pragma unroll
          for (int kk = 0; kk < SA_KT / 16; ++kk)
            tc_mma_f16_ts_if(issue, tmem, tmem + C::COL_R + s * (SA_KT / 2) + kk * 8,
                             sk_desc_mn128(aV + vst * C::T_BYTES + kk * 16 * 128, C::KV_CH, 1024), idesc_pv, 1u);
          tc_commit_if(issue, &v_empty[vst]);
          tc_commit_if(issue, &p_empty[s]);
          if (++vst == VS) {
            vst = 0;
            vph ^= 1;
          }
        }
      }
      if (!ok) break;
      more = x.next(nkv);
      ++piece;
      if (more) ok = wait(q_full, piece & 1) && issue_s(i);
    }
    if (!ok) {
      if (lane == 0 && !*abort_flag) set_status(status, ST_MBAR_TIMEOUT);
      *abort_flag = 1;
    }
  } else {
    // ---- softmax, queries, pieces: warps 2..5 take keys 0..31 of a tile, 6..9 the others; a pair's two threads sit in the same lane quadrant
    const int quad = warp & 3, half = (warp - 2) >> 2, st_tid = tid - 64;
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
    auto copy_q = [&](const SaWalk& y) {                             // 16 bytes at a time, swizzled as the products read them
      const int pieces = y.e.nrows * share * (HD / 8);
      const __nv_bfloat16* src = q + (long)y.e.row0 * q_stride + (long)y.kvh * share * HD;
      for (int c = st_tid; c < pieces; c += 256) {
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
    copy_q(x);
    give_q();
    int i = 0;
    bool more = true;
    while (more) {
      const SaWalk y = x;
      more = x.next(nkv);
      const int np = y.e.nrows * share;
      const int klen = pair < np ? min(st.kvlen[y.e.row0 + pair / share], y.e.k1) : 0;
      const bool active = quad * 32 < np;                            // (the same for both warps of a quadrant)
      float m_ref = -INFINITY, l = 0.f;
      for (int j = 0; j < y.n; ++j, ++i) {
        const int s = i & 1, t0 = y.token(j);
        const bool need_mask = t0 < y.e.k0 || t0 + SA_KT > y.e.kmin;
        wait(&s_full[s], (i >> 1) & 1);
        if (j + 1 == y.n && more && !dead) copy_q(x);                // every product that reads the queries is through
        if constexpr (OUT) if (need_mask) {
          // Values of keys that some row does not see meet weights of zero: those that no row sees become zeros, those that some see are looked at,
          // and where one is no finite number the key's values become zeros and its score NaN for the rows that see it.
          if (!dead) {
            wait(&v_full[i % VS], (i / VS) & 1);
          }
          if (!dead) {
            const int key = st_tid >> 2, part = st_tid & 3, tok = t0 + key;
            unsigned char* base = sV + (i % VS) * C::T_BYTES;
            constexpr int PER = HD / 32;                             // 16-byte pieces of a thread
            auto at = [&](int e) { return reinterpret_cast<uint4*>(base + ((part * PER + e) >> 3) * C::KV_CH + key * 128 + ((part * PER + e) & 7) * 16); };
            bool zero = tok < y.e.k0 || tok >= y.e.k1;
            bool bad = false;
            if (!zero && tok >= y.e.kmin) {
#pragma unroll
              for (int e = 0; e < PER; ++e) {
                const uint4 u = *at(e);
                const uint32_t a[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) bad |= (a[k] & 0x7f80u) == 0x7f80u || (a[k] & 0x7f800000u) == 0x7f800000u;
              }
            }
            const uint32_t bal = __ballot_sync(0xffffffffu, bad);
            zero |= (bal >> (lane & 28)) & 15u;
            if (zero)
#pragma unroll
              for (int e = 0; e < PER; ++e) *at(e) = make_uint4(0, 0, 0, 0);
            if (lane == 0) {
              uint32_t bits = 0;
              for (int k = 0; k < 8; ++k) bits |= ((bal >> (4 * k)) & 15u) ? 1u << k : 0u;
              ms.bad[s][st_tid >> 5] = (uint8_t)bits;
            }
            fence_proxy_async();
          }
          asm volatile("bar.sync 5, 256;" ::: "memory");
        }
        if (!active) {
          __syncwarp();
          if (lane == 0 && !dead) {
            mbar_arrive(&s_empty[s]);
            if (OUT) mbar_arrive(&p_full[s]);
          }
          continue;
        }
        uint32_t sr[HC];
        float mx = -INFINITY;
        if (!dead) {
          tc_fence_after();
          tmem_ld32(tmem + lane_addr + C::COL_S + s * SA_KT + half * HC, sr);
          tmem_ld_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_empty[s]);
          if (need_mask) {
            const int c0 = t0 + half * HC;
            const uint32_t bad = OUT ? reinterpret_cast<const uint32_t*>(ms.bad[s])[half] : 0u;
#pragma unroll
            for (int c = 0; c < HC; ++c) {
              float v = __uint_as_float(sr[c]) * scale_log2;
              if (bad >> c & 1u) v = NAN;
              if (c0 + c < y.e.k0 || c0 + c >= klen) v = -INFINITY;
              sr[c] = __float_as_uint(v);
              mx = fmaxf(mx, v);
            }
          } else {
#pragma unroll
            for (int c = 0; c < HC; ++c) {
              const float v = __uint_as_float(sr[c]) * scale_log2;
              sr[c] = __float_as_uint(v);
              mx = fmaxf(mx, v);
            }
          }
        }
        ms.mx[s][half][pair] = mx;
        asm volatile("bar.sync %0, 64;" ::"r"(1 + quad) : "memory");
        mx = pair < np ? fmaxf(mx, ms.mx[s][half ^ 1][pair]) : -INFINITY;      // (what lies behind the pairs moves no maximum)
        const bool any = __any_sync(0xffffffffu, mx > m_ref + 8.f);
        if (OUT) {
          // P(i - 2) has been read; where O is rescaled, PV(i - 1) is through
          if (i >= 2) wait(&p_empty[s], ((i >> 1) - 1) & 1);
          if (any && j > 0) wait(&p_empty[s ^ 1], ((i - 1) >> 1) & 1);
        }
        if (dead) continue;
        if (OUT) tc_fence_after();
        if (any) {
          const float m_new = fmaxf(m_ref, mx);
          const float f = m_ref == -INFINITY ? 0.f : sk_exp2(m_ref - m_new);
          l = m_ref == -INFINITY ? l : l * f;                        // (a sum that is no number stays one)
          if (OUT && j > 0) {
#pragma unroll 1
            for (int c0 = 0; c0 < OC; c0 += 32) {
              uint32_t o[32];
              tmem_ld32(tmem + lane_addr + half * OC + c0, o);
              tmem_ld_wait();
#pragma unroll
              for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * f);
              tmem_st32(tmem + lane_addr + half * OC + c0, o);
            }
            tmem_st_wait();
          }
          m_ref = m_new;
        }
        const float mr = m_ref == -INFINITY ? 0.f : m_ref;
        float sum = 0.f;
        uint32_t pr[HC / 2], px[HC / 2];
#pragma unroll
        for (int c = 0; c < HC / 2; ++c) {
          const float p0 = sk_exp2(__uint_as_float(sr[2 * c]) - mr), p1 = sk_exp2(__uint_as_float(sr[2 * c + 1]) - mr);
          sum += p0 + p1;
          if constexpr (OUT) {
            pr[c] = pack_bf2(p0, p1);
            px[c] = pack_bf2(p0 - bf_lo(pr[c]), p1 - bf_hi(pr[c]));
          }
        }
        l += sum;
        if constexpr (OUT) {
          sk_tmem_st16(tmem + lane_addr + C::COL_P + s * (SA_KT / 2) + half * (HC / 2), pr);
          sk_tmem_st16(tmem + lane_addr + C::COL_R + s * (SA_KT / 2) + half * (HC / 2), px);
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[s]);
        }
      }
      if (more) give_q();
      // ---- the piece: record number = CTA + unit, which no other piece has
      const bool grp = y.b < group_blocks;
      const long rec = (long)blockIdx.x + (long)(y.b - (grp ? 0 : group_blocks)) * nkv + y.kvh;
      const int stride = grp ? SA_PAIRS : w.seg_pairs;
      if (active && pair < np && !dead) {
        float* ml = reinterpret_cast<float*>((grp ? w.ml_grp : w.ml_seg) + rec * stride + pair);
        if (half == 0) *reinterpret_cast<float2*>(ml) = make_float2(m_ref, l);
        else ml[2] = l;
      }
      if constexpr (OUT) {
        wait(&p_empty[(i - 1) & 1], ((i - 1) >> 1) & 1);
        if (active && !dead) {
          tc_fence_after();
          float* o = (grp ? w.o_grp : w.o_seg) + (rec * stride) * HD + half * OC + 2 * (lane & 3);
#pragma unroll 1
          for (int r0 = quad * 32; r0 < min(np, quad * 32 + 32); r0 += 16) {
            const int ra = r0 + (lane >> 2), rb = ra + 8;
#pragma unroll 1
            for (int c0 = 0; c0 < OC; c0 += 32) {
              uint32_t v[16];
              sk_tmem_ld16x32(tmem + ((uint32_t)r0 << 16) + half * OC + c0, v);
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                if (ra < np) *reinterpret_cast<float2*>(o + (long)ra * HD + c0 + 8 * k) = make_float2(__uint_as_float(v[4 * k]), __uint_as_float(v[4 * k + 1]));
                if (rb < np) *reinterpret_cast<float2*>(o + (long)rb * HD + c0 + 8 * k) = make_float2(__uint_as_float(v[4 * k + 2]), __uint_as_float(v[4 * k + 3]));
              }
            }
          }
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0 && !dead) mbar_arrive(o_empty);
      }
    }
  }
done:
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, C::COLS);
}

// Pieces of a row's heads that share a kv head -> output and logarithm. grid: rows x kv heads.
__global__ void __launch_bounds__(256) shared_join_kernel(__nv_bfloat16* out, float* lse, const __nv_bfloat16* proj, long proj_stride, FbSharedStep st, SaSpace w,
                                                          int nkv, int share, int hd, int ctas) {
  __shared__ float top_s[SA_PAIRS], inv_s[SA_PAIRS];
  const int row = blockIdx.x, kvh = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_launch_dependents();
  pdl_wait();
  bool mine = false;
  for (int s = tid; s < st.nseg; s += 256) mine |= row >= st.seg_row0[s] && row - st.seg_row0[s] < st.seg_nrows[s];
  if (!__syncthreads_or(mine)) return;                               // a row of no segment
  const long long per = w.head[0];
  const int group_blocks = (int)w.head[1], n = st.kvlen[row];
  if (per <= 0) return;                                              // the step did not fit
  // a row's two runs of records; checked, since a launch that gave up has not written all of this
  const float4* ml[2];
  const float* o[2];
  int pieces[2], stride[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    pieces[k] = 0;
    const int b = w.rows[2 * row + k];
    if (b < 0 || b >= w.max_blocks || (k == 0) != (b < group_blocks) || group_blocks > w.max_group_blocks) continue;
    const SharedBlock e = w.table[b];
    const long long at = (long long)e.tile0 * nkv + (long long)kvh * e.nt;
    const long long c0 = at / per, c1 = (at + e.nt - 1) / per;
    const int r = row - e.row0;
    if (e.nt <= 0 || e.tile0 < 0 || c1 >= ctas || r < 0 || r >= e.nrows || (k && b - group_blocks >= w.max_blocks - w.max_group_blocks)) continue;
    stride[k] = k == 0 ? SA_PAIRS : w.seg_pairs;
    const long rec = (long)c0 + (long)(b - (k ? group_blocks : 0)) * nkv + kvh;
    if ((r + 1) * share > stride[k]) continue;
    ml[k] = (k == 0 ? w.ml_grp : w.ml_seg) + rec * stride[k] + r * share;
    o[k] = (k == 0 ? w.o_grp : w.o_seg) + (rec * stride[k] + r * share) * hd;
    pieces[k] = (int)(c1 - c0) + 1;
  }
  const int total = pieces[0] + pieces[1];
  auto stat = [&](int i, int g) { return i < pieces[0] ? ml[0][(long)i * stride[0] + g] : ml[1][(long)(i - pieces[0]) * stride[1] + g]; };
  for (int g = warp; g < share; g += 8) {
    float top = -INFINITY, sum = 0.f;
    for (int i = lane; i < total; i += 32) top = fmaxf(top, stat(i, g).x);
    top = warp_max(top);
    for (int i = lane; i < total; i += 32) {
      const float4 v = stat(i, g);
      const float l = v.y + v.z;
      sum += v.x == -INFINITY ? (l != l ? l : 0.f) : l * sk_exp2(v.x - top);
    }
    sum = warp_sum(sum);
    if (lane == 0) {
      const int h = kvh * share + g;
      top_s[g] = top;
      inv_s[g] = n <= 0 ? 0.f : sum == 0.f ? NAN : 1.f / sum;        // (scores of minus infinity only: 0 / 0)
      if (lse) lse[(long)row * nkv * share + h] = n <= 0 ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
    }
  }
  if (!out) return;
  __syncthreads();
  for (int c = tid; c < share * (hd / 4); c += 256) {
    const int g = c / (hd / 4), d = c % (hd / 4) * 4, h = kvh * share + g;
    const float top = top_s[g], inv = inv_s[g];
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll 8
      for (int i = 0; i < pieces[k]; ++i) {
        const float4 v = *reinterpret_cast<const float4*>(o[k] + ((long)i * stride[k] + g) * hd + d);
        const float m = ml[k][(long)i * stride[k] + g].x, f = m == -INFINITY ? 0.f : sk_exp2(m - top);
        a.x = fmaf(v.x, f, a.x); a.y = fmaf(v.y, f, a.y); a.z = fmaf(v.z, f, a.z); a.w = fmaf(v.w, f, a.w);
      }
    a.x *= inv; a.y *= inv; a.z *= inv; a.w *= inv;
    if (proj) {
      const __nv_bfloat16* gate = proj + (long)row * proj_stride + (long)h * 2 * hd + hd + d;
      a.x *= sigmoidf_(bf2f(gate[0])); a.y *= sigmoidf_(bf2f(gate[1])); a.z *= sigmoidf_(bf2f(gate[2])); a.w *= sigmoidf_(bf2f(gate[3]));
    }
    *reinterpret_cast<uint2*>(out + ((long)row * nkv * share + h) * hd + d) = make_uint2(pack_bf2(a.x, a.y), pack_bf2(a.z, a.w));
  }
}

}  // namespace fb

using namespace fb;

// The workspace: header | table | rows | statistics | sums. -> floats in all
static long sa_space(SaSpace* w, float* ws, int rows, int nseg, int max_rows, int ngrp, int nq, int nkv, int hd, int ctas, int want_out) {
  const int share = nq / nkv, R = SA_PAIRS / share;
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
  v.rows = (int*)take(2l * rows);
  v.ml_grp = (float4*)take(recs[0] * 4);
  v.ml_seg = (float4*)take(recs[1] * 4);
  v.o_grp = take(want_out ? recs[0] * hd : 0);
  v.o_seg = take(want_out ? recs[1] * hd : 0);
  v.max_blocks = (int)std::min(gb + sb, 0x7fffffffl);
  v.max_group_blocks = (int)std::min(gb, 0x7fffffffl);
  v.seg_pairs = (int)pairs;
  if (w) *w = v;
  return at - ws;
}

extern "C" long fb_attention_shared_floats(int rows, int nseg, int max_rows, int ngrp, int nq, int nkv, int hd, int ctas, int want_out) {
  if (rows <= 0 || nseg <= 0 || nkv < 1 || nq / nkv < 1 || nq / nkv > SA_PAIRS) return 0;
  return sa_space(nullptr, nullptr, rows, nseg, max_rows, ngrp, nq, nkv, hd, ctas, want_out);
}

extern "C" int fb_attention_shared(void* out, float* lse, float* ws, long ws_floats, const void* q, long q_stride, const void* k, const void* v,
                                   const void* proj, long proj_stride, FbSharedStep st, int nq, int nkv, int hd, int ctas, int* status, cudaStream_t s) {
  if (st.rows <= 0 || st.nseg <= 0) return 0;
  if (nkv < 1 || nq % nkv || nq / nkv > SA_PAIRS || st.kv_block % SA_KT || st.nseg > SK_SEGS || st.ngrp > SK_SEGS || ctas < 1) return -1;
  SaSpace w;
  if (ws_floats < sa_space(&w, ws, st.rows, st.nseg, st.max_rows, st.ngrp, nq, nkv, hd, ctas, out != nullptr)) return -3;
  if (st.rows / (SA_PAIRS / (nq / nkv)) * (st.ngrp ? 2l : 1l) > SK_BLOCKS - st.nseg - st.ngrp) return -2;        // more rows than a plan has room for
  const int share = nq / nkv;
  const float scale = 1.4426950408889634f / sqrtf((float)hd);
  CUtensorMap tmK, tmV;
  int rc;
  const uint64_t cache_rows = (uint64_t)st.pages * st.kv_block, width = (uint64_t)nkv * hd;
  if ((rc = make_tmap_bf16_2d(&tmK, k, cache_rows, width, width, SA_KT))) return rc;
  if ((rc = make_tmap_bf16_2d(&tmV, v, cache_rows, width, width, SA_KT))) return rc;
  cudaError_t e = cudaErrorInvalidValue;
#define FB_SA(H, OUTV)                                                                                                                              \
  if (hd == H && (out != nullptr) == OUTV) {                                                                                                        \
    auto kern = shared_attn_kernel<H, OUTV>;                                                                                                        \
    const size_t smem = SaCfg<H, OUTV>::MISC_AT + sizeof(SaMisc);                                                                                   \
    static_assert(SaCfg<H, OUTV>::MISC_AT + sizeof(SaMisc) <= 232448, "shared memory of an SM");                                                    \
    FB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));                                              \
    e = launch_pdl(kern, dim3(ctas), dim3(SA_THREADS), smem, s, tmK, tmV, (const __nv_bfloat16*)q, q_stride, st, w, nkv, share, scale, status);     \
  }
  FB_SA(64, true) FB_SA(128, true) FB_SA(256, true) FB_SA(64, false) FB_SA(128, false) FB_SA(256, false)
#undef FB_SA
  if (e != cudaSuccess) return (int)e;
  return (int)launch_pdl(shared_join_kernel, dim3(st.rows, nkv), dim3(256), 0, s, (__nv_bfloat16*)out, lse, (const __nv_bfloat16*)proj, proj_stride, st, w,
                         nkv, share, hd, ctas);
}

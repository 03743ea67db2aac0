// Attention over a latent cache in 4 or 8 bits (rows as in mla_cache.cuh) on the 5th-generation tensor cores, absorbed form: every head attends the same
// rows, o = softmax(scale * q . [value | key part]) value.
//
// Keys are the wide side of both products (M = 128), (row, head) pairs of a segment the narrow one (N = 16, 32 or 64): one unpacking of the codes serves
// N pairs and both products.
//
//   S^T [128 keys x N]  = [K | key part] Q^T     A: the tile's values, rows of keys; B: the pairs' queries
//   O^T [L x N]        += V^T P^T                A: the SAME tile in shared memory, read along its columns; B: the weights, written by the softmax
//
// Warps 0..7 unpack (two threads a key, 32 of every 64 values each): a word of eight 4-bit codes takes a shift, a mask and one fma per two values, fp16(16 +
// code + 8) * s - 24 s, exact in fp16 as the value itself is (a power of two times seven bits). The codes of the next tile are in flight in registers meanwhile.
// Warps 8..15 run the softmax: a thread has a key (its TMEM lane) and half of the pairs. Warp 16 issues the products.
// The values' products run in fp16, so that a weight keeps 11 bits; a query is brought to 2^10 by a power of two of its own, which keeps its bf16 bits down
// to 2^-27 of its largest value. The key part stays in bf16 (its products go to the same sums).
//
// Softmax along the lanes: a column's maximum would need all 128 threads, every tile. Instead a piece's first tile gives the reference r (its maximum - 4),
// and weights are 2^(x - r): exact whatever r is, as long as fp16 holds them. Only where a later score passes r by 2^15 (a vote of the 256 threads,
// every tile) is the maximum taken anew and O rescaled.
//
// Work is cut evenly, not by row: the tiles of all (segment, group of N pairs) units form one list, every CTA takes the same number of consecutive
// ones, from what the lengths on the device say (so a captured call follows its contexts). Units that span CTAs leave their sums in 32 bits,
// and a second kernel joins them in order. A row's bits therefore depend on what else is in the step, and on nothing else.
//
// A key of which a group is no number gets the score NaN and a finite place in the tile, so that rows ahead of it, whose weight for it is zero, stay clean.
// Every wait is bounded: one that runs out sets the status word and an abort flag, all roles leave and the CTA frees its TMEM.
#include "api_ext.h"
#include "gemm_core.cuh"
#include "mla_cache.cuh"

namespace fb {

constexpr int LA_KT = 128;                       // keys of a tile
constexpr int LA_CH = LA_KT * 128;               // bytes of 64 values of all of them
constexpr int LA_THREADS = 17 * 32;
constexpr float LA_TOP = 4.f, LA_LIMIT = 15.f;   // log2 of a piece's first largest weight; of the largest one that a weight may be

template <int BITS, int NC, int N>
struct LatentAttn {
  static constexpr int L = NC * 64, CW = N / 2;                    // CW: pairs of a softmax thread
  static constexpr int NP = (NC + 1) / 2;                          // pairs of 64 values: rows of 128 of O^T
  static constexpr int NB = NC == 8 ? (N == 64 ? 4 : 5) : 2 * NP;  // buffers of them
  static constexpr bool SHARE = NC == 8 && N == 64;                // the weights take the place of the tile's key part
  static constexpr int PD = BITS == 8 && NC == 8 ? 4 : NC;         // 64s of values in flight
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
  uint32_t bad[4][8];                            // of the last tiles: keys that are no number, two bits a key
  long long scan[18];
  int start[4];
  uint64_t bars[2 * 5 + 7];
  uint32_t tmem;
  int abort, fail;
};

struct LatentSegs {
  const int *slot, *row0, *nrows, *kvlen;
  int nseg, nq;
  long limit;                                    // keys that a table has room for
};
struct LatentWalk {                              // a place in the list of tiles
  int s, u, t, units, nt, kv, row0, nrows;
  template <int N>
  __device__ __forceinline__ void load(const LatentSegs& g) {
    nrows = g.nrows[s]; row0 = g.row0[s];
    kv = nrows > 0 ? (int)min((long)max(g.kvlen[row0 + nrows - 1], 0), g.limit) : 0;
    units = (int)(((long)max(nrows, 0) * g.nq + N - 1) / N);
    nt = max(1, (kv + LA_KT - 1) / LA_KT);
  }
  template <int N>
  __device__ __forceinline__ void next_unit(const LatentSegs& g) {
    t = 0;
    if (++u < units) return;
    u = 0;
    units = 0;
    while (++s < g.nseg) {
      load<N>(g);
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
  float a[W];
#pragma unroll
  for (int i = 0; i < W; ++i) a[i] = v[i];
#pragma unroll
  for (int off = W / 2; off > 0; off >>= 1) {
    const bool up = lane & off;
#pragma unroll
    for (int i = 0; i < off; ++i) {
      const float keep = up ? a[i + off] : a[i], give = up ? a[i] : a[i + off];
      a[i] = op(keep, __shfl_xor_sync(0xffffffffu, give, off));
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

// 32 values of a key: codes -> fp16 in four 16-byte places of the key's 128 bytes
template <int BITS>
__device__ __forceinline__ void unpack32(const uint4 (&raw)[BITS / 4], uint32_t sb0, uint32_t sb1, unsigned char* row, int first, int turn) {
  if constexpr (BITS == 4) {
    const uint32_t w[4] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const __half2 s = __float2half2_rn(latent_scale<4>(q < 2 ? sb0 : sb1)), m = __hmul2(s, __float2half2_rn(-24.f));
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t t = ((i == 0 ? w[q] << 6 : i == 1 ? w[q] << 2 : i == 2 ? w[q] >> 2 : w[q] >> 6) & 0x03c003c0u) | 0x4c004c00u;
        const __half2 h = __hfma2(*reinterpret_cast<const __half2*>(&t), s, m);
        o[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
      *reinterpret_cast<uint4*>(row + (((first + q) ^ turn) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  } else {
    const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
    const __half2 s = __float2half2_rn(latent_scale<8>(sb0));
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[2 * q + i / 2] >> (16 * (i % 2))), __NV_E4M3);
        const __half2 h = __hmul2(*reinterpret_cast<const __half2*>(&r), s);
        o[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
      *reinterpret_cast<uint4*>(row + (((first + q) ^ turn) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
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
           *ofull = qfull + 1, *oempty = ofull + 1;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort_flag = &ms.abort;
  pdl_launch_dependents();
  if (tid == 0) {
    ms.abort = 0; ms.fail = 0;
    for (int i = 0; i < NB; ++i) { mbar_init(&kfull[i], 8); mbar_init(&kempty[i], 1); }
    mbar_init(rfull, 8); mbar_init(rempty, 1); mbar_init(sfull, 1); mbar_init(pfull, 8); mbar_init(qfull, 8); mbar_init(ofull, 1); mbar_init(oempty, 8);
    fence_mbar_init();
  }
  pdl_wait();
  qabs = after_wait(qabs); cache = after_wait(cache); block_table = after_wait(block_table);
  g.slot = after_wait(g.slot); g.row0 = after_wait(g.row0); g.nrows = after_wait(g.nrows); g.kvlen = after_wait(g.kvlen);

  // ---- this CTA's share of the list: prefix sums of the segments' tiles (low 40 bits) and units (the rest) -----------------------------------------
  const int per_thread = (g.nseg + LA_THREADS - 1) / LA_THREADS;
  const int s_lo = min(tid * per_thread, g.nseg), s_hi = min(s_lo + per_thread, g.nseg);
  LatentWalk w;
  long long mine = 0;
  for (w.s = s_lo; w.s < s_hi; ++w.s) {
    w.load<N>(g);
    mine += (long long)w.units * w.nt + ((long long)w.units << 40);
    if (blockIdx.x == 0 && w.nrows > 0 && (long)g.kvlen[w.row0 + w.nrows - 1] > g.limit) set_status(status, ST_BOUNDS);
  }
  long long before = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += v;
  }
  if (lane == 31) ms.scan[warp] = before;
  __syncthreads();
  long long total = 0;
  before -= mine;
  for (int i = 0; i < LA_THREADS / 32; ++i) {
    if (i < warp) before += ms.scan[i];
    total += ms.scan[i];
  }
  constexpr long long TILES = (1ll << 40) - 1;
  const int all = (int)(total & TILES), share = max(1, (all + (int)gridDim.x - 1) / (int)gridDim.x);
  const int f0 = min((int)blockIdx.x * share, all), f1 = min(f0 + share, all), tiles = f1 - f0;
  if (by_unit) {
    if (blockIdx.x == 0)
      for (int i = (int)(total >> 40) + tid; i < entries; i += LA_THREADS) join[i] = make_int4(0, 0, 0, 0);
  } else if (tid == 0) {
    join[blockIdx.x] = make_int4(0, 0, 0, 0);
  }
  if (by_unit && (int)(total >> 40) > entries) {                     // segments of more rows than the caller said
    if (tid == 0) set_status(status, ST_CAPACITY);
    return;
  }
  if (tiles == 0) return;                                            // the same for the whole CTA, before any allocation
  if (smem_u32(smem) & 1023u) {                                      // the swizzled tiles need the 1024-byte base
    if (tid == 0) set_status(status, ST_BOUNDS);
    return;
  }
  if (f0 >= (before & TILES) && f0 < (before & TILES) + (mine & TILES)) {
    int at = f0 - (int)(before & TILES), unit = (int)(before >> 40);
    for (w.s = s_lo; w.s < s_hi; ++w.s) {
      w.load<N>(g);
      if (at < w.units * w.nt) break;
      at -= w.units * w.nt;
      unit += w.units;
    }
    ms.start[0] = w.s; ms.start[1] = at / w.nt; ms.start[2] = at % w.nt; ms.start[3] = unit + at / w.nt;
  }
  if (warp == 16) {
    tmem_alloc(&ms.tmem, C::TMEM);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ms.tmem;
  w.s = ms.start[0]; w.u = ms.start[1]; w.t = ms.start[2];
  w.load<N>(g);

  if (warp < 8) {
    // ---- unpack: thread = (key, half of every 64 values) ---------------------------------------------------------------------------------------
    const int row = warp * 16 + (lane >> 1), half = lane & 1;
    unsigned char* const krow = smem + C::K_AT + row * 128;
    unsigned char* const rrow = smem + C::R_AT + row * 128;
    const int turn = row & 7;
    constexpr int CB = BITS * 4, SW = Row::per_half * NC;            // bytes of 32 codes; of this half's scales
    // page of a key of the walk's tile, -1 where there is none
    auto page_of = [&](int& off) -> int {
      const int key = w.t * LA_KT + row;
      off = 0;
      if (w.s >= g.nseg || key >= w.kv) return -2;
      const int p = key / kv_block;
      off = key - p * kv_block;
      return block_table[(size_t)g.slot[w.s] * max_blocks + p];
    };
    auto place = [&](int blk, int off) -> const uint8_t* {
      if (blk >= 0 && blk < pages) return cache + ((size_t)blk * kv_block + off) * RB;
      if (blk != -2) set_status(status, ST_BOUNDS);
      return nullptr;
    };
    auto step = [&] { if (w.s < g.nseg && ++w.t == w.nt) w.next_unit<N>(g); };
    uint4 raw[C::PD][BITS / 4];
    auto fetch = [&](uint4 (&r)[BITS / 4], const uint8_t* p, int c) {
#pragma unroll
      for (int i = 0; i < BITS / 4; ++i)
        r[i] = p ? ldg_stream(p + c * 2 * CB + half * CB + i * 16) : BITS == 4 ? make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u) : make_uint4(0, 0, 0, 0);
    };
    constexpr int SCW = (SW + 3) / 4;
    auto scales = [&](uint32_t (&v)[SCW], const uint8_t* p) {
#pragma unroll
      for (int i = 0; i < SCW; ++i) v[i] = 0;
      if (!p) return;
      const uint8_t* at = p + Row::scale_at(L) + half * SW;
      if constexpr (SW >= 4) {
#pragma unroll
        for (int i = 0; i < SCW; ++i) v[i] = *reinterpret_cast<const uint32_t*>(at + 4 * i);
      } else if constexpr (SW == 2) {
        v[0] = *reinterpret_cast<const uint16_t*>(at);
      } else {
        v[0] = *at;
      }
    };
    int off;
    int blk = page_of(off);
    const uint8_t* p0 = place(blk, off);
#pragma unroll
    for (int c = 0; c < C::PD; ++c) fetch(raw[c], p0, c);
    uint32_t sc0[SCW], sc1[SCW];
    scales(sc0, p0);
    step();
    blk = page_of(off);
    const uint8_t* p1 = place(blk, off);
    int buf = 0;
    uint32_t kph = 1;                                                // (a fresh barrier passes a wait for parity 1)
    bool ok = true;
    for (int i = 0; i < tiles; ++i) {
      step();
      blk = i + 2 < tiles ? page_of(off) : -2;
      uint4 rope[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) rope[j] = p0 ? ldg_stream(p0 + Row::rope_at(L) + half * 64 + j * 16) : make_uint4(0, 0, 0, 0);
      scales(sc1, i + 1 < tiles ? p1 : nullptr);
      uint32_t nan = 0;
#pragma unroll
      for (int j = 0; j < SCW; ++j) {
        const uint32_t m = __vcmpgeu4(sc0[j], BITS == 4 ? 0xf8f8f8f8u : 0x87878787u);
        nan |= m;
        sc0[j] &= ~m;
      }
      nan = __ballot_sync(0xffffffffu, nan != 0);
      if (lane == 0) ms.bad[i & 3][warp] = nan;
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        ok = ok && mbar_wait_or_flag(&kempty[buf], kph, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int c = 2 * j + e;
          if (c < NC) {
            uint32_t b0, b1;
            if constexpr (BITS == 4) { b0 = sc0[c / 2] >> (16 * (c % 2)) & 255u; b1 = sc0[c / 2] >> (16 * (c % 2) + 8) & 255u; }
            else { b0 = sc0[c / 4] >> (8 * (c % 4)) & 255u; b1 = b0; }
            unpack32<BITS>(raw[c % C::PD], b0, b1, krow + buf * 2 * LA_CH + e * LA_CH, half * 4, turn);
            if (c + C::PD < NC) fetch(raw[c % C::PD], p0, c + C::PD);
            else if (i + 1 < tiles) fetch(raw[c % C::PD], p1, c + C::PD - NC);
          }
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&kfull[buf]);
        if (++buf == NB) { buf = 0; kph ^= 1; }
      }
      if (!ok) break;
      ok = mbar_wait_or_flag(rempty, (i & 1) ^ 1, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
#pragma unroll
      for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(rrow + (((half * 4 + j) ^ turn) << 4)) = rope[j];
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(rfull);
      p0 = p1;
      p1 = place(blk, off);
#pragma unroll
      for (int j = 0; j < SCW; ++j) sc0[j] = sc1[j];
    }
    if (!ok) { set_status(status, ST_MBAR_TIMEOUT); *abort_flag = 1; }
  } else if (warp == 16) {
    // ---- products: the whole warp, one lane of it by predicate ------------------------------------------------------------------------------------
    constexpr uint32_t id_s = umma_idesc(0, 0, 128, N), id_r = umma_idesc(1, 1, 128, N), id_o = umma_idesc(0, 0, 128, N) | 1u << 15 | 1u << 16;
    constexpr uint32_t P_ROW = N * 2, P_SW = N == 64 ? 2 : N == 32 ? 4 : 6;        // the weights' rows: swizzled over 128, 64 or 32 bytes
    const uint32_t aq = smem_u32(smem), ak = smem_u32(smem + C::K_AT), ar = smem_u32(smem + C::R_AT), ap = smem_u32(smem + C::P_AT);
    const uint32_t ts = tmem + NP * N;
    const bool issue = elect_one();
    auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_or_flag(bar, parity, abort_flag)); };
    int buf = 0, i = 0, piece = 0;
    uint32_t kph = 0;
    bool ok = true;
    while (ok && i < tiles) {
      const int n = min(w.nt - w.t, tiles - i);
      ok = wait(qfull, piece & 1);
      for (int k = 0; ok && k < n; ++k, ++i) {
        const int b0 = buf;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
          if (!ok || !wait(&kfull[buf], kph)) { ok = false; break; }
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < 8; ++kk) {
            const int c = 2 * j + kk / 4;
            if (c < NC)
              tc_mma_f16_if(issue, ts, umma_desc_k128(ak + buf * 2 * LA_CH + (kk / 4) * LA_CH + (kk & 3) * 32),
                            umma_desc_k128(aq + c * N * 128 + (kk & 3) * 32), id_s, j > 0 || kk > 0);
          }
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
#pragma unroll
        for (int j = 0; j < NP; ++j) {
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            tc_mma_f16_if(issue, tmem + j * N, umma_desc_mn(ak + b * 2 * LA_CH + kk * 2048, LA_CH, 1024, 2),
                          umma_desc_mn(ap + kk * 16 * P_ROW, 0, 8 * P_ROW, P_SW), id_o, k > 0 || kk > 0);
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
  } else {
    // ---- softmax: thread = (key, half of the pairs) ----------------------------------------------------------------------------------------------
    const int quad = warp & 3, hc = (warp - 8) >> 2, st = tid - 256, key = quad * 32 + lane;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16, ts = tmem + lanes + NP * N + hc * CW, to = tmem + lanes + hc * CW;
    auto fmx = [](float a, float b) { return fmaxf(a, b); };
    auto fad = [](float a, float b) { return a + b; };
    auto pairs_of = [&](const LatentWalk& x) { return (int)min((long)N, (long)x.nrows * g.nq - (long)x.u * N); };

    // queries of the walk's unit -> shared memory, and what belongs to each pair
    auto load_q = [&](int par) {
      const int np = pairs_of(w);
      const __nv_bfloat16* q0 = qabs + ((size_t)w.row0 * g.nq + (size_t)w.u * N) * D;
      constexpr int PER = N / 8, AT_ONCE = PER < 4 ? PER : 4, UV = (L / 8 + 31) / 32;
#pragma unroll 1
      for (int b = 0; b < PER; b += AT_ONCE) {
        uint4 v[AT_ONCE][UV], r[AT_ONCE];
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
          const int n = (b + k) * 8 + warp - 8;
          const uint4* src = reinterpret_cast<const uint4*>(q0 + (size_t)n * D);
#pragma unroll
          for (int x = 0; x < UV; ++x) v[k][x] = n < np && x * 32 + lane < L / 8 ? __ldg(src + x * 32 + lane) : make_uint4(0, 0, 0, 0);
          r[k] = n < np && lane < 8 ? __ldg(src + L / 8 + lane) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
          const int n = (b + k) * 8 + warp - 8;
          float top = 0.f;
          auto look = [&](const uint4& u) {
            const uint32_t a[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) top = fmaxf(top, fmaxf(fabsf(bf_lo(a[e])), fabsf(bf_hi(a[e]))));
          };
#pragma unroll
          for (int x = 0; x < UV; ++x) look(v[k][x]);
          look(r[k]);
          top = warp_max(top);
          int ex = (int)(__float_as_uint(top) >> 23) - 127;
          ex = top == 0.f || ex > 127 ? 10 : max(ex, -110);                         // (a value that is no number stays one)
          const float mul = __uint_as_float((uint32_t)(10 - ex + 127) << 23);
#pragma unroll
          for (int x = 0; x < UV; ++x) {
            const int at = x * 32 + lane;
            const uint32_t a[4] = {v[k][x].x, v[k][x].y, v[k][x].z, v[k][x].w};
            uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const __half2 h = __floats2half2_rn(bf_lo(a[e]) * mul, bf_hi(a[e]) * mul);
              o[e] = *reinterpret_cast<const uint32_t*>(&h);
            }
            if (at < L / 8)
              *reinterpret_cast<uint4*>(smem + (at / 8) * N * 128 + n * 128 + (((at & 7) ^ (n & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
          }
          if (lane < 8) {
            const uint32_t a[4] = {r[k].x, r[k].y, r[k].z, r[k].w};
            uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = pack_bf2(bf_lo(a[e]) * mul, bf_hi(a[e]) * mul);
            *reinterpret_cast<uint4*>(smem + NC * N * 128 + n * 128 + ((lane ^ (n & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
          }
          if (lane == 0) {
            ms.c[par][n] = scale_log2 * __uint_as_float((uint32_t)(ex - 10 + 127) << 23);
            ms.see[par][n] = n < np ? min(max(g.kvlen[w.row0 + (int)(((long)w.u * N + n) / g.nq)], 0), w.kv) : w.kv;
          }
        }
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(qfull);
    };

    int i = 0, piece = 0, unit = ms.start[3];
    int flat = f0;
    bool broke = false;
    load_q(0);
    while (i < tiles) {
      const int par = piece & 1, n = min(w.nt - w.t, tiles - i), t0 = w.t, nt = w.nt, np = pairs_of(w);
      const size_t base = (size_t)w.row0 * g.nq + (size_t)w.u * N;
      softmax_sync();                                                // what load_q wrote beside the queries
      const int least = ms.see[par][0];                              // rows of a segment see no fewer keys than those ahead of them
      uint64_t sum[CW / 2];
#pragma unroll
      for (int e = 0; e < CW / 2; ++e) sum[e] = f2_pack(0.f, 0.f);
      for (int k = 0; k < n; ++k, ++i) {
        bool ok = mbar_wait_or_flag(sfull, i & 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        float v[CW];
        {
          uint32_t s[CW];
          tc_fence_after();
          tmem_ld<CW>(ts, s);
          tmem_ld_wait();
          tc_fence_before();
#pragma unroll
          for (int e = 0; e < CW; ++e) v[e] = __uint_as_float(s[e]);
        }
        const int at = (t0 + k) * LA_KT + key;
        if (ms.bad[i & 3][key >> 4] >> (2 * (key & 15)) & 3u) {
#pragma unroll
          for (int e = 0; e < CW; ++e) v[e] = __uint_as_float(0x7fc00000u);
        }
        const bool edge = (t0 + k + 1) * LA_KT > least;
        if (k == 0) {
          float x[CW];
#pragma unroll
          for (int e = 0; e < CW; ++e) {
            x[e] = v[e] * ms.c[par][hc * CW + e];
            if (edge && at >= ms.see[par][hc * CW + e]) x[e] = -INFINITY;
          }
          const float m = columns<CW>(x, lane, fmx);
          if (lane < CW) ms.mx[quad][hc * CW + lane] = m;
          softmax_sync();
          if (st < N) {
            const float top = fmaxf(fmaxf(ms.mx[0][st], ms.mx[1][st]), fmaxf(ms.mx[2][st], ms.mx[3][st]));
            ms.nr[par][st] = top == -INFINITY ? 0.f : LA_TOP - top;
          }
          softmax_sync();
        }
        bool past = !ok;
#pragma unroll
        for (int e = 0; e < CW; e += 2) {
          const float2 c = *reinterpret_cast<const float2*>(&ms.c[par][hc * CW + e]), nr = *reinterpret_cast<const float2*>(&ms.nr[par][hc * CW + e]);
          const float2 x = f2_unpack(f2_fma(f2_pack(v[e], v[e + 1]), f2_pack(c.x, c.y), f2_pack(nr.x, nr.y)));
          v[e] = x.x; v[e + 1] = x.y;
        }
        if (edge) {
#pragma unroll
          for (int e = 0; e < CW; ++e)
            if (at >= ms.see[par][hc * CW + e]) v[e] = -INFINITY;
        }
        float top = v[0];
#pragma unroll
        for (int e = 1; e < CW; ++e) top = fmaxf(top, v[e]);
        past |= top > LA_LIMIT;
        if (softmax_any(past)) {
          if (!ok) ms.fail = 1;
          const float m = columns<CW>(v, lane, fmx);
          if (lane < CW) ms.mx[quad][hc * CW + lane] = m;
          softmax_sync();
          if (ms.fail) { broke = true; break; }
          if (st < N) {
            const float most = fmaxf(fmaxf(ms.mx[0][st], ms.mx[1][st]), fmaxf(ms.mx[2][st], ms.mx[3][st]));
            const float d = most > LA_TOP ? most - LA_TOP : 0.f;
            ms.d[st] = d;
            ms.nr[par][st] -= d;
          }
          softmax_sync();
          float f[CW];
#pragma unroll
          for (int e = 0; e < CW; ++e) {
            const float d = ms.d[hc * CW + e];
            v[e] -= d;
            f[e] = ex2(-d);
          }
#pragma unroll
          for (int e = 0; e < CW / 2; ++e) sum[e] = f2_mul(sum[e], f2_pack(f[2 * e], f[2 * e + 1]));
          if (k > 0) {                                               // (the tile's scores are complete, so the products ahead of them are)
#pragma unroll 1
            for (int j = 0; j < NP; ++j) {
              uint32_t o[CW];
              tmem_ld<CW>(to + j * N, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < CW; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f[e]);
              tmem_st<CW>(to + j * N, o);
            }
            tmem_st_wait();
            tc_fence_before();
          }
        }
        uint32_t pw[CW / 2];
#pragma unroll
        for (int e = 0; e < CW / 2; ++e) {
          const float a = ex2(v[2 * e]), b = ex2(v[2 * e + 1]);
          sum[e] = f2_add(sum[e], f2_pack(a, b));
          const __half2 h = __floats2half2_rn(a, b);
          pw[e] = *reinterpret_cast<const uint32_t*>(&h);
        }
        unsigned char* prow = smem + C::P_AT + key * N * 2;
        const int pturn = N == 64 ? key & 7 : N == 32 ? key >> 1 & 3 : key >> 2 & 1;
#pragma unroll
        for (int e = 0; e < CW / 8; ++e)
          *reinterpret_cast<uint4*>(prow + (((hc * (CW / 8) + e) ^ pturn) << 4)) = make_uint4(pw[4 * e], pw[4 * e + 1], pw[4 * e + 2], pw[4 * e + 3]);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(pfull);
      }
      if (broke) break;
      // ---- the piece's end; the next one's queries first (its scores no longer need this one's) ------------------------------------------------
      const bool whole = t0 == 0 && n == nt;
      const int my_unit = unit, first_flat = flat - t0;
      flat += n;
      if (t0 + n == nt) { w.next_unit<N>(g); ++unit; }
      if (i < tiles) load_q(par ^ 1);
      float a[CW];
#pragma unroll
      for (int e = 0; e < CW / 2; ++e) {
        const float2 x = f2_unpack(sum[e]);
        a[2 * e] = x.x; a[2 * e + 1] = x.y;
      }
      const float l = columns<CW>(a, lane, fad);
      if (lane < CW) ms.mx[quad][hc * CW + lane] = l;
      bool ok = mbar_wait_or_flag(ofull, piece & 1, abort_flag);
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
      if (st == 0) {
        if (t0 == 0 && (by_unit || !whole))
          join[by_unit ? my_unit : (int)blockIdx.x] = make_int4((int)base, whole ? 0 : np, rec, (first_flat + nt - 1) / share);
      }
      softmax_sync();
      tc_fence_after();
#pragma unroll 1
      for (int j = 0; j < NP; ++j) {
        uint32_t o[CW];
        tmem_ld<CW>(to + j * N, o);
        tmem_ld_wait();
        const int e0 = j * 128 + quad * 32 + lane;
        if (e0 < L) {
          if (whole) {
            __nv_bfloat16* dst = out + (base + hc * CW) * L + e0;
#pragma unroll
            for (int e = 0; e < CW; ++e)
              if (hc * CW + e < np) dst[(size_t)e * L] = f2bf(__uint_as_float(o[e]) * ms.d[hc * CW + e]);
          } else {
            float* dst = o_part + ((size_t)rec * N + hc * CW) * L + e0;
#pragma unroll
            for (int e = 0; e < CW; ++e)
              if (hc * CW + e < np) dst[(size_t)e * L] = __uint_as_float(o[e]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(oempty);
      ++piece;
    }
    if (broke && st == 0) { set_status(status, ST_MBAR_TIMEOUT); *abort_flag = 1; }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 16) tmem_dealloc(tmem, C::TMEM);
}

// Units that span CTAs. grid (entries, N), 128 threads: a CTA a pair, its records in the order of their keys.
__global__ void __launch_bounds__(128) mla_attn_q_join_kernel(__nv_bfloat16* __restrict__ out, const float* o_part, const float* ml_part, const int4* join,
                                                              int N, int L, const int* row_kvlen, int nq) {
  extern __shared__ float wt[];                                      // [records]
  __shared__ float red[32];
  const int n = blockIdx.y, tid = threadIdx.x;
  pdl_launch_dependents();
  pdl_wait();
  o_part = after_wait(o_part); ml_part = after_wait(ml_part); row_kvlen = after_wait(row_kvlen);
  const int4 job = after_wait(join)[blockIdx.x];
  if (n >= job.y) return;
  const int c0 = job.z >> 1, count = job.w - c0 + 1;
  auto record = [&](int i) { return (size_t)(i == 0 ? job.z : 2 * (c0 + i)) * N + n; };
  float m = -INFINITY;
  for (int i = tid; i < count; i += 128) {
    wt[i] = ml_part[record(i) * 2];
    m = fmaxf(m, wt[i]);
  }
  m = block_max(m, red);
  float l = 0.f;
  for (int i = tid; i < count; i += 128) {
    // a record without weight has -inf there; a reference of +inf comes with sums that are no numbers
    const float x = wt[i] == -INFINITY ? 0.f : wt[i] == m ? 1.f : exp2f(wt[i] - m);
    wt[i] = x;
    l += x == 0.f ? 0.f : x * ml_part[record(i) * 2 + 1];
  }
  l = block_sum(l, red);                                             // (its barriers publish wt)
  const size_t pair = (size_t)job.x + n;
  const float inv = row_kvlen[pair / nq] > 0 ? 1.f / l * (l == 0.f ? 0.f : 1.f) : 0.f;
  for (int e = tid * 4; e < L; e += 512) {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int i = 0; i < count; ++i) {
      const float x = wt[i];
      const float4 v = *reinterpret_cast<const float4*>(o_part + record(i) * L + e);
      if (x != 0.f) { a.x = fmaf(x, v.x, a.x); a.y = fmaf(x, v.y, a.y); a.z = fmaf(x, v.z, a.z); a.w = fmaf(x, v.w, a.w); }
    }
    *reinterpret_cast<uint2*>(out + pair * L + e) = make_uint2(pack_bf2(a.x * inv, a.y * inv), pack_bf2(a.z * inv, a.w * inv));
  }
}

}  // namespace fb

using namespace fb;

// Pairs of a unit: the fewest of 16, 32 and 64 that hold a segment's; more are several units (an unpacked tile serves as many as it can).
static int latent_pairs(long pairs) { return pairs <= 16 ? 16 : pairs <= 32 ? 32 : 64; }

extern "C" long fb_mla_attn_q_floats(int max_rows, int nq, int L, int ctas) {
  const long N = latent_pairs((long)max_rows * nq);
  return 4l * ctas + 2l * ctas * N * (L + 2);
}

// ws: fb_mla_attn_q_floats of 32 bits; row_kvlen does not fall along a segment
extern "C" int fb_mla_attn_q(void* out, float* ws, long ws_floats, const void* qabs, const void* cache, long pages, int bits, const int* seg_slot,
                             const int* seg_row0, const int* seg_nrows, int nseg, int max_rows, const int* row_kvlen, const int* block_table,
                             int max_blocks, int kv_block, int rows, int nq, int L, int R, float scale, int ctas, int* status, cudaStream_t s) {
  if (R != LC_R || (bits != 4 && bits != 8) || nq < 1 || kv_block < 1 || ctas < 1 || max_rows < 0) return -1;
  if (((uintptr_t)qabs | (uintptr_t)cache | (uintptr_t)ws) % 16 || (uintptr_t)out % 8) return -2;
  if (rows <= 0 || nseg <= 0 || max_rows == 0) return 0;
  if (ws_floats < fb_mla_attn_q_floats(max_rows, nq, L, ctas)) return -3;
  const int N = latent_pairs((long)max_rows * nq);
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
  return (int)launch_pdl(mla_attn_q_join_kernel, dim3(entries, N), dim3(128), (size_t)ctas * 4, s, (__nv_bfloat16*)out, (const float*)op,
                         (const float*)ml, (const int4*)join, N, L, row_kvlen, nq);
}

// Attention of many query rows over the pages of a paged cache, on the tensor
// cores (tcgen05):
//   prefill  several new tokens of each request attend its pages, causally
//   prefix   one token of each request of a group attends the pages of the
//            prefix that the group shares (a partial result: the requests' own
//            tokens are added by the windowed decode kernel's PREFIX form)
//
// The query rows of one kv head are packed: row = token * G + (head in its
// group), G = Hq / Hkv, so a tile of 128 rows holds floor(128 / G) tokens and
// every K and V tile is read once for all query heads that share it.  In the
// prefix form the tokens are the requests of a group: that is the whole gain,
// 128 rows for each byte of the prefix instead of G.
//
// One CTA owns NQT tiles of 128 rows of one (segment, kv head), a segment being
// a request or a group, and walks key tiles of 128 tokens (64 at D = 64) of one
// share of the context:
//   warp LOAD  TMA producer: Q once (one box of G x floor(128 / G) rows for
//              each 64 columns), then K_j and V_j into a ring of slots, in boxes
//              of `box` rows, the largest power of two that divides the page
//              size (a box never leaves its page); a lane each looks its box's
//              page up one tile ahead
//   warp MMA   S_t = Q_t K_j^T into TMEM, O_t += P_t V_j with P_t from TMEM; the
//              whole warp in step, one lane issuing (mma_ss_warp)
//   4 warps for each query tile: thread = row = TMEM lane.  Two passes over S
//              in TMEM (maximum, then 2^(s - m) written back as 16-bit P), so
//              that a row never lives in registers whole.
// Rows and warps past the segment's last token do nothing and store nothing.
// Keys past the last visible one: scores are masked by selection, and the rows
// of V are zeroed in shared memory before the product, because 0 * NaN of
// memory that was never written would reach O.
//
// Shares of a long context (few rows: one tile for each kv head would leave most
// SMs idle) leave fp32 partial results, normalised, with their base-2 LSE; a
// merge kernel (prefill) or the decode kernel (prefix) joins them.
// P is rounded to the data's type once, as the tensor core's operand; the row
// sums add the unrounded values; statistics, O and the join are fp32.
//
// What bounds it, by the rows that share K and V:
//   many (2048 tokens behind 30 720, 32/8 heads of 128: 938-968 us from run to run,
//     1100-1135 TFLOP/s, 0.66-0.68 of a measured GEMM): the chain S - softmax - P V
//     of the two query tiles, about 3500 cycles for a key tile of both against 2048
//     of products and 1664 of exponentials.  On that case, us: issued by a single
//     thread's code 1061, by the warp 959; two threads a row 1096; S in two
//     buffers of 64 keys 1031; an issuing warp for each tile 1234; scores kept in
//     registers 1396 against 1313; the tiles taking turns at the exponentials no
//     faster.
//   few (64 requests of 4 tokens at 512 to 16 388: 357-373 us, 6.0-6.2 TB/s, 0.91-0.94 of a
//     measured copy): memory.
//   D = 64 (nine ragged prompts, 20 heads: 152-190 us by their order): latencies and
//     the exponentials, 416 (512 before 3 of 16 left the special-function unit) of
//     the 850 cycles that a step of 64 keys takes an SM.
#include "ffa_common.cuh"
#include "ffa_host.h"
#include "ffa_page_attn.h"

#include <type_traits>

namespace ffa {

constexpr int PA_BM = 128, PA_BN = 128;  // rows of a query tile; the unit of a context's shares

struct PaParams {
  const int* starts;  // [N + 1] first query token of each segment
  const int* kv_lens; // causal: [N] context lengths; else [N] prefix lengths
  const int* lens;    // [R] context lengths (prefix form: which members share)
  const int* table;   // [R, width]
  int64_t bt_stride;
  void* out;          // [T, Hq, D] (causal)
  int64_t o_st, o_sh;
  float* lse;         // [T, Hq] or nullptr (causal)
  float* o_part;      // [shares, T, Hq, D]
  float* lse_part;    // [shares, T, Hq], base 2
  int N, T, Hq, Hkv, G, TQ, D;
  int num_pages, page_size, box, max_ctx;
  int shares, chunk;  // a segment's tokens [s * chunk, (s + 1) * chunk), the last share the rest
  float scale_log2, sc_pre, sc_unit, sc_poly[3];  // scale log2 e; scale / softcap, and its inverse
  int use_softcap, keep_kv;  // keep_kv: other CTAs read the same K and V
  ErrCtx ec;
};

template <int D, int NQT, bool FEW>
struct PaCfg {
  // D = 128, NQT = 1: 6 warps, two CTAs per SM (each half the TMEM; the two
  // interleave on the tensor core).  NQT = 2: 10 warps, one CTA, K and V read once
  // for both tiles.  At most 168 registers a thread either way.
  // FEW (D = 128, at most 32 rows, NQT = 1): Q takes 8 KB, which leaves room for a
  // third slot of the ring: bound by memory, whose latency two slots do not cover.
  // (The products read 128 rows there all the same, whatever lies behind Q's.)
  // D = 64, where the exponentials outweigh the products: key tiles of 64, a quarter
  // of the TMEM, four CTAs per SM, so that some softmax always has its scores.
  static constexpr int BN = D == 64 ? 64 : 128;  // keys of a tile
  static constexpr int THREADS = (4 * NQT + 2) * 32;
  static constexpr int MIN_BLOCKS = NQT == 2 ? 1 : D == 64 ? 4 : 2;
  static constexpr int TMEM_COLS = 512 / MIN_BLOCKS;
  static constexpr int O_COL = NQT * BN;      // TMEM: S_t / P_t at [128 t, ...), O_t at O_COL + 128 t
  static constexpr int Q_ROWS = FEW ? 32 : PA_BM;
  static constexpr int TILE = Q_ROWS * D * 2;  // a tile of Q
  static constexpr int KV_TILE = BN * D * 2;  // a tile of K or V
  static constexpr int NBUF = FEW ? 3 : NQT == 1 && D == 128 ? 2 : 4;
  static constexpr int KV_OFF = NQT * TILE;
  static constexpr int BAR_OFF = KV_OFF + NBUF * KV_TILE;
  static constexpr int SMEM = BAR_OFF + 512 + 1024;
  static_assert(MIN_BLOCKS * (SMEM + 1024) <= 228 * 1024, "shared memory budget");
};

struct PaBars {
  uint64_t q_full;
  uint64_t s_full[2];
  uint64_t p_full[2][2];
  uint64_t o_done[2];
  uint64_t drain;
  uint64_t kv_full[4];
  uint64_t kv_empty[4];
  uint32_t tmem_base;
  int abort;
};

enum : uint32_t {
  SITE_PA_Q = 0x501,
  SITE_PA_KV_EMPTY = 0x502,
  SITE_PA_KV_FULL = 0x503,
  SITE_PA_P_FULL = 0x504,
  SITE_PA_S_FULL = 0x505,
  SITE_PA_O_DONE = 0x506,
  SITE_PA_DRAIN = 0x507,
};

// The item-th block of `per` query tokens over all segments, found by one warp:
// its segment, the segment's first token, tokens and keys, and the block within
// it.  CTAs that run long start early: of a segment the block with the most keys
// comes first and, where contexts are not cut into shares of one length, so do of
// every 32 segments those with the most keys (nine ragged prompts 161 -> 151 us).
// Of more segments than a warp's lanes the last blocks come first, segment by
// segment, so that of many with one block each none is searched for.
__device__ __forceinline__ bool pa_find(const PaParams& p, int per, int item, int lane, int& seg, int& first, int& n,
                                        int& kv, int& block) {
  const bool many = p.N > 32;
  auto bad = [&](int lo, int hi) -> bool {
    if (lo >= 0 && hi >= lo && hi <= p.T) return false;
    if (p.ec.err) atomicCAS(p.ec.err, 0u, SITE_PA_BAD_STARTS);
    return true;
  };
  if (many && item < p.N) {
    seg = item;
    first = p.starts[seg];
    const int end = p.starts[seg + 1];
    kv = p.kv_lens[seg];
    if (bad(first, end)) return false;
    n = end - first;
    block = (n + per - 1) / per - 1;
    return n > 0;
  }
  if (many) item -= p.N;
  int base = 0;
  for (int i0 = 0; i0 < p.N; i0 += 32) {
    const int i = i0 + lane;
    int lo = 0, hi = 0, keys = 0;
    if (i < p.N) {
      lo = p.starts[i];
      hi = p.starts[i + 1];
      keys = p.kv_lens[i];
      if (bad(lo, hi)) lo = hi = 0;
    }
    const int blocks = max((hi - lo + per - 1) / per - (many ? 1 : 0), 0);
    int before = base, all = 0;  // blocks of the segments that come before this lane's; of the 32
    if (p.shares == 1) {
      for (int k = 0; k < min(32, p.N - i0); ++k) {
        const int kk = __shfl_sync(0xffffffffu, keys, k), kb = __shfl_sync(0xffffffffu, blocks, k);
        if (kk > keys || (kk == keys && k < lane)) before += kb;
        all += kb;
      }
    } else {
      all = blocks;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, all, off);
        if (lane >= off) all += a;
      }
      before += all - blocks;
      all = __shfl_sync(0xffffffffu, all, 31);
    }
    const uint32_t mine = __ballot_sync(0xffffffffu, before <= item && item - before < blocks);
    if (mine) {
      const int o = __ffs(mine) - 1;
      seg = i0 + o;
      first = __shfl_sync(0xffffffffu, lo, o);
      n = __shfl_sync(0xffffffffu, hi - lo, o);
      kv = __shfl_sync(0xffffffffu, keys, o);
      block = __shfl_sync(0xffffffffu, before + blocks, o) - 1 - item;
      return true;
    }
    base += all;
  }
  return false;
}

// Maxima that are NaN where a score is, at the price of the others.
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^x for two lanes on the FMA and integer pipes: x = n + f with n whole and f in
// [-1/2, 1/2] (adding 1.5 2^23 rounds, and leaves n in the low bits), 2^f by a
// quartic fitted to it (least squares on Chebyshev nodes, reweighted towards
// minimax: relative error 2.7e-6 in fp32), n added to the exponent.  NaN becomes
// some number: a row whose scores have one is NaN by its maximum.
__device__ __forceinline__ float2 exp2_fma2(float2 x) {
  const float2 t = fadd2(x, f2(12582912.f));
  const float2 f = ffma2(fadd2(t, f2(-12582912.f)), f2(-1.f), x);
  float2 p = ffma2(f2(0.009570098975f), f, f2(0.05591786009f));
  p = ffma2(p, f, f2(0.240247449f));
  p = ffma2(p, f, f2(0.6931218148f));
  p = ffma2(p, f, f2(0.9999992614f));
  // (below 2^-125, -inf among them, exactly 0: a masked key must not count)
  return make_float2(x.x < -125.f ? 0.f : __int_as_float(__float_as_int(p.x) + (__float_as_int(t.x) << 23)),
                     x.y < -125.f ? 0.f : __int_as_float(__float_as_int(p.y) + (__float_as_int(t.y) << 23)));
}

template <typename T, int D, int NQT, bool FEW, bool CAUSAL>
__global__ void __launch_bounds__(PaCfg<D, NQT, FEW>::THREADS, PaCfg<D, NQT, FEW>::MIN_BLOCKS)
    ffa_page_attn_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                         const __grid_constant__ CUtensorMap tmV, const PaParams p) {
  using Cfg = PaCfg<D, NQT, FEW>;
  constexpr int WARP_MMA = 0, WARP_LOAD = 1;  // then four softmax warps for each query tile
  constexpr int O_COL = Cfg::O_COL, BN = Cfg::BN;
  constexpr int HALVES = D / 64, HALF = 128 * 128, Q_HALF = Cfg::Q_ROWS * 128;  // 64-column halves of a tile
  static_assert(HALVES == 1 || BN == 128, "a half's bytes");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sKV = smem + Cfg::KV_OFF;
  PaBars* bars = reinterpret_cast<PaBars*>(smem + Cfg::BAR_OFF);
  volatile int* abort_flag = &bars->abort;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  // a kernel launched behind this one may start once every CTA has come here
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }

  // ---------------- what this CTA works on (the same in every warp) ----------------
  const int h = blockIdx.x % p.Hkv;
  const int share = blockIdx.x / p.Hkv % p.shares;
  const int item = blockIdx.x / p.Hkv / p.shares;
  const int per = p.TQ * NQT;
  int seg, first, n, kv, block;
  if (!pa_find(p, per, item, lane, seg, first, n, kv, block)) return;
  const int tok0 = block * per;              // of the segment's query tokens
  const int toks = min(per, n - tok0);       // this CTA's
  const int tiles_q = NQT == 1 || toks <= p.TQ ? 1 : 2;
  int row, past;  // table row; tokens before the segment's first query (causal)
  bool direct = false;
  int limit;      // keys [0, limit) are visible to some row of this CTA
  if (CAUSAL) {
    if (kv < n || kv > p.max_ctx) {
      if (lane == 0 && p.ec.err) atomicCAS(p.ec.err, 0u, SITE_DEC_BAD_CTX);
      return;
    }
    row = seg;
    past = kv - n;
    limit = past + tok0 + toks;
    direct = p.shares == 1 || kv <= p.chunk;
  } else {
    if (kv < 0 || kv > p.max_ctx) {
      if (lane == 0 && p.ec.err) atomicCAS(p.ec.err, 0u, SITE_PA_BAD_STARTS);
      return;
    }
    // the first member long enough lends its pages
    row = -1;
    past = 0;
    for (int i0 = 0; i0 < n && row < 0; i0 += 32) {
      const int len = i0 + lane < n ? p.lens[first + i0 + lane] : -1;
      const uint32_t has = __ballot_sync(0xffffffffu, len >= kv && len <= p.max_ctx);
      if (has) row = first + i0 + __ffs(has) - 1;
    }
    if (row < 0) return;
    limit = kv;
  }
  const int kv0 = share * p.chunk;
  const int kv1 = share + 1 == p.shares ? limit : min(limit, kv0 + p.chunk);
  if (kv0 >= kv1) return;
  const int n_tiles = (kv1 - kv0 + BN - 1) / BN;

  if (threadIdx.x == 0) {
    mbar_init(&bars->q_full, 1);
    for (int t = 0; t < NQT; ++t) {
      mbar_init(&bars->s_full[t], 1);
      for (int k = 0; k < 2; ++k) mbar_init(&bars->p_full[t][k], 4);  // one arrival per warp
      mbar_init(&bars->o_done[t], 1);
    }
    mbar_init(&bars->drain, 1);
    for (int i = 0; i < Cfg::NBUF; ++i) {
      mbar_init(&bars->kv_full[i], 1);
      mbar_init(&bars->kv_empty[i], 1);
    }
    bars->abort = 0;
    fence_mbar_init();
  }
  if (warp == WARP_MMA) {
    tmem_alloc(&bars->tmem_base, Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;

  int issued = 0;  // (producer) slots armed so far
  if (warp == WARP_LOAD) {
    // ------------------------------- producer -------------------------------
    const uint64_t pol = p.keep_kv ? policy_evict_last() : policy_evict_first();
    if (lane == 0) {
      const int q_rows = p.TQ * p.G;
      mbar_arrive_expect_tx(&bars->q_full, tiles_q * HALVES * q_rows * 128);
      for (int t = 0; t < tiles_q; ++t)
        for (int c = 0; c < HALVES; ++c)
          tma_load_4d(&tmQ, &bars->q_full, sQ + t * Cfg::TILE + c * Q_HALF, c * 64, 0, first + tok0 + t * p.TQ, h, pol);
    }
    __syncwarp();
    const int* table = p.table + (int64_t)row * p.bt_stride;
    // pool row of this lane's box of a tile, or -1 (past the last key, or a page
    // id outside the pool, which is recorded)
    auto box_row = [&](int j) -> int {
      const int tok = kv0 + j * BN + lane * p.box;
      if (lane * p.box >= BN || tok >= kv1) return -1;
      const int i = tok / p.page_size;
      const int page = table[i];
      if ((unsigned)page >= (unsigned)p.num_pages) {
        if (p.ec.err) atomicCAS(p.ec.err, 0u, SITE_DEC_BAD_PAGE);
        return -1;
      }
      return (page * p.Hkv + h) * p.page_size + tok - i * p.page_size;
    };
    int at = box_row(0);
    bool ok = true;
    for (int j = 0; j < n_tiles && ok; ++j) {
      const int next = j + 1 < n_tiles ? box_row(j + 1) : -1;
      const uint32_t boxes = __popc(__ballot_sync(0xffffffffu, at >= 0));
      for (int v = 0; v < 2 && ok; ++v) {
        const int s = 2 * j + v, buf = s % Cfg::NBUF, use = s / Cfg::NBUF;
        if (use > 0) ok = mbar_wait(&bars->kv_empty[buf], (use - 1) & 1, p.ec, abort_flag, SITE_PA_KV_EMPTY);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&bars->kv_full[buf], boxes * p.box * 128 * HALVES);
        ++issued;
        __syncwarp();
        if (at >= 0) {
          uint8_t* dst = sKV + buf * Cfg::KV_TILE + lane * p.box * 128;
#pragma unroll
          for (int c = 0; c < HALVES; ++c)
            tma_load_4d(v ? &tmV : &tmK, &bars->kv_full[buf], dst + c * HALF, c * 64, at, 0, 0, pol);
        }
      }
      at = next;
    }
  } else if (warp == WARP_MMA) {
    // ------------------------------ MMA issuer ------------------------------
    {
      // (the lanes agree on a wait's outcome: each product needs all of them)
      auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t site) -> bool {
        return __all_sync(0xffffffffu, mbar_wait_mma(bar, parity, p.ec, abort_flag, site));
      };
      constexpr uint32_t FMT = DtypeFmt<T>::value;
      const uint32_t idesc_qk = make_idesc_f16(PA_BM, BN, FMT, 0, 0);
      const uint32_t idesc_pv = make_idesc_f16(PA_BM, D, FMT, 0, 1);
      const uint64_t q_base = make_sdesc_sw128(smem_u32(sQ), 16, 1024);
      const uint64_t k_base = make_sdesc_sw128(smem_u32(sKV), 16, 1024);
      const uint64_t v_base = make_sdesc_sw128(smem_u32(sKV), HALF, 1024);
      // every operand but the ring slot is a constant of the unrolled code
      auto issue_qk = [&](auto tile, uint64_t kb) {
        constexpr int t = decltype(tile)::value;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const int qo = t * Cfg::TILE + (ks / 4) * Q_HALF + (ks % 4) * 32, ko = (ks / 4) * HALF + (ks % 4) * 32;
          mma_ss_warp(tmem + t * 128, q_base + (uint64_t)(qo >> 4), kb + (uint64_t)(ko >> 4), idesc_qk, ks > 0);
        }
        mma_commit_warp(&bars->s_full[t]);
      };
      auto issue_pv = [&](auto tile, uint64_t vb, bool acc, auto hf) {
        constexpr int t = decltype(tile)::value, half = decltype(hf)::value;
#pragma unroll
        for (int kk = 0; kk < BN / 32; ++kk) {
          const int ks = half * (BN / 32) + kk;
          mma_ts_warp(tmem + O_COL + t * 128, tmem + t * 128 + ks * 8, vb + (uint64_t)((ks * 16 * 128) >> 4), idesc_pv,
                      (acc || ks > 0) ? 1u : 0u);
        }
      };
      auto tiles = [&](auto f) {  // f(tile) for the query tiles in use
        f(std::integral_constant<int, 0>{});
        if constexpr (NQT == 2) {
          if (tiles_q == 2) f(std::integral_constant<int, 1>{});
        }
      };
      using H0 = std::integral_constant<int, 0>;
      using H1 = std::integral_constant<int, 1>;
      // A limit of 1 ns ends one wait of a CTA at once, so that giving up can be tested:
      // this one, with copies in flight, or that for the last O, with products in flight.
      // (In the loops' waits it costs up to 4 %: a chunk 968 -> 1004 us.)
      const bool early = 2 * n_tiles <= Cfg::NBUF || blockIdx.x % 2;
      bool ok = !early || __all_sync(0xffffffffu, mbar_wait<true>(&bars->q_full, 0, p.ec, abort_flag, SITE_PA_Q));
      ok = ok && wait(&bars->q_full, 0, SITE_PA_Q) && wait(&bars->kv_full[0], 0, SITE_PA_KV_FULL);
      if (ok) {
        tc_fence_after();
        tiles([&](auto t) { issue_qk(t, k_base); });
        mma_commit_warp(&bars->kv_empty[0]);
      }
      for (int j = 0; j < n_tiles && ok; ++j) {
        const int vs = 2 * j + 1, ks = 2 * j + 2, vi = vs % Cfg::NBUF, ki = ks % Cfg::NBUF;
        const uint64_t vb = v_base + (uint64_t)((vi * Cfg::KV_TILE) >> 4), kb = k_base + (uint64_t)((ki * Cfg::KV_TILE) >> 4);
        ok = wait(&bars->kv_full[vi], (vs / Cfg::NBUF) & 1, SITE_PA_KV_FULL);
        tiles([&](auto t) {
          constexpr int n = decltype(t)::value;  // (the query tile)
          ok = ok && wait(&bars->p_full[n][0], j & 1, SITE_PA_P_FULL);
          if (!ok) return;
          tc_fence_after();
          issue_pv(t, vb, j > 0, H0{});
          ok = wait(&bars->p_full[n][1], j & 1, SITE_PA_P_FULL);
          if (!ok) return;
          tc_fence_after();
          issue_pv(t, vb, j > 0, H1{});
          mma_commit_warp(&bars->o_done[n]);
          if (n == tiles_q - 1) mma_commit_warp(&bars->kv_empty[vi]);
          if (j + 1 == n_tiles) return;
          if (n == 0) ok = wait(&bars->kv_full[ki], (ks / Cfg::NBUF) & 1, SITE_PA_KV_FULL);
          if (!ok) return;
          tc_fence_after();
          issue_qk(t, kb);
          if (n == tiles_q - 1) mma_commit_warp(&bars->kv_empty[ki]);
        });
      }
      // every MMA must retire before TMEM is released
      mma_commit_warp(&bars->drain);
      mbar_wait_mma(&bars->drain, 0, p.ec, abort_flag, SITE_PA_DRAIN, true);
    }
    __syncwarp();
  } else if ((warp - 2) / 4 < tiles_q) {
    // -------------------------------- softmax --------------------------------
    const int t = (warp - 2) / 4, r = warp % 4 * 32 + lane;  // (TMEM lanes go by the warp's number)
    const uint32_t lane_off = (uint32_t)((warp % 4) * 32) << 16;
    const uint32_t tS = tmem + lane_off + t * 128;
    const uint32_t tO = tmem + lane_off + O_COL + t * 128;
    const int t_toks = min(p.TQ, toks - t * p.TQ);   // tokens of this tile
    const bool live = (warp % 4) * 32 < t_toks * p.G;  // any row of this warp
    const int tl = r / p.G, g = r - tl * p.G;        // this row's token in the tile, and head
    // Rows that are not stored (another segment's, or whatever shared memory held) have
    // no vote on what their warp does, so that a result does not depend on them.
    const bool votes = tl < t_toks;
    // keys [0, vis) are visible to this row (a row past the segment's last token is computed like the last)
    const int vis = CAUSAL ? past + tok0 + t * p.TQ + min(tl, t_toks - 1) + 1 : limit;
    const int vis_min = CAUSAL ? past + tok0 + t * p.TQ + 1 : limit;
    constexpr bool AHEAD = D > 64;  // 32 columns are on their way while 32 are worked on
    uint32_t sc[AHEAD ? 64 : 32];   // (D = 64: other CTAs fill the wait, and registers are few)
    // First pass where scores change: softcapped, -inf from column `hi` on, written
    // back to TMEM; returns their maximum.  A softcap becomes y with tanh(k s) = k y,
    // k = scale / softcap, so that scores keep one factor: by the polynomial where
    // every argument of the warp's 32 columns is within 1/2.
    auto rewrite = [&](int hi) -> float {
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
      for (int c = 0; c < BN; c += 32) {
        uint32_t s[32];
        tmem_ld32(tS + c, s);
        tmem_ld_wait32(s);
        if (p.use_softcap) {
          float lo[4] = {0.f, 0.f, 0.f, 0.f};
          if (c + 32 <= hi) {
#pragma unroll
            for (int e = 0; e < 32; e += 8)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                lo[i] = fmax3(lo[i], fabsf(__uint_as_float(s[e + i])), fabsf(__uint_as_float(s[e + i + 4])));
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) lo[e % 4] = c + e < hi ? fmaxf(lo[e % 4], fabsf(__uint_as_float(s[e]))) : lo[e % 4];
          }
          if (__all_sync(0xffffffffu,
                         !votes || fmaxf(fmaxf(lo[0], lo[1]), fmaxf(lo[2], lo[3])) * p.sc_pre <= 0.5f)) {
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const float2 y = softcap_small2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])),
                                              p.sc_poly[0], p.sc_poly[1], p.sc_poly[2]);
              s[e] = __float_as_uint(y.x);
              s[e + 1] = __float_as_uint(y.y);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              s[e] = __float_as_uint(tanh_acc(__uint_as_float(s[e]) * p.sc_pre) * p.sc_unit);
          }
        }
        if (!__all_sync(0xffffffffu, c + 32 <= hi)) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (c + e >= hi) s[e] = __float_as_uint(-INFINITY);
        }
        tmem_st32(tS + c, s);
#pragma unroll
        for (int e = 0; e < 32; e += 8)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx[i] = max3_nan(mx[i], __uint_as_float(s[e + i]), __uint_as_float(s[e + i + 4]));
      }
      tmem_st_wait();
      return max_nan(max_nan(mx[0], mx[1]), max_nan(mx[2], mx[3]));
    };
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < n_tiles; ++j) {
      const int c0 = kv0 + j * BN;
      ok = __all_sync(0xffffffffu, mbar_wait(&bars->s_full[t], j & 1, p.ec, abort_flag, SITE_PA_S_FULL));
      if (!ok) break;
      tc_fence_after();
      if (t == 0 && c0 + BN > limit) {
        // The last tile ends past the visible keys: V's rows there become zeros.
        // (Only now: S_j is issued after V_(j-1) was waited for, so the barrier
        // is in this tile's phase; before that its parity would not tell.)
        const int s = 2 * j + 1;
        ok = __all_sync(0xffffffffu, mbar_wait(&bars->kv_full[s % Cfg::NBUF], (s / Cfg::NBUF) & 1, p.ec, abort_flag,
                                               SITE_PA_KV_FULL));
        if (!ok) break;
        uint8_t* vt = sKV + s % Cfg::NBUF * Cfg::KV_TILE;
        const int drop = (limit - c0) * 8, all = BN * 8;  // 16-byte pieces of a half
        for (int i = drop + r; i < all; i += PA_BM)
#pragma unroll
          for (int c = 0; c < HALVES; ++c) *reinterpret_cast<uint4*>(vt + c * HALF + i * 16) = make_uint4(0, 0, 0, 0);
        fence_async_smem();
        __syncwarp();
      }
      if (!live) {  // P of rows that nobody reads: whatever TMEM holds
        if (lane == 0) {
          mbar_arrive(&bars->p_full[t][0]);
          mbar_arrive(&bars->p_full[t][1]);
        }
        continue;
      }
      // First pass: the row's maximum, in base-2 units (scale is positive).  Softcaps
      // and masks are written back to TMEM in a pass of its own, so that the second
      // pass knows neither.
      float top;
      if (p.use_softcap || c0 + BN > vis_min) {
        top = rewrite(vis - c0);
        if (AHEAD) tmem_ld32(tS, sc);
      } else {
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (AHEAD) tmem_ld32(tS, sc);
#pragma unroll
        for (int c = 0; c < BN; c += 32) {
          uint32_t* s = sc + (AHEAD ? c % 64 : 0);
          if (!AHEAD) tmem_ld32(tS + c, s);
          tmem_ld_wait32(s);
          if (AHEAD) tmem_ld32(tS + (c + 32) % BN, sc + (c + 32) % 64);  // (the last one: the second pass's first)
#pragma unroll
          for (int e = 0; e < 32; e += 8)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              mx[i] = max3_nan(mx[i], __uint_as_float(s[e + i]), __uint_as_float(s[e + i + 4]));
        }
        top = max_nan(max_nan(mx[0], mx[1]), max_nan(mx[2], mx[3]));
      }
      top *= p.scale_log2;
      // A row that sees a NaN, or a score of +inf (inf - inf), is NaN from here on: its
      // maximum, so its sum, O and LSE, whatever exp2_fma2 makes of one score.
      float m_new = max_nan(m, top);
      if (__any_sync(0xffffffffu, votes && !(m_new <= m + 8.f))) {
        // lazy rescale: exact, numerator and denominator share the stale maximum
        if (m_new == INFINITY) m_new = NAN;
        const float alpha = m_new == -INFINITY ? 1.f : ex2(m - m_new);
        l *= alpha;
        m = m_new;
        if (j > 0) {
          ok = __all_sync(0xffffffffu,
                          mbar_wait(&bars->o_done[t], (j - 1) & 1, p.ec, abort_flag, SITE_PA_O_DONE));
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < D; c += 32) {
            uint32_t ov[32];
            tmem_ld32(tO + c, ov);
            tmem_ld_wait32(ov);
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              const float2 v = fmul2(make_float2(__uint_as_float(ov[e]), __uint_as_float(ov[e + 1])), f2(alpha));
              ov[e] = __float_as_uint(v.x);
              ov[e + 1] = __float_as_uint(v.y);
            }
            tmem_st32(tO + c, ov);
          }
        }
      }
      // second pass: P over S, handed over in two halves of the tile
      const float mu = m == -INFINITY ? 0.f : m;
      const float2 mul2 = f2(p.scale_log2), nmu2 = f2(-mu);
      float2 acc[2] = {f2(0.f), f2(0.f)};
#pragma unroll
      for (int c = 0; c < BN; c += 32) {
        uint32_t pk[16];
        uint32_t* s = sc + (AHEAD ? c % 64 : 0);
        if (!AHEAD) tmem_ld32(tS + c, s);
        tmem_ld_wait32(s);
        if (AHEAD && c + 32 < BN) tmem_ld32(tS + c + 32, sc + (c + 32) % 64);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float2 a = ffma2(make_float2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), mul2, nmu2);
          // three pairs of sixteen leave the special-function unit (D 128: 256 requests
          // behind 32 768 tokens 193 -> 184 us, two pairs 188; D 64: 2048 tokens behind
          // 30 720 876 -> 818, two pairs 834, four 834, five 855)
          const float2 pv = e % 5 == 3 ? exp2_fma2(a) : make_float2(ex2(a.x), ex2(a.y));
          acc[e & 1] = fadd2(acc[e & 1], pv);
          pk[e] = pack2<T>(pv.x, pv.y);
        }
        tmem_st16(tS + c / 2, pk);
        if ((c + 32) % (BN / 2) == 0) {
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->p_full[t][c / (BN / 2)]);
        }
      }
      const float2 a = fadd2(acc[0], acc[1]);
      l += a.x + a.y;
    }
    // (a wait gave up: a read of S ahead of its use may be on its way, and TMEM is given back below)
    if (AHEAD && !ok) tmem_ld_wait();
    // -------------------------------- epilogue --------------------------------
    if (ok && live) {
      ok = __all_sync(0xffffffffu,
                      mbar_wait<true>(&bars->o_done[t], (n_tiles - 1) & 1, p.ec, abort_flag, SITE_PA_O_DONE));
      if (ok) {
        tc_fence_after();
        // (a sum of NaN is no empty row: O and LSE say NaN, and so do the joins')
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int64_t tok = first + tok0 + t * p.TQ + tl;
        const int head = h * p.G + g;
        const int64_t part = ((int64_t)share * p.T + tok) * p.Hq + head;
        if (votes) {
          const float lse = l == 0.f ? -INFINITY : m + lg2(l);
          if (!(CAUSAL && direct)) p.lse_part[part] = lse;
          else if (p.lse) p.lse[tok * p.Hq + head] = lse * 0.6931471805599453f;
        }
        // O leaves through the query tile's place in shared memory (its S are all
        // done), so that a warp's store covers whole rows of the output: a thread's
        // own row at a time took 8200 cycles for fp32 partial results, 2200 for
        // 16-bit ones.  A row of W 16-byte pieces, piece k of row r at k ^ (r % W):
        // no bank conflicts either way.  fp32 rows go in two halves.
        constexpr int W = D / 8;
        uint8_t* buf = sQ + t * Cfg::TILE + warp % 4 * (W * 16 * 32);
        uint8_t* mine = buf + lane * (W * 16);
        auto leave = [&](auto* dst, int64_t own, int per, int col0) {
          __syncwarp();
#pragma unroll 4
          for (int i = 0; i < W; ++i) {
            const int row = i * (32 / W) + lane / W, k = lane % W;
            const int64_t to = __shfl_sync(0xffffffffu, own, row);
            if (to >= 0 && col0 + k * per < p.D)
              *reinterpret_cast<uint4*>(dst + to + col0 + k * per) =
                  *reinterpret_cast<const uint4*>(buf + row * (W * 16) + ((k ^ (row % W)) << 4));
          }
          __syncwarp();
        };
        if (CAUSAL && direct) {
#pragma unroll
          for (int c = 0; c < D; c += 32) {
            uint32_t ov[32];
            tmem_ld32(tO + c, ov);
            tmem_ld_wait32(ov);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t pk[4];
#pragma unroll
              for (int i = 0; i < 4; ++i)
                pk[i] = pack2<T>(__uint_as_float(ov[8 * e + 2 * i]) * inv, __uint_as_float(ov[8 * e + 2 * i + 1]) * inv);
              *reinterpret_cast<uint4*>(mine + (((c / 8 + e) ^ (lane % W)) << 4)) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
            }
          }
          leave(reinterpret_cast<T*>(p.out), votes ? tok * p.o_st + head * p.o_sh : -1, 8, 0);
        } else {
#pragma unroll
          for (int c0 = 0; c0 < D; c0 += D / 2) {
#pragma unroll
            for (int c = 0; c < D / 2; c += 32) {
              uint32_t ov[32];
              tmem_ld32(tO + c0 + c, ov);
              tmem_ld_wait32(ov);
#pragma unroll
              for (int e = 0; e < 8; ++e)
                *reinterpret_cast<float4*>(mine + (((c / 4 + e) ^ (lane % W)) << 4)) =
                    make_float4(__uint_as_float(ov[4 * e]) * inv, __uint_as_float(ov[4 * e + 1]) * inv,
                                __uint_as_float(ov[4 * e + 2]) * inv, __uint_as_float(ov[4 * e + 3]) * inv);
            }
            leave(p.o_part, votes ? part * p.D : -1, 4, c0);
          }
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == WARP_MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, Cfg::TMEM_COLS);
  }
  if (*abort_flag && warp == WARP_LOAD && lane == 0) {
    // a wait gave up somewhere: copies still in flight land before the CTA's smem is another's
    mbar_wait(&bars->q_full, 0, p.ec, abort_flag, SITE_PA_DRAIN, true);
    for (int s = max(0, issued - Cfg::NBUF); s < issued; ++s)
      mbar_wait(&bars->kv_full[s % Cfg::NBUF], (s / Cfg::NBUF) & 1, p.ec, abort_flag, SITE_PA_DRAIN, true);
  }
}

// Joins the shares of a prefill: one warp for each (token, query head) of the
// requests longer than a share, the loads of four shares in flight (one share at a
// time: 50 us behind the last CTA of a chunk of 2048 tokens, D 128, against 33).
template <typename T>
__global__ void __launch_bounds__(256, 6) ffa_page_attn_merge_kernel(const PaParams p) {
  constexpr int FOLD = 4;
  const int64_t w = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / 32;
  const int lane = threadIdx.x % 32;
  int tok = 0, head = 0, parts = 0;
  if (w < (int64_t)p.T * p.Hq) {  // (lengths and boundaries are nothing that the launch before writes)
    tok = (int)(w / p.Hq);
    head = (int)(w % p.Hq);
    const int seg = warp_search(p.starts, p.N, tok, lane);  // the request
    const int first = p.starts[seg], end = p.starts[seg + 1], kv = p.kv_lens[seg], n = end - first;
    if (first >= 0 && tok >= first && tok < end && end <= p.T && kv >= n && kv <= p.max_ctx && kv > p.chunk)
      parts = share_count(kv - n + tok - first + 1, p.chunk, p.shares);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (parts == 0) return;
  const int64_t step = (int64_t)p.T * p.Hq;
  const bool live = lane * 4 < p.D;
  float M = -INFINITY, L = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < parts; s0 += FOLD) {
    float x[FOLD], top = M;
    float4 v[FOLD];
#pragma unroll
    for (int k = 0; k < FOLD; ++k) {
      const int64_t at = w + (s0 + k) * step;
      const bool has = s0 + k < parts;
      x[k] = has ? __ldcg(p.lse_part + at) : -INFINITY;
      v[k] = has && live ? __ldcg(reinterpret_cast<const float4*>(p.o_part + at * p.D + lane * 4))
                         : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int k = 0; k < FOLD; ++k) top = fmaxf(top, x[k]);
    const float keep = M == -INFINITY ? 0.f : ex2(M - top);
    L *= keep;
    acc = make_float4(acc.x * keep, acc.y * keep, acc.z * keep, acc.w * keep);
#pragma unroll
    for (int k = 0; k < FOLD; ++k) {
      const float f = x[k] == -INFINITY ? 0.f : ex2(x[k] - top);
      L += f;
      acc.x += f * v[k].x;
      acc.y += f * v[k].y;
      acc.z += f * v[k].z;
      acc.w += f * v[k].w;
    }
    M = top;
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  if (live) {
    T* dst = reinterpret_cast<T*>(p.out) + tok * p.o_st + head * p.o_sh + lane * 4;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
  }
  if (lane == 0 && p.lse) p.lse[w] = L == 0.f ? -INFINITY : (M + lg2(L)) * 0.6931471805599453f;
}

// Shares of the context and query tiles per CTA.  Two tiles where a segment's rows
// fill more than one and the head dim is above 64 (chunk of 2048 tokens, D 128: 965
// us against 1007 with one; at D 64, whose K and V are half the bytes and whose CTAs
// are half as long, one tile: nine ragged prompts 180 us against 202).  The form for
// 32 rows where segments have at most 16 on average, so that twice as many still
// fit (64 requests of 16 rows 363 us against 378 in the form for 128; 17 requests of
// 2 to 58 rows, which take two blocks then, 165 against 94).
PaShape pa_shape(int64_t tokens, int64_t segments, int64_t kv, int Hkv, int G, int D) {
  PaShape s{};
  const int64_t mean = (tokens + segments - 1) / segments;  // tokens of a segment
  s.rows = D > 64 && mean * G <= 16 ? 32 : 128;
  const int tq = s.rows / G;
  s.nqt = D > 64 && mean > tq ? 2 : 1;
  const int64_t per = (int64_t)tq * s.nqt, slots = s.nqt == 2 ? 148 : D > 64 ? 296 : 592;
  const int64_t base = segments * ((mean + per - 1) / per) * Hkv;
  const int64_t tiles = (kv + PA_BN - 1) / PA_BN;
  // time of a CTA: 5 us of start and end, and its key tiles (us a tile, alone on an
  // SM and with its slots full; the latter at the memory's rate where nobody else
  // reads the same keys); a partial result costs its writing and reading
  const double alone = 1.9, shared = s.nqt == 2 ? 2.05 : D > 64 ? 2.1 : 3.5;
  const double fresh = PA_BN * D * 4.0 * slots / 6.5e6, full = mean > per || fresh < shared ? shared : fresh;
  // (a CTA of one query tile where others have two is done in about half the time)
  const double busy = 0.5 + 0.5 * (double)((mean + tq - 1) / tq) / (double)((mean + per - 1) / per * s.nqt);
  double least = 0;
  int64_t best = 1;
  for (int64_t n = 1; n <= tiles && n <= PA_MAX_SHARES; ++n) {
    const int64_t each = (tiles + n - 1) / n, used = (tiles + each - 1) / each;
    if (used != n) continue;
    const int64_t ctas = base * n, waves = (ctas + slots - 1) / slots;
    const double load = ctas < slots ? (double)ctas / slots : 1.0;
    double t = waves * (5.0 + each * (alone + (full > alone ? full - alone : 0.0) * load));
    if (n > 1) t += 2.0 + (double)n * tokens * Hkv * G * D * 8 / 6.0e6;
    if (n == 1 || t < least) {
      least = t, best = n;
      s.time = (float)t;
      s.idle = (float)(1.0 - (double)ctas / (double)(waves * slots) * busy);
    }
  }
  const int64_t each = (tiles + best - 1) / best;
  s.shares = (int)best;
  s.chunk = each > 0 && each < (1 << 24) ? (int)each * PA_BN : 0x7fffff80;  // (past any context: one share)
  return s;
}

template <typename T, int D, int NQT, bool FEW, bool CAUSAL>
static int launch_page_attn(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const PaParams& p,
                            int64_t grid, cudaStream_t st) {
  using Cfg = PaCfg<D, NQT, FEW>;
  auto kern = ffa_page_attn_kernel<T, D, NQT, FEW, CAUSAL>;
  static std::atomic<uint64_t> done{0};
  if (int s = smem_attr_once(kern, Cfg::SMEM, done)) return s;
  kern<<<(unsigned)grid, Cfg::THREADS, Cfg::SMEM, st>>>(mq, mk, mv, p);
  return launch_status();
}

// Tensor maps and the launch, for either form.
int page_attn(const PaCall& c, const PaShape& shape, void* stream) {
  PaParams p{};
  p.starts = c.starts;
  p.kv_lens = c.kv_lens;
  p.lens = c.lens;
  p.table = c.block_table;
  p.bt_stride = c.width;
  p.out = c.out;
  if (c.out) {
    p.o_st = c.o_strides[0];
    p.o_sh = c.o_strides[1];
  }
  p.lse = c.lse;
  p.N = c.N;
  p.T = c.T;
  p.Hq = c.Hq;
  p.Hkv = c.Hkv;
  p.G = c.Hq / c.Hkv;
  p.TQ = shape.rows / p.G;
  p.D = c.D;
  p.num_pages = c.num_pages;
  p.page_size = c.page_size;
  p.box = 8;
  while (p.box < (c.D <= 64 ? 64 : 128) && c.page_size % (2 * p.box) == 0) p.box *= 2;  // (at most a key tile)
  p.max_ctx = c.width * c.page_size;
  p.shares = shape.shares;
  p.chunk = shape.chunk;
  const int64_t rows = (int64_t)c.T * c.Hq;
  p.o_part = static_cast<float*>(c.workspace);
  p.lse_part = p.o_part + rows * shape.shares * c.D;
  p.scale_log2 = c.scale * 1.4426950408889634f;
  p.use_softcap = c.softcap > 0.f;
  p.sc_pre = p.use_softcap ? c.scale / c.softcap : 0.f;
  p.sc_unit = p.use_softcap ? c.softcap / c.scale : 0.f;
  softcap_poly_coeffs(p.sc_pre, p.sc_poly);
  const int64_t per = (int64_t)p.TQ * shape.nqt;
  const int64_t items = c.N + c.T / per;  // the sum of ceil(n / per) over segments of c.T tokens is at most this
  p.keep_kv = c.T > c.N * per;
  p.ec.err = c.dev_err;
  p.ec.limit_ns = wait_limit_ns();
  const int64_t grid = items * p.Hkv * p.shares;
  if (grid > 0x7fffffffLL) return FFA_ERR_UNSUPPORTED;

  const CUtensorMapDataType dt =
      c.dtype == FFA_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUtensorMap mq, mk, mv;
  const uint64_t pool = (uint64_t)c.num_pages * c.Hkv * c.page_size, line = (uint64_t)c.D * 2;
  int st = make_tmap_4d(&mq, c.q, dt, 2, c.D, p.G, c.T, c.Hkv, c.q_strides[1] * 2, c.q_strides[0] * 2,
                        (uint64_t)p.G * c.q_strides[1] * 2, 64, p.G, p.TQ);
  if (!st) st = make_tmap_4d(&mk, c.k_pages, dt, 2, c.D, pool, 1, 1, line, pool * line, pool * line, 64, p.box);
  if (!st) st = make_tmap_4d(&mv, c.v_pages, dt, 2, c.D, pool, 1, 1, line, pool * line, pool * line, 64, p.box);
  if (st) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto typed = [&](auto t) -> int {
    using T = decltype(t);
    auto shaped = [&](auto causal) -> int {
      constexpr bool C = decltype(causal)::value;
      if (c.D <= 64)
        return launch_page_attn<T, 64, 1, false, C>(mq, mk, mv, p, grid, s);
      if (shape.rows == 32) return launch_page_attn<T, 128, 1, true, C>(mq, mk, mv, p, grid, s);
      return shape.nqt == 1 ? launch_page_attn<T, 128, 1, false, C>(mq, mk, mv, p, grid, s)
                            : launch_page_attn<T, 128, 2, false, C>(mq, mk, mv, p, grid, s);
    };
    if (!c.causal) return shaped(std::false_type{});
    int status = shaped(std::true_type{});
    if (status || p.shares == 1) return status;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)((rows + 7) / 8));
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, ffa_page_attn_merge_kernel<T>, p));
  };
  return c.dtype == FFA_DTYPE_BF16 ? typed(__nv_bfloat16{}) : typed(__half{});
}

// Sizes, strides and pointers that both forms need.
int pa_check(const PaCall& c) {
  if (!c.q || !c.k_pages || !c.v_pages || !c.block_table || !c.starts || !c.kv_lens || !c.q_strides)
    return FFA_ERR_INVALID_ARG;
  if (c.T <= 0 || c.N <= 0 || c.Hq <= 0 || c.Hkv <= 0 || c.Hq % c.Hkv || c.D <= 0 || c.num_pages <= 0 ||
      c.page_size <= 0 || c.width <= 0 || !(c.scale > 0.f))
    return FFA_ERR_INVALID_ARG;
  if (c.dtype != FFA_DTYPE_BF16 && c.dtype != FFA_DTYPE_F16) return FFA_ERR_UNSUPPORTED;
  if (c.D % 8 || c.D > 128 || c.page_size % 8 || c.Hq / c.Hkv > 128) return FFA_ERR_UNSUPPORTED;
  // pool rows and positions are 32-bit indexes (a box reaches up to 128 past the last)
  if ((int64_t)c.num_pages * c.Hkv * c.page_size > 0x7fffffffLL || (int64_t)c.width * c.page_size > 0x7fffff00LL ||
      (int64_t)c.T * (c.Hq / c.Hkv) > 0x7fffff00LL)
    return FFA_ERR_UNSUPPORTED;
  if (!aligned16(c.q) || !aligned16(c.k_pages) || !aligned16(c.v_pages) || c.q_strides[0] % 8 || c.q_strides[1] % 8 ||
      c.q_strides[0] < 0 || c.q_strides[1] < 0)
    return FFA_ERR_INVALID_ARG;
  return FFA_OK;
}

size_t pa_workspace(int64_t T, int Hq, int D, int shares) {
  return shares > 1 ? (size_t)T * Hq * shares * (D + 1) * 4 : 0;
}

}  // namespace ffa

extern "C" size_t ffa_paged_prefill_workspace_size(int R, int T, int Hq, int Hkv, int D, int max_ctx) {
  using namespace ffa;
  if (R <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || Hq / Hkv > 128 || D <= 0 || D > 128 || max_ctx < 0)
    return 0;
  return pa_workspace(T, Hq, D, pa_shape(T, R, max_ctx, Hkv, Hq / Hkv, D).shares);
}

extern "C" int ffa_paged_prefill(const void* q, const void* k_pages, const void* v_pages, const int* block_table,
                                 const int* ctx_lens, const int* query_starts, void* out, float* lse, int dtype, int R,
                                 int T, int Hq, int Hkv, int D, int num_pages, int page_size, int max_pages_per_req,
                                 const int64_t* q_strides, const int64_t* o_strides, float scale, float softcap,
                                 int max_ctx, void* workspace, size_t workspace_bytes, uint32_t* dev_err,
                                 void* stream) {
  using namespace ffa;
  if (R == 0 || T == 0) return FFA_OK;
  PaCall c{};
  c.q = q;
  c.k_pages = k_pages;
  c.v_pages = v_pages;
  c.block_table = block_table;
  c.starts = query_starts;
  c.kv_lens = ctx_lens;
  c.out = out;
  c.lse = lse;
  c.dtype = dtype;
  c.N = R;
  c.T = T;
  c.Hq = Hq;
  c.Hkv = Hkv;
  c.D = D;
  c.num_pages = num_pages;
  c.page_size = page_size;
  c.width = max_pages_per_req;
  c.q_strides = q_strides;
  c.o_strides = o_strides;
  c.scale = scale;
  c.softcap = softcap;
  c.causal = true;
  c.workspace = workspace;
  c.dev_err = dev_err;
  if (int s = pa_check(c)) return s;
  if (!out || !o_strides || max_ctx < 0 || !aligned16(out) || o_strides[0] % 8 || o_strides[1] % 8)
    return FFA_ERR_INVALID_ARG;
  const PaShape shape = pa_shape(T, R, max_ctx, Hkv, Hq / Hkv, D);
  const size_t need = pa_workspace(T, Hq, D, shape.shares);
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace))) return FFA_ERR_WORKSPACE;
  return page_attn(c, shape, stream);
}

// Paged decode over a sliding window and the first tokens (sinks): one query
// token per request attends the last `window` tokens of its context and its
// first `sinks` tokens, straight from the page pool.  Pages outside both are
// never looked at, so a cache may have freed them.
//
// The visible tokens of a request form one virtual sequence
//   v in [0, ns)        -> token v               ns = min(sinks, w0)
//   v in [ns, nv)       -> token w0 + v - ns     w0 = max(ctx - window, 0)
// and the kernel walks 16-token chunks of it: the sinks share their chunk with
// the window's first tokens, nothing of a masked token is read, and a page may
// begin and end anywhere inside a chunk (each row has its own table look-up).
//
// One cluster of CTAs per (request, kv head, block of 16 query heads); its
// CTAs split the chunks and join their partial softmaxes through distributed
// shared memory, so a call is one launch without a workspace.  Each of a CTA's
// warps streams its own chunks of K and V into its own ring of shared memory
// with 16-byte asynchronous copies (the pool rows are contiguous; the store
// swizzles them for ldmatrix), computes S = Q K^T and O += P V for all heads of
// the block with warp-level tensor-core MMAs, and keeps its own running
// maximum and sum.  No warp waits for another before the join.
//
// HBM-bound: the K and V bytes of the visible tokens, read once per kv head;
// 64 requests, window 4096 + 4, 32/8 heads, D 128: 154 us, 6.59 TB/s (1.0 of a
// measured copy).  One request alone is bound by latencies (11 us: the launch,
// the length, the table, the rows, each warp's few chunks, two cluster barriers).
// P is rounded to the data's type for the P V product (the tensor core's
// operand), the row sums add the unrounded values; statistics, O and the join
// are fp32.
//
// The PREFIX form (ffa_prefix_decode) is the second launch of decoding behind a
// shared prefix: a request that shares attends its own tokens alone, those
// behind the prefix, and joins the partial results that ffa_page_attn.cu left
// for its rows.  It starts while that kernel still runs (programmatic launch:
// its loads need nothing of it) and waits for it only before the join.  Where
// the prefix leaves SMs idle for long, it leaves a partial result of its own
// tokens instead, and a third launch joins them, so that nothing waits.  Where
// little is shared, it is the only launch, and every request attends all of its
// tokens, those of the prefix through the table row that lends them.
#include <cooperative_groups.h>
#include <math.h>

#include "ffa_common.cuh"
#include "ffa_host.h"
#include "ffa_page_attn.h"

namespace ffa {

namespace cg = cooperative_groups;

// Tokens per chunk: one running-maximum update, one K-step of P V.  32 tokens
// took as long per token (a warp is bound by its instructions, about 30 a token)
// and left fewer warps for the same shared memory: 192 us against 165 on 64
// requests of a 4096-token window, 32/8 heads, D 128.
constexpr int WD_CHUNK = 16;

// PREFIX: partial results that a thread asks for at a time.
constexpr int FOLD = 8;

struct WdParams {
  const void* q;  // [R, Hq, D]
  int64_t q_sr, q_sh;
  const void* kp;  // [P, Hkv, page_size, D]
  const void* vp;
  const int* block_table;
  int64_t bt_stride;
  const int* ctx_lens;
  int num_pages, max_ctx;
  void* out;  // [R, Hq, D]
  int64_t o_sr, o_sh;
  float* lse;  // [R, Hq] or nullptr
  int R, Hq, Hkv, G, D, page_size, window, sinks;
  uint32_t ps_mul;  // division by page_size (WdRows)
  int ps_shift;
  int splits;       // CTAs per cluster
  int head_blocks;  // blocks of 16 query heads in a group
  float scale_log2, sc_pre, sc_post;
  float sc_poly[3];  // PREFIX: softcap_small2's
  int use_softcap;
  uint32_t* err;
  // PREFIX: requests [starts[g], starts[g + 1]) share their first prefix_lens[g]
  // tokens, whose partial results lie in o_part [shares, R, Hq, D] (normalised)
  // and lse_part [shares, R, Hq] (base 2), one for every `chunk` tokens
  const int *starts, *prefix_lens;
  int groups, shares, chunk;
  const float *o_part, *lse_part;
  // own tokens' partial results [R, Hq, D] and [R, Hq] (base 2) of requests that
  // share, for ffa_prefix_join_kernel to join with those; or nullptr
  float *o_own, *lse_own;
  int whole;  // or no launch before: each request attends its prefix too, through its group's row
};

// WARPS per CTA, each with STAGES chunks in flight.  Two shapes:
//   4 warps, 64 KB of rings (2 stages at 128 columns), three CTAs per SM;
//   2 warps, 48 KB (3 stages), four CTAs per SM, for 128 columns: more requests
//     run unsplit in one wave (at 64 columns the warps' instructions bound it).
// 8 warps, or 4 with 3 stages, leave fewer CTAs per SM: 183 us and more on 64
// requests of a 4096-token window, 32/8 heads, D 128, against 165 and less.
template <int DP, int WARPS>
struct WdCfg {
  static constexpr int THREADS = WARPS * 32;
  static constexpr int STAGES = (WARPS == 2 ? 3 : 2) * (128 / DP);
  static constexpr int HALF = WD_CHUNK * 128;        // a chunk's rows x 64 elements
  static constexpr int KV_BYTES = WD_CHUNK * DP * 2; // one chunk of K (or V)
  static constexpr int STAGE = 2 * KV_BYTES;
  static constexpr int RING = WARPS * STAGES * STAGE;
  // the joins overlay the rings, idle by then: per warp, then per CTA,
  // 16 rows x (m, l, O[DP])
  static constexpr int STATE = 16 * (DP + 2);        // floats
  static constexpr int CTA_OFF = (WARPS + 1) * STATE * 4;  // (one more for PREFIX)
  static constexpr int MERGE = CTA_OFF + STATE * 4;
  static constexpr int SMEM = (RING > MERGE ? RING : MERGE) + 1024;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// What one lane needs to turn a virtual index into a pool row.
template <bool PREFIX>
struct WdRows {
  const int* table;
  const int* lead;  // PREFIX: the table row of virtual indexes below ns
  int h, Hkv, page_size, num_pages, ns, skip, nv;  // skip: added to v >= ns
  uint32_t ps_mul;
  int ps_shift;
  uint32_t* err;
  // Table entry of virtual index v, and the token's offset in its page (any
  // values for one past the end).  Division by the page size as a product:
  // ps_mul = floor(2^(31 + k) / d) + 1 with 2^k >= d is exact below 2^31.
  __device__ __forceinline__ int page(int v, int& off) const {
    off = 0;
    if (v >= nv) return 0;
    const uint32_t tok = v < ns ? v : v + skip;
    const uint32_t i = (uint32_t)(((uint64_t)tok * ps_mul) >> ps_shift);
    off = (int)(tok - i * page_size);
    return (PREFIX && v < ns ? lead : table)[i];
  }
  // pool row, or -1: past the end, or a page id outside the pool (recorded)
  __device__ __forceinline__ int row(int v, int page, int off) const {
    if (v >= nv) return -1;
    if ((unsigned)page >= (unsigned)num_pages) {
      if (err) atomicCAS(err, 0u, SITE_DEC_BAD_PAGE);
      return -1;
    }
    return (page * Hkv + h) * page_size + off;
  }
};

template <typename T>
__device__ __forceinline__ T wd_round(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 wd_round<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half wd_round<__half>(float x) { return __float2half_rn(x); }

// Prefix length of request r's group (0: in none) and the group's first request,
// found by one warp.  A request shorter than it shares nothing.
__device__ __forceinline__ int wd_prefix(const WdParams& p, int r, int lane, int& first) {
  first = r;
  if (p.groups == 0) return 0;
  if (p.groups >= 32) {
    const int g = warp_search(p.starts, p.groups + 1, r, lane);
    if (g >= p.groups || p.starts[g] > r) return 0;
    first = p.starts[g];
    return p.prefix_lens[g];
  }
  // few groups: their lengths asked for with the starts, not after them
  const int start = lane <= p.groups ? p.starts[lane] : 0x7fffffff;
  const int len = lane < p.groups ? p.prefix_lens[lane] : 0;
  const int g = __popc(__ballot_sync(0xffffffffu, start <= r)) - 1;
  if (g < 0 || g >= p.groups) return 0;
  first = __shfl_sync(0xffffffffu, start, g);
  return __shfl_sync(0xffffffffu, len, g);
}

// The first request of [first, r] that is as long as the prefix (its table row is
// the group's), or -1, found by one warp.
__device__ __forceinline__ int wd_lead(const WdParams& p, int first, int r, int prefix, int lane) {
  for (int i0 = max(first, 0); i0 <= r; i0 += 32) {
    const int len = i0 + lane <= r ? p.ctx_lens[i0 + lane] : -1;
    const uint32_t has = __ballot_sync(0xffffffffu, len >= prefix && len <= p.max_ctx);
    if (has) return i0 + __ffs(has) - 1;
  }
  return -1;
}

template <typename T, int DP, int WARPS, bool PREFIX>
__global__ void __launch_bounds__(WARPS * 32) ffa_window_decode_kernel(const WdParams p) {
  using Cfg = WdCfg<DP, WARPS>;
  constexpr int WD_WARPS = WARPS, WD_THREADS = Cfg::THREADS;
  constexpr int S = Cfg::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int split = blockIdx.x % p.splits;
  int pair = blockIdx.x / p.splits;
  const int hb = pair % p.head_blocks;
  pair /= p.head_blocks;
  const int h = pair % p.Hkv, r = pair / p.Hkv;
  const int g0 = hb * 16, G = min(16, p.G - g0);  // query heads h * p.G + g0 + [0, G)

  const bool apart = PREFIX && p.o_own;  // the joining kernel may start, and wait
  if (apart) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  int ctx = p.ctx_lens[r];
  int first = r;
  const int prefix = PREFIX ? wd_prefix(p, r, lane, first) : 0;  // (its loads travel with the length's)
  if (ctx < 0 || ctx > p.max_ctx) {
    if (threadIdx.x == 0 && p.err) atomicCAS(p.err, 0u, SITE_DEC_BAD_CTX);
    ctx = 0;
  }
  int shared = prefix > 0 && prefix <= ctx ? prefix : 0;
  const bool whole = PREFIX && p.whole;
  int lead = r;
  if (whole) {
    if (shared) lead = wd_lead(p, first, r, prefix, lane);
    if (lead < 0) shared = 0, lead = r;  // (boundaries that decrease)
    if (blockIdx.x == 0 && p.err)
      for (int g = threadIdx.x; g < p.groups; g += WD_THREADS) {
        const int lo = p.starts[g], hi = p.starts[g + 1], len = p.prefix_lens[g];
        if (lo < 0 || hi < lo || hi > p.R || (hi > lo && (len < 0 || len > p.max_ctx)))
          atomicCAS(p.err, 0u, SITE_PA_BAD_STARTS);
      }
  }
  const int w0 = PREFIX ? shared : max(ctx - p.window, 0);
  WdRows<PREFIX> rows;
  rows.table = p.block_table + (int64_t)r * p.bt_stride;
  rows.lead = whole ? p.block_table + (int64_t)lead * p.bt_stride : rows.table;
  rows.h = h;
  rows.Hkv = p.Hkv;
  rows.page_size = p.page_size;
  rows.num_pages = p.num_pages;
  rows.ns = whole ? shared : PREFIX ? 0 : min(p.sinks, w0);
  rows.skip = w0 - rows.ns;
  rows.nv = rows.ns + ctx - w0;
  rows.ps_mul = p.ps_mul;
  rows.ps_shift = p.ps_shift;
  rows.err = p.err;
  const int chunks = (rows.nv + WD_CHUNK - 1) / WD_CHUNK;
  const int c0 = (int)((int64_t)chunks * split / p.splits), c1 = (int)((int64_t)chunks * (split + 1) / p.splits);
  const int n = max(0, (c1 - c0 - warp + WD_WARPS - 1) / WD_WARPS);  // this warp's chunks: c0 + warp + i * WD_WARPS

  uint8_t* ring = smem + warp * S * Cfg::STAGE;
  if (p.D < DP) {  // columns past the head dim stay zero: their products must be
    for (int i = lane; i < S * Cfg::STAGE / 16; i += 32) reinterpret_cast<uint4*>(ring)[i] = make_uint4(0, 0, 0, 0);
    __syncwarp();
  }
  // copies: lane takes 16-byte column `col` of rows row0, row0 + step, ...
  constexpr int COLS = DP / 8, STEP = 32 / COLS;
  const int col = lane % COLS, row0 = lane / COLS;
  const uint32_t dst0 = smem_u32(ring) + (col / 8) * Cfg::HALF;
  const int64_t row_bytes = (int64_t)p.D * 2;
  const uint8_t* kcol = static_cast<const uint8_t*>(p.kp) + col * 16;
  const uint8_t* vcol = static_cast<const uint8_t*>(p.vp) + col * 16;
  auto issue = [&](int i, int my_row) {  // chunk i of this warp; my_row: pool row of the chunk's row lane % WD_CHUNK
    const uint32_t d = dst0 + (i % S) * Cfg::STAGE;
#pragma unroll
    for (int k = 0; k < WD_CHUNK / STEP; ++k) {
      const int rr = row0 + k * STEP;
      const int row = __shfl_sync(0xffffffffu, my_row, rr);
      if (col * 8 < p.D) {
        const uint32_t dd = d + rr * 128 + (((col % 8) ^ (rr & 7)) << 4);
        const int64_t off = row < 0 ? 0 : row * row_bytes;
        cp_async16(dd, kcol + off, row >= 0);
        cp_async16(dd + Cfg::KV_BYTES, vcol + off, row >= 0);
      }
    }
  };
  auto vidx = [&](int i) { return (c0 + warp + i * WD_WARPS) * WD_CHUNK + lane % WD_CHUNK; };
  // table entries run one chunk ahead of the copies that need them
  int pages[S + 1], offs[S + 1];
#pragma unroll
  for (int i = 0; i <= S; ++i) {
    pages[i] = offs[i] = 0;
    if (i < n) pages[i] = rows.page(vidx(i), offs[i]);
  }

  // Q as the A operand: rows = the block's query heads (rows past G are zero)
  const int g = lane >> 2, t = lane & 3;
  uint32_t qa[DP / 16][4];
  {
    const T* qbase = reinterpret_cast<const T*>(p.q) + (int64_t)r * p.q_sr + (int64_t)(h * p.G + g0) * p.q_sh;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = g + 8 * (e & 1), c = kk * 16 + 2 * t + 8 * (e >> 1);
        qa[kk][e] = row < G && c < p.D ? *reinterpret_cast<const uint32_t*>(qbase + row * p.q_sh + c) : 0u;
      }
  }
#pragma unroll
  for (int i = 0; i < S; ++i) {
    if (i < n) issue(i, rows.row(vidx(i), pages[i], offs[i]));
    cp_commit();
  }
  int next_page = pages[S], next_off = offs[S];

  float o[DP / 8][4];
#pragma unroll
  for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m_lo = -INFINITY, m_hi = -INFINITY;  // rows g and g + 8 (base-2 units)
  float l_lo = 0.f, l_hi = 0.f;              // this lane's partial row sums
  const int mi = lane >> 3, mr = lane & 7;   // ldmatrix: matrix index / row within it

  for (int i = 0; i < n; ++i) {
    cp_wait<S - 1>();
    __syncwarp();
    const uint32_t kbase = smem_u32(ring + (i % S) * Cfg::STAGE);
    const uint32_t vbase = kbase + Cfg::KV_BYTES;
    constexpr int NT = WD_CHUNK / 8;  // n-tiles of 8 tokens
    float x[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) x[nt][0] = x[nt][1] = x[nt][2] = x[nt][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk) {
      const int hf = kk / 4, ch = 2 * (kk % 4) + (mi & 1);
#pragma unroll
      for (int nt = 0; nt < NT; nt += 2) {
        const int tok = nt * 8 + mr + 8 * (mi >> 1);
        uint32_t b00, b01, b10, b11;
        ldsm_x4(sw128(kbase + hf * Cfg::HALF, tok, ch), b00, b01, b10, b11);
        mma16816<T>(x[nt], qa[kk], b00, b01);
        mma16816<T>(x[nt + 1], qa[kk], b10, b11);
      }
    }
    const int left = rows.nv - (c0 + warp + i * WD_WARPS) * WD_CHUNK;  // tokens of this chunk
    float mul = p.scale_log2;
    // PREFIX: the polynomial where every argument is within 1/2, as the prefix's kernel
    // has it (the tanh's absolute error counts among few tokens of small scores: an
    // LSE of two was 1.1e-6 off, relatively)
    bool tanhs = p.use_softcap;
    if (PREFIX && p.use_softcap) {
      float top = 0.f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(x[nt][e]));
      tanhs = !__all_sync(0xffffffffu, top * p.sc_pre <= 0.5f);
      if (!tanhs) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const float2 y =
                softcap_small2(make_float2(x[nt][e], x[nt][e + 1]), p.sc_poly[0], p.sc_poly[1], p.sc_poly[2]);
            x[nt][e] = y.x;
            x[nt][e + 1] = y.y;
          }
      }
    }
    if (tanhs) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[nt][e] = tanh_acc(x[nt][e] * p.sc_pre);
      mul = p.sc_post;
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) x[nt][e] *= mul;
    if (left < WD_CHUNK) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (nt * 8 + 2 * t + (e & 1) >= left) x[nt][e] = -INFINITY;
    }
    float mx_lo = -INFINITY, mx_hi = -INFINITY;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      mx_lo = fmaxf(mx_lo, fmaxf(x[nt][0], x[nt][1]));
      mx_hi = fmaxf(mx_hi, fmaxf(x[nt][2], x[nt][3]));
    }
#pragma unroll
    for (int off = 1; off < 4; off <<= 1) {
      mx_lo = fmaxf(mx_lo, __shfl_xor_sync(0xffffffffu, mx_lo, off));
      mx_hi = fmaxf(mx_hi, __shfl_xor_sync(0xffffffffu, mx_hi, off));
    }
    // lazy rescale: only when a row max grows by more than 2^8 (exact: the sums
    // and O share the same stale maximum)
    const float mn_lo = fmaxf(m_lo, mx_lo), mn_hi = fmaxf(m_hi, mx_hi);
    if (__any_sync(0xffffffffu, mn_lo > m_lo + 8.f || mn_hi > m_hi + 8.f)) {
      const float a_lo = (mn_lo == -INFINITY) ? 1.f : ex2(m_lo - mn_lo);
      const float a_hi = (mn_hi == -INFINITY) ? 1.f : ex2(m_hi - mn_hi);
      l_lo *= a_lo;
      l_hi *= a_hi;
#pragma unroll
      for (int d = 0; d < DP / 8; ++d) {
        o[d][0] *= a_lo;
        o[d][1] *= a_lo;
        o[d][2] *= a_hi;
        o[d][3] *= a_hi;
      }
      m_lo = mn_lo;
      m_hi = mn_hi;
    }
    const float u_lo = (m_lo == -INFINITY) ? 0.f : m_lo, u_hi = (m_hi == -INFINITY) ? 0.f : m_hi;
#pragma unroll
    for (int ks = 0; ks < NT / 2; ++ks) {  // 16 tokens: one K-step of P V
      float(*pr)[4] = x + 2 * ks;
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        pr[nt][0] = ex2(pr[nt][0] - u_lo);
        pr[nt][1] = ex2(pr[nt][1] - u_lo);
        pr[nt][2] = ex2(pr[nt][2] - u_hi);
        pr[nt][3] = ex2(pr[nt][3] - u_hi);
        l_lo += pr[nt][0] + pr[nt][1];
        l_hi += pr[nt][2] + pr[nt][3];
      }
      const uint32_t pa[4] = {pack2<T>(pr[0][0], pr[0][1]), pack2<T>(pr[0][2], pr[0][3]),
                              pack2<T>(pr[1][0], pr[1][1]), pack2<T>(pr[1][2], pr[1][3])};
#pragma unroll
      for (int nt = 0; nt < DP / 8; nt += 2) {
        const int hf = nt / 8, ch = (nt % 8) + (mi >> 1);
        const int tok = 16 * ks + mr + 8 * (mi & 1);
        uint32_t b0, b1, b2, b3;
        ldsm_x4_t(sw128(vbase + hf * Cfg::HALF, tok, ch), b0, b1, b2, b3);
        mma16816<T>(o[nt], pa, b0, b1);
        mma16816<T>(o[nt + 1], pa, b2, b3);
      }
    }
    __syncwarp();  // every lane has read the stage before it is refilled
    if (i + S < n) issue(i + S, rows.row(vidx(i + S), next_page, next_off));
    cp_commit();
    if (i + S + 1 < n) next_page = rows.page(vidx(i + S + 1), next_off);
  }
  cp_wait<0>();

  // -------------------- join the warps, then the cluster -------------------
#pragma unroll
  for (int off = 1; off < 4; off <<= 1) {
    l_lo += __shfl_xor_sync(0xffffffffu, l_lo, off);
    l_hi += __shfl_xor_sync(0xffffffffu, l_hi, off);
  }
  __syncthreads();  // every ring is idle: the states overlay them
  constexpr int P2 = DP + 2;
  float* wm = reinterpret_cast<float*>(smem) + warp * Cfg::STATE;  // row: m, l, O[DP]
  if (t == 0) {
    wm[g * P2] = m_lo;
    wm[g * P2 + 1] = l_lo;
    wm[(g + 8) * P2] = m_hi;
    wm[(g + 8) * P2 + 1] = l_hi;
  }
#pragma unroll
  for (int nt = 0; nt < DP / 8; ++nt) {
    const int d = 2 + nt * 8 + 2 * t;
    *reinterpret_cast<float2*>(wm + g * P2 + d) = make_float2(o[nt][0], o[nt][1]);
    *reinterpret_cast<float2*>(wm + (g + 8) * P2 + d) = make_float2(o[nt][2], o[nt][3]);
  }
  // PREFIX: the prefix's shares, which the cluster's CTAs divide, are one more state,
  // or a launch of their own joins them.  That one waits for this kernel only, so
  // one CTA here waits for the one before.
  const bool folds = PREFIX && !apart && !whole;
  if (apart && blockIdx.x + 1 == gridDim.x) asm volatile("griddepcontrol.wait;" ::: "memory");
  if (folds) {
    const int parts = shared ? share_count(shared, p.chunk, p.shares) : 0;
    const int64_t step = (int64_t)p.R * p.Hq;
    float* fold = reinterpret_cast<float*>(smem) + WARPS * Cfg::STATE;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // they are complete
    for (int it = threadIdx.x; it < G * (p.D / 4); it += WD_THREADS) {
      const int row = it / (p.D / 4), d = it % (p.D / 4) * 4;
      const int64_t at = (int64_t)r * p.Hq + h * p.G + g0 + row;
      float M = -INFINITY, L = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int s0 = split; s0 < parts; s0 += FOLD * p.splits) {  // FOLD loads in flight
        float x[FOLD], top = M;
        float4 v[FOLD];
#pragma unroll
        for (int k = 0; k < FOLD; ++k) {
          const int s = s0 + k * p.splits;
          x[k] = s < parts ? p.lse_part[at + s * step] : -INFINITY;
          v[k] = s < parts ? *reinterpret_cast<const float4*>(p.o_part + (at + s * step) * p.D + d)
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
          acc.x += v[k].x * f;
          acc.y += v[k].y * f;
          acc.z += v[k].z * f;
          acc.w += v[k].w * f;
        }
        M = top;
      }
      float* to = fold + row * P2;
      *reinterpret_cast<float2*>(to + 2 + d) = make_float2(acc.x, acc.y);
      *reinterpret_cast<float2*>(to + 4 + d) = make_float2(acc.z, acc.w);
      if (d == 0) to[0] = M, to[1] = L;
    }
  }
  __syncthreads();
  // `state(s)`: the s-th partial state; joins two columns of one row
  auto join = [&](int parts, auto state, int row, int d, float& M, float& L, float2& acc) {
    M = -INFINITY;
    for (int s = 0; s < parts; ++s) M = fmaxf(M, state(s)[row * P2]);
    L = 0.f;
    acc = make_float2(0.f, 0.f);
    for (int s = 0; s < parts; ++s) {
      const float* st = state(s) + row * P2;
      const float f = st[0] == -INFINITY ? 0.f : ex2(st[0] - M);
      const float2 v = *reinterpret_cast<const float2*>(st + 2 + d);
      L += st[1] * f;
      acc.x += v.x * f;
      acc.y += v.y * f;
    }
  };
  auto store = [&](int row, int d, float M, float L, float2 acc) {
    const int head = h * p.G + g0 + row;
    const bool none = PREFIX ? L == 0.f : !(L > 0.f);  // (PREFIX: a sum of NaN is no empty row, its LSE is NaN too)
    const float inv = none ? 0.f : 1.f / L;
    if (apart && shared) {
      const int64_t at = (int64_t)r * p.Hq + head;
      *reinterpret_cast<float2*>(p.o_own + at * p.D + d) = make_float2(acc.x * inv, acc.y * inv);
      if (d == 0) p.lse_own[at] = none ? -INFINITY : M + lg2(L);
      return;
    }
    T* dst = reinterpret_cast<T*>(p.out) + (int64_t)r * p.o_sr + (int64_t)head * p.o_sh + d;
    dst[0] = wd_round<T>(acc.x * inv);
    dst[1] = wd_round<T>(acc.y * inv);
    if (d == 0 && p.lse) p.lse[(int64_t)r * p.Hq + head] = none ? -INFINITY : (M + lg2(L)) * 0.6931471805599453f;
  };
  const int items = G * (p.D / 2);
  const float* warps = reinterpret_cast<const float*>(smem);
  float* cta = reinterpret_cast<float*>(smem + Cfg::CTA_OFF);
  for (int it = threadIdx.x; it < items; it += WD_THREADS) {
    const int row = it / (p.D / 2), d = it % (p.D / 2) * 2;
    float M, L;
    float2 acc;
    const auto state = [&](int s) { return warps + s * Cfg::STATE; };
    // (a constant count each way, so that the loops unroll: 37 requests' groups 20.7 -> 20.0 us)
    if (folds) join(WARPS + 1, state, row, d, M, L, acc);
    else join(WARPS, state, row, d, M, L, acc);
    if (p.splits == 1) {
      store(row, d, M, L, acc);
    } else {
      *reinterpret_cast<float2*>(cta + row * P2 + 2 + d) = acc;
      if (d == 0) {
        cta[row * P2] = M;
        cta[row * P2 + 1] = L;
      }
    }
  }
  if (p.splits == 1) return;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  // the cluster's threads share the output: item by item, every CTA's state read through DSMEM
  for (int it = split * WD_THREADS + threadIdx.x; it < items; it += p.splits * WD_THREADS) {
    const int row = it / (p.D / 2), d = it % (p.D / 2) * 2;
    float M, L;
    float2 acc;
    join(p.splits, [&](int s) { return cluster.map_shared_rank(cta, s); }, row, d, M, L, acc);
    store(row, d, M, L, acc);
  }
  cluster.sync();  // no CTA leaves while another reads its shared memory
}

// Joins the prefix's shares and the own tokens of each request that shares: one
// warp for each (request, query head), FOLD partial results in flight.
template <typename T>
__global__ void __launch_bounds__(256) ffa_prefix_join_kernel(const WdParams p) {
  const int64_t at = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / 32;
  const int lane = threadIdx.x % 32;
  int r = 0, head = 0, prefix = 0, ctx = 0;
  if (at < (int64_t)p.R * p.Hq) {
    r = (int)(at / p.Hq);
    head = (int)(at % p.Hq);
    ctx = p.ctx_lens[r];
    int first;
    prefix = wd_prefix(p, r, lane, first);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");  // (every warp: what follows this launch may count on both before)
  if (prefix <= 0 || prefix > ctx || ctx > p.max_ctx) return;
  const int parts = share_count(prefix, p.chunk, p.shares);
  const int64_t step = (int64_t)p.R * p.Hq;
  const bool live = lane * 4 < p.D;
  auto load = [&](const float* o) {  // (from L2: nothing of it may be in an L1 from before the wait)
    return live ? __ldcg(reinterpret_cast<const float4*>(o + lane * 4)) : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  float M = __ldcg(p.lse_own + at), L = M == -INFINITY ? 0.f : 1.f;
  float4 acc = load(p.o_own + at * p.D);
  for (int s0 = 0; s0 < parts; s0 += FOLD) {
    float x[FOLD], top = M;
    float4 v[FOLD];
#pragma unroll
    for (int k = 0; k < FOLD; ++k) {
      const int s = min(s0 + k, parts - 1);
      x[k] = s0 + k < parts ? __ldcg(p.lse_part + at + s * step) : -INFINITY;
      v[k] = load(p.o_part + (at + s * step) * p.D);
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
      acc.x += v[k].x * f;
      acc.y += v[k].y * f;
      acc.z += v[k].z * f;
      acc.w += v[k].w * f;
    }
    M = top;
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  if (live) {
    T* dst = reinterpret_cast<T*>(p.out) + (int64_t)r * p.o_sr + (int64_t)head * p.o_sh + lane * 4;
    dst[0] = wd_round<T>(acc.x * inv);
    dst[1] = wd_round<T>(acc.y * inv);
    dst[2] = wd_round<T>(acc.z * inv);
    dst[3] = wd_round<T>(acc.w * inv);
  }
  if (lane == 0 && p.lse) p.lse[at] = L == 0.f ? -INFINITY : (M + lg2(L)) * 0.6931471805599453f;
}

// Estimated time (us) of `pairs` clusters of s CTAs over `visible` tokens each.
// Full waves of resident CTAs stream at the memory's rate and pay a start and a
// join (4 us); the last, partial one takes that rate or one CTA's own speed
// (13.6 ns a token with 4 warps at 128 columns, 10 at 64), whichever is longer,
// and 5 us.  Measured against it (us, estimate in brackets), D 128, 512 pairs of
// 4100 tokens: 4 warps split by 1, 2, 4, 8: 215 (208), 188 (184), 184 (186),
// 218 (209); 2 warps split by 1, 2, 4: 167 (170), 178 (174), 189 (188).  8 pairs
// of 4100 split by 8, 16: 13.6, 11.1; 512 pairs of 1028: 4 warps 64 (59), 2 warps
// 51 (47); 296 pairs of 4100: 4 warps unsplit 100 (101), 2 warps split by 2 103.
static double wd_time(int64_t pairs, int64_t visible, int D, int warps, int s) {
  const double per_token = 4.0 * D / 6.5e6;  // K and V bytes over bytes per us
  const double own = (D > 64 ? 0.0136 : 0.010) * 4 / warps, tokens = (double)visible / s;
  const int64_t slots = 148 * (warps == 2 ? 4 : 3), ctas = pairs * s;
  const int64_t full = ctas / slots, rest = ctas % slots;
  double t = full * (slots * tokens * per_token + 4.0);
  if (rest) t += fmax(rest * tokens * per_token, tokens * own) + 5.0;
  return t;
}

// The same for the PREFIX form, whose requests hold anything up to `visible`
// tokens: the CTAs' throughput at the mean length, or the longest one's own
// time.  Measured against it (us, estimate in brackets), D 128, 512 pairs of 1
// to 1024 tokens: 4 warps split by 1, 2, 4: 32 (31), 37 (47), 52 (78); 2 warps 39
// (34), 41, 47.  2048 pairs of 1 to 512: 4 warps 54 (66), 91 (123); 2 warps 59 (66), 88.
static double wd_time_ragged(int64_t pairs, int64_t visible, int D, int warps, int s) {
  const double per_token = 4.0 * D / 6.5e6, own = (D > 64 ? 0.0136 : 0.010) * 4 / warps;
  const double slots = 148 * (warps == 2 ? 4 : 3), mean = 0.5 * visible / s;
  const double start = s > 1 ? 8.0 : warps == 2 ? 5.5 : 4.0;
  return fmax(pairs * s / slots * (start + mean * slots * per_token), (double)visible / s * own) + (s > 1 ? 7.5 : 6.0);
}

// CTAs per cluster and warps per CTA with the least estimated time: powers of
// two up to 16, no less than a chunk per warp.
static void wd_shape(bool ragged, int64_t pairs, int64_t visible, int D, int& splits, int& warps) {
  double least = 0;
  splits = 0;
  for (int w = 4; w >= (D > 64 ? 2 : 4); w -= 2)
    for (int s = 1; s <= 16 && (s == 1 || visible >= (int64_t)s * w * WD_CHUNK); s *= 2) {
      const double t = ragged ? wd_time_ragged(pairs, visible, D, w, s) : wd_time(pairs, visible, D, w, s);
      if (!splits || t < least) splits = s, warps = w, least = t;
    }
}

template <typename T, int DP, int WARPS, bool PREFIX>
static int launch_window_decode(const WdParams& p, int64_t grid, cudaStream_t st) {
  using Cfg = WdCfg<DP, WARPS>;
  auto kern = ffa_window_decode_kernel<T, DP, WARPS, PREFIX>;
  static std::atomic<uint64_t> done{0}, wide{0};
  if (int s = smem_attr_once(kern, Cfg::SMEM, done)) return s;
  if (p.splits > 8) {  // clusters past 8 CTAs are opt-in
    int dev = 0;
    if (int s = cuda_status(cudaGetDevice(&dev))) return s;
    const uint64_t bit = dev < 64 ? (1ull << dev) : 0ull;
    if (!bit || !(wide.load(std::memory_order_acquire) & bit)) {
      if (int s = cuda_status(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1))) return s;
      if (bit) wide.fetch_or(bit, std::memory_order_acq_rel);
    }
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(Cfg::THREADS);
  cfg.dynamicSmemBytes = Cfg::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)p.splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  // (with groups the launch before this one is their partial results')
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = PREFIX && p.groups && !p.whole ? 2 : 1;
  if (int s = cuda_status(cudaLaunchKernelEx(&cfg, kern, p))) return s;
  if (!PREFIX || !p.o_own) return FFA_OK;
  cudaLaunchConfig_t join{};
  join.gridDim = dim3((unsigned)(((int64_t)p.R * p.Hq + 7) / 8));
  join.blockDim = dim3(256);
  join.stream = st;
  join.attrs = attr + 1;
  join.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&join, ffa_prefix_join_kernel<T>, p));
}

// The launch for either form; `visible`: the most tokens a request sees here;
// `before` (PREFIX): the launch of the prefix.  What it leaves idle works off own
// tokens while it runs, if their CTAs do not wait for its partial results, which
// costs the joining launch 4 us (256 requests of 1 to 512 tokens behind 32768, 32/8
// heads, D 128, where 128 CTAs take the prefix: 187 us to 174; 64 requests of 1 to
// 1024 behind 8192, where 144 do: 54 to 57).  Nothing is gained where all of them
// find room beside the prefix (four requests behind 200 tokens, if the prefix is
// done for the group: 12.3 us to 13.7).
template <bool PREFIX>
static int window_decode(WdParams& p, int dtype, int64_t visible, const PaShape& before, cudaStream_t st) {
  int k = 0;
  while ((1ll << k) < p.page_size) ++k;
  p.ps_shift = 31 + k;
  p.ps_mul = (uint32_t)((1ull << p.ps_shift) / (unsigned)p.page_size + 1);
  p.G = p.Hq / p.Hkv;
  p.head_blocks = (p.G + 15) / 16;
  const int64_t pairs = (int64_t)p.R * p.Hkv * p.head_blocks;
  int warps = 4;
  wd_shape(PREFIX && !p.whole, pairs, visible, p.D, p.splits, warps);
  const int64_t grid = pairs * p.splits;
  if (grid > 0x7fffffffLL) return FFA_ERR_UNSUPPORTED;
  if (PREFIX && (before.idle * before.time <= 6.f || grid <= before.idle * 148 * (warps == 2 ? 4 : 3)))
    p.o_own = nullptr;
  auto typed = [&](auto t) -> int {
    using T = decltype(t);
    if (p.D <= 64) return launch_window_decode<T, 64, 4, PREFIX>(p, grid, st);
    return warps == 2 ? launch_window_decode<T, 128, 2, PREFIX>(p, grid, st)
                      : launch_window_decode<T, 128, 4, PREFIX>(p, grid, st);
  };
  return dtype == FFA_DTYPE_BF16 ? typed(__nv_bfloat16{}) : typed(__half{});
}

}  // namespace ffa

extern "C" int ffa_window_decode(const void* q, const void* k_pages, const void* v_pages, const int* block_table,
                                 const int* ctx_lens, void* out, float* lse, int dtype, int R, int Hq, int Hkv,
                                 int D, int num_pages, int page_size, int max_pages_per_req,
                                 const int64_t* q_strides, const int64_t* o_strides, float scale, float softcap,
                                 int window, int sinks, int max_ctx, uint32_t* dev_err, void* stream) {
  using namespace ffa;
  if (R == 0) return FFA_OK;
  if (!q || !k_pages || !v_pages || !block_table || !ctx_lens || !out || !q_strides || !o_strides)
    return FFA_ERR_INVALID_ARG;
  if (R < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || D <= 0 || num_pages <= 0 || page_size <= 0 ||
      max_pages_per_req <= 0 || window <= 0 || sinks < 0)
    return FFA_ERR_INVALID_ARG;
  if (dtype != FFA_DTYPE_BF16 && dtype != FFA_DTYPE_F16) return FFA_ERR_UNSUPPORTED;
  if (D % 8 || D > 128) return FFA_ERR_UNSUPPORTED;
  // pool rows and context positions are 32-bit indexes in the kernel
  if ((int64_t)num_pages * Hkv * page_size > 0x7fffffffLL || (int64_t)max_pages_per_req * page_size > 0x7fffffffLL)
    return FFA_ERR_UNSUPPORTED;
  if (!aligned16(k_pages) || !aligned16(v_pages) || (reinterpret_cast<uintptr_t>(q) & 3) || q_strides[0] % 2 ||
      q_strides[1] % 2)
    return FFA_ERR_INVALID_ARG;
  WdParams p{};
  p.q = q;
  p.q_sr = q_strides[0];
  p.q_sh = q_strides[1];
  p.kp = k_pages;
  p.vp = v_pages;
  p.block_table = block_table;
  p.bt_stride = max_pages_per_req;
  p.ctx_lens = ctx_lens;
  p.num_pages = num_pages;
  p.max_ctx = max_pages_per_req * page_size;
  p.out = out;
  p.o_sr = o_strides[0];
  p.o_sh = o_strides[1];
  p.lse = lse;
  p.R = R;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.D = D;
  p.page_size = page_size;
  p.window = window;
  p.sinks = sinks;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.use_softcap = softcap > 0.f;
  p.sc_pre = p.use_softcap ? scale / softcap : 0.f;
  p.sc_post = p.use_softcap ? softcap * 1.4426950408889634f : 0.f;
  p.err = dev_err;
  // the most tokens a request can see
  int64_t visible = max_ctx > 0 && max_ctx < p.max_ctx ? max_ctx : p.max_ctx;
  if (visible > (int64_t)window + sinks) visible = (int64_t)window + sinks;
  return window_decode<false>(p, dtype, visible, PaShape{}, static_cast<cudaStream_t>(stream));
}

// The shares of a prefix: ffa_page_attn.cu's shape, with a workspace for every one.
// No share where each request reads the prefix itself (from the group's pages), in
// one launch: where that takes 5 us at most, the bytes of all of them at the
// memory's rate, or a CTA's part of the tokens at its own speed.  Shared against
// whole, us on the device with own tokens of 1 to 100, 32/8 heads of 128: 16
// requests behind 100 tokens (estimate 1) 11.9, 8.8; behind 400 (4) 12.1, 11.2;
// behind 1000 (10) 12.4, 16.6; 64 behind 100 (4) 17.4, 13.6; behind 400 (16) 18.6,
// 24; 8/2 heads of 64: 4 behind 8000 (5) 14.8, 12.2; 16 behind 4000 (5) 12.1, 12.0;
// 64 behind 1000 (5) 10.9, 12.7 (but one launch and its tensor maps less to call).
static ffa::PaShape prefix_shape(int R, int groups, int Hq, int Hkv, int D, int max_prefix) {
  ffa::PaShape s = ffa::pa_shape(R, groups, max_prefix, Hkv, Hq / Hkv, D);
  const double pairs = (double)R * Hkv * ((Hq / Hkv + 15) / 16);
  const double parts = pairs < 27 ? 16.0 : pairs < 444 ? 444.0 / pairs : 1.0;
  const double read = fmax(pairs * max_prefix * D * 4.0 / 6.5e6, max_prefix / parts * (D > 64 ? 0.0136 : 0.010));
  if (read <= 5.0) s.shares = 0;
  return s;
}

extern "C" size_t ffa_prefix_decode_workspace_size(int R, int groups, int Hq, int Hkv, int D, int max_prefix) {
  if (R <= 0 || groups <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || Hq / Hkv > 128 || D <= 0 || D > 128 ||
      max_prefix < 0)
    return 0;
  const int shares = prefix_shape(R, groups, Hq, Hkv, D, max_prefix).shares;
  return shares ? (size_t)R * Hq * (shares + 1) * (D + 1) * 4 : 0;
}

extern "C" int ffa_prefix_decode(const void* q, const void* k_pages, const void* v_pages, const int* block_table,
                                 const int* ctx_lens, const int* group_starts, const int* prefix_lens, void* out,
                                 float* lse, int dtype, int R, int groups, int Hq, int Hkv, int D, int num_pages,
                                 int page_size, int max_pages_per_req, const int64_t* q_strides,
                                 const int64_t* o_strides, float scale, float softcap, int max_prefix, int max_own,
                                 void* workspace, size_t workspace_bytes, uint32_t* dev_err, void* stream) {
  using namespace ffa;
  if (R == 0) return FFA_OK;
  PaCall c{};
  c.q = q;
  c.k_pages = k_pages;
  c.v_pages = v_pages;
  c.block_table = block_table;
  c.starts = groups ? group_starts : ctx_lens;  // (no group: neither is read)
  c.kv_lens = groups ? prefix_lens : ctx_lens;
  c.lens = ctx_lens;
  c.dtype = dtype;
  c.N = groups ? groups : 1;
  c.T = R;
  c.Hq = Hq;
  c.Hkv = Hkv;
  c.D = D;
  c.num_pages = num_pages;
  c.page_size = page_size;
  c.width = max_pages_per_req;
  c.q_strides = q_strides;
  c.scale = scale;
  c.softcap = softcap;
  c.workspace = workspace;
  c.dev_err = dev_err;
  if (int s = pa_check(c)) return s;
  if (!ctx_lens || !out || !o_strides || groups < 0 || max_prefix < 0 || max_own < 0) return FFA_ERR_INVALID_ARG;
  WdParams p{};
  PaShape shape{};
  if (groups) {
    shape = prefix_shape(R, groups, Hq, Hkv, D, max_prefix);
    p.starts = group_starts;
    p.prefix_lens = prefix_lens;
    p.groups = groups;
    p.whole = shape.shares == 0;
  }
  if (groups && !p.whole) {
    const size_t need = ffa_prefix_decode_workspace_size(R, groups, Hq, Hkv, D, max_prefix);
    if (!workspace || workspace_bytes < need || !aligned16(workspace)) return FFA_ERR_WORKSPACE;
    // [own tokens' O][shares' O][shares' lse][own tokens' lse]
    const int64_t rows = (int64_t)R * Hq;
    float* ws = static_cast<float*>(workspace);
    c.workspace = ws + rows * D;
    if (int s = page_attn(c, shape, stream)) return s;
    p.shares = shape.shares;
    p.chunk = shape.chunk;
    p.o_part = ws + rows * D;
    p.lse_part = p.o_part + rows * shape.shares * D;
    p.o_own = ws;
    p.lse_own = ws + rows * (D + (int64_t)shape.shares * (D + 1));
  }
  p.q = q;
  p.q_sr = q_strides[0];
  p.q_sh = q_strides[1];
  p.kp = k_pages;
  p.vp = v_pages;
  p.block_table = block_table;
  p.bt_stride = max_pages_per_req;
  p.ctx_lens = ctx_lens;
  p.num_pages = num_pages;
  p.max_ctx = max_pages_per_req * page_size;
  p.out = out;
  p.o_sr = o_strides[0];
  p.o_sh = o_strides[1];
  p.lse = lse;
  p.R = R;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.D = D;
  p.page_size = page_size;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.use_softcap = softcap > 0.f;
  p.sc_pre = p.use_softcap ? scale / softcap : 0.f;
  p.sc_post = p.use_softcap ? softcap * 1.4426950408889634f : 0.f;
  softcap_poly_coeffs(p.sc_pre, p.sc_poly);
  p.err = dev_err;
  int64_t visible = max_own > 0 ? max_own : p.max_ctx;
  if (p.whole) visible += max_prefix;
  if (visible > p.max_ctx) visible = p.max_ctx;
  return window_decode<true>(p, dtype, visible, shape, static_cast<cudaStream_t>(stream));
}

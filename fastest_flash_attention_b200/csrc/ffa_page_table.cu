// Block tables and slot maps of a paged cache, built on the GPU from request
// lengths: pages taken from a ring of free ones for the new tokens of a batch
// (with each token's slot and position), and the pages of finished requests
// put back behind the ring's last.  No value visits the host, so a serving
// step can be captured in a graph.
//
//   assign:   need_r = ceil((len_r + n_r) / ps) - ceil(len_r / ps)
//             page k of them = ring[(head + sum_{s<r} need_s + k) mod P]
//   release:  page k of row r -> ring[(head + count + sum_{s<r} give_s + k) mod P]
//   share:    rows that are empty get the first pages of one that holds them
//
// The first two are a scan over the requests and then independent work for every token
// and page.  One cluster of CTAs does it in one launch: every CTA scans all
// lengths into its own shared memory (a few KB, cheaper than a second launch),
// the cluster meets once all inputs have been read and checked (results may be
// written over the inputs, and an invalid call changes nothing), then the CTAs
// share tokens and pages, each of which finds its row by bisection.
// Bound by latencies in sequence: launch, lengths, scan, meeting, table entry.
// Device time: 64 requests of one token 6.0 us, 131 072 prompt tokens of 1024
// requests 12.9 (35.5 by bisection alone with 8 CTAs of 512 threads), 33 000 pages
// of 64 requests given back 6.3 (12.4).
#include <cooperative_groups.h>

#include "ffa_common.cuh"
#include "ffa_host.h"

namespace ffa {

namespace cg = cooperative_groups;

enum : uint32_t { SITE_ASSIGN = 0x3E4, SITE_RELEASE = 0x3E5, SITE_SHARE = 0x3E7 };

constexpr int PT_THREADS = 1024;
constexpr int PT_ILP = 4;  // items that a thread works on at a time
constexpr int PT_MAX_ROWS = 16384;  // three ints a row in shared memory

struct PtParams {
  int* table;  // [R, width]
  int width;
  const int* lens;
  const int* counts;    // assign: new tokens [R]; release: tokens whose pages stay taken [R], or nullptr
  const uint8_t* done;  // release: rows whose pages are given back [R]
  int* ring;            // [P]
  const int* state;     // {head, count}
  int *slots, *positions, *starts;
  int *lens_out, *state_out;
  int R, P, page_size, max_tokens;
  int vec;          // slots and positions are 16-byte aligned
  uint32_t ps_mul;  // division by page_size: floor(x / d) = x * mul >> shift with mul = floor(2^shift / d) + 1,
  int ps_shift;     // shift = 31 + k, 2^k >= d, exact below 2^31
  uint32_t* err;
};

// Rows that own items i[k] (the last ones with first[row] <= i[k]) for the lanes
// of a warp whose items all lie in [from, to]: the warp finds those two's rows by
// probing 32 places at a time, each lane its own between them by bisection (of N
// items side by side, without branches: their loads overlap).
__device__ __forceinline__ int pt_row(const int* first, int R, int i, int lane) {
  int lo = 0;
  for (int len = R; len > 1;) {
    const int step = (len + 31) / 32, at = lo + lane * step;
    const uint32_t below = __ballot_sync(0xffffffffu, lane * step < len && first[min(at, R - 1)] <= i);
    const int skip = max(__popc(below) - 1, 0) * step;
    lo += skip;
    len = min(step, len - skip);
  }
  return lo;
}
template <int N>
__device__ __forceinline__ void pt_rows(const int* first, int R, int from, int to, const int* i, int* row, int lane) {
  const int lo = pt_row(first, R, from, lane), hi = from == to ? lo : pt_row(first, R, to, lane);
#pragma unroll
  for (int k = 0; k < N; ++k) row[k] = lo;
  if (hi == lo) return;
  for (int step = 1 << (31 - __clz(hi - lo)); step > 0; step >>= 1) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int next = row[k] + step;
      const bool up = (next <= hi) & (first[min(next, hi)] <= i[k]);
      row[k] = up ? next : row[k];
    }
  }
}

template <bool ASSIGN>
__global__ void __launch_bounds__(PT_THREADS) ffa_page_table_kernel(const PtParams p) {
  extern __shared__ int smem[];
  int* page0 = smem;           // [R] pages of the rows before
  int* own = smem + p.R;       // [R] assign: the row's length; release: its first page index to give back
  int* tok0 = smem + 2 * p.R;  // [R] (assign) tokens of the rows before
  auto div_ps = [&](int x) { return (int)(((uint64_t)(uint32_t)x * p.ps_mul) >> p.ps_shift); };
  auto ceil_ps = [&](int x) { return x > 0 ? div_ps(x - 1) + 1 : 0; };
  auto base = [&](int r) { return ASSIGN ? ceil_ps(own[r]) : own[r]; };
  __shared__ long long warp_sum[2][32];
  __shared__ int bad_flag;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, threads = blockDim.x;
  const int ctas = gridDim.x, cta = blockIdx.x;  // one cluster
  if (tid == 0) bad_flag = 0;
  if (tid < 64) warp_sum[tid / 32][lane] = 0;  // (of warps that are not there)
  const int head = p.state[0], count = p.state[1];
  bool bad = head < 0 || head >= p.P || count < 0 || count > p.P;
  const long long room = (long long)p.width * p.page_size;
  // exclusive sums over the rows, a row for each thread at a time (64-bit: the
  // sum of any 32-bit lengths fits; only sums found small enough are used)
  long long pages64 = 0, toks64 = 0;  // of the rows so far, in every thread
  for (int r0 = 0; r0 < p.R; r0 += threads) {
    const int r = r0 + tid;
    long long pages = 0, toks = 0;
    int first = 0;
    if (r < p.R) {
      const long long len = p.lens[r];
      if (len < 0 || len > room) {
        bad = true;
      } else if (ASSIGN) {
        const long long n = p.counts[r];
        if (n < 0 || len + n > room) {
          bad = true;
        } else {
          first = (int)len;
          const int had = ceil_ps(first), i = div_ps(first);
          pages = ceil_ps((int)(len + n)) - had;
          toks = n;
          // tokens that go on in a page begun earlier
          if (n && i < had) bad |= (unsigned)p.table[(int64_t)r * p.width + i] >= (unsigned)p.P;
        }
      } else if (p.done[r]) {
        const long long keep = p.counts ? p.counts[r] : 0;
        if (keep < 0) {
          bad = true;
        } else {
          first = ceil_ps((int)keep);
          pages = ceil_ps((int)len) - first;
          if (pages < 0) pages = 0;
        }
      }
    }
    long long ip = pages, it = toks;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long a = __shfl_up_sync(0xffffffffu, ip, off), b = ASSIGN ? __shfl_up_sync(0xffffffffu, it, off) : 0;
      if (lane >= off) {
        ip += a;
        it += b;
      }
    }
    __syncthreads();  // (the sums of the rows before have been read)
    if (lane == 31) {
      warp_sum[0][warp] = ip;
      warp_sum[1][warp] = it;
    }
    __syncthreads();
    // every warp sums up the warps' totals
    long long wp = warp_sum[0][lane], wt = warp_sum[1][lane];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long a = __shfl_up_sync(0xffffffffu, wp, off), b = ASSIGN ? __shfl_up_sync(0xffffffffu, wt, off) : 0;
      if (lane >= off) {
        wp += a;
        wt += b;
      }
    }
    const long long bp = warp ? __shfl_sync(0xffffffffu, wp, warp - 1) : 0;
    const long long bt = ASSIGN && warp ? __shfl_sync(0xffffffffu, wt, warp - 1) : 0;
    if (r < p.R) {
      page0[r] = (int)(pages64 + bp + ip - pages);
      own[r] = first;
      if (ASSIGN) tok0[r] = (int)(toks64 + bt + it - toks);
    }
    pages64 += __shfl_sync(0xffffffffu, wp, 31);
    toks64 += ASSIGN ? __shfl_sync(0xffffffffu, wt, 31) : 0;
  }
  if (ASSIGN) bad |= pages64 > count || toks64 > p.max_tokens;
  else bad |= pages64 + count > p.P;
  // (the row sums are valid below 2^31 only; every thread knows both totals)
  const int pages = pages64 <= p.P ? (int)pages64 : 0, toks = (int)toks64;
  bad |= pages64 > p.P;
  const int step = ctas * threads, i0 = cta * threads + tid;
  // (places of pages and tokens are counted unsigned: up to 2^31, a step past it)
  auto least = [](unsigned a, int b) { return (int)min(a, (unsigned)b); };
  const bool sums_ok = __syncthreads_or(bad) == 0;
  // the page ids concerned, each checked by one thread of the cluster; `ids`
  // (release): the first PT_ILP of this thread
  int ids[PT_ILP];
  auto entry = [&](int j, int r) { return p.table + (int64_t)r * p.width + base(r) + j - page0[r]; };
  auto place = [&](int j) {  // j-th place behind the ring's first free page (assign) or last (release)
    const long long at = (long long)head + j + (ASSIGN ? 0 : count);
    return p.ring + (at >= p.P ? at - p.P : at);
  };
  // (a warp's PT_ILP pieces of 32 items follow one another)
  const unsigned w0 = (cta * threads / 32 + warp) * 32 * PT_ILP;
  auto items = [&](unsigned j0, int n, int* j) {  // this lane's of the warp's items from j0 on, all below n
#pragma unroll
    for (int k = 0; k < PT_ILP; ++k) j[k] = least(j0 + 32 * k + lane, n - 1);
  };
  if (sums_ok) {
    for (unsigned j0 = w0; j0 < (unsigned)pages; j0 += PT_ILP * step) {
      int j[PT_ILP], row[PT_ILP], id[PT_ILP];
      items(j0, pages, j);
      if (!ASSIGN) pt_rows<PT_ILP>(page0, p.R, (int)j0, least(j0 + 32 * PT_ILP, pages) - 1, j, row, lane);
#pragma unroll
      for (int k = 0; k < PT_ILP; ++k) id[k] = ASSIGN ? *place(j[k]) : *entry(j[k], row[k]);
#pragma unroll
      for (int k = 0; k < PT_ILP; ++k) {
        bad |= (unsigned)id[k] >= (unsigned)p.P;
        if (j0 == w0) ids[k] = id[k];
      }
    }
  }
  if (bad) bad_flag = 1;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  const bool ok = !__syncthreads_or(tid < ctas && *cluster.map_shared_rank(&bad_flag, tid));

  // rows: where results are written over the inputs, each row is read and
  // written by one thread
  for (int r = i0; r < p.R; r += step) {
    const int len = p.lens[r];
    if (ASSIGN) {
      p.starts[r] = ok ? tok0[r] : 0;
      p.lens_out[r] = ok ? len + p.counts[r] : len;
    } else {
      p.lens_out[r] = ok && p.done[r] ? 0 : len;
    }
  }
  if (i0 == 0) {
    if (ASSIGN) p.starts[p.R] = ok ? toks : 0;
    if (ASSIGN) {
      const long long at = (long long)head + pages;
      p.state_out[0] = ok ? (int)(at >= p.P ? at - p.P : at) : head;
      p.state_out[1] = ok ? count - pages : count;
    } else {
      p.state_out[0] = head;
      p.state_out[1] = ok ? count + pages : count;
    }
    if (!ok && p.err) atomicCAS(p.err, 0u, ASSIGN ? SITE_ASSIGN : SITE_RELEASE);
  }
  if (ok) {
    for (unsigned j0 = w0; j0 < (unsigned)pages; j0 += PT_ILP * step) {
      int j[PT_ILP], row[PT_ILP];
      items(j0, pages, j);
      if (ASSIGN || j0 > w0) pt_rows<PT_ILP>(page0, p.R, (int)j0, least(j0 + 32 * PT_ILP, pages) - 1, j, row, lane);
#pragma unroll
      for (int k = 0; k < PT_ILP; ++k) {
        if (j0 > w0) ids[k] = ASSIGN ? *place(j[k]) : *entry(j[k], row[k]);
        if (j0 + 32 * k + lane >= (unsigned)pages) continue;
        if (ASSIGN) *entry(j[k], row[k]) = ids[k];
        else *place(j[k]) = ids[k];
      }
    }
  }
  if (ASSIGN) {
    // PT_ILP tokens in a row for each thread: one store
    for (unsigned tw = w0; tw < (unsigned)p.max_tokens; tw += PT_ILP * step) {
      const unsigned t0 = tw + PT_ILP * lane;
      int pos[PT_ILP], slot[PT_ILP];
#pragma unroll
      for (int k = 0; k < PT_ILP; ++k) {
        pos[k] = 0;
        slot[k] = -1;
      }
      if (ok && tw < (unsigned)toks) {
        int t[PT_ILP], row[PT_ILP];
#pragma unroll
        for (int k = 0; k < PT_ILP; ++k) t[k] = least(t0 + k, toks - 1);
        pt_rows<PT_ILP>(tok0, p.R, (int)tw, least(tw + 32 * PT_ILP, toks) - 1, t, row, lane);
#pragma unroll
        for (int k = 0; k < PT_ILP; ++k) {
          const int r = row[k], x = own[r] + t[k] - tok0[r];
          const int i = div_ps(x), n = i - base(r);
          const int page = *(n >= 0 ? place(page0[r] + n) : p.table + (int64_t)r * p.width + i);
          if (t0 + k < (unsigned)toks) {
            pos[k] = x;
            slot[k] = page * p.page_size + x - i * p.page_size;
          }
        }
      }
      if (p.vec && t0 + PT_ILP <= (unsigned)p.max_tokens) {
        *reinterpret_cast<int4*>(p.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
        *reinterpret_cast<int4*>(p.positions + t0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
      } else {
#pragma unroll
        for (int k = 0; k < PT_ILP; ++k)
          if (t0 + k < (unsigned)p.max_tokens) {
            p.slots[t0 + k] = slot[k];
            p.positions[t0 + k] = pos[k];
          }
      }
    }
  }
  cluster.sync();  // no CTA leaves while another reads its flag
}

struct PtShare {
  int* table;  // [R, width]
  int* lens;   // [R]
  int width, owner, pages, tokens, R, P;
  uint32_t* err;
  uint32_t rows[PT_MAX_ROWS / 32];  // a bit for each row that gets the owner's first pages
};

// Every CTA checks all that is asked (a few KB read), the cluster meets, since what
// was read is written next, and the warps share pieces of 256 entries of the rows.
// Device time: 3 rows of 9 pages 3.0 us, 255 rows of 512 pages 4.8, of 2048 7.0 (as two
// copies for each row, which checked nothing, 255 rows were 510 launches).
__global__ void __launch_bounds__(PT_THREADS) ffa_page_share_kernel(const __grid_constant__ PtShare p) {
  constexpr int PIECE = 256;
  const int tid = threadIdx.x, lane = tid % 32, threads = blockDim.x;
  const int* own = p.table + (int64_t)p.owner * p.width;
  auto asked = [&](int r) { return (p.rows[r / 32] >> (r % 32)) & 1u; };
  bool bad = p.lens[p.owner] < p.tokens;
  for (int r = tid; r < p.R; r += threads)
    if (asked(r)) bad |= p.lens[r] != 0;
  for (int i = tid; i < p.pages; i += threads) bad |= (unsigned)own[i] >= (unsigned)p.P;
  const bool ok = !__syncthreads_or(bad);
  cg::this_cluster().sync();
  if (!ok) {
    if (blockIdx.x == 0 && tid == 0 && p.err) atomicCAS(p.err, 0u, SITE_SHARE);
    return;
  }
  const int pieces = (p.pages + PIECE - 1) / PIECE, warps = gridDim.x * (threads / 32);
  int r = 0, piece = blockIdx.x * (threads / 32) + tid / 32;
  for (;; piece += warps) {
    r += piece / pieces;
    piece %= pieces;
    if (r >= p.R) return;
    if (!asked(r)) continue;
    int* row = p.table + (int64_t)r * p.width;
#pragma unroll
    for (int k = 0; k < PIECE; k += 32) {
      const int i = piece * PIECE + k + lane;
      if (i < p.pages) row[i] = own[i];
    }
    if (piece == 0 && lane == 0) p.lens[r] = p.tokens;
  }
}

// CTAs of the cluster, and threads of a CTA, for so many rows, tokens or table entries.
static void pt_shape(int64_t items, unsigned& ctas, unsigned& threads) {
  ctas = items <= PT_THREADS ? 1 : items <= 8 * PT_THREADS ? 4 : 16;
  threads = items >= PT_THREADS ? PT_THREADS : items < 64 ? 64 : (unsigned)(items + 31) / 32 * 32;
}

// One cluster for so many items; `wide`: the devices where the kernel may have more than 8 CTAs.
template <typename Params>
static int launch_cluster(void (*kern)(Params), const Params& p, int64_t items, size_t smem,
                          std::atomic<uint64_t>& wide, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  unsigned ctas, threads;
  pt_shape(items, ctas, threads);
  cfg.gridDim = dim3(ctas);
  if (cfg.gridDim.x > 8) {  // clusters past 8 CTAs are opt-in
    int dev = 0;
    if (int s = cuda_status(cudaGetDevice(&dev))) return s;
    const uint64_t bit = dev < 64 ? (1ull << dev) : 0ull;
    if (!bit || !(wide.load(std::memory_order_acquire) & bit)) {
      if (int s = cuda_status(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1))) return s;
      if (bit) wide.fetch_or(bit, std::memory_order_acq_rel);
    }
  }
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cfg.gridDim.x;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, p));
}

template <bool ASSIGN>
static int launch_page_table(PtParams& p, int64_t items, cudaStream_t st) {
  int k = 0;
  while ((1ll << k) < p.page_size) ++k;
  p.ps_shift = 31 + k;
  p.ps_mul = (uint32_t)((1ull << p.ps_shift) / (unsigned)p.page_size + 1);
  static std::atomic<uint64_t> done{0}, wide{0};
  if (int s = smem_attr_once(ffa_page_table_kernel<ASSIGN>, 3 * 4 * PT_MAX_ROWS, done)) return s;
  return launch_cluster<const PtParams>(ffa_page_table_kernel<ASSIGN>, p, items, (ASSIGN ? 3 : 2) * 4 * (size_t)p.R,
                                        wide, st);
}

// Sizes that all entry points take.  Slots and table entries are 32-bit.
static int pt_check(int R, int width, int P, int page_size) {
  if (R < 0 || width <= 0 || P <= 0 || page_size <= 0) return FFA_ERR_INVALID_ARG;
  if (R > PT_MAX_ROWS || (int64_t)P * page_size > 0x7fffffffLL || (int64_t)width * page_size > 0x7fffffffLL)
    return FFA_ERR_UNSUPPORTED;
  return FFA_OK;
}

}  // namespace ffa

extern "C" int ffa_assign_slots(int* block_table, int width, const int* ctx_lens, const int* new_lens,
                                const int* free_pages, const int* free_state, int* slots, int* positions, int* starts,
                                int* ctx_lens_out, int* free_state_out, int R, int num_pages, int page_size,
                                int max_tokens, uint32_t* dev_err, void* stream) {
  using namespace ffa;
  if (int s = pt_check(R, width, num_pages, page_size)) return s;
  if (max_tokens < 0) return FFA_ERR_INVALID_ARG;
  if (!free_pages || !free_state || !starts || !free_state_out || (max_tokens > 0 && (!slots || !positions)) ||
      (R > 0 && (!block_table || !ctx_lens || !new_lens || !ctx_lens_out)))
    return FFA_ERR_INVALID_ARG;
  PtParams p{};
  p.table = block_table;
  p.width = width;
  p.lens = ctx_lens;
  p.counts = new_lens;
  p.ring = const_cast<int*>(free_pages);  // (only read)
  p.state = free_state;
  p.slots = slots;
  p.positions = positions;
  p.starts = starts;
  p.lens_out = ctx_lens_out;
  p.state_out = free_state_out;
  p.R = R;
  p.P = num_pages;
  p.page_size = page_size;
  p.max_tokens = max_tokens;
  p.vec = aligned16(slots) && aligned16(positions);
  p.err = dev_err;
  return launch_page_table<true>(p, max_tokens > R ? max_tokens : R, static_cast<cudaStream_t>(stream));
}

extern "C" int ffa_release_pages(const int* block_table, int width, const int* ctx_lens, const uint8_t* done,
                                 const int* keep, int* free_pages, const int* free_state, int* ctx_lens_out,
                                 int* free_state_out, int R, int num_pages, int page_size, uint32_t* dev_err,
                                 void* stream) {
  using namespace ffa;
  if (int s = pt_check(R, width, num_pages, page_size)) return s;
  if (!free_pages || !free_state || !free_state_out ||
      (R > 0 && (!block_table || !ctx_lens || !done || !ctx_lens_out)))
    return FFA_ERR_INVALID_ARG;
  PtParams p{};
  p.table = const_cast<int*>(block_table);  // (only read)
  p.width = width;
  p.lens = ctx_lens;
  p.counts = keep;
  p.done = done;
  p.ring = free_pages;
  p.state = free_state;
  p.lens_out = ctx_lens_out;
  p.state_out = free_state_out;
  p.R = R;
  p.P = num_pages;
  p.page_size = page_size;
  p.err = dev_err;
  return launch_page_table<false>(p, (int64_t)R * width, static_cast<cudaStream_t>(stream));
}

extern "C" int ffa_share_pages(int* block_table, int width, int* ctx_lens, int owner, const int* rows, int num_rows,
                               int R, int num_pages, int page_size, int tokens, uint32_t* dev_err, void* stream) {
  using namespace ffa;
  if (int s = pt_check(R, width, num_pages, page_size)) return s;
  if (!block_table || !ctx_lens || (num_rows > 0 && !rows) || num_rows < 0 || owner < 0 || owner >= R || tokens <= 0 ||
      tokens % page_size || tokens / page_size > width)
    return FFA_ERR_INVALID_ARG;
  PtShare p{};
  for (int i = 0; i < num_rows; ++i) {
    const int r = rows[i];
    if (r < 0 || r >= R || r == owner || ((p.rows[r / 32] >> (r % 32)) & 1u)) return FFA_ERR_INVALID_ARG;
    p.rows[r / 32] |= 1u << (r % 32);
  }
  if (num_rows == 0) return FFA_OK;
  p.table = block_table;
  p.lens = ctx_lens;
  p.width = width;
  p.owner = owner;
  p.pages = tokens / page_size;
  p.tokens = tokens;
  p.R = R;
  p.P = num_pages;
  p.err = dev_err;
  static std::atomic<uint64_t> wide{0};
  return launch_cluster<const PtShare>(ffa_page_share_kernel, p, (int64_t)num_rows * p.pages, 0, wide,
                                       static_cast<cudaStream_t>(stream));
}

// Block tables and slot maps of a paged cache, built on the GPU from request
// lengths: pages taken from a ring of free ones for the new tokens of a batch
// (with each token's slot and position), and the pages of finished requests
// put back behind the ring's last.  No value visits the host, so a serving
// step can be captured in a graph.
//
//   assign:   need_r = ceil((len_r + n_r) / ps) - ceil(len_r / ps)
//             page k of them = ring[(head + sum_{s<r} need_s + k) mod P]
//   release:  page k of row r -> ring[(head + count + sum_{s<r} give_s + k) mod P]
//
// Both are a scan over the requests and then independent work for every token
// and page.  One cluster of CTAs does it in one launch: every CTA scans all
// lengths into its own shared memory (a few KB, cheaper than a second launch),
// the cluster meets once all inputs have been read and checked (results may be
// written over the inputs, and an invalid call changes nothing), then the CTAs
// share tokens and pages, each of which finds its row by bisection.
// Bound by latencies in sequence: launch, lengths, scan, meeting, table entry.
#include <cooperative_groups.h>

#include "ffa_common.cuh"
#include "ffa_host.h"

namespace ffa {

namespace cg = cooperative_groups;

enum : uint32_t { SITE_ASSIGN = 0x3E4, SITE_RELEASE = 0x3E5 };

constexpr int PT_THREADS = 512;
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
  uint32_t* err;
};

// Row that owns item i: the last one with first[row] <= i.
__device__ __forceinline__ int pt_row(const int* first, int R, int i) {
  int lo = 0, hi = R;  // first[lo] <= i < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <bool ASSIGN>
__global__ void __launch_bounds__(PT_THREADS) ffa_page_table_kernel(const PtParams p) {
  extern __shared__ int smem[];
  int* page0 = smem;           // [R] pages of the rows before
  int* own = smem + p.R;       // [R] assign: the row's length; release: its first page index to give back
  int* tok0 = smem + 2 * p.R;  // [R] (assign) tokens of the rows before
  auto base = [&](int r) { return ASSIGN ? (own[r] + p.page_size - 1) / p.page_size : own[r]; };
  __shared__ long long warp_sum[2][PT_THREADS / 32];
  __shared__ long long carry[2];
  __shared__ int bad_flag, any_bad;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int ctas = gridDim.x, cta = blockIdx.x;  // one cluster
  if (tid == 0) {
    carry[0] = carry[1] = 0;
    bad_flag = 0;
  }
  const int head = p.state[0], count = p.state[1];
  bool bad = head < 0 || head >= p.P || count < 0 || count > p.P;
  const long long room = (long long)p.width * p.page_size;
  __syncthreads();
  // exclusive sums over the rows, PT_THREADS of them at a time (64-bit: the
  // sum of any 32-bit lengths fits; only sums found small enough are used)
  for (int r0 = 0; r0 < p.R; r0 += PT_THREADS) {
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
          pages = (len + n + p.page_size - 1) / p.page_size - (len + p.page_size - 1) / p.page_size;
          toks = n;
          // tokens that go on in a page begun earlier
          if (n && len % p.page_size)
            bad |= (unsigned)p.table[(int64_t)r * p.width + len / p.page_size] >= (unsigned)p.P;
        }
      } else if (p.done[r]) {
        const long long keep = p.counts ? p.counts[r] : 0;
        if (keep < 0) {
          bad = true;
        } else {
          first = (int)((keep + p.page_size - 1) / p.page_size);
          pages = (len + p.page_size - 1) / p.page_size - first;
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
    if (lane == 31) {
      warp_sum[0][warp] = ip;
      warp_sum[1][warp] = it;
    }
    __syncthreads();
    long long bp = carry[0], bt = carry[1];
    for (int w = 0; w < warp; ++w) {
      bp += warp_sum[0][w];
      bt += warp_sum[1][w];
    }
    if (r < p.R) {
      page0[r] = (int)(bp + ip - pages);
      own[r] = first;
      if (ASSIGN) tok0[r] = (int)(bt + it - toks);
    }
    __syncthreads();
    if (tid == PT_THREADS - 1) {
      carry[0] = bp + ip;
      carry[1] = bt + it;
    }
    __syncthreads();
  }
  const long long pages64 = carry[0], toks64 = carry[1];
  if (ASSIGN) bad |= pages64 > count || toks64 > p.max_tokens;
  else bad |= pages64 + count > p.P;
  // (the row sums are valid below 2^31 only; every thread knows both totals)
  const int pages = pages64 <= p.P ? (int)pages64 : 0, toks = (int)toks64;
  bad |= pages64 > p.P;
  const int step = ctas * PT_THREADS, i0 = cta * PT_THREADS + tid;
  const bool sums_ok = __syncthreads_or(bad) == 0;
  // the page ids concerned, each checked by one thread of the cluster
  if (sums_ok) {
    for (int j = i0; j < pages; j += step) {
      int id;
      if (ASSIGN) {
        long long at = (long long)head + j;
        id = p.ring[at >= p.P ? at - p.P : at];
      } else {
        const int r = pt_row(page0, p.R, j);
        id = p.table[(int64_t)r * p.width + base(r) + j - page0[r]];
      }
      bad |= (unsigned)id >= (unsigned)p.P;
    }
  }
  if (bad) bad_flag = 1;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.sync();
  if (tid == 0) {
    any_bad = 0;
    for (int c = 0; c < ctas; ++c) any_bad |= *cluster.map_shared_rank(&bad_flag, c);
  }
  __syncthreads();
  const bool ok = !any_bad;

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
    for (int j = i0; j < pages; j += step) {
      const int r = pt_row(page0, p.R, j);
      int* entry = p.table + (int64_t)r * p.width + base(r) + j - page0[r];
      long long at = (long long)head + j + (ASSIGN ? 0 : count);
      if (at >= p.P) at -= p.P;
      if (ASSIGN) *entry = p.ring[at];
      else p.ring[at] = *entry;
    }
  }
  if (ASSIGN) {
    for (int t = i0; t < p.max_tokens; t += step) {
      int slot = -1, pos = 0;
      if (ok && t < toks) {
        const int r = pt_row(tok0, p.R, t);
        pos = own[r] + t - tok0[r];
        const int i = pos / p.page_size, k = i - base(r);
        int page;
        if (k >= 0) {
          long long at = (long long)head + page0[r] + k;
          page = p.ring[at >= p.P ? at - p.P : at];
        } else {
          page = p.table[(int64_t)r * p.width + i];
        }
        slot = page * p.page_size + pos - i * p.page_size;
      }
      p.slots[t] = slot;
      p.positions[t] = pos;
    }
  }
  cluster.sync();  // no CTA leaves while another reads its flag
}

template <bool ASSIGN>
static int launch_page_table(const PtParams& p, int64_t items, cudaStream_t st) {
  auto kern = ffa_page_table_kernel<ASSIGN>;
  static std::atomic<uint64_t> done{0};
  if (int s = smem_attr_once(kern, 3 * 4 * PT_MAX_ROWS, done)) return s;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(items > 4 * PT_THREADS ? 8 : 1);
  cfg.blockDim = dim3(PT_THREADS);
  cfg.dynamicSmemBytes = (ASSIGN ? 3 : 2) * 4 * (size_t)p.R;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cfg.gridDim.x;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, kern, p));
}

// Sizes that both entry points take.  Slots and table entries are 32-bit.
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

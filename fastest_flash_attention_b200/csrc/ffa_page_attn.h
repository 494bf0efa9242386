// Attention of many query rows over a paged cache (ffa_page_attn.cu): the call
// that ffa_paged_prefill and the first launch of ffa_prefix_decode share.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace ffa {

// Request boundaries or a prefix length that mean nothing (not an expired wait).
enum : uint32_t { SITE_PA_BAD_STARTS = 0x3E6 };

constexpr int PA_MAX_SHARES = 64;

#ifdef __CUDACC__
// Last i in [0, n) with a[i] <= x in ascending a (0 if there is none), by one warp:
// 32 places at a time.
__device__ __forceinline__ int warp_search(const int* a, int n, int x, int lane) {
  int lo = 0;
  for (int len = n; len > 1;) {
    const int step = (len + 31) / 32, at = lo + lane * step;
    const uint32_t below = __ballot_sync(0xffffffffu, lane * step < len && a[at < n ? at : n - 1] <= x);
    const int skip = (below ? 31 - __clz(below) : 0) * step;
    lo += skip;
    len = step < len - skip ? step : len - skip;
  }
  return lo;
}

// Shares that hold `keys` tokens (one or more; no sum that could pass 2^31).
__device__ __forceinline__ int share_count(int keys, int chunk, int shares) {
  return min(shares, (keys - 1) / chunk + 1);
}
#endif

struct PaCall {
  const void *q, *k_pages, *v_pages;
  const int* block_table;
  const int* starts;   // [N + 1]
  const int* kv_lens;  // [N]
  const int* lens;     // prefix form: [R] context lengths
  void* out;           // causal form
  float* lse;
  int dtype, N, T, Hq, Hkv, D, num_pages, page_size, width;
  const int64_t *q_strides, *o_strides;  // {token, head}
  float scale, softcap;
  bool causal;
  void* workspace;
  uint32_t* dev_err;
};

// Query tiles per CTA and rows in use of each (128, or 32), and the shares that a
// context is cut into: share s takes tokens [s * chunk, (s + 1) * chunk), the last
// one all that follow.  `time`: estimated (us); `idle`: the part of its CTAs'
// slots that is empty meanwhile.
struct PaShape {
  int nqt, rows, shares, chunk;
  float time, idle;
};

PaShape pa_shape(int64_t tokens, int64_t segments, int64_t kv, int Hkv, int G, int D);
int pa_check(const PaCall& c);
size_t pa_workspace(int64_t T, int Hq, int D, int shares);
int page_attn(const PaCall& c, const PaShape& shape, void* stream);

}  // namespace ffa

// Paged KV-cache append: one warp per (token, kv head) copies a D-element
// row of K and of V into its page slot with 16-byte vector stores.
// Replaces the per-token Python loop of ops/kv_cache.py:192-204.
#include "ffa_common.cuh"
#include "ffa_host.h"

namespace ffa {

__global__ void ffa_paged_append_kernel(const uint16_t* __restrict__ k_new, const uint16_t* __restrict__ v_new,
                                        uint16_t* __restrict__ k_pages, uint16_t* __restrict__ v_pages,
                                        const int* __restrict__ slots, int n_tokens, int Hkv, int D, int page_size,
                                        int num_pages, int64_t s_head, int64_t s_tok) {
  const int w = (blockIdx.x * blockDim.x + threadIdx.x) / 32;
  const int lane = threadIdx.x % 32;
  if (w >= n_tokens * Hkv) return;
  const int tok = w / Hkv, h = w % Hkv;
  const int slot = slots[tok];
  const int page = slot / page_size, off = slot % page_size;
  if (slot < 0 || page >= num_pages) return;  // rejected on the host; never write outside the pool
  const int64_t dst = (((int64_t)page * Hkv + h) * page_size + off) * D;
  const int64_t src = (int64_t)h * s_head + (int64_t)tok * s_tok;
  for (int d = lane * 8; d < D; d += 256) {
    *reinterpret_cast<uint4*>(k_pages + dst + d) = *reinterpret_cast<const uint4*>(k_new + src + d);
    *reinterpret_cast<uint4*>(v_pages + dst + d) = *reinterpret_cast<const uint4*>(v_new + src + d);
  }
}

}  // namespace ffa

extern "C" int ffa_paged_append(const void* k_new, const void* v_new, void* k_pages, void* v_pages,
                                const int* slots, int dtype, int n_tokens, int Hkv, int D, int page_size,
                                int num_pages, const int64_t* new_strides, void* stream) {
  using namespace ffa;
  if (!k_new || !v_new || !k_pages || !v_pages || !slots || !new_strides) return FFA_ERR_INVALID_ARG;
  if (n_tokens < 0 || Hkv <= 0 || D <= 0 || page_size <= 0 || num_pages <= 0) return FFA_ERR_INVALID_ARG;
  if (dtype != FFA_DTYPE_BF16 && dtype != FFA_DTYPE_F16) return FFA_ERR_UNSUPPORTED;
  if (D % 8 || new_strides[0] % 8 || new_strides[1] % 8 || !aligned16(k_new) || !aligned16(v_new) ||
      !aligned16(k_pages) || !aligned16(v_pages))
    return FFA_ERR_INVALID_ARG;
  if (n_tokens == 0) return FFA_OK;
  const int warps = n_tokens * Hkv;
  ffa_paged_append_kernel<<<(warps * 32 + 255) / 256, 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const uint16_t*>(k_new), static_cast<const uint16_t*>(v_new), static_cast<uint16_t*>(k_pages),
      static_cast<uint16_t*>(v_pages), slots, n_tokens, Hkv, D, page_size, num_pages, new_strides[0],
      new_strides[1]);
  return launch_status();
}

namespace ffa {
// ---------------------------------------------------------------------------
// Copies inside the page pools: whole pages (a fork's last page, a
// defragmentation) and single token rows (a sequence compacted to its first
// tokens and its window).  Both move bytes and compute nothing: the floor is
// one read and one write of what moves, at the rate of a plain copy.
// Sources and destinations are disjoint (the caller's contract), so no order
// between the copies is needed.
// ---------------------------------------------------------------------------
// Invalid ids (not expired waits): a page id outside [0, num_pages), a slot
// outside [0, num_pages * page_size).  The copy of that entry is left out.
enum : uint32_t { SITE_COPY_BAD_ID = 0x3E2 };

constexpr int COPY_THREADS = 256;
constexpr int COPY_VECS = 4;  // vectors each thread has in flight

// One CTA copies COPY_THREADS * COPY_VECS vectors of one page of one pool.
template <typename V>
__global__ void __launch_bounds__(COPY_THREADS)
    ffa_page_copy_kernel(uint8_t* k_pages, uint8_t* v_pages, const int* __restrict__ src,
                         const int* __restrict__ dst, int num_pages, int64_t vecs_per_page, int ctas_per_page,
                         uint32_t* err) {
  const int64_t unit = blockIdx.x / ctas_per_page;
  const int part = blockIdx.x % ctas_per_page;
  const int s = src[unit], d = dst[unit];
  if ((unsigned)s >= (unsigned)num_pages || (unsigned)d >= (unsigned)num_pages) {
    if (threadIdx.x == 0 && err) atomicCAS(err, 0u, SITE_COPY_BAD_ID);
    return;
  }
  V* pool = reinterpret_cast<V*>(blockIdx.y ? v_pages : k_pages);
  const V* from = pool + (int64_t)s * vecs_per_page;
  V* to = pool + (int64_t)d * vecs_per_page;
  const int64_t v0 = (int64_t)part * (COPY_THREADS * COPY_VECS) + threadIdx.x;
  V x[COPY_VECS];
#pragma unroll
  for (int i = 0; i < COPY_VECS; ++i)
    if (v0 + i * COPY_THREADS < vecs_per_page) x[i] = from[v0 + i * COPY_THREADS];
#pragma unroll
  for (int i = 0; i < COPY_VECS; ++i)
    if (v0 + i * COPY_THREADS < vecs_per_page) to[v0 + i * COPY_THREADS] = x[i];
}

// One thread moves one vector of a token's row for every kv head, COPY_VECS
// heads in flight at a time: the two slots are read and divided once, and the
// lanes of neighbouring tokens (mostly neighbours in their pages too) touch
// neighbouring rows.
template <typename V>
__global__ void __launch_bounds__(COPY_THREADS)
    ffa_token_move_kernel(uint8_t* k_pages, uint8_t* v_pages, const int* __restrict__ src,
                          const int* __restrict__ dst, int n, int Hkv, int page_size, int64_t n_slots,
                          int vecs_per_row, uint32_t* err) {
  const int64_t t = (int64_t)blockIdx.x * COPY_THREADS + threadIdx.x;
  const int64_t tok = t / vecs_per_row;
  const int c = (int)(t % vecs_per_row);
  if (tok >= n) return;
  const int s = src[tok], d = dst[tok];
  if (s < 0 || s >= n_slots || d < 0 || d >= n_slots) {
    if (c == 0 && err) atomicCAS(err, 0u, SITE_COPY_BAD_ID);
    return;
  }
  V* pool = reinterpret_cast<V*>(blockIdx.y ? v_pages : k_pages);
  const int64_t head = (int64_t)page_size * vecs_per_row;  // vectors between a page's heads
  const V* from = pool + (int64_t)(s / page_size) * Hkv * head + (int64_t)(s % page_size) * vecs_per_row + c;
  V* to = pool + (int64_t)(d / page_size) * Hkv * head + (int64_t)(d % page_size) * vecs_per_row + c;
  for (int h0 = 0; h0 < Hkv; h0 += COPY_VECS) {
    V x[COPY_VECS];
#pragma unroll
    for (int i = 0; i < COPY_VECS; ++i)
      if (h0 + i < Hkv) x[i] = from[(h0 + i) * head];
#pragma unroll
    for (int i = 0; i < COPY_VECS; ++i)
      if (h0 + i < Hkv) to[(h0 + i) * head] = x[i];
  }
}

}  // namespace ffa

extern "C" int ffa_page_copy(void* k_pages, void* v_pages, const int* src, const int* dst, int n, int num_pages,
                             int64_t page_bytes, uint32_t* dev_err, void* stream) {
  using namespace ffa;
  if (n == 0) return FFA_OK;
  if (!k_pages || !src || !dst || n < 0 || num_pages <= 0 || page_bytes <= 0) return FFA_ERR_INVALID_ARG;
  if (page_bytes % 2) return FFA_ERR_UNSUPPORTED;
  const bool vec = page_bytes % 16 == 0 && aligned16(k_pages) && aligned16(v_pages);
  if (!vec && ((reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages)) & 1))
    return FFA_ERR_INVALID_ARG;
  const int64_t vecs = page_bytes / (vec ? 16 : 2);
  const int64_t per = (vecs + COPY_THREADS * COPY_VECS - 1) / (COPY_THREADS * COPY_VECS);
  if (per * n > 0x7fffffffLL) return FFA_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)(per * n), v_pages ? 2 : 1);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* kp = static_cast<uint8_t*>(k_pages);
  uint8_t* vp = static_cast<uint8_t*>(v_pages);
  if (vec)
    ffa_page_copy_kernel<uint4><<<grid, COPY_THREADS, 0, st>>>(kp, vp, src, dst, num_pages, vecs, (int)per, dev_err);
  else
    ffa_page_copy_kernel<uint16_t>
        <<<grid, COPY_THREADS, 0, st>>>(kp, vp, src, dst, num_pages, vecs, (int)per, dev_err);
  return launch_status();
}

extern "C" int ffa_token_move(void* k_pages, void* v_pages, const int* src_slots, const int* dst_slots, int n,
                              int Hkv, int page_size, int num_pages, int row_bytes, uint32_t* dev_err,
                              void* stream) {
  using namespace ffa;
  if (n == 0) return FFA_OK;
  if (!k_pages || !src_slots || !dst_slots || n < 0 || Hkv <= 0 || page_size <= 0 || num_pages <= 0 ||
      row_bytes <= 0)
    return FFA_ERR_INVALID_ARG;
  if (row_bytes % 2) return FFA_ERR_UNSUPPORTED;
  const bool vec = row_bytes % 16 == 0 && aligned16(k_pages) && aligned16(v_pages);
  if (!vec && ((reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages)) & 1))
    return FFA_ERR_INVALID_ARG;
  const int vecs = row_bytes / (vec ? 16 : 2);
  const int64_t blocks = ((int64_t)n * vecs + COPY_THREADS - 1) / COPY_THREADS;
  if (blocks > 0x7fffffffLL) return FFA_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)blocks, v_pages ? 2 : 1);
  const int64_t n_slots = (int64_t)num_pages * page_size;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* kp = static_cast<uint8_t*>(k_pages);
  uint8_t* vp = static_cast<uint8_t*>(v_pages);
  if (vec)
    ffa_token_move_kernel<uint4>
        <<<grid, COPY_THREADS, 0, st>>>(kp, vp, src_slots, dst_slots, n, Hkv, page_size, n_slots, vecs, dev_err);
  else
    ffa_token_move_kernel<uint16_t>
        <<<grid, COPY_THREADS, 0, st>>>(kp, vp, src_slots, dst_slots, n, Hkv, page_size, n_slots, vecs, dev_err);
  return launch_status();
}

// Host-side plumbing shared by the C-ABI entry points: CUDA error capture,
// the per-thread wait limit, and TMA tensor-map encoding through the driver
// entry point (so the library does not link libcuda directly).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "ffa_b200.h"

namespace ffa {

void set_last_error(const char* msg);
unsigned long long wait_limit_ns();

// Records the CUDA error string (if any) and maps it to a status.
inline int cuda_status(cudaError_t e) {
  if (e == cudaSuccess) return FFA_OK;
  set_last_error(cudaGetErrorString(e));
  return FFA_ERR_CUDA;
}

// Status of the most recent launch on this thread.
inline int launch_status() { return cuda_status(cudaGetLastError()); }

// Encodes a 4-D tiled TMA map over a row-major tensor whose innermost dim is
// contiguous: dims {d0 (contiguous), d1, d2, d3}, byte strides for d1..d3,
// box {b0, b1, 1, 1}, 128-byte swizzle, zero fill out of bounds.
int make_tmap_4d(CUtensorMap* map, const void* base, CUtensorMapDataType dt, uint32_t elem_bytes, uint64_t d0,
                 uint64_t d1, uint64_t d2, uint64_t d3, uint64_t s1_bytes, uint64_t s2_bytes, uint64_t s3_bytes,
                 uint32_t b0, uint32_t b1);

// Raises a kernel's dynamic shared-memory limit once per device.  The
// attribute belongs to the device's context, so the "done" record is a bit
// per device; the record is atomic because entry points may be called from
// several host threads (setting the attribute twice is harmless).
template <typename Kernel>
int smem_attr_once(Kernel kern, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  int s = cuda_status(cudaGetDevice(&dev));
  if (s) return s;
  const uint64_t bit = dev < 64 ? (1ull << dev) : 0ull;
  if (bit && (done.load(std::memory_order_acquire) & bit)) return FFA_OK;
  s = cuda_status(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (s) return s;
  if (bit) done.fetch_or(bit, std::memory_order_acq_rel);
  return FFA_OK;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// fp32 kernels on the CUDA cores (ffa_f32.cu), reached through ffa_fwd /
// ffa_bwd / ffa_bwd_masked with dtype FFA_DTYPE_F32.
int f32_fwd(const void* q, const void* k, const void* v, void* o, float* lse, int B, int Hq, int Hkv, int Sq,
            int Skv, int D, int Dv, const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
            const int64_t* o_strides, float scale, int causal, int q_offset, int window, int sink, float softcap,
            const uint8_t* block_mask, int n_br, int n_bc, int mask_bq, int mask_bkv, void* stream);
int f32_bwd(const void* dout, const void* q, const void* k, const void* v, const void* o, const float* lse,
            void* dq, void* dk, void* dv, int B, int Hq, int Hkv, int Sq, int Skv, int D, int Dv,
            const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
            const int64_t* o_strides, const int64_t* do_strides, const int64_t* dq_strides,
            const int64_t* dk_strides, const int64_t* dv_strides, float scale, int causal, int q_offset,
            int window, int sink, float softcap, const uint8_t* block_mask, int n_br, int n_bc, int mask_bq, int mask_bkv,
            void* workspace, float* sink_ws, void* stream);

// A window past any length: the kernels add positions to it in 32 bits.
inline int bounded_window(int window) { return window < (1 << 30) ? window : 1 << 30; }

// Head dims of the attention kernel that serves (D, Dv).  The sink kernels take
// any multiples of 8 up to (192, 128): their TMA copies read zeros past the
// true head dim and write nothing there, so narrower heads run on the next
// wider tile without a padded copy.  The others take exactly these widths.
inline bool attention_tile(int D, int Dv, bool sinks, int& KD, int& KV) {
  KD = D <= 64 && Dv <= 64 ? 64 : D <= 128 ? 128 : 192;
  KV = KD == 64 ? 64 : 128;
  if (D <= 0 || Dv <= 0 || D > KD || Dv > KV) return false;
  return sinks ? D % 8 == 0 && Dv % 8 == 0 : D == KD && Dv == KV;
}

// Backward with sinks: the `tile`-key tiles that hold them, [0, tiles), see
// every later query, so `parts` CTAs share each one's queries: about as many
// 64-query units per CTA as the window gives another key tile, so that no CTA
// runs much longer than the rest; at most 64 shares in all, since many sink
// tiles are parallel work enough and every share holds fp32 sums.
inline void bwd_sink_shape(int tile, int Sq, int Skv, int window, int sink, int& tiles, int& parts) {
  const int keys = sink < Skv ? sink : Skv;
  tiles = (keys + tile - 1) / tile;
  const int64_t n_q = ((int64_t)Sq + 63) / 64;
  const int64_t usual = ((int64_t)window + tile + 63) / 64 + 1;
  const int64_t n = (n_q + usual - 1) / usual, most = tiles > 32 ? 1 : 64 / (tiles > 0 ? tiles : 1);
  parts = (int)(n < 1 ? 1 : n > most ? most : n);
}

// The same for the fp32 kernels' 64-key tiles, whose units are many times
// slower: where the key tiles would keep half of the SMs idle, every tile's
// queries are shared (B1 H32/8 S216 D64: 32 CTAs of up to 16 units, about 230
// us, against 45 shared).  Larger grids are not worth it, since a share also loads its K and V
// and leaves its sums (256 CTAs of 5 units in three shares each: 124 -> 165 us).
inline void f32_bwd_sink_shape(int B, int Hq, int Hkv, int Sq, int Skv, int window, int sink, int& tiles,
                               int& parts) {
  bwd_sink_shape(64, Sq, Skv, window, sink, tiles, parts);
  const int64_t all = ((int64_t)Skv + 63) / 64, ctas = all * B * Hkv;
  if (ctas > 74) return;
  const int64_t units = ((int64_t)Sq + 63) / 64 * (Hq / Hkv), n = 4 * 148 / ctas;
  tiles = (int)all;
  parts = (int)(n < units ? n : units);
}

}  // namespace ffa

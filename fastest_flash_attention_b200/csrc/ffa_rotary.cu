// Rotary positions: queries and keys turned by their tokens' angles, for
// training (forward and, by the negative angle, the gradient) and for serving
// (fused with the scatter of keys and values into their cache pages).
//
//   (a, b) -> (a cos - b sin, b cos + a sin)
// for each pair (a, b) of the head's first `rot` values: (x[i], x[i + rot/2])
// in the half layout, (x[2i], x[2i+1]) in the interleaved one; the values from
// `rot` on pass through.  The rotation is orthogonal, so its gradient is the
// rotation by the negative angle.  cos / sin come from fp32 tables of
// [positions, rot / 2] that the caller builds once (in 64 bits, so long
// positions lose nothing); products and sums are fp32, rounded once to the
// data's type.
//
// HBM-bound: every value is read and written once; a token's table row is read
// once per thread and serves all of its heads.  Measured on q [4, 32, 4096, 128]
// and k [4, 8, 4096, 128] bf16: 56 us a launch, 6.06 TB/s (0.92 of a measured
// copy); one thread per pair took 359 us, and addressing each head's row from
// the operand table inside the loop 92 us (integer work).
#include "ffa_common.cuh"
#include "ffa_host.h"

namespace ffa {

// A position outside the tables: the token's values pass through unturned.
enum : uint32_t { SITE_ROT_BAD_POS = 0x3E3 };

constexpr int ROT_THREADS = 256;

struct RotTensor {  // one operand: source and destination with their element strides
  const void* src;
  void* dst;
  int64_t sb, sh, ss;  // source {batch, head, token}
  int64_t db, dh, ds;  // destination
};

struct RotParams {
  RotTensor q, k, v;  // v: serving only (copied, not turned)
  const float* cos;
  const float* sin;
  const void* pos;
  int64_t pos_sb;  // elements between the batch rows of pos (0: one row for all)
  int pos64;       // pos is int64 (else int32)
  int64_t table_len;
  const int* slots;  // serving: token t's cache slot (k.dst / v.dst are then the page pools), else nullptr
  int page_size, num_pages;
  int B, S, Hq, Hkv, D, rot;
  float sign;  // -1: the gradient
  int interleaved;
  int heads_per_thread;  // vector kernel
  uint32_t* err;
};

template <typename T>
__device__ __forceinline__ float rot_to_f(T x);
template <>
__device__ __forceinline__ float rot_to_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ float rot_to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float rot_to_f<__half>(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T rot_from_f(float x);
template <>
__device__ __forceinline__ float rot_from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 rot_from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half rot_from_f<__half>(float x) { return __float2half_rn(x); }

// Table row of token (b, s), or -1 (recorded) if its position has none.
__device__ __forceinline__ int64_t rot_row(const RotParams& p, int b, int s) {
  const int64_t i = (int64_t)b * p.pos_sb + s;
  const int64_t pos = p.pos64 ? static_cast<const int64_t*>(p.pos)[i] : (int64_t) static_cast<const int*>(p.pos)[i];
  if (pos >= 0 && pos < p.table_len) return pos;
  if (p.err) atomicCAS(p.err, 0u, SITE_ROT_BAD_POS);
  return -1;
}

// Head `x` of the token's Hq + Hkv (+ Hkv) rows: its source and destination.
// Returns false for a row that is not written (a slot outside the pool).
template <typename T>
__device__ __forceinline__ bool rot_head(const RotParams& p, int x, int b, int s, int slot, const T*& src, T*& dst,
                                         bool& turn) {
  const RotTensor& o = x < p.Hq ? p.q : (x < p.Hq + p.Hkv ? p.k : p.v);
  const int h = x < p.Hq ? x : (x < p.Hq + p.Hkv ? x - p.Hq : x - p.Hq - p.Hkv);
  turn = x < p.Hq + p.Hkv;
  src = static_cast<const T*>(o.src) + b * o.sb + h * o.sh + (int64_t)s * o.ss;
  if (p.slots != nullptr && x >= p.Hq) {
    const int page = slot / p.page_size;
    if (slot < 0 || page >= p.num_pages) return false;
    dst = static_cast<T*>(o.dst) + (((int64_t)page * p.Hkv + h) * p.page_size + slot % p.page_size) * p.D;
  } else {
    dst = static_cast<T*>(o.dst) + b * o.db + h * o.dh + (int64_t)s * o.ds;
  }
  return true;
}

// One thread per value pair of one head of one token (pass-through values: one
// each): any rot, D, stride and alignment.
template <typename T>
__global__ void __launch_bounds__(ROT_THREADS) ffa_rotary_any_kernel(const RotParams p) {
  const int half = p.rot / 2;
  const int items = half + (p.D - p.rot);
  const int heads = p.Hq + p.Hkv * (p.slots != nullptr ? 2 : 1);
  const int64_t i = (int64_t)blockIdx.x * ROT_THREADS + threadIdx.x;
  const int64_t row = i / items;
  const int c = (int)(i % items);
  const int64_t tok = row / heads;
  if (tok >= (int64_t)p.B * p.S) return;
  const int x = (int)(row % heads), b = (int)(tok / p.S), s = (int)(tok % p.S);
  const T* src;
  T* dst;
  bool turn;
  const int slot = p.slots != nullptr ? p.slots[tok] : 0;
  if (!rot_head<T>(p, x, b, s, slot, src, dst, turn)) return;
  if (c >= half) {
    dst[p.rot + c - half] = src[p.rot + c - half];
    return;
  }
  const int ia = p.interleaved ? 2 * c : c, ib = p.interleaved ? 2 * c + 1 : c + half;
  const int64_t t = turn ? rot_row(p, b, s) : -1;
  if (t < 0) {
    dst[ia] = src[ia];
    dst[ib] = src[ib];
    return;
  }
  const float cs = p.cos[t * half + c], sn = p.sign * p.sin[t * half + c];
  const float a = rot_to_f<T>(src[ia]), z = rot_to_f<T>(src[ib]);
  dst[ia] = rot_from_f<T>(a * cs - z * sn);
  dst[ib] = rot_from_f<T>(z * cs + a * sn);
}

// Eight pairs of values as two 8-value runs (a: the first run, z: the second).
// Half layout: a holds the pairs' first values, z their second ones;
// interleaved: pairs lie side by side, four in each run.
template <typename T>
struct RotRun {  // 8 values
  static constexpr int VECS = 8 * sizeof(T) / 16;
  uint4 v[VECS];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < VECS; ++i) v[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < VECS; ++i) reinterpret_cast<uint4*>(p)[i] = v[i];
  }
  __device__ __forceinline__ void get(float* f) const {
    const T* t = reinterpret_cast<const T*>(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = rot_to_f<T>(t[i]);
  }
  __device__ __forceinline__ void set(const float* f) {
    T* t = reinterpret_cast<T*>(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = rot_from_f<T>(f[i]);
  }
};

// Rotated widths and head dims that are multiples of 16, 16-byte aligned rows:
// one thread holds eight pairs' cos / sin (one read of the token's table row)
// and walks p.heads_per_thread heads with them, ROT_BATCH heads' loads in
// flight at a time.  D / 16 neighbouring threads cover a row, neighbouring
// tokens follow.
constexpr int ROT_BATCH = 4;

// Heads [0, n) of one operand: `src` / `dst` address this token's first head
// of them, `sh` / `dh` step to the next.
template <typename T, bool INTERLEAVED, bool TURN>
__device__ __forceinline__ void rot_walk(const T* src, int64_t sh, T* dst, int64_t dh, int n, int oa, int oz,
                                         const float* cs, const float* sn) {
  constexpr int BATCH = sizeof(T) == 4 ? ROT_BATCH / 2 : ROT_BATCH;
  for (int x = 0; x < n; x += BATCH) {
    RotRun<T> a[BATCH], z[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      if (x + i < n) {
        a[i].load(src + i * sh + oa);
        z[i].load(src + i * sh + oz);
      }
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      if (x + i >= n) continue;
      if (TURN) {
        float f[16], g[16];
        a[i].get(f);
        z[i].get(f + 8);
        if (INTERLEAVED) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            g[2 * e] = f[2 * e] * cs[e] - f[2 * e + 1] * sn[e];
            g[2 * e + 1] = f[2 * e + 1] * cs[e] + f[2 * e] * sn[e];
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            g[e] = f[e] * cs[e] - f[8 + e] * sn[e];
            g[8 + e] = f[8 + e] * cs[e] + f[e] * sn[e];
          }
        }
        a[i].set(g);
        z[i].set(g + 8);
      }
      a[i].store(dst + i * dh + oa);
      z[i].store(dst + i * dh + oz);
    }
    src += BATCH * sh;
    dst += BATCH * dh;
  }
}

template <typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(ROT_THREADS) ffa_rotary_vec_kernel(const RotParams p) {
  const int lanes = p.D / 16;
  const int per_cta = ROT_THREADS / lanes;
  const int c = threadIdx.x % lanes, in_cta = threadIdx.x / lanes;
  const uint32_t tok = blockIdx.x * (uint32_t)per_cta + in_cta;
  if (in_cta >= per_cta || tok >= (uint32_t)p.B * (uint32_t)p.S) return;
  const int b = (int)(tok / (uint32_t)p.S), s = (int)(tok % (uint32_t)p.S);
  const int half = p.rot / 2;
  const bool turned = 16 * c < p.rot;
  int64_t row = -1;
  if (turned) row = rot_row(p, b, s);
  float cs[8], sn[8];
  if (row >= 0) {
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const float4 u = *reinterpret_cast<const float4*>(p.cos + row * half + 8 * c + i);
      const float4 w = *reinterpret_cast<const float4*>(p.sin + row * half + 8 * c + i);
      cs[i] = u.x, cs[i + 1] = u.y, cs[i + 2] = u.z, cs[i + 3] = u.w;
      sn[i] = p.sign * w.x, sn[i + 1] = p.sign * w.y, sn[i + 2] = p.sign * w.z, sn[i + 3] = p.sign * w.w;
    }
  }
  // the two runs of this thread in every row
  const int oa = turned && !INTERLEAVED ? 8 * c : 16 * c;
  const int oz = turned && !INTERLEAVED ? half + 8 * c : 16 * c + 8;
  // this CTA's heads among the token's Hq + Hkv (+ Hkv) rows
  const int x0 = blockIdx.y * p.heads_per_thread, x1 = x0 + p.heads_per_thread;
  const bool paged = p.slots != nullptr;
  int64_t page_row = -1;  // paged: element offset of head 0's row in the pools
  if (paged && x1 > p.Hq) {
    const int slot = p.slots[tok], page = slot / p.page_size;
    if (slot >= 0 && page < p.num_pages)
      page_row = ((int64_t)page * p.Hkv * p.page_size + slot % p.page_size) * p.D;
  }
  auto part = [&](const RotTensor& o, int first, int count, bool kv, bool turn) {
    const int h0 = max(x0 - first, 0), n = min(x1 - first, count) - h0;
    if (n <= 0 || (kv && paged && page_row < 0)) return;
    const T* src = static_cast<const T*>(o.src) + b * o.sb + h0 * o.sh + s * o.ss;
    const int64_t dh = kv && paged ? (int64_t)p.page_size * p.D : o.dh;
    T* dst = static_cast<T*>(o.dst) + (kv && paged ? page_row : b * o.db + s * o.ds) + h0 * dh;
    if (turn && row >= 0)
      rot_walk<T, INTERLEAVED, true>(src, o.sh, dst, dh, n, oa, oz, cs, sn);
    else
      rot_walk<T, INTERLEAVED, false>(src, o.sh, dst, dh, n, oa, oz, cs, sn);
  };
  part(p.q, 0, p.Hq, false, true);
  part(p.k, p.Hq, p.Hkv, true, true);
  if (paged) part(p.v, p.Hq + p.Hkv, p.Hkv, true, false);
}

// 16-byte rows in every operand the launch touches.
template <typename T>
static bool rot_vec_ready(const RotParams& p) {
  constexpr int64_t E = 16 / sizeof(T);
  if (p.D % 16 || p.rot % 16 || p.D > 16 * ROT_THREADS || (int64_t)p.B * p.S > 0x7fffffffLL) return false;
  if (!aligned16(p.cos) || !aligned16(p.sin)) return false;
  const RotTensor* ops[3] = {&p.q, &p.k, &p.v};
  for (const RotTensor* o : ops) {
    if (!aligned16(o->src) || !aligned16(o->dst)) return false;
    for (int64_t s : {o->sb, o->sh, o->ss, o->db, o->dh, o->ds})
      if (s % E) return false;
  }
  return true;
}

// CTAs for each SM that a launch aims at before a thread walks more heads: with
// 2 a launch of the case above takes 56 us, with 4, 8 and 16 58, with 32 62 (the
// table rows are read more often).  Evict-first loads, and batches of 2 heads at
// four resident CTAs, measured 57 to 63 beside it.
constexpr int ROT_CTAS_PER_SM = 2;

template <typename T>
static int launch_rotary(RotParams p, cudaStream_t st) {
  if (rot_vec_ready<T>(p)) {
    const int heads = p.Hq + p.Hkv * (p.slots != nullptr ? 2 : 1);
    const int per_cta = ROT_THREADS / (p.D / 16);
    const int64_t blocks = ((int64_t)p.B * p.S + per_cta - 1) / per_cta;
    // heads per thread: all of them would read each table row once, but the
    // grid should have several CTAs for each SM
    int64_t groups = (148 * ROT_CTAS_PER_SM + blocks - 1) / blocks;
    const int64_t most = (heads + ROT_BATCH - 1) / ROT_BATCH;
    if (groups > most) groups = most;
    p.heads_per_thread = (int)(((heads + groups - 1) / groups + ROT_BATCH - 1) / ROT_BATCH * ROT_BATCH);
    const dim3 grid((unsigned)blocks, (unsigned)((heads + p.heads_per_thread - 1) / p.heads_per_thread));
    if (p.interleaved)
      ffa_rotary_vec_kernel<T, true><<<grid, ROT_THREADS, 0, st>>>(p);
    else
      ffa_rotary_vec_kernel<T, false><<<grid, ROT_THREADS, 0, st>>>(p);
    return launch_status();
  }
  const int64_t heads = p.Hq + (int64_t)p.Hkv * (p.slots != nullptr ? 2 : 1);
  const int64_t items = (int64_t)p.B * p.S * heads * (p.D - p.rot / 2);
  const int64_t blocks = (items + ROT_THREADS - 1) / ROT_THREADS;
  if (blocks > 0x7fffffffLL) return FFA_ERR_UNSUPPORTED;
  ffa_rotary_any_kernel<T><<<(unsigned)blocks, ROT_THREADS, 0, st>>>(p);
  return launch_status();
}

static int rotary_dispatch(const RotParams& p, int dtype, cudaStream_t st) {
  if (dtype == FFA_DTYPE_BF16) return launch_rotary<__nv_bfloat16>(p, st);
  if (dtype == FFA_DTYPE_F16) return launch_rotary<__half>(p, st);
  if (dtype == FFA_DTYPE_F32) return launch_rotary<float>(p, st);
  return FFA_ERR_UNSUPPORTED;
}

static RotTensor rot_tensor(const void* src, const int64_t* s, void* dst, const int64_t* d) {
  RotTensor t{};
  t.src = src;
  t.dst = dst;
  if (s) t.sb = s[0], t.sh = s[1], t.ss = s[2];
  if (d) t.db = d[0], t.dh = d[1], t.ds = d[2];
  return t;
}

}  // namespace ffa

extern "C" int ffa_rotary(const void* q, const int64_t* q_strides, void* q_out, const int64_t* qo_strides,
                          const void* k, const int64_t* k_strides, void* k_out, const int64_t* ko_strides,
                          const float* cos, const float* sin, int64_t table_len, const void* pos, int pos64,
                          int64_t pos_batch_stride, int dtype, int B, int S, int Hq, int Hkv, int D, int rot,
                          int interleaved, int inverse, uint32_t* dev_err, void* stream) {
  using namespace ffa;
  if (B == 0 || S == 0) return FFA_OK;
  if (!q || !q_strides || !q_out || !qo_strides || !cos || !sin || !pos) return FFA_ERR_INVALID_ARG;
  if (Hkv > 0 && (!k || !k_strides || !k_out || !ko_strides)) return FFA_ERR_INVALID_ARG;
  if (B < 0 || S < 0 || Hq <= 0 || Hkv < 0 || D <= 0 || rot <= 0 || rot > D || rot % 2 || table_len <= 0)
    return FFA_ERR_INVALID_ARG;
  RotParams p{};
  p.q = rot_tensor(q, q_strides, q_out, qo_strides);
  p.k = rot_tensor(k, k_strides, k_out, ko_strides);
  p.cos = cos;
  p.sin = sin;
  p.pos = pos;
  p.pos_sb = pos_batch_stride;
  p.pos64 = pos64;
  p.table_len = table_len;
  p.B = B;
  p.S = S;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.D = D;
  p.rot = rot;
  p.sign = inverse ? -1.f : 1.f;
  p.interleaved = interleaved;
  p.err = dev_err;
  return rotary_dispatch(p, dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int ffa_rotary_append(const void* q, const int64_t* q_strides, void* q_out, const int64_t* qo_strides,
                                 const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                 const float* cos, const float* sin, int64_t table_len, const void* pos, int pos64,
                                 const int* slots, void* k_pages, void* v_pages, int dtype, int n_tokens, int Hq,
                                 int Hkv, int D, int rot, int interleaved, int page_size, int num_pages,
                                 uint32_t* dev_err, void* stream) {
  using namespace ffa;
  if (n_tokens == 0) return FFA_OK;
  if (!q || !q_strides || !q_out || !qo_strides || !k || !k_strides || !v || !v_strides || !cos || !sin || !pos ||
      !slots || !k_pages || !v_pages)
    return FFA_ERR_INVALID_ARG;
  if (n_tokens < 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || rot <= 0 || rot > D || rot % 2 || table_len <= 0 ||
      page_size <= 0 || num_pages <= 0)
    return FFA_ERR_INVALID_ARG;
  // tokens along the "batch" axis: strides {token, head}
  const int64_t qs[3] = {q_strides[0], q_strides[1], 0}, qd[3] = {qo_strides[0], qo_strides[1], 0};
  const int64_t ks[3] = {k_strides[0], k_strides[1], 0}, vs[3] = {v_strides[0], v_strides[1], 0};
  RotParams p{};
  p.q = rot_tensor(q, qs, q_out, qd);
  p.k = rot_tensor(k, ks, k_pages, nullptr);
  p.v = rot_tensor(v, vs, v_pages, nullptr);
  p.cos = cos;
  p.sin = sin;
  p.pos = pos;
  p.pos_sb = 1;
  p.pos64 = pos64;
  p.table_len = table_len;
  p.slots = slots;
  p.page_size = page_size;
  p.num_pages = num_pages;
  p.B = n_tokens;
  p.S = 1;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.D = D;
  p.rot = rot;
  p.sign = 1.f;
  p.interleaved = interleaved;
  p.err = dev_err;
  return rotary_dispatch(p, dtype, static_cast<cudaStream_t>(stream));
}

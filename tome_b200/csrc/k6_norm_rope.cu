// K6: norms of queries and keys for each head with the rotary position rotation, one pass
// (HBM-bound): forward, backward, and the serving form that appends keys and values to the
// paged cache.  The reference's own kernel for the forward is mlx-impl/model.py:105-194.
//
// For a head x of D elements at position p, in fp32:
//   r = rsqrt(mean(x^2) + eps),  y = x * r * w,
//   z[i] = y[i] cos[p, i] - y[i + D/2] sin[p, i],   z[i + D/2] = y[i + D/2] cos[p, i] + y[i] sin[p, i]
// rounded once, on the store.  Backward of dz:
//   dy = the rotation by -p of dz,  dw += dy * x * r,  g = dy * w,
//   dx = r * (g - x r * mean(g * x r)).
//
// A head is shared by a small group of threads, each holding eight elements of the first half
// and the eight they are rotated with of the second half: both 16-byte vectors (two per half
// in fp32), no exchange but the sum of squares.  A group takes several heads of one token at a
// time, so that cos and sin are fetched once for them and enough loads are in flight.
//
// Measured (CUDA-graph replay; bytes read and written once), 20480 tokens of 16 + 8 heads of 128,
// bf16: forward 44 to 46 us, 5.6 to 5.8 TB/s (0.85 to 0.89 of a copy); backward 98 us, 4.75 TB/s (0.73): 128 registers
// leave 16 warps per SM, which wait for their loads.  Appending 4084
// tokens of 32 + 8 heads 21 us, 8 tokens 2.7 us.  Blocks of 64 threads took 111 us backward and 48
// forward, of 256 threads 111 to 139 and 90, one head per group 112 to 128 backward, and fetching the
// next item's loads ahead into registers 110 to 145.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "host_common.h"
#include "ptx.cuh"

namespace tome {

constexpr int K6_THREADS = 128;
constexpr int K6_MAX_DIM = 256;
// heads per group, blocks per SM that the registers are limited for
constexpr int K6_F_HPG = 4, K6_F_MINB = 5;  // forward
constexpr int K6_B_HPG = 2, K6_B_MINB = 4;  // backward

struct K6Params {
  const void* qkv;          // [T, (heads + 2 kv_heads) * D], token stride qkv_stride
  int64_t qkv_stride;       // elements
  const void* q_weight;     // [D]
  const void* k_weight;     // [D]
  const float* cos_sin;     // [n_positions, D]: cos of the D/2 angles, then sin
  const int32_t* positions; // [T]
  int64_t tokens;
  int32_t n_positions, heads, kv_heads, dim;
  float eps;
  void* q_out;              // [T, heads, D]            (backward: unused)
  void* k_out;              // [T, kv_heads, D]; null: keys and values go to the pools
  // append
  const int32_t* seq_ids;   // [T] or null (token t belongs to sequence t)
  const int32_t* tables;    // [n_seq, max_blocks]
  const int32_t* cache_pos; // [T]; negative: not cached
  void* k_pool;             // [num_blocks, kv_heads, block_size, D]
  void* v_pool;
  int32_t n_seq, max_blocks, num_blocks, block_size;
  // backward
  const void* grad_q;       // [T, heads, D]
  const void* grad_k;       // [T, kv_heads, D]
  const void* grad_v;       // [T, kv_heads, D] or null (zeros)
  void* grad_qkv;           // [T, (heads + 2 kv_heads) * D]
  float* partial;           // [gridDim.x, 2, D] weight-gradient sums of each block
  int32_t* status;
};

__device__ __forceinline__ void k6_raise(int32_t* status, int32_t bit) {
  if (status != nullptr) atomicOr(status, bit);
}

// ------------------------------------------------------------------ eight elements <-> fp32
// (pairs, for the packed fp32 arithmetic: two elements per instruction)
struct K6Eight {
  float2 v[4];
};
__device__ __forceinline__ float2 k6_both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 k6_neg(float2 x) { return make_float2(-x.x, -x.y); }

template <typename T>
struct K6Raw {  // eight elements as they sit in memory
  uint4 a;
};
template <>
struct K6Raw<float> {
  uint4 a, b;
};

template <typename T>
__device__ __forceinline__ K6Raw<T> k6_load(const T* p) {
  K6Raw<T> r;
  const uint4* s = reinterpret_cast<const uint4*>(p);
  r.a = __ldcs(s);
  if constexpr (sizeof(T) == 4) r.b = __ldcs(s + 1);
  return r;
}

template <typename T>
__device__ __forceinline__ K6Raw<T> k6_load_cached(const T* p) {  // for what is read again soon
  K6Raw<T> r;
  const uint4* s = reinterpret_cast<const uint4*>(p);
  r.a = __ldg(s);
  if constexpr (sizeof(T) == 4) r.b = __ldg(s + 1);
  return r;
}

template <typename T>
__device__ __forceinline__ void k6_store(T* p, const K6Raw<T>& r) {
  stg128_streaming(p, r.a);
  if constexpr (sizeof(T) == 4) stg128_streaming(p + 4, r.b);
}

__device__ __forceinline__ float2 k6_pair(uint32_t w, __nv_bfloat16) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 k6_pair(uint32_t w, __half) {
  return __half22float2(*reinterpret_cast<__half2*>(&w));
}
__device__ __forceinline__ uint32_t k6_pack(float2 f, __nv_bfloat16) {
  const __nv_bfloat162 h = __float22bfloat162_rn(f);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t k6_pack(float2 f, __half) {
  const __half2 h = __float22half2_rn(f);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ K6Eight k6_unpack(const K6Raw<T>& r) {
  K6Eight e;
  if constexpr (sizeof(T) == 4) {
    e.v[0] = make_float2(__uint_as_float(r.a.x), __uint_as_float(r.a.y));
    e.v[1] = make_float2(__uint_as_float(r.a.z), __uint_as_float(r.a.w));
    e.v[2] = make_float2(__uint_as_float(r.b.x), __uint_as_float(r.b.y));
    e.v[3] = make_float2(__uint_as_float(r.b.z), __uint_as_float(r.b.w));
  } else {
    e.v[0] = k6_pair(r.a.x, T());
    e.v[1] = k6_pair(r.a.y, T());
    e.v[2] = k6_pair(r.a.z, T());
    e.v[3] = k6_pair(r.a.w, T());
  }
  return e;
}

template <typename T>
__device__ __forceinline__ K6Raw<T> k6_pack8(const K6Eight& e) {
  K6Raw<T> r;
  if constexpr (sizeof(T) == 4) {
    r.a = make_uint4(__float_as_uint(e.v[0].x), __float_as_uint(e.v[0].y), __float_as_uint(e.v[1].x),
                     __float_as_uint(e.v[1].y));
    r.b = make_uint4(__float_as_uint(e.v[2].x), __float_as_uint(e.v[2].y), __float_as_uint(e.v[3].x),
                     __float_as_uint(e.v[3].y));
  } else {
    r.a = make_uint4(k6_pack(e.v[0], T()), k6_pack(e.v[1], T()), k6_pack(e.v[2], T()), k6_pack(e.v[3], T()));
  }
  return r;
}

// Sum of the squares of a thread's sixteen elements.
__device__ __forceinline__ float k6_squares(const K6Eight& a, const K6Eight& b) {
  float2 s = __fmul2_rn(a.v[0], a.v[0]);
#pragma unroll
  for (int e = 1; e < 4; ++e) s = __ffma2_rn(a.v[e], a.v[e], s);
#pragma unroll
  for (int e = 0; e < 4; ++e) s = __ffma2_rn(b.v[e], b.v[e], s);
  return s.x + s.y;
}

__device__ __forceinline__ K6Eight k6_eight(const float* p) { return k6_unpack(k6_load_cached(p)); }

// Sum over the 2^k threads of a head's group.
template <int G>
__device__ __forceinline__ float k6_group_sum(float x) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// Token and slot of item (first + i), i < 2^16: the quotient of the block's first item is the same for
// all its threads, the rest is small.
struct K6Place {
  int64_t token;
  int32_t slot;
};
__device__ __forceinline__ K6Place k6_place(int64_t first, int32_t i, int32_t per_token) {
  const int64_t t0 = (first >> 31) == 0
                         ? static_cast<int64_t>(static_cast<uint32_t>(first) / static_cast<uint32_t>(per_token))
                         : first / per_token;
  const uint32_t rest = static_cast<uint32_t>(first - t0 * per_token) + static_cast<uint32_t>(i);
  const uint32_t q = rest / static_cast<uint32_t>(per_token);
  return K6Place{t0 + q, static_cast<int32_t>(rest - q * per_token)};
}

// ------------------------------------------------------------------ forward and append
// Work items of a token: ceil(heads / HPG) of queries, ceil(kv_heads / HPG) of keys and, when
// appending, as many of values (copied).  G threads share a head.
template <typename T, int G, int HPG>
__global__ void __launch_bounds__(K6_THREADS, HPG == 1 ? 3 : (sizeof(T) == 4 ? 1 : K6_F_MINB)) k6_forward_kernel(const K6Params p) {
  const int j = threadIdx.x % G;  // which eight elements of a half
  const int half = p.dim >> 1;
  const bool on = j * 8 < half;   // groups are a power of two: some threads may have no elements
  const int64_t groups = static_cast<int64_t>(gridDim.x) * (K6_THREADS / G);
  const int q_items = (p.heads + HPG - 1) / HPG, k_items = (p.kv_heads + HPG - 1) / HPG;
  const int per_token = q_items + k_items * (p.k_out == nullptr ? 2 : 1);
  const int64_t items = p.tokens * per_token;
  const float inv_dim = 1.0f / static_cast<float>(p.dim);
  // whole warps stay together for the shuffles: the bound is rounded up to a warp's groups
  const int64_t rounded = (items + 32 / G - 1) / (32 / G) * (32 / G);
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * (K6_THREADS / G) + threadIdx.x / G;
       item < rounded; item += groups) {
    const bool live = on && item < items;
    const K6Place at_item = k6_place(item - threadIdx.x / G, threadIdx.x / G, per_token);
    const int64_t t = live ? at_item.token : 0;
    int slot = at_item.slot;
    const int kind = slot < q_items ? 0 : (slot < q_items + k_items ? 1 : 2);
    slot -= kind == 0 ? 0 : (kind == 1 ? q_items : q_items + k_items);
    const int h0 = slot * HPG;
    const int n = live ? min(HPG, (kind == 0 ? p.heads : p.kv_heads) - h0) : 0;
    const T* src = reinterpret_cast<const T*>(p.qkv) + t * p.qkv_stride +
                   static_cast<int64_t>(h0 + (kind == 0 ? 0 : p.heads + (kind == 1 ? 0 : p.kv_heads))) *
                       p.dim + j * 8;
    K6Raw<T> lo[HPG], hi[HPG];
#pragma unroll
    for (int i = 0; i < HPG; ++i)
      if (i < n) {
        lo[i] = k6_load(src + i * p.dim);
        hi[i] = k6_load(src + i * p.dim + half);
      }
    // where the heads go: h0 .. h0 + n of q / k, or the token's row of the pools' blocks
    T* dst = nullptr;
    int64_t pitch = p.dim;
    if (n > 0) {
      if (kind == 0) {
        dst = reinterpret_cast<T*>(p.q_out) + (t * p.heads + h0) * p.dim + j * 8;
      } else if (p.k_out != nullptr) {
        dst = reinterpret_cast<T*>(p.k_out) + (t * p.kv_heads + h0) * p.dim + j * 8;
      } else {
        const int32_t at = p.cache_pos[t], pos = p.positions[t];
        // a token whose rotary position is bad (its keys report it) is not cached at all
        if (at >= 0 && pos >= 0 && pos < p.n_positions) {
          const int64_t seq = p.seq_ids != nullptr ? static_cast<int64_t>(p.seq_ids[t]) : t;
          const int32_t blk = at / p.block_size;
          int32_t page = -1;
          if (seq >= 0 && seq < p.n_seq && blk < p.max_blocks)
            page = p.tables[seq * p.max_blocks + blk];
          if (page >= 0 && page < p.num_blocks) {
            pitch = static_cast<int64_t>(p.block_size) * p.dim;
            dst = reinterpret_cast<T*>(kind == 1 ? p.k_pool : p.v_pool) +
                  (static_cast<int64_t>(page) * p.kv_heads + h0) * pitch +
                  static_cast<int64_t>(at - blk * p.block_size) * p.dim + j * 8;
          } else if (j == 0) {
            k6_raise(p.status, TOME_DEV_BLOCK_OUT_OF_RANGE);
          }
        }
      }
    }
    if (kind == 2) {  // values are copied (and take part in the shuffles below like the others)
#pragma unroll
      for (int i = 0; i < HPG; ++i)
        if (i < n && dst != nullptr) {
          k6_store(dst + i * pitch, lo[i]);
          k6_store(dst + i * pitch + half, hi[i]);
        }
    }
    K6Eight w_lo = {}, w_hi = {}, co = {}, si = {};
    bool bad = false;
    if (n > 0 && kind != 2) {
      const T* w = reinterpret_cast<const T*>(kind == 0 ? p.q_weight : p.k_weight) + j * 8;
      w_lo = k6_unpack(k6_load_cached(w));
      w_hi = k6_unpack(k6_load_cached(w + half));
      const int32_t pos = p.positions[t];
      bad = pos < 0 || pos >= p.n_positions;
      if (bad && j == 0) k6_raise(p.status, TOME_DEV_POSITION_OUT_OF_RANGE);
      const float* cs = p.cos_sin + static_cast<int64_t>(bad ? 0 : pos) * p.dim + j * 8;
      co = k6_eight(cs);
      si = k6_eight(cs + half);
    }
#pragma unroll
    for (int i = 0; i < HPG; ++i) {
      K6Eight a = {}, b = {};
      if (i < n) {
        a = k6_unpack(lo[i]);
        b = k6_unpack(hi[i]);
      }
      const float ss = k6_group_sum<G>(k6_squares(a, b));
      float r = rsqrtf(fmaf(ss, inv_dim, p.eps));
      if (bad) r = __int_as_float(0x7fc00000);
      K6Eight za, zb;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 ya = __fmul2_rn(__fmul2_rn(a.v[e], k6_both(r)), w_lo.v[e]);
        const float2 yb = __fmul2_rn(__fmul2_rn(b.v[e], k6_both(r)), w_hi.v[e]);
        za.v[e] = __ffma2_rn(ya, co.v[e], __fmul2_rn(k6_neg(yb), si.v[e]));
        zb.v[e] = __ffma2_rn(yb, co.v[e], __fmul2_rn(ya, si.v[e]));
      }
      if (i < n && kind != 2 && dst != nullptr) {
        k6_store(dst + i * pitch, k6_pack8<T>(za));
        k6_store(dst + i * pitch + half, k6_pack8<T>(zb));
      }
    }
  }
}

// ------------------------------------------------------------------ backward
// One kind of heads at a time, queries, then keys, then the values' copy: each thread sums the weight
// gradients of its elements over all its heads of a kind, a block adds its groups' sums in a fixed
// order and leaves them in `partial`, which k6_weight_grad_kernel adds over the blocks: the result
// does not depend on timing.
template <typename T, int G, int HPG>
__global__ void __launch_bounds__(K6_THREADS, sizeof(T) == 4 ? 1 : K6_B_MINB) k6_backward_kernel(const K6Params p) {
  const int j = threadIdx.x % G;
  const int half = p.dim >> 1;
  const bool on = j * 8 < half;
  constexpr int PER_BLOCK = K6_THREADS / G;
  const int64_t width = static_cast<int64_t>(p.heads + 2 * p.kv_heads) * p.dim;
  const float inv_dim = 1.0f / static_cast<float>(p.dim);
  __shared__ float sums[K6_THREADS / 32][2][K6_MAX_DIM];
  griddep_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

#pragma unroll 1
  for (int kind = 0; kind < 2; ++kind) {
    const int heads = kind == 0 ? p.heads : p.kv_heads;
    const int per_token = (heads + HPG - 1) / HPG;
    const int64_t items = p.tokens * per_token;
    const int64_t rounded = (items + 32 / G - 1) / (32 / G) * (32 / G);  // whole warps for the shuffles
    const T* grads = reinterpret_cast<const T*>(kind == 0 ? p.grad_q : p.grad_k) + j * 8;
    const int64_t column0 = (kind == 0 ? 0 : static_cast<int64_t>(p.heads) * p.dim) + j * 8;
    K6Raw<T> w_lo = {}, w_hi = {};
    if (on) {
      const T* w = reinterpret_cast<const T*>(kind == 0 ? p.q_weight : p.k_weight) + j * 8;
      w_lo = k6_load_cached(w);
      w_hi = k6_load_cached(w + half);
    }
    float2 dw[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[i] = make_float2(0.0f, 0.0f);
    for (int64_t first = static_cast<int64_t>(blockIdx.x) * PER_BLOCK; first + threadIdx.x / G < rounded;
         first += static_cast<int64_t>(gridDim.x) * PER_BLOCK) {
      const K6Place at = k6_place(first, threadIdx.x / G, per_token);
      const bool live = on && at.token < p.tokens;
      const int64_t t = live ? at.token : 0;
      const int h0 = at.slot * HPG;
      const int n = live ? min(HPG, heads - h0) : 0;
      const T* x = reinterpret_cast<const T*>(p.qkv) + t * p.qkv_stride + column0 + h0 * p.dim;
      const T* g = grads + (t * heads + h0) * p.dim;
      T* dst = reinterpret_cast<T*>(p.grad_qkv) + t * width + column0 + h0 * p.dim;
      K6Raw<T> xl[HPG] = {}, xh[HPG] = {}, gl[HPG] = {}, gh[HPG] = {};
#pragma unroll
      for (int i = 0; i < HPG; ++i)
        if (i < n) {
          xl[i] = k6_load(x + i * p.dim);
          xh[i] = k6_load(x + i * p.dim + half);
          gl[i] = k6_load(g + i * p.dim);
          gh[i] = k6_load(g + i * p.dim + half);
        }
      K6Eight co = {}, si = {};
      bool bad = false;
      if (n > 0) {
        const int32_t pos = p.positions[t];
        bad = pos < 0 || pos >= p.n_positions;
        if (bad && j == 0) k6_raise(p.status, TOME_DEV_POSITION_OUT_OF_RANGE);
        const float* cs = p.cos_sin + static_cast<int64_t>(bad ? 0 : pos) * p.dim + j * 8;
        co = k6_eight(cs);
        si = k6_eight(cs + half);
      }
#pragma unroll
      for (int i = 0; i < HPG; ++i) {
        const K6Eight a = k6_unpack(xl[i]), b = k6_unpack(xh[i]);
        const float ss = k6_group_sum<G>(k6_squares(a, b));
        // 0 for a head that is not there: with an eps of 0 its zeros would become NaN in the sums
        float r = i < n ? rsqrtf(fmaf(ss, inv_dim, p.eps)) : 0.0f;
        if (bad) r = __int_as_float(0x7fc00000);
        const K6Eight da = k6_unpack(gl[i]), db = k6_unpack(gh[i]), wa = k6_unpack(w_lo), wb = k6_unpack(w_hi);
        K6Eight ya, yb;  // gradient of the normed head (rotation turned back), times the weight
        float2 dot2 = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 na = __fmul2_rn(a.v[e], k6_both(r)), nb = __fmul2_rn(b.v[e], k6_both(r));
          ya.v[e] = __ffma2_rn(da.v[e], co.v[e], __fmul2_rn(db.v[e], si.v[e]));
          yb.v[e] = __ffma2_rn(db.v[e], co.v[e], __fmul2_rn(k6_neg(da.v[e]), si.v[e]));
          dw[e] = __ffma2_rn(ya.v[e], na, dw[e]);  // (heads that are not there have zeros)
          dw[4 + e] = __ffma2_rn(yb.v[e], nb, dw[4 + e]);
          ya.v[e] = __fmul2_rn(ya.v[e], wa.v[e]);
          yb.v[e] = __fmul2_rn(yb.v[e], wb.v[e]);
          dot2 = __ffma2_rn(ya.v[e], na, __ffma2_rn(yb.v[e], nb, dot2));
        }
        const float dot = -k6_group_sum<G>(dot2.x + dot2.y) * inv_dim * r;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          ya.v[e] = __fmul2_rn(k6_both(r), __ffma2_rn(a.v[e], k6_both(dot), ya.v[e]));
          yb.v[e] = __fmul2_rn(k6_both(r), __ffma2_rn(b.v[e], k6_both(dot), yb.v[e]));
        }
        if (i < n) {
          k6_store(dst + i * p.dim, k6_pack8<T>(ya));
          k6_store(dst + i * p.dim + half, k6_pack8<T>(yb));
        }
      }
    }
    // the warp's sums, over its groups (lanes that differ in their group's bits)
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int o = 16; o >= G; o >>= 1) {
        dw[e].x += __shfl_xor_sync(0xffffffffu, dw[e].x, o);
        dw[e].y += __shfl_xor_sync(0xffffffffu, dw[e].y, o);
      }
    if (lane < G && on)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        *reinterpret_cast<float2*>(&sums[warp][kind][j * 8 + 2 * e]) = dw[e];
        *reinterpret_cast<float2*>(&sums[warp][kind][half + j * 8 + 2 * e]) = dw[4 + e];
      }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * p.dim; i += K6_THREADS) {
    const int kind = i >= p.dim, e = i - kind * p.dim;
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < K6_THREADS / 32; ++w) s += sums[w][kind][e];
    p.partial[static_cast<int64_t>(blockIdx.x) * 2 * p.dim + i] = s;
  }

  // the values' part: copied, or zeros
  constexpr int ES = 16 / sizeof(T);
  const int64_t per_token = static_cast<int64_t>(p.kv_heads) * p.dim / ES, all = p.tokens * per_token;
  const int64_t step = static_cast<int64_t>(gridDim.x) * K6_THREADS;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * K6_THREADS + threadIdx.x; i < all; i += step) {
    const int64_t t = (i >> 31) == 0 ? static_cast<int64_t>(static_cast<uint32_t>(i) / static_cast<uint32_t>(per_token))
                                     : i / per_token;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (p.grad_v != nullptr) v = __ldcs(reinterpret_cast<const uint4*>(p.grad_v) + i);
    stg128_streaming(reinterpret_cast<T*>(p.grad_qkv) + t * width + static_cast<int64_t>(p.heads + p.kv_heads) * p.dim +
                         (i - t * per_token) * ES, v);
  }
}

// out[i] = sum over the blocks of partial[block, i], i < 2 * dim: 32 columns per block, the
// rows dealt to 32 warps and their sums added in order.
__global__ void __launch_bounds__(1024) k6_weight_grad_kernel(const float* partial, int blocks,
                                                              int dim, float* q_out, float* k_out) {
  __shared__ float sums[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int i = blockIdx.x * 32 + lane;
  griddep_wait();
  float s = 0.0f;
  if (i < 2 * dim)
    for (int b = warp; b < blocks; b += 32) s += partial[static_cast<int64_t>(b) * 2 * dim + i];
  sums[warp][lane] = s;
  __syncthreads();
  float v = sums[lane][warp];  // column `warp` of this block's 32
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int c = blockIdx.x * 32 + warp;
  if (lane == 0 && c < 2 * dim) {
    if (c < dim) q_out[c] = v; else k_out[c - dim] = v;
  }
}

// ------------------------------------------------------------------ host side
// Blocks of the backward's grid at most (K6_B_MINB per SM: 592 on 148 SMs, and room for a larger
// part); also the rows of the partial sums that the workspace has to hold.
constexpr int K6_MAX_BLOCKS = 1024;

static int k6_group_of(int dim) {
  int g = 1;
  while (g * 16 < dim) g <<= 1;
  return g;
}

static int32_t k6_check(const K6Params& p, int32_t dtype, const void* const* required, int n_required) {
  if (dtype != TOME_F32 && dtype != TOME_BF16 && dtype != TOME_F16)
    return fail(TOME_ERR_BAD_DTYPE, "dtype=%d", dtype);
  if (p.tokens < 0 || p.heads <= 0 || p.kv_heads <= 0 || p.heads > 65536 || p.kv_heads > 65536 ||
      p.n_positions <= 0)
    return fail(TOME_ERR_BAD_SHAPE, "tokens=%lld heads=%d kv_heads=%d n_positions=%d",
                (long long)p.tokens, p.heads, p.kv_heads, p.n_positions);
  if (p.dim < 16 || p.dim > K6_MAX_DIM || p.dim % 16 != 0)
    return fail(TOME_ERR_UNSUPPORTED, "head_dim=%d must be a multiple of 16 in [16, %d]", p.dim,
                K6_MAX_DIM);
  if (!(p.eps >= 0.0f) || p.eps > 1.0f) return fail(TOME_ERR_BAD_SHAPE, "eps=%g", (double)p.eps);
  if (p.tokens == 0) return TOME_OK;
  const int64_t es = dtype == TOME_F32 ? 4 : 2;
  if (p.qkv_stride < static_cast<int64_t>(p.heads + 2 * p.kv_heads) * p.dim ||
      (p.qkv_stride * es) % 16 != 0)
    return fail(TOME_ERR_BAD_STRIDE, "qkv_stride=%lld", (long long)p.qkv_stride);
  for (int i = 0; i < n_required; ++i) {
    if (required[i] == nullptr) return fail(TOME_ERR_NULL_POINTER, "a required pointer is NULL");
    if (!aligned16(required[i]))
      return fail(TOME_ERR_MISALIGNED, "tensors must be 16-byte aligned");
  }
  if (p.positions == nullptr) return fail(TOME_ERR_NULL_POINTER, "positions is NULL");
  return TOME_OK;
}

template <typename T, int HPG, bool BACK>
static const void* k6_kernel_of(int g) {
  switch (g) {
#define K6_CASE(G)                                                                  \
  case G:                                                                           \
    return BACK ? reinterpret_cast<const void*>(&k6_backward_kernel<T, G, HPG>)     \
                : reinterpret_cast<const void*>(&k6_forward_kernel<T, G, HPG>);
    K6_CASE(1)
    K6_CASE(2)
    K6_CASE(4)
    K6_CASE(8)
    K6_CASE(16)
#undef K6_CASE
  }
  return nullptr;
}

template <bool BACK>
static int32_t k6_launch(const K6Params& p, int32_t dtype, cudaStream_t stream, int* blocks_out) {
  DeviceInfo info;
  const int32_t st = current_device_info(&info);
  if (st != TOME_OK) return st;
  const int g = k6_group_of(p.dim);
  const int per_block = K6_THREADS / g;
  const int sections = (BACK || p.k_out == nullptr) ? 2 : 1;
  const int64_t heads_in_all = p.tokens * (p.heads + sections * p.kv_heads);
  // One head per group while that still fills no more than the device once (a decode step:
  // latency), else several heads of a token share its cos and sin.
  const int many = BACK ? K6_B_HPG : K6_F_HPG;
  const bool one = heads_in_all <= static_cast<int64_t>(info.sm_count) * 2 * per_block;
  const int hpg = one ? 1 : many;
  const int64_t items =
      p.tokens * ((p.heads + hpg - 1) / hpg + sections * ((p.kv_heads + hpg - 1) / hpg));
  const int64_t want = (items + per_block - 1) / per_block;
  int64_t blocks = std::max<int64_t>(1, want);
  if (BACK) blocks = std::min<int64_t>(blocks, std::min(info.sm_count * K6_B_MINB, K6_MAX_BLOCKS));
  else blocks = std::min<int64_t>(blocks, static_cast<int64_t>(1) << 30);
  const void* kernel = nullptr;
  if (dtype == TOME_F32)
    kernel = one ? k6_kernel_of<float, 1, BACK>(g) : k6_kernel_of<float, BACK ? K6_B_HPG : K6_F_HPG, BACK>(g);
  else if (dtype == TOME_BF16)
    kernel = one ? k6_kernel_of<__nv_bfloat16, 1, BACK>(g)
                 : k6_kernel_of<__nv_bfloat16, BACK ? K6_B_HPG : K6_F_HPG, BACK>(g);
  else
    kernel = one ? k6_kernel_of<__half, 1, BACK>(g) : k6_kernel_of<__half, BACK ? K6_B_HPG : K6_F_HPG, BACK>(g);
  void* args[] = {const_cast<K6Params*>(&p)};
  if (blocks_out != nullptr) *blocks_out = static_cast<int>(blocks);
  return check_cuda(cudaLaunchKernel(kernel, dim3(static_cast<unsigned>(blocks)), dim3(K6_THREADS),
                                     args, 0, stream),
                    BACK ? "norm rope backward launch" : "norm rope launch");
}

}  // namespace tome

using namespace tome;

extern "C" int32_t tome_qk_norm_rope(const void* qkv, int32_t dtype, int64_t tokens, int32_t heads,
                                     int32_t kv_heads, int32_t head_dim, int64_t qkv_stride,
                                     const void* q_weight, const void* k_weight,
                                     const float* cos_sin, int32_t n_positions,
                                     const int32_t* positions, float eps, void* q_out, void* k_out,
                                     int32_t* dev_status, void* stream) {
  K6Params p = {};
  p.qkv = qkv;
  p.qkv_stride = qkv_stride;
  p.q_weight = q_weight;
  p.k_weight = k_weight;
  p.cos_sin = cos_sin;
  p.n_positions = n_positions;
  p.positions = positions;
  p.tokens = tokens;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.dim = head_dim;
  p.eps = eps;
  p.q_out = q_out;
  p.k_out = k_out;
  p.status = dev_status;
  const void* required[] = {qkv, q_weight, k_weight, cos_sin, q_out, k_out};
  const int32_t st = k6_check(p, dtype, required, 6);
  if (st != TOME_OK || tokens == 0) return st;
  return k6_launch<false>(p, dtype, static_cast<cudaStream_t>(stream), nullptr);
}

extern "C" int32_t tome_qk_norm_rope_append(
    const void* qkv, int32_t dtype, int64_t tokens, int32_t heads, int32_t kv_heads,
    int32_t head_dim, int64_t qkv_stride, const void* q_weight, const void* k_weight,
    const float* cos_sin, int32_t n_positions, const int32_t* positions, float eps,
    const int32_t* seq_ids, const int32_t* block_tables, const int32_t* cache_positions,
    int64_t n_seq, int32_t block_size, int32_t max_blocks, int32_t num_blocks, void* q_out,
    void* k_pool, void* v_pool, int32_t* dev_status, void* stream) {
  K6Params p = {};
  p.qkv = qkv;
  p.qkv_stride = qkv_stride;
  p.q_weight = q_weight;
  p.k_weight = k_weight;
  p.cos_sin = cos_sin;
  p.n_positions = n_positions;
  p.positions = positions;
  p.tokens = tokens;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.dim = head_dim;
  p.eps = eps;
  p.q_out = q_out;
  p.seq_ids = seq_ids;
  p.tables = block_tables;
  p.cache_pos = cache_positions;
  p.k_pool = k_pool;
  p.v_pool = v_pool;
  p.n_seq = static_cast<int32_t>(n_seq);
  p.block_size = block_size;
  p.max_blocks = max_blocks;
  p.num_blocks = num_blocks;
  p.status = dev_status;
  const void* required[] = {qkv, q_weight, k_weight, cos_sin, q_out, k_pool, v_pool};
  const int32_t st = k6_check(p, dtype, required, 7);
  if (st != TOME_OK) return st;
  if (n_seq < 0 || n_seq > 0x7fffffff || block_size <= 0 || max_blocks < 0 || num_blocks < 0 ||
      (seq_ids == nullptr && n_seq != tokens))
    return fail(TOME_ERR_BAD_SHAPE, "n_seq=%lld block_size=%d max_blocks=%d num_blocks=%d",
                (long long)n_seq, block_size, max_blocks, num_blocks);
  if (tokens == 0) return TOME_OK;
  if (block_tables == nullptr || cache_positions == nullptr)
    return fail(TOME_ERR_NULL_POINTER, "a required pointer is NULL");
  return k6_launch<false>(p, dtype, static_cast<cudaStream_t>(stream), nullptr);
}

extern "C" size_t tome_qk_norm_rope_backward_workspace_bytes(int32_t head_dim) {
  if (head_dim <= 0 || head_dim > K6_MAX_DIM) return 0;
  return static_cast<size_t>(K6_MAX_BLOCKS) * 2 * head_dim * sizeof(float);
}

extern "C" int32_t tome_qk_norm_rope_backward(
    const void* grad_q, const void* grad_k, const void* grad_v, const void* qkv, int32_t dtype,
    int64_t tokens, int32_t heads, int32_t kv_heads, int32_t head_dim, int64_t qkv_stride,
    const void* q_weight, const void* k_weight, const float* cos_sin, int32_t n_positions,
    const int32_t* positions, float eps, void* grad_qkv, float* grad_q_weight,
    float* grad_k_weight, void* workspace, size_t workspace_bytes, int32_t* dev_status,
    void* stream) {
  K6Params p = {};
  p.qkv = qkv;
  p.qkv_stride = qkv_stride;
  p.q_weight = q_weight;
  p.k_weight = k_weight;
  p.cos_sin = cos_sin;
  p.n_positions = n_positions;
  p.positions = positions;
  p.tokens = tokens;
  p.heads = heads;
  p.kv_heads = kv_heads;
  p.dim = head_dim;
  p.eps = eps;
  p.grad_q = grad_q;
  p.grad_k = grad_k;
  p.grad_v = grad_v;
  p.grad_qkv = grad_qkv;
  p.partial = static_cast<float*>(workspace);
  p.status = dev_status;
  const void* required[] = {qkv, q_weight, k_weight, cos_sin, grad_q, grad_k, grad_qkv};
  int32_t st = k6_check(p, dtype, required, 7);
  if (st != TOME_OK) return st;
  if (grad_q_weight == nullptr || grad_k_weight == nullptr)
    return fail(TOME_ERR_NULL_POINTER, "a weight gradient is NULL");
  if (grad_v != nullptr && !aligned16(grad_v))
    return fail(TOME_ERR_MISALIGNED, "grad_v must be 16-byte aligned");
  if (workspace == nullptr || workspace_bytes < tome_qk_norm_rope_backward_workspace_bytes(head_dim))
    return fail(TOME_ERR_WORKSPACE_TOO_SMALL, "workspace of %zu bytes, %zu needed", workspace_bytes,
                tome_qk_norm_rope_backward_workspace_bytes(head_dim));
  if (!aligned16(workspace)) return fail(TOME_ERR_MISALIGNED, "workspace must be 16-byte aligned");
  int blocks = 0;
  if (tokens > 0) {
    st = k6_launch<true>(p, dtype, static_cast<cudaStream_t>(stream), &blocks);
    if (st != TOME_OK) return st;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((2 * head_dim + 31) / 32));
  cfg.blockDim = dim3(1024);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr;  // set up while the kernel before drains
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, k6_weight_grad_kernel,
                                       static_cast<const float*>(p.partial), blocks, head_dim,
                                       grad_q_weight, grad_k_weight),
                    "norm rope weight gradient launch");
}

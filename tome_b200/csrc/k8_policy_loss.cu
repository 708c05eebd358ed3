// K8: clipped policy loss with a KL term, and its gradient with respect to the logits
// (HBM-bound).  It is what the log-probs and the k3 KL of tome_dual_logprob_kl are computed
// for; the reference leaves the loss to its external trainer (no counterpart).
//
// For an active position with logits x, token t, T the temperature:
//   lp    = x[t]/T - logsumexp(x/T)
//   rho   = exp(lp - old),   a = advantage of the sequence
//   l     = -min(rho a, clamp(rho, 1 - clip_low, 1 + clip_high) a) + beta (exp(d) - d - 1),  d = ref - lp
//   loss  = sum of w l,  w = 1 / (active positions)  or  1 / (sequences * length of the sequence)
//   dl/dlp = -a rho [the first branch of the min is taken] + beta (1 - exp(d))
//   grad[j] = scale w dl/dlp (1[j = t] - softmax(x/T)[j]) / T
//
// A row is needed twice: for its sum of exponentials and for the gradient.  As in the
// full-matrix kernel a cluster of CTAs shares a row, each CTA streaming its part through a ring
// of bulk copies; pass 2 fetches the part again while it is still in L2, so that HBM sees the
// logits once and the gradient once.  Rows outside the windows are not read; their gradient is
// written as zeros by the same CTAs.
//
// Measured (CUDA-graph replay, vocabulary 151936, windows of random length): 32 x 256 bf16 rows 680 to
// 720 us (box to box), 5.2 to 5.5 TB/s (0.79 to 0.83 of a copy); 24 fp32 rows 12.4 to 13.2 us.  1080
// bf16 rows of 50257 50 us, 3.3 TB/s: few rows per cluster, which do not
// come out even.  Dealing the rows of the windows evenly among the clusters by a search in the prefix
// sums of their lengths took 46 to 48 us there, but 3.5 % more with many rows and 5 % with few.
#include "k1_common.cuh"
#include "row_geom.cuh"

namespace tome {

constexpr int K8_CONSUMER_WARPS = 8;
constexpr int K8_CONSUMERS = K8_CONSUMER_WARPS * 32;
constexpr int K8_THREADS = K8_CONSUMERS + 32;
constexpr int K8_SLOTS = 4;
constexpr int K8_CHUNK_BYTES = 25600;
constexpr int K8_MAX_CLUSTER = 8;
constexpr int K8_CTAS_PER_SM = 2;

struct K8Params {
  const void* logits;       // [n_seq * seq_len, vocab], contiguous
  void* grad;               // same shape, or null: no gradient
  int64_t rows, vocab;      // rows = n_seq * seq_len
  int32_t n_seq, seq_len;
  const int32_t* targets;   // [rows]
  const float* old_lp;      // [rows]
  const float* ref_lp;      // [rows] or null (no KL term)
  const float* advantages;  // [n_seq], or [rows] with adv_per_token
  const int32_t* lengths;   // [n_seq]
  const int32_t* starts;    // [n_seq] or null
  int32_t adv_per_token, per_sequence;
  float c, inv_temp;        // log2(e)/T, 1/T
  double inv_temp_64;
  float low, high, beta, scale;
  float* out_lp;            // [rows], 0 outside the windows
  float* out_loss;
  int32_t chunk_bytes;
  int32_t* status;
};

struct K8Smem {
  static constexpr int DATA = K8_SLOTS * K8_CHUNK_BYTES;
  static constexpr int FULL_BAR = DATA;
  static constexpr int EMPTY_BAR = FULL_BAR + K8_SLOTS * 8;
  static constexpr int XCHG_BAR = EMPTY_BAR + K8_SLOTS * 8;          // 2 (row parity)
  static constexpr int PART = XCHG_BAR + 16;                         // [2][WARPS] float2
  static constexpr int PAIRS = PART + 2 * K8_CONSUMER_WARPS * 8;     // [2][MAX_CLUSTER] float2
  static constexpr int BOX = PAIRS + 2 * K8_MAX_CLUSTER * 8;         // [2] float4
  static constexpr int TOTAL_LEN = BOX + 32;                         // int64
  static constexpr int TOTAL = TOTAL_LEN + 16;
};

__device__ __forceinline__ void k8_window(const K8Params& p, int i, int& start, int& len) {
  start = (p.starts != nullptr) ? p.starts[i] : 0;
  start = max(0, min(start, p.seq_len));
  len = max(0, min(p.lengths[i], p.seq_len - start));
}

// The loss of a position, and its slope in the log-prob, from lp - old and ref - lp.
struct K8Term {
  float l, slope;
};
__device__ __forceinline__ K8Term k8_term(const K8Params& p, float from_old, float d, float adv) {
  const float rho = expf(from_old);
  const float kept = fminf(fmaxf(rho, 1.0f - p.low), 1.0f + p.high);
  const bool open = !(rho * adv > kept * adv);  // a NaN takes this branch and stays one
  K8Term t;
  t.l = open ? -(rho * adv) : -(kept * adv);
  t.slope = open ? -(rho * adv) : 0.0f;
  if (p.ref_lp != nullptr) {
    const float em = expm1f(d);
    t.l = fmaf(p.beta, em - d, t.l);
    t.slope = fmaf(-p.beta, em, t.slope);
  }
  return t;
}

// Eight (four) logits -> gradient, away from the target column: k * 2^((x - m) c), k = -slope / s.
// x - m is formed first: with x c - m c a large maximum would leave its rounding in every term.
__device__ __forceinline__ uint32_t k8_grad_bf16x2(uint32_t w, float2 negm2, float2 c2, float2 k2) {
  const float2 d = __fmul2_rn(__fadd2_rn(make_float2(bf16_lo(w), bf16_hi(w)), negm2), c2);
  const float2 g = __fmul2_rn(make_float2(ex2f(d.x), ex2f(d.y)), k2);
  uint32_t o;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(o) : "f"(g.y), "f"(g.x));
  return o;
}

__device__ __forceinline__ uint4 k8_grad_vec(uint4 v, float m, float c, float k, __nv_bfloat16) {
  const float2 n2 = make_float2(-m, -m), c2 = make_float2(c, c), k2 = make_float2(k, k);
  uint4 o;
  o.x = k8_grad_bf16x2(v.x, n2, c2, k2);
  o.y = k8_grad_bf16x2(v.y, n2, c2, k2);
  o.z = k8_grad_bf16x2(v.z, n2, c2, k2);
  o.w = k8_grad_bf16x2(v.w, n2, c2, k2);
  return o;
}

__device__ __forceinline__ uint4 k8_grad_vec(uint4 v, float m, float c, float k, float) {
  uint4 o;
  o.x = __float_as_uint(k * ex2f((__uint_as_float(v.x) - m) * c));
  o.y = __float_as_uint(k * ex2f((__uint_as_float(v.y) - m) * c));
  o.z = __float_as_uint(k * ex2f((__uint_as_float(v.z) - m) * c));
  o.w = __float_as_uint(k * ex2f((__uint_as_float(v.w) - m) * c));
  return o;
}

__device__ __forceinline__ void k8_put(float* p, float v) { *p = v; }
__device__ __forceinline__ void k8_put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <typename T>
__global__ void __launch_bounds__(K8_THREADS, K8_CTAS_PER_SM)
k8_policy_loss_kernel(const K8Params p, const int cluster, const int chunks_per_cta) {
  extern __shared__ __align__(1024) uint8_t smem[];
  constexpr int ES = sizeof(T);
  const uint32_t smem_base = smem_u32(smem);
  const uint32_t full_bar = smem_base + K8Smem::FULL_BAR;
  const uint32_t empty_bar = smem_base + K8Smem::EMPTY_BAR;
  const uint32_t xchg_bar = smem_base + K8Smem::XCHG_BAR;
  float2* part = reinterpret_cast<float2*>(smem + K8Smem::PART);
  float2* pairs = reinterpret_cast<float2*>(smem + K8Smem::PAIRS);
  volatile float4* box = reinterpret_cast<volatile float4*>(smem + K8Smem::BOX);
  int64_t* total_len = reinterpret_cast<int64_t*>(smem + K8Smem::TOTAL_LEN);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int64_t n_clusters = gridDim.x / cluster;
  const int64_t first_row = blockIdx.x / cluster;

  if (threadIdx.x == 0) {
    for (int i = 0; i < K8_SLOTS; ++i) {
      mbar_init(full_bar + i * 8, 1);
      mbar_init(empty_bar + i * 8, K8_CONSUMER_WARPS);
    }
    mbar_init(xchg_bar, cluster > 1 ? cluster - 1 : 1);
    mbar_init(xchg_bar + 8, cluster > 1 ? cluster - 1 : 1);
    fence_mbar_init();
  }
  if (warp == 0 && !p.per_sequence) {  // active positions of the whole batch
    int64_t sum = 0;
    for (int i = lane; i < p.n_seq; i += 32) {
      int st, ln;
      k8_window(p, i, st, ln);
      sum += ln;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) *total_len = sum;
  }
  __syncthreads();
  griddep_launch_dependents();
  if (cluster > 1) cluster_sync_all();  // nobody arrives on a barrier that is not there yet

  const int64_t bulk_most = (p.vocab * ES) & ~static_cast<int64_t>(15);
  const int64_t chunk_bytes = p.chunk_bytes;
  const int64_t part_begin = static_cast<int64_t>(rank) * chunks_per_cta * chunk_bytes;
  int my_chunks = 0;
  for (int k = 0; k < chunks_per_cta; ++k)
    if (part_begin + k * chunk_bytes < bulk_most) ++my_chunks;
  const bool owns_ends = (rank == static_cast<uint32_t>(cluster) - 1);
  const int passes = p.grad != nullptr ? 2 : 1;
  auto chunk_size = [&](int64_t bulk_bytes, int k) {
    return static_cast<uint32_t>(
        max(int64_t{0}, min(chunk_bytes, bulk_bytes - part_begin - k * chunk_bytes)));
  };

  if (warp == K8_CONSUMER_WARPS) {
    // ---------------- producer
    if (lane == 0) {
      const uint64_t policy = policy_evict_first();
      uint32_t it = 0;
      bool ok = true;
      for (int64_t row = first_row; row < p.rows && ok; row += n_clusters) {
        const int seq = static_cast<int>(row / p.seq_len);
        const int pos = static_cast<int>(row - static_cast<int64_t>(seq) * p.seq_len);
        int st, ln;
        k8_window(p, seq, st, ln);
        if (pos < st || pos >= st + ln) continue;
        const T* row_src = reinterpret_cast<const T*>(p.logits) + row * p.vocab;
        const K1RowGeom geom = k1_row_geom(row_src, p.vocab);
        const uint8_t* src = reinterpret_cast<const uint8_t*>(row_src + geom.head) + part_begin;
        for (int pass = 0; pass < passes && ok; ++pass) {
          for (int k = 0; k < my_chunks; ++k, ++it) {
            const uint32_t slot = it % K8_SLOTS;
            const uint32_t phase = (it / K8_SLOTS) & 1u;
            if (!mbar_wait(empty_bar + slot * 8, phase ^ 1u)) {
              raise_status(p.status, TOME_DEV_TIMEOUT);
              ok = false;
              break;
            }
            const int64_t off = k * chunk_bytes;
            const uint32_t bytes = chunk_size(geom.bulk_bytes, k);
            mbar_arrive_expect_tx(full_bar + slot * 8, bytes);
            if (bytes == 0) continue;
            if (pass == passes - 1)  // the last use
              bulk_g2s_hint(smem_base + slot * K8_CHUNK_BYTES, src + off, bytes,
                            full_bar + slot * 8, policy);
            else
              bulk_g2s(smem_base + slot * K8_CHUNK_BYTES, src + off, bytes, full_bar + slot * 8);
          }
        }
      }
    }
    __syncwarp();
  } else {
    // ---------------- consumers.  One whose wait ran out stops touching data but stays in step
    // with its cluster.
    const int ctid = threadIdx.x;
    uint32_t it = 0;
    uint32_t row_it = 0;
    bool dead = false;
    for (int64_t row = first_row; row < p.rows; row += n_clusters) {
      const int seq = static_cast<int>(row / p.seq_len);
      const int pos = static_cast<int>(row - static_cast<int64_t>(seq) * p.seq_len);
      int win_start, win_len;
      k8_window(p, seq, win_start, win_len);
      const T* src = reinterpret_cast<const T*>(p.logits) + row * p.vocab;
      T* dst = reinterpret_cast<T*>(p.grad) + row * p.vocab;
      const K1RowGeom geom = k1_row_geom(src, p.vocab);  // the gradient's row sits alike
      if (pos < win_start || pos >= win_start + win_len) {
        if (p.grad != nullptr) {
          for (int k = 0; k < my_chunks; ++k) {
            const uint32_t nvec = chunk_size(geom.bulk_bytes, k) >> 4;
            uint8_t* drow = reinterpret_cast<uint8_t*>(dst + geom.head) + part_begin + k * chunk_bytes;
            for (uint32_t v = ctid; v < nvec; v += K8_CONSUMERS)
              stg128_streaming(drow + static_cast<size_t>(v) * 16, make_uint4(0, 0, 0, 0));
          }
          if (owns_ends && ctid == 0) {
            for (int64_t j = 0; j < geom.head; ++j) k8_put(dst + j, 0.0f);
            for (int64_t j = geom.tail_begin; j < p.vocab; ++j) k8_put(dst + j, 0.0f);
          }
        }
        if (rank == 0 && ctid == 0) {
          p.out_lp[row] = 0.0f;
        }
        continue;
      }
      const uint32_t par = row_it & 1u;
      const int64_t target = p.targets[row];
      const bool target_ok = target >= 0 && target < p.vocab;
      // what the first warp needs of the row besides its sum, asked for ahead of the stream
      float x_t = 0.0f, old_lp = 0.0f, ref_lp = 0.0f, adv = 0.0f;
      if (warp == 0) {
        x_t = target_ok ? to_float(src[target]) : __int_as_float(0x7fc00000);
        old_lp = p.old_lp[row];
        ref_lp = p.ref_lp != nullptr ? p.ref_lp[row] : 0.0f;
        adv = p.advantages[p.adv_per_token ? row : seq];
      }
      // ---- pass 1: (m, s) of this CTA's part
      Fast fs;
      fast_init(fs, p.c);
      for (int k = 0; k < my_chunks; ++k) {
        const uint32_t slot = (it + k) % K8_SLOTS;
        const uint32_t phase = ((it + k) / K8_SLOTS) & 1u;
        if (!dead && !mbar_wait(full_bar + slot * 8, phase)) {
          raise_status(p.status, TOME_DEV_TIMEOUT);
          dead = true;
        }
        if (dead) break;
        const uint32_t nvec = chunk_size(geom.bulk_bytes, k) >> 4;
        const uint32_t sbase = smem_base + slot * K8_CHUNK_BYTES;
#pragma unroll 4
        for (uint32_t v = ctid; v < nvec; v += K8_CONSUMERS)
          fast_update<0>(fs, lds128(sbase + v * 16), p.c, T());
        __syncwarp();
        if (lane == 0) mbar_arrive(empty_bar + slot * 8);
      }
      it += static_cast<uint32_t>(my_chunks);
      Online st = fast_finish(fs, p.c);
      if (owns_ends && ctid == 0) {
        for (int64_t j = 0; j < geom.head; ++j) online_update_scalar(st, to_float(src[j]), p.c);
        for (int64_t j = geom.tail_begin; j < p.vocab; ++j)
          online_update_scalar(st, to_float(src[j]), p.c);
      }
      online_warp_reduce(st, p.c);
      if (lane == 0) part[par * K8_CONSUMER_WARPS + warp] = make_float2(st.m, st.s);
      named_bar_sync(1, K8_CONSUMERS);
      if (warp == 0) {
        const float2 w = (lane < K8_CONSUMER_WARPS) ? part[par * K8_CONSUMER_WARPS + lane]
                                                    : make_float2(-FLT_MAX, 0.0f);
        Online cta = {w.x, w.y};
        online_warp_reduce(cta, p.c);
        if (lane < cluster) {
          if (static_cast<uint32_t>(lane) == rank) {
            pairs[par * K8_MAX_CLUSTER + rank] = make_float2(cta.m, cta.s);
          } else {
            st_cluster_f32x2(mapa_shared(smem_u32(&pairs[par * K8_MAX_CLUSTER + rank]), lane),
                             cta.m, cta.s);
            mbar_arrive_cluster(mapa_shared(xchg_bar + par * 8, lane));
          }
        }
        __syncwarp();
        bool ok = true;
        if (cluster > 1) ok = mbar_wait_cluster(xchg_bar + par * 8, (row_it >> 1) & 1u);
        const float2 o = (lane < cluster) ? pairs[par * K8_MAX_CLUSTER + lane]
                                          : make_float2(-FLT_MAX, 0.0f);
        Online all = {o.x, o.y};
        online_warp_reduce(all, p.c);
        float m = all.m, s = all.s;
        if (!(s >= 0.5f && s <= FLT_MAX)) exact_row(src, p.vocab, p.c, lane, m, s);
        // The difference to the maximum first: x_t / T - (m / T + log s) rounds three times at the size
        // of m / T.  It stays in 64 bits until the other log-prob is taken off, since the ratio
        // multiplies the whole row of gradients (its relative error, rms over 60 modelled rows with a
        // largest logit of 12: 7e-7 in the first form, 6e-7 with 32-bit differences, 7e-8 so).
        double lp = (static_cast<double>(x_t) - static_cast<double>(m)) * p.inv_temp_64 -
                    static_cast<double>(logf(s));
        if (!ok) {  // a peer never delivered: report, poison the row, keep the CTA in step
          raise_status(p.status, TOME_DEV_TIMEOUT);
          lp = static_cast<double>(__int_as_float(0x7fc00000));
        }
        const float slope = k8_term(p, static_cast<float>(lp - static_cast<double>(old_lp)),
                                    static_cast<float>(static_cast<double>(ref_lp) - lp), adv).slope;
        const float weight =
            p.per_sequence ? 1.0f / (static_cast<float>(p.n_seq) * static_cast<float>(win_len))
                           : 1.0f / static_cast<float>(*total_len);
        const float g = slope * weight * p.scale * p.inv_temp;
        if (lane == 0) {
          box[par].x = m;
          box[par].y = -g / s;
          box[par].z = fmaf(-g / s, ex2f((x_t - m) * p.c), g);  // the target column's gradient
          if (rank == 0) {
            p.out_lp[row] = static_cast<float>(lp);
            if (!target_ok) raise_status(p.status, TOME_DEV_TARGET_OUT_OF_RANGE);
          }
        }
      }
      ++row_it;
      named_bar_sync(1, K8_CONSUMERS);
      if (p.grad == nullptr) continue;
      const float m = box[par].x, kf = box[par].y, g_t = box[par].z;
      // the target column: byte offset in the body (behind the head), or an end element
      const int64_t t_off = target_ok ? (target - geom.head) * ES - part_begin : -1;
      // ---- pass 2: gradients; a slot is released once it is written out
      for (int k = 0; k < my_chunks; ++k, ++it) {
        const uint32_t slot = it % K8_SLOTS;
        if (!dead && !mbar_wait(full_bar + slot * 8, (it / K8_SLOTS) & 1u)) {
          raise_status(p.status, TOME_DEV_TIMEOUT);
          dead = true;
        }
        const int64_t off = k * chunk_bytes;
        const uint32_t bytes = chunk_size(geom.bulk_bytes, k);
        const uint32_t nvec = dead ? 0u : (bytes >> 4);
        const uint32_t sbase = smem_base + slot * K8_CHUNK_BYTES;
        uint8_t* drow = reinterpret_cast<uint8_t*>(dst + geom.head) + part_begin + off;
#pragma unroll 4
        for (uint32_t v = ctid; v < nvec; v += K8_CONSUMERS)
          stg128_streaming(drow + static_cast<size_t>(v) * 16,
                           k8_grad_vec(lds128(sbase + v * 16), m, p.c, kf, T()));
        // the target's element, written over by the thread that wrote its vector
        if (t_off >= off && t_off < off + static_cast<int64_t>(nvec) * 16 &&
            ((t_off - off) >> 4) % K8_CONSUMERS == ctid)
          k8_put(dst + target, g_t);
        __syncwarp();
        if (lane == 0) mbar_arrive(empty_bar + slot * 8);
      }
      if (owns_ends && ctid == 0) {
        for (int64_t j = 0; j < geom.head; ++j)
          k8_put(dst + j, j == target ? g_t : kf * ex2f((to_float(src[j]) - m) * p.c));
        for (int64_t j = geom.tail_begin; j < p.vocab; ++j)
          k8_put(dst + j, j == target ? g_t : kf * ex2f((to_float(src[j]) - m) * p.c));
      }
    }
  }
  // no CTA leaves while a peer may still store into its shared memory or arrive on its barriers
  if (cluster > 1) cluster_sync_all();
}

// loss = sum of w l over the windows, from the log-probs that the kernel above left, in 64 bits and
// in an order that depends on the sizes alone.
__global__ void __launch_bounds__(1024) k8_sum_kernel(const K8Params p) {
  __shared__ double sums[32];
  __shared__ int64_t counts[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  griddep_wait();
  double s = 0.0;
  int64_t active = 0;
  for (int64_t i = threadIdx.x; i < p.rows; i += 1024) {
    const int seq = static_cast<int>(i / p.seq_len);
    const int pos = static_cast<int>(i - static_cast<int64_t>(seq) * p.seq_len);
    int st, ln;
    k8_window(p, seq, st, ln);
    if (pos < st || pos >= st + ln) continue;
    const float lp = p.out_lp[i];
    const float l = k8_term(p, lp - p.old_lp[i], p.ref_lp != nullptr ? p.ref_lp[i] - lp : 0.0f,
                            p.advantages[p.adv_per_token ? i : seq]).l;
    s += p.per_sequence ? static_cast<double>(l) / (static_cast<double>(p.n_seq) * ln) : static_cast<double>(l);
    ++active;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    active += __shfl_xor_sync(0xffffffffu, active, o);
  }
  if (lane == 0) {
    sums[warp] = s;
    counts[warp] = active;
  }
  __syncthreads();
  if (warp == 0) {
    s = sums[lane];
    active = counts[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      active += __shfl_xor_sync(0xffffffffu, active, o);
    }
    if (lane == 0)
      *p.out_loss = static_cast<float>(p.per_sequence || active == 0 ? s : s / static_cast<double>(active));
  }
}

// Chunks of a row for a cluster: `n` per CTA, equal, on 1 KB boundaries (short rows: 16 bytes
// would do, but nothing is gained), at most one ring slot long.
static void k8_plan(int64_t bulk_bytes, int cluster, int* chunks_per_cta, int32_t* chunk_bytes) {
  const int64_t al = K1_CHUNK_ALIGN;
  const int64_t per_cta = (bulk_bytes + cluster - 1) / cluster;
  int64_t n = std::max<int64_t>(1, (per_cta + K8_CHUNK_BYTES - 1) / K8_CHUNK_BYTES);
  auto size = [&](int64_t k) {
    const int64_t total = k * cluster;
    return std::max<int64_t>(al, ((bulk_bytes + total - 1) / total + al - 1) / al * al);
  };
  while (size(n) > K8_CHUNK_BYTES) ++n;  // rounding pushed a chunk over the slot
  *chunks_per_cta = static_cast<int>(n);
  *chunk_bytes = static_cast<int32_t>(size(n));
}

template <typename T>
static int32_t k8_launch(K8Params p, int sm_count, cudaStream_t stream) {
  void (*kernel)(K8Params, int, int) = k8_policy_loss_kernel<T>;
  const void* fn = reinterpret_cast<const void*>(kernel);
  int32_t st = ensure_dynamic_smem(fn, K8Smem::TOTAL);
  if (st != TOME_OK) return st;
  // As for the full-matrix kernel: the smallest cluster whose CTAs get at most 160 KB of a row
  // (the rows in flight then stay in L2 between the passes); with fewer rows than clusters a
  // row is spread wider, while that still finds SMs without work.
  const int64_t bulk_bytes = (p.vocab * static_cast<int64_t>(sizeof(T))) & ~15ll;
  int cluster = 1;
  while (cluster < K8_MAX_CLUSTER && bulk_bytes > 160 * 1024 * static_cast<int64_t>(cluster))
    cluster <<= 1;
  while (cluster < K8_MAX_CLUSTER && p.rows * cluster * 2 <= sm_count * K8_CTAS_PER_SM &&
         bulk_bytes >= 8192 * static_cast<int64_t>(cluster))
    cluster <<= 1;
  int chunks_per_cta = 0;
  k8_plan(bulk_bytes, cluster, &chunks_per_cta, &p.chunk_bytes);
  int fit = max_active_clusters(fn, K8_THREADS, K8Smem::TOTAL, cluster);
  if (fit <= 0) fit = std::max(1, sm_count * K8_CTAS_PER_SM / cluster);
  const int64_t n_clusters = std::max<int64_t>(1, std::min<int64_t>(fit, p.rows));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(n_clusters * cluster), 1, 1);
  cfg.blockDim = dim3(K8_THREADS, 1, 1);
  cfg.dynamicSmemBytes = K8Smem::TOTAL;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = static_cast<unsigned>(cluster);
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  st = check_cuda(cudaLaunchKernelEx(&cfg, kernel, p, cluster, chunks_per_cta), "policy loss launch");
  if (st != TOME_OK) return st;
  cudaLaunchConfig_t sum = {};
  sum.gridDim = dim3(1);
  sum.blockDim = dim3(1024);
  sum.stream = stream;
  cudaLaunchAttribute early;  // set up while the kernel before drains
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  sum.attrs = &early;
  sum.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&sum, k8_sum_kernel, p), "policy loss sum launch");
}

}  // namespace tome

using namespace tome;

extern "C" int32_t tome_grpo_policy_loss(
    const void* logits, int32_t dtype, int64_t n_seq, int64_t seq_len, int64_t vocab,
    const int32_t* targets, const float* old_logprob, const float* ref_logprob,
    const float* advantages, int32_t advantage_per_token, const int32_t* lengths,
    const int32_t* starts, float temperature, float clip_low, float clip_high, float kl_coef,
    int32_t per_sequence, float grad_scale, float* out_loss, float* out_logprob, void* out_grad,
    int32_t* dev_status, void* stream) {
  if (dtype != TOME_F32 && dtype != TOME_BF16) return fail(TOME_ERR_BAD_DTYPE, "dtype=%d", dtype);
  if (n_seq < 0 || seq_len < 0 || vocab <= 0 || n_seq > 0x7fffffff || seq_len > 0x7fffffff)
    return fail(TOME_ERR_BAD_SHAPE, "n_seq=%lld seq_len=%lld vocab=%lld", (long long)n_seq,
                (long long)seq_len, (long long)vocab);
  if (!temperature_ok(temperature))
    return fail(TOME_ERR_BAD_TEMPERATURE, "temperature=%g must be positive and finite",
                (double)temperature);
  if (!(clip_low >= 0.0f) || !(clip_high >= 0.0f) || !(kl_coef >= 0.0f) || clip_low > 3.0e38f ||
      clip_high > 3.0e38f || kl_coef > 3.0e38f || !(grad_scale >= -3.0e38f && grad_scale <= 3.0e38f))
    return fail(TOME_ERR_BAD_SHAPE, "clip_low=%g clip_high=%g kl_coef=%g grad_scale=%g",
                (double)clip_low, (double)clip_high, (double)kl_coef, (double)grad_scale);
  if (out_loss == nullptr) return fail(TOME_ERR_NULL_POINTER, "out_loss is NULL");
  const int64_t rows = n_seq * seq_len;
  K8Params p = {};
  p.rows = rows;
  p.out_loss = out_loss;
  if (rows > 0) {
    if (logits == nullptr || targets == nullptr || old_logprob == nullptr || advantages == nullptr ||
        lengths == nullptr || out_logprob == nullptr)
      return fail(TOME_ERR_NULL_POINTER, "a required pointer is NULL");
    if (kl_coef != 0.0f && ref_logprob == nullptr)
      return fail(TOME_ERR_NULL_POINTER, "kl_coef=%g without ref_logprob", (double)kl_coef);
    if (!aligned16(logits) || (out_grad != nullptr && !aligned16(out_grad)))
      return fail(TOME_ERR_MISALIGNED, "logits and the gradient must be 16-byte aligned");
  }
  DeviceInfo info;
  const int32_t st = current_device_info(&info);
  if (st != TOME_OK) return st;
  if (rows == 0) {
    k8_sum_kernel<<<1, 1024, 0, static_cast<cudaStream_t>(stream)>>>(p);
    return check_cuda(cudaGetLastError(), "policy loss sum launch");
  }
  p.logits = logits;
  p.grad = out_grad;
  p.vocab = vocab;
  p.n_seq = static_cast<int32_t>(n_seq);
  p.seq_len = static_cast<int32_t>(seq_len);
  p.targets = targets;
  p.old_lp = old_logprob;
  p.ref_lp = kl_coef != 0.0f ? ref_logprob : nullptr;
  p.advantages = advantages;
  p.lengths = lengths;
  p.starts = starts;
  p.adv_per_token = advantage_per_token;
  p.per_sequence = per_sequence;
  p.c = LOG2E / temperature;
  p.inv_temp = 1.0f / temperature;
  p.inv_temp_64 = 1.0 / static_cast<double>(temperature);
  p.low = clip_low;
  p.high = clip_high;
  p.beta = kl_coef;
  p.scale = grad_scale;
  p.out_lp = out_logprob;
  p.status = dev_status;
  if (dtype == TOME_F32) return k8_launch<float>(p, info.sm_count, static_cast<cudaStream_t>(stream));
  return k8_launch<__nv_bfloat16>(p, info.sm_count, static_cast<cudaStream_t>(stream));
}

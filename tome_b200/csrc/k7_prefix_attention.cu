// K7: single-token attention over a paged KV cache whose prefix is shared by a group of
// sequences (HBM-bound: each prefix is read once for its whole group, each suffix once).
//
// A GRPO rollout draws G completions of one prompt; the reference copies the prompt's cache G
// times and lets every copy be read (mlx-impl/node.py:529-555, model.py:428).  Here the pages of
// the prompt are named by the group's table and the pages of a completion by the sequence's.
// For query head h of sequence b (its KV head is h / (heads / kv_heads)):
//   o = softmax(scale q [K_prefix; K_suffix]^T) [V_prefix; V_suffix].
//
// Work.  An item is (KV head, up to 128 query rows that read the same keys): the rows of a
// group against its prefix, or of one sequence against its suffix.  Items are cut into tiles of
// 64 keys, all tiles are laid end to end and every CTA takes an equal run of them, whatever the
// lengths: the split follows from the lengths on the device alone.  A CTA's part of an item is a
// piece; it leaves (sum of p v, row maximum, row sum) in the workspace, and a second kernel
// joins the pieces of a row.  A row's pieces lie at (item index + CTA index), which no two pieces
// share since at least one of the two grows from piece to piece.
//
// Pipeline of a CTA (one per SM): two warps copy keys and values (16-byte asynchronous copies:
// pages of any size, rows past the end filled with zeros) into a ring of three stages, one
// thread issues the tensor-core products S = Q K^T (128 x 64 x D) and O = P V (128 x D x 64),
// four warps own a row per thread: running maximum and sum, P rounded to the type of V
// into shared memory, O added up in registers.  S, P and O are double-buffered, so the product
// of one tile, the softmax of the next and the loads of the ones behind it overlap.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>

#include <algorithm>
#include <type_traits>

#include "host_common.h"
#include "ptx.cuh"

namespace tome {

constexpr int K7_ROWS = 128;   // query rows of an item (TMEM lanes)
constexpr int K7_KEYS = 64;    // keys of a tile
constexpr int K7_STAGES = 3;
constexpr int K7_SOFTMAX_WARPS = 4;
constexpr int K7_MMA_WARP = 4;
constexpr int K7_COPY_THREADS = 64;
constexpr int K7_THREADS = (K7_SOFTMAX_WARPS + 1) * 32 + K7_COPY_THREADS;
constexpr int K7_MAX_SEQ = 4096;
constexpr int K7_MAX_GROUPS = 1024;

struct K7Params {
  const void* q;              // [n_seq, heads, D], sequence stride q_stride
  int64_t q_stride;
  const void* k_pool;         // [num_blocks, kv_heads, block_size, D]
  const void* v_pool;
  const int32_t* prefix_tables;  // [n_groups, prefix_blocks]
  const int32_t* prefix_lens;    // [n_groups]
  const int32_t* group_starts;   // [n_groups + 1]
  const int32_t* tables;         // [n_seq, seq_blocks]
  const int32_t* lengths;        // [n_seq]
  int32_t n_seq, n_groups, heads, kv_heads, ratio, block_size, prefix_blocks, seq_blocks, num_blocks;
  uint32_t div_magic;         // key / block_size = (key * div_magic) >> div_shift
  int32_t div_shift;
  float c;                    // scale * log2(e)
  int32_t ctas;               // CTAs of the main kernel
  // workspace
  int32_t* plan;              // [0]: tiles in all; then int4 [n_seq] and int2 [n_seq], see K7Plan
  float* prefix_o;            // [prefix slots, 128, D]
  float2* prefix_ml;          // [prefix slots, 128] (maximum * c, sum)
  float* suffix_o;            // [suffix slots, ratio, D]
  float2* suffix_ml;          // [suffix slots, ratio]
  void* out;                  // [n_seq, heads, D]
  float* out_lse;             // [n_seq, heads] or null
  int32_t* status;
};

__device__ __forceinline__ void k7_raise(int32_t* status, int32_t bit) {
  if (status != nullptr) atomicOr(status, bit);
}

// Length of a table's keys: never negative, never past the table.
__device__ __forceinline__ int32_t k7_length(const K7Params& p, int32_t len, int32_t blocks) {
  const int64_t most = static_cast<int64_t>(blocks) * p.block_size;
  return static_cast<int32_t>(max(int64_t{0}, min(static_cast<int64_t>(len), most)));
}

// What every CTA works out of the lengths, in shared memory.
struct K7Plan {
  int32_t* group;   // [n_groups + 1] first sequence of each group (clamped, not decreasing)
  int32_t* block;   // [n_groups + 1] row blocks (of 128 rows) before each group
  int32_t* prefix;  // [n_groups + 1] prefix tiles before each group, all KV heads
  int32_t* suffix;  // [n_seq + 1] suffix tiles before each sequence, all KV heads
};

__device__ __forceinline__ int32_t k7_tiles(int32_t len) { return (len + K7_KEYS - 1) / K7_KEYS; }

__device__ __forceinline__ int32_t k7_scan_add(int32_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int32_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}
__device__ __forceinline__ int32_t k7_scan_max(int32_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int32_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = max(v, u);
  }
  return v;
}

// Warp 0: the groups; warp 1: the sequences.
__device__ __forceinline__ void k7_build_plan(const K7Params& p, const K7Plan& pl, int warp, int lane) {
  if (warp == 0) {
    int32_t top = 0;
    for (int base = 0; base <= p.n_groups; base += 32) {
      const int i = base + lane;
      int32_t v = (i <= p.n_groups && p.n_groups > 0) ? p.group_starts[i] : 0;
      v = max(top, k7_scan_max(min(max(v, 0), p.n_seq), lane));
      if (i <= p.n_groups) pl.group[i] = v;
      top = __shfl_sync(0xffffffffu, v, 31);
    }
    __syncwarp();
    int32_t blocks = 0, tiles = 0;
    for (int base = 0; base < p.n_groups; base += 32) {
      const int i = base + lane;
      int32_t b = 0, t = 0;
      if (i < p.n_groups) {
        b = ((pl.group[i + 1] - pl.group[i]) * p.ratio + K7_ROWS - 1) / K7_ROWS;
        t = b * p.kv_heads * k7_tiles(k7_length(p, p.prefix_lens[i], p.prefix_blocks));
      }
      const int32_t bs = k7_scan_add(b, lane), ts = k7_scan_add(t, lane);
      if (i < p.n_groups) {
        pl.block[i] = blocks + bs - b;
        pl.prefix[i] = tiles + ts - t;
      }
      blocks += __shfl_sync(0xffffffffu, bs, 31);
      tiles += __shfl_sync(0xffffffffu, ts, 31);
    }
    if (lane == 0) {
      pl.block[p.n_groups] = blocks;
      pl.prefix[p.n_groups] = tiles;
    }
  } else if (warp == 1) {
    int32_t tiles = 0;
    for (int base = 0; base < p.n_seq; base += 32) {
      const int i = base + lane;
      int32_t t = 0;
      if (i < p.n_seq) t = p.kv_heads * k7_tiles(k7_length(p, p.lengths[i], p.seq_blocks));
      const int32_t ts = k7_scan_add(t, lane);
      if (i < p.n_seq) pl.suffix[i] = tiles + ts - t;
      tiles += __shfl_sync(0xffffffffu, ts, 31);
    }
    if (lane == 0) pl.suffix[p.n_seq] = tiles;
  }
}

// The CTAs that take part (each has a tile, so that an item's pieces lie in neighbouring ones),
// the first tile of one of them, and the one that holds a tile.
__device__ __forceinline__ int32_t k7_working(int32_t tiles, int32_t ctas) { return min(tiles, ctas); }
__device__ __forceinline__ int32_t k7_first_tile(int32_t tiles, int32_t ctas, int32_t cta) {
  return static_cast<int32_t>(static_cast<int64_t>(cta) * tiles / ctas);
}
__device__ __forceinline__ int32_t k7_cta_of(int32_t tiles, int32_t ctas, int32_t tile) {
  return static_cast<int32_t>(((static_cast<int64_t>(tile) + 1) * ctas + tiles - 1) / tiles - 1);
}

// A piece: tiles [tile, tile + n) of an item.
struct K7Piece {
  const int32_t* table;
  int32_t len;        // keys of the item
  int32_t tile, n;
  int32_t kv_head;
  int32_t seq0;       // first sequence of the rows
  int32_t row0;       // first row (row = (sequence - seq0) * ratio + head within the KV head)
  int32_t rows;
  int32_t item;       // index among the prefix or suffix items
  bool prefix;
};

// largest i in [0, n) with cum[i] <= x (cum not decreasing, cum[0] = 0 <= x < cum[n])
__device__ __forceinline__ int k7_find(const int32_t* cum, int n, int32_t x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cum[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// The piece that begins at tile `at` (of all tiles) and ends at the item's end or at `end`.
__device__ __forceinline__ K7Piece k7_piece(const K7Params& p, const K7Plan& pl, int32_t at, int32_t end) {
  K7Piece x;
  const int32_t in_prefix = pl.prefix[p.n_groups];
  x.prefix = at < in_prefix;
  if (x.prefix) {
    const int g = k7_find(pl.prefix, p.n_groups, at);
    x.len = k7_length(p, p.prefix_lens[g], p.prefix_blocks);
    const int32_t tiles = k7_tiles(x.len), rem = at - pl.prefix[g];
    const int32_t i = rem / tiles;  // (row block, KV head)
    x.tile = rem - i * tiles;
    x.n = min(tiles - x.tile, end - at);
    const int32_t mb = i / p.kv_heads;
    x.kv_head = i - mb * p.kv_heads;
    x.seq0 = pl.group[g];
    x.row0 = mb * K7_ROWS;
    x.rows = min(K7_ROWS, (pl.group[g + 1] - x.seq0) * p.ratio - x.row0);
    x.item = (pl.block[g] + mb) * p.kv_heads + x.kv_head;
    x.table = p.prefix_tables + static_cast<int64_t>(g) * p.prefix_blocks;
  } else {
    const int b = k7_find(pl.suffix, p.n_seq, at - in_prefix);
    x.len = k7_length(p, p.lengths[b], p.seq_blocks);
    const int32_t tiles = k7_tiles(x.len), rem = at - in_prefix - pl.suffix[b];
    x.kv_head = rem / tiles;
    x.tile = rem - x.kv_head * tiles;
    x.n = min(tiles - x.tile, end - at);
    x.seq0 = b;
    x.row0 = 0;
    x.rows = p.ratio;
    x.item = b * p.kv_heads + x.kv_head;
    x.table = p.tables + static_cast<int64_t>(b) * p.seq_blocks;
  }
  return x;
}

// ------------------------------------------------------------------ shared memory and products
// Tiles of 128-byte rows, 128-byte swizzle: 16-byte piece c of row r of a 64-column block sits
// at r * 128 + ((c ^ (r & 7)) << 4).
template <int D>
struct K7Smem {
  static constexpr int TMEM_COLS = D == 64 ? 256 : 512;    // S 2 x 64, O 2 x D, a power of two
  static constexpr int Q_BYTES = K7_ROWS * D * 2;
  static constexpr int KV_BYTES = K7_KEYS * D * 2;
  static constexpr int P_BYTES = K7_ROWS * K7_KEYS * 2;
  static constexpr int STAGE = 2 * KV_BYTES;
  static constexpr int Q = 0;                              // 2 buffers (piece parity)
  static constexpr int P = Q + 2 * Q_BYTES;                // 2 buffers (tile parity)
  static constexpr int KV = P + 2 * P_BYTES;
  static constexpr int BARS = KV + K7_STAGES * STAGE;
  static constexpr int FULL = BARS;                        // STAGES
  static constexpr int EMPTY = FULL + K7_STAGES * 8;       // STAGES
  static constexpr int S_FULL = EMPTY + K7_STAGES * 8;     // 2
  static constexpr int P_FULL = S_FULL + 16;               // 2
  static constexpr int O_FULL = P_FULL + 16;               // 2
  static constexpr int Q_EMPTY = O_FULL + 16;              // 2
  static constexpr int TMEM = Q_EMPTY + 16;
  static constexpr int PLAN = TMEM + 16;
  static constexpr int plan_bytes(int n_groups, int n_seq) {
    return 4 * (3 * (n_groups + 1) + n_seq + 1);
  }
};

// K-major operand tile (rows of 128 bytes, 8-row groups 1024 bytes apart).
__device__ __forceinline__ uint64_t k7_desc_k(uint32_t addr) {
  return static_cast<uint64_t>((addr & 0x3ffffu) >> 4) | (static_cast<uint64_t>(1) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) |
         (static_cast<uint64_t>(2) << 61);
}
// The same bytes read with the row index as the contraction (MN-major): blocks of 64 columns
// `block_bytes` apart, groups of eight rows 1024 bytes apart.
__device__ __forceinline__ uint64_t k7_desc_mn(uint32_t addr, uint32_t block_bytes) {
  return static_cast<uint64_t>((addr & 0x3ffffu) >> 4) |
         (static_cast<uint64_t>(block_bytes >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) |
         (static_cast<uint64_t>(2) << 61);
}

// kind::f16 instruction descriptor, fp32 accumulator, A and B of type T; B MN-major if asked.
template <typename T>
__host__ __device__ constexpr uint32_t k7_idesc(int n, bool b_mn) {
  const uint32_t f = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | ((b_mn ? 1u : 0u) << 16) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(K7_ROWS >> 4) << 24);
}

__device__ __forceinline__ void k7_copy16(uint32_t dst, const void* src, bool there) {
  const uint32_t bytes = there ? 16u : 0u;  // 0: the 16 bytes are filled with zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
// The barrier counts this thread once all its copies so far have landed.
__device__ __forceinline__ void k7_copies_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ uint32_t k7_pack(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __float22bfloat162_rn(make_float2(a, b));
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t k7_pack(float a, float b, __half) {
  const __half2 h = __float22half2_rn(make_float2(a, b));
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void k7_sts128(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(K7_THREADS, 1) k7_attention_kernel(const K7Params p) {
  using S = K7Smem<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;  // swizzled tiles want 1024-byte alignment
  uint8_t* smem = smem_raw + (base - raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  K7Plan pl;
  pl.group = reinterpret_cast<int32_t*>(smem + S::PLAN);
  pl.block = pl.group + p.n_groups + 1;
  pl.prefix = pl.block + p.n_groups + 1;
  pl.suffix = pl.prefix + p.n_groups + 1;

  if (threadIdx.x == K7_MMA_WARP * 32) {
    for (int i = 0; i < K7_STAGES; ++i) {
      mbar_init(base + S::FULL + i * 8, K7_COPY_THREADS);
      mbar_init(base + S::EMPTY + i * 8, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(base + S::S_FULL + i * 8, 1);
      mbar_init(base + S::P_FULL + i * 8, K7_SOFTMAX_WARPS);
      mbar_init(base + S::O_FULL + i * 8, 1);
      mbar_init(base + S::Q_EMPTY + i * 8, 1);
    }
    fence_mbar_init();
  }
  if (warp == K7_MMA_WARP) {
    __syncwarp();
    tmem_alloc(base + S::TMEM, S::TMEM_COLS);
    tmem_relinquish();
  }
  k7_build_plan(p, pl, warp, lane);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + S::TMEM);
  const int32_t tiles = pl.prefix[p.n_groups] + pl.suffix[p.n_seq];
  const int32_t working = k7_working(tiles, p.ctas);
  const bool works = static_cast<int32_t>(blockIdx.x) < working;
  const int32_t first = works ? k7_first_tile(tiles, working, blockIdx.x) : 0;
  const int32_t last = works ? k7_first_tile(tiles, working, blockIdx.x + 1) : 0;
  griddep_launch_dependents();

  if (warp < K7_SOFTMAX_WARPS) {
    // ------------------------------------------------------------ softmax: thread = row
    const int row = threadIdx.x;
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    uint32_t t = 0;
    bool ok = true;
    // the sequences' places for the joining kernel, dealt over the CTAs
    for (int b = blockIdx.x * K7_SOFTMAX_WARPS * 32 + threadIdx.x; b < p.n_seq;
         b += gridDim.x * K7_SOFTMAX_WARPS * 32) {
      int4 a = make_int4(0, 0, 0, 0);  // row within the group, row blocks and tiles before it, tiles per item
      if (p.n_groups > 0 && b >= pl.group[0] && b < pl.group[p.n_groups]) {
        const int g = k7_find(pl.group, p.n_groups, b);
        a = make_int4((b - pl.group[g]) * p.ratio, pl.block[g], pl.prefix[g],
                      k7_tiles(k7_length(p, p.prefix_lens[g], p.prefix_blocks)));
        if (p.prefix_lens[g] > static_cast<int64_t>(p.prefix_blocks) * p.block_size)
          k7_raise(p.status, TOME_DEV_BLOCK_OUT_OF_RANGE);
      }
      const int32_t len = k7_length(p, p.lengths[b], p.seq_blocks);
      if (p.lengths[b] > len) k7_raise(p.status, TOME_DEV_BLOCK_OUT_OF_RANGE);
      reinterpret_cast<int4*>(p.plan + 4)[b] = a;
      reinterpret_cast<int2*>(p.plan + 4 + 4 * static_cast<int64_t>(p.n_seq))[b] =
          make_int2(pl.prefix[p.n_groups] + pl.suffix[b], k7_tiles(len));
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) p.plan[0] = tiles;

    for (int32_t at = first; at < last && ok;) {
      const K7Piece x = k7_piece(p, pl, at, last);
      at += x.n;
      const bool active = warp * 32 < x.rows;  // warps without a row only keep step
      float o[D];
#pragma unroll
      for (int i = 0; i < D; ++i) o[i] = 0.0f;
      float top = -INFINITY, mc = -INFINITY, sum = 0.0f, alpha = 0.0f;
      auto add_o = [&](uint32_t tile) {  // o = o * alpha + P V of `tile`
        if (!mbar_wait(base + S::O_FULL + (tile & 1u) * 8, (tile >> 1) & 1u)) {
          k7_raise(p.status, TOME_DEV_TIMEOUT);
          ok = false;
          return;
        }
        __syncwarp();
        tc_fence_after_sync();
#pragma unroll
        for (int h = 0; h < D / 32; ++h) {
          uint32_t r[32];
          tmem_ld32(tmem + lanes + 2 * K7_KEYS + (tile & 1u) * D + h * 32, r);
          tmem_ld_wait_dep(r);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[h * 32 + i] = fmaf(o[h * 32 + i], alpha, __uint_as_float(r[i]));
        }
        tc_fence_before_sync();
      };
      for (int32_t j = 0; j < x.n && ok; ++j, ++t) {
        const uint32_t buf = t & 1u;
        if (!mbar_wait(base + S::S_FULL + buf * 8, (t >> 1) & 1u)) {
          k7_raise(p.status, TOME_DEV_TIMEOUT);
          ok = false;
          break;
        }
        float next_alpha = alpha;
        __syncwarp();
        if (active) {
          tc_fence_after_sync();
          uint32_t s0[32], s1[32];
          tmem_ld32(tmem + lanes + buf * K7_KEYS, s0);
          tmem_ld32(tmem + lanes + buf * K7_KEYS + 32, s1);
          tmem_ld_wait_dep(s0);
          tmem_ld_wait_dep(s1);
          const int32_t valid = x.len - (x.tile + j) * K7_KEYS;
          if (valid < K7_KEYS) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              if (i >= valid) s0[i] = 0xff800000u;
              if (i + 32 >= valid) s1[i] = 0xff800000u;
            }
          }
          float big = top;
#pragma unroll
          for (int i = 0; i < 32; ++i) big = fmaxf(big, fmaxf(__uint_as_float(s0[i]), __uint_as_float(s1[i])));
          // a row that has seen nothing but -inf keeps 0 as its reference: all its p are 0
          const float mc_new = big == -INFINITY ? 0.0f : big * p.c;
          next_alpha = top == -INFINITY ? 0.0f : ex2f(mc - mc_new);
          top = big;
          mc = mc_new;
          float l = 0.0f;
          const uint32_t prow = base + S::P + buf * S::P_BYTES + row * 128;
#pragma unroll
          for (int h = 0; h < 8; ++h) {  // eight keys: one 16-byte piece of P
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint32_t w = h < 4 ? s0[(h & 3) * 8 + i] : s1[(h & 3) * 8 + i];
              e[i] = ex2f(fmaf(__uint_as_float(w), p.c, -mc));
              l += e[i];
            }
            k7_sts128(prow + ((h ^ (row & 7)) << 4),
                      make_uint4(k7_pack(e[0], e[1], T()), k7_pack(e[2], e[3], T()),
                                 k7_pack(e[4], e[5], T()), k7_pack(e[6], e[7], T())));
          }
          sum = fmaf(sum, next_alpha, l);
          fence_proxy_async();
          tc_fence_before_sync();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(base + S::P_FULL + buf * 8);
        if (active && j > 0) add_o(t - 1);
        alpha = next_alpha;
      }
      if (active && ok) add_o(t - 1);
      if (ok && row < x.rows) {
        const int64_t slot = static_cast<int64_t>(x.item) + blockIdx.x;
        const int64_t at_row = x.prefix ? slot * K7_ROWS + row : slot * p.ratio + row;
        float* dst = (x.prefix ? p.prefix_o : p.suffix_o) + at_row * D;
#pragma unroll
        for (int i = 0; i < D; i += 4)
          *reinterpret_cast<float4*>(dst + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        (x.prefix ? p.prefix_ml : p.suffix_ml)[at_row] = make_float2(mc, sum);
      }
    }
  } else if (warp == K7_MMA_WARP) {
    // ------------------------------------------------------------ tensor-core products
    if (lane == 0) {
      uint32_t t = 0, piece = 0;
      bool ok = true;
      auto multiply_pv = [&](uint32_t tile) {  // O = P V of `tile`, and its stage is free
        if (!mbar_wait(base + S::P_FULL + (tile & 1u) * 8, (tile >> 1) & 1u)) {
          k7_raise(p.status, TOME_DEV_TIMEOUT);
          ok = false;
          return;
        }
        tc_fence_after_sync();
        const uint32_t stage = tile % K7_STAGES;
        const uint64_t a = k7_desc_k(base + S::P + (tile & 1u) * S::P_BYTES);
        const uint64_t b = k7_desc_mn(base + S::KV + stage * S::STAGE + S::KV_BYTES, K7_KEYS * 128);
#pragma unroll
        for (int k = 0; k < K7_KEYS / 16; ++k)  // 16 keys: 32 bytes of a P row, 16 rows of V
          umma_bf16_ss(tmem + 2 * K7_KEYS + (tile & 1u) * D, a + 2 * k, b + (2048 >> 4) * k,
                       k7_idesc<T>(D, true), k != 0);
        umma_commit(base + S::O_FULL + (tile & 1u) * 8);
        umma_commit(base + S::EMPTY + stage * 8);
      };
      for (int32_t at = first; at < last && ok; ++piece) {
        const int32_t n = k7_piece(p, pl, at, last).n;
        at += n;
        for (int32_t j = 0; j < n && ok; ++j, ++t) {
          const uint32_t stage = t % K7_STAGES;
          if (!mbar_wait(base + S::FULL + stage * 8, (t / K7_STAGES) & 1u)) {
            k7_raise(p.status, TOME_DEV_TIMEOUT);
            ok = false;
            break;
          }
          fence_proxy_async();  // the copies are ordinary writes: visible to the tensor core from here
          tc_fence_after_sync();
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint64_t a = k7_desc_k(base + S::Q + (piece & 1u) * S::Q_BYTES + (k / 4) * (K7_ROWS * 128)) + 2 * (k % 4);
            const uint64_t b = k7_desc_k(base + S::KV + stage * S::STAGE + (k / 4) * (K7_KEYS * 128)) + 2 * (k % 4);
            umma_bf16_ss(tmem + (t & 1u) * K7_KEYS, a, b, k7_idesc<T>(K7_KEYS, false), k != 0);
          }
          umma_commit(base + S::S_FULL + (t & 1u) * 8);
          if (j == n - 1) umma_commit(base + S::Q_EMPTY + (piece & 1u) * 8);
          if (t > 0) multiply_pv(t - 1);
        }
      }
      if (ok && t > 0) multiply_pv(t - 1);
      // nothing may still be under way when the block leaves
      if (ok && t > 0 && !mbar_wait(base + S::EMPTY + ((t - 1) % K7_STAGES) * 8, ((t - 1) / K7_STAGES) & 1u))
        k7_raise(p.status, TOME_DEV_TIMEOUT);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ copies
    constexpr int PIECES = D / 8;                        // 16-byte pieces of a row
    constexpr int STEP = K7_COPY_THREADS / PIECES;       // rows per sweep
    constexpr int SWEEPS = K7_KEYS / STEP;
    const int ct = threadIdx.x - (K7_MMA_WARP + 1) * 32;
    const int c = ct % PIECES, r0 = ct / PIECES;
    const T* kp = reinterpret_cast<const T*>(p.k_pool) + c * 8;
    const T* vp = reinterpret_cast<const T*>(p.v_pool) + c * 8;
    uint32_t t = 0, piece = 0;
    bool ok = true;
    for (int32_t at = first; at < last && ok; ++piece) {
      const K7Piece x = k7_piece(p, pl, at, last);
      at += x.n;
      if (piece >= 2 && !mbar_wait(base + S::Q_EMPTY + (piece & 1u) * 8, ((piece >> 1) - 1) & 1u)) {
        k7_raise(p.status, TOME_DEV_TIMEOUT);
        ok = false;
        break;
      }
      for (int i = r0; i < x.rows; i += STEP) {
        const int32_t row = x.row0 + i, s = row / p.ratio;
        const T* src = reinterpret_cast<const T*>(p.q) + (x.seq0 + s) * p.q_stride +
                       static_cast<int64_t>(x.kv_head * p.ratio + (row - s * p.ratio)) * D + c * 8;
        k7_copy16(base + S::Q + (piece & 1u) * S::Q_BYTES + (c >> 3) * (K7_ROWS * 128) + i * 128 +
                      (((c & 7) ^ (i & 7)) << 4),
                  src, true);
      }
      for (int32_t j = 0; j < x.n && ok; ++j, ++t) {
        const uint32_t stage = t % K7_STAGES;
        // where the keys are, ahead of the wait for the stage
        int64_t src[SWEEPS];
#pragma unroll
        for (int i = 0; i < SWEEPS; ++i) {
          const int32_t key = (x.tile + j) * K7_KEYS + r0 + i * STEP;
          src[i] = -1;
          if (key < x.len) {
            const int32_t blk = static_cast<int32_t>((static_cast<uint64_t>(key) * p.div_magic) >> p.div_shift);
            const int32_t page = __ldg(x.table + blk);
            if (page >= 0 && page < p.num_blocks)
              src[i] = ((static_cast<int64_t>(page) * p.kv_heads + x.kv_head) * p.block_size +
                        (key - blk * p.block_size)) * D;
            else
              k7_raise(p.status, TOME_DEV_BLOCK_OUT_OF_RANGE);  // reads as zeros, as gather does
          }
        }
        if (t >= K7_STAGES && !mbar_wait(base + S::EMPTY + stage * 8, (t / K7_STAGES - 1) & 1u)) {
          k7_raise(p.status, TOME_DEV_TIMEOUT);
          ok = false;
          break;
        }
        const uint32_t dst = base + S::KV + stage * S::STAGE + (c >> 3) * (K7_KEYS * 128);
#pragma unroll
        for (int i = 0; i < SWEEPS; ++i) {
          const int r = r0 + i * STEP;
          const uint32_t d = dst + r * 128 + (((c & 7) ^ (r & 7)) << 4);
          const int64_t off = src[i] < 0 ? 0 : src[i];
          k7_copy16(d, kp + off, src[i] >= 0);
          k7_copy16(d + S::KV_BYTES, vp + off, src[i] >= 0);
        }
        k7_copies_arrive(base + S::FULL + stage * 8);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == K7_MMA_WARP) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, S::TMEM_COLS);
  }
}

// ------------------------------------------------------------------ joining the pieces
// One warp per (sequence, head).  With maxima m_i, sums l_i and sums of p v o_i of its pieces:
// M = max m_i, out = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i.  A row without a key is 0 with
// log-sum -inf.
template <typename T, int D>
__global__ void __launch_bounds__(128) k7_join_kernel(const K7Params p) {
  constexpr int E = D / 32;  // elements per lane
  const int lane = threadIdx.x & 31;
  const int64_t w = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  griddep_wait();
  if (w >= static_cast<int64_t>(p.n_seq) * p.heads) return;
  const int32_t b = static_cast<int32_t>(w / p.heads), h = static_cast<int32_t>(w - static_cast<int64_t>(b) * p.heads);
  const int32_t kv = h / p.ratio;
  const int32_t tiles = p.plan[0], working = k7_working(tiles, p.ctas);
  const int4 a = reinterpret_cast<const int4*>(p.plan + 4)[b];
  const int2 s = reinterpret_cast<const int2*>(p.plan + 4 + 4 * static_cast<int64_t>(p.n_seq))[b];
  const int32_t row = a.x + (h - kv * p.ratio), mb = row / K7_ROWS;
  int32_t n_prefix = 0, n_suffix = 0;
  int64_t at_prefix = 0, at_suffix = 0;  // row index of the first piece; pieces are K7_ROWS / ratio rows apart
  if (a.w > 0) {
    const int32_t i = mb * p.kv_heads + kv, u = a.z + i * a.w;
    const int32_t c0 = k7_cta_of(tiles, working, u), c1 = k7_cta_of(tiles, working, u + a.w - 1);
    n_prefix = c1 - c0 + 1;
    at_prefix = (static_cast<int64_t>(a.y) * p.kv_heads + i + c0) * K7_ROWS + (row - mb * K7_ROWS);
  }
  if (s.y > 0) {
    const int32_t u = s.x + kv * s.y;
    const int32_t c0 = k7_cta_of(tiles, working, u), c1 = k7_cta_of(tiles, working, u + s.y - 1);
    n_suffix = c1 - c0 + 1;
    at_suffix = (static_cast<int64_t>(b) * p.kv_heads + kv + c0) * p.ratio + (h - kv * p.ratio);
  }
  const int32_t n = n_prefix + n_suffix;
  float top = -INFINITY, total = 0.0f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.0f;
  for (int32_t base = 0; base < n; base += 32) {
    const int32_t i = base + lane;
    float2 ml = make_float2(-INFINITY, 0.0f);
    if (i < n_prefix) ml = p.prefix_ml[at_prefix + static_cast<int64_t>(i) * K7_ROWS];
    else if (i < n) ml = p.suffix_ml[at_suffix + static_cast<int64_t>(i - n_prefix) * p.ratio];
    if (ml.y == 0.0f) ml.x = -INFINITY;  // a piece that saw nothing but -inf
    float m = ml.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    m = fmaxf(m, top);
    const float keep = top == -INFINITY ? 0.0f : ex2f(top - m);
    top = m;
    const float wgt = ml.x == -INFINITY ? 0.0f : ex2f(ml.x - m);
    float l = wgt * ml.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    total = fmaf(total, keep, l);
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= keep;
    const int32_t here = min(32, n - base);
#pragma unroll 4
    for (int32_t k = 0; k < here; ++k) {
      const float f = __shfl_sync(0xffffffffu, wgt, k);
      const int32_t q = base + k;
      const float* src = q < n_prefix
                             ? p.prefix_o + (at_prefix + static_cast<int64_t>(q) * K7_ROWS) * D
                             : p.suffix_o + (at_suffix + static_cast<int64_t>(q - n_prefix) * p.ratio) * D;
      float v[E];
      if constexpr (E == 4) {
        const float4 x = *reinterpret_cast<const float4*>(src + lane * 4);
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
      } else {
        const float2 x = *reinterpret_cast<const float2*>(src + lane * 2);
        v[0] = x.x; v[1] = x.y;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = fmaf(f, v[e], acc[e]);
    }
  }
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  T* out = reinterpret_cast<T*>(p.out) + w * D + lane * E;
  uint32_t r[E / 2];
#pragma unroll
  for (int e = 0; e < E; e += 2) r[e / 2] = k7_pack(acc[e] * inv, acc[e + 1] * inv, T());
  if constexpr (E == 4) *reinterpret_cast<uint2*>(out) = make_uint2(r[0], r[1]);
  else *reinterpret_cast<uint32_t*>(out) = r[0];
  if (p.out_lse != nullptr && lane == 0)
    p.out_lse[w] = total == 0.0f ? -INFINITY : (top + log2f(total)) * 0.6931471805599453f;
}

// ------------------------------------------------------------------ host side
struct K7Layout {
  size_t plan, prefix_o, prefix_ml, suffix_o, suffix_ml, total;
};

static size_t k7_up(size_t n) { return (n + 255) / 256 * 256; }

// The split takes at most this many CTAs (one per SM); the workspace does not depend on the
// device that it is asked for on.
constexpr int K7_MAX_CTAS = 160;

static K7Layout k7_layout(int64_t n_seq, int64_t n_groups, int64_t heads, int64_t kv_heads, int64_t dim) {
  const int64_t ratio = heads / kv_heads;
  // row blocks of all groups: each group rounds up once
  const int64_t blocks = n_groups == 0 ? 0 : n_groups + n_seq * ratio / K7_ROWS;
  const int64_t prefix_slots = blocks == 0 ? 0 : blocks * kv_heads + K7_MAX_CTAS;
  const int64_t suffix_slots = n_seq * kv_heads + K7_MAX_CTAS;
  K7Layout l;
  l.plan = 0;
  l.prefix_o = k7_up(static_cast<size_t>(16 + 24 * n_seq));
  l.prefix_ml = l.prefix_o + k7_up(static_cast<size_t>(prefix_slots * K7_ROWS * dim * 4));
  l.suffix_o = l.prefix_ml + k7_up(static_cast<size_t>(prefix_slots * K7_ROWS * 8));
  l.suffix_ml = l.suffix_o + k7_up(static_cast<size_t>(suffix_slots * ratio * dim * 4));
  l.total = l.suffix_ml + k7_up(static_cast<size_t>(suffix_slots * ratio * 8));
  return l;
}

static int32_t k7_shape(int64_t n_seq, int64_t n_groups, int64_t heads, int64_t kv_heads, int64_t dim) {
  if (n_seq < 0 || n_groups < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0)
    return fail(TOME_ERR_BAD_SHAPE, "n_seq=%lld n_groups=%lld heads=%lld kv_heads=%lld",
                (long long)n_seq, (long long)n_groups, (long long)heads, (long long)kv_heads);
  if (n_seq > K7_MAX_SEQ || n_groups > K7_MAX_GROUPS || heads > 65536)
    return fail(TOME_ERR_TOO_LARGE, "at most %d sequences and %d groups per call", K7_MAX_SEQ,
                K7_MAX_GROUPS);
  if (dim != 64 && dim != 128)
    return fail(TOME_ERR_UNSUPPORTED, "head_dim=%lld must be 64 or 128", (long long)dim);
  if (heads / kv_heads > K7_ROWS)
    return fail(TOME_ERR_UNSUPPORTED, "at most %d query heads per KV head", K7_ROWS);
  return TOME_OK;
}

template <typename T, int D>
static int32_t k7_launch(const K7Params& p, cudaStream_t stream) {
  using S = K7Smem<D>;
  void (*kernel)(K7Params) = k7_attention_kernel<T, D>;
  const int bytes = S::PLAN + S::plan_bytes(p.n_groups, p.n_seq) + 1024;
  // set once for the largest plan, so that no later call has to raise it
  const int most = S::PLAN + S::plan_bytes(K7_MAX_GROUPS, K7_MAX_SEQ) + 1024;
  static_assert(S::PLAN + S::plan_bytes(K7_MAX_GROUPS, K7_MAX_SEQ) + 1024 <= 232448, "shared memory");
  int32_t st = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), most);
  if (st != TOME_OK) return st;
  kernel<<<p.ctas, K7_THREADS, bytes, stream>>>(p);
  st = check_cuda(cudaGetLastError(), "prefix attention launch");
  if (st != TOME_OK) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((static_cast<int64_t>(p.n_seq) * p.heads + 3) / 4));
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  void (*join)(K7Params) = k7_join_kernel<T, D>;
  return check_cuda(cudaLaunchKernelEx(&cfg, join, p), "prefix attention join launch");
}

}  // namespace tome

using namespace tome;

extern "C" size_t tome_shared_prefix_attention_workspace_bytes(int64_t n_seq, int64_t n_groups,
                                                               int64_t heads, int64_t kv_heads,
                                                               int64_t head_dim) {
  if (n_seq <= 0 || k7_shape(n_seq, n_groups, heads, kv_heads, head_dim) != TOME_OK) return 0;
  return k7_layout(n_seq, n_groups, heads, kv_heads, head_dim).total;
}

extern "C" int32_t tome_shared_prefix_attention(
    const void* q, int32_t dtype, int64_t n_seq, int64_t heads, int64_t kv_heads, int64_t head_dim,
    int64_t q_stride, const void* k_pool, const void* v_pool, int32_t block_size, int32_t num_blocks,
    const int32_t* prefix_tables, const int32_t* prefix_lens, const int32_t* group_starts,
    int64_t n_groups, int32_t prefix_blocks, const int32_t* block_tables, const int32_t* lengths,
    int32_t max_blocks, float scale, void* out, float* out_lse, void* workspace,
    size_t workspace_bytes, int32_t* dev_status, void* stream) {
  if (dtype != TOME_BF16 && dtype != TOME_F16) return fail(TOME_ERR_BAD_DTYPE, "dtype=%d", dtype);
  int32_t st = k7_shape(n_seq, n_groups, heads, kv_heads, head_dim);
  if (st != TOME_OK) return st;
  if (block_size <= 0 || num_blocks < 0 || prefix_blocks < 0 || max_blocks < 0)
    return fail(TOME_ERR_BAD_SHAPE, "block_size=%d num_blocks=%d prefix_blocks=%d max_blocks=%d",
                block_size, num_blocks, prefix_blocks, max_blocks);
  if (!(scale > 0.0f) || scale > 3.0e38f)
    return fail(TOME_ERR_BAD_SHAPE, "scale=%g must be positive and finite", (double)scale);
  if (n_seq == 0) return TOME_OK;
  if (q_stride < heads * head_dim || (q_stride * 2) % 16 != 0)
    return fail(TOME_ERR_BAD_STRIDE, "q_stride=%lld", (long long)q_stride);
  if (q == nullptr || k_pool == nullptr || v_pool == nullptr || lengths == nullptr || out == nullptr ||
      (max_blocks > 0 && block_tables == nullptr) ||
      (n_groups > 0 && (prefix_lens == nullptr || group_starts == nullptr ||
                        (prefix_blocks > 0 && prefix_tables == nullptr))))
    return fail(TOME_ERR_NULL_POINTER, "a required pointer is NULL");
  if (!aligned16(q) || !aligned16(k_pool) || !aligned16(v_pool) || !aligned16(out) || !aligned16(workspace))
    return fail(TOME_ERR_MISALIGNED, "tensors must be 16-byte aligned");
  const K7Layout l = k7_layout(n_seq, n_groups, heads, kv_heads, head_dim);
  if (workspace == nullptr || workspace_bytes < l.total)
    return fail(TOME_ERR_WORKSPACE_TOO_SMALL, "workspace of %zu bytes, %zu needed", workspace_bytes, l.total);
  // tiles in all are counted in 32 bits
  const int64_t ratio = heads / kv_heads;
  const int64_t key_tiles = (static_cast<int64_t>(prefix_blocks) * block_size + K7_KEYS - 1) / K7_KEYS;
  const int64_t seq_tiles = (static_cast<int64_t>(max_blocks) * block_size + K7_KEYS - 1) / K7_KEYS;
  const int64_t row_blocks = n_groups == 0 ? 0 : n_groups + n_seq * ratio / K7_ROWS;
  if (static_cast<int64_t>(prefix_blocks) * block_size > 0x3fffffff ||
      static_cast<int64_t>(max_blocks) * block_size > 0x3fffffff ||
      row_blocks * kv_heads * key_tiles + n_seq * kv_heads * seq_tiles > 0x3fffffff)
    return fail(TOME_ERR_TOO_LARGE, "the tables name too many keys for one call");
  DeviceInfo info;
  st = current_device_info(&info);
  if (st != TOME_OK) return st;
  K7Params p = {};
  p.q = q;
  p.q_stride = q_stride;
  p.k_pool = k_pool;
  p.v_pool = v_pool;
  p.prefix_tables = prefix_tables;
  p.prefix_lens = prefix_lens;
  p.group_starts = group_starts;
  p.tables = block_tables;
  p.lengths = lengths;
  p.n_seq = static_cast<int32_t>(n_seq);
  p.n_groups = static_cast<int32_t>(n_groups);
  p.heads = static_cast<int32_t>(heads);
  p.kv_heads = static_cast<int32_t>(kv_heads);
  p.ratio = static_cast<int32_t>(ratio);
  p.block_size = block_size;
  p.prefix_blocks = prefix_blocks;
  p.seq_blocks = max_blocks;
  p.num_blocks = num_blocks;
  // key / block_size for keys below 2^31: with s = ceil(log2 d), (2^(31+s) / d + 1) fits 32 bits
  // and its product with the key, shifted back, is exact
  int s = 0;
  while ((1ll << s) < block_size) ++s;
  p.div_shift = 31 + s;
  p.div_magic = static_cast<uint32_t>((1ull << (31 + s)) / static_cast<uint64_t>(block_size) + 1);
  p.c = scale * LOG2E;
  p.ctas = std::max(1, std::min(info.sm_count, K7_MAX_CTAS));
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.plan = reinterpret_cast<int32_t*>(ws + l.plan);
  p.prefix_o = reinterpret_cast<float*>(ws + l.prefix_o);
  p.prefix_ml = reinterpret_cast<float2*>(ws + l.prefix_ml);
  p.suffix_o = reinterpret_cast<float*>(ws + l.suffix_o);
  p.suffix_ml = reinterpret_cast<float2*>(ws + l.suffix_ml);
  p.out = out;
  p.out_lse = out_lse;
  p.status = dev_status;
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if (dtype == TOME_BF16)
    return head_dim == 64 ? k7_launch<__nv_bfloat16, 64>(p, cs) : k7_launch<__nv_bfloat16, 128>(p, cs);
  return head_dim == 64 ? k7_launch<__half, 64>(p, cs) : k7_launch<__half, 128>(p, cs);
}

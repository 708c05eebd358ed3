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
// 64 keys, weighed by what they cost (an item K7_ITEM_COST, a tile K7_SMALL_COST or K7_BIG_COST, see
// there) and laid end to end; every CTA takes an equal run of the whole, whatever the lengths: the
// split follows from the lengths on the device alone.  A CTA's part of an item is a
// piece; it leaves (sum of p v, row maximum, row sum) in the workspace, and a second kernel
// joins the pieces of a row.  A row's pieces lie at (item index + CTA index), which no two pieces
// share since at least one of the two grows from piece to piece.
//
// Pipeline of a CTA (one per SM): two warps copy keys and values (16-byte asynchronous copies:
// pages of any size, rows past the end filled with zeros) into a ring of four stages, one
// thread issues the tensor-core products S = Q K^T (128 x 64 x D) and O = P V (128 x D x 64),
// four warps own a row per thread: running maximum and sum, P rounded to the type of V
// into shared memory; O adds up in tensor memory.  S is double-buffered, so the products
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
constexpr int K7_STAGES = 4;
constexpr int K7_SOFTMAX_WARPS = 4;
constexpr int K7_MMA_WARP = 4;
constexpr int K7_COPY_THREADS = 64;  // a warp fetches half of a tile's keys and values
constexpr int K7_THREADS = (K7_SOFTMAX_WARPS + 1) * 32 + K7_COPY_THREADS;
constexpr int K7_SMALL_ROWS = 16;  // pieces of up to this many rows take the warp-level products
// Costs, in thirds of a tile of few rows: a tile of up to 16 rows, one of more, and what a piece
// costs besides its tiles (the ring runs dry while the queries come, the warps' results meet).
constexpr int K7_SMALL_COST = 3;
constexpr int K7_BIG_COST = 4;
constexpr int K7_ITEM_COST = 4;
// Cards of pieces in flight.  One is written over four pieces later; the copying warps are at most
// two pieces ahead of a Q buffer's release, and that comes after the softmax warps took the card.
constexpr int K7_CARDS = 4;
constexpr int K7_MAX_SEQ = 2048;
constexpr int K7_MAX_GROUPS = 512;

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
  int32_t* plan;              // [0]: the cost of all items; then two int4 [n_seq], see the kernel
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
  int32_t* prefix;  // [n_groups + 1] cost of the prefix items before each group
  int32_t* suffix;  // [n_seq + 1] cost of the suffix items before each sequence
};

__device__ __forceinline__ int32_t k7_tiles(int32_t len) { return (len + K7_KEYS - 1) / K7_KEYS; }

// Cost of a tile of an item whose rows number `rows`, and of an item; tiles that lie before the
// offset `cost` of an item.
__device__ __forceinline__ int32_t k7_tile_cost(int32_t rows) {
  return rows <= K7_SMALL_ROWS ? K7_SMALL_COST : K7_BIG_COST;
}
__device__ __forceinline__ int32_t k7_item_cost(int32_t tiles, int32_t tile_cost) {
  return tiles == 0 ? 0 : K7_ITEM_COST + tiles * tile_cost;
}
__device__ __forceinline__ int32_t k7_cut(int32_t cost, int32_t tile_cost) {
  return max(cost - K7_ITEM_COST + tile_cost / 2, 0) / tile_cost;
}

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
        const int32_t rows = (pl.group[i + 1] - pl.group[i]) * p.ratio;
        b = (rows + K7_ROWS - 1) / K7_ROWS;
        t = b * p.kv_heads * k7_item_cost(k7_tiles(k7_length(p, p.prefix_lens[i], p.prefix_blocks)),
                                          k7_tile_cost(rows));
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
      if (i < p.n_seq)
        t = p.kv_heads * k7_item_cost(k7_tiles(k7_length(p, p.lengths[i], p.seq_blocks)),
                                      k7_tile_cost(p.ratio));
      const int32_t ts = k7_scan_add(t, lane);
      if (i < p.n_seq) pl.suffix[i] = tiles + ts - t;
      tiles += __shfl_sync(0xffffffffu, ts, 31);
    }
    if (lane == 0) pl.suffix[p.n_seq] = tiles;
  }
}

// The CTAs that take part (each has some cost, so that an item's pieces lie in neighbouring
// ones), where the run of one begins, and the one that holds a place.
__device__ __forceinline__ int32_t k7_working(int32_t cost, int32_t ctas) { return min(cost, ctas); }
__device__ __forceinline__ int32_t k7_begin(int32_t cost, int32_t ctas, int32_t cta) {
  return static_cast<int32_t>(static_cast<int64_t>(cta) * cost / ctas);
}
__device__ __forceinline__ int32_t k7_cta_of(int32_t cost, int32_t ctas, int32_t place) {
  return static_cast<int32_t>(((static_cast<int64_t>(place) + 1) * ctas + cost - 1) / cost - 1);
}

// A piece: tiles [tile, tile + n) of an item.
struct K7Piece {
  const int32_t* table;
  int32_t len;        // keys of the item
  int32_t tile, n;
  int32_t tile_cost;
  int32_t end;        // place where the item ends
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

// Tiles of the item that ends at x.end between the places `at` and `last`.
__device__ __forceinline__ void k7_cut_piece(K7Piece& x, int32_t at, int32_t last) {
  const int32_t begin = x.end - k7_item_cost(k7_tiles(x.len), x.tile_cost);
  x.tile = k7_cut(at - begin, x.tile_cost);
  x.n = k7_cut(min(last, x.end) - begin, x.tile_cost) - x.tile;
}

// The part of the item at the place `at` that lies before `last`.
__device__ __forceinline__ K7Piece k7_piece(const K7Params& p, const K7Plan& pl, int32_t at, int32_t last) {
  K7Piece x;
  const int32_t in_prefix = pl.prefix[p.n_groups];
  x.prefix = at < in_prefix;
  if (x.prefix) {
    const int g = k7_find(pl.prefix, p.n_groups, at);
    x.seq0 = pl.group[g];
    const int32_t rows = (pl.group[g + 1] - x.seq0) * p.ratio;
    x.len = k7_length(p, p.prefix_lens[g], p.prefix_blocks);
    x.tile_cost = k7_tile_cost(rows);
    const int32_t cost = k7_item_cost(k7_tiles(x.len), x.tile_cost);
    const int32_t i = (at - pl.prefix[g]) / cost;  // (row block, KV head)
    x.end = pl.prefix[g] + (i + 1) * cost;
    const int32_t mb = i / p.kv_heads;
    x.kv_head = i - mb * p.kv_heads;
    x.row0 = mb * K7_ROWS;
    x.rows = min(K7_ROWS, rows - x.row0);
    x.item = (pl.block[g] + mb) * p.kv_heads + x.kv_head;
    x.table = p.prefix_tables + static_cast<int64_t>(g) * p.prefix_blocks;
  } else {
    const int b = k7_find(pl.suffix, p.n_seq, at - in_prefix);
    x.seq0 = b;
    x.len = k7_length(p, p.lengths[b], p.seq_blocks);
    x.tile_cost = k7_tile_cost(p.ratio);
    const int32_t cost = k7_item_cost(k7_tiles(x.len), x.tile_cost), begin = in_prefix + pl.suffix[b];
    x.kv_head = (at - begin) / cost;
    x.end = begin + (x.kv_head + 1) * cost;
    x.row0 = 0;
    x.rows = p.ratio;
    x.item = b * p.kv_heads + x.kv_head;
    x.table = p.tables + static_cast<int64_t>(b) * p.seq_blocks;
  }
  k7_cut_piece(x, at, last);
  return x;
}

// Next piece with a tile of the run that goes on at `at` (x is the piece before, if `have`); moves
// `at` behind it.  As a rule it is the next KV head of the same rows and keys, else it is looked up.
__device__ __forceinline__ bool k7_next(const K7Params& p, const K7Plan& pl, K7Piece& x, bool have,
                                        int32_t& at, int32_t last) {
  while (at < last) {
    if (have && at == x.end && x.kv_head + 1 < p.kv_heads) {
      x.kv_head += 1;
      x.item += 1;
      x.end += k7_item_cost(k7_tiles(x.len), x.tile_cost);
      k7_cut_piece(x, at, last);
    } else {
      x = k7_piece(p, pl, at, last);
      have = true;
    }
    at = min(last, x.end);
    if (x.n > 0) return true;
  }
  return false;
}

// What the softmax warps need of a piece, written by the first copying thread ahead of them; n = 0
// behind the last one.
struct K7Card {
  int32_t len, tile, n, rows, item, prefix;
};

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
  static constexpr int P = Q + 2 * Q_BYTES;
  static constexpr int KV = P + P_BYTES;
  static constexpr int BARS = KV + K7_STAGES * STAGE;
  static constexpr int FULL = BARS;                        // STAGES
  static constexpr int EMPTY = FULL + K7_STAGES * 8;       // STAGES
  static constexpr int S_FULL = EMPTY + K7_STAGES * 8;     // 2
  static constexpr int P_FULL = S_FULL + 16;               // 2
  static constexpr int O_FULL = P_FULL + 16;               // 2
  static constexpr int Q_EMPTY = O_FULL + 16;              // 2
  static constexpr int TMEM = Q_EMPTY + 16;
  static constexpr int WARP_ML = TMEM + 16;                // [4 warps][8 rows] float2
  static constexpr int CARD_FULL = WARP_ML + K7_SOFTMAX_WARPS * 8 * 8;  // K7_CARDS
  static constexpr int CARDS = CARD_FULL + K7_CARDS * 8;
  static constexpr int PLAN = CARDS + K7_CARDS * static_cast<int>(sizeof(K7Card));
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

__device__ __forceinline__ void k7_ldmatrix(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void k7_ldmatrix_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// c[16 x 8] += a[16 x 16] b[16 x 8] by one warp
__device__ __forceinline__ void k7_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                       __nv_bfloat16) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void k7_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1,
                                       __half) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A piece of up to 16 rows (a sequence's own tokens, as a rule two to eight rows): each of the
// four warps takes 16 keys of every tile through warp-level products, with its own running
// maximum and sum and its sums of p v in registers; they meet at the end of the piece.  The
// tensor-core path below would compute 128 rows for these few and pass each tile through four
// barriers; here a tile costs a warp 32 small products and is given back at once.
template <typename T, int D>
__device__ __forceinline__ bool k7_small_piece(const K7Params& p, uint8_t* smem, uint32_t base,
                                               const K7Card& x, uint32_t& t, uint32_t piece, int warp,
                                               int lane, float* out_o, float2* out_ml) {
  using S = K7Smem<D>;
  const int g = lane >> 2;  // this thread's rows: g and g + 8; its columns: 2 (lane & 3) + {0, 1} of eight
  bool ok = true;
  uint32_t qf[D / 16][4];
  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;
  float ref[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
  // where this lane points the matrix loads to: row and 16-byte piece of Q, K and V tiles
  const int q_row = lane & 15, q_c = lane >> 4;
  const int k_row = warp * 16 + (lane & 7) + ((lane >> 4) << 3), k_c = (lane >> 3) & 1;
  const int v_row = warp * 16 + (lane & 15), v_c = lane >> 4;
  for (int32_t j = 0; j < x.n; ++j, ++t) {
    const uint32_t stage = t % K7_STAGES;
    if (ok && !mbar_wait(base + S::FULL + stage * 8, (t / K7_STAGES) & 1u)) {
      k7_raise(p.status, TOME_DEV_TIMEOUT);
      ok = false;
    }
    __syncwarp();
    if (j == 0) {  // the queries came with the first tile
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const int c = 2 * k + q_c;
        k7_ldmatrix(base + S::Q + (piece & 1u) * S::Q_BYTES + (c >> 3) * (K7_ROWS * 128) + q_row * 128 +
                        (((c & 7) ^ (q_row & 7)) << 4),
                    qf[k]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(base + S::Q_EMPTY + (piece & 1u) * 8);
    }
    const int32_t valid = x.len - (x.tile + j) * K7_KEYS - warp * 16;  // of this warp's 16 keys
    // All matrix loads first, then the stage is given back: the ring is as good as one stage
    // longer, and no load's latency stands before a product.
    const uint32_t kt = base + S::KV + stage * S::STAGE, vt = kt + S::KV_BYTES;
    uint32_t kf[D / 16][4], vf[D / 16][4];
    if (valid > 0) {
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const int c = 2 * k + k_c;
        k7_ldmatrix(kt + (c >> 3) * (K7_KEYS * 128) + k_row * 128 + (((c & 7) ^ (k_row & 7)) << 4), kf[k]);
      }
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const int c = 2 * k + v_c;
        k7_ldmatrix_trans(vt + (c >> 3) * (K7_KEYS * 128) + v_row * 128 + (((c & 7) ^ (v_row & 7)) << 4), vf[k]);
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(base + S::EMPTY + stage * 8);
    if (valid > 0) {
      float s[2][4] = {}, s2[2][4] = {};  // two chains of products for each eight keys
#pragma unroll
      for (int k = 0; k < D / 16; k += 2) {
        k7_mma(s[0], qf[k], kf[k][0], kf[k][1], T());
        k7_mma(s[1], qf[k], kf[k][2], kf[k][3], T());
        k7_mma(s2[0], qf[k + 1], kf[k + 1][0], kf[k + 1][1], T());
        k7_mma(s2[1], qf[k + 1], kf[k + 1][2], kf[k + 1][3], T());
      }
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] += s2[n][e];
      if (valid < 16) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n * 8 + 2 * (lane & 3) + (e & 1) >= valid) s[n][e] = -INFINITY;
      }
      // The exponents' reference moves only when a score exceeds it by more than 2^8, which one
      // vote finds out; the row maxima are formed only then.
      float top[2];
      bool grow = false;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        top[r] = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1])) * p.c;
        grow |= g + 8 * r < x.rows && (top[r] > ref[r] + 8.0f);
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
          top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
          const float next = fmaxf(ref[r], top[r]);
          const float alpha = next == -INFINITY ? 1.0f : ex2f(ref[r] - next);
          ref[r] = next;
          sum[r] *= alpha;
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            o[i][2 * r] *= alpha;
            o[i][2 * r + 1] *= alpha;
          }
        }
      }
      const float off[2] = {ref[0] == -INFINITY ? 0.0f : -ref[0], ref[1] == -INFINITY ? 0.0f : -ref[1]};
      uint32_t pf[4];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float a = ex2f(fmaf(s[n][2 * r], p.c, off[r])), b = ex2f(fmaf(s[n][2 * r + 1], p.c, off[r]));
          sum[r] += a + b;
          pf[2 * n + r] = k7_pack(a, b, T());
        }
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        k7_mma(o[2 * i], pf, vf[i][0], vf[i][1], T());
        k7_mma(o[2 * i + 1], pf, vf[i][2], vf[i][3], T());
      }
    }
  }
  // The warps' results meet in the space of P, which is free between pieces, eight rows at a time:
  // [warp][row][D], pairs of a row turned by its index so that the rows of a store fall on
  // different banks.
  float2* const area = reinterpret_cast<float2*>(smem + S::P);
  float2* const ml = reinterpret_cast<float2*>(smem + S::WARP_ML);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    if (8 * r >= x.rows) break;
    sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
    sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
    if (g + 8 * r < x.rows) {
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
        area[(warp * 8 + g) * (D / 2) + ((4 * i + (lane & 3)) ^ (g << 2))] =
            make_float2(o[i][2 * r], o[i][2 * r + 1]);
      if ((lane & 3) == 0) ml[warp * 8 + g] = make_float2(ref[r], sum[r]);
    }
    named_bar_sync(1, K7_SOFTMAX_WARPS * 32);
    const int rows = min(8, x.rows - 8 * r);
    for (int i = warp * 32 + lane; i < rows * (D / 2); i += K7_SOFTMAX_WARPS * 32) {
      const int row = i / (D / 2), f = i - row * (D / 2);
      float2 w[K7_SOFTMAX_WARPS];
      float top = -INFINITY;
#pragma unroll
      for (int k = 0; k < K7_SOFTMAX_WARPS; ++k) {
        w[k] = ml[k * 8 + row];
        top = fmaxf(top, w[k].x);
      }
      float2 v = make_float2(0.0f, 0.0f);
      float l = 0.0f;
#pragma unroll
      for (int k = 0; k < K7_SOFTMAX_WARPS; ++k) {
        // a warp without a finite score has the weight 0, or 1 where it holds a NaN
        const float a = w[k].x == -INFINITY ? (w[k].y == 0.0f ? 0.0f : 1.0f) : ex2f(w[k].x - top);
        const float2 q = area[(k * 8 + row) * (D / 2) + (f ^ (row << 2))];
        v.x = fmaf(a, q.x, v.x);
        v.y = fmaf(a, q.y, v.y);
        l = fmaf(a, w[k].y, l);
      }
      *reinterpret_cast<float2*>(out_o + (8 * r + row) * D + 2 * f) = v;
      if (f == 0) out_ml[8 * r + row] = make_float2(top, l);
    }
    named_bar_sync(1, K7_SOFTMAX_WARPS * 32);  // the space may be written again
  }
  return ok;
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

  K7Card* const cards = reinterpret_cast<K7Card*>(smem + S::CARDS);

  if (threadIdx.x == K7_MMA_WARP * 32) {
    for (int i = 0; i < K7_STAGES; ++i) {
      mbar_init(base + S::FULL + i * 8, K7_COPY_THREADS);
      mbar_init(base + S::EMPTY + i * 8, K7_SOFTMAX_WARPS);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(base + S::S_FULL + i * 8, 1);
      mbar_init(base + S::P_FULL + i * 8, K7_SOFTMAX_WARPS);
      mbar_init(base + S::O_FULL + i * 8, 1);
      mbar_init(base + S::Q_EMPTY + i * 8, K7_SOFTMAX_WARPS);
    }
    for (int i = 0; i < K7_CARDS; ++i) mbar_init(base + S::CARD_FULL + i * 8, 1);
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
  const int32_t cost = pl.prefix[p.n_groups] + pl.suffix[p.n_seq];
  const int32_t working = k7_working(cost, p.ctas);
  const bool works = static_cast<int32_t>(blockIdx.x) < working;
  const int32_t first = works ? k7_begin(cost, working, blockIdx.x) : 0;
  const int32_t last = works ? k7_begin(cost, working, blockIdx.x + 1) : 0;
  griddep_launch_dependents();

  if (warp < K7_SOFTMAX_WARPS) {
    // ------------------------------------------------------------ softmax: thread = row
    const int row = threadIdx.x;
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    // counts of tiles (the ring), of tiles and pieces on the tensor core, of all pieces
    uint32_t t = 0, u = 0, big_piece = 0, piece = 0;
    bool ok = true;
    // For the joining kernel, dealt over the CTAs: where a sequence's items lie.
    for (int b = blockIdx.x * K7_SOFTMAX_WARPS * 32 + threadIdx.x; b < p.n_seq;
         b += gridDim.x * K7_SOFTMAX_WARPS * 32) {
      int4 a = make_int4(0, 0, 0, 0);  // its row within the group, the group's first row block and place, tiles
      int32_t prefix_tile = K7_SMALL_COST;
      if (p.n_groups > 0 && b >= pl.group[0] && b < pl.group[p.n_groups]) {
        const int g = k7_find(pl.group, p.n_groups, b);
        a = make_int4((b - pl.group[g]) * p.ratio, pl.block[g], pl.prefix[g],
                      k7_tiles(k7_length(p, p.prefix_lens[g], p.prefix_blocks)));
        prefix_tile = k7_tile_cost((pl.group[g + 1] - pl.group[g]) * p.ratio);
        if (p.prefix_lens[g] > static_cast<int64_t>(p.prefix_blocks) * p.block_size)
          k7_raise(p.status, TOME_DEV_BLOCK_OUT_OF_RANGE);
      }
      const int32_t len = k7_length(p, p.lengths[b], p.seq_blocks);
      if (p.lengths[b] > len) k7_raise(p.status, TOME_DEV_BLOCK_OUT_OF_RANGE);
      reinterpret_cast<int4*>(p.plan + 4)[2 * b] = a;
      reinterpret_cast<int4*>(p.plan + 4)[2 * b + 1] =
          make_int4(pl.prefix[p.n_groups] + pl.suffix[b], k7_tiles(len), prefix_tile, k7_tile_cost(p.ratio));
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) p.plan[0] = cost;

    for (; ok; ++piece) {
      if (!mbar_wait(base + S::CARD_FULL + (piece % K7_CARDS) * 8, (piece / K7_CARDS) & 1u)) {
        k7_raise(p.status, TOME_DEV_TIMEOUT);
        break;
      }
      const K7Card x = cards[piece % K7_CARDS];
      if (x.n == 0) break;
      const int64_t slot = static_cast<int64_t>(x.item) + blockIdx.x;
      const int64_t rows_at = x.prefix ? slot * K7_ROWS : slot * p.ratio;
      float* const out_o = (x.prefix ? p.prefix_o : p.suffix_o) + rows_at * D;
      float2* const out_ml = (x.prefix ? p.prefix_ml : p.suffix_ml) + rows_at;
      if (x.rows <= K7_SMALL_ROWS) {
        ok = k7_small_piece<T, D>(p, smem, base, x, t, piece, warp, lane, out_o, out_ml);
        continue;
      }
      const bool active = warp * 32 < x.rows;  // warps without a row only keep step
      const uint32_t o_addr = tmem + lanes + 2 * K7_KEYS + (big_piece & 1u) * D;
      // `ref` is what the exponents are relative to, in the log2 domain.  It follows the row's
      // maximum only when that has grown by more than 2^8: the sums in tensor memory then
      // have to be rescaled, which hardly ever happens after the first tiles.
      float ref = -INFINITY, sum = 0.0f;
      for (int32_t j = 0; j < x.n && ok; ++j, ++t, ++u) {
        const uint32_t buf = u & 1u;
        if (!mbar_wait(base + S::S_FULL + buf * 8, (u >> 1) & 1u)) {
          k7_raise(p.status, TOME_DEV_TIMEOUT);
          ok = false;
          break;
        }
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
          float big[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 32; ++i)
            big[i & 3] = fmax3(big[i & 3], __uint_as_float(s0[i]), __uint_as_float(s1[i]));
          const float top = fmaxf(fmaxf(big[0], big[1]), fmaxf(big[2], big[3])) * p.c;
          // (lanes beyond the rows hold whatever the last piece left)
          const bool grow = row < x.rows && (top > ref + 8.0f || (j == 0 && top > ref));
          // P V of the tile before is done: P may be written again, and the sums be rescaled
          if (j > 0) {
            if (!mbar_wait(base + S::O_FULL + ((u - 1) & 1u) * 8, ((u - 1) >> 1) & 1u)) {
              k7_raise(p.status, TOME_DEV_TIMEOUT);
              ok = false;
            }
            __syncwarp();
          }
          if (__any_sync(0xffffffffu, grow)) {
            const float next = grow ? top : ref;
            const float alpha = next == -INFINITY ? 1.0f : ex2f(ref - next);
            sum *= alpha;
            ref = next;
            if (j > 0) {
              tc_fence_after_sync();
#pragma unroll 1
              for (int h = 0; h < D; h += 32) {
                uint32_t r[32];
                tmem_ld32(o_addr + h, r);
                tmem_ld_wait_dep(r);
#pragma unroll
                for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
                tmem_st32(o_addr + h, r);
              }
              tmem_st_wait();
            }
          }
          // a row that has seen nothing but -inf takes 0 as its reference: all its p are 0
          const float off = ref == -INFINITY ? 0.0f : -ref;
          const float2 c2 = make_float2(p.c, p.c), off2 = make_float2(off, off);
          float2 la = make_float2(0.0f, 0.0f), lb = la;
          const uint32_t prow = base + S::P + row * 128;
#pragma unroll
          for (int h = 0; h < 8; ++h) {  // eight keys: one 16-byte piece of P
            float2 e[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int w = (h & 3) * 8 + 2 * i;
              e[i] = h < 4 ? make_float2(__uint_as_float(s0[w]), __uint_as_float(s0[w + 1]))
                           : make_float2(__uint_as_float(s1[w]), __uint_as_float(s1[w + 1]));
              e[i] = __ffma2_rn(e[i], c2, off2);
              e[i].x = ex2f(e[i].x);
              e[i].y = ex2f(e[i].y);
            }
            la = __fadd2_rn(la, __fadd2_rn(e[0], e[1]));
            lb = __fadd2_rn(lb, __fadd2_rn(e[2], e[3]));
            k7_sts128(prow + ((h ^ (row & 7)) << 4),
                      make_uint4(k7_pack(e[0].x, e[0].y, T()), k7_pack(e[1].x, e[1].y, T()),
                                 k7_pack(e[2].x, e[2].y, T()), k7_pack(e[3].x, e[3].y, T())));
          }
          sum += (la.x + la.y) + (lb.x + lb.y);
          fence_proxy_async();
          tc_fence_before_sync();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(base + S::P_FULL + buf * 8);
      }
      ++big_piece;
      // (warps without a row wait too: what follows may write where the products read P)
      if (ok && !mbar_wait(base + S::O_FULL + ((u - 1) & 1u) * 8, ((u - 1) >> 1) & 1u)) {
        k7_raise(p.status, TOME_DEV_TIMEOUT);
        ok = false;
      }
      if (!active || !ok) continue;
      __syncwarp();
      tc_fence_after_sync();
      float* dst = out_o + row * D;
#pragma unroll 1
      for (int h = 0; h < D; h += 32) {
        uint32_t r[32];
        tmem_ld32(o_addr + h, r);
        tmem_ld_wait_dep(r);
        if (row < x.rows) {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            stg128(dst + h + i, make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]));
        }
      }
      tc_fence_before_sync();
      if (row < x.rows) out_ml[row] = make_float2(ref, sum);
    }
  } else if (warp == K7_MMA_WARP) {
    // ------------------------------------------------------------ tensor-core products
    if (lane == 0) {
      // counts as above; the product P V of a tile is issued after Q K of the next one
      uint32_t t = 0, u = 0, big_piece = 0, piece = 0;
      bool ok = true, pending = false, pending_add = false;
      uint32_t pending_stage = 0, pending_o = 0;
      auto multiply_pv = [&]() {  // O (+)= P V of tile u - 1
        pending = false;
        const uint32_t buf = (u - 1) & 1u;
        if (!mbar_wait(base + S::P_FULL + buf * 8, ((u - 1) >> 1) & 1u)) {
          k7_raise(p.status, TOME_DEV_TIMEOUT);
          ok = false;
          return;
        }
        tc_fence_after_sync();
        const uint64_t a = k7_desc_k(base + S::P);
        const uint64_t b = k7_desc_mn(base + S::KV + pending_stage * S::STAGE + S::KV_BYTES, K7_KEYS * 128);
#pragma unroll
        for (int k = 0; k < K7_KEYS / 16; ++k)  // 16 keys: 32 bytes of a P row, 16 rows of V
          umma_bf16_ss(tmem + 2 * K7_KEYS + pending_o * D, a + 2 * k, b + (2048 >> 4) * k,
                       k7_idesc<T>(D, true), pending_add || k != 0);
        // a stage is given back by four arrivals (of four warps, where those do the products)
        for (int i = 1; i < K7_SOFTMAX_WARPS; ++i) mbar_arrive(base + S::EMPTY + pending_stage * 8);
        umma_commit(base + S::EMPTY + pending_stage * 8);
        umma_commit(base + S::O_FULL + buf * 8);
      };
      K7Piece x;
      int32_t at = first;
      for (; ok && k7_next(p, pl, x, piece > 0, at, last); ++piece) {
        if (x.rows <= K7_SMALL_ROWS) {
          if (pending) multiply_pv();
          t += x.n;
          continue;
        }
        for (int32_t j = 0; j < x.n && ok; ++j, ++t) {
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
            umma_bf16_ss(tmem + (u & 1u) * K7_KEYS, a, b, k7_idesc<T>(K7_KEYS, false), k != 0);
          }
          umma_commit(base + S::S_FULL + (u & 1u) * 8);
          if (j == x.n - 1) {
            for (int i = 1; i < K7_SOFTMAX_WARPS; ++i) mbar_arrive(base + S::Q_EMPTY + (piece & 1u) * 8);
            umma_commit(base + S::Q_EMPTY + (piece & 1u) * 8);
          }
          if (pending) multiply_pv();
          pending = true;
          pending_add = j > 0;
          pending_stage = stage;
          pending_o = big_piece & 1u;
          ++u;
        }
        ++big_piece;
      }
      if (ok && pending) multiply_pv();
      // nothing may still be under way when the block leaves
      if (ok && u > 0 && !mbar_wait(base + S::O_FULL + ((u - 1) & 1u) * 8, ((u - 1) >> 1) & 1u))
        k7_raise(p.status, TOME_DEV_TIMEOUT);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ copies
    constexpr int PIECES = D / 8;                  // 16-byte pieces of a row
    constexpr int AT_ONCE = 32 / PIECES;           // rows that a warp copies per step
    constexpr int STEPS = 32 / AT_ONCE;            // a warp has 32 of the 64 keys
    const int cw = warp - (K7_MMA_WARP + 1);
    const int c = lane % PIECES, sub = lane / PIECES;
    const int my_row = cw * 32;
    const T* k_pool = reinterpret_cast<const T*>(p.k_pool) + c * 8;
    const T* v_pool = reinterpret_cast<const T*>(p.v_pool) + c * 8;
    const uint32_t area = base + S::KV + (c >> 3) * (K7_KEYS * 128);
    auto block_of = [&](int32_t key) {
      return static_cast<int32_t>(static_cast<uint64_t>(key) * p.div_magic >> p.div_shift);
    };
    // 64 entries of the table from block `first` on, two per lane: a tile's pages come from there by
    // shuffles, and the entries behind them are asked for long before they are needed.
    struct Pages {
      int32_t first, a, b;
    };
    auto ask = [&](const K7Piece& y, int32_t block) {
      return block <= block_of(y.len - 1) ? __ldg(y.table + block) : -1;
    };
    auto open_pages = [&](const K7Piece& y) {
      const int32_t f = block_of(min(y.tile * K7_KEYS + my_row, y.len - 1));
      return Pages{f, ask(y, f + lane), ask(y, f + 32 + lane)};
    };
    // The pool's row (blocks and heads flattened) of key (tile * 64 + my_row + lane), or -1.
    auto pool_row_of = [&](const K7Piece& y, Pages& w, int32_t tile) -> int32_t {
      const int32_t key0 = tile * K7_KEYS + my_row, key = key0 + lane;
      if (key0 >= y.len) return -1;
      const int32_t lo = block_of(key0);
      if (lo - w.first >= 32) {
        if (lo - w.first < 64) w = Pages{w.first + 32, w.b, ask(y, w.first + 64 + lane)};
        else w = Pages{lo, ask(y, lo + lane), ask(y, lo + 32 + lane)};
      }
      const int32_t blk = block_of(min(key, y.len - 1)), rel = blk - w.first;  // 0 .. 62
      const int32_t pa = __shfl_sync(0xffffffffu, w.a, rel & 31), pb = __shfl_sync(0xffffffffu, w.b, rel & 31);
      const int32_t page = rel < 32 ? pa : pb;
      if (key >= y.len) return -1;
      if (page < 0 || page >= p.num_blocks) {
        k7_raise(p.status, TOME_DEV_BLOCK_OUT_OF_RANGE);  // reads as zeros, as gather does
        return -1;
      }
      return (page * p.kv_heads + y.kv_head) * p.block_size + (key - blk * p.block_size);
    };
    auto show = [&](const K7Piece& y, uint32_t index, bool there) {  // to the softmax warps
      if (cw == 0 && lane == 0) {
        cards[index % K7_CARDS] = K7Card{y.len, y.tile, there ? y.n : 0, y.rows, y.item, y.prefix ? 1 : 0};
        mbar_arrive(base + S::CARD_FULL + (index % K7_CARDS) * 8);
      }
    };
    uint32_t t = 0, piece = 0;
    bool ok = true;
    int32_t at = first;
    K7Piece x = {};
    Pages pages = {};
    bool there = k7_next(p, pl, x, false, at, last);
    show(x, 0, there);
    if (there) pages = open_pages(x);
    while (there && ok) {
      if (piece >= 2 && !mbar_wait(base + S::Q_EMPTY + (piece & 1u) * 8, ((piece >> 1) - 1) & 1u)) {
        k7_raise(p.status, TOME_DEV_TIMEOUT);
        ok = false;
        break;
      }
      for (int i = cw * AT_ONCE + sub; i < x.rows; i += 2 * AT_ONCE) {
        const int32_t row = x.row0 + i, s = row / p.ratio;
        const T* src = reinterpret_cast<const T*>(p.q) + (x.seq0 + s) * p.q_stride +
                       static_cast<int64_t>(x.kv_head * p.ratio + (row - s * p.ratio)) * D + c * 8;
        k7_copy16(base + S::Q + (piece & 1u) * S::Q_BYTES + (c >> 3) * (K7_ROWS * 128) + i * 128 +
                      (((c & 7) ^ (i & 7)) << 4),
                  src, true);
      }
      K7Piece next = x;
      Pages next_pages = {};
      bool next_there = false;
      for (int32_t j = 0; j < x.n; ++j, ++t) {
        const uint32_t stage = t % K7_STAGES;
        if (j + 1 == x.n) {  // the piece behind is looked up while this one's loads are under way
          next_there = k7_next(p, pl, next, true, at, last);
          show(next, piece + 1, next_there);
          if (next_there) next_pages = open_pages(next);
        }
        if (t >= K7_STAGES && !mbar_wait(base + S::EMPTY + stage * 8, (t / K7_STAGES - 1) & 1u)) {
          k7_raise(p.status, TOME_DEV_TIMEOUT);
          ok = false;
          break;
        }
        __syncwarp();
        const int32_t pool_row = pool_row_of(x, pages, x.tile + j);
        const uint32_t dst = area + stage * S::STAGE;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
          const int r = my_row + i * AT_ONCE + sub;
          const int32_t from = __shfl_sync(0xffffffffu, pool_row, i * AT_ONCE + sub);
          const int64_t off = static_cast<int64_t>(max(from, 0)) * D;
          const uint32_t to = dst + r * 128 + (((c & 7) ^ (r & 7)) << 4);
          k7_copy16(to, k_pool + off, from >= 0);
          k7_copy16(to + S::KV_BYTES, v_pool + off, from >= 0);
        }
        k7_copies_arrive(base + S::FULL + stage * 8);
      }
      x = next;
      pages = next_pages;
      there = next_there;
      ++piece;
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
  const int32_t cost = p.plan[0], working = k7_working(cost, p.ctas);
  const int4 a = reinterpret_cast<const int4*>(p.plan + 4)[2 * b];
  const int4 s = reinterpret_cast<const int4*>(p.plan + 4)[2 * b + 1];
  const int32_t row = a.x + (h - kv * p.ratio), mb = row / K7_ROWS;
  // the CTAs that hold parts of the row's two items, and the row's place in the first one's slot
  int32_t n_prefix = 0, n_suffix = 0, prefix_cta = 0, suffix_cta = 0, prefix_begin = 0, suffix_begin = 0;
  int64_t at_prefix = 0, at_suffix = 0;
  const int32_t prefix_cost = k7_item_cost(a.w, s.z), suffix_cost = k7_item_cost(s.y, s.w);
  if (a.w > 0) {
    const int32_t i = mb * p.kv_heads + kv;
    prefix_begin = a.z + i * prefix_cost;
    prefix_cta = k7_cta_of(cost, working, prefix_begin);
    n_prefix = k7_cta_of(cost, working, prefix_begin + prefix_cost - 1) - prefix_cta + 1;
    at_prefix = (static_cast<int64_t>(a.y) * p.kv_heads + i + prefix_cta) * K7_ROWS + (row - mb * K7_ROWS);
  }
  if (s.y > 0) {
    suffix_begin = s.x + kv * suffix_cost;
    suffix_cta = k7_cta_of(cost, working, suffix_begin);
    n_suffix = k7_cta_of(cost, working, suffix_begin + suffix_cost - 1) - suffix_cta + 1;
    at_suffix = (static_cast<int64_t>(b) * p.kv_heads + kv + suffix_cta) * p.ratio + (h - kv * p.ratio);
  }
  const int32_t n = n_prefix + n_suffix;
  float top = -INFINITY, total = 0.0f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.0f;
  for (int32_t base = 0; base < n; base += 32) {
    const int32_t i = base + lane;
    float2 ml = make_float2(-INFINITY, 0.0f);
    bool there = false;  // a CTA's run may hold less than a tile of the item
    if (i < n) {
      const bool pre = i < n_prefix;
      const int32_t cta = pre ? prefix_cta + i : suffix_cta + i - n_prefix;
      const int32_t begin = pre ? prefix_begin : suffix_begin, end = begin + (pre ? prefix_cost : suffix_cost);
      const int32_t from = max(k7_begin(cost, working, cta), begin), to = min(k7_begin(cost, working, cta + 1), end);
      const int32_t w1 = pre ? s.z : s.w;
      there = k7_cut(to - begin, w1) > k7_cut(from - begin, w1);
      if (there)
        ml = pre ? p.prefix_ml[at_prefix + static_cast<int64_t>(i) * K7_ROWS]
                 : p.suffix_ml[at_suffix + static_cast<int64_t>(i - n_prefix) * p.ratio];
    }
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
    const uint32_t which = __ballot_sync(0xffffffffu, there);
    const int32_t here = min(32, n - base);
#pragma unroll 4
    for (int32_t k = 0; k < here; ++k) {
      const float f = __shfl_sync(0xffffffffu, wgt, k);
      if (!(which >> k & 1u)) continue;
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
  l.prefix_o = k7_up(static_cast<size_t>(16 + 32 * n_seq));
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
  // the cost of all items is counted in 32 bits
  const int64_t ratio = heads / kv_heads;
  const int64_t prefix_keys = static_cast<int64_t>(prefix_blocks) * block_size;
  const int64_t seq_keys = static_cast<int64_t>(max_blocks) * block_size;
  const int64_t row_blocks = n_groups == 0 ? 0 : n_groups + n_seq * ratio / K7_ROWS;
  auto most = [&](int64_t keys) { return K7_ITEM_COST + K7_BIG_COST * ((keys + K7_KEYS - 1) / K7_KEYS); };
  if (prefix_keys > 0x3fffffff || seq_keys > 0x3fffffff ||
      row_blocks * kv_heads * most(prefix_keys) + n_seq * kv_heads * most(seq_keys) > 0x3fffffff)
    return fail(TOME_ERR_TOO_LARGE, "the tables name too many keys for one call");
  if (static_cast<int64_t>(num_blocks) * kv_heads > 0x7fffffff / block_size)
    return fail(TOME_ERR_TOO_LARGE, "the pool has more than 2^31 - 1 rows");
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

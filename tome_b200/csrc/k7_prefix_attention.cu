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
// group against its prefix, or of one sequence against its suffix.  Items of more than 16 rows are
// "big": they go through the 5th-generation tensor core, tiles of 64 keys, a CTA at a time.  Items
// of up to 16 rows are "small": a warp alone takes one, tiles of 16 keys, through warp-level
// products (on the tensor-core path two to eight rows would cost what 128 do).  The tiles of each
// kind are laid end to end, and every CTA takes an equal run of the big ones, then each of its
// twelve warps an equal run of the small ones, whatever the lengths: the split follows from the
// lengths on the device alone.  A worker's part of an item is a piece; it leaves (sum of p v, row
// maximum, row sum) in the workspace, and a second kernel joins the pieces of a row.  A piece lies
// at (item index + worker index), which no two pieces share since at least one of the two grows
// from piece to piece.
//
// Measured (CUDA-graph replay; head_dim 128, ratio 4 unless said): 8 prompts of 8192 tokens with 16
// completions of up to 2048 each, 142 us, 5.3 TB/s (0.81 of a copy); 60000 tokens shared by 8 / 32
// sequences 57 / 66 us (0.66 / 0.57), one sequence of 60000 61 us; 16381 tokens shared by 64
// sequences, two row blocks that each read them, 48.6 us; 4 x 8 of 512 + 640 tokens (ratio 2) 18.5;
// 1 x 8 of 100 + 24 tokens (ratio 2) 10 us, of which this kernel works 3.8 (1.4 until the split is
// known); the rest is two launches and the second kernel.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>

#include <algorithm>
#include <type_traits>

#include "host_common.h"
#include "ptx.cuh"
#include "tensor_map.h"

namespace tome {

constexpr int K7_ROWS = 128;         // query rows of a big item at most (TMEM lanes)
constexpr int K7_SMALL_ROWS = 16;    // of a small one
constexpr int K7_KEYS = 64;          // keys of a big tile
constexpr int K7_SMALL_KEYS = 16;    // of a small one
// Rings of big tiles.  Even, so that a team meets a stage's phases one by one; values stay longer,
// from their load until the softmax of their tile is done.
constexpr int K7_K_STAGES = 4;
constexpr int K7_V_STAGES = 6;
constexpr int K7_SMALL_STAGES = 2;   // each warp's ring of small tiles
constexpr int K7_TEAM_WARPS = 4;     // a team takes every other big tile
constexpr int K7_SOFTMAX_WARPS = 2 * K7_TEAM_WARPS;
constexpr int K7_ISSUE_WARP = K7_SOFTMAX_WARPS;        // issues the products of the first team,
constexpr int K7_ISSUE_WARP_2 = K7_ISSUE_WARP + 1;     // of the second one
constexpr int K7_COPY_WARP = K7_ISSUE_WARP_2 + 1;      // fetches keys, the next one values
constexpr int K7_WARPS = K7_COPY_WARP + 2;             // all of them take small items
constexpr int K7_THREADS = K7_WARPS * 32;
// Cost of a small item besides its tiles, in tiles: the warp's ring runs dry where the queries come.
constexpr int K7_SMALL_ITEM_COST = 2;
// Cards of pieces in flight.  The warp that writes them is at most the ring's tiles ahead of the
// softmax warps (each piece has a tile), and a card is written over more pieces later than that.
constexpr int K7_CARDS = 8;
static_assert(K7_CARDS >= K7_K_STAGES + 3, "cards");
constexpr int K7_MAX_SEQ = 2048;
constexpr int K7_MAX_GROUPS = 512;
// The split takes at most this many CTAs (one per SM); the workspace does not depend on the
// device that it is asked for on.
constexpr int K7_MAX_CTAS = 160;
constexpr int K7_MAX_WORKERS = K7_MAX_CTAS * K7_WARPS;

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
  uint32_t div_magic, ratio_magic;  // x / block_size and x / ratio, see k7_div
  int32_t div_shift, ratio_shift;
  float c;                    // scale * log2(e)
  bool whole_pages;           // pages of a multiple of 16 tokens: tiles go by tensor copies
  int32_t big_box;            // sixteens of rows per tensor copy of a big tile: 1, 2 or 4
  int32_t ctas;               // CTAs of the main kernel
  double inv_ctas;            // 1 / ctas
  // workspace: the pieces' rows, those of big prefix items (128 per piece), of small ones (16) from
  // row small_rows on, of suffix items (ratio) from row suffix_rows on
  int4* plan;                 // [n_seq, heads] where a row's pieces are, see K7Where
  float* part_o;              // [rows, D]
  float2* part_ml;            // [rows] (maximum * c, sum)
  int64_t small_rows, suffix_rows;
  void* out;                  // [n_seq, heads, D]
  float* out_lse;             // [n_seq, heads] or null
  int32_t* status;
};

// A row's record: x, y first row and number of its prefix pieces, z, w of its suffix pieces.  The
// number of prefix pieces is negative where they are 16 rows apart.

__device__ __forceinline__ void k7_raise(int32_t* status, int32_t bit) {
  if (status != nullptr) atomicOr(status, bit);
}

// x / d for 0 <= x < 2^31 with s = ceil(log2 d), magic = floor(2^(31+s) / d) + 1, shift = 31 + s.
__device__ __forceinline__ int32_t k7_div(int32_t x, uint32_t magic, int32_t shift) {
  return static_cast<int32_t>(static_cast<uint64_t>(x) * magic >> shift);
}

// Length of a table's keys: never negative, never past the table.
__device__ __forceinline__ int32_t k7_length(const K7Params& p, int32_t len, int32_t blocks) {
  const int64_t most = static_cast<int64_t>(blocks) * p.block_size;
  return static_cast<int32_t>(max(int64_t{0}, min(static_cast<int64_t>(len), most)));
}

// ------------------------------------------------------------------ the split
__host__ __device__ constexpr int k7_keys(bool big) { return big ? K7_KEYS : K7_SMALL_KEYS; }
// Cost of an item besides its tiles.
__host__ __device__ constexpr int k7_extra(bool big) { return big ? 0 : K7_SMALL_ITEM_COST; }

__device__ __forceinline__ bool k7_is_big(int32_t rows) { return rows > K7_SMALL_ROWS; }
__device__ __forceinline__ int32_t k7_tiles(int32_t len, bool big) {
  return (len + k7_keys(big) - 1) / k7_keys(big);
}
__device__ __forceinline__ int32_t k7_item_cost(int32_t len, bool big) {
  return len == 0 ? 0 : k7_extra(big) + k7_tiles(len, big);
}
// Tiles that lie before the offset `cost` of an item.
__device__ __forceinline__ int32_t k7_cut(int32_t cost, bool big) { return max(cost - k7_extra(big), 0); }

// What every CTA works out of the lengths, in shared memory.
struct K7Plan {
  int32_t* group;     // [n_groups + 1] first sequence of each group (clamped, not decreasing)
  int32_t* block;     // [n_groups + 1] row blocks (of 128 rows) of the big groups before each group
  int32_t* prefix[2]; // [n_groups + 1] cost of the small [0] and big [1] prefix items before each group
  int32_t* suffix;    // [n_seq + 1] cost of the suffix items before each sequence
};

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

// Four values per lane from an array of n, 128 from `base` on; 0 past the end.  (All four loads are
// under way before the first scan waits for one.)
struct K7Four {
  int32_t v[4];
};
__device__ __forceinline__ K7Four k7_four(const int32_t* src, int n, int base, int lane) {
  K7Four f;
#pragma unroll
  for (int k = 0; k < 4; ++k) f.v[k] = base + 32 * k + lane < n ? __ldg(src + base + 32 * k + lane) : 0;
  return f;
}

// Warp 0: the groups; warp 1: the sequences.
__device__ __forceinline__ void k7_build_plan(const K7Params& p, const K7Plan& pl, int warp, int lane) {
  if (warp == 0) {
    K7Four len = k7_four(p.prefix_lens, p.n_groups, 0, lane);
    int32_t top = 0;
    for (int base = 0; base <= p.n_groups; base += 128) {
      const K7Four f = k7_four(p.group_starts, p.n_groups > 0 ? p.n_groups + 1 : 0, base, lane);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = base + 32 * k + lane;
        if (base + 32 * k > p.n_groups) break;
        const int32_t v = max(top, k7_scan_max(min(max(f.v[k], 0), p.n_seq), lane));
        if (i <= p.n_groups) pl.group[i] = v;
        top = __shfl_sync(0xffffffffu, v, 31);
      }
    }
    __syncwarp();
    int32_t blocks = 0, cost[2] = {0, 0};
    for (int base = 0; base < p.n_groups; base += 128) {
      if (base > 0) len = k7_four(p.prefix_lens, p.n_groups, base, lane);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = base + 32 * k + lane;
        if (base + 32 * k >= p.n_groups) break;
        int32_t b = 0, c[2] = {0, 0};
        if (i < p.n_groups) {
          const int32_t rows = (pl.group[i + 1] - pl.group[i]) * p.ratio, n = k7_length(p, len.v[k], p.prefix_blocks);
          if (k7_is_big(rows)) {
            b = (rows + K7_ROWS - 1) / K7_ROWS;
            c[1] = b * p.kv_heads * k7_item_cost(n, true);
          } else if (rows > 0) {
            c[0] = p.kv_heads * k7_item_cost(n, false);
          }
        }
        const int32_t bs = k7_scan_add(b, lane);
        if (i < p.n_groups) pl.block[i] = blocks + bs - b;
        blocks += __shfl_sync(0xffffffffu, bs, 31);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int32_t cs = k7_scan_add(c[s], lane);
          if (i < p.n_groups) pl.prefix[s][i] = cost[s] + cs - c[s];
          cost[s] += __shfl_sync(0xffffffffu, cs, 31);
        }
      }
    }
    if (lane == 0) {
      pl.block[p.n_groups] = blocks;
      pl.prefix[0][p.n_groups] = cost[0];
      pl.prefix[1][p.n_groups] = cost[1];
    }
  } else if (warp == 1) {
    const bool big = k7_is_big(p.ratio);
    int32_t cost = 0;
    for (int base = 0; base < p.n_seq; base += 128) {
      const K7Four len = k7_four(p.lengths, p.n_seq, base, lane);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i = base + 32 * k + lane;
        if (base + 32 * k >= p.n_seq) break;
        const int32_t c = i < p.n_seq ? p.kv_heads * k7_item_cost(k7_length(p, len.v[k], p.seq_blocks), big) : 0;
        const int32_t cs = k7_scan_add(c, lane);
        if (i < p.n_seq) pl.suffix[i] = cost + cs - c;
        cost += __shfl_sync(0xffffffffu, cs, 31);
      }
    }
    if (lane == 0) pl.suffix[p.n_seq] = cost;
  }
}

// Cost of all big or all small items.
__device__ __forceinline__ int32_t k7_cost(const K7Params& p, const K7Plan& pl, bool big) {
  return pl.prefix[big][p.n_groups] + (k7_is_big(p.ratio) == big ? pl.suffix[p.n_seq] : 0);
}

// The split of a kind's cost over the workers that take part: where the run of one begins, and the
// one that holds a place.  Every run is long enough to hold a tile of any item it goes through, but
// for the item's first and last run.  Quotients of up to 2^41 by products with a reciprocal, put
// right by one.
struct K7Split {
  int32_t cost, workers;
  double inv_workers;
  __device__ __forceinline__ K7Split(int32_t all, int32_t most, double inv_most, bool big)
      : cost(all),
        workers(all == 0 ? 0 : min(max(all / (k7_extra(big) + 1), 1), most)),
        inv_workers(workers == most ? inv_most : 1.0 / max(workers, 1)) {}
  static __device__ __forceinline__ int32_t quotient(int64_t a, int32_t b, double inv) {
    int64_t q = static_cast<int64_t>(static_cast<double>(a) * inv);
    const int64_t r = a - q * b;
    q += (r >= b) - (r < 0);
    return static_cast<int32_t>(q);
  }
  __device__ __forceinline__ int32_t begin(int32_t worker) const {
    return quotient(static_cast<int64_t>(worker) * cost, workers, inv_workers);
  }
  // the last worker that begins at the place or before it
  __device__ __forceinline__ int32_t holder(int32_t place) const {
    return quotient((static_cast<int64_t>(place) + 1) * workers - 1, cost, 1.0 / cost);
  }
};

// First of the workers that hold tiles of the item of `len` > 0 keys that begins at the place
// `begin`, and how many do.  (The first and the last run may hold less than a tile of it.)
__device__ __forceinline__ int2 k7_holders(const K7Split& split, int32_t begin, int32_t len, bool big) {
  const int32_t cost = k7_item_cost(len, big);
  int32_t w0 = split.holder(begin), w1 = split.holder(begin + cost - 1);
  if (k7_cut(min(split.begin(w0 + 1) - begin, cost), big) == 0) ++w0;
  if (k7_cut(max(split.begin(w1) - begin, 0), big) == k7_tiles(len, big)) --w1;
  return make_int2(w0, w1 - w0 + 1);
}

// A piece: tiles [tile, tile + n) of an item.
struct K7Piece {
  const int32_t* table;
  int32_t len;        // keys of the item
  int32_t tile, n;
  int32_t end;        // place where the item ends
  int32_t kv_head;
  int32_t seq0;       // first sequence of the rows
  int32_t row0;       // first row (row = (sequence - seq0) * ratio + head within the KV head)
  int32_t rows;
  int32_t item;       // index among the big prefix, small prefix or suffix items
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
__device__ __forceinline__ void k7_cut_piece(K7Piece& x, int32_t at, int32_t last, bool big) {
  const int32_t begin = x.end - k7_item_cost(x.len, big);
  x.tile = k7_cut(at - begin, big);
  x.n = k7_cut(min(last, x.end) - begin, big) - x.tile;
}

// The part of the item at the place `at` that lies before `last`.
template <bool BIG>
__device__ __forceinline__ K7Piece k7_piece(const K7Params& p, const K7Plan& pl, int32_t at, int32_t last) {
  K7Piece x;
  const int32_t* cum = pl.prefix[BIG];
  const int32_t in_prefix = cum[p.n_groups];
  x.prefix = at < in_prefix;
  if (x.prefix) {
    const int g = k7_find(cum, p.n_groups, at);
    x.seq0 = pl.group[g];
    const int32_t rows = (pl.group[g + 1] - x.seq0) * p.ratio;
    x.len = k7_length(p, p.prefix_lens[g], p.prefix_blocks);
    const int32_t cost = k7_item_cost(x.len, BIG);
    const int32_t i = (at - cum[g]) / cost;  // (row block, KV head)
    x.end = cum[g] + (i + 1) * cost;
    const int32_t mb = i / p.kv_heads;       // 0 for a small item
    x.kv_head = i - mb * p.kv_heads;
    x.row0 = mb * K7_ROWS;
    x.rows = min(K7_ROWS, rows - x.row0);
    x.item = ((BIG ? pl.block[g] : g) + mb) * p.kv_heads + x.kv_head;
    x.table = p.prefix_tables + static_cast<int64_t>(g) * p.prefix_blocks;
  } else {
    const int b = k7_find(pl.suffix, p.n_seq, at - in_prefix);
    x.seq0 = b;
    x.len = k7_length(p, p.lengths[b], p.seq_blocks);
    const int32_t cost = k7_item_cost(x.len, BIG), begin = in_prefix + pl.suffix[b];
    x.kv_head = (at - begin) / cost;
    x.end = begin + (x.kv_head + 1) * cost;
    x.row0 = 0;
    x.rows = p.ratio;
    x.item = b * p.kv_heads + x.kv_head;
    x.table = p.tables + static_cast<int64_t>(b) * p.seq_blocks;
  }
  k7_cut_piece(x, at, last, BIG);
  return x;
}

// Next piece with a tile of the run that goes on at `at` (x is the piece before, if `have`); moves
// `at` behind it.  As a rule it is the next KV head of the same rows and keys, else it is looked up.
template <bool BIG>
__device__ __forceinline__ bool k7_next(const K7Params& p, const K7Plan& pl, K7Piece& x, bool have,
                                        int32_t& at, int32_t last) {
  while (at < last) {
    if (have && at == x.end && x.kv_head + 1 < p.kv_heads) {
      x.kv_head += 1;
      x.item += 1;
      x.end += k7_item_cost(x.len, BIG);
      k7_cut_piece(x, at, last, BIG);
    } else {
      x = k7_piece<BIG>(p, pl, at, last);
      have = true;
    }
    at = min(last, x.end);
    if (x.n > 0) return true;
  }
  return false;
}

// First of the workspace's rows that belong to a piece.
__device__ __forceinline__ int64_t k7_out_row(const K7Params& p, bool prefix, bool big, int32_t item, int32_t worker) {
  const int64_t slot = static_cast<int64_t>(item) + worker;
  if (!prefix) return p.suffix_rows + slot * p.ratio;
  return big ? slot * K7_ROWS : p.small_rows + slot * K7_SMALL_ROWS;
}

// Pages of keys.  64 entries of the table from block `first` on, two per lane: a tile's pages come
// from there by shuffles, and the entries behind them are asked for long before they are needed.
struct K7Pages {
  int32_t first, a, b;
};
__device__ __forceinline__ int32_t k7_block(const K7Params& p, int32_t key) {
  return k7_div(key, p.div_magic, p.div_shift);
}
__device__ __forceinline__ int32_t k7_entry(const K7Params& p, const K7Piece& y, int32_t block) {
  return block <= k7_block(p, y.len - 1) ? __ldg(y.table + block) : -1;
}
__device__ __forceinline__ K7Pages k7_open_pages(const K7Params& p, const K7Piece& y, int32_t key0, int lane) {
  const int32_t f = k7_block(p, min(key0, y.len - 1));
  return K7Pages{f, k7_entry(p, y, f + lane), k7_entry(p, y, f + 32 + lane)};
}
// Moves the entries on so that `block`, which does not fall from call to call, is among the first 32.
__device__ __forceinline__ void k7_turn_pages(const K7Params& p, const K7Piece& y, K7Pages& w, int32_t block, int lane) {
  if (block - w.first < 32) return;
  if (block - w.first < 64) w = K7Pages{w.first + 32, w.b, k7_entry(p, y, w.first + 64 + lane)};
  else w = K7Pages{block, k7_entry(p, y, block + lane), k7_entry(p, y, block + 32 + lane)};
}
// The page of each lane's `block`, at most 31 behind `first` (the same for the whole warp).
__device__ __forceinline__ int32_t k7_page(const K7Params& p, const K7Piece& y, K7Pages& w, int32_t first,
                                           int32_t block, int lane) {
  k7_turn_pages(p, y, w, first, lane);
  const int32_t rel = block - w.first;  // 0 .. 62
  const int32_t a = __shfl_sync(0xffffffffu, w.a, rel & 31), b = __shfl_sync(0xffffffffu, w.b, rel & 31);
  return rel < 32 ? a : b;
}
// The pool's row (blocks and heads flattened) of key (key0 + lane), or -1; key0 does not fall from
// call to call, and no more than 32 keys from it on are asked for.
__device__ __forceinline__ int32_t k7_pool_row(const K7Params& p, const K7Piece& y, K7Pages& w, int32_t key0, int lane) {
  if (key0 >= y.len) return -1;
  const int32_t key = key0 + lane, lo = k7_block(p, key0);
  const int32_t blk = k7_block(p, min(key, y.len - 1)), page = k7_page(p, y, w, lo, blk, lane);
  if (key >= y.len) return -1;
  if (page < 0 || page >= p.num_blocks) {
    k7_raise(p.status, TOME_DEV_BLOCK_OUT_OF_RANGE);  // reads as zeros, as gather does
    return -1;
  }
  return (page * p.kv_heads + y.kv_head) * p.block_size + (key - blk * p.block_size);
}

// The pool's row of key0 where it and the fifteen behind it lie in one page of whole tiles, else -1.
// The same for the whole warp.
__device__ __forceinline__ int32_t k7_whole_row(const K7Params& p, const K7Piece& y, K7Pages& w, int32_t key0, int lane) {
  if (!p.whole_pages || key0 + 16 > y.len) return -1;
  const int32_t blk = k7_block(p, key0);
  k7_turn_pages(p, y, w, blk, lane);
  const int32_t page = __shfl_sync(0xffffffffu, w.a, blk - w.first);
  if (page < 0 || page >= p.num_blocks) return -1;
  return (page * p.kv_heads + y.kv_head) * p.block_size + (key0 - blk * p.block_size);
}

// What the softmax warps need of a big piece, written by the first copying thread ahead of them;
// n = 0 behind the last one.
struct K7Card {
  int32_t len, tile, n, rows, item, prefix, seq0, row0, kv_head;
};

// ------------------------------------------------------------------ shared memory and products
// Tiles of 128-byte rows, 128-byte swizzle: 16-byte piece c of row r of a 64-column block sits
// at r * 128 + ((c ^ (r & 7)) << 4).
template <int D>
struct K7Smem {
  // tensor memory: each team's two S (64 columns; P, two 16-bit values per column, takes the place of
  // the S it is made of), then each team's O
  static constexpr int O_COL = 4 * K7_KEYS;
  static constexpr int TMEM_COLS = 512;
  static_assert(O_COL + 2 * D <= TMEM_COLS, "tensor memory");
  static constexpr int Q_BYTES = K7_ROWS * D * 2;
  static constexpr int KV_BYTES = K7_KEYS * D * 2;
  static constexpr int Q = 0;
  static constexpr int K = Q + Q_BYTES;                    // K_STAGES
  static constexpr int V = K + K7_K_STAGES * KV_BYTES;     // V_STAGES
  // small items: each warp's ring of tiles lies in the same space
  static constexpr int SMALL_KV = K7_SMALL_KEYS * D * 2;
  static constexpr int SMALL_STAGE = 2 * SMALL_KV;
  static constexpr int SMALL = K7_WARPS * K7_SMALL_STAGES * SMALL_STAGE;
  static constexpr int MEET_ML = V + K7_V_STAGES * KV_BYTES; // [2 teams][128] float2
  static_assert(SMALL <= MEET_ML, "small tiles");
  static constexpr int BARS = MEET_ML + 2 * K7_ROWS * 8;
  static constexpr int K_FULL = BARS;                      // stages, as the next three
  static constexpr int K_EMPTY = K_FULL + K7_K_STAGES * 8;
  static constexpr int V_FULL = K_EMPTY + K7_K_STAGES * 8;
  static constexpr int V_EMPTY = V_FULL + K7_V_STAGES * 8;
  static constexpr int S_FULL = V_EMPTY + K7_V_STAGES * 8; // 2 (teams) x 2, as the next
  static constexpr int P_FULL = S_FULL + 32;
  static constexpr int O_FULL = P_FULL + 32;               // 2 (teams), as the next
  static constexpr int Q_FULL = O_FULL + 16;
  static constexpr int MEET = Q_FULL + 16;                 // the softmax warps among themselves
  static constexpr int TMEM = MEET + 16;
  static constexpr int CARD_FULL = TMEM + 16;              // K7_CARDS
  static constexpr int CARDS = CARD_FULL + K7_CARDS * 8;
  static constexpr int SMALL_FULL = CARDS + K7_CARDS * static_cast<int>(sizeof(K7Card));  // each warp's, STAGES
  static constexpr int PLAN = SMALL_FULL + K7_WARPS * K7_SMALL_STAGES * 8;
  static constexpr int plan_bytes(int n_groups, int n_seq) {
    return 4 * (4 * (n_groups + 1) + n_seq + 1);
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

// A whole warp waits.  Either all its lanes go on or none does: one lane whose wait ran out must not
// leave the others at a vote.
__device__ __forceinline__ bool k7_wait(uint32_t bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity));
}

// All softmax warps meet: what each wrote before is visible to all behind.  An mbarrier rather than
// a hardware barrier, so that the wait has a limit too; `met` counts the meetings.
__device__ __forceinline__ void k7_meet(const K7Params& p, uint32_t bar, uint32_t& met, int lane, bool& ok) {
  __syncwarp();
  if (lane == 0) mbar_arrive(bar);
  if (ok && !k7_wait(bar, met & 1u)) {
    k7_raise(p.status, TOME_DEV_TIMEOUT);
    ok = false;
  }
  ++met;
  __syncwarp();
}

// ------------------------------------------------------------------ small items
// A warp's run of small tiles.  It fetches its own keys and values, a tile ahead, and keeps running
// maximum, sum and the sums of p v in registers: nothing is shared with another warp, and twelve of
// them hide one another's latencies.  A tile that lies within a page (pages of a multiple of 16
// tokens) comes by tensor copies, swizzled as the matrix loads want it, which one lane issues; the
// asynchronous copies of 16 bytes that the others take keep a warp busy for 900 clocks per tile.
template <typename T, int D>
__device__ __forceinline__ void k7_small_run(const K7Params& p, const CUtensorMap* k_map, const CUtensorMap* v_map,
                                             const K7Plan& pl, uint32_t ring, uint32_t full, int32_t worker,
                                             int32_t first, int32_t last, int lane) {
  using S = K7Smem<D>;
  constexpr int PIECES = D / 8;                     // 16-byte pieces of a row
  constexpr int AT_ONCE = 32 / PIECES;              // rows copied per step
  constexpr int STEPS = K7_SMALL_KEYS / AT_ONCE;
  constexpr int BLOCK = K7_SMALL_KEYS * 128;        // bytes of a 64-column block of a tile
  // the copying side, a tile ahead of the products
  K7Piece cp = {};
  int32_t cp_at = first, cp_j = 0;
  K7Pages pages = {};
  bool cp_there = true, cp_have = false;
  const int c = lane % PIECES, sub = lane / PIECES;
  const T* k_pool = reinterpret_cast<const T*>(p.k_pool) + c * 8;
  const T* v_pool = reinterpret_cast<const T*>(p.v_pool) + c * 8;
  uint32_t filled = 0, used = 0;  // tiles
  uint32_t by_hand = 0;           // stages whose last tile did not come by tensor copies
  auto fill = [&]() {  // the next tile into the ring (or nothing)
    if (cp_j == cp.n && cp_there) {
      const int32_t* table = cp.table;
      cp_there = k7_next<false>(p, pl, cp, cp_have, cp_at, last);
      cp_have = true;
      cp_j = 0;
      if (cp_there) {  // the next KV head's keys lie in the same pages
        const int32_t key0 = cp.tile * K7_SMALL_KEYS, ahead = k7_block(p, key0) - pages.first;
        if (cp.table != table || ahead < 0 || ahead >= 32) pages = k7_open_pages(p, cp, key0, lane);
      }
    }
    if (cp_there) {
      const int32_t key0 = (cp.tile + cp_j) * K7_SMALL_KEYS;
      const uint32_t stage = filled % K7_SMALL_STAGES, bar = full + stage * 8, dst = ring + stage * S::SMALL_STAGE;
      const int32_t row0 = k7_whole_row(p, cp, pages, key0, lane);
      if (row0 >= 0) {
        if (by_hand >> stage & 1u) {  // ordinary writes before the tensor copy's
          fence_proxy_async();
          __syncwarp();
          by_hand &= ~(1u << stage);
        }
        if (lane == 0) {
          mbar_expect_tx(bar, S::SMALL_STAGE);
          mbar_arrive_many(bar, 32);
#pragma unroll
          for (int h = 0; h < D / 64; ++h) {
            tma_load_2d(dst + h * BLOCK, k_map, h * 64, row0, bar);
            tma_load_2d(dst + S::SMALL_KV + h * BLOCK, v_map, h * 64, row0, bar);
          }
        }
      } else {
        by_hand |= 1u << stage;
        const int32_t row = k7_pool_row(p, cp, pages, key0, lane);
#pragma unroll 1
        for (int i = 0; i < STEPS; ++i) {
          const int r = i * AT_ONCE + sub;
          const int32_t from = __shfl_sync(0xffffffffu, row, r);
          const int64_t off = static_cast<int64_t>(max(from, 0)) * D;
          const uint32_t to = dst + (c >> 3) * BLOCK + r * 128 + (((c & 7) ^ (r & 7)) << 4);
          k7_copy16(to, k_pool + off, from >= 0);
          k7_copy16(to + S::SMALL_KV, v_pool + off, from >= 0);
        }
        k7_copies_arrive(bar);
      }
      ++filled;
      ++cp_j;
    }
  };
  fill();

  const int g = lane >> 2;  // this thread's rows: g and g + 8; its columns: 2 (lane & 3) + {0, 1} of eight
  const int k_row = (lane & 7) + ((lane >> 4) << 3), k_c = (lane >> 3) & 1;  // where the lane points
  const int v_row = lane & 15, v_c = lane >> 4;                              // the matrix loads to
  // places in a tile that the lane's matrix loads read: column pairs k, k + 4 lie a block apart
  uint32_t k_spot[4], v_spot[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    k_spot[k] = ring + k_row * 128 + (((2 * k + k_c) ^ (k_row & 7)) << 4);
    v_spot[k] = ring + S::SMALL_KV + v_row * 128 + (((2 * k + v_c) ^ (v_row & 7)) << 4);
  }
  while (cp_there) {
    // the piece of the tile that was copied last; its other tiles follow
    const int32_t len = cp.len, tile = cp.tile, n = cp.n, rows = cp.rows;
    const int64_t out_row = k7_out_row(p, cp.prefix, false, cp.item, worker);
    // queries, straight into the products' layout
    uint32_t qf[D / 16][4];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int32_t row = g + 8 * r, s = k7_div(row, p.ratio_magic, p.ratio_shift);
      const uint32_t* src = reinterpret_cast<const uint32_t*>(
          reinterpret_cast<const T*>(p.q) + (cp.seq0 + s) * p.q_stride +
          static_cast<int64_t>(cp.kv_head * p.ratio + (row - s * p.ratio)) * D) + (lane & 3);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        qf[k][r] = row < rows ? __ldg(src + 8 * k) : 0u;
        qf[k][2 + r] = row < rows ? __ldg(src + 8 * k + 4) : 0u;
      }
    }
    float o[D / 8][4];
#pragma unroll
    for (int k = 0; k < D / 8; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[k][e] = 0.0f;
    float ref[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
#pragma unroll 1
    for (int32_t j = 0; j < n; ++j) {
      __syncwarp();  // the tile before, whose place is filled now, is done with
      fill();
      const uint32_t read_at = (used % K7_SMALL_STAGES) * S::SMALL_STAGE;
      // (whether it came is voted on below, together with the maxima: a vote of its own took another 1.5 %)
      const bool there = mbar_wait(full + (used % K7_SMALL_STAGES) * 8, (used / K7_SMALL_STAGES) & 1u);
      __syncwarp();
      ++used;
      float s[2][4] = {}, s2[2][4] = {};  // two chains of products for each eight keys
      uint32_t f[D / 16][4];
      // all loads of the keys first: no load's latency stands before a product
#pragma unroll
      for (int k = 0; k < D / 16; ++k) k7_ldmatrix(k_spot[k % 4] + read_at + (k / 4) * BLOCK, f[k]);
#pragma unroll
      for (int k = 0; k < D / 16; k += 2) {
        k7_mma(s[0], qf[k], f[k][0], f[k][1], T());
        k7_mma(s[1], qf[k], f[k][2], f[k][3], T());
        k7_mma(s2[0], qf[k + 1], f[k + 1][0], f[k + 1][1], T());
        k7_mma(s2[1], qf[k + 1], f[k + 1][2], f[k + 1][3], T());
      }
#pragma unroll
      for (int k = 0; k < D / 16; ++k) k7_ldmatrix_trans(v_spot[k % 4] + read_at + (k / 4) * BLOCK, f[k]);
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] += s2[n][e];
      const int32_t valid = len - (tile + j) * K7_SMALL_KEYS;
      if (valid < K7_SMALL_KEYS) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n * 8 + 2 * (lane & 3) + (e & 1) >= valid) s[n][e] = -INFINITY;
      }
      // The exponents' reference moves only when a score exceeds it by more than 2^8, which one
      // vote finds out; the row maxima are formed only then.
      float top[2];
      bool grow = !there;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        top[r] = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1])) * p.c;
        grow |= top[r] > ref[r] + 8.0f;
      }
      if (__any_sync(0xffffffffu, grow)) {
        if (!__all_sync(0xffffffffu, there)) {  // the whole warp gives up
          k7_raise(p.status, TOME_DEV_TIMEOUT);
          asm volatile("cp.async.wait_all;" ::: "memory");
          return;
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
          top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
          const float next = fmaxf(ref[r], top[r]);
          const float alpha = next == -INFINITY ? 1.0f : ex2f(ref[r] - next);
          ref[r] = next;
          sum[r] *= alpha;
#pragma unroll
          for (int k = 0; k < D / 8; ++k) {
            o[k][2 * r] *= alpha;
            o[k][2 * r + 1] *= alpha;
          }
        }
      }
      // a row that has seen nothing but -inf takes 0 as its reference: all its p are 0
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
      for (int k = 0; k < D / 16; ++k) {
        k7_mma(o[2 * k], pf, f[k][0], f[k][1], T());
        k7_mma(o[2 * k + 1], pf, f[k][2], f[k][3], T());
      }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
      if (g + 8 * r < rows) {
        float* dst = p.part_o + (out_row + g + 8 * r) * D + 2 * (lane & 3);
#pragma unroll
        for (int k = 0; k < D / 8; ++k) *reinterpret_cast<float2*>(dst + 8 * k) = make_float2(o[k][2 * r], o[k][2 * r + 1]);
        if ((lane & 3) == 0) p.part_ml[out_row + g + 8 * r] = make_float2(ref[r], sum[r]);
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// ------------------------------------------------------------------ big items
// Softmax of a piece: thread = row, the team's tiles in turn.
template <typename T, int D>
__device__ __forceinline__ bool k7_big_piece(const K7Params& p, uint8_t* smem, uint32_t base, uint32_t tmem,
                                             const K7Card& x, uint32_t& u, int warp, int lane,
                                             float* out_o, float2* out_ml, uint32_t& met) {
  using S = K7Smem<D>;
  const uint32_t team = warp / K7_TEAM_WARPS;
  const int row = (warp % K7_TEAM_WARPS) * 32 + lane;
  const uint32_t lanes = static_cast<uint32_t>((warp % K7_TEAM_WARPS) * 32) << 16;
  const bool active = (warp % K7_TEAM_WARPS) * 32 < x.rows;  // warps without a row only keep step
  const uint32_t o_addr = tmem + lanes + S::O_COL;
  bool ok = true;
  {  // the piece's queries, a warp's share of the rows (nothing reads the last piece's any more)
    constexpr int PIECES = D / 8, AT_ONCE = 32 / PIECES;
    const int c = lane % PIECES;
    for (int i = warp * AT_ONCE + lane / PIECES; i < x.rows; i += K7_SOFTMAX_WARPS * AT_ONCE) {
      const int32_t r = x.row0 + i, s = k7_div(r, p.ratio_magic, p.ratio_shift);
      k7_copy16(base + S::Q + (c >> 3) * (K7_ROWS * 128) + i * 128 + (((c & 7) ^ (i & 7)) << 4),
                reinterpret_cast<const T*>(p.q) + (x.seq0 + s) * p.q_stride +
                    static_cast<int64_t>(x.kv_head * p.ratio + (r - s * p.ratio)) * D + c * 8,
                true);
    }
    for (uint32_t t = 0; t < 2; ++t)  // tell the teams that have a tile of the piece
      if (x.n > 1 || (u & 1u) == t) k7_copies_arrive(base + S::Q_FULL + t * 8);
  }
  // `ref` is what the exponents are relative to, in the log2 domain.  It follows the row's maximum
  // only when that has grown by more than 2^8: the sums in tensor memory then have to be
  // rescaled, which hardly ever happens after the first tiles.
  float ref = -INFINITY, sum = 0.0f;
  const uint32_t end = u + x.n, mine = u + ((u ^ team) & 1u);
  for (uint32_t i = mine; i < end && ok; i += 2) {
    const uint32_t n = i >> 1, half = 2 * team + (n & 1u);  // the team's n-th tile, in its S number n & 1
    const uint32_t s_addr = tmem + lanes + half * K7_KEYS;
    if (!k7_wait(base + S::S_FULL + half * 8, (n >> 1) & 1u)) {
      k7_raise(p.status, TOME_DEV_TIMEOUT);
      ok = false;
    }
    if (active) {
      tc_fence_after_sync();
      uint32_t s0[32], s1[32];
      tmem_ld32(s_addr, s0);
      tmem_ld32(s_addr + 32, s1);
      tmem_ld_wait_dep(s0);
      tmem_ld_wait_dep(s1);
      const int32_t valid = x.len - (x.tile + static_cast<int32_t>(i - u)) * K7_KEYS;
      if (valid < K7_KEYS) {
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          if (k >= valid) s0[k] = 0xff800000u;
          if (k + 32 >= valid) s1[k] = 0xff800000u;
        }
      }
      float big[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int k = 0; k < 32; ++k)
        big[k & 3] = fmax3(big[k & 3], __uint_as_float(s0[k]), __uint_as_float(s1[k]));
      const float top = fmaxf(fmaxf(big[0], big[1]), fmaxf(big[2], big[3])) * p.c;
      // (lanes beyond the rows hold whatever the last piece left)
      const bool grow = row < x.rows && (top > ref + 8.0f || (i == mine && top > ref));
      if (__any_sync(0xffffffffu, grow)) {
        const float next = grow ? top : ref;
        const float alpha = next == -INFINITY ? 1.0f : ex2f(ref - next);
        sum *= alpha;
        ref = next;
        if (i > mine) {
          // P V of the team's tile before is done (the next one waits for this tile's P)
          if (!k7_wait(base + S::O_FULL + team * 8, (n - 1) & 1u)) {
            k7_raise(p.status, TOME_DEV_TIMEOUT);
            ok = false;
          }
          tc_fence_after_sync();
#pragma unroll 1
          for (int h = 0; h < D; h += 32) {
            uint32_t r[32];
            tmem_ld32(o_addr + team * D + h, r);
            tmem_ld_wait_dep(r);
#pragma unroll
            for (int k = 0; k < 32; ++k) r[k] = __float_as_uint(__uint_as_float(r[k]) * alpha);
            tmem_st32(o_addr + team * D + h, r);
          }
        }
      }
      // a row that has seen nothing but -inf takes 0 as its reference: all its p are 0
      const float off = ref == -INFINITY ? 0.0f : -ref;
      const float2 c2 = make_float2(p.c, p.c), off2 = make_float2(off, off);
      float2 la = make_float2(0.0f, 0.0f), lb = la;
      uint32_t pw[32];
#pragma unroll
      for (int k = 0; k < 32; ++k) {  // two keys
        float2 e = k < 16 ? make_float2(__uint_as_float(s0[2 * k]), __uint_as_float(s0[2 * k + 1]))
                          : make_float2(__uint_as_float(s1[2 * k - 32]), __uint_as_float(s1[2 * k - 31]));
        e = __ffma2_rn(e, c2, off2);
        e.x = ex2f(e.x);
        e.y = ex2f(e.y);
        if (k & 1) la = __fadd2_rn(la, e);
        else lb = __fadd2_rn(lb, e);
        pw[k] = k7_pack(e.x, e.y, T());
      }
      tmem_st32(s_addr, pw);
      sum += (la.x + la.y) + (lb.x + lb.y);
      tmem_st_wait();
      tc_fence_before_sync();
    }
    // The piece's last P is handed over when P V of the tile before is done: a phase is known by its
    // parity alone, so that the wait for the last P V must not find the one before under way.  (The
    // phase before that one is over, S of this tile was made behind it.)
    if (i > mine && i + 2 >= end && !k7_wait(base + S::O_FULL + team * 8, (n - 1) & 1u)) {
      k7_raise(p.status, TOME_DEV_TIMEOUT);
      ok = false;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(base + S::P_FULL + half * 8);
  }
  // The teams' sums meet: each team brings the rows' reference and sum, then writes half of the
  // columns from both teams' O.
  float2* const ml = reinterpret_cast<float2*>(smem + S::MEET_ML);
  if (mine < end && ok) {
    const uint32_t n = (end - 1 - ((end - 1 - mine) & 1u)) >> 1;  // the team's last tile
    if (!k7_wait(base + S::O_FULL + team * 8, n & 1u)) {
      k7_raise(p.status, TOME_DEV_TIMEOUT);
      ok = false;
    }
    tc_fence_after_sync();
  }
  u = end;
  ml[team * K7_ROWS + row] = make_float2(ref, sum);
  tc_fence_before_sync();
  k7_meet(p, base + S::MEET, met, lane, ok);
  tc_fence_after_sync();
  if (active) {
    const float2 a = ml[row], b = ml[K7_ROWS + row];
    const float top = fmaxf(a.x, b.x);
    // a team without a finite score has the weight 0 (also one without a tile, whose O is
    // another piece's), or 1 where it holds a NaN
    const float wa = a.x == -INFINITY ? (a.y == 0.0f ? 0.0f : 1.0f) : ex2f(a.x - top);
    const float wb = b.x == -INFINITY ? (b.y == 0.0f ? 0.0f : 1.0f) : ex2f(b.x - top);
    float* dst = out_o + row * D + team * (D / 2);
#pragma unroll 1
    for (int h = 0; h < D / 2; h += 32) {
      uint32_t ra[32], rb[32];
      tmem_ld32(o_addr + team * (D / 2) + h, ra);
      tmem_ld32(o_addr + D + team * (D / 2) + h, rb);
      tmem_ld_wait_dep(ra);
      tmem_ld_wait_dep(rb);
      if (row < x.rows) {
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          const float va = wa == 0.0f ? 0.0f : __uint_as_float(ra[k]) * wa;
          ra[k] = __float_as_uint(wb == 0.0f ? va : fmaf(__uint_as_float(rb[k]), wb, va));
        }
#pragma unroll
        for (int k = 0; k < 32; k += 4) stg128(dst + h + k, make_uint4(ra[k], ra[k + 1], ra[k + 2], ra[k + 3]));
      }
    }
    if (team == 0 && row < x.rows) out_ml[row] = make_float2(top, fmaf(wa, a.y, wb * b.y));
  }
  tc_fence_before_sync();
  k7_meet(p, base + S::MEET, met, lane, ok);  // O, and the space of the exchange, may be written again
  return ok;
}

// Pipeline of the big items: two warps fetch keys and values (tensor copies of 16 to 64 rows where pages
// allow it, else asynchronous copies of 16 bytes; rows past the end are zeros) into rings
// which drain at their own pace.  Two teams take the tiles in turn: a thread issues
// S = Q K^T (128 x 64 x D) and O += P V (128 x D x 64, P read from tensor memory), four warps own a row
// per thread and keep its running maximum and sum; the teams' O meet at the end of a piece.  A
// team has two S, so that the products of its next tile run under the softmax of this one.
//
// Per tile at D = 128: 32 KB from HBM at its rate 1400 clocks, the tensor pipe 640 (48 clocks per
// 128 x 64 x 16 with A from shared memory, 64 per 128 x 128 x 16), a warp's softmax 1250 for every
// other tile.  One thread for both teams' products bound the kernel at 1700 clocks per tile, one
// S per team at 1370 together with a copying warp that looked up every tile's pages and issued eight
// copies of 16 rows (1200 clocks); queries in tensor memory made no difference.
template <typename T, int D>
__global__ void __launch_bounds__(K7_THREADS, 1) k7_attention_kernel(
    const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
    const __grid_constant__ CUtensorMap k_map_16, const __grid_constant__ CUtensorMap v_map_16, const K7Params p) {
  using S = K7Smem<D>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;  // swizzled tiles want 1024-byte alignment
  uint8_t* smem = smem_raw + (base - raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  K7Plan pl;
  pl.group = reinterpret_cast<int32_t*>(smem + S::PLAN);
  pl.block = pl.group + p.n_groups + 1;
  pl.prefix[0] = pl.block + p.n_groups + 1;
  pl.prefix[1] = pl.prefix[0] + p.n_groups + 1;
  pl.suffix = pl.prefix[1] + p.n_groups + 1;
  K7Card* const cards = reinterpret_cast<K7Card*>(smem + S::CARDS);

  if (threadIdx.x == K7_ISSUE_WARP * 32) {
    for (int i = 0; i < K7_K_STAGES; ++i) {
      mbar_init(base + S::K_FULL + i * 8, 32);
      mbar_init(base + S::K_EMPTY + i * 8, 1);
    }
    for (int i = 0; i < K7_V_STAGES; ++i) {
      mbar_init(base + S::V_FULL + i * 8, 32);
      mbar_init(base + S::V_EMPTY + i * 8, 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(base + S::S_FULL + i * 8, 1);
      mbar_init(base + S::P_FULL + i * 8, K7_TEAM_WARPS);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(base + S::O_FULL + i * 8, 1);
      mbar_init(base + S::Q_FULL + i * 8, K7_SOFTMAX_WARPS * 32);
    }
    mbar_init(base + S::MEET, K7_SOFTMAX_WARPS);
    for (int i = 0; i < K7_CARDS; ++i) mbar_init(base + S::CARD_FULL + i * 8, 1);
    for (int i = 0; i < K7_WARPS * K7_SMALL_STAGES; ++i) mbar_init(base + S::SMALL_FULL + i * 8, 32);
    fence_mbar_init();
  }
  griddep_wait();  // what the kernels before write is read from here on
  griddep_launch_dependents();
  k7_build_plan(p, pl, warp, lane);
  __syncthreads();
  const K7Split big(k7_cost(p, pl, true), p.ctas, p.inv_ctas, true);
  const K7Split small(k7_cost(p, pl, false), p.ctas * K7_WARPS, p.inv_ctas / K7_WARPS, false);

  if (big.cost > 0) {  // (the same for all threads of all CTAs)
    if (warp == K7_ISSUE_WARP) {
      tmem_alloc(base + S::TMEM, S::TMEM_COLS);
      tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + S::TMEM);
    const bool works = static_cast<int32_t>(blockIdx.x) < big.workers;
    const int32_t first = works ? big.begin(blockIdx.x) : 0;
    const int32_t last = works ? big.begin(blockIdx.x + 1) : 0;
    if (warp < K7_SOFTMAX_WARPS) {
      // ---------------------------------------------------------- softmax
      uint32_t u = 0, piece = 0, met = 0;  // tiles, pieces, meetings so far; a tile's team is its parity
      for (bool ok = true; ok; ++piece) {
        if (!k7_wait(base + S::CARD_FULL + (piece % K7_CARDS) * 8, (piece / K7_CARDS) & 1u)) {
          k7_raise(p.status, TOME_DEV_TIMEOUT);
          break;
        }
        const K7Card x = cards[piece % K7_CARDS];
        if (x.n == 0) break;
        const int64_t out_row = k7_out_row(p, x.prefix != 0, true, x.item, blockIdx.x);
        ok = k7_big_piece<T, D>(p, smem, base, tmem, x, u, warp, lane, p.part_o + out_row * D, p.part_ml + out_row, met);
      }
    } else if (warp == K7_ISSUE_WARP || warp == K7_ISSUE_WARP_2) {
      // ---------------------------------------------------------- tensor-core products of a team
      if (lane == 0) {
        const uint32_t team = warp == K7_ISSUE_WARP ? 0u : 1u;
        const uint64_t q_desc = k7_desc_k(base + S::Q), k_desc = k7_desc_k(base + S::K);
        const uint64_t v_desc = k7_desc_mn(base + S::V, K7_KEYS * 128);
        const uint32_t s_addr = tmem + 2 * team * K7_KEYS, o_addr = tmem + S::O_COL + team * D;
        const uint32_t s_full = base + S::S_FULL + 16 * team, p_full = base + S::P_FULL + 16 * team;
        const uint32_t o_full = base + S::O_FULL + 8 * team;
        uint32_t u = 0, piece = 0, pieces = 0, last_mine = 0;  // `pieces`: those with a tile of the team
        bool ok = true, any = false;
        auto multiply_qk = [&](uint32_t i) {  // S = Q K^T of tile i
          const uint32_t stage = i % K7_K_STAGES, half = (i >> 1) & 1u;
          if (!mbar_wait(base + S::K_FULL + stage * 8, (i / K7_K_STAGES) & 1u)) ok = false;
          if (!ok) return;
          fence_proxy_async();  // tiles that did not come by tensor copies are ordinary writes
          tc_fence_after_sync();
          const uint64_t a = q_desc, b = k_desc + stage * (S::KV_BYTES >> 4);
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            umma_bf16_ss(s_addr + half * K7_KEYS, a + (k / 4) * (K7_ROWS * 128 >> 4) + 2 * (k % 4),
                         b + (k / 4) * (K7_KEYS * 128 >> 4) + 2 * (k % 4), k7_idesc<T>(K7_KEYS, false), k != 0);
          umma_commit(s_full + half * 8);
          umma_commit(base + S::K_EMPTY + stage * 8);
        };
        auto multiply_pv = [&](uint32_t i, bool add) {  // O (+)= P V of tile i
          const uint32_t stage = i % K7_V_STAGES, half = (i >> 1) & 1u;
          if (!mbar_wait(p_full + half * 8, (i >> 2) & 1u)) ok = false;
          if (!mbar_wait(base + S::V_FULL + stage * 8, (i / K7_V_STAGES) & 1u)) ok = false;
          if (!ok) return;
          fence_proxy_async();
          tc_fence_after_sync();
          const uint64_t b = v_desc + stage * (S::KV_BYTES >> 4);
#pragma unroll
          for (int k = 0; k < K7_KEYS / 16; ++k)  // 16 keys: 8 columns of P, 16 rows of V
            umma_f16_ts(o_addr, s_addr + half * K7_KEYS + 8 * k, b + (2048 >> 4) * k, k7_idesc<T>(D, true), add || k != 0);
          umma_commit(o_full);
          umma_commit(base + S::V_EMPTY + stage * 8);
          any = true;
          last_mine = i;
        };
        K7Piece x;
        int32_t at = first;
        for (; ok && k7_next<true>(p, pl, x, piece > 0, at, last); ++piece) {
          const uint32_t end = u + x.n, mine = u + ((u ^ team) & 1u);
          if (mine < end) {
            if (!mbar_wait(base + S::Q_FULL + team * 8, pieces++ & 1u)) ok = false;
            if (ok) multiply_qk(mine);
            if (ok && mine + 2 < end) multiply_qk(mine + 2);
          }
          for (uint32_t i = mine; i < end && ok; i += 2) {
            multiply_pv(i, i > mine);
            if (!ok || i + 4 >= end) continue;
            // the S that the tile's P lay in is free once that has been read
            if (!mbar_wait(o_full, (i >> 1) & 1u)) ok = false;
            if (ok) multiply_qk(i + 4);
          }
          u = end;
        }
        // nothing may still be under way when the space is used otherwise
        if (any && !mbar_wait(o_full, (last_mine >> 1) & 1u)) ok = false;
        if (!ok) k7_raise(p.status, TOME_DEV_TIMEOUT);
      }
      __syncwarp();
    } else {
      // ---------------------------------------------------------- copies
      constexpr int PIECES = D / 8;                  // 16-byte pieces of a row
      constexpr int AT_ONCE = 32 / PIECES;           // rows copied per step
      constexpr int STEPS = 16 / AT_ONCE;            // for sixteen rows
      const bool keys = warp == K7_COPY_WARP;        // the other one: values
      const int c = lane % PIECES, sub = lane / PIECES;
      const T* pool = reinterpret_cast<const T*>(keys ? p.k_pool : p.v_pool) + c * 8;
      const CUtensorMap* map = keys ? &k_map : &v_map;
      const uint32_t stages = keys ? K7_K_STAGES : K7_V_STAGES;
      const uint32_t area = base + (keys ? S::K : S::V);
      const uint32_t full = base + (keys ? S::K_FULL : S::V_FULL), empty = base + (keys ? S::K_EMPTY : S::V_EMPTY);
      auto show = [&](const K7Piece& y, uint32_t index, bool there) {  // to the softmax warps
        if (keys && lane == 0) {
          cards[index % K7_CARDS] = K7Card{y.len, y.tile, there ? y.n : 0, y.rows, y.item, y.prefix ? 1 : 0, y.seq0, y.row0, y.kv_head};
          mbar_arrive(base + S::CARD_FULL + (index % K7_CARDS) * 8);
        }
      };
      uint32_t t = 0, piece = 0, by_hand = 0;
      bool ok = true;
      int32_t at = first;
      K7Piece x = {};
      K7Pages pages = {};
      // Where whole pages hold them, the pool rows of a piece's groups of sixteen keys are looked up 32
      // at a time, one per lane, and the pages behind those are asked for meanwhile: with a look-up per
      // tile this warp, not the memory, set the pace.
      auto page_of = [&](const K7Piece& y, int32_t group) {
        const int32_t key = (group + lane) * 16;
        return p.whole_pages && key + 16 <= y.len ? __ldg(y.table + k7_block(p, key)) : -1;
      };
      int32_t ahead = -1, row = -1;
      uint32_t good = 0;  // the groups that have a row
      bool there = k7_next<true>(p, pl, x, false, at, last);
      show(x, 0, there);
      if (there) {
        pages = k7_open_pages(p, x, x.tile * K7_KEYS, lane);
        ahead = page_of(x, x.tile * (K7_KEYS / 16));
      }
      while (there && ok) {
        K7Piece next = x;
        K7Pages next_pages = {};
        int32_t next_ahead = -1;
        bool next_there = false;
        for (int32_t j = 0; j < x.n; ++j, ++t) {
          const uint32_t stage = t % stages;
          if (j + 1 == x.n) {  // the piece behind is looked up while this one's loads are under way
            next_there = k7_next<true>(p, pl, next, true, at, last);
            show(next, piece + 1, next_there);
            if (next_there) {
              next_pages = k7_open_pages(p, next, next.tile * K7_KEYS, lane);
              next_ahead = page_of(next, next.tile * (K7_KEYS / 16));
            }
          }
          if (j % 8 == 0) {
            const int32_t group = (x.tile + j) * (K7_KEYS / 16), key = (group + lane) * 16;
            row = ahead < 0 || ahead >= p.num_blocks
                      ? -1
                      : (ahead * p.kv_heads + x.kv_head) * p.block_size + (key - k7_block(p, key) * p.block_size);
            good = __ballot_sync(0xffffffffu, row >= 0);
            if (j + 8 < x.n) ahead = page_of(x, group + 32);
          }
          if (t >= stages && !k7_wait(empty + stage * 8, (t / stages - 1) & 1u)) {
            k7_raise(p.status, TOME_DEV_TIMEOUT);
            ok = false;
            break;
          }
          __syncwarp();
          const uint32_t dst = area + stage * S::KV_BYTES;
          const int32_t key0 = (x.tile + j) * K7_KEYS;
          const int32_t in_batch = (j % 8) * (K7_KEYS / 16);
          const bool whole = (good >> in_batch & 0xfu) == 0xfu;
          if (whole) {
            if (by_hand >> stage & 1u) {  // ordinary writes before the tensor copies'
              fence_proxy_async();
              __syncwarp();
              by_hand &= ~(1u << stage);
            }
            int32_t rows[K7_KEYS / 16];
#pragma unroll
            for (int h = 0; h < K7_KEYS / 16; ++h) rows[h] = __shfl_sync(0xffffffffu, row, in_batch + h);
            if (lane == 0) {
              mbar_expect_tx(full + stage * 8, S::KV_BYTES);
              mbar_arrive_many(full + stage * 8, 32);
#pragma unroll
              for (int h = 0; h < K7_KEYS / 16; ++h) {
                if (h & (p.big_box - 1)) continue;
#pragma unroll
                for (int b = 0; b < D / 64; ++b)
                  tma_load_2d(dst + b * (K7_KEYS * 128) + h * 2048, map, b * 64, rows[h], full + stage * 8);
              }
            }
          } else {
            by_hand |= 1u << stage;
#pragma unroll 1
            for (int h = 0; h < K7_KEYS; h += 16) {
              const int32_t pool_row = k7_pool_row(p, x, pages, key0 + h, lane);
#pragma unroll 1
              for (int i = 0; i < STEPS; ++i) {
                const int r = i * AT_ONCE + sub;
                const int32_t from = __shfl_sync(0xffffffffu, pool_row, r);
                k7_copy16(dst + (c >> 3) * (K7_KEYS * 128) + (h + r) * 128 + (((c & 7) ^ (r & 7)) << 4),
                          pool + static_cast<int64_t>(max(from, 0)) * D, from >= 0);
              }
            }
            k7_copies_arrive(full + stage * 8);
          }
        }
        x = next;
        pages = next_pages;
        ahead = next_ahead;
        there = next_there;
        ++piece;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
    fence_proxy_async();  // the space is filled by tensor copies again
    tc_fence_before_sync();
    __syncthreads();
    if (warp == K7_ISSUE_WARP) {
      tc_fence_after_sync();
      tmem_dealloc(tmem, S::TMEM_COLS);
    }
  }

  if (warp == K7_WARPS - 1) {
    // For the joining kernel, dealt over the CTAs: where a row's pieces lie.
    for (int64_t i = blockIdx.x * 32 + lane; i < static_cast<int64_t>(p.n_seq) * p.heads; i += gridDim.x * 32) {
      const int32_t b = static_cast<int32_t>(i / p.heads), h = static_cast<int32_t>(i - static_cast<int64_t>(b) * p.heads);
      const int32_t kv = h / p.ratio, hr = h - kv * p.ratio;
      int4 where = make_int4(0, 0, 0, 0);
      if (p.n_groups > 0 && b >= pl.group[0] && b < pl.group[p.n_groups]) {
        const int g = k7_find(pl.group, p.n_groups, b);
        const int32_t len = k7_length(p, p.prefix_lens[g], p.prefix_blocks);
        const bool is_big = k7_is_big((pl.group[g + 1] - pl.group[g]) * p.ratio);
        const int32_t row = (b - pl.group[g]) * p.ratio + hr, mb = is_big ? row / K7_ROWS : 0, in_group = mb * p.kv_heads + kv;
        if (len > 0) {
          const int2 w = k7_holders(is_big ? big : small, pl.prefix[is_big][g] + in_group * k7_item_cost(len, is_big), len, is_big);
          const int32_t item = (is_big ? pl.block[g] : g) * p.kv_heads + in_group;
          where.x = static_cast<int32_t>(k7_out_row(p, true, is_big, item, w.x)) + (row - mb * K7_ROWS);
          where.y = is_big ? w.y : -w.y;
        }
        if (p.prefix_lens[g] > len) k7_raise(p.status, TOME_DEV_BLOCK_OUT_OF_RANGE);
      }
      const int32_t len = k7_length(p, p.lengths[b], p.seq_blocks);
      if (p.lengths[b] > len) k7_raise(p.status, TOME_DEV_BLOCK_OUT_OF_RANGE);
      if (len > 0) {
        const bool is_big = k7_is_big(p.ratio);
        const int2 w = k7_holders(is_big ? big : small,
                                  pl.prefix[is_big][p.n_groups] + pl.suffix[b] + kv * k7_item_cost(len, is_big), len, is_big);
        where.z = static_cast<int32_t>(k7_out_row(p, false, is_big, b * p.kv_heads + kv, w.x)) + hr;
        where.w = w.y;
      }
      p.plan[i] = where;
    }
  }
  // the first workers are spread over the CTAs
  const int32_t worker = warp * gridDim.x + blockIdx.x;
  if (worker < small.workers)
    k7_small_run<T, D>(p, &k_map_16, &v_map_16, pl, base + warp * (K7_SMALL_STAGES * S::SMALL_STAGE),
                       base + S::SMALL_FULL + warp * (K7_SMALL_STAGES * 8), worker, small.begin(worker),
                       small.begin(worker + 1), lane);
}

// ------------------------------------------------------------------ joining the pieces
// With maxima m_i, sums l_i and sums of p v o_i of a row's pieces: M = max m_i,
// out = sum 2^(m_i - M) o_i / sum 2^(m_i - M) l_i.  A row without a key is 0 with log-sum -inf.
// WARPS warps share a row's pieces.  Little but the latency of two loads: where the pieces are,
// then all of them at once.
constexpr int K7_JOIN_WARPS = 4;

template <typename T, int D, int WARPS>
__global__ void __launch_bounds__(K7_JOIN_WARPS * 32) k7_join_kernel(const K7Params p) {
  constexpr int E = D / 32;       // elements per lane
  constexpr int TOGETHER = 8;     // pieces whose loads are under way at a time
  __shared__ float part[WARPS][D];
  __shared__ float2 part_ml[WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t w = WARPS > 1 ? static_cast<int64_t>(blockIdx.x)
                              : static_cast<int64_t>(blockIdx.x) * K7_JOIN_WARPS + warp;
  griddep_wait();
  griddep_launch_dependents();
  if (w >= static_cast<int64_t>(p.n_seq) * p.heads) return;  // (never with WARPS > 1)
  const int4 where = p.plan[w];
  const int32_t n_prefix = abs(where.y), n = n_prefix + where.w;
  const int32_t prefix_step = where.y < 0 ? K7_SMALL_ROWS : K7_ROWS;
  float top = -INFINITY, total = 0.0f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.0f;
  // takes (m, l) and o of one more piece each; a sum of 0 is a piece that saw nothing but -inf, a
  // maximum of -inf with a sum is one of NaN scores
  auto take = [&](const float2 (&ml)[TOGETHER], const float (&v)[TOGETHER][E], int32_t count) {
    float m = top;
#pragma unroll
    for (int k = 0; k < TOGETHER; ++k)
      if (k < count && ml[k].y != 0.0f) m = fmaxf(m, ml[k].x);
    const float keep = top == -INFINITY ? (total == 0.0f ? 0.0f : 1.0f) : ex2f(top - m);
    top = m;
    total *= keep;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] *= keep;
#pragma unroll
    for (int k = 0; k < TOGETHER; ++k) {
      if (k >= count || ml[k].y == 0.0f) continue;
      const float f = ml[k].x == -INFINITY ? 1.0f : ex2f(ml[k].x - m);
      total = fmaf(f, ml[k].y, total);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = fmaf(f, v[k][e], acc[e]);
    }
  };
  for (int32_t base = WARPS > 1 ? warp * TOGETHER : 0; base < n; base += WARPS * TOGETHER) {
    float v[TOGETHER][E];
    float2 ml[TOGETHER];
#pragma unroll
    for (int k = 0; k < TOGETHER; ++k) {
      const int32_t i = min(base + k, n - 1);
      const int64_t row = i < n_prefix ? where.x + static_cast<int64_t>(i) * prefix_step
                                       : where.z + static_cast<int64_t>(i - n_prefix) * p.ratio;
      ml[k] = p.part_ml[row];
      const float* src = p.part_o + row * D + lane * E;
      if constexpr (E == 4) {
        const float4 x = *reinterpret_cast<const float4*>(src);
        v[k][0] = x.x; v[k][1] = x.y; v[k][2] = x.z; v[k][3] = x.w;
      } else {
        const float2 x = *reinterpret_cast<const float2*>(src);
        v[k][0] = x.x; v[k][1] = x.y;
      }
    }
    take(ml, v, n - base);
  }
  if constexpr (WARPS > 1) {
#pragma unroll
    for (int e = 0; e < E; ++e) part[warp][lane * E + e] = acc[e];
    if (lane == 0) part_ml[warp] = make_float2(top, total);
    __syncthreads();
    if (warp > 0) return;
    float v[TOGETHER][E];
    float2 ml[TOGETHER];
#pragma unroll
    for (int k = 1; k < WARPS; ++k) {
      ml[k - 1] = part_ml[k];
#pragma unroll
      for (int e = 0; e < E; ++e) v[k - 1][e] = part[k][lane * E + e];
    }
    take(ml, v, WARPS - 1);
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
  int64_t small_rows, suffix_rows, rows;
  size_t plan, part_o, part_ml, total;
};

static size_t k7_up(size_t n) { return (n + 255) / 256 * 256; }

static K7Layout k7_layout(int64_t n_seq, int64_t n_groups, int64_t heads, int64_t kv_heads, int64_t dim) {
  const int64_t ratio = heads / kv_heads;
  // row blocks of all groups: each group rounds up once
  const int64_t blocks = n_groups == 0 ? 0 : n_groups + n_seq * ratio / K7_ROWS;
  K7Layout l;
  l.small_rows = n_groups == 0 ? 0 : (blocks * kv_heads + K7_MAX_CTAS) * K7_ROWS;
  l.suffix_rows = l.small_rows + (n_groups == 0 ? 0 : (n_groups * kv_heads + K7_MAX_WORKERS) * K7_SMALL_ROWS);
  l.rows = l.suffix_rows + (n_seq * kv_heads + (ratio > K7_SMALL_ROWS ? K7_MAX_CTAS : K7_MAX_WORKERS)) * ratio;
  l.plan = 0;
  l.part_o = k7_up(static_cast<size_t>(16 * n_seq * heads));
  l.part_ml = l.part_o + k7_up(static_cast<size_t>(l.rows * dim * 4));
  l.total = l.part_ml + k7_up(static_cast<size_t>(l.rows * 8));
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
  void (*kernel)(CUtensorMap, CUtensorMap, CUtensorMap, CUtensorMap, K7Params) = k7_attention_kernel<T, D>;
  const int bytes = S::PLAN + S::plan_bytes(p.n_groups, p.n_seq) + 1024;
  // set once for the largest plan, so that no later call has to raise it
  const int most = S::PLAN + S::plan_bytes(K7_MAX_GROUPS, K7_MAX_SEQ) + 1024;
  static_assert(S::PLAN + S::plan_bytes(K7_MAX_GROUPS, K7_MAX_SEQ) + 1024 <= 232448, "shared memory");
  int32_t st = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), most);
  if (st != TOME_OK) return st;
  // the pools as matrices of 64-column blocks, for small tiles sixteen rows at a time, for big ones as
  // many as divide a page
  CUtensorMap k_map = {}, v_map = {}, k_map_16 = {}, v_map_16 = {};
  if (p.whole_pages) {
    const int64_t rows = static_cast<int64_t>(p.num_blocks) * p.kv_heads * p.block_size;
    st = tensor_map_16bit(&k_map_16, p.k_pool, rows, D, 16);
    if (st == TOME_OK) st = tensor_map_16bit(&v_map_16, p.v_pool, rows, D, 16);
    k_map = k_map_16;
    v_map = v_map_16;
    if (p.big_box > 1 && st == TOME_OK) st = tensor_map_16bit(&k_map, p.k_pool, rows, D, 16 * p.big_box);
    if (p.big_box > 1 && st == TOME_OK) st = tensor_map_16bit(&v_map, p.v_pool, rows, D, 16 * p.big_box);
    if (st != TOME_OK) return st;
  }
  cudaLaunchAttribute attr;  // each kernel is set up while the one before it drains
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.ctas));
  cfg.blockDim = dim3(K7_THREADS);
  cfg.dynamicSmemBytes = static_cast<size_t>(bytes);
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  st = check_cuda(cudaLaunchKernelEx(&cfg, kernel, k_map, v_map, k_map_16, v_map_16, p), "prefix attention launch");
  if (st != TOME_OK) return st;
  // Few rows have many pieces each: a block of warps per row then, else a warp.
  const int64_t rows = static_cast<int64_t>(p.n_seq) * p.heads;
  const bool few = rows <= K7_MAX_CTAS * 8;
  cfg.gridDim = dim3(static_cast<unsigned>(few ? rows : (rows + K7_JOIN_WARPS - 1) / K7_JOIN_WARPS));
  cfg.blockDim = dim3(K7_JOIN_WARPS * 32);
  cfg.dynamicSmemBytes = 0;
  void (*join)(K7Params) = few ? k7_join_kernel<T, D, K7_JOIN_WARPS> : k7_join_kernel<T, D, 1>;
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
  // places and rows of the workspace are counted in 32 bits
  const int64_t ratio = heads / kv_heads;
  const int64_t prefix_keys = static_cast<int64_t>(prefix_blocks) * block_size;
  const int64_t seq_keys = static_cast<int64_t>(max_blocks) * block_size;
  const int64_t row_blocks = n_groups == 0 ? 0 : n_groups + n_seq * ratio / K7_ROWS;
  auto most = [&](int64_t keys) { return K7_SMALL_ITEM_COST + (keys + K7_SMALL_KEYS - 1) / K7_SMALL_KEYS; };
  if (l.rows > 0x7fffffff) return fail(TOME_ERR_TOO_LARGE, "too many rows for one call");
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
  auto divisor = [](int32_t d, uint32_t* magic, int32_t* shift) {
    int s = 0;
    while ((1ll << s) < d) ++s;
    *shift = 31 + s;
    *magic = static_cast<uint32_t>((1ull << (31 + s)) / static_cast<uint64_t>(d) + 1);
  };
  divisor(block_size, &p.div_magic, &p.div_shift);
  divisor(p.ratio, &p.ratio_magic, &p.ratio_shift);
  p.c = scale * LOG2E;
  p.whole_pages = block_size % 16 == 0 && num_blocks > 0;
  p.big_box = block_size % 64 == 0 ? 4 : (block_size % 32 == 0 ? 2 : 1);
  p.ctas = std::max(1, std::min(info.sm_count, K7_MAX_CTAS));
  p.inv_ctas = 1.0 / p.ctas;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.plan = reinterpret_cast<int4*>(ws + l.plan);
  p.part_o = reinterpret_cast<float*>(ws + l.part_o);
  p.part_ml = reinterpret_cast<float2*>(ws + l.part_ml);
  p.small_rows = l.small_rows;
  p.suffix_rows = l.suffix_rows;
  p.out = out;
  p.out_lse = out_lse;
  p.status = dev_status;
  const cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if (dtype == TOME_BF16)
    return head_dim == 64 ? k7_launch<__nv_bfloat16, 64>(p, cs) : k7_launch<__nv_bfloat16, 128>(p, cs);
  return head_dim == 64 ? k7_launch<__half, 64>(p, cs) : k7_launch<__half, 128>(p, cs);
}

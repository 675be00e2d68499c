// Attention of a step's tokens - one, a chunk of a prompt, a tree of drafts - over a paged
// key/value cache.
//
//   out = sum_p softmax_p(scale q . k_p) v_p   over the cache_lens[b] tokens that were there and
//   the step's tokens that tree_mask (or causal order) lets the query see.
//
// The T * group query rows that share a key/value head are one (128-row) tensor-core tile,
// padded: with at most that many rows the step is bound by reading K and V once from HBM, and
// the padding costs nothing that the memory does not wait for (a key tile of 64 KB takes an SM
// about 2800 cycles to receive, its two 128 x 128 x 128 products 1024).
//
// Work is split by key tiles, not by sequences: the key tiles of all (sequence, head, row tile)
// items laid end to end are cut into equal ranges, one per CTA, from the lengths in device
// memory.  A CTA walks its range; an item that lies in one range is finished there, the others
// leave partial softmax states (row maximum, sum, accumulator) that a second kernel joins in
// range order.  The split is a function of the lengths alone, so results do not depend on
// timing.
//
// One CTA per SM, two softmax groups A and B whose work interleaves on the tensor cores, so that
// one's softmax overlaps the other's matrix products:
//   split  (at most 128 rows)   A and B take the CTA's key tiles in turn, each with its own running
//                               maximum, sum and O; the group of a run's last tile joins the two
//                               states at its end, while the other already works on the next
//                               run's first tile, whose S was issued before (Q has two places)
//   quad   (at most 16 rows,    split, with the rows four times in the tile: warp q of a group takes
//          many items: see      keys [32 q, 32 q + 32) of every tile, its P is zero elsewhere, and
//          lay_out_rows)        its rows are a partial state of their own.  A warp's 128
//                               exponentials, 1000 cycles of the special-function unit whether
//                               one lane has a row or all, become 32, on four schedulers
//   pair   (more rows)          A and B are two row tiles of 128, every key tile serves both
//
//   warps 0, 10  TMA producers of K and of V: a box per run of slots inside a page, into rings
//   warp 11      TMA producer of Q: a box of group heads x tokens is a row tile, token by token
//   warp 1       MMA issuer: S_x = Q K^T, O_x += P_x V (P from tensor memory)
//   warps 2..5   softmax group A, warps 6..9 group B: a query row per thread
//
// What a run does once (masks, values that are not finite) is kept in
// rolled loops: unrolled, the kernel was 180 KB of code, more than the instruction cache.
//
// Measured (bf16, heads of 128, 32 on 8): 32 sequences of 2048 - 8192 keys, a token each, 115 - 119 us =
// 5.7 - 5.9 TB/s, 0.87 - 0.89 of a copy (quad; a tile of 64 KB every 2230 cycles); 8 x 16 drafts of the
// same lengths 44 us = 3.9 TB/s, where the first copies, the last softmax and the join are a third; 4 x 64 drafts of 8192 -
// 32768 keys 124 us: 2.0 - 2.2 us for a tile of 256 rows (pair), bound by the chain S, softmax, P V of a row
// tile.  One token of 32 heads and 1024 keys (fp16) 13.0 us: launch, lengths -> pages -> K, join.
//
// Slots behind a sequence's last token may hold anything: their scores are masked by index and
// their rows of V are cleared in shared memory, since 0 * NaN is not 0.  Values of the step's own tokens
// that are not finite are cleared too, and added to the rows that see them.  A row that sees no key is
// zero; NaN in a query, or in a key that the row sees, makes it NaN, whoever finishes or joins it.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cfloat>

#include "common.cuh"
#include "host.h"
#include "softmax.cuh"

namespace b200k {
namespace {

constexpr int kPaBM = 128;             // query rows of a tile
constexpr int kPaBN = 128;             // keys of a tile
constexpr int kPaThreads = 384;        // K warp, MMA warp, two softmax groups of four warps, V and Q warps
constexpr int kPaQuadRows = 16;        // rows up to which quad is taken
constexpr int kPaMaxBatch = 65535;     // every warp that looks for its place reads all lengths
constexpr int kPaTmemCols = 512;       // S_A, S_B, O_A, O_B; P over S

// Rings of K and V tiles in what Q's two tiles leave of 224 KB.  V tiles wait for the softmax, so V
// gets the odd one.
enum Mode : int { kSplit = 0, kPair = 1, kQuad = 2 };

template <int D> struct Rings {
  static constexpr int kTile = 128 * D * 2;
  static constexpr int kQ = 2;                        // two runs' rows (split), two halves (pair)
  static constexpr int kTiles = 224 * 1024 / kTile - kQ;
  static constexpr int kK = kTiles / 2, kV = kTiles - kK;
  static constexpr int kSmem = (kQ + kTiles) * kTile + 1472 + 8 * 2 * 13 * 4;
};

struct PagedParams {
  const uint16_t* q;
  const uint16_t* v;                   // as plain memory: the rare path of values that are not finite
  uint16_t* out;
  const int* page_table;
  const int* cache_lens;
  const int* new_lens;
  const uint8_t* mask;
  int64_t o_b, o_h, o_t, vc_p, vc_h, vc_s, mask_b, mask_t, mask_j;
  int64_t page_table_stride, num_pages;
  int batch, tokens, heads_kv, group, dim;
  int row_tiles, half_tokens;          // row tiles; tokens of a 128-row half: half_tokens * group <= 128 rows
  int tile_rows;                       // rows of a tile's partial state
  int page_size, max_pages, box_rows;
  int page_shift;                      // log2 of the page size, -1 where it is no power of two
  int ctas;
  int join_blocks;                     // blocks of the joining kernel for an item
  int o_vec;                           // rows of out on 16-byte boundaries
  int zero_padding;
  float scale_log2;
  float* ws_ml;                        // (slots, tile_rows, 2): row maximum and sum
  float* ws_acc;                       // (slots, D / 4, tile_rows, 4): two slots per CTA (quad: and one per item)
  int* status;
};

// Lengths of a sequence, kept inside what its page table can name (at most 2^29 tokens: every count
// of tokens and of key tiles fits 32 bits).
struct SeqInfo {
  int have, fresh, len, tiles;         // tokens before the step, of the step, their sum, key tiles
};
__device__ __forceinline__ SeqInfo seq_info(const PagedParams& p, int b) {
  SeqInfo s;
  const int cap = p.max_pages * p.page_size;
  s.fresh = p.new_lens != nullptr ? max(0, min(p.new_lens[b], p.tokens)) : p.tokens;
  s.have = max(0, min(p.cache_lens[b], cap));
  s.len = s.fresh == 0 ? 0 : min(s.have + s.fresh, cap);
  s.tiles = (s.len + kPaBN - 1) / kPaBN;
  return s;
}
__device__ __forceinline__ bool lengths_fit(const PagedParams& p, int b) {
  const int fresh = p.new_lens != nullptr ? max(0, min(p.new_lens[b], p.tokens)) : p.tokens;
  const int have = p.cache_lens[b];
  return fresh == 0 || (have >= 0 && have <= p.max_pages * p.page_size - fresh);
}

__device__ __forceinline__ int warp_sum(int v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// `total` tiles in `ctas` ranges, the first total % ctas of them one tile longer: first tile of
// range c, and the range that holds tile x.
struct Ranges {
  int base, longer;
  __device__ __forceinline__ Ranges(int total, int ctas) : base(total / ctas), longer(total % ctas) {}
  __device__ __forceinline__ int begin(int c) const { return c * base + min(c, longer); }
  __device__ __forceinline__ int owner(int x) const {
    const int in_longer = longer * (base + 1);
    return x < in_longer ? x / (base + 1) : longer + (x - in_longer) / base;
  }
};

// A CTA's walk over its range: runs of key tiles of one item.
struct Walk {
  int left;                            // tiles still to come
  int b, item, tile;                   // sequence; head * row_tiles + row tile; first key tile
};
struct Run {
  SeqInfo seq;
  int b, head, row_tile, first, last;  // key tiles [first, last)
};
// The run at the walk's place, whose sequence r.seq is, and the walk behind it.
__device__ __forceinline__ void take_run(const PagedParams& p, Walk& w, Run& r) {
  r.b = w.b;
  r.head = p.row_tiles == 1 ? w.item : w.item / p.row_tiles;
  r.row_tile = w.item - r.head * p.row_tiles;
  r.first = w.tile;
  r.last = min(r.seq.tiles, w.tile + w.left);
  w.left -= r.last - r.first;
  w.tile = 0;
  if (++w.item == p.heads_kv * p.row_tiles) {
    w.item = 0;
    ++w.b;
  }
}
__device__ __forceinline__ bool next_run(const PagedParams& p, Walk& w, Run& r) {
  if (w.left <= 0) return false;
  do {                                 // sequences without tokens have no tiles
    if (w.b >= p.batch) return false;
    r.seq = seq_info(p, w.b);
  } while (r.seq.tiles == 0 && ++w.b > 0);
  take_run(p, w, r);
  return true;
}

// This CTA's range and its first run, warp-collective; false where it has none.  Up to 32 sequences
// their lengths are read once (every further trip to the L2 costs 700 cycles before the first copy).
__device__ __forceinline__ bool first_run(const PagedParams& p, int lane, Walk& w, Run& r) {
  const int per_seq = p.heads_kv * p.row_tiles;
  SeqInfo seq = {0, 0, 0, 0};
  if (lane < p.batch) seq = seq_info(p, lane);
  int all = seq.tiles;
#pragma unroll 1
  for (int b = lane + 32; b < p.batch; b += 32) all += seq_info(p, b).tiles;
  const Ranges ranges(warp_sum(all) * per_seq, p.ctas);
  const int begin = ranges.begin(blockIdx.x);
  w.left = ranges.begin(blockIdx.x + 1) - begin;
  if (w.left <= 0) return false;
  int before = 0;
#pragma unroll 1
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    if (b0 > 0) {
      seq = {0, 0, 0, 0};
      if (b0 + lane < p.batch) seq = seq_info(p, b0 + lane);
    }
    const int mine = seq.tiles * per_seq;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const uint32_t here = __ballot_sync(0xffffffffu, begin >= before + upto - mine && begin < before + upto);
    if (here != 0) {
      const int from = __ffs(here) - 1;
      r.seq.have = __shfl_sync(0xffffffffu, seq.have, from);
      r.seq.fresh = __shfl_sync(0xffffffffu, seq.fresh, from);
      r.seq.len = __shfl_sync(0xffffffffu, seq.len, from);
      r.seq.tiles = __shfl_sync(0xffffffffu, seq.tiles, from);
      const int in_seq = begin - before - __shfl_sync(0xffffffffu, upto - mine, from);
      w.b = b0 + from;
      w.item = in_seq / r.seq.tiles;
      w.tile = in_seq - w.item * r.seq.tiles;
      take_run(p, w, r);
      return true;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  return false;
}

// A softmax warp's walk and run, in shared memory: what a run needs at its two ends only would
// otherwise be spilled to local memory, whose lines the 20 KB of L1 beside the tiles do not hold.
constexpr int kRunWords = 13;
__device__ __forceinline__ void save_run(volatile int* w, const Walk& k, const Run& r) {
  w[0] = k.left; w[1] = k.b; w[2] = k.item; w[3] = k.tile;
  w[4] = r.seq.have; w[5] = r.seq.fresh; w[6] = r.seq.len; w[7] = r.seq.tiles;
  w[8] = r.b; w[9] = r.head; w[10] = r.row_tile; w[11] = r.first; w[12] = r.last;
}
__device__ __forceinline__ Walk saved_walk(volatile int* w) {
  Walk k;
  k.left = w[0]; k.b = w[1]; k.item = w[2]; k.tile = w[3];
  return k;
}
__device__ __forceinline__ Run saved_run(volatile int* w) {
  Run r;
  r.seq.have = w[4]; r.seq.fresh = w[5]; r.seq.len = w[6]; r.seq.tiles = w[7];
  r.b = w[8]; r.head = w[9]; r.row_tile = w[10]; r.first = w[11]; r.last = w[12];
  return r;
}

// 1 / l of a row: 0 where it saw no key (the maximum is -inf).  A sum of 0 over keys that it saw, whose
// scores are all -inf, is the softmax's 0 / 0; a sum that is NaN stays NaN.
__device__ __forceinline__ float softmax_factor(float m, float l) {
  if (l > 0.0f) return __fdividef(1.0f, l);
  return m == -INFINITY ? l : __int_as_float(0x7fc00000);
}

// Ones in the halves of a word whose 16-bit floats are finite.
template <bool BF16>
__device__ __forceinline__ uint32_t finite_halves(uint32_t w) {
  const uint32_t e = BF16 ? 0x7f80u : 0x7c00u;
  return ((w & e) == e ? 0u : 0xffffu) | (((w >> 16) & e) == e ? 0u : 0xffff0000u);
}
template <bool BF16>
__device__ __forceinline__ float half_to_float(uint16_t h) {
  if constexpr (BF16) return __uint_as_float(static_cast<uint32_t>(h) << 16);
  else return __half2float(*reinterpret_cast<const __half*>(&h));
}

// Which of the keys [k0, k0 + 32) a row sees, as bits, warp-collective: lane i fetches key i's entry
// for one token of the warp's rows after the other (neighbouring bytes, eight tokens on their
// way at once), and a vote makes the word.  `t` is the lane's own token, [t0, t1] the warp's.
__device__ __forceinline__ uint32_t visible_keys(const PagedParams& p, const SeqInfo& seq, int b, int t, int t0, int t1,
                                                 int k0, int lane) {
  const int old = seq.have - k0;              // tokens from before the step
  if (old >= 32) return 0xffffffffu;
  if (k0 >= seq.len) return 0u;
  if (p.mask == nullptr) {                    // drafts up to t
    const int n = min(t, seq.fresh - 1) + 1 + old;
    return n >= 32 ? 0xffffffffu : (n > 0 ? (1u << n) - 1u : 0u);
  }
  uint32_t bits = old > 0 ? (1u << old) - 1u : 0u;
  const int draft = lane - old;
  const bool in = draft >= 0 && draft < seq.fresh && k0 + lane < seq.len;
  const uint8_t* at = p.mask + b * p.mask_b + t0 * p.mask_t + (in ? draft * p.mask_j : 0);
#pragma unroll 1
  for (int tt = t0; tt <= t1; tt += 8) {
    uint8_t v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = in && tt + u <= t1 ? at[u * p.mask_t] : 0;
    at += 8 * p.mask_t;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const uint32_t vote = __ballot_sync(0xffffffffu, v[u] != 0);
      if (t == tt + u) bits |= vote;
    }
  }
  return bits;
}

// Adds to a row that has been written, to out (`whole`) or as a partial state (column k at
// acc[k / 4][.][k % 4]), the values that are not finite in the V of the step's tokens that token t
// sees, among keys [from, to): they were taken out of the tile, and any weight leaves them what they
// are.  `quarter` (quad): only the keys of that quarter of a tile, -1: all.
template <bool BF16>
__device__ __forceinline__ void add_not_finite(const PagedParams& p, const Run& run, int t, int quarter, bool whole,
                                               uint16_t* o_row, float* acc) {
  const int from = max(run.seq.have, run.first * kPaBN);
  int to = min(run.seq.len, run.last * kPaBN);
  if (p.mask == nullptr) to = min(to, run.seq.have + t + 1);
  const uint8_t* mask = p.mask + run.b * p.mask_b + t * p.mask_t;
  const int* pages = p.page_table + run.b * p.page_table_stride;
#pragma unroll 1
  for (int c0 = 0; c0 < p.dim; c0 += 8) {
    const uint16_t* v = p.v + run.head * p.vc_h + c0;
    float sum[8] = {};
    bool all_nan = false;
    // four slots of a page on their way at once
#pragma unroll 1
    for (int k0 = from & ~3; k0 < to && !all_nan; k0 += 4) {
      if (quarter >= 0 && ((k0 >> 5) & 3) != quarter) continue;
      const int entry = k0 / p.page_size, page = pages[entry];
      if (page < 0 || page >= p.num_pages) continue;
      const uint16_t* at = v + page * p.vc_p + (k0 - entry * p.page_size) * p.vc_s;
      uint4 rows[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int key = k0 + u;
        const bool sees = key >= from && key < to && (p.mask == nullptr || mask[(key - run.seq.have) * p.mask_j] != 0);
        rows[u] = sees ? *reinterpret_cast<const uint4*>(at + u * p.vc_s) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint32_t w[4] = {rows[u].x, rows[u].y, rows[u].z, rows[u].w};
        uint32_t bad[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) bad[i] = w[i] & ~finite_halves<BF16>(w[i]);
        if ((bad[0] | bad[1] | bad[2] | bad[3]) == 0u) continue;
        all_nan = true;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sum[2 * i] += half_to_float<BF16>(static_cast<uint16_t>(bad[i] & 0xffffu));
          sum[2 * i + 1] += half_to_float<BF16>(static_cast<uint16_t>(bad[i] >> 16));
          all_nan = all_nan && sum[2 * i] != sum[2 * i] && sum[2 * i + 1] != sum[2 * i + 1];
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (sum[e] == 0.f) continue;
      if (whole) {
        const float y = half_to_float<BF16>(o_row[c0 + e]) + sum[e];
        if constexpr (BF16) reinterpret_cast<__nv_bfloat16*>(o_row)[c0 + e] = __float2bfloat16_rn(y);
        else reinterpret_cast<__half*>(o_row)[c0 + e] = __float2half_rn(y);
      } else {
        acc[static_cast<int64_t>((c0 + e) / 4) * p.tile_rows * 4 + (c0 + e) % 4] += sum[e];
      }
    }
  }
}

template <int D, bool BF16, int MODE>
__global__ void __launch_bounds__(kPaThreads, 1)
paged_attention_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                       const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ PagedParams p) {
  constexpr bool PAIR = MODE == kPair, QUAD = MODE == kQuad;
  using R = Rings<D>;
  constexpr int kBoxes = D / 64;            // 64-element (128-byte) slices of the head dim
  constexpr int kBoxBytes = 128 * 128;
  // no room for rounding the base up: the swizzle atoms need the declared alignment
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {
    report_status(p.status, 89, 0);
    return;
  }
  const uint32_t q_smem = smem_u32(smem);
  const uint32_t k_smem = q_smem + R::kQ * R::kTile;
  const uint32_t v_smem = k_smem + R::kK * R::kTile;
  uint8_t* tail = smem + (R::kQ + R::kTiles) * R::kTile;
  const uint32_t bar0 = smem_u32(tail);
  enum { Q_FULL = 0, Q_EMPTY = Q_FULL + 2, S_FULL = Q_EMPTY + 2, P_HALF = S_FULL + 2, P_FULL = P_HALF + 2, PV_DONE = P_FULL + 2,
         RUN_DONE = PV_DONE + 2, O_READ, K_FULL, K_EMPTY = K_FULL + R::kK, V_FULL = K_EMPTY + R::kK,
         V_EMPTY = V_FULL + R::kV, NUM_BARS = V_EMPTY + R::kV };
  static_assert(8 * NUM_BARS <= 384, "barriers fit their place");
  auto bar = [&](int i) { return bar0 + 8u * i; };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail + 384);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 392);
  volatile int* bad_draft = reinterpret_cast<volatile int*>(tail + 400);   // [2], by run parity
  float2* state_b = reinterpret_cast<float2*>(tail + 448);                 // [128] maximum and sum of the other group's rows
  volatile int* run_words = reinterpret_cast<volatile int*>(tail + 1472);  // [8 softmax warps][2][kRunWords]

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < NUM_BARS; ++i) {
      int count = 1;
      if (i >= P_HALF && i < PV_DONE) count = 4;
      if (i == RUN_DONE) count = 8;
      if (i == O_READ) count = 4;
      mbar_init(bar(i), count);
    }
    *abort_flag = 0;
    bad_draft[0] = bad_draft[1] = -1;
    fence_barrier_init();
    tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  if (warp == 0 && lane < 2) {
    // the page table and the queries are asked for only after the lengths have come: their address
    // translations start now
    const void* early = lane == 0 ? static_cast<const void*>(p.page_table) : static_cast<const void*>(p.q);
    asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<uint64_t>(early)));
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), kPaTmemCols);
    tmem_relinquish();
  }
  // what the kernel before this one in the stream writes is read from here on
  pdl_wait();
  // The joining kernel may be set up now.  Not earlier: it reads the lengths before it waits for this
  // grid, and a kernel that writes them may have let its own successor start before its end.
  pdl_launch_dependents();
  // where this CTA begins, and its first pages: every warp finds its own, without a wait for
  // another's
  Walk walk;
  Run run;
  bool have_run = first_run(p, lane, walk, run);
  // the K and V producers' lane i looks up the i-th run of slots of a tile, all of one page
  const int boxes_per_tile = kPaBN / p.box_rows;
  auto find = [&](int j, int& page, int& slot) {
    const int key = j * kPaBN + lane * p.box_rows;
    page = slot = 0;
    if (lane < boxes_per_tile && key < run.seq.len) {
      const int entry = p.page_shift >= 0 ? key >> p.page_shift : key / p.page_size;
      slot = key - entry * p.page_size;
      page = p.page_table[run.b * p.page_table_stride + entry];
    }
  };
  int page = 0, slot = 0;
  if (have_run && (warp == 0 || warp == 10)) find(run.first, page, slot);
  if (blockIdx.x == 0 && warp == 2) {
#pragma unroll 1
    for (int b = lane; b < p.batch; b += 32)
      if (!lengths_fit(p, b)) report_bad_index(p.status, kRolePage, b);
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  constexpr uint32_t kFmt = BF16 ? kFmtBF16 : kFmtF16;

  if (warp == 11) {
    // the Q producer: a run's rows once their place's last S is through.  Pair has one place: the
    // next run's rows are prefetched into the L2 (cold, they took 10 us of a full memory system)
    Run next;
    bool ok = true;
    const bool elected = elect_one();
    constexpr int kHalves = PAIR ? 2 : 1, kCopies = QUAD ? 4 : 1;
    const uint32_t bytes = static_cast<uint32_t>(p.half_tokens * p.group) * 128u * kBoxes * kHalves * kCopies;
    int runs = 0;
    for (; have_run && ok; ++runs) {
      // split: run r in place r % 2, once run r - 2 is through
      const int place = PAIR ? 0 : runs & 1, fill = PAIR ? runs : runs >> 1;
      if (fill > 0 && !mbar_wait(bar(Q_EMPTY + place), (fill - 1) & 1, abort_flag)) {
        report_status(p.status, 98, runs);
        *abort_flag = 1;
        ok = false;
        break;
      }
      if (elected) mbar_arrive_expect_tx(bar(Q_FULL + place), bytes);
      const bool more = next_run(p, walk, next);
#pragma unroll
      for (int x = 0; x < kHalves; ++x) {
#pragma unroll
        for (int h = 0; h < kBoxes; ++h) {
          if (elected) {
#pragma unroll
            for (int copy = 0; copy < kCopies; ++copy)
              tma_load_4d(q_smem + (place + x) * R::kTile + h * kBoxBytes + copy * 32 * 128, &tmap_q, bar(Q_FULL + place),
                          h * 64, run.head * p.group, (run.row_tile * kHalves + x) * p.half_tokens, run.b);
            if (PAIR && more)
              tma_prefetch_4d(&tmap_q, h * 64, next.head * p.group, (next.row_tile * kHalves + x) * p.half_tokens, next.b);
          }
        }
      }
      __syncwarp();
      run = next;
      have_run = more;
    }
    // nothing in flight when the CTA leaves
    for (int i = 0; i < (PAIR ? 1 : 2) && i < runs; ++i)
      mbar_wait(bar(Q_FULL + i), (PAIR ? runs - 1 : (runs - 1 - i) >> 1) & 1, abort_flag);
    __syncwarp();
  } else if (warp == 0 || warp == 10) {
    const bool is_v = warp != 0;
    const CUtensorMap* tmap = is_v ? &tmap_v : &tmap_k;
    const int full = is_v ? V_FULL : K_FULL, empty = is_v ? V_EMPTY : K_EMPTY, places = is_v ? R::kV : R::kK;
    const uint32_t ring = is_v ? v_smem : k_smem;
    const uint32_t box_bytes = p.box_rows * 128u;
    const bool elected = elect_one();
    bool ok = true;
    int place = 0, fills = 0;
    uint32_t parity = 1;                       // a fresh ring is empty
    for (int runs = 0; have_run && ok; ++runs) {
      if (runs > 0) find(run.first, page, slot);
      for (int j = run.first; j < run.last; ++j) {
        int next_page = 0, next_slot = 0;
        if (j + 1 < run.last) find(j + 1, next_page, next_slot);   // on its way while this tile is issued
        const int boxes = min(boxes_per_tile, (run.seq.len - j * kPaBN + p.box_rows - 1) / p.box_rows);
        if (lane < boxes && (page < 0 || page >= p.num_pages)) {
          report_bad_index(p.status, kRolePage, run.b);
          page = static_cast<int>(p.num_pages);   // behind the last page: filled with zeros
        }
        if (!mbar_wait(bar(empty + place), parity, abort_flag)) {
          report_status(p.status, is_v ? 91 : 90, j);
          *abort_flag = 1;
          ok = false;
          break;
        }
        const uint32_t dst = ring + place * R::kTile, done = bar(full + place);
        if (elected) mbar_arrive_expect_tx(done, static_cast<uint32_t>(boxes) * box_bytes * kBoxes);
        // warp-uniform coordinates: one elected lane issues box after box (lanes with coordinates
        // of their own cost three times as much per box)
#pragma unroll 1
        for (int i = 0; i < boxes; ++i) {
          const int pg = __shfl_sync(0xffffffffu, page, i), sl = __shfl_sync(0xffffffffu, slot, i);
          if (elected) {
#pragma unroll
            for (int h = 0; h < kBoxes; ++h)
              tma_load_4d(dst + h * kBoxBytes + i * box_bytes, tmap, done, h * 64, sl, run.head, pg);
          }
        }
        __syncwarp();
        ++fills;
        if (++place == places) { place = 0; parity ^= 1; }
        page = next_page;
        slot = next_slot;
      }
      have_run = next_run(p, walk, run);
    }
    // no copy of this warp is in flight when the CTA leaves (bounded, also after a failure): the
    // last fill of every ring place
    for (int i = 0; i < places && i < fills; ++i)
      mbar_wait(bar(full + i), ((fills - 1 - i) / places) & 1, abort_flag);
    __syncwarp();
  } else if (warp == 1) {
    const bool elected = elect_one();
    constexpr uint32_t idesc_qk = make_idesc(kFmt, kFmt, false, false, kPaBM, kPaBN);
    constexpr uint32_t idesc_pv = make_idesc(kFmt, kFmt, false, true, kPaBM, D);
    int ks = 0, vs = 0;
    uint32_t kp = 0, vp = 0, pp[2] = {0, 0};   // ring places and parities; parity of the groups' P
    bool ok = true;
    auto give_up = [&](int role, int detail) {
      report_status(p.status, role, detail);
      *abort_flag = 1;
      ok = false;
    };
    // S_x = Q_x K^T: both operands K-major, 16 elements (32 bytes) of the head dim per MMA
    auto issue_s = [&](int x, int q_place) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint32_t off = (kk / 4) * kBoxBytes;
        const uint64_t qd = make_smem_desc(q_smem + q_place * R::kTile + off, 16, 1024, kSwizzle128B) + 2 * (kk % 4);
        const uint64_t kd = make_smem_desc(k_smem + ks * R::kTile + off, 16, 1024, kSwizzle128B) + 2 * (kk % 4);
        if (elected) umma<kKindF16>(tmem_base + x * 128, qd, kd, idesc_qk, kk > 0 ? 1u : 0u);
      }
      if (elected) tc_commit(bar(S_FULL + x));
    };
    auto free_k = [&]() {
      if (elected) tc_commit(bar(K_EMPTY + ks));
      if (++ks == R::kK) { ks = 0; kp ^= 1; }
    };
    // O_x += P_x V in two halves of 64 keys: P from tensor memory, V (keys, D) with D contiguous
    auto issue_pv = [&](int x, bool first, int j) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (!mbar_wait(bar((half == 0 ? P_HALF : P_FULL) + x), pp[x], abort_flag)) {
          give_up(94, j);
          return;
        }
        tc_fence_after_sync();
#pragma unroll
        for (int k4 = 0; k4 < kPaBN / 32; ++k4) {
          const int kk = half * (kPaBN / 32) + k4;
          const uint64_t vd = make_smem_desc(v_smem + vs * R::kTile + kk * 2048, kBoxBytes, 1024, kSwizzle128B);
          if (elected)
            umma_f16_ts(tmem_base + 256 + x * 128, tmem_base + x * 128 + kk * 8, vd, idesc_pv, (!first || kk > 0) ? 1u : 0u);
        }
      }
      pp[x] ^= 1;
      if (elected) tc_commit(bar(PV_DONE + x));
    };
    auto free_v = [&]() {
      if (elected) tc_commit(bar(V_EMPTY + vs));
      if (++vs == R::kV) { vs = 0; vp ^= 1; }
    };
    if constexpr (PAIR) {
      for (int runs = 0; ok && have_run; ++runs, have_run = next_run(p, walk, run)) {
        const int n = run.last - run.first;
        if (!mbar_wait(bar(Q_FULL), runs & 1, abort_flag) || !mbar_wait(bar(K_FULL + ks), kp, abort_flag)) {
          give_up(92, runs);
          break;
        }
        tc_fence_after_sync();
        issue_s(0, 0);
        issue_s(1, 1);
        free_k();
        if (n == 1 && elected) tc_commit(bar(Q_EMPTY));
        for (int i = 0; i < n && ok; ++i) {
          // P V (A, i)  S (A, i + 1)  P V (B, i)  S (B, i + 1)
          const bool more = i + 1 < n;
          if (!mbar_wait(bar(V_FULL + vs), vp, abort_flag) || (more && !mbar_wait(bar(K_FULL + ks), kp, abort_flag))) {
            give_up(93, i);
            break;
          }
          tc_fence_after_sync();
          issue_pv(0, i == 0, i);
          if (ok && more) issue_s(0, 0);
          if (ok) issue_pv(1, i == 0, i);
          if (ok && more) {
            issue_s(1, 1);
            free_k();
            if (i + 1 == n - 1 && elected) tc_commit(bar(Q_EMPTY));
          }
          if (ok) free_v();
        }
      }
    } else {
      // tiles in the order of the CTA's range, group tile % 2; S two tiles ahead of P V, across runs
      int i = 0, runs = 0, issued = 0;
      bool first[2] = {true, true};            // the group's next P V is its first of a run
      Run next;
      bool have_next = false;
      auto next_s = [&]() {
        if (!have_run) return;
        const int x = issued & 1, n = run.last - run.first;
        if ((i == 0 && !mbar_wait(bar(Q_FULL + (runs & 1)), (runs >> 1) & 1, abort_flag)) ||
            !mbar_wait(bar(K_FULL + ks), kp, abort_flag)) {
          give_up(93, issued);
          return;
        }
        tc_fence_after_sync();
        issue_s(x, runs & 1);
        free_k();
        first[x] = i < 2;
        ++issued;
        if (i == 0) have_next = next_run(p, walk, next);   // found while nothing waits for it
        if (++i == n) {
          if (elected) tc_commit(bar(Q_EMPTY + (runs & 1)));
          run = next;
          have_run = have_next;
          i = 0;
          ++runs;
        }
      };
      next_s();
      if (ok) next_s();
      for (int done = 0; ok && done < issued; ++done) {
        if (!mbar_wait(bar(V_FULL + vs), vp, abort_flag)) {
          give_up(95, done);
          break;
        }
        issue_pv(done & 1, first[done & 1], done);
        if (ok) free_v();
        if (ok) next_s();
      }
    }
    __syncwarp();
  } else {
    const int x = (warp - 2) >> 2;              // group A or B
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_addr = uint32_t(quarter * 32) << 16;
    const uint32_t tmem_s = tmem_base + x * 128 + lane_addr;
    const uint32_t tmem_o = tmem_base + 256 + x * 128 + lane_addr;
    bool ok = true;
    int runs = 0;
    int tile0 = 0, other_tiles = 0;             // key tiles of the CTA's earlier runs; split: the other group's so far
    uint32_t sp = 0;                            // parity of the group's next S (and P V)
    auto give_up = [&](int role, int detail) {
      report_status(p.status, role, detail);
      *abort_flag = 1;
      ok = false;
    };
    volatile int* words = run_words + (warp - 2) * 2 * kRunWords;   // this run's and the next one's
    // the query row this thread has in a run: token and head, and whether there is one
    struct Place {
      int t, hq;
      bool live;
    };
    auto place_in = [&](const Run& run) {
      Place q;
      const int in_tile = QUAD ? lane : row, in_half = in_tile / p.group;
      q.t = (PAIR ? run.row_tile * 2 + x : run.row_tile) * p.half_tokens + in_half;
      q.hq = run.head * p.group + (in_tile - in_half * p.group);
      q.live = in_half < p.half_tokens && q.t < run.seq.fresh;
      return q;
    };
    if (lane == 0) save_run(words, walk, run);
    __syncwarp();
    for (; have_run && ok; ++runs) {
      volatile int* mine = words + (runs & 1) * kRunWords;
      int n, first_tile, have;
      bool live, any_live;
      {
        const Run run = saved_run(mine);
        live = place_in(run).live;
        any_live = __any_sync(0xffffffffu, live);
        n = run.last - run.first;
        first_tile = run.first;
        have = run.seq.have;
      }
      // split: the first of the run's tiles that is this group's; the group of the last one finishes
      const int i0 = PAIR ? 0 : (tile0 ^ x) & 1, di = PAIR ? 1 : 2;
      const bool finish = PAIR || ((tile0 + n - 1 - x) & 1) == 0;
      float m_used = -INFINITY, l = 0.0f;
      // the run is this warp's no more than to its last P: what others read of it is in place
      auto leave_run = [&]() {
        if (!finish) state_b[row] = make_float2(m_used, l);
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(RUN_DONE));
      };
      // the group that finished the run before has read this one's O of it: the first P V of this
      // run may begin to overwrite it
      auto await_o_read = [&](int i) {
        if (!PAIR && i == 0 && runs > 0 && !mbar_wait(bar(O_READ), (runs - 1) & 1, abort_flag)) give_up(99, runs);
      };
      if (i0 >= n) leave_run();                 // no share of a single tile
      for (int i = i0; i < n; i += di) {
        const int j = first_tile + i;
        const int key0 = j * kPaBN;
        const bool edge = key0 + kPaBN > have;       // the step's tokens, or slots behind the last one
        uint32_t sees[4] = {0u, 0u, 0u, 0u};
        if (edge && any_live) {
          const Run run = saved_run(mine);
          const int t = place_in(run).t;
          const int t0 = __shfl_sync(0xffffffffu, t, 0);
          const int t1 = min(__shfl_sync(0xffffffffu, t, 31), run.seq.fresh - 1);
          if constexpr (QUAD) {
            sees[0] = visible_keys(p, run.seq, run.b, t, t0, t1, key0 + 32 * quarter, lane);
          } else {
#pragma unroll 1
            for (int w = 0; w < 4; ++w) {                // rolled: the words move up
              sees[0] = sees[1];
              sees[1] = sees[2];
              sees[2] = sees[3];
              sees[3] = visible_keys(p, run.seq, run.b, t, t0, t1, key0 + 32 * w, lane);
            }
          }
        }
        if (!mbar_wait(bar(S_FULL + x), sp, abort_flag)) {
          give_up(96, j);
          break;
        }
        // Row `row` of the tile's V is cleared where no token lies; in a token of the step that some query
        // may not see, the values that are not finite are (the epilogue adds them to the rows that see
        // them).  After the softmax of the first half, so that V has had that long to come.  S_FULL said that the P V two
        // tiles back is done, so V_FULL's phase is this tile's or the one before.
        auto clear_v = [&]() {
          const int vi = tile0 + i, vs = vi % R::kV;
          if (!mbar_wait(bar(V_FULL + vs), (vi / R::kV) & 1, abort_flag)) {
            give_up(95, j);
            return;
          }
          // (rows lie 128 bytes apart: every lane starts at another 16-byte piece, or all would
          // meet in the same banks)
          const uint32_t v_row = v_smem + vs * R::kTile + row * 128;
          const int key = key0 + row;
          if (key >= mine[6]) {                           // the sequence's length
#pragma unroll 2
            for (int c = 0; c < D / 8; ++c) st_shared_v4(v_row + (c / 8) * kBoxBytes + ((c ^ row) & 7) * 16, 0u, 0u, 0u, 0u);
          } else if (key >= have && (p.mask != nullptr || p.tokens > 1)) {
            bool bad = false;
#pragma unroll 2
            for (int c = 0; c < D / 8; ++c) {
              const uint32_t at = v_row + (c / 8) * kBoxBytes + ((c ^ row) & 7) * 16;
              uint32_t y[4], keep[4];
              ld_shared_v4(at, y);
#pragma unroll
              for (int i = 0; i < 4; ++i) keep[i] = finite_halves<BF16>(y[i]);
              if ((keep[0] & keep[1] & keep[2] & keep[3]) != 0xffffffffu) {
                st_shared_v4(at, y[0] & keep[0], y[1] & keep[1], y[2] & keep[2], y[3] & keep[3]);
                bad = true;
              }
            }
            if (bad) bad_draft[runs & 1] = runs;
          }
          fence_proxy_async_smem();
          __syncwarp();
        };
        tc_fence_after_sync();
        if (any_live) {                                   // a warp of padding rows only keeps step
          float sq[32];                                   // quad: the warp's 32 keys
          // S in halves of 64 scores, once for the maximum and once for the exponentials: a row of 128
          // in registers would spill, and local memory is what the L1 beside 224 KB of tiles
          // serves worst
          auto load_scores = [&](int half, float (&s)[64]) {
            uint32_t y[64];
            tmem_ld_32x32b_x64(tmem_s + half * 64, y);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 64; ++k) s[k] = __uint_as_float(y[k]);
            const uint32_t lo = half == 0 ? sees[0] : sees[2], hi = half == 0 ? sees[1] : sees[3];
            if (edge && !__all_sync(0xffffffffu, (lo & hi) == 0xffffffffu)) {
#pragma unroll
              for (int k = 0; k < 64; ++k)
                if ((((k < 32 ? lo : hi) >> (k % 32)) & 1u) == 0u) s[k] = -INFINITY;
            }
          };
          // halves behind the last key that any row of the warp sees are left out
          const int halves = edge && !__any_sync(0xffffffffu, (sees[2] | sees[3]) != 0u) ? 1 : 2;
          float mx = -INFINITY;
          if constexpr (QUAD) {
            uint32_t y[32];
            tmem_ld_32x32b_x32(tmem_s + quarter * 32, y);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 32; ++k) sq[k] = __uint_as_float(y[k]);
            if (edge) {
#pragma unroll
              for (int k = 0; k < 32; ++k)
                if (((sees[0] >> k) & 1u) == 0u) sq[k] = -INFINITY;
            }
            float m2[2] = {fmax3(sq[0], sq[1], sq[2]), fmax3(sq[16], sq[17], sq[18])};
#pragma unroll
            for (int k = 3; k < 15; k += 2) {
              m2[0] = fmax3(m2[0], sq[k], sq[k + 1]);
              m2[1] = fmax3(m2[1], sq[16 + k], sq[17 + k]);
            }
            mx = fmaxf(fmax3(m2[0], m2[1], sq[15]), sq[31]);
          } else {
#pragma unroll 1
            for (int half = 0; half < halves; ++half) {
              float s[64];
              load_scores(half, s);
              float m4[4];
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                m4[c] = fmax3(s[16 * c], s[16 * c + 1], s[16 * c + 2]);
#pragma unroll
                for (int k = 3; k < 15; k += 2) m4[c] = fmax3(m4[c], s[16 * c + k], s[16 * c + k + 1]);
                m4[c] = fmaxf(m4[c], s[16 * c + 15]);
              }
              mx = fmaxf(mx, fmax3(m4[0], m4[1], fmaxf(m4[2], m4[3])));
            }
          }
          // a row that sees a key has a maximum above -inf, also where its scores are -inf or NaN
          const bool some = !edge || (sees[0] | sees[1] | sees[2] | sees[3]) != 0u;
          const float m_new = fmax3(m_used, mx * p.scale_log2, some ? -FLT_MAX : -INFINITY);
          const bool grow = (m_new - m_used > kRescaleThreshold) || (m_used == -INFINITY && m_new > -INFINITY);
          const bool any_grow = __any_sync(0xffffffffu, grow);
          float alpha = 1.0f;
          if (grow) {
            alpha = (m_used == -INFINITY) ? 0.0f : fast_exp2(m_used - m_new);
            m_used = m_new;
          }
          if (any_grow && i > i0) {
            // this S was committed after the group's last P V, so O is quiescent
            l *= alpha;
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t y[32];
              tmem_ld_32x32b_x32(tmem_o + c * 32, y);
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 32; ++k) y[k] = __float_as_uint(__uint_as_float(y[k]) * alpha);
              tmem_st_32x32b_x32(tmem_o + c * 32, y);
            }
          }
          const float neg_m = (m_used == -INFINITY) ? 0.0f : -m_used;
          const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
          const float2 negm2 = make_float2(neg_m, neg_m);
          float2 sum2[4] = {};
          if constexpr (QUAD) {
            uint32_t pk[16], none[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const float2 y = __ffma2_rn(make_float2(sq[2 * k], sq[2 * k + 1]), scale2, negm2);
              const float2 e = make_float2(fast_exp2(y.x), fast_exp2(y.y));
              sum2[k & 3] = __fadd2_rn(sum2[k & 3], e);
              pk[k] = BF16 ? pack_bf16x2(e.x, e.y) : pack_f16x2(e.x, e.y);
              none[k] = 0u;
            }
            // the other warps' keys: zero, where S lay
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              if (w == quarter) tmem_st_32x32b_x16(tmem_s + w * 16, pk);
              else tmem_st_32x32b_x16(tmem_s + w * 16, none);
            }
            if (edge) clear_v();
            await_o_read(i);
            tmem_st_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(P_HALF + x));
          } else {
#pragma unroll 1
            for (int c = 0; c < 2; ++c) {
              uint32_t pk[32];
              if (c < halves) {
                float s[64];
                load_scores(c, s);                            // P of the first half lies over scores already used
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                  const float2 y = __ffma2_rn(make_float2(s[2 * k], s[2 * k + 1]), scale2, negm2);
                  // pair: every fourth pair on the FMA pipe, as two row tiles keep the special-function
                  // unit busier than the tensor cores (133 -> 130 us); split waits for memory.  7.5e-5 of a
                  // weight, where its rounding to 16 bits below takes up to 2^-8 or 2^-11
                  const bool poly = PAIR && k % kFmhaPolyEvery == kFmhaPolyEvery - 1;
                  const float2 e = poly ? exp2_poly_pair<true>(y) : make_float2(fast_exp2(y.x), fast_exp2(y.y));
                  sum2[k & 3] = __fadd2_rn(sum2[k & 3], e);
                  // P is rounded to the input type: it is the tensor cores' operand
                  pk[k] = BF16 ? pack_bf16x2(e.x, e.y) : pack_f16x2(e.x, e.y);
                }
              } else {
#pragma unroll
                for (int k = 0; k < 32; ++k) pk[k] = 0u;
              }
              tmem_st_32x32b_x32(tmem_s + c * 32, pk);
              if (c == 0) {                                 // the first 64 keys are enough for half of P V
                if (edge && (!PAIR || x == 0)) clear_v();
                await_o_read(i);
                tmem_st_wait();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(P_HALF + x));
              }
            }
          }
          l += ((sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y)) + ((sum2[2].x + sum2[2].y) + (sum2[3].x + sum2[3].y));
          tmem_st_wait();
        } else {
          if (edge && (!PAIR || x == 0)) clear_v();
          await_o_read(i);
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(P_HALF + x));
        }
        if (!ok) break;
        sp ^= 1;
        // before the last P: whoever finds the run's products done finds these arrivals made, so
        // the phases of RUN_DONE cannot lie two apart
        if (i + di >= n) leave_run();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(P_FULL + x));
      }
      tile0 += n;
      if (!ok) break;
      {
        Walk on = saved_walk(mine);
        Run next;
        have_run = next_run(p, on, next);
        __syncwarp();
        if (lane == 0) save_run(words + ((runs + 1) & 1) * kRunWords, on, next);
        __syncwarp();
      }
      other_tiles += (n + i0) / 2;
      if (!finish) continue;                              // the other group finishes the run
      const bool edges = (first_tile + n) * kPaBN > have;
      const bool two = !PAIR && n > 1;                    // the other group has a share of it
      if (!mbar_wait(bar(PV_DONE + x), sp ^ 1, abort_flag) ||
          (two && !mbar_wait(bar(PV_DONE + (x ^ 1)), (other_tiles - 1) & 1, abort_flag)) ||
          ((!PAIR || edges) && !mbar_wait(bar(RUN_DONE), runs & 1, abort_flag))) {
        give_up(97, runs);
        break;
      }
      tc_fence_after_sync();

      // the run's result: the output where the run is the whole item, else a partial state
      float fa = 1.0f, fb = 0.0f;
      if (two) {
        const float2 sb = state_b[row];
        const float m = fmaxf(m_used, sb.x);
        fa = (m_used == -INFINITY) ? 0.0f : fast_exp2(m_used - m);
        fb = (sb.x == -INFINITY) ? 0.0f : fast_exp2(sb.x - m);
        l = l * fa + sb.y * fb;
        m_used = m;
      }
      const Run run = saved_run(mine);
      const Place at = place_in(run);
      // quad always leaves its four states, a whole item's in a slot of the item's
      const bool all = run.first == 0 && run.last == run.seq.tiles, whole = !QUAD && all;
      const int64_t slot = QUAD && all ? 2 * static_cast<int64_t>(p.ctas) + run.b * p.heads_kv + run.head
                                       : 2 * static_cast<int64_t>(blockIdx.x) + (runs == 0 ? 0 : 1);
      // quad: every quarter's rows are a state of their own
      const int tile_row = QUAD ? quarter * (p.tile_rows / 4) + lane : (PAIR ? x * kPaBM : 0) + row;
      const float inv_l = softmax_factor(m_used, l);
      const bool by_hand = edges && bad_draft[runs & 1] == runs;
      uint16_t* o_row = p.out + run.b * p.o_b + at.hq * p.o_h + at.t * p.o_t;
      float4* acc = reinterpret_cast<float4*>(p.ws_acc) + slot * (D / 4) * p.tile_rows + tile_row;
      if (live && !whole) reinterpret_cast<float2*>(p.ws_ml)[slot * p.tile_rows + tile_row] = make_float2(m_used, l);
      if (any_live) {
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
          {
            uint32_t y[32];
            tmem_ld_32x32b_x32(tmem_o + c * 32, y);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = __uint_as_float(y[k]);
            if (two) {                                    // the other group's O lies in the same lanes
              tmem_ld_32x32b_x32(tmem_base + 256 + (x ^ 1) * 128 + lane_addr + c * 32, y);
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = o[k] * fa + __uint_as_float(y[k]) * fb;
            }
          }
          if (live && whole) {
            uint32_t pk[16];
#pragma unroll
            for (int k = 0; k < 16; ++k)
              pk[k] = BF16 ? pack_bf16x2(o[2 * k] * inv_l, o[2 * k + 1] * inv_l)
                           : pack_f16x2(o[2 * k] * inv_l, o[2 * k + 1] * inv_l);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int d0 = c * 32 + 8 * k;
              if (d0 < p.dim) {
                if (p.o_vec) {
                  *reinterpret_cast<uint4*>(o_row + d0) = make_uint4(pk[4 * k], pk[4 * k + 1], pk[4 * k + 2], pk[4 * k + 3]);
                } else {
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    o_row[d0 + 2 * e] = static_cast<uint16_t>(pk[4 * k + e] & 0xffff);
                    o_row[d0 + 2 * e + 1] = static_cast<uint16_t>(pk[4 * k + e] >> 16);
                  }
                }
              }
            }
          } else if (live) {
#pragma unroll
            for (int k = 0; k < 8; ++k)                   // neighbouring rows side by side
              acc[static_cast<int64_t>(c * 8 + k) * p.tile_rows] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
          }
          __syncwarp();
        }
        // (a sum of NaN makes the row NaN anyway)
        if (by_hand && live && l == l)
          add_not_finite<BF16>(p, run, at.t, QUAD ? quarter : -1, whole, o_row, reinterpret_cast<float*>(acc));
        __syncwarp();
      }
      tc_fence_before_sync();
      if (!PAIR) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(O_READ));
      }
    }
    __syncwarp();
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, kPaTmemCols);
  }
}

// Four columns of a row, from column c0, with those that are NaN taken from V itself: the sum of the
// values there that are not finite, over the keys that token t sees.  With a weight above zero each is
// what it is, and beside them the finite ones do not matter.  Where there is no such value, the
// NaN stays.
template <bool BF16>
__device__ __forceinline__ float4 infinite_values(const PagedParams& p, const SeqInfo& seq, int b, int head, int t, int c0,
                                               float4 o) {
  const uint8_t* mask = p.mask + b * p.mask_b + t * p.mask_t;
  const int* pages = p.page_table + b * p.page_table_stride;
  const uint16_t* v = p.v + head * p.vc_h + c0;
  const int to = p.mask == nullptr ? min(seq.len, seq.have + t + 1) : seq.len;
  float sum[4] = {};
  bool all_nan = false;
#pragma unroll 1
  for (int k0 = 0; k0 < to && !all_nan; k0 += 4) {            // four slots of a page
    const int entry = k0 / p.page_size, page = pages[entry];
    if (page < 0 || page >= p.num_pages) continue;
    const uint16_t* at = v + page * p.vc_p + (k0 - entry * p.page_size) * p.vc_s;
    uint2 rows[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int key = k0 + u;
      const bool sees = key < to && (p.mask == nullptr || key < seq.have || mask[(key - seq.have) * p.mask_j] != 0);
      rows[u] = sees ? *reinterpret_cast<const uint2*>(at + u * p.vc_s) : make_uint2(0u, 0u);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint32_t bad[2] = {rows[u].x & ~finite_halves<BF16>(rows[u].x), rows[u].y & ~finite_halves<BF16>(rows[u].y)};
      if ((bad[0] | bad[1]) == 0u) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] += half_to_float<BF16>(static_cast<uint16_t>(bad[i / 2] >> (16 * (i & 1))));
      all_nan = sum[0] != sum[0] && sum[1] != sum[1] && sum[2] != sum[2] && sum[3] != sum[3];
    }
  }
  const auto chosen = [](float old, float found) { return old != old && found != 0.f ? found : old; };
  return make_float4(chosen(o.x, sum[0]), chosen(o.y, sum[1]), chosen(o.z, sum[2]), chosen(o.w, sum[3]));
}

// Joins the partial states of items that several CTAs share, and clears padding rows.  A thread owns
// four columns of a row (neighbouring threads neighbouring rows, as the states are stored) and
// takes every G-th state in range order; its G partners' results meet in shared memory.
template <int D, bool BF16, int MODE, int E, int G>
__global__ void __launch_bounds__(E * G)
paged_attention_join_kernel(const __grid_constant__ PagedParams p) {
  const int lane = threadIdx.x & 31;
  pdl_launch_dependents();
  const int per_seq = p.heads_kv * p.row_tiles;
  const int any_item = blockIdx.x / p.join_blocks;      // of all sequences
  const int b = any_item / per_seq, item = any_item - b * per_seq;
  const int head = item / p.row_tiles, row_tile = item - head * p.row_tiles;
  const int element = (blockIdx.x - any_item * p.join_blocks) * E + threadIdx.x % E;
  constexpr bool PAIR = MODE == kPair;
  constexpr int kStates = MODE == kQuad ? 4 : 1;     // partial states of a row that a run leaves
  const int out_rows = p.tile_rows / kStates;
  const int quad = element / out_rows, row = element - quad * out_rows;
  const SeqInfo seq = seq_info(p, b);
  int all = 0, before = 0;             // key tiles of all sequences, of those before this one
#pragma unroll 1
  for (int i = lane; i < p.batch; i += 32) {
    const int tiles = seq_info(p, i).tiles;
    all += tiles;
    before += i < b ? tiles : 0;
  }
  const Ranges ranges(warp_sum(all) * per_seq, p.ctas);
  const int first = warp_sum(before) * per_seq + item * seq.tiles;
  const int half = row / kPaBM, in_half = (row - half * kPaBM) / p.group;
  const int hq = head * p.group + (row - half * kPaBM) - in_half * p.group;
  const int t = (PAIR ? row_tile * 2 + half : row_tile) * p.half_tokens + in_half;
  const bool mine = quad * 4 < p.dim && in_half < p.half_tokens && t < p.tokens;
  const bool real = mine && t < seq.fresh;
  const int c0 = seq.tiles > 0 ? ranges.owner(first) : 0, c1 = seq.tiles > 0 ? ranges.owner(first + seq.tiles - 1) : 0;
  // a row of an item that one CTA has finished is in place; a padding row is cleared on request
  const bool store = mine && (real ? kStates > 1 || c0 != c1 || seq.tiles == 0 : p.zero_padding != 0);
  uint16_t* dst = p.out + b * p.o_b + static_cast<int64_t>(hq) * p.o_h + t * p.o_t + quad * 4;
  const int g = threadIdx.x / E, e = threadIdx.x % E;
  __shared__ float2 sm_ml[G][E];
  __shared__ float4 sm_o[G][E];
  if (store) asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<uint64_t>(dst)));
  // Everything below runs twice: once on whatever the workspace holds, with nothing stored, while
  // the kernel before still computes - its instructions and address translations are then at
  // hand, which took longer than the join itself - and once, after that kernel's end, in earnest.
  // Loads go past the L1, so nothing of the first pass is seen in the second.  A block's start
  // waits for a CTA of that kernel to leave its SM, so the first pass is for the blocks that come
  // into the first free places, and for kernels that last: with it 8 heads and 8000 keys 17.8 us
  // against 18.4, 32 sequences of 2048 keys 53.1 against 53.9; without it a token of 32 heads and 1024
  // keys (less than two tiles a CTA) 13.5 against 14.1, 16 x 32 rows of 4 (8192 blocks) 41.8 against 43.
  const bool rehearse = ranges.base >= 3 && blockIdx.x < p.ctas;
#pragma unroll 1
  for (int pass = rehearse ? 0 : 1; pass < 2; ++pass) {
    // the partial states come from the kernel launched just before; every thread waits for it, so
    // that this kernel's end is that one's end too
    if (pass == 1) pdl_wait();
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    // A state that saw nothing has a maximum of -inf and a sum of 0; the sum of one that saw NaN is
    // NaN, which no factor of 0 removes.  Without a branch, so that the loads of several states are
    // under way at once.
    auto take = [&](float mc, float lc, const float4& a) {
      const float top = fmaxf(m, mc);
      const float f = (m == -INFINITY) ? 0.f : fast_exp2(m - top), h = (mc == -INFINITY) ? 0.f : fast_exp2(mc - top);
      l = l * f + lc * h;
      o.x = o.x * f + a.x * h;
      o.y = o.y * f + a.y * h;
      o.z = o.z * f + a.z * h;
      o.w = o.w * f + a.w * h;
      m = top;
    };
    if ((kStates > 1 || c0 != c1) && real && seq.tiles > 0) {
      const float4* acc = reinterpret_cast<const float4*>(p.ws_acc);
      const float2* ml = reinterpret_cast<const float2*>(p.ws_ml);
      const int states = (c1 - c0 + 1) * kStates, last = pass == 0 ? min(states, G) : states;
#pragma unroll 4
      for (int k = g; k < last; k += G) {
        const int c = c0 + k / kStates, at = (k % kStates) * out_rows + row;
        // only the first of an item's CTAs may have begun with an earlier item
        const int64_t slot = kStates > 1 && c0 == c1 ? 2 * static_cast<int64_t>(p.ctas) + any_item
                                                     : 2 * static_cast<int64_t>(c) + (ranges.begin(c) >= first ? 0 : 1);
        const float2 state = __ldcg(ml + slot * p.tile_rows + at);
        take(state.x, state.y, __ldcg(acc + (slot * (D / 4) + quad) * p.tile_rows + at));
      }
    }
    if constexpr (G > 1) {
      __syncthreads();
      sm_ml[g][e] = make_float2(m, l);
      sm_o[g][e] = o;
      __syncthreads();
      if (g == 0) {
#pragma unroll
        for (int k = 1; k < G; ++k) take(sm_ml[k][e].x, sm_ml[k][e].y, sm_o[k][e]);
      }
    }
    // quad: the three quarters that have no share of a key multiply its V by zeros, and 0 * inf is NaN
    if (kStates > 1 && pass == 1 && store && g == 0 && real && l == l && !(o.x + o.y + o.z + o.w == o.x + o.y + o.z + o.w))
      o = infinite_values<BF16>(p, seq, b, head, t, quad * 4, o);
    const float inv_l = softmax_factor(m, l);
    const uint32_t lo = BF16 ? pack_bf16x2(o.x * inv_l, o.y * inv_l) : pack_f16x2(o.x * inv_l, o.y * inv_l);
    const uint32_t hi = BF16 ? pack_bf16x2(o.z * inv_l, o.w * inv_l) : pack_f16x2(o.z * inv_l, o.w * inv_l);
    if (pass == 1 && store && g == 0) {
      if (p.o_vec) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
      } else {
        dst[0] = static_cast<uint16_t>(lo & 0xffff);
        dst[1] = static_cast<uint16_t>(lo >> 16);
        dst[2] = static_cast<uint16_t>(hi & 0xffff);
        dst[3] = static_cast<uint16_t>(hi >> 16);
      }
    }
  }
}

// ---- host ------------------------------------------------------------------------------------

int padded_dim(const b200k_paged_attention_args* a) { return a->head_dim <= 64 ? 64 : 128; }

// The rows that share a key/value head, token by token, and how they are cut: one 128-row half
// ("split"; "quad" where there are few rows and many items), or tiles of two halves ("pair") where there
// are more.  A half holds whole tokens.
struct Rows {
  Mode mode;
  int64_t half_tokens, tiles, per_tile;      // per_tile: rows of a partial state
  int64_t slots(const b200k_paged_attention_args* a, int64_t ctas) const {   // partial states
    return 2 * ctas + (mode == kQuad ? a->batch * a->heads_kv : 0);
  }
};
Rows lay_out_rows(const b200k_paged_attention_args* a, int sms) {
  const int64_t group = a->heads_q / a->heads_kv;
  Rows r;
  const int64_t rows = a->tokens * group;
  // quad shortens a tile's softmax and pays with four states per item: it gains where CTAs walk
  // several short items (64 sequences of up to 500 keys, 8 heads: 49 -> 38 us; of 1000 63 -> 47; 64
  // items of 2000 keys 17.2 -> 16.5), not where many CTAs share one (32 items 13.7 -> 14.6; 8 items
  // 17.9 -> 18.5), nor with more rows to write (16 rows 67 -> 61, 32 rows 28.9 -> 32.1)
  r.mode = rows <= kPaQuadRows && 3 * a->batch * a->heads_kv >= sms ? kQuad : (rows <= kPaBM ? kSplit : kPair);
  r.half_tokens = r.mode == kPair ? kPaBM / group : a->tokens;
  r.tiles = r.mode == kPair ? ceil_div(a->tokens, 2 * r.half_tokens) : 1;
  r.per_tile = r.mode == kPair ? 2 * kPaBM : (r.mode == kQuad ? 4 * rows : rows);
  return r;
}

// CTAs of a call: one per SM, fewer where there cannot be as many key tiles.
int64_t pick_ctas(const b200k_paged_attention_args* a, int sms) {
  const int64_t items = a->batch * a->heads_kv * lay_out_rows(a, sms).tiles;
  const int64_t most = items * ceil_div(static_cast<int64_t>(a->max_pages) * a->page_size, kPaBN);
  const int64_t n = most < sms ? most : sms;
  return n < 1 ? 1 : n;
}

int check_args(const b200k_paged_attention_args* a) {
  if (a == nullptr) return fail(B200K_INVALID_ARG, "null args");
  if (a->batch < 0 || a->tokens < 0 || a->heads_q < 0 || a->heads_kv <= 0 || a->num_pages < 0 || a->max_pages < 0)
    return fail(B200K_INVALID_ARG, "negative dimension, or no key/value heads");
  if (a->heads_q % a->heads_kv != 0) return fail(B200K_INVALID_ARG, "heads_q must be a multiple of heads_kv");
  if (a->heads_q > kPaBM * a->heads_kv)
    return fail(B200K_UNSUPPORTED, "at most %d query heads per key/value head", kPaBM);
  if (a->dtype != B200K_F16 && a->dtype != B200K_BF16) return fail(B200K_INVALID_ARG, "dtype must be f16 or bf16");
  if (a->head_dim <= 0 || a->head_dim > 128 || a->head_dim % 8 != 0)
    return fail(B200K_UNSUPPORTED, "head_dim must be a multiple of 8 up to 128 (got %d)", a->head_dim);
  if (!(a->qk_scale > 0.f) || a->qk_scale > 2.0e38f)   // times log2(e) it is finite, too
    return fail(B200K_INVALID_ARG, "qk_scale must be positive and at most 2e38");
  if (a->page_size <= 0 || a->page_size % 8 != 0)
    return fail(B200K_UNSUPPORTED, "page_size must be a positive multiple of 8 (got %d)", a->page_size);
  const int64_t limit = int64_t(1) << 29;   // sums of two such counts fit 32 bits
  const int64_t width = static_cast<int64_t>(a->max_pages) * a->page_size;   // tokens that a sequence's table can name
  if (a->tokens > limit || a->heads_q > limit || a->tokens * a->heads_q > limit || width > limit ||
      a->num_pages >= limit || a->batch > kPaMaxBatch || a->heads_kv > limit ||
      // key tiles of all items, were every table full: never summed with another such count
      a->batch * a->heads_kv * lay_out_rows(a, 1).tiles > INT32_MAX / (width > kPaBN ? ceil_div(width, kPaBN) : 1))
    return fail(B200K_UNSUPPORTED, "more rows, pages or sequences than the kernel counts");
  return B200K_OK;
}

template <int D, bool BF16, int MODE>
int launch_paged_as(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, PagedParams p, int64_t items,
                    cudaStream_t stream) {
  constexpr int kSmem = Rings<D>::kSmem;
  auto kernel = paged_attention_kernel<D, BF16, MODE>;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess)
      return fail(B200K_CUDA_ERROR, "cudaFuncSetAttribute(%d): %s", kSmem, cudaGetErrorString(e));
    configured[dev] = true;
  }
  // Many outputs: a thread for each.  Few mean few items, each shared by many CTAs: several threads
  // to an output, in blocks of a warp of outputs (a token of 32 heads and 1024 keys 13.7 us with
  // eight, 13.9 with four, 14.4 with sixteen; 8 heads and 8000 keys 17.9, 19.3, 18.4).  Quad has at
  // least a third as many items as CTAs, so few states each: four threads and larger blocks (32
  // sequences of 2048 keys, 256 items: 53.2 us against 56.5 with eight and 64.5 with sixteen).
  constexpr int kFewE = MODE == kQuad ? 128 : 32, kFewG = MODE == kQuad ? 4 : 8;
  const int64_t outputs = static_cast<int64_t>(p.tile_rows / (MODE == kQuad ? 4 : 1)) * (D / 4);
  static_assert(kSmem <= 227 * 1024, "shared memory of one CTA");
  const bool many = outputs * items >= 256 * current_sm_count();
  p.join_blocks = static_cast<int>(ceil_div(outputs, many ? 128 : kFewE));
  if (items * p.join_blocks > INT32_MAX) return fail(B200K_UNSUPPORTED, "more row tiles than a grid has blocks");
  // programmatic launches: this kernel's set-up (barriers, tensor memory, descriptors) overlaps the
  // end of the kernel before it, and its end the set-up of the joining kernel
  cudaError_t e = launch_after_predecessor(kernel, dim3(p.ctas), dim3(kPaThreads), kSmem, stream, tq, tk, tv, p);
  if (e != cudaSuccess) return fail(B200K_CUDA_ERROR, "paged attention launch: %s", cudaGetErrorString(e));
  const dim3 grid(static_cast<unsigned>(items * p.join_blocks));
  e = many ? launch_after_predecessor(paged_attention_join_kernel<D, BF16, MODE, 128, 1>, grid, dim3(128), 0, stream, p)
           : launch_after_predecessor(paged_attention_join_kernel<D, BF16, MODE, kFewE, kFewG>, grid, dim3(kFewE * kFewG),
                                      0, stream, p);
  if (e != cudaSuccess) return fail(B200K_CUDA_ERROR, "paged attention join launch: %s", cudaGetErrorString(e));
  return B200K_OK;
}

template <int D, bool BF16>
int launch_paged(Mode mode, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const PagedParams& p,
                 int64_t items, cudaStream_t stream) {
  if (mode == kQuad) return launch_paged_as<D, BF16, kQuad>(tq, tk, tv, p, items, stream);
  if (mode == kSplit) return launch_paged_as<D, BF16, kSplit>(tq, tk, tv, p, items, stream);
  return launch_paged_as<D, BF16, kPair>(tq, tk, tv, p, items, stream);
}

}  // namespace
}  // namespace b200k

using namespace b200k;

extern "C" int64_t b200k_paged_attention_workspace_bytes(const b200k_paged_attention_args* a) {
  if (a == nullptr || a->batch <= 0 || a->tokens <= 0 || a->heads_kv <= 0 || a->heads_q < a->heads_kv ||
      a->page_size <= 0 || a->max_pages < 0 || a->head_dim <= 0 || a->head_dim > 128)
    return 0;
  const int sms = current_sm_count();
  if (sms <= 0) return 0;
  const Rows rows = lay_out_rows(a, sms);
  return rows.slots(a, pick_ctas(a, sms)) * rows.per_tile * (padded_dim(a) + 2) * 4;
}

extern "C" int b200k_paged_attention(const b200k_paged_attention_args* a, b200k_stream stream_) {
  const int rc = check_args(a);
  if (rc != B200K_OK) return rc;
  if (a->batch == 0 || a->tokens == 0 || a->heads_q == 0) return B200K_OK;
  if (!a->q || !a->k_cache || !a->v_cache || !a->out || !a->page_table || !a->cache_lens)
    return fail(B200K_INVALID_ARG, "null pointer");
  for (int64_t s : {a->q_stride_b, a->q_stride_h, a->q_stride_t, a->kc_stride_p, a->kc_stride_h, a->kc_stride_s,
                    a->vc_stride_p, a->vc_stride_h, a->vc_stride_s})
    if (s < 0 || s % 8 != 0) return fail(B200K_UNSUPPORTED, "query and cache strides must be multiples of 16 bytes");
  if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k_cache) |
       reinterpret_cast<uintptr_t>(a->v_cache)) & 15)
    return fail(B200K_UNSUPPORTED, "queries and caches must be 16-byte aligned");
  if (a->num_pages == 0) return fail(B200K_INVALID_ARG, "the cache has no pages");
  const int sms = current_sm_count();
  if (sms <= 0) return fail(B200K_CUDA_ERROR, "no current CUDA device");
  if (a->workspace == nullptr || (reinterpret_cast<uintptr_t>(a->workspace) & 15) ||
      a->workspace_bytes < b200k_paged_attention_workspace_bytes(a))
    return fail(B200K_INVALID_ARG, "workspace missing, unaligned or too small");

  PagedParams p = {};
  p.q = static_cast<const uint16_t*>(a->q);
  p.v = static_cast<const uint16_t*>(a->v_cache);
  p.out = static_cast<uint16_t*>(a->out);
  p.page_table = a->page_table;
  p.cache_lens = a->cache_lens;
  p.new_lens = a->new_lens;
  p.mask = a->tree_mask;
  p.o_b = a->o_stride_b; p.o_h = a->o_stride_h; p.o_t = a->o_stride_t;
  p.vc_p = a->vc_stride_p; p.vc_h = a->vc_stride_h; p.vc_s = a->vc_stride_s;
  p.mask_b = a->mask_stride_b; p.mask_t = a->mask_stride_t; p.mask_j = a->mask_stride_j;
  p.page_table_stride = a->page_table_stride;
  p.num_pages = a->num_pages;
  p.batch = static_cast<int>(a->batch);
  p.tokens = static_cast<int>(a->tokens);
  p.heads_kv = static_cast<int>(a->heads_kv);
  p.group = static_cast<int>(a->heads_q / a->heads_kv);
  p.dim = a->head_dim;
  const Rows rows = lay_out_rows(a, sms);
  p.half_tokens = static_cast<int>(rows.half_tokens);
  p.row_tiles = static_cast<int>(rows.tiles);
  p.tile_rows = static_cast<int>(rows.per_tile);
  p.page_size = a->page_size;
  p.max_pages = a->max_pages;
  // slots per TMA box: the largest power of two (8 to 128) that divides a page, so that a box
  // lies in one page and starts on a whole eight-row swizzle atom of the tile
  p.box_rows = 8;
  while (p.box_rows < kPaBN && a->page_size % (p.box_rows * 2) == 0) p.box_rows *= 2;
  p.page_shift = -1;
  for (int i = 3; i < 30; ++i)
    if (a->page_size == 1 << i) p.page_shift = i;
  p.ctas = static_cast<int>(pick_ctas(a, sms));
  const auto vec = [](const void* base, int64_t sb, int64_t sh, int64_t st) {
    return (reinterpret_cast<uintptr_t>(base) & 15) == 0 && sb % 8 == 0 && sh % 8 == 0 && st % 8 == 0;
  };
  p.o_vec = vec(a->out, p.o_b, p.o_h, p.o_t);
  p.zero_padding = a->zero_padding;
  p.scale_log2 = a->qk_scale * 1.4426950408889634f;
  const int d = padded_dim(a);
  p.ws_acc = static_cast<float*>(a->workspace);
  p.ws_ml = p.ws_acc + rows.slots(a, p.ctas) * p.tile_rows * d;
  p.status = device_status_word();

  const CUtensorMapDataType dt =
      a->dtype == B200K_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUtensorMap tq, tk, tv;
  // the stride of an axis of one entry is never used, but has to be one that a tensor map takes
  const auto bytes = [](int64_t entries, int64_t stride) -> uint64_t { return entries == 1 ? 16 : stride * 2; };
  if (!encode_tmap_4d(&tq, dt, a->q, a->head_dim, a->heads_q, a->tokens, a->batch, bytes(a->heads_q, a->q_stride_h),
                      bytes(a->tokens, a->q_stride_t), bytes(a->batch, a->q_stride_b), 64, p.group, p.half_tokens, 1,
                      CU_TENSOR_MAP_SWIZZLE_128B) ||
      !encode_tmap_4d(&tk, dt, a->k_cache, a->head_dim, a->page_size, a->heads_kv, a->num_pages,
                      bytes(a->page_size, a->kc_stride_s), bytes(a->heads_kv, a->kc_stride_h), bytes(a->num_pages, a->kc_stride_p), 64,
                      p.box_rows, 1, 1, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !encode_tmap_4d(&tv, dt, a->v_cache, a->head_dim, a->page_size, a->heads_kv, a->num_pages,
                      bytes(a->page_size, p.vc_s), bytes(a->heads_kv, p.vc_h), bytes(a->num_pages, p.vc_p), 64,
                      p.box_rows, 1, 1, CU_TENSOR_MAP_SWIZZLE_128B))
    return B200K_INVALID_ARG;
  const int64_t items = a->batch * a->heads_kv * p.row_tiles;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const bool bf16 = a->dtype == B200K_BF16;
  if (d == 128)
    return bf16 ? launch_paged<128, true>(rows.mode, tq, tk, tv, p, items, stream)
                : launch_paged<128, false>(rows.mode, tq, tk, tv, p, items, stream);
  return bf16 ? launch_paged<64, true>(rows.mode, tq, tk, tv, p, items, stream)
              : launch_paged<64, false>(rows.mode, tq, tk, tv, p, items, stream);
}

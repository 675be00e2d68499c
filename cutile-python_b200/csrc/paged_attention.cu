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
// timing.  Two CTAs share an SM: one's softmax overlaps the other's matrix products and loads.
//
//   warp 0      TMA producer: one box per run of slots inside a page
//   warp 1      MMA issuer: S = Q K^T, O += P V (P from tensor memory)
//   warps 2..5  Q to shared memory, softmax (a row per thread), epilogue
//
// Slots behind a sequence's last token may hold anything: their scores are masked by index and
// their rows of V are cleared in shared memory, since 0 * NaN is not 0.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "host.h"
#include "softmax.cuh"

namespace b200k {
namespace {

constexpr int kPaBM = 128;             // query rows of a tile
constexpr int kPaBN = 128;             // keys of a tile
constexpr int kPaThreads = 192;
constexpr int kPaTmemCols = 256;
constexpr int kPaCtasPerSM = 2;
constexpr int kPaMergeThreads = 128;

struct PagedParams {
  const uint16_t* q;
  const uint16_t* k;                   // caches as plain memory: the rare path of non-finite drafts
  const uint16_t* v;
  uint16_t* out;
  const int* page_table;
  const int* cache_lens;
  const int* new_lens;
  const uint8_t* mask;
  int64_t q_b, q_h, q_t, o_b, o_h, o_t, kc_p, kc_h, kc_s, vc_p, vc_h, vc_s, mask_b, mask_t, mask_j;
  int64_t page_table_stride, num_pages;
  int batch, tokens, heads_kv, group, dim;
  int rows, row_tiles, tile_rows;      // tokens * group; tiles of 128 of them; min(rows, 128)
  int page_size, max_pages, box_rows;
  int ctas;
  int q_vec, o_vec;                    // rows of q / out on 16-byte boundaries
  int zero_padding;
  float scale_log2;
  float* ws_ml;                        // (2 ctas, tile_rows, 2): row maximum and sum
  float* ws_acc;                       // (2 ctas, tile_rows, D)
  int* status;
};

// Lengths of a sequence, kept inside what its page table can name.
struct SeqInfo {
  int have, fresh, len, tiles;         // tokens before the step, of the step, their sum, key tiles
};
__device__ __forceinline__ SeqInfo seq_info(const PagedParams& p, int b) {
  SeqInfo s;
  const int64_t cap = static_cast<int64_t>(p.max_pages) * p.page_size;
  const int64_t have = p.cache_lens[b];
  int64_t fresh = p.tokens;
  if (p.new_lens != nullptr) fresh = max(0, min(p.new_lens[b], p.tokens));
  s.fresh = static_cast<int>(fresh);
  s.have = static_cast<int>(max(static_cast<int64_t>(0), min(have, cap)));
  s.len = static_cast<int>(min(s.have + fresh, cap));
  if (fresh == 0) s.len = 0;
  s.tiles = (s.len + kPaBN - 1) / kPaBN;
  return s;
}
__device__ __forceinline__ bool lengths_fit(const PagedParams& p, int b) {
  const int64_t have = p.cache_lens[b];
  const int64_t fresh = p.new_lens != nullptr ? max(0, min(p.new_lens[b], p.tokens)) : p.tokens;
  return fresh == 0 || (have >= 0 && have + fresh <= static_cast<int64_t>(p.max_pages) * p.page_size);
}

__device__ __forceinline__ int64_t warp_sum64(int64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Key tiles of the sequences [0, count), warp-collective.
__device__ __forceinline__ int64_t tiles_before(const PagedParams& p, int count, int lane) {
  int64_t sum = 0;
  for (int b = lane; b < count; b += 32) sum += seq_info(p, b).tiles;
  return warp_sum64(sum);
}

// First tile of CTA c's range; the ranges cover `total` tiles.
__device__ __forceinline__ int64_t range_begin(int c, int64_t total, int ctas) { return c * total / ctas; }
// The CTA whose range holds tile x.
__device__ __forceinline__ int range_owner(int64_t x, int64_t total, int ctas) {
  return static_cast<int>(((x + 1) * ctas - 1) / total);
}

// A CTA's walk over its range: runs of key tiles of one item.
struct Walk {
  int64_t left;                        // tiles still to come
  int b, item, tile;                   // sequence; head * row_tiles + row tile; first key tile
};
struct Run {
  SeqInfo seq;
  int b, head, row_tile, first, last;  // key tiles [first, last)
};
__device__ __forceinline__ bool next_run(const PagedParams& p, Walk& w, Run& r) {
  if (w.left <= 0) return false;
  do {                                 // sequences without tokens have no tiles
    if (w.b >= p.batch) return false;
    r.seq = seq_info(p, w.b);
  } while (r.seq.tiles == 0 && ++w.b > 0);
  r.b = w.b;
  r.head = w.item / p.row_tiles;
  r.row_tile = w.item - r.head * p.row_tiles;
  r.first = w.tile;
  r.last = static_cast<int>(min(static_cast<int64_t>(r.seq.tiles), w.tile + w.left));
  w.left -= r.last - r.first;
  w.tile = 0;
  if (++w.item == p.heads_kv * p.row_tiles) {
    w.item = 0;
    ++w.b;
  }
  return true;
}

// Whether a 16-bit float is an infinity or NaN, for the two halves of a word.
template <bool BF16>
__device__ __forceinline__ bool word_not_finite(uint32_t w) {
  const uint32_t e = BF16 ? 0x7f80u : 0x7c00u;
  return (w & e) == e || ((w >> 16) & e) == e;
}
template <bool BF16>
__device__ __forceinline__ float half_to_float(uint16_t h) {
  if constexpr (BF16) return __uint_as_float(static_cast<uint32_t>(h) << 16);
  else return __half2float(*reinterpret_cast<const __half*>(&h));
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kPaThreads, kPaCtasPerSM)
paged_attention_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                       const __grid_constant__ PagedParams p) {
  constexpr int kBoxes = D / 64;            // 64-element (128-byte) slices of the head dim
  constexpr int kTileBytes = 128 * D * 2;
  constexpr int kBoxBytes = 128 * 128;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t q_smem = base;
  const uint32_t k_smem = base + kTileBytes;
  const uint32_t v_smem = base + 2 * kTileBytes;
  uint8_t* tail = smem + 3 * kTileBytes;
  const uint32_t bar0 = smem_u32(tail);
  enum { Q_FULL = 0, K_FULL, K_EMPTY, V_FULL, V_EMPTY, S_FULL, P_FULL, PV_DONE, EDGE_DONE, NUM_BARS };
  auto bar = [&](int i) { return bar0 + 8u * i; };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail + 8 * NUM_BARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + 8 * NUM_BARS + 8);
  volatile int* bad_draft = reinterpret_cast<volatile int*>(tail + 8 * NUM_BARS + 16);   // [2], by run parity
  Walk* walk_start = reinterpret_cast<Walk*>(tail + 8 * NUM_BARS + 32);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  pdl_launch_dependents();   // the joining kernel may be set up now; it waits for this grid
  if (threadIdx.x == 0) {
    for (int i = 0; i < NUM_BARS; ++i) mbar_init(bar(i), (i == P_FULL || i == Q_FULL || i == EDGE_DONE) ? 4 : 1);
    *abort_flag = 0;
    bad_draft[0] = bad_draft[1] = -1;
    fence_barrier_init();
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), kPaTmemCols);
    tmem_relinquish();
  }
  if (warp == 2) {
    // this CTA's range of key tiles and the item it begins in
    const int per_seq = p.heads_kv * p.row_tiles;
    const int64_t total = tiles_before(p, p.batch, lane) * per_seq;
    Walk w;
    const int64_t begin = range_begin(blockIdx.x, total, p.ctas);
    w.left = range_begin(blockIdx.x + 1, total, p.ctas) - begin;
    w.b = 0;
    w.item = 0;
    w.tile = 0;
    int64_t before = 0;
    for (int b0 = 0; b0 < p.batch && w.left > 0; b0 += 32) {
      const int b = b0 + lane;
      const int64_t mine = b < p.batch ? static_cast<int64_t>(seq_info(p, b).tiles) * per_seq : 0;
      int64_t upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const bool here = begin >= before + upto - mine && begin < before + upto;
      const uint32_t who = __ballot_sync(0xffffffffu, here);
      if (who != 0) {
        if (here) {
          const int tiles = static_cast<int>(mine / per_seq);
          const int64_t in_seq = begin - (before + upto - mine);
          w.b = b;
          w.item = static_cast<int>(in_seq / tiles);
          w.tile = static_cast<int>(in_seq - static_cast<int64_t>(w.item) * tiles);
          *walk_start = w;
        }
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (w.left <= 0 && lane == 0) *walk_start = w;
    if (blockIdx.x == 0) {
      for (int b = lane; b < p.batch; b += 32)
        if (!lengths_fit(p, b)) report_bad_index(p.status, kRolePage, b);
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t tmem_s = tmem_base;          // S: 128 columns; P aliases its first 64
  const uint32_t tmem_o = tmem_base + 128;    // O: D columns
  constexpr uint32_t kFmt = BF16 ? kFmtBF16 : kFmtF16;
  Walk walk = *walk_start;
  Run run;

  if (warp == 0) {
    const int boxes_per_tile = kPaBN / p.box_rows;
    const bool elected = elect_one();
    bool ok = true;
    int it = 0;                                // key tiles so far, over all runs
    while (ok && next_run(p, walk, run)) {
      const int* pages = p.page_table + run.b * p.page_table_stride;
      for (int j = run.first; j < run.last; ++j, ++it) {
        const uint32_t ph = it & 1;
        const int boxes = min(boxes_per_tile, (run.seq.len - j * kPaBN + p.box_rows - 1) / p.box_rows);
        // lane i: the i-th run of slots, all of one page
        int page = 0, slot = 0;
        if (lane < boxes) {
          const int key = j * kPaBN + lane * p.box_rows;
          const int entry = key / p.page_size;
          slot = key - entry * p.page_size;
          page = pages[entry];
          if (page < 0 || page >= p.num_pages) {
            report_bad_index(p.status, kRolePage, run.b);
            page = static_cast<int>(p.num_pages);   // behind the last page: filled with zeros
          }
        }
        const uint32_t bytes = static_cast<uint32_t>(boxes) * p.box_rows * 128u * kBoxes;
        if (!mbar_wait(bar(K_EMPTY), ph ^ 1, abort_flag)) {
          report_status(p.status, 90, j);
          *abort_flag = 1;
          ok = false;
          break;
        }
        if (elected) mbar_arrive_expect_tx(bar(K_FULL), bytes);
        __syncwarp();
        if (lane < boxes) {
#pragma unroll
          for (int i = 0; i < kBoxes; ++i)
            tma_load_4d(k_smem + i * kBoxBytes + lane * p.box_rows * 128, &tmap_k, bar(K_FULL), i * 64, slot,
                        run.head, page);
        }
        __syncwarp();
        if (!mbar_wait(bar(V_EMPTY), ph ^ 1, abort_flag)) {
          report_status(p.status, 91, j);
          *abort_flag = 1;
          mbar_wait(bar(K_FULL), ph, abort_flag);
          ok = false;
          break;
        }
        if (elected) mbar_arrive_expect_tx(bar(V_FULL), bytes);
        __syncwarp();
        if (lane < boxes) {
#pragma unroll
          for (int i = 0; i < kBoxes; ++i)
            tma_load_4d(v_smem + i * kBoxBytes + lane * p.box_rows * 128, &tmap_v, bar(V_FULL), i * 64, slot,
                        run.head, page);
        }
        __syncwarp();
      }
    }
    if (it > 0) {   // no copy of this CTA is in flight when it leaves (bounded, also after a failure)
      mbar_wait(bar(K_FULL), (it - 1) & 1, abort_flag);
      mbar_wait(bar(V_FULL), (it - 1) & 1, abort_flag);
    }
    __syncwarp();
  } else if (warp == 1) {
    const bool elected = elect_one();
    constexpr uint32_t idesc_qk = make_idesc(kFmt, kFmt, false, false, kPaBM, kPaBN);
    constexpr uint32_t idesc_pv = make_idesc(kFmt, kFmt, false, true, kPaBM, D);
    bool ok = true;
    int it = 0, runs = 0;
    for (; ok && next_run(p, walk, run); ++runs) {
      if (!mbar_wait(bar(Q_FULL), runs & 1, abort_flag)) {
        report_status(p.status, 92, runs);
        *abort_flag = 1;
        break;
      }
      for (int j = run.first; j < run.last; ++j, ++it) {
        const uint32_t ph = it & 1;
        if (!mbar_wait(bar(K_FULL), ph, abort_flag)) {
          report_status(p.status, 93, j);
          *abort_flag = 1;
          ok = false;
          break;
        }
        tc_fence_after_sync();
        // S = Q K^T: both operands K-major, 16 elements (32 bytes) of the head dim per MMA
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk / 4) * kBoxBytes;
          const uint64_t qd = make_smem_desc(q_smem + off, 16, 1024, kSwizzle128B) + 2 * (kk % 4);
          const uint64_t kd = make_smem_desc(k_smem + off, 16, 1024, kSwizzle128B) + 2 * (kk % 4);
          if (elected) umma<kKindF16>(tmem_s, qd, kd, idesc_qk, kk > 0 ? 1u : 0u);
        }
        if (elected) {
          tc_commit(bar(K_EMPTY));
          tc_commit(bar(S_FULL));
        }
        if (!mbar_wait(bar(P_FULL), ph, abort_flag) || !mbar_wait(bar(V_FULL), ph, abort_flag)) {
          report_status(p.status, 94, j);
          *abort_flag = 1;
          ok = false;
          break;
        }
        tc_fence_after_sync();
        // O += P V: P from tensor memory, V (keys, D) with D contiguous = MN-major B
#pragma unroll
        for (int kk = 0; kk < kPaBN / 16; ++kk) {
          const uint64_t vd = make_smem_desc(v_smem + kk * 2048, kBoxBytes, 1024, kSwizzle128B);
          if (elected) umma_f16_ts(tmem_o, tmem_s + kk * 8, vd, idesc_pv, (j > run.first || kk > 0) ? 1u : 0u);
        }
        if (elected) {
          tc_commit(bar(V_EMPTY));
          tc_commit(bar(PV_DONE));
        }
      }
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_addr = uint32_t(quarter * 32) << 16;
    bool ok = true;
    int it = 0, runs = 0, edges = 0;           // key tiles, runs, tiles with an edge so far
    for (; ok && next_run(p, walk, run); ++runs) {
      const SeqInfo seq = run.seq;
      const int edges_before = edges;
      const int r = run.row_tile * kPaBM + row;          // row of the item: token * group + head
      const int t = r / p.group;
      const int hq = run.head * p.group + (r - t * p.group);
      const bool live = r < p.rows && t < seq.fresh;
      const bool any_live = __any_sync(0xffffffffu, live);
      const uint16_t* q_row = p.q + run.b * p.q_b + hq * p.q_h + t * p.q_t;
      // Q: this row in 16-byte pieces, in the 128-byte swizzle of the MMA operand.  The last S
      // of the previous run has been read (S_FULL), so nothing reads the old rows any more.
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        uint32_t w[4] = {0u, 0u, 0u, 0u};
        if (live && c * 8 < p.dim) {
          if (p.q_vec) {
            const uint4 x = *reinterpret_cast<const uint4*>(q_row + c * 8);
            w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              w[i] = static_cast<uint32_t>(q_row[c * 8 + 2 * i]) | (static_cast<uint32_t>(q_row[c * 8 + 2 * i + 1]) << 16);
          }
        }
        st_shared_v4(q_smem + (c / 8) * kBoxBytes + row * 128 + (((c % 8) ^ (row & 7)) * 16), w[0], w[1], w[2], w[3]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(Q_FULL));

      float m_used = -INFINITY, l = 0.0f;
      for (int j = run.first; j < run.last; ++j, ++it) {
        const uint32_t ph = it & 1;
        const int key0 = j * kPaBN;
        const bool edge = key0 + kPaBN > seq.have;       // the step's tokens, or slots behind the last one
        if (!mbar_wait(bar(S_FULL), ph, abort_flag)) {
          report_status(p.status, 96, j);
          *abort_flag = 1;
          ok = false;
          break;
        }
        if (edge) {
          // (S_FULL also says that P V of the last tile is done: only now is V_FULL's phase this
          // tile's, and V this tile's rows.)  Row `row` of V is cleared where no token lies, and where a token of the step that some
          // query may not see is not finite (added by hand in the epilogue)
          if (!mbar_wait(bar(V_FULL), ph, abort_flag)) {
            report_status(p.status, 95, j);
            *abort_flag = 1;
            ok = false;
            break;
          }
          const int key = key0 + row;
          bool clear = key >= seq.len;
          if (!clear && key >= seq.have && (p.mask != nullptr || p.tokens > 1)) {
#pragma unroll 4
            for (int c = 0; c < D / 8; ++c) {
              uint32_t x[4];
              ld_shared_v4(v_smem + (c / 8) * kBoxBytes + row * 128 + (c % 8) * 16, x);
              clear = clear || word_not_finite<BF16>(x[0]) || word_not_finite<BF16>(x[1]) ||
                      word_not_finite<BF16>(x[2]) || word_not_finite<BF16>(x[3]);
            }
            if (clear) bad_draft[runs & 1] = runs;
          }
          if (clear) {
#pragma unroll 4
            for (int c = 0; c < D / 8; ++c)
              st_shared_v4(v_smem + (c / 8) * kBoxBytes + row * 128 + (c % 8) * 16, 0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(EDGE_DONE));
          ++edges;
        }
        tc_fence_after_sync();
        if (any_live) {                                   // a warp of padding rows only keeps step
          float s[128];
          {
            uint32_t x[128];
            tmem_ld_32x32b_x128(tmem_s + lane_addr, x);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 128; ++i) s[i] = __uint_as_float(x[i]);
          }
          if (edge) {
            uint32_t sees[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              uint32_t bits = 0;
              const int k0 = key0 + 32 * w;
              if (k0 + 32 <= seq.have) {
                bits = 0xffffffffu;
              } else if (live && k0 < seq.len) {
                const uint8_t* mrow = p.mask + run.b * p.mask_b + t * p.mask_t;
#pragma unroll 1
                for (int i = 0; i < 32; ++i) {
                  const int key = k0 + i, draft = key - seq.have;
                  bool v = draft < 0;
                  if (!v && key < seq.len) v = p.mask != nullptr ? mrow[draft * p.mask_j] != 0 : draft <= t;
                  bits |= static_cast<uint32_t>(v) << i;
                }
              }
              sees[w] = bits;
            }
#pragma unroll
            for (int i = 0; i < 128; ++i)
              if (((sees[i / 32] >> (i % 32)) & 1u) == 0u) s[i] = -INFINITY;
            __syncwarp();
          }
          float mx8[8];
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            float m = fmax3(s[16 * c], s[16 * c + 1], s[16 * c + 2]);
#pragma unroll
            for (int i = 3; i < 15; i += 2) m = fmax3(m, s[16 * c + i], s[16 * c + i + 1]);
            mx8[c] = fmaxf(m, s[16 * c + 15]);
          }
          const float mx = fmax3(fmax3(mx8[0], mx8[1], mx8[2]), fmax3(mx8[3], mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7]));
          const float m_new = fmaxf(m_used, mx * p.scale_log2);
          const bool grow = (m_new - m_used > kRescaleThreshold) || (m_used == -INFINITY && m_new > -INFINITY);
          const bool any_grow = __any_sync(0xffffffffu, grow);
          float alpha = 1.0f;
          if (grow) {
            alpha = (m_used == -INFINITY) ? 0.0f : fast_exp2(m_used - m_new);
            m_used = m_new;
          }
          if (any_grow && j > run.first) {
            // S_FULL of this tile was committed after P V of the last one, so O is quiescent
            l *= alpha;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              uint32_t x[32];
              tmem_ld_32x32b_x32(tmem_o + lane_addr + c * 32, x);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * alpha);
              tmem_st_32x32b_x32(tmem_o + lane_addr + c * 32, x);
            }
          }
          const float neg_m = (m_used == -INFINITY) ? 0.0f : -m_used;
          const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
          const float2 negm2 = make_float2(neg_m, neg_m);
          float2 sum2[4] = {};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t pk[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float2 x = __ffma2_rn(make_float2(s[c * 64 + 2 * i], s[c * 64 + 2 * i + 1]), scale2, negm2);
              const float2 e = make_float2(fast_exp2(x.x), fast_exp2(x.y));
              sum2[i & 3] = __fadd2_rn(sum2[i & 3], e);
              // P is rounded to the input type: it is the tensor cores' operand
              pk[i] = BF16 ? pack_bf16x2(e.x, e.y) : pack_f16x2(e.x, e.y);
            }
            tmem_st_32x32b_x32(tmem_s + lane_addr + c * 32, pk);
          }
          l += ((sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y)) + ((sum2[2].x + sum2[2].y) + (sum2[3].x + sum2[3].y));
          tmem_st_wait();
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(P_FULL));
      }
      // every warp has looked at its rows of V before any reads bad_draft (a tile's V comes after
      // all four warps have left the tile before it, so the phases cannot lie two apart)
      if (ok && (!mbar_wait(bar(PV_DONE), (it - 1) & 1, abort_flag) ||
                 (edges > edges_before && !mbar_wait(bar(EDGE_DONE), (edges - 1) & 1, abort_flag)))) {
        report_status(p.status, 97, 0);
        *abort_flag = 1;
        ok = false;
      }
      if (!ok) break;
      tc_fence_after_sync();
      if (!any_live) continue;

      // the run's result: the output where the run is the whole item, else a partial state
      const bool whole = run.first == 0 && run.last == seq.tiles;
      const int64_t slot = (2 * static_cast<int64_t>(blockIdx.x) + (runs == 0 ? 0 : 1)) * p.tile_rows + row;
      const float inv_l = (l > 0.0f) ? __fdividef(1.0f, l) : (l == 0.0f ? 0.0f : l);
      uint16_t* o_row = p.out + run.b * p.o_b + hq * p.o_h + t * p.o_t;
      const bool by_hand = bad_draft[runs & 1] == runs;
      if (live && !whole) {
        p.ws_ml[2 * slot] = m_used;
        p.ws_ml[2 * slot + 1] = l;
      }
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        float o[32];
        {
          uint32_t x[32];
          tmem_ld_32x32b_x32(tmem_o + lane_addr + c * 32, x);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __uint_as_float(x[i]);
        }
        if (live) {
          if (by_hand) {
            // tokens of the step whose row of V was cleared for being not finite: their share,
            // for the rows that see them
            const int k_end = min(seq.len, run.last * kPaBN);
            for (int key = max(seq.have, run.first * kPaBN); key < k_end; ++key) {
              const int draft = key - seq.have;
              const bool v = p.mask != nullptr ? p.mask[run.b * p.mask_b + t * p.mask_t + draft * p.mask_j] != 0 : draft <= t;
              const int page = p.page_table[run.b * p.page_table_stride + key / p.page_size];
              if (!v || page < 0 || page >= p.num_pages) continue;
              const uint16_t* v_row = p.v + page * p.vc_p + run.head * p.vc_h + (key % p.page_size) * p.vc_s;
              bool bad = false;
              for (int i = 0; i < p.dim; ++i) bad = bad || word_not_finite<BF16>(v_row[i]);
              if (!bad) continue;
              const uint16_t* k_row = p.k + page * p.kc_p + run.head * p.kc_h + (key % p.page_size) * p.kc_s;
              float score = 0.f;
              for (int i = 0; i < p.dim; ++i) score += half_to_float<BF16>(q_row[i]) * half_to_float<BF16>(k_row[i]);
              const float e = fast_exp2(score * p.scale_log2 - m_used);
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (c * 32 + i < p.dim) o[i] += e * half_to_float<BF16>(v_row[c * 32 + i]);
            }
          }
          if (whole) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 16; ++i)
              pk[i] = BF16 ? pack_bf16x2(o[2 * i] * inv_l, o[2 * i + 1] * inv_l) : pack_f16x2(o[2 * i] * inv_l, o[2 * i + 1] * inv_l);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int d0 = c * 32 + 8 * i;
              if (d0 < p.dim) {
                if (p.o_vec) {
                  *reinterpret_cast<uint4*>(o_row + d0) = make_uint4(pk[4 * i], pk[4 * i + 1], pk[4 * i + 2], pk[4 * i + 3]);
                } else {
#pragma unroll
                  for (int k = 0; k < 4; ++k) {
                    o_row[d0 + 2 * k] = static_cast<uint16_t>(pk[4 * i + k] & 0xffff);
                    o_row[d0 + 2 * k + 1] = static_cast<uint16_t>(pk[4 * i + k] >> 16);
                  }
                }
              }
            }
          } else {
            float4* dst = reinterpret_cast<float4*>(p.ws_acc + slot * D + c * 32);
#pragma unroll
            for (int i = 0; i < 8; ++i) dst[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
        }
        __syncwarp();
      }
      tc_fence_before_sync();
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

// Joins the partial states of items that several CTAs share, and clears padding rows.  A warp
// owns a row: lanes read the partial maxima and sums side by side, then every lane adds up its
// columns over the partials.
template <int D, bool BF16>
__global__ void __launch_bounds__(kPaMergeThreads)
paged_attention_join_kernel(const __grid_constant__ PagedParams p) {
  constexpr int kCols = D / 32;              // columns of a lane
  const int lane = threadIdx.x & 31;
  const int per_seq = p.heads_kv * p.row_tiles;
  const int b = blockIdx.y / per_seq, item = blockIdx.y - b * per_seq;
  const int head = item / p.row_tiles, row_tile = item - head * p.row_tiles;
  const int row = blockIdx.x * (kPaMergeThreads / 32) + (threadIdx.x >> 5);
  const int r = row_tile * kPaBM + row;
  const SeqInfo seq = seq_info(p, b);
  const int64_t total = tiles_before(p, p.batch, lane) * per_seq;
  const int64_t first = tiles_before(p, b, lane) * per_seq + static_cast<int64_t>(item) * seq.tiles;
  // the partial states come from the kernel launched just before; every thread waits for it, so
  // that this kernel's end is that one's end too
  pdl_wait();
  if (row >= kPaBM || r >= p.rows) return;
  const int t = r / p.group;
  uint16_t* o_row = p.out + b * p.o_b + static_cast<int64_t>(head * p.group + (r - t * p.group)) * p.o_h + t * p.o_t;
  const int d0 = lane * kCols;
  float o[kCols];
#pragma unroll
  for (int i = 0; i < kCols; ++i) o[i] = 0.f;
  bool store = false;
  if (t < seq.fresh && seq.tiles == 0) {
    store = true;                            // nothing to see: zeros
  } else if (t < seq.fresh) {
    const int c0 = range_owner(first, total, p.ctas), c1 = range_owner(first + seq.tiles - 1, total, p.ctas);
    if (c0 != c1) {
      store = true;
      // only the first of an item's CTAs may have begun with an earlier item
      auto slot = [&](int c) {
        return (2 * static_cast<int64_t>(c) + (range_begin(c, total, p.ctas) >= first ? 0 : 1)) * p.tile_rows + row;
      };
      float m = -INFINITY;
      for (int c = c0 + lane; c <= c1; c += 32)
        if (range_begin(c, total, p.ctas) < range_begin(c + 1, total, p.ctas)) m = fmaxf(m, p.ws_ml[2 * slot(c)]);
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
      float l = 0.f;
      for (int base = c0; base <= c1; base += 32) {
        float f = 0.f;
        int64_t at = 0;
        const int c = base + lane;
        // a range may be empty where there are fewer tiles than CTAs
        if (c <= c1 && range_begin(c, total, p.ctas) < range_begin(c + 1, total, p.ctas)) {
          at = slot(c);
          const float mc = p.ws_ml[2 * at];
          f = (mc == -INFINITY) ? 0.f : exp2f(mc - m);
          l += f * p.ws_ml[2 * at + 1];
        }
        const int n = min(32, c1 - base + 1);
#pragma unroll 4
        for (int k = 0; k < n; ++k) {
          const float fk = __shfl_sync(0xffffffffu, f, k);
          const int64_t ak = __shfl_sync(0xffffffffu, at, k);
          if (fk != 0.f) {
            const float* src = p.ws_acc + ak * D + d0;
#pragma unroll
            for (int i = 0; i < kCols; ++i) o[i] = fmaf(fk, src[i], o[i]);
          }
        }
      }
#pragma unroll
      for (int s = 16; s > 0; s >>= 1) l += __shfl_xor_sync(0xffffffffu, l, s);
      const float inv_l = (l > 0.0f) ? __fdividef(1.0f, l) : (l == 0.0f ? 0.0f : l);
#pragma unroll
      for (int i = 0; i < kCols; ++i) o[i] *= inv_l;
    }
  } else {
    store = p.zero_padding != 0;
  }
  if (!store) return;
#pragma unroll
  for (int i = 0; i < kCols; ++i) {
    if (d0 + i < p.dim) {
      if constexpr (BF16) reinterpret_cast<__nv_bfloat16*>(o_row)[d0 + i] = __float2bfloat16_rn(o[i]);
      else reinterpret_cast<__half*>(o_row)[d0 + i] = __float2half_rn(o[i]);
    }
  }
}

// ---- host ------------------------------------------------------------------------------------

int padded_dim(const b200k_paged_attention_args* a) { return a->head_dim <= 64 ? 64 : 128; }

// CTAs of a call: two per SM, fewer where there cannot be as many key tiles.
int64_t pick_ctas(const b200k_paged_attention_args* a, int sms) {
  const int64_t rows = a->tokens * (a->heads_q / a->heads_kv);
  const int64_t items = a->batch * a->heads_kv * ceil_div(rows, kPaBM);
  const int64_t most = items * ceil_div(static_cast<int64_t>(a->max_pages) * a->page_size, kPaBN);
  const int64_t want = static_cast<int64_t>(sms) * kPaCtasPerSM;
  const int64_t n = most < want ? most : want;
  return n < 1 ? 1 : n;
}

int check_args(const b200k_paged_attention_args* a) {
  if (a == nullptr) return fail(B200K_INVALID_ARG, "null args");
  if (a->batch < 0 || a->tokens < 0 || a->heads_q < 0 || a->heads_kv <= 0 || a->num_pages < 0 || a->max_pages < 0)
    return fail(B200K_INVALID_ARG, "negative dimension, or no key/value heads");
  if (a->heads_q % a->heads_kv != 0) return fail(B200K_INVALID_ARG, "heads_q must be a multiple of heads_kv");
  if (a->dtype != B200K_F16 && a->dtype != B200K_BF16) return fail(B200K_INVALID_ARG, "dtype must be f16 or bf16");
  if (a->head_dim <= 0 || a->head_dim > 128 || a->head_dim % 8 != 0)
    return fail(B200K_UNSUPPORTED, "head_dim must be a multiple of 8 up to 128 (got %d)", a->head_dim);
  if (!(a->qk_scale > 0.f) || a->qk_scale > 3.0e38f)
    return fail(B200K_INVALID_ARG, "qk_scale must be positive and finite");
  if (a->page_size <= 0 || a->page_size % 8 != 0)
    return fail(B200K_UNSUPPORTED, "page_size must be a positive multiple of 8 (got %d)", a->page_size);
  const int64_t limit = int64_t(1) << 30;
  if (a->tokens * a->heads_q > limit || static_cast<int64_t>(a->max_pages) * a->page_size > limit ||
      a->num_pages >= limit || a->batch * a->heads_kv > 65535)
    return fail(B200K_UNSUPPORTED, "more rows, pages or sequences than the kernel counts");
  return B200K_OK;
}

template <int D, bool BF16>
int launch_paged(const CUtensorMap& tk, const CUtensorMap& tv, const PagedParams& p, int64_t items, cudaStream_t stream) {
  constexpr int kSmem = 1024 + 3 * 128 * D * 2 + 256;
  auto kernel = paged_attention_kernel<D, BF16>;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess)
      return fail(B200K_CUDA_ERROR, "cudaFuncSetAttribute(%d): %s", kSmem, cudaGetErrorString(e));
    configured[dev] = true;
  }
  kernel<<<p.ctas, kPaThreads, kSmem, stream>>>(tk, tv, p);
  B200K_CHECK_LAUNCH("paged attention launch");
  const dim3 grid(static_cast<unsigned>(ceil_div(p.tile_rows, kPaMergeThreads / 32)), static_cast<unsigned>(items));
  const cudaError_t e = launch_after_predecessor(paged_attention_join_kernel<D, BF16>, grid, dim3(kPaMergeThreads), 0,
                                                 stream, p);
  if (e != cudaSuccess) return fail(B200K_CUDA_ERROR, "paged attention join launch: %s", cudaGetErrorString(e));
  return B200K_OK;
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
  const int64_t rows = a->tokens * (a->heads_q / a->heads_kv);
  const int64_t tile_rows = rows < kPaBM ? rows : kPaBM;
  return pick_ctas(a, sms) * 2 * tile_rows * (padded_dim(a) + 2) * 4;
}

extern "C" int b200k_paged_attention(const b200k_paged_attention_args* a, b200k_stream stream_) {
  const int rc = check_args(a);
  if (rc != B200K_OK) return rc;
  if (a->batch == 0 || a->tokens == 0 || a->heads_q == 0) return B200K_OK;
  if (!a->q || !a->k_cache || !a->v_cache || !a->out || !a->page_table || !a->cache_lens)
    return fail(B200K_INVALID_ARG, "null pointer");
  for (int64_t s : {a->kc_stride_p, a->kc_stride_h, a->kc_stride_s, a->vc_stride_p, a->vc_stride_h, a->vc_stride_s})
    if (s < 0 || s % 8 != 0) return fail(B200K_UNSUPPORTED, "cache strides must be multiples of 16 bytes");
  if ((reinterpret_cast<uintptr_t>(a->k_cache) | reinterpret_cast<uintptr_t>(a->v_cache)) & 15)
    return fail(B200K_UNSUPPORTED, "caches must be 16-byte aligned");
  if (a->num_pages == 0) return fail(B200K_INVALID_ARG, "the cache has no pages");
  const int sms = current_sm_count();
  if (sms <= 0) return fail(B200K_CUDA_ERROR, "no current CUDA device");
  if (a->workspace == nullptr || (reinterpret_cast<uintptr_t>(a->workspace) & 15) ||
      a->workspace_bytes < b200k_paged_attention_workspace_bytes(a))
    return fail(B200K_INVALID_ARG, "workspace missing, unaligned or too small");

  PagedParams p = {};
  p.q = static_cast<const uint16_t*>(a->q);
  p.k = static_cast<const uint16_t*>(a->k_cache);
  p.v = static_cast<const uint16_t*>(a->v_cache);
  p.out = static_cast<uint16_t*>(a->out);
  p.page_table = a->page_table;
  p.cache_lens = a->cache_lens;
  p.new_lens = a->new_lens;
  p.mask = a->tree_mask;
  p.q_b = a->q_stride_b; p.q_h = a->q_stride_h; p.q_t = a->q_stride_t;
  p.o_b = a->o_stride_b; p.o_h = a->o_stride_h; p.o_t = a->o_stride_t;
  p.kc_p = a->kc_stride_p; p.kc_h = a->kc_stride_h; p.kc_s = a->kc_stride_s;
  p.vc_p = a->vc_stride_p; p.vc_h = a->vc_stride_h; p.vc_s = a->vc_stride_s;
  p.mask_b = a->mask_stride_b; p.mask_t = a->mask_stride_t; p.mask_j = a->mask_stride_j;
  p.page_table_stride = a->page_table_stride;
  p.num_pages = a->num_pages;
  p.batch = static_cast<int>(a->batch);
  p.tokens = static_cast<int>(a->tokens);
  p.heads_kv = static_cast<int>(a->heads_kv);
  p.group = static_cast<int>(a->heads_q / a->heads_kv);
  p.dim = a->head_dim;
  p.rows = p.tokens * p.group;
  p.row_tiles = static_cast<int>(ceil_div(p.rows, kPaBM));
  p.tile_rows = p.rows < kPaBM ? p.rows : kPaBM;
  p.page_size = a->page_size;
  p.max_pages = a->max_pages;
  // slots per TMA box: the largest power of two (8 to 128) that divides a page, so that a box
  // lies in one page and starts on a whole eight-row swizzle atom of the tile
  p.box_rows = 8;
  while (p.box_rows < kPaBN && a->page_size % (p.box_rows * 2) == 0) p.box_rows *= 2;
  p.ctas = static_cast<int>(pick_ctas(a, sms));
  const auto vec = [](const void* base, int64_t sb, int64_t sh, int64_t st) {
    return (reinterpret_cast<uintptr_t>(base) & 15) == 0 && sb % 8 == 0 && sh % 8 == 0 && st % 8 == 0;
  };
  p.q_vec = vec(a->q, p.q_b, p.q_h, p.q_t);
  p.o_vec = vec(a->out, p.o_b, p.o_h, p.o_t);
  p.zero_padding = a->zero_padding;
  p.scale_log2 = a->qk_scale * 1.4426950408889634f;
  const int d = padded_dim(a);
  p.ws_acc = static_cast<float*>(a->workspace);
  p.ws_ml = p.ws_acc + static_cast<int64_t>(p.ctas) * 2 * p.tile_rows * d;
  p.status = device_status_word();

  const CUtensorMapDataType dt =
      a->dtype == B200K_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  CUtensorMap tk, tv;
  if (!encode_tmap_4d(&tk, dt, a->k_cache, a->head_dim, a->page_size, a->heads_kv, a->num_pages, p.kc_s * 2, p.kc_h * 2,
                      p.kc_p * 2, 64, p.box_rows, 1, 1, CU_TENSOR_MAP_SWIZZLE_128B) ||
      !encode_tmap_4d(&tv, dt, a->v_cache, a->head_dim, a->page_size, a->heads_kv, a->num_pages, p.vc_s * 2, p.vc_h * 2,
                      p.vc_p * 2, 64, p.box_rows, 1, 1, CU_TENSOR_MAP_SWIZZLE_128B))
    return B200K_INVALID_ARG;
  const int64_t items = a->batch * a->heads_kv * p.row_tiles;
  if (items > 65535) return fail(B200K_UNSUPPORTED, "more row tiles than the kernel counts");
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const bool bf16 = a->dtype == B200K_BF16;
  if (d == 128)
    return bf16 ? launch_paged<128, true>(tk, tv, p, items, stream) : launch_paged<128, false>(tk, tv, p, items, stream);
  return bf16 ? launch_paged<64, true>(tk, tv, p, items, stream) : launch_paged<64, false>(tk, tv, p, items, stream);
}

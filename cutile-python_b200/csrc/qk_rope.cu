// Norm of every query / key head and rotation by position in one pass over the rows, its
// gradient, and the same pass with a paged cache as its destination (a serving step's append).
//
//   n = x * rsqrt(mean(x^2) + eps) * w          (weight absent: n = x)
//   y = Rot(p) n                                 p: the token's position
// Rot(p) turns rotary_dim / 2 pairs of the row by the angles of table row p: half split
// (i, i + R / 2) or interleaved (2 i, 2 i + 1); the other D - R values pass through.  Backward,
// with u = x * rsqrt(..), g = Rot(p)^T dy, h = g * w:
//   dw = sum over rows of g * u                  dx = rsqrt(..) * (h - u * mean(h * u))
//
// All of it is HBM-bound: about twenty operations per element that is read and written once.
// A group of 4, 8 or 16 lanes owns one row, a lane 16 of its values in 16-byte pieces chosen so
// that both halves of every rotated pair sit in the same lane: no exchange but the sum of squares.
// A group keeps one token and walks its heads, so the cosines, sines and weights of its columns
// are fetched once for several rows.  Rows come through shared memory by asynchronous copies,
// which keep 64 KB (forward) to 160 KB (backward) per SM in flight without holding registers.
// Everything is computed in fp32 and rounded once, at the store.
//
// Measured (4 x 4096 tokens, 32 + 8 heads of 128, bf16; of the 6.55 TB/s a copy reaches): forward 63 us
// = 5.4 TB/s (registers instead of shared memory 69.5 us; the table's reads and the two passes of a
// block, fetch and store, are what is left); backward 89 us = 5.7 TB/s (199 us with rows in
// registers, 101 with scalar fp32 and weights in conflicting banks); append of 8 x 2048 ragged
// tokens 61 us = 5.0 TB/s; a decode step of 32 sequences 3.0 us, an append step of 64 3.9 us.

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "host.h"

namespace b200k {
namespace {

constexpr int kRopeThreads = 128;
constexpr int kMaxHeads = 65536;
constexpr int kBackwardStages = 5;      // rows of 16-bit values on their way to a lane group
constexpr int kBackwardMinBlocks = 4;

// One tensor of a call: (batch, heads, tokens, D) rows in, rows out.
struct RopeSide {
  const void* x;
  const void* dy;        // backward only: gradient of the output rows
  void* y;               // output rows; backward: gradient of x
  const void* w;         // (D) norm weight or null
  float* dw;             // backward: this side's partial sums, (blocks, D)
  int64_t x_b, x_h, x_t, dy_b, dy_h, dy_t, y_b, y_h, y_t;   // elements; paged output: page, head, slot
  int heads;
  int chunks;            // ceil(heads / heads per group)
  int per;               // backward: heads per group, the chunks as even as they come
  int rotate;
  int paged;
  int zero_padding;      // tokens behind new_lens[b] give zero rows (else they are left alone)
  int first_block, blocks;
};

struct RopeParams {
  RopeSide side[3];
  int sides;
  int dim, units, pairs, rotary;    // pairs: units that are rotated
  int interleaved, w_is_f32, w_vec;   // w_vec: the weights start on 16-byte boundaries
  int heads_per_group;
  int64_t tokens, total_tokens;     // per sequence, of all sequences
  const float* cos;
  const float* sin;
  int64_t table_stride, table_rows;
  const void* positions;            // null: token index (or cache_lens[b] + token index)
  int64_t pos_b, pos_t;
  int pos_is_i64;
  const int* cache_lens;
  const int* new_lens;
  const int* page_table;
  int64_t page_table_stride;
  int page_size, max_pages;
  int64_t num_pages;
  float eps, inv_dim;
  int* status;
};

template <typename T> __device__ __forceinline__ float rope_to_f32(T v);
template <> __device__ __forceinline__ float rope_to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float rope_to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float rope_to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T rope_from_f32(float v);
template <> __device__ __forceinline__ float rope_from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half rope_from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 rope_from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// A lane's values come in pieces of 16 bytes: two of eight 16-bit values or four of four fp32.
template <typename T> struct Piece {
  static constexpr int kValues = 16 / sizeof(T), kCount = 16 / kValues;
};

// A lane's sixteen values as the pairs (lo, hi) that a rotation turns, two pairs to a register
// pair: fp32 products and sums are issued two at a time.  Half split: lo is the first half of the
// values, hi the second.  Interleaved: lo the even, hi the odd ones.
struct Pairs {
  float2 lo[4], hi[4];
};
template <bool INTER>
__device__ __forceinline__ Pairs to_pairs(const float (&v)[16]) {
  Pairs r;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (INTER) {
      r.lo[k] = make_float2(v[4 * k], v[4 * k + 2]);
      r.hi[k] = make_float2(v[4 * k + 1], v[4 * k + 3]);
    } else {
      r.lo[k] = make_float2(v[2 * k], v[2 * k + 1]);
      r.hi[k] = make_float2(v[8 + 2 * k], v[8 + 2 * k + 1]);
    }
  }
  return r;
}
template <bool INTER>
__device__ __forceinline__ void from_pairs(const Pairs& r, float (&v)[16]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (INTER) {
      v[4 * k] = r.lo[k].x; v[4 * k + 1] = r.hi[k].x; v[4 * k + 2] = r.lo[k].y; v[4 * k + 3] = r.hi[k].y;
    } else {
      v[2 * k] = r.lo[k].x; v[2 * k + 1] = r.lo[k].y;
      v[8 + 2 * k] = r.hi[k].x; v[8 + 2 * k + 1] = r.hi[k].y;
    }
  }
}

// The values of a piece.
template <typename T>
__device__ __forceinline__ void unpack_piece(const uint4& q, float* f) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      f[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store_piece(T* p, const float* f) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(f[i]);
    else w[i] = std::is_same<T, __half>::value ? pack_f16x2(f[2 * i], f[2 * i + 1]) : pack_bf16x2(f[2 * i], f[2 * i + 1]);
  }
  if constexpr (VEC) {
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int i = 0; i < Piece<T>::kValues; ++i) p[i] = e[i];
  }
}

// Norm weights of a lane's columns; zeros where it has none.
template <typename T, bool INTER, typename Columns>
__device__ __forceinline__ Pairs load_weights(const RopeParams& p, const void* w, const Columns& col) {
  constexpr int kValues = Piece<T>::kValues;
  float v[16];
#pragma unroll
  for (int q = 0; q < Piece<T>::kCount; ++q) {
    float* f = v + q * kValues;
#pragma unroll
    for (int i = 0; i < kValues; ++i) f[i] = 0.f;
    if (!col.has[q]) continue;
    if (p.w_vec && !p.w_is_f32) {
      unpack_piece<T>(*reinterpret_cast<const uint4*>(static_cast<const T*>(w) + col.at[q]), f);
    } else if (p.w_vec) {
#pragma unroll
      for (int i = 0; i < kValues; i += 4)
        unpack_piece<float>(*reinterpret_cast<const uint4*>(static_cast<const float*>(w) + col.at[q] + i), f + i);
    } else {
#pragma unroll 1
      for (int i = 0; i < kValues; ++i) {
        const int at = col.at[q] + i;
        const float x = p.w_is_f32 ? static_cast<const float*>(w)[at] : rope_to_f32<T>(static_cast<const T*>(w)[at]);
#pragma unroll
        for (int j = 0; j < kValues; ++j)
          if (j == i) f[j] = x;
      }
    }
  }
  return to_pairs<INTER>(v);
}

// Cosines and sines of the lane's pairs; with `minus` the negated sines.
struct Angles {
  float2 c[4], s[4], minus[4];
};
// (lo, hi) -> (lo c - hi s, hi c + lo s); BACK turns the other way.
template <bool BACK>
__device__ __forceinline__ void rotate_pairs(Pairs& r, const Angles& g) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 lo = r.lo[k], hi = r.hi[k];
    r.lo[k] = __ffma2_rn(lo, g.c[k], __fmul2_rn(hi, BACK ? g.s[k] : g.minus[k]));
    r.hi[k] = __ffma2_rn(hi, g.c[k], __fmul2_rn(lo, BACK ? g.minus[k] : g.s[k]));
  }
}

template <int GS>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = GS / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Which columns a lane holds: those of its pieces, `unit` the lane's number in the row's group.
// 16-bit rows: pieces at 8 u and R / 2 + 8 u (half split), or side by side (interleaved).  fp32
// rows: piece q at q R / 4 + 4 u, so that a group's lanes read and write 16 neighbouring bytes
// each (32 bytes of a lane side by side cost twice the sectors: 107 us against 79 for 12749 tokens
// of 36 heads of 128).  Without a piece: column 0, so that addresses stay in the row.
template <typename T>
struct LaneColumns {
  int at[Piece<T>::kCount];
  bool has[Piece<T>::kCount];
  bool rotated;
};

template <typename T, bool INTER>
__device__ __forceinline__ LaneColumns<T> lane_columns(const RopeParams& p, int unit) {
  constexpr int kCount = Piece<T>::kCount, kValues = Piece<T>::kValues;
  LaneColumns<T> c;
  c.rotated = unit < p.pairs;
#pragma unroll
  for (int q = 0; q < kCount; ++q) {
    if (c.rotated) {
      c.at[q] = kCount == 4 ? q * 4 * p.pairs + 4 * unit : (INTER ? unit * 16 + 8 * q : unit * 8 + q * (p.rotary / 2));
      c.has[q] = true;
    } else {
      const int rest = p.units - p.pairs, u = unit - p.pairs;   // lanes of the columns that pass through
      c.at[q] = p.rotary + (kCount == 4 ? q * kValues * rest + kValues * u : u * 16 + 8 * q);
      c.has[q] = unit < p.units && c.at[q] < p.dim;
      if (!c.has[q]) c.at[q] = 0;
    }
  }
  return c;
}

__device__ __forceinline__ int64_t position_of(const RopeParams& p, int64_t b, int64_t t) {
  if (p.positions != nullptr) {
    const int64_t at = b * p.pos_b + t * p.pos_t;
    return p.pos_is_i64 ? static_cast<const int64_t*>(p.positions)[at] : static_cast<const int*>(p.positions)[at];
  }
  return (p.cache_lens != nullptr ? p.cache_lens[b] : 0) + t;
}

// Cosines and sines of a position for the lane's pairs.  A position outside the table is recorded
// in the status word and makes the rotated values NaN: nothing is read out of range.
template <typename T, bool INTER>
__device__ __forceinline__ void load_angles(const RopeParams& p, int64_t pos, int64_t t, int unit,
                                            const LaneColumns<T>& col, Angles& g) {
  if (pos < 0 || pos >= p.table_rows) {
    if (unit == 0) report_bad_index(p.status, kRolePosition, t);
    const float nan = __int_as_float(0x7fc00000);
#pragma unroll
    for (int k = 0; k < 4; ++k) g.c[k] = g.s[k] = g.minus[k] = make_float2(nan, nan);
    return;
  }
  const float* cr = p.cos + pos * p.table_stride;
  const float* sr = p.sin + pos * p.table_stride;
  if constexpr (Piece<T>::kCount == 4 && INTER) {   // two of the rotation's pairs to a piece
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      g.c[k] = *reinterpret_cast<const float2*>(cr + col.at[k] / 2);
      g.s[k] = *reinterpret_cast<const float2*>(sr + col.at[k] / 2);
    }
  } else {                                          // four side by side
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int from = Piece<T>::kCount == 4 ? col.at[i] : unit * 8 + 4 * i;
      const float4 c = *reinterpret_cast<const float4*>(cr + from), s = *reinterpret_cast<const float4*>(sr + from);
      g.c[2 * i] = make_float2(c.x, c.y);
      g.c[2 * i + 1] = make_float2(c.z, c.w);
      g.s[2 * i] = make_float2(s.x, s.y);
      g.s[2 * i + 1] = make_float2(s.z, s.w);
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) g.minus[k] = make_float2(-g.s[k].x, -g.s[k].y);
}

// A lane's pieces of a row (zeros where it has none), fetched into its own slots of shared memory:
// [piece][thread], so neighbouring threads hit neighbouring banks.  With VEC the copies are
// asynchronous and cost no registers while they are in flight; a thread waits for its own copies
// only, so no barrier is needed.
template <typename T, bool VEC>
__device__ __forceinline__ void stage_row(uint4* slot, const T* row, const LaneColumns<T>& col, bool on) {
#pragma unroll
  for (int q = 0; q < Piece<T>::kCount; ++q) {
    const T* src = row + col.at[q];
    if constexpr (VEC) {
      const uint32_t dst = smem_u32(slot + q * kRopeThreads);
      // a source size of 0 fills the slot with zeros and reads nothing
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(src)),
                   "r"(col.has[q] && on ? 16 : 0)
                   : "memory");
    } else {
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      T* e = reinterpret_cast<T*>(&v);
      if (col.has[q] && on) {
#pragma unroll
        for (int i = 0; i < Piece<T>::kValues; ++i) e[i] = src[i];
      }
      slot[q * kRopeThreads] = v;
    }
  }
}
__device__ __forceinline__ void stage_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void stage_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <typename T, bool INTER>
__device__ __forceinline__ Pairs read_staged(const uint4* slot) {
  float v[16];
#pragma unroll
  for (int q = 0; q < Piece<T>::kCount; ++q) unpack_piece<T>(slot[q * kRopeThreads], v + q * Piece<T>::kValues);
  return to_pairs<INTER>(v);
}
template <typename T, bool INTER, bool VEC>
__device__ __forceinline__ void store_pairs(T* row, const LaneColumns<T>& col, const Pairs& r) {
  float v[16];
  from_pairs<INTER>(r, v);
#pragma unroll
  for (int q = 0; q < Piece<T>::kCount; ++q)
    if (col.has[q]) store_piece<T, VEC>(row + col.at[q], v + q * Piece<T>::kValues);
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// Forward.  grid.x: one block per kRopeThreads / GS tokens; grid.y: (side, chunk of heads).  All
// rows of the chunk are requested at once, then normed and rotated batch by batch as they come.
template <typename T> struct ForwardRows {          // heads a group walks; 16 KB of shared memory
  static constexpr int kMax = sizeof(T) == 4 ? 2 : 4;
};

template <typename T, int GS, bool INTER, bool VEC>
__global__ void __launch_bounds__(kRopeThreads)
qk_rope_kernel(const __grid_constant__ RopeParams p) {
  constexpr int kRows = ForwardRows<T>::kMax, kBatch = kRows / 2;
  constexpr int kSlot = Piece<T>::kCount * kRopeThreads;
  __shared__ uint4 stage[kRows * kSlot];
  uint4* mine = stage + threadIdx.x;
  const int unit = threadIdx.x % GS;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * (kRopeThreads / GS) + threadIdx.x / GS;
  int chunk = blockIdx.y, which = 0;
  while (which + 1 < p.sides && chunk >= p.side[which].chunks) chunk -= p.side[which++].chunks;
  const RopeSide& sd = p.side[which];
  const bool live = n < p.total_tokens;
  const int64_t b = live ? n / p.tokens : 0, t = live ? n - b * p.tokens : 0;
  const LaneColumns<T> col = lane_columns<T, INTER>(p, unit);
  const bool padded = live && p.new_lens != nullptr && t >= p.new_lens[b];

  const T* x = static_cast<const T*>(sd.x) + b * sd.x_b + t * sd.x_t;
  const int h_begin = chunk * p.heads_per_group;
  const int rows = min(sd.heads - h_begin, p.heads_per_group);   // at most kRows
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const bool on = live && !padded && u < rows;
    stage_row<T, VEC>(mine + u * kSlot, x + (on ? h_begin + u : 0) * sd.x_h, col, on);
    if (u == kBatch - 1) stage_commit();
  }
  stage_commit();

  // where this token's rows go
  int64_t out = b * sd.y_b + t * sd.y_t;
  bool store = live && (!padded || sd.zero_padding);
  if (sd.paged && store) {
    const int64_t at = static_cast<int64_t>(p.cache_lens[b]) + t;
    const int64_t entry = at >= 0 ? at / p.page_size : -1;
    int64_t page = -1;
    if (entry >= 0 && entry < p.max_pages) page = p.page_table[b * p.page_table_stride + entry];
    if (page < 0 || page >= p.num_pages) {
      if (unit == 0) report_bad_index(p.status, kRolePage, b);
      store = false;
    } else {
      out = page * sd.y_b + (at - entry * p.page_size) * sd.y_t;
    }
  }
  Angles angles;
  const bool rotate = sd.rotate != 0 && col.rotated && store && !padded;
  if (rotate) load_angles<T, INTER>(p, position_of(p, b, t), t, unit, col, angles);
  const bool norm = sd.w != nullptr;
  Pairs w;
  if (norm) w = load_weights<T, INTER>(p, sd.w, col);

  T* y = static_cast<T*>(sd.y) + out + h_begin * sd.y_h;
#pragma unroll
  for (int batch = 0; batch < 2; ++batch) {
    if (batch == 0) stage_wait<1>();
    else stage_wait<0>();
#pragma unroll
    for (int v = 0; v < kBatch; ++v) {
      const int u = batch * kBatch + v;
      if (u >= rows) break;                      // the same for the whole block
      Pairs r = read_staged<T, INTER>(mine + u * kSlot);
      if (norm) {
        float2 sq = both(0.f), sq2 = both(0.f);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          sq = __ffma2_rn(r.lo[k], r.lo[k], sq);
          sq2 = __ffma2_rn(r.hi[k], r.hi[k], sq2);
        }
        sq = __fadd2_rn(sq, sq2);
        const float2 inv = both(rsqrtf(group_sum<GS>(sq.x + sq.y) * p.inv_dim + p.eps));
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          r.lo[k] = __fmul2_rn(r.lo[k], __fmul2_rn(inv, w.lo[k]));
          r.hi[k] = __fmul2_rn(r.hi[k], __fmul2_rn(inv, w.hi[k]));
        }
      }
      if (rotate) rotate_pairs<false>(r, angles);
      if (padded) {
#pragma unroll
        for (int k = 0; k < 4; ++k) r.lo[k] = r.hi[k] = both(0.f);
      }
      if (store) store_pairs<T, INTER, VEC>(y + u * sd.y_h, col, r);
    }
  }
}

// Backward.  Block-strided over (token, chunk of heads) of one side, kStages rows of x and dy
// ahead of the row in hand; every lane sums its columns' weight gradient over its rows in fp32,
// the block's groups are summed through shared memory in a fixed order and the block leaves one
// partial row: the result does not depend on the order in which blocks run.
template <typename T, int GS, bool INTER, bool VEC>
__global__ void __launch_bounds__(kRopeThreads, kBackwardMinBlocks)
qk_rope_backward_kernel(const __grid_constant__ RopeParams p) {
  constexpr int kStages = sizeof(T) == 4 ? kBackwardStages / 2 : kBackwardStages;
  constexpr int kGroups = kRopeThreads / GS;
  constexpr int kSlot = Piece<T>::kCount * kRopeThreads;
  __shared__ uint4 stage[kStages * 2 * kSlot];
  __shared__ float4 weights[4][GS];   // [piece][unit]: neighbouring lanes read neighbouring banks
  pdl_launch_dependents();   // the sum of the partial rows may be set up now; it waits for this grid
  uint4* mine = stage + threadIdx.x;
  const int unit = threadIdx.x % GS, group = threadIdx.x / GS;
  int which = 0;
  while (which + 1 < p.sides && static_cast<int>(blockIdx.x) >= p.side[which + 1].first_block) ++which;
  const RopeSide& sd = p.side[which];
  const int block = blockIdx.x - sd.first_block;
  const LaneColumns<T> col = lane_columns<T, INTER>(p, unit);
  const bool norm = sd.w != nullptr;
  const bool rotated = col.rotated && sd.rotate != 0;
  Pairs grad;                     // weight gradient of the lane's columns
#pragma unroll
  for (int k = 0; k < 4; ++k) grad.lo[k] = grad.hi[k] = both(0.f);

  // a group's rows: the heads of the chunk that is its task 0, those of task 1, ...; the same number
  // for every group of the block (the sums below are warp-collective)
  const int tasks = static_cast<int>(p.total_tokens) * sd.chunks;   // at most 2^30, checked at the launch
  const int step = sd.blocks * kGroups, first = block * kGroups + group;
  const int per = sd.per;
  const int rounds = (tasks + step - 1) / step;
  struct Place {
    int b, t, h, heads;           // sequence, token, first head, heads of this chunk (0: no such task)
  };
  auto place_of = [&](int round) {
    const int task = round * step + first;
    Place q = {0, 0, 0, 0};
    if (task < tasks && round < rounds) {
      const int n = task / sd.chunks, tokens = static_cast<int>(p.tokens);
      q.h = (task - n * sd.chunks) * per;
      q.heads = min(sd.heads - q.h, per);
      q.b = n / tokens;
      q.t = n - q.b * tokens;
    }
    return q;
  };
  const T* xs = static_cast<const T*>(sd.x);
  const T* dys = static_cast<const T*>(sd.dy);
  int fetch_heads = 0;            // of the chunk that is being requested
  int fetch_round = 0, fetch_u = 0;
  auto request = [&](uint4* slot) {
    const int u = fetch_u;
    if (u == 0) {
      const Place q = place_of(fetch_round);
      fetch_heads = q.heads;
      xs = static_cast<const T*>(sd.x) + q.b * sd.x_b + q.t * sd.x_t + q.h * sd.x_h;
      dys = static_cast<const T*>(sd.dy) + q.b * sd.dy_b + q.t * sd.dy_t + q.h * sd.dy_h;
    }
    stage_row<T, VEC>(slot, xs, col, u < fetch_heads);
    stage_row<T, VEC>(slot + kSlot, dys, col, u < fetch_heads);
    if (u + 1 < fetch_heads) {
      xs += sd.x_h;
      dys += sd.dy_h;
    }
    if (++fetch_u == per) {
      fetch_u = 0;
      ++fetch_round;
    }
    stage_commit();
  };
  for (int i = 0; i < kStages - 1; ++i) request(mine + i * 2 * kSlot);
  if (norm && threadIdx.x < GS) {
    const Pairs v = load_weights<T, INTER>(p, sd.w, col);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      weights[k][unit] = make_float4(v.lo[2 * k].x, v.lo[2 * k].y, v.lo[2 * k + 1].x, v.lo[2 * k + 1].y);
      weights[2 + k][unit] = make_float4(v.hi[2 * k].x, v.hi[2 * k].y, v.hi[2 * k + 1].x, v.hi[2 * k + 1].y);
    }
  }
  __syncthreads();

  int use = 0, fill = kStages - 1;
  for (int round = 0; round < rounds; ++round) {
    const Place here = place_of(round);
    const int heads = here.heads;
    const bool turns = heads > 0 && rotated;
    Angles angles;
    if (turns) load_angles<T, INTER>(p, position_of(p, here.b, here.t), here.t, unit, col, angles);
    T* dx = static_cast<T*>(sd.y) + here.b * sd.y_b + here.t * sd.y_t + here.h * sd.y_h;
    for (int u = 0; u < per; ++u) {
      request(mine + fill * 2 * kSlot);
      fill = fill + 1 == kStages ? 0 : fill + 1;
      stage_wait<kStages - 1>();
      const uint4* slot = mine + use * 2 * kSlot;
      use = use + 1 == kStages ? 0 : use + 1;
      Pairs g = read_staged<T, INTER>(slot + kSlot);
      if (turns) rotate_pairs<true>(g, angles);
      if (norm) {
        const Pairs x = read_staged<T, INTER>(slot);
        Pairs gx, w;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float4 l = weights[k][unit], h = weights[2 + k][unit];
          w.lo[2 * k] = make_float2(l.x, l.y);
          w.lo[2 * k + 1] = make_float2(l.z, l.w);
          w.hi[2 * k] = make_float2(h.x, h.y);
          w.hi[2 * k + 1] = make_float2(h.z, h.w);
        }
        float2 sq[2] = {both(0.f), both(0.f)}, dot[2] = {both(0.f), both(0.f)};   // sum x^2, sum x g w
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          gx.lo[k] = __fmul2_rn(g.lo[k], x.lo[k]);
          gx.hi[k] = __fmul2_rn(g.hi[k], x.hi[k]);
          sq[0] = __ffma2_rn(x.lo[k], x.lo[k], sq[0]);
          sq[1] = __ffma2_rn(x.hi[k], x.hi[k], sq[1]);
          dot[0] = __ffma2_rn(gx.lo[k], w.lo[k], dot[0]);
          dot[1] = __ffma2_rn(gx.hi[k], w.hi[k], dot[1]);
        }
        const float2 sqs = __fadd2_rn(sq[0], sq[1]), dots = __fadd2_rn(dot[0], dot[1]);
        const float r = rsqrtf(group_sum<GS>(sqs.x + sqs.y) * p.inv_dim + p.eps);
        const float along = group_sum<GS>(dots.x + dots.y) * p.inv_dim * r * r;   // mean(h u) / (x / u)
        // rows that are not there are zeros and add nothing
        const float2 r2 = both(u < heads ? r : 0.f), m2 = both(u < heads ? -r * along : 0.f);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          grad.lo[k] = __ffma2_rn(gx.lo[k], r2, grad.lo[k]);
          grad.hi[k] = __ffma2_rn(gx.hi[k], r2, grad.hi[k]);
          g.lo[k] = __ffma2_rn(x.lo[k], m2, __fmul2_rn(__fmul2_rn(g.lo[k], w.lo[k]), r2));
          g.hi[k] = __ffma2_rn(x.hi[k], m2, __fmul2_rn(__fmul2_rn(g.hi[k], w.hi[k]), r2));
        }
      }
      if (u < heads) {
        store_pairs<T, INTER, VEC>(dx, col, g);
        dx += sd.y_h;
      }
    }
  }
  stage_wait<0>();

  if (!norm) return;   // the same for the whole block
  float (*sums)[GS * 16 + 1] = reinterpret_cast<float (*)[GS * 16 + 1]>(stage);
  static_assert(sizeof(stage) >= kGroups * (GS * 16 + 1) * 4, "the stages are reused for the sums");
  __syncthreads();
  {
    float v[16];
    from_pairs<INTER>(grad, v);
#pragma unroll
    for (int k = 0; k < 16; ++k) sums[group][unit * 16 + k] = v[k];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < GS * 16; i += kRopeThreads) {
    const LaneColumns<T> lc = lane_columns<T, INTER>(p, i / 16);
    constexpr int kValues = Piece<T>::kValues;
    int column = -1;
#pragma unroll
    for (int q = 0; q < Piece<T>::kCount; ++q)
      if (q == i % 16 / kValues && lc.has[q]) column = lc.at[q] + i % kValues;
    if (column >= 0) {
      float v = 0.f;
#pragma unroll 8
      for (int g = 0; g < kGroups; ++g) v += sums[g][i];
      sd.dw[static_cast<int64_t>(block) * p.dim + column] = v;
    }
  }
}

// Sum of the partial rows: a block takes 32 columns of one side, 32 threads per column.
struct WeightGradParams {
  const float* partial[2];
  void* out[2];
  int blocks[2];
  int dim;
};

template <typename W>
__global__ void __launch_bounds__(1024)
weight_grad_sum_kernel(const __grid_constant__ WeightGradParams p) {
  const int lane = threadIdx.x % 32, row = threadIdx.x / 32;
  const int col = blockIdx.x * 32 + lane;
  const int which = blockIdx.y;
  __shared__ float sums[32][33];
  pdl_wait();
  float v = 0.f;
  if (col < p.dim) {
#pragma unroll 4
    for (int i = row; i < p.blocks[which]; i += 32) v += p.partial[which][static_cast<int64_t>(i) * p.dim + col];
  }
  sums[row][lane] = v;
  __syncthreads();
  // lane of warp `row` = the partial sum number; the warp owns column `row` of the block
  float total = sums[lane][row];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  const int out_col = blockIdx.x * 32 + row;
  if (lane == 0 && out_col < p.dim && p.out[which] != nullptr)
    static_cast<W*>(p.out[which])[out_col] = rope_from_f32<W>(total);
}

// ---- host ----------------------------------------------------------------------------------

bool multiple_of_16_bytes(const void* base, int64_t elem, std::initializer_list<int64_t> strides) {
  if (reinterpret_cast<uintptr_t>(base) & 15) return false;
  for (int64_t s : strides)
    if ((s * elem) & 15) return false;
  return true;
}

bool side_vectors(const RopeSide& s, int64_t elem) {
  return multiple_of_16_bytes(s.x, elem, {s.x_b, s.x_h, s.x_t}) &&
         multiple_of_16_bytes(s.y, elem, {s.y_b, s.y_h, s.y_t}) &&
         (s.dy == nullptr || multiple_of_16_bytes(s.dy, elem, {s.dy_b, s.dy_h, s.dy_t}));
}

int weight_vectors(const RopeParams& p) {
  uintptr_t bits = 0;
  for (int i = 0; i < p.sides; ++i) bits |= reinterpret_cast<uintptr_t>(p.side[i].w);
  return (bits & 15) == 0;
}

// Lanes per row: the smallest group whose lanes hold 16 values each.
int lanes_per_row(int units) { return units <= 4 ? 4 : (units <= 8 ? 8 : 16); }

// Heads a group walks with one token's angles, a power of two: as many as leave every SM about a
// thousand threads.
int pick_heads_per_group(int64_t total_tokens, int heads_all, int lanes, int most, int sms) {
  int per = most;
  while (per > 1 && total_tokens * lanes * ceil_div(heads_all, per) < static_cast<int64_t>(sms) * 1024) per /= 2;
  return per;
}

int fill_geometry(RopeParams& p, int64_t batch, int64_t tokens, int dim, int rotary, int interleaved,
                  const float* cos, const float* sin, int64_t table_stride, int64_t table_rows, int w_dtype,
                  int dtype, float eps) {
  if (batch < 0 || tokens < 0) return fail(B200K_INVALID_ARG, "negative dimension");
  if (dtype != B200K_F16 && dtype != B200K_BF16 && dtype != B200K_F32)
    return fail(B200K_INVALID_ARG, "dtype must be f16, bf16 or f32");
  if (w_dtype != dtype && w_dtype != B200K_F32)
    return fail(B200K_INVALID_ARG, "norm weights must have the rows' dtype or be f32");
  if (dim <= 0 || dim > 256 || dim % 8 != 0)
    return fail(B200K_UNSUPPORTED, "head_dim must be a multiple of 8 up to 256 (got %d)", dim);
  if (rotary < 0 || rotary > dim || rotary % 16 != 0)
    return fail(B200K_UNSUPPORTED, "rotary_dim must be a multiple of 16 up to head_dim (got %d)", rotary);
  if (rotary > 0) {
    if (cos == nullptr || sin == nullptr) return fail(B200K_INVALID_ARG, "null rotation table");
    if (table_rows <= 0 || table_stride < rotary / 2)
      return fail(B200K_INVALID_ARG, "rotation table of %lld rows, row stride %lld", (long long)table_rows,
                  (long long)table_stride);
    if (((reinterpret_cast<uintptr_t>(cos) | reinterpret_cast<uintptr_t>(sin)) & 15) || table_stride % 4 != 0)
      return fail(B200K_UNSUPPORTED, "rotation table rows must start on 16-byte boundaries");
  }
  if (!(eps >= 0.f)) return fail(B200K_INVALID_ARG, "eps must be >= 0");
  p.dim = dim;
  p.rotary = rotary;
  p.pairs = rotary / 16;
  p.units = p.pairs + (dim - rotary + 15) / 16;
  p.interleaved = interleaved;
  p.w_is_f32 = w_dtype == B200K_F32;
  p.tokens = tokens;
  p.total_tokens = batch * tokens;
  p.cos = cos;
  p.sin = sin;
  p.table_stride = table_stride;
  p.table_rows = table_rows;
  p.eps = eps;
  p.inv_dim = 1.0f / static_cast<float>(dim);
  p.status = device_status_word();
  return B200K_OK;
}

template <typename T, int GS>
int launch_rope(const RopeParams& p, bool vec, dim3 grid, cudaStream_t stream) {
  if (p.interleaved) {
    if (vec) qk_rope_kernel<T, GS, true, true><<<grid, kRopeThreads, 0, stream>>>(p);
    else qk_rope_kernel<T, GS, true, false><<<grid, kRopeThreads, 0, stream>>>(p);
  } else {
    if (vec) qk_rope_kernel<T, GS, false, true><<<grid, kRopeThreads, 0, stream>>>(p);
    else qk_rope_kernel<T, GS, false, false><<<grid, kRopeThreads, 0, stream>>>(p);
  }
  B200K_CHECK_LAUNCH("qk_rope launch");
  return B200K_OK;
}

template <typename T>
int launch_rope_type(const RopeParams& p, int lanes, bool vec, dim3 grid, cudaStream_t stream) {
  if (lanes == 4) return launch_rope<T, 4>(p, vec, grid, stream);
  if (lanes == 8) return launch_rope<T, 8>(p, vec, grid, stream);
  return launch_rope<T, 16>(p, vec, grid, stream);
}

int launch_forward(RopeParams& p, int dtype, cudaStream_t stream) {
  const int sms = current_sm_count();
  if (sms <= 0) return fail(B200K_CUDA_ERROR, "no current CUDA device");
  const int lanes = lanes_per_row(p.units);
  int heads_all = 0;
  bool vec = true;
  for (int i = 0; i < p.sides; ++i) {
    heads_all += p.side[i].heads;
    vec = vec && side_vectors(p.side[i], dtype == B200K_F32 ? 4 : 2);
  }
  p.w_vec = weight_vectors(p);
  p.heads_per_group = pick_heads_per_group(p.total_tokens, heads_all, lanes,
                                           dtype == B200K_F32 ? ForwardRows<float>::kMax : ForwardRows<__half>::kMax, sms);
  int64_t chunks = 0;
  for (int i = 0; i < p.sides; ++i) {
    p.side[i].chunks = static_cast<int>(ceil_div(p.side[i].heads, p.heads_per_group));
    chunks += p.side[i].chunks;
  }
  const int64_t blocks = ceil_div(p.total_tokens, kRopeThreads / lanes);
  if (blocks > INT32_MAX || chunks > 65535) return fail(B200K_UNSUPPORTED, "too many rows");
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(chunks));
  if (dtype == B200K_BF16) return launch_rope_type<__nv_bfloat16>(p, lanes, vec, grid, stream);
  if (dtype == B200K_F16) return launch_rope_type<__half>(p, lanes, vec, grid, stream);
  return launch_rope_type<float>(p, lanes, vec, grid, stream);
}

template <typename T, int GS>
int launch_backward(const RopeParams& p, bool vec, int grid, cudaStream_t stream) {
  if (p.interleaved) {
    if (vec) qk_rope_backward_kernel<T, GS, true, true><<<grid, kRopeThreads, 0, stream>>>(p);
    else qk_rope_backward_kernel<T, GS, true, false><<<grid, kRopeThreads, 0, stream>>>(p);
  } else {
    if (vec) qk_rope_backward_kernel<T, GS, false, true><<<grid, kRopeThreads, 0, stream>>>(p);
    else qk_rope_backward_kernel<T, GS, false, false><<<grid, kRopeThreads, 0, stream>>>(p);
  }
  B200K_CHECK_LAUNCH("qk_rope backward launch");
  return B200K_OK;
}

template <typename T>
int launch_backward_type(const RopeParams& p, int lanes, bool vec, int grid, cudaStream_t stream) {
  if (lanes == 4) return launch_backward<T, 4>(p, vec, grid, stream);
  if (lanes == 8) return launch_backward<T, 8>(p, vec, grid, stream);
  return launch_backward<T, 16>(p, vec, grid, stream);
}

// Blocks of the backward pass per SM: enough rows in flight, few partial rows.
constexpr int kBackwardBlocksPerSM = kBackwardMinBlocks;

}  // namespace
}  // namespace b200k

using namespace b200k;

extern "C" int b200k_qk_norm_rope(const b200k_qk_norm_rope_args* a, b200k_stream stream) {
  if (a == nullptr) return fail(B200K_INVALID_ARG, "null args");
  if (a->heads_q < 0 || a->heads_kv < 0 || a->heads_q > kMaxHeads || a->heads_kv > kMaxHeads)
    return fail(B200K_INVALID_ARG, "heads must lie between 0 and %d", kMaxHeads);
  RopeParams p = {};
  const int rc = fill_geometry(p, a->batch, a->tokens, a->head_dim, a->rotary_dim, a->interleaved, a->cos, a->sin,
                               a->table_stride, a->table_rows, a->weight_dtype, a->dtype, a->eps);
  if (rc != B200K_OK) return rc;
  if (p.total_tokens == 0) return B200K_OK;
  p.positions = a->positions;
  p.pos_b = a->position_stride_b;
  p.pos_t = a->position_stride_t;
  p.pos_is_i64 = a->positions_are_int64;
  if (a->heads_q > 0) {
    if (!a->q || !a->q_out) return fail(B200K_INVALID_ARG, "null pointer");
    RopeSide& s = p.side[p.sides++];
    s.x = a->q; s.y = a->q_out; s.w = a->q_weight;
    s.x_b = a->q_stride_b; s.x_h = a->q_stride_h; s.x_t = a->q_stride_t;
    s.y_b = a->qo_stride_b; s.y_h = a->qo_stride_h; s.y_t = a->qo_stride_t;
    s.heads = static_cast<int>(a->heads_q);
    s.rotate = a->rotary_dim > 0;
  }
  if (a->heads_kv > 0) {
    if (!a->k || !a->k_out) return fail(B200K_INVALID_ARG, "null pointer");
    RopeSide& s = p.side[p.sides++];
    s.x = a->k; s.y = a->k_out; s.w = a->k_weight;
    s.x_b = a->k_stride_b; s.x_h = a->k_stride_h; s.x_t = a->k_stride_t;
    s.y_b = a->ko_stride_b; s.y_h = a->ko_stride_h; s.y_t = a->ko_stride_t;
    s.heads = static_cast<int>(a->heads_kv);
    s.rotate = a->rotary_dim > 0;
  }
  if (p.sides == 0) return B200K_OK;
  return launch_forward(p, a->dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int64_t b200k_qk_norm_rope_backward_workspace_bytes(const b200k_qk_norm_rope_args* a) {
  if (a == nullptr || a->head_dim <= 0) return 0;
  const int sms = current_sm_count();
  if (sms <= 0) return 0;
  return static_cast<int64_t>(sms) * kBackwardBlocksPerSM * a->head_dim * 4;
}

extern "C" int b200k_qk_norm_rope_backward(const b200k_qk_norm_rope_args* a, b200k_stream stream_) {
  if (a == nullptr) return fail(B200K_INVALID_ARG, "null args");
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (a->heads_q < 0 || a->heads_kv < 0 || a->heads_q > kMaxHeads || a->heads_kv > kMaxHeads)
    return fail(B200K_INVALID_ARG, "heads must lie between 0 and %d", kMaxHeads);
  RopeParams p = {};
  const int rc = fill_geometry(p, a->batch, a->tokens, a->head_dim, a->rotary_dim, a->interleaved, a->cos, a->sin,
                               a->table_stride, a->table_rows, a->weight_dtype, a->dtype, a->eps);
  if (rc != B200K_OK) return rc;
  if ((a->q_weight != nullptr) != (a->dq_weight != nullptr) || (a->k_weight != nullptr) != (a->dk_weight != nullptr))
    return fail(B200K_INVALID_ARG, "a weight and its gradient come together");
  const int sms = current_sm_count();
  if (sms <= 0) return fail(B200K_CUDA_ERROR, "no current CUDA device");
  const int64_t rows_q = p.total_tokens * a->heads_q, rows_k = p.total_tokens * a->heads_kv;
  const bool sums = a->dq_weight != nullptr || a->dk_weight != nullptr;
  if (sums && (a->workspace == nullptr || (reinterpret_cast<uintptr_t>(a->workspace) & 15) ||
               a->workspace_bytes < b200k_qk_norm_rope_backward_workspace_bytes(a)))
    return fail(B200K_INVALID_ARG, "workspace missing, unaligned or too small");
  p.positions = a->positions;
  p.pos_b = a->position_stride_b;
  p.pos_t = a->position_stride_t;
  p.pos_is_i64 = a->positions_are_int64;

  const int lanes = lanes_per_row(p.units);
  const int groups = kRopeThreads / lanes;
  const int most = pick_heads_per_group(p.total_tokens, static_cast<int>(a->heads_q + a->heads_kv), lanes, 8, sms);
  WeightGradParams g = {};
  g.dim = p.dim;
  g.out[0] = a->dq_weight;
  g.out[1] = a->dk_weight;
  float* partial = static_cast<float*>(a->workspace);
  g.partial[0] = g.partial[1] = partial;
  // the blocks are shared out over the two sides by their rows
  const int budget = sms * kBackwardBlocksPerSM;
  int first = 0;
  for (int which = 0; which < 2; ++which) {
    const int64_t heads = which == 0 ? a->heads_q : a->heads_kv;
    const int64_t rows = which == 0 ? rows_q : rows_k;
    if (rows == 0) continue;
    if (!(which == 0 ? a->q && a->dq_out && a->q_out : a->k && a->dk_out && a->k_out))
      return fail(B200K_INVALID_ARG, "null pointer");
    RopeSide& s = p.side[p.sides++];
    if (which == 0) {
      s.x = a->q; s.dy = a->dq_out; s.y = a->q_out; s.w = a->q_weight;
      s.x_b = a->q_stride_b; s.x_h = a->q_stride_h; s.x_t = a->q_stride_t;
      s.dy_b = a->dq_stride_b; s.dy_h = a->dq_stride_h; s.dy_t = a->dq_stride_t;
      s.y_b = a->qo_stride_b; s.y_h = a->qo_stride_h; s.y_t = a->qo_stride_t;
    } else {
      s.x = a->k; s.dy = a->dk_out; s.y = a->k_out; s.w = a->k_weight;
      s.x_b = a->k_stride_b; s.x_h = a->k_stride_h; s.x_t = a->k_stride_t;
      s.dy_b = a->dk_stride_b; s.dy_h = a->dk_stride_h; s.dy_t = a->dk_stride_t;
      s.y_b = a->ko_stride_b; s.y_h = a->ko_stride_h; s.y_t = a->ko_stride_t;
    }
    s.heads = static_cast<int>(heads);
    s.rotate = a->rotary_dim > 0;
    s.chunks = static_cast<int>(ceil_div(heads, most));
    s.per = static_cast<int>(ceil_div(heads, s.chunks));
    if (p.total_tokens > (1 << 30) || p.total_tokens * s.chunks > (1 << 30))
      return fail(B200K_UNSUPPORTED, "too many rows");
    const int64_t need = ceil_div(p.total_tokens * s.chunks, groups);
    int64_t share = budget * rows / (rows_q + rows_k);
    if (share < 1) share = 1;
    if (which == 1 && first + share > budget) share = budget - first;
    if (which == 0 && rows_k > 0 && share > budget - 1) share = budget - 1;
    s.blocks = static_cast<int>(need < share ? need : share);
    s.first_block = first;
    s.dw = partial == nullptr ? nullptr : partial + static_cast<int64_t>(first) * p.dim;
    g.partial[which] = s.dw;
    g.blocks[which] = s.blocks;
    first += s.blocks;
  }
  if (p.sides > 0) {
    bool vec = true;
    for (int i = 0; i < p.sides; ++i) vec = vec && side_vectors(p.side[i], a->dtype == B200K_F32 ? 4 : 2);
    p.w_vec = weight_vectors(p);
    int e;
    if (a->dtype == B200K_BF16) e = launch_backward_type<__nv_bfloat16>(p, lanes, vec, first, stream);
    else if (a->dtype == B200K_F16) e = launch_backward_type<__half>(p, lanes, vec, first, stream);
    else e = launch_backward_type<float>(p, lanes, vec, first, stream);
    if (e != B200K_OK) return e;
  }
  if (!sums) return B200K_OK;
  const dim3 grid(static_cast<unsigned>(ceil_div(p.dim, 32)), 2);
  cudaError_t e;
  if (a->weight_dtype == B200K_F32)
    e = launch_after_predecessor(weight_grad_sum_kernel<float>, grid, dim3(1024), 0, stream, g);
  else if (a->weight_dtype == B200K_BF16)
    e = launch_after_predecessor(weight_grad_sum_kernel<__nv_bfloat16>, grid, dim3(1024), 0, stream, g);
  else
    e = launch_after_predecessor(weight_grad_sum_kernel<__half>, grid, dim3(1024), 0, stream, g);
  if (e != cudaSuccess) return fail(B200K_CUDA_ERROR, "weight gradient launch: %s", cudaGetErrorString(e));
  return B200K_OK;
}

extern "C" int b200k_paged_kv_append(const b200k_paged_kv_append_args* a, b200k_stream stream) {
  if (a == nullptr) return fail(B200K_INVALID_ARG, "null args");
  if (a->heads_q < 0 || a->heads_kv < 0 || a->heads_q > kMaxHeads || a->heads_kv > kMaxHeads)
    return fail(B200K_INVALID_ARG, "heads must lie between 0 and %d", kMaxHeads);
  if (a->dtype != B200K_F16 && a->dtype != B200K_BF16)
    return fail(B200K_INVALID_ARG, "dtype must be f16 or bf16");
  RopeParams p = {};
  const int rc = fill_geometry(p, a->batch, a->tokens, a->head_dim, a->rotary_dim, a->interleaved, a->cos, a->sin,
                               a->table_stride, a->table_rows, a->weight_dtype, a->dtype, a->eps);
  if (rc != B200K_OK) return rc;
  if (a->page_size <= 0 || a->num_pages < 0 || a->max_pages < 0)
    return fail(B200K_INVALID_ARG, "page_size must be positive, page counts not negative");
  if (p.total_tokens == 0) return B200K_OK;
  if (!a->cache_lens || (a->heads_kv > 0 && (!a->k || !a->v || !a->k_cache || !a->v_cache || !a->page_table)))
    return fail(B200K_INVALID_ARG, "null pointer");
  p.positions = a->positions;
  p.pos_b = a->position_stride_b;
  p.pos_t = a->position_stride_t;
  p.pos_is_i64 = a->positions_are_int64;
  p.cache_lens = a->cache_lens;
  p.new_lens = a->new_lens;
  p.page_table = a->page_table;
  p.page_table_stride = a->page_table_stride;
  p.page_size = a->page_size;
  p.max_pages = a->max_pages;
  p.num_pages = a->num_pages;
  if (a->q != nullptr && a->heads_q > 0) {
    if (!a->q_out) return fail(B200K_INVALID_ARG, "null pointer");
    RopeSide& s = p.side[p.sides++];
    s.x = a->q; s.y = a->q_out; s.w = a->q_weight;
    s.x_b = a->q_stride_b; s.x_h = a->q_stride_h; s.x_t = a->q_stride_t;
    s.y_b = a->qo_stride_b; s.y_h = a->qo_stride_h; s.y_t = a->qo_stride_t;
    s.heads = static_cast<int>(a->heads_q);
    s.rotate = a->rotary_dim > 0;
    s.zero_padding = a->zero_padding;
  }
  for (int which = 0; which < 2 && a->heads_kv > 0; ++which) {
    RopeSide& s = p.side[p.sides++];
    s.heads = static_cast<int>(a->heads_kv);
    s.paged = 1;
    if (which == 0) {
      s.x = a->k; s.y = a->k_cache; s.w = a->k_weight;
      s.x_b = a->k_stride_b; s.x_h = a->k_stride_h; s.x_t = a->k_stride_t;
      s.y_b = a->kc_stride_p; s.y_h = a->kc_stride_h; s.y_t = a->kc_stride_s;
      s.rotate = a->rotary_dim > 0;
    } else {
      s.x = a->v; s.y = a->v_cache;
      s.x_b = a->v_stride_b; s.x_h = a->v_stride_h; s.x_t = a->v_stride_t;
      s.y_b = a->vc_stride_p; s.y_h = a->vc_stride_h; s.y_t = a->vc_stride_s;
    }
  }
  if (p.sides == 0) return B200K_OK;
  return launch_forward(p, a->dtype, static_cast<cudaStream_t>(stream));
}

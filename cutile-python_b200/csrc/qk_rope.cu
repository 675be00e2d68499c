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
// A group of 4, 8 or 16 lanes owns one row, a lane 16 of its values as two 16-byte-multiple
// vectors chosen so that both halves of every rotated pair sit in the same lane (vectors at i
// and i + R / 2, or two neighbours): no exchange but the sum of squares.  A group keeps one
// token and walks its heads, so the cosines, sines and weights of its columns stay in
// registers.  Everything is computed in fp32 and rounded once, at the store.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "host.h"

namespace b200k {
namespace {

constexpr int kRopeThreads = 128;
constexpr int kMaxHeads = 65536;

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
  int rotate;
  int paged;
  int zero_padding;      // tokens behind new_lens[b] give zero rows (else they are left alone)
  int first_block, blocks;
};

struct RopeParams {
  RopeSide side[3];
  int sides;
  int dim, units, pairs, rotary;    // pairs: units that are rotated
  int interleaved, w_is_f32;
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

// Eight values as they lie in memory: 16 bytes (16-bit types) or 32 bytes (fp32).
template <typename T> struct Oct {
  static constexpr int kWords = sizeof(T) / 2;   // uint4s
  uint4 q[kWords];
};

template <typename T, bool VEC>
__device__ __forceinline__ Oct<T> load_oct(const T* p) {
  Oct<T> o;
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < Oct<T>::kWords; ++i) o.q[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  } else {
    T* e = reinterpret_cast<T*>(&o);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = p[i];
  }
  return o;
}

template <typename T, bool VEC>
__device__ __forceinline__ void store_oct(T* p, const float (&f)[8]) {
  Oct<T> o;
  T* e = reinterpret_cast<T*>(&o);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = rope_from_f32<T>(f[i]);
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < Oct<T>::kWords; ++i) reinterpret_cast<uint4*>(p)[i] = o.q[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = e[i];
  }
}

template <typename T>
__device__ __forceinline__ void unpack_oct(const Oct<T>& o, float (&f)[8]) {
  const T* e = reinterpret_cast<const T*>(&o);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = rope_to_f32<T>(e[i]);
}

template <typename T>
__device__ __forceinline__ void load_weight(const RopeParams& p, const void* w, int col, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    f[i] = p.w_is_f32 ? static_cast<const float*>(w)[col + i]
                      : rope_to_f32<T>(static_cast<const T*>(w)[col + i]);
  }
}

// A pair of the lane's values turned by (c, s); `back` turns the other way.
__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
  const float ta = a * c - b * s;
  b = b * c + a * s;
  a = ta;
}

// The lane's pairs: half split (lo[i], hi[i]); interleaved (lo[2i], lo[2i+1]), (hi[2i], hi[2i+1]).
__device__ __forceinline__ void rotate_lane(float (&lo)[8], float (&hi)[8], const float (&c)[8], const float (&s)[8],
                                            int interleaved) {
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      turn(lo[2 * i], lo[2 * i + 1], c[i], s[i]);
      turn(hi[2 * i], hi[2 * i + 1], c[4 + i], s[4 + i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) turn(lo[i], hi[i], c[i], s[i]);
  }
}

template <int GS>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = GS / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Which columns a lane holds.
struct LaneColumns {
  int lo, hi;             // first column of each vector
  bool has_lo, has_hi;
  bool rotated;
};

__device__ __forceinline__ LaneColumns lane_columns(const RopeParams& p, int unit) {
  LaneColumns c;
  c.rotated = unit < p.pairs;
  if (c.rotated) {
    c.lo = p.interleaved ? unit * 16 : unit * 8;
    c.hi = p.interleaved ? unit * 16 + 8 : unit * 8 + p.rotary / 2;
    c.has_lo = c.has_hi = true;
  } else {
    c.lo = p.rotary + (unit - p.pairs) * 16;
    c.hi = c.lo + 8;
    c.has_lo = unit < p.units;
    c.has_hi = c.has_lo && c.hi < p.dim;
  }
  return c;
}

// Cosines and sines of a token's position for the lane's pairs.  A position outside the table
// is recorded in the status word and gives NaN rows: nothing is read out of range.
__device__ __forceinline__ void load_angles(const RopeParams& p, int64_t b, int64_t t, const LaneColumns& col, int unit,
                                            float (&c)[8], float (&s)[8]) {
  int64_t pos;
  if (p.positions != nullptr) {
    const int64_t at = b * p.pos_b + t * p.pos_t;
    pos = p.pos_is_i64 ? static_cast<const int64_t*>(p.positions)[at] : static_cast<const int*>(p.positions)[at];
  } else {
    pos = (p.cache_lens != nullptr ? p.cache_lens[b] : 0) + t;
  }
  if (pos < 0 || pos >= p.table_rows) {
    if (unit == 0) report_bad_index(p.status, kRolePosition, static_cast<int>(t));
#pragma unroll
    for (int i = 0; i < 8; ++i) c[i] = s[i] = __int_as_float(0x7fc00000);
    return;
  }
  const float* cr = p.cos + pos * p.table_stride + unit * 8;
  const float* sr = p.sin + pos * p.table_stride + unit * 8;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 cv = reinterpret_cast<const float4*>(cr)[i];
    const float4 sv = reinterpret_cast<const float4*>(sr)[i];
    c[4 * i] = cv.x; c[4 * i + 1] = cv.y; c[4 * i + 2] = cv.z; c[4 * i + 3] = cv.w;
    s[4 * i] = sv.x; s[4 * i + 1] = sv.y; s[4 * i + 2] = sv.z; s[4 * i + 3] = sv.w;
  }
}

// Forward.  grid.x: one block per kRopeThreads / GS tokens; grid.y: (side, chunk of heads).
// U rows are requested together before the first is used.
template <typename T, int GS, bool VEC>
__global__ void __launch_bounds__(kRopeThreads)
qk_rope_kernel(const __grid_constant__ RopeParams p) {
  constexpr int U = sizeof(T) == 4 ? 2 : 4;
  const int unit = threadIdx.x % GS;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * (kRopeThreads / GS) + threadIdx.x / GS;
  int chunk = blockIdx.y, which = 0;
  while (which + 1 < p.sides && chunk >= p.side[which].chunks) chunk -= p.side[which++].chunks;
  const RopeSide& sd = p.side[which];
  const bool live = n < p.total_tokens;
  const int64_t b = live ? n / p.tokens : 0, t = live ? n - b * p.tokens : 0;
  const LaneColumns col = lane_columns(p, unit);
  const bool padded = live && p.new_lens != nullptr && t >= p.new_lens[b];

  // where this token's rows go
  int64_t out = b * sd.y_b + t * sd.y_t;
  bool store = live && (!padded || sd.zero_padding);
  if (sd.paged && store) {
    const int64_t at = static_cast<int64_t>(p.cache_lens[b]) + t;
    const int64_t entry = at >= 0 ? at / p.page_size : -1;
    int64_t page = -1;
    if (entry >= 0 && entry < p.max_pages) page = p.page_table[b * p.page_table_stride + entry];
    if (page < 0 || page >= p.num_pages) {
      if (unit == 0) report_bad_index(p.status, kRolePage, static_cast<int>(b));
      store = false;
    } else {
      out = page * sd.y_b + (at - entry * p.page_size) * sd.y_t;
    }
  }
  const bool read = store && !padded;

  float c[8], s[8], wlo[8], whi[8];
  const bool rotate = sd.rotate != 0 && col.rotated && read;
  if (rotate) load_angles(p, b, t, col, unit, c, s);
  const bool norm = sd.w != nullptr;
  if (norm) {
    if (col.has_lo) load_weight<T>(p, sd.w, col.lo, wlo);
    if (col.has_hi) load_weight<T>(p, sd.w, col.hi, whi);
  }

  const T* x = static_cast<const T*>(sd.x) + b * sd.x_b + t * sd.x_t;
  T* y = static_cast<T*>(sd.y) + out;
  const int h_end = min(sd.heads, (chunk + 1) * p.heads_per_group);
  for (int h0 = chunk * p.heads_per_group; h0 < h_end; h0 += U) {
    Oct<T> lo[U], hi[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool on = read && h0 + u < h_end;
      lo[u] = hi[u] = Oct<T>{};
      if (on && col.has_lo) lo[u] = load_oct<T, VEC>(x + (h0 + u) * sd.x_h + col.lo);
      if (on && col.has_hi) hi[u] = load_oct<T, VEC>(x + (h0 + u) * sd.x_h + col.hi);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float a[8], d[8];
      unpack_oct<T>(lo[u], a);
      unpack_oct<T>(hi[u], d);
      if (norm) {
        float sq = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sq += a[i] * a[i] + d[i] * d[i];
        const float r = rsqrtf(group_sum<GS>(sq) * p.inv_dim + p.eps);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          a[i] *= r * wlo[i];
          d[i] *= r * whi[i];
        }
      }
      if (rotate) rotate_lane(a, d, c, s, p.interleaved);
      if (padded) {
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = d[i] = 0.f;
      }
      if (store && h0 + u < h_end) {
        T* row = y + (h0 + u) * sd.y_h;
        if (col.has_lo) store_oct<T, VEC>(row + col.lo, a);
        if (col.has_hi) store_oct<T, VEC>(row + col.hi, d);
      }
    }
  }
}

// Backward.  Block-strided over (token, chunk of heads) of one side; every lane sums its
// columns' weight gradient over its rows in fp32, the block's groups are summed through shared
// memory in a fixed order and the block leaves one partial row: the result does not depend on
// the order in which blocks run.
template <typename T, int GS, bool VEC>
__global__ void __launch_bounds__(kRopeThreads)
qk_rope_backward_kernel(const __grid_constant__ RopeParams p) {
  constexpr int U = 2;
  constexpr int kGroups = kRopeThreads / GS;
  pdl_launch_dependents();   // the sum of the partial rows may be set up now; it waits for this grid
  const int unit = threadIdx.x % GS, group = threadIdx.x / GS;
  int which = 0;
  while (which + 1 < p.sides && static_cast<int>(blockIdx.x) >= p.side[which + 1].first_block) ++which;
  const RopeSide& sd = p.side[which];
  const int block = blockIdx.x - sd.first_block;
  const LaneColumns col = lane_columns(p, unit);
  const bool norm = sd.w != nullptr;
  float wlo[8] = {}, whi[8] = {};
  if (norm) {
    if (col.has_lo) load_weight<T>(p, sd.w, col.lo, wlo);
    if (col.has_hi) load_weight<T>(p, sd.w, col.hi, whi);
  }
  float glo[8] = {}, ghi[8] = {};   // weight gradient of the lane's columns

  const int64_t tasks = p.total_tokens * sd.chunks;
  const int64_t step = static_cast<int64_t>(sd.blocks) * kGroups;
  // the loop's bound is the same for the lanes of a warp (group_sum is warp-collective)
  const int64_t rounds = (tasks + step - 1) / step;
  for (int64_t i = 0; i < rounds; ++i) {
    const int64_t task = i * step + static_cast<int64_t>(block) * kGroups + group;
    const bool live = task < tasks;
    const int64_t n = live ? task / sd.chunks : 0;
    const int chunk = live ? static_cast<int>(task - n * sd.chunks) : 0;
    const int64_t b = n / p.tokens, t = n - b * p.tokens;
    float c[8], s[8];
    const bool rotate = live && col.rotated;
    if (rotate) {
      load_angles(p, b, t, col, unit, c, s);
#pragma unroll
      for (int k = 0; k < 8; ++k) s[k] = -s[k];
    }
    const T* x = static_cast<const T*>(sd.x) + b * sd.x_b + t * sd.x_t;
    const T* dy = static_cast<const T*>(sd.dy) + b * sd.dy_b + t * sd.dy_t;
    T* dx = static_cast<T*>(sd.y) + b * sd.y_b + t * sd.y_t;
    const int h_begin = chunk * p.heads_per_group;
    const int h_end = live ? min(sd.heads, h_begin + p.heads_per_group) : h_begin;
    // as many rounds for every group of the warp: a full chunk's heads, not this chunk's
    for (int h0 = h_begin; h0 < h_begin + min(p.heads_per_group, sd.heads); h0 += U) {
      Oct<T> xlo[U], xhi[U], dlo[U], dhi[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool on = h0 + u < h_end;
        xlo[u] = xhi[u] = dlo[u] = dhi[u] = Oct<T>{};
        if (on && col.has_lo) {
          xlo[u] = load_oct<T, VEC>(x + (h0 + u) * sd.x_h + col.lo);
          dlo[u] = load_oct<T, VEC>(dy + (h0 + u) * sd.dy_h + col.lo);
        }
        if (on && col.has_hi) {
          xhi[u] = load_oct<T, VEC>(x + (h0 + u) * sd.x_h + col.hi);
          dhi[u] = load_oct<T, VEC>(dy + (h0 + u) * sd.dy_h + col.hi);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float gl[8], gh[8];
        unpack_oct<T>(dlo[u], gl);
        unpack_oct<T>(dhi[u], gh);
        if (rotate) rotate_lane(gl, gh, c, s, p.interleaved);
        if (norm) {
          float a[8], d[8];
          unpack_oct<T>(xlo[u], a);
          unpack_oct<T>(xhi[u], d);
          float sq = 0.f, dot = 0.f;   // sum x^2, sum x * g * w
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            sq += a[k] * a[k] + d[k] * d[k];
            dot += a[k] * (gl[k] * wlo[k]) + d[k] * (gh[k] * whi[k]);
          }
          const float r = rsqrtf(group_sum<GS>(sq) * p.inv_dim + p.eps);
          const float along = group_sum<GS>(dot) * p.inv_dim * r * r;   // mean(h u) / (x / u)
          if (h0 + u < h_end) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              glo[k] += gl[k] * (a[k] * r);
              ghi[k] += gh[k] * (d[k] * r);
            }
          }
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            gl[k] = r * (gl[k] * wlo[k] - a[k] * along);
            gh[k] = r * (gh[k] * whi[k] - d[k] * along);
          }
        }
        if (h0 + u < h_end) {
          T* row = dx + (h0 + u) * sd.y_h;
          if (col.has_lo) store_oct<T, VEC>(row + col.lo, gl);
          if (col.has_hi) store_oct<T, VEC>(row + col.hi, gh);
        }
      }
    }
  }

  if (!norm) return;   // the same for the whole block
  __shared__ float sums[kGroups][GS * 16 + 1];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    sums[group][unit * 16 + k] = glo[k];
    sums[group][unit * 16 + 8 + k] = ghi[k];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < GS * 16; i += kRopeThreads) {
    const LaneColumns lc = lane_columns(p, i / 16);
    const bool high = (i % 16) >= 8;
    if (high ? lc.has_hi : lc.has_lo) {
      float v = 0.f;
#pragma unroll 8
      for (int g = 0; g < kGroups; ++g) v += sums[g][i];
      sd.dw[static_cast<int64_t>(block) * p.dim + (high ? lc.hi : lc.lo) + (i % 8)] = v;
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

// Lanes per row: the smallest group whose lanes hold 16 values each.
int lanes_per_row(int units) { return units <= 4 ? 4 : (units <= 8 ? 8 : 16); }

// Heads a group walks with one token's angles: as many as leave every SM about a thousand
// threads, at least the rows that are requested together.
int pick_heads_per_group(int64_t total_tokens, int heads_all, int lanes, int at_least, int sms) {
  int per = 16;
  while (per > at_least && total_tokens * lanes * ceil_div(heads_all, per) < static_cast<int64_t>(sms) * 1024) per /= 2;
  return per < at_least ? at_least : per;
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
  if (vec) qk_rope_kernel<T, GS, true><<<grid, kRopeThreads, 0, stream>>>(p);
  else qk_rope_kernel<T, GS, false><<<grid, kRopeThreads, 0, stream>>>(p);
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
  p.heads_per_group = pick_heads_per_group(p.total_tokens, heads_all, lanes, dtype == B200K_F32 ? 2 : 4, sms);
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
  if (vec) qk_rope_backward_kernel<T, GS, true><<<grid, kRopeThreads, 0, stream>>>(p);
  else qk_rope_backward_kernel<T, GS, false><<<grid, kRopeThreads, 0, stream>>>(p);
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
constexpr int kBackwardBlocksPerSM = 6;

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
  p.heads_per_group = pick_heads_per_group(p.total_tokens, static_cast<int>(a->heads_q + a->heads_kv), lanes, 2, sms);
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
    s.chunks = static_cast<int>(ceil_div(heads, p.heads_per_group));
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
  if (p.total_tokens == 0 || a->heads_kv == 0) return B200K_OK;
  if (!a->k || !a->v || !a->k_cache || !a->v_cache || !a->page_table || !a->cache_lens)
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
  for (int which = 0; which < 2; ++which) {
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
  return launch_forward(p, a->dtype, static_cast<cudaStream_t>(stream));
}

// attention.cu -- attention within packed segments (an encoder's users, documents): queries
// [Tq, H, D] and keys/values [Tk, Hk, D] of S segments lie one behind the other, and a query
// sees keys of its own segment only.  For query i (of n) and key j (of m) of a segment, head h:
//
//   x = scale q_i . k_j      s = cap tanh(x / cap)  (or x)  - slope_h |i + m - n - j|
//   seen(i, j) = not causal, or j <= i + m - n, or j < prefix
//   p_ij = exp(s_ij) / sum over seen exp(s)     out_i = sum_j p_ij v_j     (0 where nothing is seen)
//
// and, with dp_ij = dout_i . v_j, delta_i = dout_i . out_i, e_ij = p_ij (dp_ij - delta_i) (1 - tanh^2) scale:
//
//   dv_j = sum_i p_ij dout_i     dq_i = sum_j e_ij k_j     dk_j = sum_i e_ij q_i
//
// (dk, dv: summed over the query heads that share the key head).
//
// What every kernel uses: the mask of a row is ONE interval [lo, hi) of the packed keys, whatever mixes into it
// (segments, causal order, prefix).  plan_kernel (delta_kernel for the gradients) computes it once a call for all heads, so
// that tiles need not follow segments: a tile is 128 rows of the packed order, its keys are the union of its rows'
// intervals, and a block of keys that all rows see is not masked at all.
//
// The kernels of a call start under one another's tails.  What one of them writes (the workspace) the next reads by plain
// loads behind its griddepcontrol.wait, never by __ldg, which asks for memory that nobody writes while the kernel lives.
#include "common.cuh"

#include <algorithm>
#include <climits>
#include <cmath>
#include <mutex>
#include <type_traits>

namespace rb {
namespace attn {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kMaxWidth = 256;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Params {
  const void *q, *k, *v, *o, *g;  // o, g: the forward call's output and the gradient it got
  void *out, *dq, *dk, *dv;
  float* lse;                     // [H, Tq] log of the sum of exp(s), -inf where nothing is seen
  float* delta;                   // [H, Tq] dout . out, then (behind the queries' gradients) the sum of p dp; in fp16, from
                                  // the tiles, times range_of
  int4* rows;                     // [Tq]: lo, hi, place of the query among the packed keys, segment (-1: in none)
  int4* tiles;                    // of the queries: rows [x, y), the keys that they see [z, w)
  int4* key_tiles;                // (backward) of the keys: rows [x, y), queries that may see them [z, w)
  int32_t* key_segments;          // (fp16 backward) [Tk]: of the keys, -1: in none
  uint32_t* next;                 // tickets for work
  int2* redo;                     // (forward tiles) [tiles x heads][4]: rows of 32 to be taken again, the entry before it
  float* part;                    // few queries: of every row and split, the sums [D], their maximum and their weights' sum
  int splits, parts;
  const void *q_off, *k_off, *prefix;
  const float* slopes;
  int64_t q_t, q_h, k_t, k_h, v_t, v_h, g_t, g_h;  // elements from token to token and from head to head
  int Tq, Tk, S, H, Hk, G, D, off64, causal;
  float scale, cap;
  uint32_t* peaks;                // fp16 backward: [S, Hk] the largest squared norms of a row of g and of v
  int by_segment, n_tiles;        // tiles follow segments (else: 128 rows of the packed order)
  int keys_by_segment, n_key_tiles;
};

__device__ __forceinline__ int64_t entry(const void* a, int wide, int64_t i) {
  return wide ? __ldg(static_cast<const int64_t*>(a) + i) : (int64_t)__ldg(static_cast<const int32_t*>(a) + i);
}
// an offset as it may be used: whatever the array holds, no row outside [0, total] is named
__device__ __forceinline__ int offset_at(const void* a, int wide, int i, int total) {
  return (int)min(max(entry(a, wide, i), (int64_t)0), (int64_t)total);
}
// the last segment that starts at or before row r, or -1
__device__ __forceinline__ int segment_of(const void* off, int wide, int S, int total, int r) {
  int a = 0, b = S;  // segments [0, a) start at or before r, [b, S) behind it
  while (a < b) {
    const int m = (a + b) >> 1;
    if (offset_at(off, wide, m, total) <= r) a = m + 1;
    else b = m;
  }
  return a - 1;
}

__device__ __forceinline__ int4 row_of(const Params& p, int r) {
  const int s = segment_of(p.q_off, p.off64, p.S, p.Tq, r);
  if (s < 0) return make_int4(0, 0, 0, -1);
  const int q0 = offset_at(p.q_off, p.off64, s, p.Tq), q1 = offset_at(p.q_off, p.off64, s + 1, p.Tq);
  if (r >= q1) return make_int4(0, 0, 0, -1);
  const int k0 = offset_at(p.k_off, p.off64, s, p.Tk), k1 = max(k0, offset_at(p.k_off, p.off64, s + 1, p.Tk));
  const int place = k0 + (r - q0) + (k1 - k0) - (q1 - q0);
  int hi = k1;
  if (p.causal) {
    const int seen = p.prefix != nullptr ? (int)min(max(entry(p.prefix, p.off64, s), (int64_t)0), (int64_t)(k1 - k0)) : 0;
    hi = min(k1, max(place + 1, k0 + seen));
  }
  return hi > k0 ? make_int4(k0, hi, place, s) : make_int4(0, 0, place, s);
}

template <typename T>
__device__ __forceinline__ float to_f32(T v) { return (float)v; }

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// tanh from exp: 1 - 2 / (1 + e^2x).  Near 0 it is off by 2^-22 of 1, not of x: in the score that is 2^-22 cap, where
// the hardware's own tanh is off by 2^-11 of x.  Caps above kWideCap, for which that would be 2^-14 and more, take the
// series below 1/4 (its next term is 2^-26 of x there), in tile kernels of their own (WIDE, of 128 columns for all widths):
// as a branch of the others it cost those 2 to 5 % by its registers.
constexpr float kWideCap = 256.0f;
__device__ __forceinline__ float tanh_of(float x) { return fmaf(-2.0f, rcp_fast(1.0f + exp2_fast(x * (2.0f * kLog2e))), 1.0f); }
__device__ __forceinline__ float tanh_wide(float x) {
  const float z = x * x;
  float s = fmaf(z, 62.0f / 2835.0f, -17.0f / 315.0f);
  s = fmaf(z, s, 2.0f / 15.0f);
  s = fmaf(z, s, -1.0f / 3.0f);
  return z < 0.0625f ? fmaf(x * z, s, x) : tanh_of(x);
}
// 1 - tanh^2: with w = e^-2|x| and m = 2 w / (1 + w) = 1 - |tanh| it is m (2 - m), right to a few 2^-24 of itself however
// near to 1 the tanh is (1 - t t is off by 2^-23 of 1)
__device__ __forceinline__ float slant_of(float x) {
  const float w = exp2_fast(-fabsf(x) * (2.0f * kLog2e)), m = 2.0f * w * rcp_fast(1.0f + w);
  return m * (2.0f - m);
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}

constexpr int kTile = 128;  // rows of a tile: the lanes of TMEM

// The rows [x, y) of tile b of `size` rows.  By the packed order, 128 rows a tile.  By segment, segment s has room for
// tiles from floor(start / size) + s on, which is as much as it needs and known without a sum over segments; the rows
// before the first and behind the last count as segments too, and a tile that its segment does not need is empty.
// A token may be `factor` rows.
__device__ __forceinline__ int2 tile_rows(const void* off, int wide, int S, int total, int b, int by_segment, int size = kTile, int factor = 1) {
  if (!by_segment) return make_int2(min(b * size, total * factor), min((b + 1) * size, total * factor));
  // starts 0, off[0], ..., off[S]: the last i with floor(start_i / size) + i <= b
  int lo = 0, hi = S + 2;
  const int lane = threadIdx.x & 31;
  while (hi - lo > 1) {  // 32 probes at once
    const int step = (hi - lo + 31) / 32;
    const int i = lo + (lane + 1) * step;
    const bool below = i < hi && offset_at(off, wide, i - 1, total) * factor / size + i <= b;
    const int n = __popc(__ballot_sync(kAll, below));
    lo += n * step;
    hi = min(hi, lo + step);
  }
  const int start = lo == 0 ? 0 : offset_at(off, wide, lo - 1, total) * factor;
  const int end = lo == S + 1 ? total * factor : offset_at(off, wide, lo, total) * factor;
  const int first = start + max(b - (start / size + lo), 0) * size;
  return make_int2(min(first, end), min(first + size, end));
}

// The rows' intervals, once a call for all heads, a CTA a tile; and what its rows see together.  A tile that sees nothing
// is finished here (zeros).
template <typename T>
__global__ void __launch_bounds__(kTile) plan_kernel(const __grid_constant__ Params p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ int s_lo[4], s_hi[4];
  if (blockIdx.x == 0 && threadIdx.x == 0 && p.next != nullptr) *p.next = 0;
  const int2 span = tile_rows(p.q_off, p.off64, p.S, p.Tq, blockIdx.x, p.by_segment);
  const int r = span.x + threadIdx.x, warp = threadIdx.x >> 5;
  int4 row = make_int4(0, 0, 0, 0);
  if (r < span.y) {
    row = row_of(p, r);
    p.rows[r] = row;
  }
  const int lo = __reduce_min_sync(kAll, row.y > row.x ? row.x : INT_MAX), hi = __reduce_max_sync(kAll, row.y > row.x ? row.y : 0);
  if ((threadIdx.x & 31) == 0) {
    s_lo[warp] = lo;
    s_hi[warp] = hi;
  }
  __syncthreads();
  const int first = min(min(s_lo[0], s_lo[1]), min(s_lo[2], s_lo[3])), last = max(max(s_hi[0], s_hi[1]), max(s_hi[2], s_hi[3]));
  if (threadIdx.x == 0 && p.tiles != nullptr) p.tiles[blockIdx.x] = make_int4(span.x, span.y, first, last);
  if (first >= last && p.tiles != nullptr) {
    T* out = static_cast<T*>(p.out) + (int64_t)span.x * p.H * p.D;
    for (int64_t i = threadIdx.x; i < (int64_t)max(span.y - span.x, 0) * p.H * p.D; i += kTile) out[i] = T(0.0f);
    if (p.lse != nullptr && r < span.y)
      for (int h = 0; h < p.H; ++h) p.lse[(int64_t)h * p.Tq + r] = -INFINITY;
  }
}

// ------------------------------------------------------------ one row, one warp
// The formulas as they stand, a warp for a row of one head, each lane D / 32 columns.  These take the shapes that the
// tiles do not (D off 8 or above 128, rows off 16 bytes), and every row of a tile whose result is not finite: a tile
// adds the keys that a row does not see times a zero weight, and a zero times an infinity or NaN there is a NaN.
constexpr int kPerLane = kMaxWidth / 32;

template <typename T>
__device__ __forceinline__ void load_row(const void* base, int64_t at, int D, int lane, float* v) {
  const T* t = static_cast<const T*>(base) + at;
#pragma unroll
  for (int c = 0; c < kPerLane; ++c) v[c] = lane + 32 * c < D ? to_f32(t[lane + 32 * c]) : 0.0f;
}
template <typename T>
__device__ __forceinline__ void store_row(void* base, int64_t at, int D, int lane, const float* v, float w) {
  T* t = static_cast<T*>(base) + at;
#pragma unroll
  for (int c = 0; c < kPerLane; ++c)
    if (lane + 32 * c < D) t[lane + 32 * c] = T(v[c] * w);
}
__device__ __forceinline__ float dot_row(const float* a, const float* b) {
  float s = 0.0f;
#pragma unroll
  for (int c = 0; c < kPerLane; ++c) s = fmaf(a[c], b[c], s);
  return warp_sum(s);
}
// the score in units of log 2, and 1 - tanh^2
__device__ __forceinline__ float score_of(const Params& p, float x, int place, int j, float slope, float& slant) {
  x *= p.scale;
  slant = 1.0f;
  if (p.cap > 0.0f) {
    slant = slant_of(x / p.cap);
    x = p.cap * (p.cap > kWideCap ? tanh_wide(x / p.cap) : tanh_of(x / p.cap));
  }
  return kLog2e * fmaf(-slope, (float)abs(place - j), x);
}

template <typename T>
__device__ __noinline__ void row_forward(const Params& p, int r, int h) {
  const int lane = threadIdx.x & 31, hk = h / p.G;
  const int4 row = p.rows[r];
  const float slope = p.slopes != nullptr ? __ldg(p.slopes + h) : 0.0f;
  float q[kPerLane], o[kPerLane], x[kPerLane], top = -INFINITY, total = 0.0f, slant;
  load_row<T>(p.q, r * p.q_t + h * p.q_h, p.D, lane, q);
#pragma unroll
  for (int c = 0; c < kPerLane; ++c) o[c] = 0.0f;
#pragma unroll 1
  for (int j = row.x; j < row.y; ++j) {
    load_row<T>(p.k, j * p.k_t + hk * p.k_h, p.D, lane, x);
    const float s = score_of(p, dot_row(q, x), row.z, j, slope, slant);
    const float higher = fmaxf(top, s);
    const float keep = higher == top ? 1.0f : exp2_fast(top - higher);
    const float w = higher == -INFINITY ? s - s + 0.0f : exp2_fast(s - higher);  // (a score of -inf: nothing, or NaN)
    top = higher;
    const float e = s == -INFINITY ? 0.0f : w;
    total = fmaf(total, keep, e);
    load_row<T>(p.v, j * p.v_t + hk * p.v_h, p.D, lane, x);
#pragma unroll
    for (int c = 0; c < kPerLane; ++c) o[c] = fmaf(o[c], keep, e * x[c]);
  }
  store_row<T>(p.out, ((int64_t)r * p.H + h) * p.D, p.D, lane, o, total == 0.0f ? 0.0f : 1.0f / total);
  if (p.lse != nullptr && lane == 0) p.lse[(int64_t)h * p.Tq + r] = total == 0.0f ? -INFINITY : kLn2 * (top + log2f(total));
}

// in units of log 2; +inf (all weights 0) for a row that sees nothing
__device__ __forceinline__ float lse_of(const Params& p, int r, int h) {
  const float l = __ldg(p.lse + (int64_t)h * p.Tq + r);
  return l == -INFINITY ? INFINITY : kLog2e * l;
}

// (fp16) the power of two that keeps |dP - delta| of a segment's rows times it under 1
__device__ __forceinline__ float range_of(const Params& p, int segment, int hk) {
  if (segment < 0) return 1.0f;
  const uint32_t* peak = p.peaks + ((int64_t)segment * p.Hk + hk) * 2;
  const float bound = 2.0f * sqrtf(__uint_as_float(peak[0])) * sqrtf(__uint_as_float(peak[1]));  // of |dP - delta|
  const int e = (int)(__float_as_uint(bound) >> 23) - 126;                                       // bound < 2^e
  return bound > 0.0f && bound < INFINITY ? __uint_as_float((uint32_t)min(max(127 - e, 1), 254) << 23) : 1.0f;
}

// delta of a row, which the tiles of fp16 queries leave times its range
template <typename T>
__device__ __forceinline__ float delta_unit(const Params& p, int r, int h) {
  return std::is_same<T, __half>::value && p.key_tiles != nullptr ? range_of(p, p.rows[r].w, h / p.G) : 1.0f;
}
// (delta and what it is off by: at backward_kernel)
template <typename T>
__device__ __noinline__ void row_dq(const Params& p, int r, int h) {
  const int lane = threadIdx.x & 31, hk = h / p.G;
  const int4 row = p.rows[r];
  const float slope = p.slopes != nullptr ? __ldg(p.slopes + h) : 0.0f;
  const float lse = lse_of(p, r, h), range = delta_unit<T>(p, r, h), delta = p.delta[(int64_t)h * p.Tq + r] / range;
  float q[kPerLane], g[kPerLane], dq[kPerLane], mean[kPerLane], k[kPerLane], v[kPerLane], slant, off = 0.0f;
  load_row<T>(p.q, r * p.q_t + h * p.q_h, p.D, lane, q);
  load_row<T>(p.g, r * p.g_t + h * p.g_h, p.D, lane, g);
#pragma unroll
  for (int c = 0; c < kPerLane; ++c) dq[c] = mean[c] = 0.0f;
#pragma unroll 1
  for (int j = row.x; j < row.y; ++j) {
    load_row<T>(p.k, j * p.k_t + hk * p.k_h, p.D, lane, k);
    load_row<T>(p.v, j * p.v_t + hk * p.v_h, p.D, lane, v);
    const float s = score_of(p, dot_row(q, k), row.z, j, slope, slant);
    const float w = exp2_fast(s - lse), d = w * (dot_row(g, v) - delta);
    off += d;
#pragma unroll
    for (int c = 0; c < kPerLane; ++c) {
      dq[c] = fmaf(d * slant, k[c], dq[c]);
      mean[c] = fmaf(w * slant, k[c], mean[c]);
    }
  }
#pragma unroll
  for (int c = 0; c < kPerLane; ++c) dq[c] = fmaf(-off, mean[c], dq[c]);
  if (lane == 0) p.delta[(int64_t)h * p.Tq + r] = (delta + off) * range;
  store_row<T>(p.dq, ((int64_t)r * p.H + h) * p.D, p.D, lane, dq, p.scale);
}

// the segment that a row is in, or -1
__device__ __forceinline__ int segment_with(const Params& p, const void* off, int total, int r) {
  const int s = segment_of(off, p.off64, p.S, total, r);
  return s >= 0 && r < offset_at(off, p.off64, s + 1, total) ? s : -1;
}
// the queries of the segment that key j belongs to: [x, y)
__device__ __forceinline__ int2 queries_of(const Params& p, int j) {
  const int s = segment_with(p, p.k_off, p.Tk, j);
  if (s < 0) return make_int2(0, 0);
  return make_int2(offset_at(p.q_off, p.off64, s, p.Tq), offset_at(p.q_off, p.off64, s + 1, p.Tq));
}

template <typename T>
__device__ __noinline__ void row_dkv(const Params& p, int j, int hk) {
  const int lane = threadIdx.x & 31;
  const int2 span = queries_of(p, j);
  float k[kPerLane], v[kPerLane], dk[kPerLane], dv[kPerLane], q[kPerLane], g[kPerLane], slant;
  load_row<T>(p.k, j * p.k_t + hk * p.k_h, p.D, lane, k);
  load_row<T>(p.v, j * p.v_t + hk * p.v_h, p.D, lane, v);
#pragma unroll
  for (int c = 0; c < kPerLane; ++c) dk[c] = dv[c] = 0.0f;
#pragma unroll 1
  for (int h = hk * p.G; h < (hk + 1) * p.G; ++h) {
    const float slope = p.slopes != nullptr ? __ldg(p.slopes + h) : 0.0f;
#pragma unroll 1
    for (int r = span.x; r < span.y; ++r) {
      const int4 row = p.rows[r];
      if (j < row.x || j >= row.y) continue;
      load_row<T>(p.q, r * p.q_t + h * p.q_h, p.D, lane, q);
      load_row<T>(p.g, r * p.g_t + h * p.g_h, p.D, lane, g);
      const float s = score_of(p, dot_row(q, k), row.z, j, slope, slant);
      const float w = exp2_fast(s - lse_of(p, r, h));
      const float e = w * (dot_row(g, v) - p.delta[(int64_t)h * p.Tq + r] / delta_unit<T>(p, r, h)) * slant;
#pragma unroll
      for (int c = 0; c < kPerLane; ++c) {
        dk[c] = fmaf(e, q[c], dk[c]);
        dv[c] = fmaf(w, g[c], dv[c]);
      }
    }
  }
  const int64_t at = ((int64_t)j * p.Hk + hk) * p.D;
  store_row<T>(p.dk, at, p.D, lane, dk, p.scale);
  store_row<T>(p.dv, at, p.D, lane, dv, 1.0f);
}

enum RowPass : int { kRowForward, kRowDq, kRowDkv };
template <typename T, int PASS>
__global__ void __launch_bounds__(256) row_kernel(const __grid_constant__ Params p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int heads = PASS == kRowDkv ? p.Hk : p.H;
  const int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (i >= (int64_t)(PASS == kRowDkv ? p.Tk : p.Tq) * heads) return;
  const int r = (int)(i / heads), h = (int)(i % heads);
  if constexpr (PASS == kRowForward) row_forward<T>(p, r, h);
  else if constexpr (PASS == kRowDq) row_dq<T>(p, r, h);
  else row_dkv<T>(p, r, h);
}

// What the gradients need: each query's interval and the lists of tiles (the first CTAs), delta_i = dout_i . out_i, and in
// fp16, for each segment and key head, the largest squared norms of a row of dout and of v (those that are finite), as bits
// of positive floats, which order as numbers do.  LANES lanes take a row of one head by 16 bytes each (32, value by value, where rows do not allow that).
constexpr int kDeltaCtas = 6;  // an SM, at most (fp16, 60 users of 10 to 1000 items: 35.4 us, with 8 and fewer registers 37.7)
template <typename T>
__device__ __forceinline__ float2 widen2(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return make_float2(bf16_lo(w), bf16_hi(w));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
// sums over the lanes of a row
template <int LANES>
__device__ __forceinline__ float2 lanes_sum(float2 s) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    s.x += __shfl_xor_sync(kAll, s.x, o);
    s.y += __shfl_xor_sync(kAll, s.y, o);
  }
  return s;
}
// a warp a tile: the rows of tile b of the queries and the keys that any of them sees
__device__ __forceinline__ void list_queries(const Params& p, int b) {
  const int lane = threadIdx.x & 31;
  const int2 span = tile_rows(p.q_off, p.off64, p.S, p.Tq, b, p.by_segment);
  int lo = INT_MAX, hi = 0;
  for (int r = span.x + lane; r < span.y; r += 32) {
    const int4 row = row_of(p, r);
    if (row.y > row.x) {
      lo = min(lo, row.x);
      hi = max(hi, row.y);
    }
  }
  lo = __reduce_min_sync(kAll, lo);
  hi = __reduce_max_sync(kAll, hi);
  if (lane == 0) p.tiles[b] = make_int4(span.x, span.y, lo, hi);
}
// and of tile b of the keys, with the queries of the segments from the first key's to the last key's (in causal order,
// from the first that sees the first key)
__device__ __forceinline__ void list_keys(const Params& p, int b) {
  const int2 span = tile_rows(p.k_off, p.off64, p.S, p.Tk, b, p.keys_by_segment);
  if ((threadIdx.x & 31) != 0) return;
  int lo = INT_MAX, hi = 0;
  if (span.y > span.x) {
    const int sa = max(segment_of(p.k_off, p.off64, p.S, p.Tk, span.x), 0), sb = segment_of(p.k_off, p.off64, p.S, p.Tk, span.y - 1);
    if (sb >= 0) {
      const int q0 = offset_at(p.q_off, p.off64, sa, p.Tq), k0 = offset_at(p.k_off, p.off64, sa, p.Tk);
      const int n = max(0, offset_at(p.q_off, p.off64, sa + 1, p.Tq) - q0), m = max(0, offset_at(p.k_off, p.off64, sa + 1, p.Tk) - k0);
      lo = q0;
      hi = offset_at(p.q_off, p.off64, sb + 1, p.Tq);
      if (p.causal) {
        const int seen = p.prefix != nullptr ? (int)min(max(entry(p.prefix, p.off64, sa), (int64_t)0), (int64_t)m) : 0;
        if (span.x - k0 >= seen) lo = q0 + min(max(span.x - k0 - m + n, 0), n);
      }
    }
  }
  p.key_tiles[b] = make_int4(span.x, span.y, lo, hi);
}

template <typename T, int LANES, bool VEC>
__global__ void __launch_bounds__(256, kDeltaCtas) delta_kernel(const __grid_constant__ Params p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  constexpr bool kPeaks = std::is_same<T, __half>::value;
  const int query_ctas = (p.Tq + 255) / 256, list_ctas = query_ctas + (kPeaks ? (p.Tk + 255) / 256 : 0);
  const int row_ctas = list_ctas + (p.n_tiles + p.n_key_tiles + 7) / 8;
  if ((int)blockIdx.x < query_ctas) {
    const int r = blockIdx.x * 256 + threadIdx.x;
    if (r < p.Tq) p.rows[r] = row_of(p, r);
    return;
  }
  if (kPeaks && (int)blockIdx.x < list_ctas) {
    const int j = (blockIdx.x - query_ctas) * 256 + threadIdx.x;
    if (j < p.Tk) p.key_segments[j] = segment_with(p, p.k_off, p.Tk, j);
    return;
  }
  if ((int)blockIdx.x < row_ctas) {
    const int b = (blockIdx.x - list_ctas) * 8 + (threadIdx.x >> 5);
    if (b < p.n_tiles) list_queries(p, b);
    else if (b < p.n_tiles + p.n_key_tiles) list_keys(p, b - p.n_tiles);
    return;
  }
  // (fp16) the largest square of the rows of one segment and key head that this thread meets one behind the other
  uint32_t* peak = nullptr;
  float high = 0.0f;
  // of the last row, and the first row behind it: at first those of the CTA's first row, found by a warp with 32 probes
  int segment = -1, until = 0;
  __shared__ int2 s_first[2];
  const int64_t ctas = gridDim.x - row_ctas, cta = blockIdx.x - row_ctas;
  if (kPeaks) {
    if (threadIdx.x < 64) {
      const void* off = threadIdx.x < 32 ? p.q_off : p.k_off;
      const int total = threadIdx.x < 32 ? p.Tq : p.Tk, r = (int)(total * cta / ctas);
      int a = 0, b = p.S;  // segments [0, a) start at or before r, [b, S) behind it
      while (a < b) {
        const int step = (b - a + 31) / 32, m = a + (int)(threadIdx.x % 32) * step;
        const int n = __popc(__ballot_sync(kAll, m < b && offset_at(off, p.off64, m, total) <= r));
        b = min(b, a + n * step);
        if (n > 0) a += (n - 1) * step + 1;
      }
      const int end = a > 0 ? offset_at(off, p.off64, a, total) : 0;
      if (threadIdx.x % 32 == 0) s_first[threadIdx.x / 32] = end > r ? make_int2(a - 1, end) : make_int2(-1, r);
    }
    __syncthreads();
    segment = s_first[0].x;
    until = s_first[0].y;
  }
  auto raise = [&](uint32_t* next) {
    if (peak != nullptr) atomicMax(peak, __float_as_uint(high));
    peak = next;
    high = 0.0f;
  };
  auto meet = [&](const void* off, int total, int r, int hk, int which, float square) {
    if (r >= until) {
      segment = segment_with(p, off, total, r);
      until = segment < 0 ? r + 1 : offset_at(off, p.off64, segment + 1, total);
    }
    uint32_t* mine = segment < 0 ? nullptr : p.peaks + ((int64_t)segment * p.Hk + hk) * 2 + which;
    if (mine != peak) raise(mine);
    if (square < INFINITY) high = fmaxf(high, square);
  };
  constexpr int kRows = 256 / LANES, kTwo = 2;  // rows of a CTA at a time, twice
  const int lane = threadIdx.x % LANES, c = lane * 8;
  // rows (token, head) [0, tokens * heads), a run of tokens a CTA; from one to this thread's next without a quotient
  auto scan = [&](int all_tokens, int heads, auto source, auto use) {
    const int d_token = kRows / heads, d_head = kRows % heads, first = threadIdx.x / LANES;
    const int64_t tokens = all_tokens * (cta + 1) / ctas;
    int64_t token = all_tokens * cta / ctas + first / heads;
    int head = first % heads;
    while (__any_sync(kAll, token < tokens)) {
      int64_t at[kTwo];
      int h[kTwo];
      const T *x[kTwo], *y[kTwo];
      float2 s[kTwo];
#pragma unroll
      for (int u = 0; u < kTwo; ++u) {
        at[u] = token;
        h[u] = head;
        x[u] = y[u] = nullptr;
        if (token < tokens) source(token, head, x[u], y[u]);
        s[u] = make_float2(0.0f, 0.0f);
        token += d_token;
        head += d_head;
        if (head >= heads) {
          head -= heads;
          ++token;
        }
      }
      if constexpr (VEC) {  // (a lane's sixteen bytes are its part of a row)
        uint4 xv[kTwo], yv[kTwo];
#pragma unroll
        for (int u = 0; u < kTwo; ++u) {
          xv[u] = x[u] != nullptr && c < p.D ? __ldg(reinterpret_cast<const uint4*>(x[u] + c)) : make_uint4(0u, 0u, 0u, 0u);
          yv[u] = y[u] != nullptr && c < p.D ? __ldg(reinterpret_cast<const uint4*>(y[u] + c)) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int u = 0; u < kTwo; ++u) {
          const uint32_t xw[4] = {xv[u].x, xv[u].y, xv[u].z, xv[u].w}, yw[4] = {yv[u].x, yv[u].y, yv[u].z, yv[u].w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 f = widen2<T>(xw[k]), g = widen2<T>(yw[k]);
            s[u].x = fmaf(f.x, g.x, fmaf(f.y, g.y, s[u].x));
            if (kPeaks) s[u].y = fmaf(g.x, g.x, fmaf(g.y, g.y, s[u].y));
          }
        }
      } else {
        for (int u = 0; u < kTwo; ++u)
          for (int k = lane; y[u] != nullptr && k < p.D; k += LANES) {
            const float g = to_f32(y[u][k]);
            if (x[u] != nullptr) s[u].x = fmaf(to_f32(x[u][k]), g, s[u].x);
            s[u].y = fmaf(g, g, s[u].y);
          }
      }
#pragma unroll
      for (int u = 0; u < kTwo; ++u) {
        s[u] = lanes_sum<LANES>(s[u]);
        if (lane == 0 && y[u] != nullptr) use(at[u], h[u], s[u]);
      }
    }
  };
  scan(p.Tq, p.H,
       [&](int64_t r, int h, const T*& x, const T*& y) {
         x = static_cast<const T*>(p.o) + (r * p.H + h) * p.D;
         y = static_cast<const T*>(p.g) + r * p.g_t + h * p.g_h;
       },
       [&](int64_t r, int h, float2 s) {
         p.delta[(int64_t)h * p.Tq + r] = s.x;
         if (kPeaks) meet(p.q_off, p.Tq, (int)r, h / p.G, 0, s.y);
       });
  if constexpr (kPeaks) {
    raise(nullptr);
    segment = s_first[1].x;
    until = s_first[1].y;
    scan(p.Tk, p.Hk, [&](int64_t r, int h, const T*&, const T*& y) { y = static_cast<const T*>(p.v) + r * p.v_t + h * p.v_h; },
         [&](int64_t r, int h, float2 s) { meet(p.k_off, p.Tk, (int)r, h, 1, s.y); });
    raise(nullptr);
  }
}

// ------------------------------------------------------- tensor-core helpers
constexpr int kBlock = 64;    // of the other side that a step takes

// A wait for others of the CTA, with mbar_wait_bounded's budget, in as little code as will do: a wait stands between any
// two pieces of work here.  A try may sleep for up to a millisecond; the clock is read once in 64.
constexpr uint64_t kGivenUp = ~0ull;
__device__ __noinline__ uint64_t later(uint64_t since, int code, volatile int* abort_flag) {
  if (abort_flag != nullptr && *abort_flag) return kGivenUp;
  const uint64_t now = global_ns();
  if (since == 0) return now;
  if (now - since < kWaitBudgetNs) return since;
  raise_device_error(code);
  if (abort_flag != nullptr) *abort_flag = 1;
  return kGivenUp;
}
__device__ __forceinline__ bool wait_on(uint64_t* bar, uint32_t parity, int code, volatile int* abort_flag) {
  const uint32_t at = smem_u32(bar);
  uint32_t tries = 0, done;
  uint64_t since = 0;
  while (true) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(at), "r"(parity & 1u), "r"(1000000u)
        : "memory");
    if (done) return true;
    if ((++tries & 63u) == 0 && (since = later(since, code, abort_flag)) == kGivenUp) return false;
  }
}

// one arrival for a warp, whose lanes have all come here
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(smem_u32(bar));
}

// Operands under the 128-byte swizzle: 64 columns (128 bytes) a row, groups of eight rows 1024 bytes apart.  Their
// descriptors differ in the low word alone: the address, and how far on the next 64 columns lie where rows run along K.
// One thread issues all products, and what it computes between two of them holds the tensor cores up: so low words,
// loops unrolled, no division.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t rows_desc(uint32_t saddr) { return (saddr >> 4) | (1u << 16); }
__device__ __forceinline__ uint32_t columns_desc(uint32_t saddr, uint32_t next) { return (saddr >> 4) | ((next >> 4) << 16); }
// (without the operand that switches lanes of D off: with it one thread issued a product in 95 cycles, without in 50)
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)acc), "r"(kDescHigh));
}
// A from TMEM: sixteen 16-bit values of a row are eight words of its lane
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)acc), "r"(kDescHigh));
}
// where in operands of `rows` rows the i-th sixteen columns lie, in 16-byte units
__host__ __device__ constexpr uint32_t sixteenth(int i, int rows) { return (uint32_t)((i >> 2) * rows * 8 + (i & 3) * 2); }
// a position in a ring of S slots, and the parity of its use
template <int S>
struct Turn {
  int slot = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void next() {
    if (++slot == S) {
      slot = 0;
      parity ^= 1;
    }
  }
};
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* tm, int c0, int c1, int c2, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 32 columns of this thread's lane, to be used after tmem_wait_ld
__device__ __forceinline__ void tmem_get32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_put32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_get16(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_put8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_put16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return pack_bf16x2(lo, hi);
  else return pack_f16x2(lo, hi);
}
template <typename T>
__host__ __device__ constexpr uint32_t type_bits() { return std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u; }
// D fp32, M = 128, N columns; TURNED: B's rows run along K
template <typename T>
__host__ __device__ constexpr uint32_t idesc_of(int n, bool turned) {
  return (1u << 4) | type_bits<T>() | (turned ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}

// Weights meet the values as two values of the type: what a weight is rounded to, and what is left, rounded (2^-18 of it
// bf16, 2^-22 fp16).  In fp16 they are 2^7 times as large, so that those of 2^-25 of a row's largest are still there.
template <typename T>
constexpr float kLift = std::is_same<T, __half>::value ? 7.0f : 0.0f;
template <typename T>
__device__ __forceinline__ void two_values(F2 v, uint32_t& whole, uint32_t& rest) {
  const float2 f = un(v);
  whole = pack2<T>(f.x, f.y);
  const float2 top = widen2<T>(whole), left = un(sub2(v, f2(top.x, top.y)));
  rest = pack2<T>(left.x, left.y);
}

// A row of fp32 sums of `n` columns times w, as the type, to 16-byte aligned memory
template <typename T>
__device__ __forceinline__ void store_sums(T* to, const uint32_t* v, int n, float w, bool wide) {
#pragma unroll
  for (int c = 0; c < 32; c += 16) {
    uint32_t o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = pack2<T>(__uint_as_float(v[c + 2 * i]) * w, __uint_as_float(v[c + 2 * i + 1]) * w);
    if (c + 16 <= n && wide) {
      stg_v8(to + c, o);
    } else {
      if (c + 8 <= n) *reinterpret_cast<uint4*>(to + c) = make_uint4(o[0], o[1], o[2], o[3]);
      if (c + 16 <= n) *reinterpret_cast<uint4*>(to + c + 8) = make_uint4(o[4], o[5], o[6], o[7]);
    }
  }
}
__device__ __forceinline__ bool finite32(const uint32_t* v) {
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int q = 0; q < 32; ++q) s[q & 3] = fmaf(__uint_as_float(v[q]), 0.0f, s[q & 3]);
  const float all = (s[0] + s[1]) + (s[2] + s[3]);
  return all == all;
}

// whether all of the rows' N threads say so; they meet here
template <int N>
__device__ __forceinline__ bool rows_all(bool ok) {
  uint32_t every;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(every)
      : "r"((uint32_t)ok), "n"(N)
      : "memory");
  return every != 0;
}

// Half a block of neighbouring keys and the rows of a warp: seen by none of them, by all, or by some.
enum Seen : int { kNone = 0, kSome = 1, kEvery = 2 };
constexpr int kHalf = 32;
struct Span {  // of a warp's rows' intervals
  int lo_min, lo_max, hi_min, hi_max;
  __device__ Seen of(int j, int width = kHalf) const {  // of keys [j, j + width)
    return j + width <= lo_min || j >= hi_max ? kNone : j >= lo_max && j + width <= hi_min ? kEvery : kSome;
  }
};
__device__ __forceinline__ Span span_of(int4 row) {
  const bool sees = row.y > row.x;
  Span s;
  s.lo_min = __reduce_min_sync(kAll, sees ? row.x : INT_MAX);
  s.hi_max = __reduce_max_sync(kAll, sees ? row.y : 0);
  s.lo_max = __reduce_max_sync(kAll, row.x);
  s.hi_min = __reduce_min_sync(kAll, row.y);  // 0 with a row that sees nothing: kEvery never
  return s;
}

__device__ __forceinline__ F2 pair(const uint32_t* x) { return f2(__uint_as_float(x[0]), __uint_as_float(x[1])); }
__device__ __forceinline__ void put(uint32_t* x, F2 v) {
  const float2 f = un(v);
  x[0] = __float_as_uint(f.x);
  x[1] = __float_as_uint(f.y);
}
// scores in place of raw products, in units of log 2, of the 32 keys from j on
template <bool WIDE>
__device__ __forceinline__ void transform(const Params& p, uint32_t* raw, float slope2, int place, int j) {
  if constexpr (WIDE) {
    const float in = p.scale / p.cap, cap2 = p.cap * kLog2e;
#pragma unroll
    for (int c = 0; c < kHalf; ++c) raw[c] = __float_as_uint(cap2 * tanh_wide(__uint_as_float(raw[c]) * in));
  } else if (p.cap > 0.0f) {  // cap tanh(y) = cap - 2 cap / (1 + e^2y), as tanh_of has it
    const float in = p.scale / p.cap * (2.0f * kLog2e), cap2 = p.cap * kLog2e;
    const F2 in2 = f2(in, in), one = f2(1.0f, 1.0f), base = f2(cap2, cap2), minus = f2(-2.0f * cap2, -2.0f * cap2);
#pragma unroll
    for (int c = 0; c < kHalf; c += 2) {
      const float2 y = un(mul2(pair(raw + c), in2));
      const float2 d = un(add2(f2(exp2_fast(y.x), exp2_fast(y.y)), one));
      put(raw + c, fma2(f2(rcp_fast(d.x), rcp_fast(d.y)), minus, base));
    }
  }
  if (slope2 != 0.0f) {
    const float first = (float)(place - j), unit = p.cap > 0.0f ? 1.0f : p.scale * kLog2e;
#pragma unroll
    for (int c = 0; c < kHalf; ++c)
      raw[c] = __float_as_uint(fmaf(-slope2, fabsf(first - (float)c), __uint_as_float(raw[c]) * unit));
  }
}

// ---------------------------------------------------------------- forward
// A persistent CTA takes tiles of 128 rows of one head, the next by a ticket (long ones first), and treats their blocks
// of 64 keys as one stream: the thread that issues copies and MMAs asks for a block's keys and values kStages blocks
// ahead, in the next tile where this one ends, so that no tile waits for memory at its start.  With a CTA a tile, 1024
// users took 265 us: three quarters of a CTA's life went to its start and end.
//
// A row's thread goes over the block's scores in TMEM twice, 32 at a time: the maximum (scores that are masked or capped
// or fall with distance are put back in their place), then the weights, which go back as 16-bit values for the second
// product.  The running sum is fp32; the accumulator is rescaled only when a maximum has grown by more than 2^8 over
// what it is scaled to.  A weight goes into the second product as two values of the type (with the first alone `out` was
// 1.4 times as far from the exact sums as its own rounding makes it).  Rows whose sums are not finite are noted and taken again at the CTA's end.
//
// Bound by the row warps' issue slots (45 to 52 % used): 1024 users of 1 to 200 items in 8 heads of 64 take 132 us (their
// bytes 65; with weights of one value 117); two causal documents of 4100 to 7001 rows, 8 heads of 128, capped scores, 446 us
// (412).
template <int DP>
struct Forward {
  static constexpr int kChunks = DP / 64;              // 64 columns, a swizzled row
  static constexpr int kQBytes = kTile * 128 * kChunks;
  static constexpr int kKvBytes = kBlock * 128 * kChunks;
  static constexpr int kStages = 2;
  static constexpr int kSmem = 1024 + kQBytes + 2 * kStages * kKvBytes;
  // DP 64: the weights (both of their values) lie where the scores were, 128 columns in all, and four CTAs an SM fill each
  // other's waits; DP 128: apart, two CTAs, and the next block's scores are computed meanwhile
  static constexpr bool kApart = DP == 128;
  static constexpr int kPAt = kApart ? 64 : 0, kOAt = kApart ? 128 : 64;
  static constexpr int kTmemCols = kApart ? 256 : 128;
  static constexpr int kCtas = kApart ? 2 : 4;
  // warps that share 32 rows, each with half of a block's keys: sixteen warps of rows an SM either way
  static constexpr int kSets = kApart ? 2 : 1;
  static constexpr int kRowThreads = 128 * kSets, kThreads = 32 + kRowThreads;
};
constexpr int kItems = 4;  // tiles that are posted to the rows: theirs, up to two ahead, and one more
struct Item {
  int r0, r1, head, key0, blocks, unit;  // blocks 0: no more; unit: the ticket
};

template <typename T, int DP, bool WIDE>
__global__ void __launch_bounds__(Forward<DP>::kThreads, Forward<DP>::kCtas)
    forward_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                   const __grid_constant__ CUtensorMap tmV, const __grid_constant__ Params p) {
  using C = Forward<DP>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + C::kQBytes;
  uint8_t* sV = sK + C::kStages * C::kKvBytes;
  __shared__ __align__(8) uint64_t qfull, kfull[C::kStages], vfull[C::kStages], ifull[kItems];
  __shared__ __align__(8) uint64_t sfull, sfree, pready, pvdone, drained;
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  __shared__ Item s_item[kItems];
  // what the two warps of 32 rows tell each other: a row's maximum of either half (of this block and the next), its sums,
  // whether they are finite
  __shared__ __align__(8) uint64_t pairs[4];
  __shared__ float s_max[2][2][C::kSets == 2 ? kTile : 1], s_total[2][C::kSets == 2 ? kTile : 1];
  __shared__ int s_redo[C::kSets == 2 ? kTile : 1];
  __shared__ int s_redo_last[4];  // of 32 rows: the last unit with rows that are taken again, or -1
  volatile int* abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&qfull), 1);
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(smem_u32(&kfull[s]), 1);
      mbar_init(smem_u32(&vfull[s]), 1);
    }
    for (int s = 0; s < kItems; ++s) mbar_init(smem_u32(&ifull[s]), 1);
    mbar_init(smem_u32(&sfull), 1);
    mbar_init(smem_u32(&sfree), C::kRowThreads / 32);
    mbar_init(smem_u32(&pready), C::kRowThreads / 32);
    mbar_init(smem_u32(&pvdone), 1);
    mbar_init(smem_u32(&drained), 1);
    for (int q = 0; q < 4; ++q) {
      mbar_init(smem_u32(&pairs[q]), 2);
      s_redo_last[q] = -1;
    }
    abort_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmQ)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmK)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmV)) : "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(C::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = tmem_slot;
  asm volatile("griddepcontrol.wait;" ::: "memory");

  if (warp == 0) {
    if (lane == 0) {
      // -------------------------------------------------- copies and MMAs
      constexpr uint32_t idesc_s = idesc_of<T>(kBlock, false), idesc_o = idesc_of<T>(DP, true);
      auto wait = [&](uint64_t* bar, int n) { return wait_on(bar, (uint32_t)n, kWaitTimeoutMma, abort_flag); };
      const uint32_t items = (uint32_t)p.n_tiles * p.H;
      const uint32_t q_at = smem_u32(sQ), k_at = smem_u32(sK), v_at = smem_u32(sV);
      // `ahead`: the tile whose keys are asked for, the `posted`th, from block a_block on; the values follow, block v_block
      // of tile v_tile.  Posting overwrites what was posted four tiles ago: its blocks lie three tiles back at least and
      // the rows are past them.
      Item ahead{};
      int posted = 0, a_block = 0, k_asked = 0, v_tile = 0, v_block = 0, v_asked = 0, queried = 0;
      Turn<C::kStages> k_ask, v_ask, k_use, v_use;
      uint32_t ticket = atomicAdd(p.next, 1u);
      auto take = [&] {
        ahead.blocks = 0;
        a_block = 0;
        while (ticket < items && ahead.blocks == 0) {
          const int4 t = p.tiles[p.n_tiles - 1 - ticket / p.H];
          ahead = Item{t.x, t.y, (int)(ticket % p.H), t.z, t.w > t.z ? (t.w - t.z + kBlock - 1) / kBlock : 0, (int)ticket};
          ticket = atomicAdd(p.next, 1u);  // (needed a tile later)
        }
        s_item[posted % kItems] = ahead;
        mbar_arrive(smem_u32(&ifull[posted % kItems]));
        ++posted;
      };
      auto copy = [&](uint64_t* full, uint32_t to, const CUtensorMap* tm, int slot, int head, int key) {
        const uint32_t bar = smem_u32(&full[slot]);
        mbar_arrive_expect_tx(bar, C::kKvBytes);
#pragma unroll
        for (int c = 0; c < C::kChunks; ++c) tma_load_3d(to + slot * C::kKvBytes + c * kBlock * 128, tm, 64 * c, head / p.G, key, bar);
      };
      auto ask_k = [&] {  // for the next block's keys, whose slot is free
        if (ahead.blocks == 0) return;
        copy(kfull, k_at, &tmK, k_ask.slot, ahead.head, ahead.key0 + a_block * kBlock);
        k_ask.next();
        ++k_asked;
        if (++a_block == ahead.blocks) take();
      };
      auto ask_v = [&] {  // for its values
        if (v_asked == k_asked) return;
        const Item& it = s_item[v_tile % kItems];
        copy(vfull, v_at, &tmV, v_ask.slot, it.head, it.key0 + v_block * kBlock);
        v_ask.next();
        ++v_asked;
        if (++v_block == it.blocks) {
          v_block = 0;
          ++v_tile;
        }
      };
      auto ask_queries = [&](const Item& it) {
        const uint32_t bar = smem_u32(&qfull);
        mbar_arrive_expect_tx(bar, C::kQBytes);
#pragma unroll
        for (int c = 0; c < C::kChunks; ++c) tma_load_3d(q_at + c * kTile * 128, &tmQ, 64 * c, it.head, it.r0, bar);
        ++queried;
      };
      const int steps = (p.D + 15) / 16;  // of 16 columns (the rest of a row is zeros)
      auto scores = [&](bool first) {  // of the next block
        if (first && !wait(&qfull, queried - 1)) return false;
        if (!wait(&kfull[k_use.slot], k_use.parity)) return false;
        tc::tc_fence_after();
        const uint32_t qd = rows_desc(q_at), kd = rows_desc(k_at + k_use.slot * C::kKvBytes);
#pragma unroll
        for (int i = 0; i < DP / 16; ++i)
          if (i < steps) mma_ss(tmem, qd + sixteenth(i, kTile), kd + sixteenth(i, kBlock), idesc_s, i > 0);
        tc::umma_commit(smem_u32(&sfull));
        k_use.next();
        return true;
      };
      take();
      Item now = ahead;
      bool ok = true;
      if (now.blocks > 0) {
        ask_queries(now);
        for (int s = 0; s < C::kStages; ++s) {
          ask_k();
          ask_v();
        }
        ok = scores(true);
      }
      int t = 0;  // block of all tiles
      for (int tile = 0; now.blocks > 0 && ok; ++tile) {
        Item next{};
        for (int n = 0; n < now.blocks && ok; ++n, ++t) {
          const bool last = n + 1 == now.blocks;
          // (a tile is posted when the last block before it is asked for, kStages before this one is done)
          if (C::kApart) {  // the rows' threads have the scores: their columns are free, and their keys' slot
            ok = wait(&sfree, t);
            if (ok) {
              tc::tc_fence_after();
              if (!last) ok = scores(false);
              ask_k();
            }
          }
          ok = ok && wait(&vfull[v_use.slot], v_use.parity) && wait(&pready, t);
          if (!ok) break;
          tc::tc_fence_after();
          const uint32_t vd = columns_desc(v_at + v_use.slot * C::kKvBytes, kBlock * 128);
#pragma unroll
          for (int i = 0; i < kBlock / 16; ++i) {
            const uint32_t w = tmem + C::kPAt + (i >> 1) * kHalf + (i & 1) * 8;
            mma_ts(tmem + C::kOAt, w, vd + i * (16 * 128 / 16), idesc_o, n > 0 || i > 0);
            mma_ts(tmem + C::kOAt, w + kHalf / 2, vd + i * (16 * 128 / 16), idesc_o, true);
          }
          tc::umma_commit(smem_u32(&pvdone));
          v_use.next();
          if (last) {
            next = s_item[(tile + 1) % kItems];
            if (next.blocks > 0) ask_queries(next);
          }
          const bool more = !last || next.blocks > 0;
          if (C::kApart) {
            if (t > 0) ask_v();  // (into the slot of the block before: its product had ended before these weights were written)
            if (last && more) ok = scores(true);
          } else if (more) {
            ok = wait(&pvdone, t);
            if (ok) ok = scores(last);
            ask_k();
            ask_v();
          }
        }
        now = next;
      }
      if (!ok) {  // given up: no MMA in flight behind this CTA
        tc::umma_commit(smem_u32(&drained));
        wait_on(&drained, 0, kWaitTimeoutMma, nullptr);
      }
      // nor a copy
      if (queried > 0) wait_on(&qfull, (uint32_t)(queried - 1), kWaitTimeoutProducer, nullptr);
      for (int i = max(0, k_asked - C::kStages); i < k_asked; ++i) wait_on(&kfull[i % C::kStages], (uint32_t)(i / C::kStages), kWaitTimeoutProducer, nullptr);
      for (int i = max(0, v_asked - C::kStages); i < v_asked; ++i) wait_on(&vfull[i % C::kStages], (uint32_t)(i / C::kStages), kWaitTimeoutProducer, nullptr);
    }
  } else {
    // -------------------------------------------------------------- rows
    const int quarter = warp & 3, set = (warp - 1) >> 2;  // of the lanes of TMEM; of the columns
    const uint32_t mine = tmem + ((uint32_t)(quarter * 32) << 16);
    auto wait = [&](uint64_t* bar, int n) {
      return __all_sync(kAll, wait_on(bar, (uint32_t)n, kWaitTimeoutEpilogue, abort_flag)) != 0;
    };
    int met = 0;
    auto meet = [&] {  // the two warps of a quarter
      warp_arrive(&pairs[quarter]);
      return wait(&pairs[quarter], met++);
    };
    bool ok = wait(&ifull[0], 0);
    Item it = s_item[0];
    int4 row = make_int4(0, 0, 0, 0);
    if (ok && it.blocks > 0 && it.r0 + quarter * 32 + lane < it.r1) row = p.rows[it.r0 + quarter * 32 + lane];
    int t = 0;  // block of all tiles
    for (int tile = 0; ok && it.blocks > 0; ++tile) {
      const int r = it.r0 + quarter * 32 + lane, h = it.head;
      const float slope2 = p.slopes != nullptr ? kLog2e * __ldg(p.slopes + h) : 0.0f;
      const bool plain = p.cap == 0.0f && slope2 == 0.0f;
      const float unit = plain ? p.scale * kLog2e : 1.0f;
      const Span reach = span_of(row);
      float top = -INFINITY, total = 0.0f;  // top: what the weights are scaled to, in the scores' units
      for (int n = 0; n < it.blocks && ok; ++n, ++t) {
        const int j0 = it.key0 + n * kBlock;
        ok = wait(&sfull, t);
        if (!ok) break;
        tc::tc_fence_after();
        float high = -INFINITY;
        auto prepare = [&](uint32_t* x, int j, Seen seen) {  // scores of 32 keys, and their maximum
          if (!plain) transform<WIDE>(p, x, slope2, row.z, j);
          if (seen == kSome) {
            const int lo = row.x - j, len = max(row.y - row.x, 0);
#pragma unroll
            for (int c = 0; c < kHalf; ++c)
              if ((unsigned)(c - lo) >= (unsigned)len) x[c] = 0xff800000u;
          }
          float m[4] = {high, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < kHalf; c += 2) m[(c >> 1) & 3] = fmaxf(fmaxf(m[(c >> 1) & 3], __uint_as_float(x[c])), __uint_as_float(x[c + 1]));
          high = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
        };
        uint32_t held[C::kSets == 2 ? kHalf : 1];
        if constexpr (C::kSets == 2) {
          tmem_get32(mine + set * kHalf, held);
          tmem_wait_ld();
          tc::tc_fence_before();
          warp_arrive(&sfree);
          const Seen seen = reach.of(j0 + set * kHalf);
          if (seen != kNone) prepare(held, j0 + set * kHalf, seen);
          s_max[t & 1][set][quarter * 32 + lane] = high;
          ok = meet();
          high = fmaxf(high, s_max[t & 1][set ^ 1][quarter * 32 + lane]);
        } else {
          bool kept = false;
#pragma unroll 1
          for (int c0 = 0; c0 < kBlock; c0 += kHalf) {
            const Seen seen = reach.of(j0 + c0);
            if (seen == kNone) continue;
            uint32_t x[kHalf];
            tmem_get32(mine + c0, x);
            tmem_wait_ld();
            prepare(x, j0 + c0, seen);
            if (!plain || seen == kSome) {
              tmem_put32(mine + c0, x);
              kept = true;
            }
          }
          if (kept) tmem_wait_st();
        }
        const bool grow = (high - top) * unit > 8.0f || (top == -INFINITY && high > -INFINITY);
        if (C::kApart && n > 0) ok = ok && wait(&pvdone, t - 1);  // the product before has read its weights
        if (!ok) break;
        if (__any_sync(kAll, grow)) {
          if (n > 0) {
            const float keep = grow ? exp2_fast((top - high) * unit) : 1.0f;
            total *= keep;
            tc::tc_fence_after();
#pragma unroll 1
            for (int c = 32 * set; c < DP; c += 32 * C::kSets) {
              uint32_t o[32];
              tmem_get32(mine + C::kOAt + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
              tmem_put32(mine + C::kOAt + c, o);
            }
          }
          if (grow) top = high;
        }
        const float shift = top == -INFINITY ? 0.0f : fmaf(-top, unit, kLift<T>);
        const F2 unit2 = f2(unit, unit), shift2 = f2(shift, shift);
        F2 sum[2] = {f2(0.0f, 0.0f), f2(0.0f, 0.0f)};
        auto weigh = [&](const uint32_t* x, uint32_t* w) {
#pragma unroll
          for (int c = 0; c < kHalf; c += 2) {
            const float2 e = un(fma2(f2(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), unit2, shift2));
            const float a = exp2_fast(e.x), b = exp2_fast(e.y);
            sum[(c >> 1) & 1] = add2(sum[(c >> 1) & 1], f2(a, b));
            two_values<T>(f2(a, b), w[c / 2], w[kHalf / 2 + c / 2]);
          }
        };
#pragma unroll 1
        for (int c0 = C::kSets == 2 ? set * kHalf : 0; c0 < (C::kSets == 2 ? (set + 1) * kHalf : kBlock); c0 += kHalf) {
          uint32_t w[kHalf];  // of 32 keys: what the weights are rounded to, and what is left, in the scores' columns
          if (reach.of(j0 + c0) == kNone) {
#pragma unroll
            for (int c = 0; c < kHalf; ++c) w[c] = 0u;
          } else if constexpr (C::kSets == 2) {
            weigh(held, w);
          } else {
            uint32_t x[kHalf];
            tmem_get32(mine + c0, x);
            tmem_wait_ld();
            weigh(x, w);
          }
          tmem_put32(mine + C::kPAt + c0, w);
        }
        const float2 s2 = un(add2(sum[0], sum[1]));
        total += s2.x + s2.y;
        tmem_wait_st();
        tc::tc_fence_before();
        warp_arrive(&pready);
      }
      // the next tile's intervals come while the last product runs
      ok = ok && wait(&ifull[(tile + 1) % kItems], (tile + 1) / kItems);
      if (!ok) break;
      const Item next = s_item[(tile + 1) % kItems];
      int4 next_row = make_int4(0, 0, 0, 0);
      if (next.blocks > 0 && next.r0 + quarter * 32 + lane < next.r1) next_row = p.rows[next.r0 + quarter * 32 + lane];
      ok = wait(&pvdone, t - 1);
      if (!ok) break;
      tc::tc_fence_after();
      const bool sees = row.y > row.x, there = r < it.r1;
      if constexpr (C::kSets == 2) {
        s_total[set][quarter * 32 + lane] = total;
        ok = meet();
        if (!ok) break;
        total += s_total[set ^ 1][quarter * 32 + lane];
      }
      const float w = total == 0.0f ? 0.0f : 1.0f / total;
      T* out = static_cast<T*>(p.out) + ((int64_t)r * p.H + h) * p.D;
      const bool wide = p.D % 16 == 0 && aligned(p.out, 32);
      bool redo = sees && !(total < INFINITY);
#pragma unroll 1
      for (int c = 32 * set; c < p.D; c += 32 * C::kSets) {
        uint32_t o[32];
        tmem_get32(mine + C::kOAt + c, o);
        tmem_wait_ld();
        if (!sees) {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        } else {
          redo = redo || !finite32(o);
        }
        if (there) store_sums<T>(out + c, o, p.D - c, sees ? w : 0.0f, wide);
      }
      if (there && p.lse != nullptr && set == 0)
        p.lse[(int64_t)h * p.Tq + r] = sees && total != 0.0f ? kLn2 * fmaf(top, unit, log2f(total) - kLift<T>) : -INFINITY;
      if constexpr (C::kSets == 2) {  // what either finds not finite in its columns the first takes again, once both have stored
        if (set == 1) s_redo[quarter * 32 + lane] = redo;
        ok = meet();
        if (!ok) break;
        redo = set == 0 && (redo || s_redo[quarter * 32 + lane] != 0);
      }
      // (not here: others of this CTA wait for the next tile's rows, and a row over long keys takes longer than they do)
      const uint32_t again = __ballot_sync(kAll, redo && there);
      if (again != 0 && lane == 0) {
        p.redo[(int64_t)it.unit * 4 + quarter] = make_int2((int)again, s_redo_last[quarter]);
        s_redo_last[quarter] = it.unit;
      }
      it = next;
      row = next_row;
    }
    // the rows that were not finite, one by one, when nothing waits for this warp but the CTA's end
    __syncwarp();
    for (int unit = set == 0 ? s_redo_last[quarter] : -1; unit >= 0;) {
      const int2 entry = p.redo[(int64_t)unit * 4 + quarter];
      const int r0 = p.tiles[p.n_tiles - 1 - unit / p.H].x + quarter * 32, h = unit % p.H;
      for (uint32_t again = (uint32_t)entry.x; again != 0; again &= again - 1) {
        row_forward<T>(p, r0 + __ffs(again) - 1, h);
        __syncwarp();
      }
      unit = entry.y;
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmemCols) : "memory");
  }
}

// ------------------------------------------------- few queries, long histories
// Some queries of a segment over many keys (a user's new items over a cached history): bound by reading the keys and
// values once.  A CTA takes 16 rows (a key head's query heads, for one token or several) and one of `splits` parts of
// the segment's keys, so that a single query still fills the GPU; a producer warp keeps kStages blocks of 64 keys
// coming, and each of four warps takes 16 keys of a block with products of 16 x 8 x 16 (most of the 128 rows of the
// larger tensor-core products would be empty here).  Warps, then parts, are added up in their order.  64 queries of 16 heads
// (4 key heads of 128) over 1000 to 16000 keys each: 204 us, 0.9 of the copy rate.
template <int DP>
struct Few {
  static constexpr int kRows = 16, kWarps = 4, kThreads = 32 * (kWarps + 1);
  static constexpr int kChunks = DP / 64;
  static constexpr int kBytes = kBlock * 128 * kChunks;  // of a block's keys, and of its values
  static constexpr int kStages = DP == 64 ? 4 : 3;
  static constexpr int kSmem = 1024 + kStages * 2 * kBytes;
  static constexpr int kCtas = DP == 64 ? 3 : 2;
  static_assert(kWarps * kRows * (DP + 4) * 4 <= kStages * 2 * kBytes, "the warps' sums lie where the blocks did");
};
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_turned(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T, int DP>
__global__ void __launch_bounds__(Few<DP>::kThreads, Few<DP>::kCtas)
    few_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ Params p) {
  using C = Few<DP>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(8) uint64_t full[C::kStages], empty[C::kStages];
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = blockIdx.x / p.splits, split = blockIdx.x % p.splits, hk = blockIdx.y;
  const int2 span = tile_rows(p.q_off, p.off64, p.S, p.Tq, tile, 1, C::kRows, p.G);
  if (span.x >= span.y) return;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), C::kWarps);
    }
    abort_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncthreads();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // rows g and g + 8 of the tile are this thread's; a row is (token, head of the group)
  const int g = lane >> 2, q4 = lane & 3;
  int4 mine[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = span.x + g + 8 * i;
    mine[i] = row < span.y ? p.rows[row / p.G] : make_int4(0, 0, 0, 0);
  }
  const Span a = span_of(mine[0]), b = span_of(mine[1]);
  const int lo = min(a.lo_min, b.lo_min), hi = max(a.hi_max, b.hi_max);  // of all rows
  const int all_lo = max(a.lo_max, b.lo_max), all_hi = min(a.hi_min, b.hi_min);
  // this part of the keys: whole blocks
  const int blocks_all = hi > lo ? (hi - lo + kBlock - 1) / kBlock : 0;
  const int first = (int)((int64_t)blocks_all * split / p.splits), blocks = (int)((int64_t)blocks_all * (split + 1) / p.splits) - first;
  const int key0 = lo + first * kBlock;

  if (warp == C::kWarps) {
    if (lane == 0) {
      int n = 0;
      for (; n < blocks; ++n) {
        const int s = n % C::kStages;
        if (!wait_on(&empty[s], (uint32_t)(n / C::kStages) ^ 1u, kWaitTimeoutProducer, abort_flag)) break;
        const uint32_t bar = smem_u32(&full[s]), to = smem_u32(smem + s * 2 * C::kBytes);
        mbar_arrive_expect_tx(bar, 2 * C::kBytes);
        for (int c = 0; c < C::kChunks; ++c) {
          tma_load_3d(to + c * kBlock * 128, &tmK, 64 * c, hk, key0 + n * kBlock, bar);
          tma_load_3d(to + C::kBytes + c * kBlock * 128, &tmV, 64 * c, hk, key0 + n * kBlock, bar);
        }
      }
      for (int i = max(0, n - C::kStages); i < n; ++i) wait_on(&full[i % C::kStages], (uint32_t)(i / C::kStages), kWaitTimeoutProducer, nullptr);
    }
  }
  float top[2] = {-INFINITY, -INFINITY}, total[2] = {0.0f, 0.0f}, o[DP / 8][4];
#pragma unroll
  for (int i = 0; i < DP / 8; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) o[i][c] = 0.0f;
  bool ok = true;
  if (warp < C::kWarps && blocks > 0) {
    uint32_t q[DP / 16][4];
#pragma unroll
    for (int k = 0; k < DP / 16; ++k)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int row = span.x + g + 8 * (c & 1), col = 16 * k + 8 * (c >> 1) + 2 * q4;
        const T* from = static_cast<const T*>(p.q) + (int64_t)(row / p.G) * p.q_t + (int64_t)(hk * p.G + row % p.G) * p.q_h + col;
        q[k][c] = row < span.y && col < p.D ? __ldg(reinterpret_cast<const uint32_t*>(from)) : 0u;
      }
    float slope2[2] = {0.0f, 0.0f};
    if (p.slopes != nullptr)
#pragma unroll
      for (int i = 0; i < 2; ++i) slope2[i] = kLog2e * __ldg(p.slopes + hk * p.G + (span.x + g + 8 * i) % p.G);
    const float unit = p.cap > 0.0f ? 1.0f : p.scale * kLog2e;
    const int key = 16 * warp + (lane & 7) + 8 * ((lane >> 3) & 1);  // the row of a block that this lane points ldmatrix at
    const int half = lane >> 4;                                      // and which eight of sixteen columns
    for (int n = 0; n < blocks; ++n) {
      const int s = n % C::kStages, j0 = key0 + n * kBlock + 16 * warp;
      ok = __all_sync(kAll, wait_on(&full[s], (uint32_t)(n / C::kStages), kWaitTimeoutEpilogue, abort_flag));
      if (!ok) break;
      if (j0 < hi) {
        const uint32_t at = smem_u32(smem + s * 2 * C::kBytes) + key * 128;
        float x[2][4];
#pragma unroll
        for (int c = 0; c < 4; ++c) x[0][c] = x[1][c] = 0.0f;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          uint32_t r[4];  // keys 0-7 and 8-15 of the first eight columns, then of the second
          ldsm4(at + (k >> 2) * kBlock * 128 + ((((k & 3) * 2 + half) ^ (key & 7)) << 4), r);
          mma16<T>(x[0], q[k], r[0], r[2]);
          mma16<T>(x[1], q[k], r[1], r[3]);
        }
        // x[e][2 i + d]: row g + 8 i, key j0 + 8 e + 2 q4 + d
        const bool every = j0 >= all_lo && j0 + 16 <= all_hi;
        float high[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int i = c >> 1, j = j0 + 8 * e + 2 * q4 + (c & 1);
            float v = x[e][c];
            if (p.cap > kWideCap) v = p.cap * kLog2e * tanh_wide(v * (p.scale / p.cap));
            else if (p.cap > 0.0f) v = p.cap * kLog2e * tanh_of(v * (p.scale / p.cap));
            else v *= unit;
            v = fmaf(-slope2[i], (float)abs(mine[i].z - j), v);
            if (!every && !(j >= mine[i].x && j < mine[i].y)) v = -INFINITY;
            x[e][c] = v;
            high[i] = fmaxf(high[i], v);
          }
        float keep[2], shift[2];
        bool grow = false;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          high[i] = fmaxf(high[i], __shfl_xor_sync(kAll, high[i], 1));
          high[i] = fmaxf(high[i], __shfl_xor_sync(kAll, high[i], 2));
          keep[i] = 1.0f;
          if (high[i] > top[i] + 8.0f || (top[i] == -INFINITY && high[i] > -INFINITY)) {
            keep[i] = exp2_fast(top[i] - high[i]);
            top[i] = high[i];
            grow = true;
          }
          shift[i] = top[i] == -INFINITY ? 0.0f : top[i] - kLift<T>;
        }
        if (__any_sync(kAll, grow)) {
#pragma unroll
          for (int i = 0; i < DP / 8; ++i) {
            o[i][0] *= keep[0];
            o[i][1] *= keep[0];
            o[i][2] *= keep[1];
            o[i][3] *= keep[1];
          }
          total[0] *= keep[0];
          total[1] *= keep[1];
        }
        uint32_t w[4], rest[4];
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float u = exp2_fast(x[e][2 * i] - shift[i]), v = exp2_fast(x[e][2 * i + 1] - shift[i]);
            total[i] += u + v;
            two_values<T>(f2(u, v), w[2 * e + i], rest[2 * e + i]);
          }
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          uint32_t r[4];  // keys 0-7 and 8-15 of eight columns, then of the next eight
          ldsm4_turned(at + C::kBytes + (k >> 2) * kBlock * 128 + ((((k & 3) * 2 + half) ^ (key & 7)) << 4), r);
          mma16<T>(o[2 * k], w, r[0], r[1]);
          mma16<T>(o[2 * k + 1], w, r[2], r[3]);
          mma16<T>(o[2 * k], rest, r[0], r[1]);
          mma16<T>(o[2 * k + 1], rest, r[2], r[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&empty[s]));
    }
  }
  ok = __syncthreads_and(ok);
  if (!ok) return;
  // the warps' sums, on one maximum: [warp][row][D], then maximum and sum
  float* sums = reinterpret_cast<float*>(smem);
  float* tops = sums + C::kWarps * C::kRows * DP;
  float* totals = tops + C::kWarps * C::kRows;
  if (warp < C::kWarps) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      total[i] += __shfl_xor_sync(kAll, total[i], 1);
      total[i] += __shfl_xor_sync(kAll, total[i], 2);
      if (q4 == 0) {
        tops[warp * C::kRows + g + 8 * i] = top[i];
        totals[warp * C::kRows + g + 8 * i] = total[i];
      }
    }
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) {
      float* to = sums + (warp * C::kRows + g) * DP + 8 * i + 2 * q4;
      *reinterpret_cast<float2*>(to) = make_float2(o[i][0], o[i][1]);
      *reinterpret_cast<float2*>(to + 8 * DP) = make_float2(o[i][2], o[i][3]);
    }
  }
  __syncthreads();
  const int rows = span.y - span.x;
  for (int r = warp; r < rows; r += C::kWarps + 1) {  // a warp a row
    float high = -INFINITY, sum = 0.0f, scale[C::kWarps];
#pragma unroll
    for (int w = 0; w < C::kWarps; ++w) high = fmaxf(high, tops[w * C::kRows + r]);
#pragma unroll
    for (int w = 0; w < C::kWarps; ++w) {
      scale[w] = high == -INFINITY ? 1.0f : exp2_fast(tops[w * C::kRows + r] - high);
      sum = fmaf(scale[w], totals[w * C::kRows + r], sum);
    }
    const int token = (span.x + r) / p.G, h = hk * p.G + (span.x + r) % p.G;
    const int64_t at = (int64_t)token * p.H + h;
    bool finite = sum < INFINITY;
    for (int c = lane; c < p.D; c += 32) {
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < C::kWarps; ++w) v = fmaf(scale[w], sums[(w * C::kRows + r) * DP + c], v);
      if (p.splits > 1) {
        p.part[(at * p.splits + split) * (p.D + 2) + c] = v;
      } else {
        finite = finite && fabsf(v) < INFINITY;
        static_cast<T*>(p.out)[at * p.D + c] = T(sum == 0.0f ? 0.0f : v / sum);
      }
    }
    if (p.splits > 1) {
      if (lane < 2) p.part[(at * p.splits + split) * (p.D + 2) + p.D + lane] = lane ? sum : high;
    } else {
      if (lane == 0 && p.lse != nullptr) p.lse[(int64_t)h * p.Tq + token] = sum == 0.0f ? -INFINITY : kLn2 * (high + (log2f(sum) - kLift<T>));
      if (!__all_sync(kAll, finite)) {
        __syncwarp();
        row_forward<T>(p, token, h);
      }
    }
  }
}

// the parts of a row, a warp a row of one head
template <typename T>
__global__ void __launch_bounds__(256) few_join_kernel(const __grid_constant__ Params p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int64_t at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (at >= (int64_t)p.Tq * p.H) return;
  const float* part = p.part + at * p.splits * (p.D + 2);
  float high = -INFINITY, sum = 0.0f;
  for (int s = lane; s < p.splits; s += 32) high = fmaxf(high, part[s * (p.D + 2) + p.D]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) high = fmaxf(high, __shfl_xor_sync(kAll, high, o));
  for (int s = 0; s < p.splits; ++s) {
    const float w = high == -INFINITY ? 1.0f : exp2_fast(part[s * (p.D + 2) + p.D] - high);
    sum = fmaf(w, part[s * (p.D + 2) + p.D + 1], sum);
  }
  bool finite = sum < INFINITY;
  for (int c = lane; c < p.D; c += 32) {
    float v = 0.0f;
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) {
      const float w = high == -INFINITY ? 1.0f : exp2_fast(part[s * (p.D + 2) + p.D] - high);
      v = fmaf(w, part[s * (p.D + 2) + c], v);
    }
    finite = finite && fabsf(v) < INFINITY;
    static_cast<T*>(p.out)[at * p.D + c] = T(sum == 0.0f ? 0.0f : v / sum);
  }
  const int token = (int)(at / p.H), h = (int)(at % p.H);
  if (lane == 0 && p.lse != nullptr) p.lse[(int64_t)h * p.Tq + token] = sum == 0.0f ? -INFINITY : kLn2 * (high + (log2f(sum) - kLift<T>));
  if (!__all_sync(kAll, finite)) {
    __syncwarp();
    row_forward<T>(p, token, h);
  }
}


// --------------------------------------------------------------- backward
// Two kernels of one form, and no atomics: the same bits every time.  KEYS false: a CTA's 128 rows are queries of one
// head, it goes over blocks of 64 keys and sums dq.  KEYS true: its rows are keys of one key head, it goes over blocks
// of 64 queries of every head that shares it and sums dk and dv.  With (A1, A2) the resident tiles and (B1, B2) the
// blocks, (Q, dO) and (K, V) or the other way round, a block is
//
//   S = A1 B1^T   dP = A2 B2^T   p = exp(s - lse)   e = p (dP - delta) (1 - tanh^2)   acc += e B1   [dv += p B2]
//
// delta_i = sum_j p_ij dP_ij.  As dO_i . out_i, which delta_kernel has, it is off by what rounding `out` left off, and where
// few keys hold a row's weight dP - delta is a small difference beside that (dq and dk of such rows had no right digit).
// The queries' kernel comes first and sums what it is off by: d_i = sum_j p_ij (dP_ij - delta_i), and with it
// dq_i = acc_i - d_i sum_j p_ij (1 - tanh^2)_ij k_j, whose last sum is its second accumulator (of p rounded once: d is
// small).  delta_i + d_i is what the keys' kernel gets.
//
// seven products for both where one kernel that adds dq by atomics has five, the queries' second sum apart.  p and e go to the second products as two
// values of the type each, out of TMEM: what they are rounded to, and what is left, rounded.  (With the first alone dq, dk
// and dv are 1.3 to 1.4 times as far from the exact sums, 2.4e-3 for 1.7e-3 in bf16.)  In fp16 they are brought into the
// type's range first: p by 2^15, e by that and the power of two that keeps |dP - delta| of the row's own segment and key head
// under 1 (from the largest norms of a row of dO and of V there): what other users hold does not take bits from a row.
//
// Bound by the row warps' issue slots (44 to 55 % used, the tensor pipe 36 to 39 % busy at 128 columns): two causal documents
// of 4100 to 7001 rows, 8 heads over 2 of 128: dk and dv 604 us, dq 486; 60 users of 10 to 1000 items, 8 heads of 64, fp16:
// 209 and 182, the latter (38 % of the slots) waiting for products, since its second accumulator leaves S and dP no columns
// beside p and e (138 with one accumulator and p and e apart).
template <int DP, bool KEYS>
struct Backward {
  static constexpr int kChunks = DP / 64;
  static constexpr int kABytes = kTile * 128 * kChunks;   // each of A1, A2
  static constexpr int kBBytes = kBlock * 128 * kChunks;  // each of B1, B2
  static constexpr int kStages = 4;
  static constexpr int kSmem = 1024 + 2 * kABytes + 2 * kStages * kBBytes;
  // Warps that share 32 rows, each with its part of a block's columns, kPart at a time: sixteen warps of rows an SM.  (With
  // eight, issue slots were used to 25 % and two long documents' gradients took 1.69 ms.)
  static constexpr int kSets = DP == 64 ? 2 : 4, kPart = 16, kSteps = kBlock / kPart / kSets;
  static constexpr int kRowThreads = 128 * kSets, kThreads = 64 + kRowThreads;
  static constexpr int kCtas = DP == 64 ? 2 : 1;
  // TMEM: S, dP, then the sums; the 16-bit values beside them (the next S and dP are then computed meanwhile) or in
  // place of S and dP, where two CTAs of 256 columns leave no room
  static constexpr int kAccAt = 128, kAcc2At = 128 + DP;
  static constexpr bool kApart = DP != 64;
  static constexpr int kEAt = kApart ? kAcc2At + DP : 64;
  static constexpr int kPAt = kApart ? kEAt + 64 : 0;
  static constexpr int kStride = 16;                      // sixteen of p or e as they are rounded, then what is left of them
  static constexpr int kTmemCols = DP == 64 ? 256 : 512;
};

template <typename T, int DP, bool KEYS, bool WIDE>
__global__ void __launch_bounds__(Backward<DP, KEYS>::kThreads, Backward<DP, KEYS>::kCtas)
    backward_kernel(const __grid_constant__ CUtensorMap tmA1, const __grid_constant__ CUtensorMap tmA2,
                    const __grid_constant__ CUtensorMap tmB1, const __grid_constant__ CUtensorMap tmB2,
                    const __grid_constant__ Params p) {
  using C = Backward<DP, KEYS>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* sA1 = smem;
  uint8_t* sA2 = sA1 + C::kABytes;
  uint8_t* sB1 = sA2 + C::kABytes;
  uint8_t* sB2 = sB1 + C::kStages * C::kBBytes;
  __shared__ __align__(8) uint64_t afull, bfull[C::kStages], sfull, sfree, ready, done, drained[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word, s_bad[kTile];
  // of the block's queries (KEYS), for this block and the next: lse and delta (negative), interval and place; and, of its
  // halves, what all of them see together
  __shared__ __align__(16) float s_lse[2][KEYS ? kBlock : 4], s_delta[2][KEYS ? kBlock : 4];
  __shared__ int4 s_row[2][KEYS ? kBlock : 1];
  __shared__ Span s_span[2][2];
  __shared__ float s_off[KEYS ? 1 : C::kSets][KEYS ? 1 : kTile];  // (queries) what delta is off by, of a set's columns
  volatile int* abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // (KEYS) blockIdx.z: one of the heads that share the key head, where there are parts; else all of them
  const int head = blockIdx.y, heads = KEYS && p.parts ? 1 : p.G, first_head = head * p.G + (KEYS ? (int)blockIdx.z : 0);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 span = *(KEYS ? p.key_tiles + blockIdx.x : p.tiles + (gridDim.x - 1 - blockIdx.x));  // (long ones first)
  if (span.x >= span.y) return;

  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&afull), 1);
    for (int s = 0; s < C::kStages; ++s) mbar_init(smem_u32(&bfull[s]), 1);
    mbar_init(smem_u32(&sfull), 1);
    mbar_init(smem_u32(&sfree), C::kRowThreads / 32);
    mbar_init(smem_u32(&ready), C::kRowThreads / 32);
    mbar_init(smem_u32(&done), 1);
    for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&drained[i]), 1);
    abort_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (threadIdx.x < kTile) s_bad[threadIdx.x] = 0;
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(C::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  const int quarter = warp & 3, set = (warp - 2) >> 2;
  const int r = span.x + quarter * 32 + lane;  // the thread's query or key
  int4 row = make_int4(0, 0, 0, 0);
  if (!KEYS && warp >= 2 && r < span.y) row = p.rows[r];
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const int other0 = span.z, other1 = span.w;
  const int each = other1 > other0 ? (other1 - other0 + kBlock - 1) / kBlock : 0;  // blocks of a head
  const int blocks = KEYS ? each * heads : each;
  const int up = std::is_same<T, __half>::value ? 15 : 0;
  float sigma = 1.0f;  // of the thread's row
  if (up != 0 && warp >= 2 && r < span.y) sigma = range_of(p, KEYS ? p.key_segments[r] : row.w, KEYS ? head : head / p.G);

  if (warp == 0) {
    if (lane == 0 && blocks > 0) {
      // ----------------------------------------- the resident tiles, S and dP
      constexpr uint32_t idesc = idesc_of<T>(kBlock, false);
      auto wait = [&](uint64_t* bar, uint32_t parity) { return wait_on(bar, parity, kWaitTimeoutMma, abort_flag); };
      const uint32_t a1_at = smem_u32(sA1), a2_at = smem_u32(sA2), b1_at = smem_u32(sB1), b2_at = smem_u32(sB2), ab = smem_u32(&afull);
      mbar_arrive_expect_tx(ab, 2 * C::kABytes);
#pragma unroll
      for (int c = 0; c < C::kChunks; ++c) {
        tma_load_3d(a1_at + c * kTile * 128, &tmA1, 64 * c, head, span.x, ab);
        tma_load_3d(a2_at + c * kTile * 128, &tmA2, 64 * c, head, span.x, ab);
      }
      Turn<C::kStages> used;
      const int steps = (p.D + 15) / 16;
      const uint32_t a1 = rows_desc(a1_at), a2 = rows_desc(a2_at);
      bool ok = wait(&afull, 0);
      for (int n = 0; n < blocks && ok; ++n) {
        ok = wait(&bfull[used.slot], used.parity);
        if (n > 0) ok = ok && wait(C::kApart ? &sfree : &done, (uint32_t)(n - 1));  // S's and dP's columns
        if (!ok) break;
        tc::tc_fence_after();
        const uint32_t b1 = rows_desc(b1_at + used.slot * C::kBBytes), b2 = rows_desc(b2_at + used.slot * C::kBBytes);
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
          if (i >= steps) continue;
          mma_ss(tmem, a1 + sixteenth(i, kTile), b1 + sixteenth(i, kBlock), idesc, i > 0);
          mma_ss(tmem + 64, a2 + sixteenth(i, kTile), b2 + sixteenth(i, kBlock), idesc, i > 0);
        }
        tc::umma_commit(smem_u32(&sfull));
        used.next();
      }
      if (!ok) {  // given up: no MMA in flight behind this CTA
        tc::umma_commit(smem_u32(&drained[0]));
        wait_on(&drained[0], 0, kWaitTimeoutMma, nullptr);
      }
      wait_on(&afull, 0, kWaitTimeoutProducer, nullptr);  // nor a copy
    }
  } else if (warp == 1) {
    if (lane == 0 && blocks > 0) {
      // ---------------------------------------------- the blocks, the sums
      constexpr uint32_t idesc = idesc_of<T>(DP, true);
      auto wait = [&](uint64_t* bar, uint32_t parity) { return wait_on(bar, parity, kWaitTimeoutMma, abort_flag); };
      const uint32_t b1_at = smem_u32(sB1), b2_at = smem_u32(sB2);
      int asked = 0, a_block = 0, a_head = KEYS ? first_head : head / p.G;
      Turn<C::kStages> ring, held;  // what is asked for next, what the sums take next
      auto ask = [&] {
        if (asked >= blocks) return;
        ++asked;
        const int at = other0 + a_block * kBlock;
        const uint32_t bar = smem_u32(&bfull[ring.slot]), to = ring.slot * C::kBBytes;
        mbar_arrive_expect_tx(bar, 2 * C::kBBytes);
#pragma unroll
        for (int c = 0; c < C::kChunks; ++c) {
          tma_load_3d(b1_at + to + c * kBlock * 128, &tmB1, 64 * c, a_head, at, bar);
          tma_load_3d(b2_at + to + c * kBlock * 128, &tmB2, 64 * c, a_head, at, bar);
        }
        ring.next();
        if (++a_block == each) {
          a_block = 0;
          ++a_head;
        }
      };
      for (int s = 0; s < C::kStages; ++s) ask();
      bool ok = true;
      for (int n = 0; n < blocks; ++n) {
        ok = wait(&bfull[held.slot], held.parity) && wait(&ready, (uint32_t)n);
        if (!ok) break;
        tc::tc_fence_after();
        const uint32_t b1 = columns_desc(b1_at + held.slot * C::kBBytes, kBlock * 128), b2 = columns_desc(b2_at + held.slot * C::kBBytes, kBlock * 128);
#pragma unroll
        for (int i = 0; i < kBlock / 16; ++i) {
          mma_ts(tmem + C::kAcc2At, tmem + C::kPAt + C::kStride * i, (KEYS ? b2 : b1) + i * (16 * 128 / 16), idesc, n > 0 || i > 0);
          if (KEYS) mma_ts(tmem + C::kAcc2At, tmem + C::kPAt + C::kStride * i + 8, b2 + i * (16 * 128 / 16), idesc, true);
          mma_ts(tmem + C::kAccAt, tmem + C::kEAt + C::kStride * i, b1 + i * (16 * 128 / 16), idesc, n > 0 || i > 0);
          mma_ts(tmem + C::kAccAt, tmem + C::kEAt + C::kStride * i + 8, b1 + i * (16 * 128 / 16), idesc, true);
        }
        tc::umma_commit(smem_u32(&done));
        held.next();
        if (n > 0) ask();  // (into the slot of the block before: its sums had ended before these values were written)
      }
      if (!ok) {
        tc::umma_commit(smem_u32(&drained[1]));
        wait_on(&drained[1], 0, kWaitTimeoutMma, nullptr);
      }
      for (int i = max(0, asked - C::kStages); i < asked; ++i) wait_on(&bfull[i % C::kStages], (uint32_t)(i / C::kStages), kWaitTimeoutProducer, nullptr);
    }
  } else {
    // -------------------------------------------------------------- rows
    const int t = threadIdx.x - 64;
    const uint32_t mine = tmem + ((uint32_t)(quarter * 32) << 16);
    const float unit = p.cap > 0.0f ? p.cap * kLog2e : p.scale * kLog2e;
    float slope2 = 0.0f, lse = 0.0f, delta = 0.0f;
    F2 off = f2(0.0f, 0.0f);
    Span reach{};
    if (!KEYS) reach = span_of(row);
    if (!KEYS) {
      slope2 = p.slopes != nullptr ? kLog2e * __ldg(p.slopes + head) : 0.0f;
      lse = r < span.y ? lse_of(p, r, head) - up : INFINITY;
      delta = r < span.y ? sigma * p.delta[(int64_t)head * p.Tq + r] : 0.0f;
    }
    // a block's queries, by the first two warps of the rows: from memory, then to shared memory
    float next_lse = INFINITY, next_delta = 0.0f;
    int4 next_row = make_int4(0, 0, 0, 0);
    auto fetch = [&](int n) {
      if (t >= kBlock) return;
      const int i = other0 + (n % each) * kBlock + t, h = first_head + n / each;
      const bool there = i < other1;
      next_row = there ? p.rows[i] : make_int4(0, 0, 0, 0);
      next_lse = there ? lse_of(p, i, h) - up : INFINITY;
      next_delta = there ? p.delta[(int64_t)h * p.Tq + i] : 0.0f;  // (times the range, which a query and its keys share)
    };
    auto deposit = [&](int n) {
      if (t < kBlock) {
        s_lse[n & 1][t] = -next_lse;
        s_delta[n & 1][t] = -next_delta;
        s_row[n & 1][t] = next_row;
        const Span span = span_of(next_row);
        if (lane == 0) s_span[n & 1][t >> 5] = span;
      }
    };
    auto meet = [](bool good) { return rows_all<C::kRowThreads>(good); };
    bool ok = true;
    if (KEYS && blocks > 0) {
      fetch(0);
      deposit(0);
      meet(true);
      if (blocks > 1) fetch(1);
    }
    for (int n = 0; n < blocks && ok; ++n) {
      const int o0 = other0 + (KEYS ? n % each : n) * kBlock;
      if (KEYS) slope2 = p.slopes != nullptr ? kLog2e * __ldg(p.slopes + first_head + n / each) : 0.0f;
      ok = __all_sync(kAll, wait_on(&sfull, (uint32_t)n, kWaitTimeoutEpilogue, abort_flag));
      tc::tc_fence_after();
#pragma unroll 1
      for (int step = 0; step < C::kSteps && ok; ++step) {
        const int c0 = (set * C::kSteps + step) * C::kPart;
        // of these keys (queries) and the warp's rows: is there one that sees, do all
        const Seen seen = KEYS ? s_span[n & 1][c0 / kHalf].of(span.x + quarter * 32) : reach.of(o0 + c0, C::kPart);
        uint32_t w[C::kPart], e[C::kPart];
        if (seen != kNone) {
          uint32_t x[C::kPart], y[C::kPart], slant[KEYS ? 1 : C::kPart];
          tmem_get16(mine + c0, x);
          tmem_get16(mine + 64 + c0, y);
          tmem_wait_ld();
          if (C::kApart && step == C::kSteps - 1) {  // the next block's products may begin
            tc::tc_fence_before();
            warp_arrive(&sfree);
          }
          // y: dP - delta (KEYS: times the slant 1 - tanh^2); x: the score in units of log 2 (over `unit`)
#pragma unroll
          for (int c = 0; c < C::kPart; c += 2) {
            const F2 d = KEYS ? *reinterpret_cast<const F2*>(&s_delta[n & 1][c0 + c]) : f2(-delta, -delta);
            const float2 v = un(fma2(f2(__uint_as_float(y[c]), __uint_as_float(y[c + 1])), f2(sigma, sigma), d));
            y[c] = __float_as_uint(v.x);
            y[c + 1] = __float_as_uint(v.y);
          }
          float left = unit;
          if constexpr (WIDE) {
            const float in = p.scale / p.cap;
#pragma unroll
            for (int c = 0; c < C::kPart; ++c) {
              const float v = __uint_as_float(x[c]) * in, sl = slant_of(v);
              x[c] = __float_as_uint(tanh_wide(v));
              if (KEYS) y[c] = __float_as_uint(__uint_as_float(y[c]) * sl);
              else slant[c] = __float_as_uint(sl);
            }
          } else if (p.cap > 0.0f) {
            const float in = p.scale / p.cap * (2.0f * kLog2e);
            const F2 in2 = f2(in, in), one = f2(1.0f, 1.0f);
#pragma unroll
            for (int c = 0; c < C::kPart; c += 2) {  // as slant_of has it, and the tanh 1 - m with x's sign
              const float2 v = un(mul2(pair(x + c), in2));
              const F2 w = f2(exp2_fast(-fabsf(v.x)), exp2_fast(-fabsf(v.y)));
              const float2 d = un(add2(w, one));
              const F2 m = mul2(add2(w, w), f2(rcp_fast(d.x), rcp_fast(d.y))), th = sub2(one, m);
              const float2 t = un(th);
              x[c] = __float_as_uint(copysignf(t.x, v.x));
              x[c + 1] = __float_as_uint(copysignf(t.y, v.y));
              const F2 sl = mul2(m, add2(th, one));
              if (KEYS) put(y + c, mul2(pair(y + c), sl));
              else put(slant + c, sl);
            }
          }
          if (slope2 != 0.0f) {
#pragma unroll
            for (int c = 0; c < C::kPart; ++c) {
              const int far = KEYS ? s_row[n & 1][c0 + c].z - r : row.z - (o0 + c0 + c);
              x[c] = __float_as_uint(fmaf(-slope2, fabsf((float)far), __uint_as_float(x[c]) * left));
            }
            left = 1.0f;
          }
          if (seen == kSome) {
#pragma unroll
            for (int c = 0; c < C::kPart; ++c) {
              int4 q = row;
              if (KEYS) q = s_row[n & 1][c0 + c];
              const int j = KEYS ? r : o0 + c0 + c;
              if (!(j >= q.x && j < q.y)) {
                x[c] = 0xff800000u;
                y[c] = 0u;
              }
            }
          }
          auto weigh = [&](auto capped) {
#pragma unroll
            for (int c = 0; c < C::kPart; c += 2) {
              const F2 l = KEYS ? *reinterpret_cast<const F2*>(&s_lse[n & 1][c0 + c]) : f2(-lse, -lse);
              const float2 v = un(fma2(f2(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), f2(left, left), l));
              F2 a = f2(exp2_fast(v.x), exp2_fast(v.y)), g = mul2(a, pair(y + c));
              if constexpr (KEYS) {
                two_values<T>(a, w[c / 2], w[C::kPart / 2 + c / 2]);
              } else {
                off = add2(off, g);
                if constexpr (decltype(capped)::value) {
                  a = mul2(a, pair(slant + c));
                  g = mul2(g, pair(slant + c));
                }
                const float2 f = un(a);
                w[c / 2] = pack2<T>(f.x, f.y);
              }
              two_values<T>(g, e[c / 2], e[C::kPart / 2 + c / 2]);
            }
          };
          if (!KEYS && p.cap > 0.0f) weigh(std::true_type());
          else weigh(std::false_type());
        } else {
#pragma unroll
          for (int c = 0; c < C::kPart; ++c) w[c] = e[c] = 0u;
          if (C::kApart && step == C::kSteps - 1) {
            tc::tc_fence_before();
            warp_arrive(&sfree);
          }
        }
        if (C::kApart && n > 0 && step == 0) {  // the products before have read their values
          ok = __all_sync(kAll, wait_on(&done, (uint32_t)(n - 1), kWaitTimeoutEpilogue, abort_flag));
          tc::tc_fence_after();
        }
        if (ok) {
          if (KEYS) tmem_put16(mine + C::kPAt + c0 / C::kPart * C::kStride, w);
          else tmem_put8(mine + C::kPAt + c0 / C::kPart * C::kStride, w);
          tmem_put16(mine + C::kEAt + c0 / C::kPart * C::kStride, e);
        }
      }
      if (ok) {
        tmem_wait_st();
        tc::tc_fence_before();
        warp_arrive(&ready);
      }
      if (KEYS && n + 1 < blocks) {  // (a give-up is everyone's: all meet here)
        deposit(n + 1);
        ok = meet(ok);
        if (n + 2 < blocks) fetch(n + 2);
      }
    }
    if (ok && blocks > 0) {
      ok = wait_on(&done, (uint32_t)(blocks - 1) & 1u, kWaitTimeoutEpilogue, abort_flag);
      tc::tc_fence_after();
    }
    if constexpr (!KEYS) {
      const float2 both = un(off);
      s_off[set][quarter * 32 + lane] = both.x + both.y;
    }
    ok = meet(ok);
    // a row that is not finite is taken again by itself; the sums' columns are shared by the sets
    const float down = up != 0 ? 0x1p-15f : 1.0f, w1 = p.scale * down / sigma;
    const int64_t at = ((int64_t)r * (KEYS ? p.Hk : p.H) + head) * p.D;
    const bool mine_too = KEYS || row.y > row.x, there = r < span.y;
    float d = 0.0f;  // what delta is off by, as p and dP are scaled
    if constexpr (!KEYS) {
      for (int i = 0; i < C::kSets; ++i) d += s_off[i][quarter * 32 + lane];
      d *= down;
      if (ok && set == 0 && there && mine_too) p.delta[(int64_t)head * p.Tq + r] = delta + d;  // (fp16: times the range)
    }
    if (ok) {
      bool bad = false;
      for (int which = 0; which < (KEYS ? 2 : 1); ++which) {
        T* out = static_cast<T*>(which ? p.dv : KEYS ? p.dk : p.dq);
        const bool wide = p.D % 16 == 0 && aligned(out, 32);
#pragma unroll 1
        for (int c = 32 * set; c < p.D; c += 32 * C::kSets) {
          uint32_t o[32];
          __syncwarp();
          if (blocks > 0) {
            tmem_get32(mine + (which ? C::kAcc2At : C::kAccAt) + c, o);
            tmem_wait_ld();
          }
          if (!KEYS && blocks > 0) {
            uint32_t k[32];
            tmem_get32(mine + C::kAcc2At + c, k);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(fmaf(-d, __uint_as_float(k[i]), __uint_as_float(o[i])));
          }
          if (blocks == 0 || !mine_too) {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0u;
          }
          if (KEYS && p.parts) {  // (whatever they are: their sum is looked at)
            float* to = p.part + ((int64_t)(which * p.G + blockIdx.z) * p.Tk * p.Hk * p.D) + at + c;
            if (there)
#pragma unroll
              for (int i = 0; i < 32; i += 4)
                if (c + i < p.D)
                  *reinterpret_cast<float4*>(to + i) = make_float4(__uint_as_float(o[i]), __uint_as_float(o[i + 1]), __uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
          } else if (there) {
            bad = bad || !finite32(o);
            store_sums<T>(out + at + c, o, p.D - c, which ? down : w1, wide);
          }
        }
      }
      if (bad) s_bad[quarter * 32 + lane] = 1;
      meet(true);  // (all have stored)
    }
    if (ok && set == 0) {
      uint32_t again = __ballot_sync(kAll, there && s_bad[quarter * 32 + lane]);
      while (again != 0) {
        const int i = __ffs(again) - 1;
        again &= again - 1;
        if (KEYS) row_dkv<T>(p, span.x + quarter * 32 + i, head);
        else row_dq<T>(p, span.x + quarter * 32 + i, head);
        __syncwarp();
      }
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmemCols) : "memory");
  }
}

// dk and dv of a key head from its query heads' parts, a warp a row
template <typename T>
__global__ void __launch_bounds__(256) keys_join_kernel(const __grid_constant__ Params p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5), rows = (int64_t)p.Tk * p.Hk;
  if (row >= rows) return;
  constexpr bool kHalfType = std::is_same<T, __half>::value;
  const float down = kHalfType ? 0x1p-15f : 1.0f, w1 = p.scale * down / (kHalfType ? range_of(p, p.key_segments[row / p.Hk], (int)(row % p.Hk)) : 1.0f);
  bool finite = true;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    T* out = static_cast<T*>(which ? p.dv : p.dk) + row * p.D;
    for (int c = lane * 4; c < p.D; c += 128) {
      float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
      for (int g = 0; g < p.G; ++g) {
        const float4 v = *reinterpret_cast<const float4*>(p.part + (int64_t)(which * p.G + g) * rows * p.D + row * p.D + c);
        s.x += v.x;
        s.y += v.y;
        s.z += v.z;
        s.w += v.w;
      }
      const float w = which ? down : w1, any = s.x * 0.0f + s.y * 0.0f + s.z * 0.0f + s.w * 0.0f;
      finite = finite && any == any;
      *reinterpret_cast<uint2*>(out + c) = make_uint2(pack2<T>(s.x * w, s.y * w), pack2<T>(s.z * w, s.w * w));
    }
  }
  if (!__all_sync(kAll, finite)) {
    __syncwarp();
    row_dkv<T>(p, (int)(row / p.Hk), (int)(row % p.Hk));
  }
}

// ------------------------------------------------------------------- host
static int make_map(CUtensorMap* tm, const void* base, int D, int heads, int64_t T, int64_t t_stride, int64_t h_stride, int rows,
                    CUtensorMapDataType dt) {
  auto enc = tc::encode_fn();
  if (enc == nullptr) return fail(RB_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)T};
  cuuint64_t strides[2] = {(cuuint64_t)(heads > 1 ? h_stride : D) * 2, (cuuint64_t)(T > 1 ? t_stride : D) * 2};
  cuuint32_t box[3] = {64, 1, (cuuint32_t)rows};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = enc(tm, dt, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(RB_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return RB_OK;
}

// whether a tensor map can be made of it: 16-byte rows and strides (of the dimensions that have a second entry)
static bool mappable(const void* base, int64_t T, int heads, int64_t t_stride, int64_t h_stride) {
  auto fits = [](int64_t s) { return s > 0 && s % 8 == 0 && s < (int64_t)1 << 39; };
  return aligned(base, 16) && (T <= 1 || fits(t_stride)) && (heads <= 1 || fits(h_stride));
}

template <typename K>
static int launch(K kernel, dim3 grid, int threads, int smem, bool after, cudaStream_t st, const char* what, void** args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = after ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelExC(&cfg, reinterpret_cast<const void*>(kernel), args), what);
}

// Tiles by the packed order or by segment: which takes less time, were all segments alike.  By segment, every segment has
// its own (partly empty) tiles; by the packed order a tile's rows see keys of several segments.  A tile costs about two
// blocks besides its own, fewer tiles than the GPU holds at once take as long as those, and the last are half alone.  Eight heads of 64, us packed |
// by segment: 2048 users of 40: 88 | 111 (gradients 419 | 784), 700 of 128: 76 | 82 (393 | 517), 512 of mean 200, uneven:
// 158 | 151 (723 | 770), 128 of mean 700, uneven: 290 | 285, 512 single queries over 16 keys each: 73 | 32, 512 times 30 over
// 256: 132 | 85.
static bool choose_by_segment(int64_t Tq, int64_t Tk, int64_t S, int heads) {
  if (S <= 0) return false;
  const double nq = (double)Tq / S, nk = (double)Tk / S, wave = 4.0 * sm_count();
  auto time = [&](double tiles, double keys) { return (std::max(tiles * heads, wave) + wave / 2) * (keys / kBlock + 0.5 + 2.0); };
  return time(S * std::max(nq / kTile + 0.5, 1.0), nk) < time((double)Tq / kTile + 0.5, nk * (1.0 + kTile / std::max(nq, 1.0)));
}

static int tiles_of(int64_t T, int64_t S, bool by_segment) { return (int)(by_segment ? T / kTile + S + 2 : (T + kTile - 1) / kTile); }

template <typename T, int DP, bool WIDE>
static int run_forward(Params& p, CUtensorMapDataType dt, cudaStream_t st) {
  using C = Forward<DP>;
  static std::once_flag once[64];
  int dev = 0, rc;
  cudaGetDevice(&dev);
  cudaError_t e = cudaSuccess;
  std::call_once(once[dev & 63], [&] {
    e = cudaFuncSetAttribute(forward_kernel<T, DP, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  });
  if (e != cudaSuccess) return check_cuda(e, "cudaFuncSetAttribute(attention forward_kernel)");
  CUtensorMap tmQ, tmK, tmV;
  if ((rc = make_map(&tmQ, p.q, p.D, p.H, p.Tq, p.q_t, p.q_h, kTile, dt))) return rc;
  if ((rc = make_map(&tmK, p.k, p.D, p.Hk, p.Tk, p.k_t, p.k_h, kBlock, dt))) return rc;
  if ((rc = make_map(&tmV, p.v, p.D, p.Hk, p.Tk, p.v_t, p.v_h, kBlock, dt))) return rc;
  const int64_t ctas = std::min<int64_t>((int64_t)p.n_tiles * p.H, (int64_t)sm_count() * C::kCtas);
  void* args[] = {&tmQ, &tmK, &tmV, &p};
  return launch(forward_kernel<T, DP, WIDE>, dim3((unsigned)ctas), C::kThreads, C::kSmem, true, st, "attention forward_kernel launch", args);
}

// How many parts the keys of a segment are split into where there are few queries, 0: not that kernel.  It reads a key
// head's keys for 16 rows, each query's heads among them; the tiles read them for 128 rows of one head, most of them empty.
// So 16 rows cost 0.7 of a tile and half a tile for each segment, while fewer tiles than five an SM take as long as those
// (64 segments of 4000 keys, tiles | this, us: 1 query of 8 heads over 8, 282 | 122; over 1, 278 | 28; 16 over 1, 281 |
// 110; 64 over 8, 277 | 309; 512 segments of 1000 keys: 1 over 8, 260 | 256, 8 over 1, 265 | 114).
// Parts fill the GPU once (of 256 keys or more); where it holds fewer than three of each, segments of different lengths
// are evened out by up to eight CTAs an SM, of 1024 keys or more (64 histories of 1000 to 16000 keys, 16 heads over 4: whole
// 283, in two 240, in five, which are eight CTAs an SM, 204, in nine 199; 64 times 4 queries over 4000 keys, 8 heads over 2:
// whole 69, in three, which fill the GPU once, 55, in eight 54).
static int splits_of(int64_t Tq, int64_t Tk, int64_t S, int H, int Hk, int D) {
  const int64_t G = H / Hk, sm = sm_count(), used = std::min(S, Tq);  // segments with queries, at most
  if (used <= 0 || D % 8 != 0 || D > 128 || Tk < 4 * Tq || Tq * G > 1 << 30) return 0;
  if (7 * Hk * (Tq * G / 16 + used) + 5 * Hk * used >= 10 * std::max<int64_t>(H * (Tq / kTile + used), 5 * sm)) return 0;
  const int64_t ctas = used * ((Tq * G / used + 15) / 16) * Hk, keys = Tk / S;
  const int64_t once = sm * (D > 64 ? Few<128>::kCtas : Few<64>::kCtas) / ctas;
  int64_t parts = once > 2 ? std::min(once, keys / 256) : std::max(std::min(once, keys / 256), std::min((8 * sm + ctas - 1) / ctas, keys / 1024));
  parts = std::min(parts, 64 * sm / (Tq * G / 16 + S + 2));  // (the grid has a place for every segment, queries or not)
  return (int)std::max<int64_t>(1, std::min<int64_t>(parts, 64));
}

template <typename T, int DP>
static int run_few(Params& p, CUtensorMapDataType dt, cudaStream_t st) {
  using C = Few<DP>;
  static std::once_flag once[64];
  int dev = 0, rc;
  cudaGetDevice(&dev);
  cudaError_t e = cudaSuccess;
  std::call_once(once[dev & 63], [&] {
    e = cudaFuncSetAttribute(few_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  });
  if (e != cudaSuccess) return check_cuda(e, "cudaFuncSetAttribute(attention few_kernel)");
  CUtensorMap tmK, tmV;
  if ((rc = make_map(&tmK, p.k, p.D, p.Hk, p.Tk, p.k_t, p.k_h, kBlock, dt))) return rc;
  if ((rc = make_map(&tmV, p.v, p.D, p.Hk, p.Tk, p.v_t, p.v_h, kBlock, dt))) return rc;
  const int64_t tiles = (int64_t)p.Tq * p.G / C::kRows + p.S + 2;
  void* args[] = {&tmK, &tmV, &p};
  if ((rc = launch(few_kernel<T, DP>, dim3((unsigned)(tiles * p.splits), p.Hk), C::kThreads, C::kSmem, true, st, "attention few_kernel launch", args)))
    return rc;
  if (p.splits == 1) return RB_OK;
  void* join[] = {&p};
  return launch(few_join_kernel<T>, dim3((unsigned)(((int64_t)p.Tq * p.H + 7) / 8)), 256, 0, true, st, "attention few_join_kernel launch", join);
}

static bool tiled(const Params& p) {
  return p.D % 8 == 0 && p.D <= 128 && mappable(p.q, p.Tq, p.H, p.q_t, p.q_h) && mappable(p.k, p.Tk, p.Hk, p.k_t, p.k_h) &&
         mappable(p.v, p.Tk, p.Hk, p.v_t, p.v_h);
}

template <typename T>
static int forward(Params& p, CUtensorMapDataType dt, cudaStream_t st) {
  int rc;
  const bool tiles = tiled(p) && p.Tk > 0 && aligned(p.out, 16);
  p.by_segment = choose_by_segment(p.Tq, p.Tk, p.S, p.H);
  p.splits = tiles ? splits_of(p.Tq, p.Tk, p.S, p.H, p.Hk, p.D) : 0;
  p.n_tiles = tiles_of(p.Tq, p.S, p.by_segment);
  if (!tiles || p.splits > 0) p.tiles = nullptr;
  plan_kernel<T><<<p.n_tiles, kTile, 0, st>>>(p);
  if ((rc = check_cuda(cudaGetLastError(), "attention plan_kernel launch"))) return rc;
  if (p.splits > 0) return p.D <= 64 ? run_few<T, 64>(p, dt, st) : run_few<T, 128>(p, dt, st);
  if (tiles && p.cap > kWideCap) return run_forward<T, 128, true>(p, dt, st);
  if (tiles) return p.D <= 64 ? run_forward<T, 64, false>(p, dt, st) : run_forward<T, 128, false>(p, dt, st);
  void* args[] = {&p};
  return launch(row_kernel<T, kRowForward>, dim3((unsigned)(((int64_t)p.Tq * p.H + 7) / 8)), 256, 0, true, st,
                "attention row_kernel launch", args);
}

// Whether the query heads that share a key head go to CTAs of their own, whose sums are added up after (each part is
// written and read once, in 32 bits): with few tiles of keys an SM the longest take too long by themselves.  Eight heads
// over two, both gradients, together | apart, us: 1 document of 6100 keys (0.6 tiles an SM) 744 | 511; 2 of them 913 | 891,
// in heads of 64 values 1306 | 906; 8 of 3000 (2.5 tiles) 921 | 966; 64 users of 150 (1.0) 120 | 183; 16 of 300 (0.5) 76 | 95.
static bool key_parts(int64_t Tk, int64_t S, int H, int Hk) {
  if (H <= Hk || H / Hk > 64 || Tk < kTile) return false;
  const int64_t tiles = Tk / kTile * Hk, sm = sm_count();
  return 2 * tiles < sm || (tiles < 2 * sm && Tk >= 1024 * S);
}

template <typename T, int DP, bool KEYS, bool WIDE>
static int run_backward(Params& p, CUtensorMapDataType dt, cudaStream_t st) {
  using C = Backward<DP, KEYS>;
  static std::once_flag once[64];
  int dev = 0, rc;
  cudaGetDevice(&dev);
  cudaError_t e = cudaSuccess;
  std::call_once(once[dev & 63], [&] {
    e = cudaFuncSetAttribute(backward_kernel<T, DP, KEYS, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  });
  if (e != cudaSuccess) return check_cuda(e, "cudaFuncSetAttribute(attention backward_kernel)");
  const int q_rows = KEYS ? kBlock : kTile, k_rows = KEYS ? kTile : kBlock;
  CUtensorMap q, g, k, v;
  if ((rc = make_map(&q, p.q, p.D, p.H, p.Tq, p.q_t, p.q_h, q_rows, dt))) return rc;
  if ((rc = make_map(&g, p.g, p.D, p.H, p.Tq, p.g_t, p.g_h, q_rows, dt))) return rc;
  if ((rc = make_map(&k, p.k, p.D, p.Hk, p.Tk, p.k_t, p.k_h, k_rows, dt))) return rc;
  if ((rc = make_map(&v, p.v, p.D, p.Hk, p.Tk, p.v_t, p.v_h, k_rows, dt))) return rc;
  const int tiles = KEYS ? p.n_key_tiles : p.n_tiles;
  void* args[] = {KEYS ? &k : &q, KEYS ? &v : &g, KEYS ? &q : &k, KEYS ? &g : &v, &p};
  if ((rc = launch(backward_kernel<T, DP, KEYS, WIDE>, dim3((unsigned)tiles, KEYS ? p.Hk : p.H, KEYS && p.parts ? p.G : 1), C::kThreads, C::kSmem,
                   true, st, "attention backward_kernel launch", args)))
    return rc;
  if (!KEYS || !p.parts) return RB_OK;
  void* join[] = {&p};
  return launch(keys_join_kernel<T>, dim3((unsigned)(((int64_t)p.Tk * p.Hk + 7) / 8)), 256, 0, true, st, "attention keys_join_kernel launch", join);
}

template <typename T>
static int backward(Params& p, CUtensorMapDataType dt, cudaStream_t st) {
  int rc;
  const bool peaks = std::is_same<T, __half>::value;
  if (peaks && p.S > 0 && (rc = check_cuda(cudaMemsetAsync(p.peaks, 0, (size_t)p.S * p.Hk * 8, st), "attention peaks"))) return rc;
  const bool tiles = tiled(p) && p.Tq > 0 && p.Tk > 0 && mappable(p.g, p.Tq, p.H, p.g_t, p.g_h) && aligned(p.dq, 16) &&
                     aligned(p.dk, 16) && aligned(p.dv, 16);
  if (tiles) {
    p.by_segment = choose_by_segment(p.Tq, p.Tk, p.S, p.H);
    p.keys_by_segment = choose_by_segment(p.Tk, p.Tq, p.S, p.Hk);
    p.n_tiles = tiles_of(p.Tq, p.S, p.by_segment);
    p.n_key_tiles = tiles_of(p.Tk, p.S, p.keys_by_segment);
    p.key_tiles = p.tiles + p.n_tiles;
  }
  const int64_t heads = (int64_t)p.Tq * p.H + (peaks ? (int64_t)p.Tk * p.Hk : 0);
  if (heads > 0) {
    const bool vec = p.D % 8 == 0 && aligned(p.o, 16) && mappable(p.g, p.Tq, p.H, p.g_t, p.g_h) && mappable(p.v, p.Tk, p.Hk, p.v_t, p.v_h);
    const int lanes = !vec || p.D > 128 ? 32 : p.D > 64 ? 16 : 8;
    const unsigned grid = (unsigned)((p.Tq + 255) / 256 + (peaks ? (p.Tk + 255) / 256 : 0) + (p.n_tiles + p.n_key_tiles + 7) / 8 + std::min<int64_t>((heads * lanes + 255) / 256, (int64_t)sm_count() * kDeltaCtas));
    if (!vec) delta_kernel<T, 32, false><<<grid, 256, 0, st>>>(p);
    else if (lanes == 32) delta_kernel<T, 32, true><<<grid, 256, 0, st>>>(p);
    else if (lanes == 16) delta_kernel<T, 16, true><<<grid, 256, 0, st>>>(p);
    else delta_kernel<T, 8, true><<<grid, 256, 0, st>>>(p);
    if ((rc = check_cuda(cudaGetLastError(), "attention delta_kernel launch"))) return rc;
  }
  if (tiles) {
    // the queries first: they give the keys their delta
    p.parts = key_parts(p.Tk, p.S, p.H, p.Hk);
    if (p.cap > kWideCap) {
      if ((rc = run_backward<T, 128, false, true>(p, dt, st))) return rc;
      return run_backward<T, 128, true, true>(p, dt, st);
    }
    if ((rc = p.D <= 64 ? run_backward<T, 64, false, false>(p, dt, st) : run_backward<T, 128, false, false>(p, dt, st))) return rc;
    return p.D <= 64 ? run_backward<T, 64, true, false>(p, dt, st) : run_backward<T, 128, true, false>(p, dt, st);
  }
  void* args[] = {&p};
  if (p.Tq > 0 && (rc = launch(row_kernel<T, kRowDq>, dim3((unsigned)(((int64_t)p.Tq * p.H + 7) / 8)), 256, 0, false, st,
                               "attention row_kernel launch", args)))
    return rc;
  if (p.Tk == 0) return RB_OK;
  return launch(row_kernel<T, kRowDkv>, dim3((unsigned)(((int64_t)p.Tk * p.Hk + 7) / 8)), 256, 0, false, st,
                "attention row_kernel launch", args);
}

static int check(const Params& p, int dtype, int64_t Tq, int64_t Tk, int64_t S, int idx_dtype) {
  if (Tq < 0 || Tk < 0 || S < 0 || p.H <= 0 || p.Hk <= 0 || p.D <= 0) return fail(RB_ERR_VALUE, "negative or empty attention shape");
  if (dtype != RB_BF16 && dtype != RB_F16) return fail(RB_ERR_UNSUPPORTED, "attention takes bf16 or f16");
  if (idx_dtype != RB_I64 && idx_dtype != RB_I32) return fail(RB_ERR_VALUE, "offsets must be int64 or int32");
  if (p.H % p.Hk != 0) return fail(RB_ERR_VALUE, "%d query heads cannot share %d key heads", p.H, p.Hk);
  if (p.D > kMaxWidth) return fail(RB_ERR_UNSUPPORTED, "heads wider than %d", kMaxWidth);
  if (Tq > 1 << 30 || Tk > 1 << 30 || S > 1 << 30 || p.H > 65535) return fail(RB_ERR_UNSUPPORTED, "more than 2^30 tokens or segments, or 65535 heads");
  if ((Tq / kTile + Tk / kTile + S + 2) * p.H > 0x7fffffffLL) return fail(RB_ERR_UNSUPPORTED, "more than 2^31 tiles of all heads");
  if (!(p.scale > 0.0f) || !(p.scale < INFINITY)) return fail(RB_ERR_VALUE, "scale must be positive");
  if (!(p.cap >= 0.0f) || !(p.cap < INFINITY)) return fail(RB_ERR_VALUE, "cap must be positive, or 0 for none");
  return RB_OK;
}

}  // namespace attn
}  // namespace rb

using namespace rb;

extern "C" int64_t rb_segment_attention_workspace_size(int64_t Tq, int64_t Tk, int64_t S, int H, int Hk, int D) {
  if (Tq < 0 || Tk < 0 || S < 0 || H <= 0 || Hk <= 0 || D <= 0 || Tq > 1 << 30) return -1;
  const int64_t splits = H % Hk == 0 ? attn::splits_of(Tq, Tk, S, H, Hk, D) : 0;
  const int64_t tiles = Tq / attn::kTile + S + 2, lists = 16 + Tq * 16 + tiles * 16;
  if (splits > 0) return lists + (splits > 1 ? Tq * H * splits * (D + 2) * 4 : 0);
  return lists + (D % 8 == 0 && D <= 128 ? tiles * H * 32 : 0);
}

extern "C" int rb_segment_attention(const void* q, int64_t q_t, int64_t q_h, const void* k, int64_t k_t, int64_t k_h,
                                    const void* v, int64_t v_t, int64_t v_h, int dtype, int64_t Tq, int64_t Tk, int H, int Hk,
                                    int D, const void* q_offsets, const void* k_offsets, const void* prefix, int idx_dtype,
                                    int64_t S, int causal, const float* slopes, float cap, float scale, void* workspace,
                                    int64_t workspace_bytes, void* out, float* lse, void* stream) {
  using namespace rb::attn;
  Params p{};
  p.H = H;
  p.Hk = Hk;
  p.D = D;
  p.scale = scale;
  p.cap = cap;
  int rc;
  if ((rc = check(p, dtype, Tq, Tk, S, idx_dtype))) return rc;
  if (Tq > 0 && (q == nullptr || out == nullptr || (S > 0 && (q_offsets == nullptr || k_offsets == nullptr))))
    return fail(RB_ERR_VALUE, "null operand");
  if (Tk > 0 && (k == nullptr || v == nullptr)) return fail(RB_ERR_VALUE, "null operand");
  const int64_t need = rb_segment_attention_workspace_size(Tq, Tk, S, H, Hk, D);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(RB_ERR_VALUE, "workspace of %lld bytes (16-byte aligned) needed, %lld given", (long long)need,
                (long long)workspace_bytes);
  if (!device_is_sm100()) return fail(RB_ERR_DEVICE, "rb_segment_attention needs an sm_100 (B200) device");
  if (Tq == 0) return RB_OK;
  p.q = q;
  p.k = k;
  p.v = v;
  p.out = out;
  p.lse = lse;
  p.next = static_cast<uint32_t*>(workspace);
  p.rows = static_cast<int4*>(workspace) + 1;
  p.tiles = p.rows + Tq;
  p.part = reinterpret_cast<float*>(p.tiles + (Tq / kTile + S + 2));
  p.redo = reinterpret_cast<int2*>(p.part);  // (no kernel uses both)
  p.q_off = q_offsets;
  p.k_off = k_offsets;
  p.prefix = prefix;
  p.slopes = slopes;
  p.q_t = q_t;
  p.q_h = q_h;
  p.k_t = k_t;
  p.k_h = k_h;
  p.v_t = v_t;
  p.v_h = v_h;
  p.Tq = (int)Tq;
  p.Tk = (int)Tk;
  p.S = (int)S;
  p.G = H / Hk;
  p.off64 = idx_dtype == RB_I64;
  p.causal = causal != 0;
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == RB_BF16 ? forward<__nv_bfloat16>(p, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, st)
                          : forward<__half>(p, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, st);
}

extern "C" int64_t rb_segment_attention_backward_workspace_size(int64_t Tq, int64_t Tk, int64_t S, int H, int Hk, int D) {
  if (Tq < 0 || Tk < 0 || S < 0 || H <= 0 || Hk <= 0 || D <= 0 || Tq > 1 << 30) return -1;
  const int64_t parts = H % Hk == 0 && D % 8 == 0 && D <= 128 && attn::key_parts(Tk, S, H, Hk) ? (int64_t)2 * H * Tk * D * 4 : 0;
  const int64_t lists = (Tq + Tq / attn::kTile + Tk / attn::kTile + 2 * S + 4) * 16;
  return (S * Hk * 8 + 15) / 16 * 16 + lists + ((int64_t)H * Tq * 4 + 15) / 16 * 16 + (Tk * 4 + 15) / 16 * 16 + parts;
}

extern "C" int rb_segment_attention_backward(const void* grad, int64_t g_t, int64_t g_h, const void* q, int64_t q_t, int64_t q_h,
                                             const void* k, int64_t k_t, int64_t k_h, const void* v, int64_t v_t, int64_t v_h,
                                             const void* out, const float* lse, int dtype, int64_t Tq, int64_t Tk, int H, int Hk,
                                             int D, const void* q_offsets, const void* k_offsets, const void* prefix,
                                             int idx_dtype, int64_t S, int causal, const float* slopes, float cap, float scale,
                                             void* workspace, int64_t workspace_bytes, void* dq, void* dk, void* dv, void* stream) {
  using namespace rb::attn;
  Params p{};
  p.H = H;
  p.Hk = Hk;
  p.D = D;
  p.scale = scale;
  p.cap = cap;
  int rc;
  if ((rc = check(p, dtype, Tq, Tk, S, idx_dtype))) return rc;
  if (S > 0 && (q_offsets == nullptr || k_offsets == nullptr)) return fail(RB_ERR_VALUE, "null offsets");
  if (Tq > 0 && (grad == nullptr || q == nullptr || out == nullptr || lse == nullptr || dq == nullptr)) return fail(RB_ERR_VALUE, "null operand");
  if (Tk > 0 && (k == nullptr || v == nullptr || dk == nullptr || dv == nullptr)) return fail(RB_ERR_VALUE, "null operand");
  const int64_t need = rb_segment_attention_backward_workspace_size(Tq, Tk, S, H, Hk, D);
  if (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16))
    return fail(RB_ERR_VALUE, "workspace of %lld bytes (16-byte aligned) needed, %lld given", (long long)need,
                (long long)workspace_bytes);
  if (!device_is_sm100()) return fail(RB_ERR_DEVICE, "rb_segment_attention_backward needs an sm_100 (B200) device");
  p.g = grad;
  p.q = q;
  p.k = k;
  p.v = v;
  p.o = out;
  p.lse = const_cast<float*>(lse);
  p.dq = dq;
  p.dk = dk;
  p.dv = dv;
  p.peaks = static_cast<uint32_t*>(workspace);
  p.rows = reinterpret_cast<int4*>(static_cast<uint8_t*>(workspace) + (S * Hk * 8 + 15) / 16 * 16);
  p.tiles = p.rows + Tq;
  p.delta = reinterpret_cast<float*>(p.tiles + (Tq / kTile + Tk / kTile + 2 * S + 4));
  p.key_segments = reinterpret_cast<int32_t*>(p.delta + ((int64_t)H * Tq + 3) / 4 * 4);
  p.part = reinterpret_cast<float*>(p.key_segments + (Tk + 3) / 4 * 4);
  p.q_off = q_offsets;
  p.k_off = k_offsets;
  p.prefix = prefix;
  p.slopes = slopes;
  p.g_t = g_t;
  p.g_h = g_h;
  p.q_t = q_t;
  p.q_h = q_h;
  p.k_t = k_t;
  p.k_h = k_h;
  p.v_t = v_t;
  p.v_h = v_h;
  p.Tq = (int)Tq;
  p.Tk = (int)Tk;
  p.S = (int)S;
  p.G = H / Hk;
  p.off64 = idx_dtype == RB_I64;
  p.causal = causal != 0;
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == RB_BF16 ? backward<__nv_bfloat16>(p, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, st)
                          : backward<__half>(p, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, st);
}

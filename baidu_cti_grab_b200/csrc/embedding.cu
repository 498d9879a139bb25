// embedding.cu -- rows of an embedding table by id, scaled, and the table's gradient.
//
//   out[i] = scale table[id_i]                                      (ids clamped to the table)
//   dtable[r] = scale sum over i with id_i = r of grad[row(i)]      row(i) = i, or the bag that id i lies in
//
// The lookup is a copy and bound by HBM.  The gradient reads each id's row of grad once and writes each table row
// once; what stands between is finding the ids that share a row.  Ids are sorted (a stable radix sort of the bits
// that the table needs, the row of grad as its payload), so the sums are taken in the order of the ids: no atomics on
// values, the same bits every time.  Then
//   sums_kernel     a team of threads takes a run of sorted ids, sums in fp32 and writes every row whose ids lie in its
//                   run; what goes on in the next run, or came from the one before, goes to a partial sum
//   combine_kernel  adds the partial sums of a row that crosses runs, in their order
// The partial sums of one row are added up by one CTA: a row that many ids ask for waits for it (150,000 ids of 512 bf16
// values: 84 us over 50,000 rows, 440 over two, 650 over one).
//
// 103,725 ids of 50,000 rows of 512 bf16 values: lookup 30 us, gradient 80 (the sort about a third).  1.45 million ids in bags
// over 2.8 million rows of 512, the touched rows: 483 us, 366 of them sums that wait for rows of grad in the ids' order
// (each row of grad and of the result once: 252 us at the copy rate).
#include "common.cuh"

#include <algorithm>
#include <mutex>
#include <type_traits>

namespace rb {
namespace embed {

constexpr unsigned kAll = 0xffffffffu;

struct Params {
  const void *table, *grad, *ids, *bags;
  void *out;                     // looked-up rows | the table's gradient | the touched rows
  int64_t* out_ids;              // sparse: the touched rows' numbers
  int32_t* count;                // sparse: how many
  int64_t ld_table, ld_grad, ld_out, V, n, n_bags, padding;
  float scale;
  int D, wide_ids, out_dtype, accumulate, sparse;
  // workspace: written by one kernel of a call and read by the next, which starts under its tail, so by plain loads behind
  // griddepcontrol.wait and never by __ldg, which asks for memory that nobody writes while the kernel lives
  int32_t *key[2], *row[2];      // ids and their rows of grad, before and after a pass
  int32_t* counts;               // of a pass: [tiles][256], or [256][tiles] scanned
  int32_t* totals;               // [256]
  int32_t* heads;                // sparse: rows that start in a run, then before it
  float* part;                   // [runs][2][D]: of the row that comes from before, of the row that goes on
  int tiles, shift, bits, scanned, run, runs, run_log, team;
  int64_t zero_bytes;            // of `out`, written by CTAs behind the tiles'
};

template <typename T>
__device__ __forceinline__ float to_f32(T v) { return (float)v; }

template <typename T, int VEC>
struct Raw {  // VEC values as they lie in memory
  static constexpr int kWords = VEC * (int)sizeof(T) / 4;
  using Word = typename std::conditional<kWords <= 1, uint32_t, typename std::conditional<kWords == 2, uint2, uint4>::type>::type;
  typename std::conditional<VEC == 1, T, Word>::type v;
  __device__ void load(const T* from) { v = __ldg(reinterpret_cast<const decltype(v)*>(from)); }
  __device__ void widen(float* f) const {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = 0.0f;
    add_to(f);
  }
  __device__ void add_to(float* acc) const {
    if constexpr (VEC == 1) {
      acc[0] += to_f32(v);
    } else {
      uint32_t u[kWords];
      if constexpr (kWords == 1) u[0] = v;
      else u[0] = v.x, u[1] = v.y;
      if constexpr (kWords == 4) u[2] = v.z, u[3] = v.w;
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        if constexpr (std::is_same<T, float>::value) {
          acc[i] += __uint_as_float(u[i]);
        } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          acc[2 * i] += bf16_lo(u[i]);
          acc[2 * i + 1] += bf16_hi(u[i]);
        } else {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
          acc[2 * i] += f.x;
          acc[2 * i + 1] += f.y;
        }
      }
    }
  }
};

// VEC values to memory as T2, whole words where there are several (from an aligned address)
template <typename T2, int VEC>
__device__ __forceinline__ void store_as(T2* p, const float* v) {
  if constexpr (VEC == 1) {
    p[0] = T2(v[0]);
  } else if constexpr (std::is_same<T2, float>::value && VEC == 2) {
    *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
  } else if constexpr (std::is_same<T2, float>::value) {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  } else {
    uint32_t u[VEC / 2];
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      if constexpr (std::is_same<T2, __nv_bfloat16>::value) u[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
      else u[i] = pack_f16x2(v[2 * i], v[2 * i + 1]);
    }
    if constexpr (VEC == 2) *reinterpret_cast<uint32_t*>(p) = u[0];
    else if constexpr (VEC == 4) *reinterpret_cast<uint2*>(p) = make_uint2(u[0], u[1]);
    else *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
  }
}
template <int VEC>
__device__ __forceinline__ void load_any(const void* p, int dtype, int64_t i, float* v) {
#pragma unroll
  for (int c = 0; c < VEC; ++c) v[c] = load_as_f32(p, dtype, i + c);
}
// sums of VEC columns to row `r` of the gradient, times the scale, added to what is there when asked to
template <int VEC>
__device__ __forceinline__ void store_sums(const Params& p, int64_t r, int c, float* v) {
  const int64_t at = r * p.ld_out + c;
#pragma unroll
  for (int i = 0; i < VEC; ++i) v[i] *= p.scale;
  if (p.accumulate) {
    float old[VEC];
    load_any<VEC>(p.out, p.out_dtype, at, old);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] += old[i];
  }
  switch (p.out_dtype) {
    case RB_BF16: store_as<__nv_bfloat16, VEC>(static_cast<__nv_bfloat16*>(p.out) + at, v); break;
    case RB_F16: store_as<__half, VEC>(static_cast<__half*>(p.out) + at, v); break;
    default: store_as<float, VEC>(static_cast<float*>(p.out) + at, v);
  }
}

__device__ __forceinline__ int64_t id_at(const void* ids, int wide, int64_t i) {
  return wide ? __ldg(static_cast<const int64_t*>(ids) + i) : (int64_t)__ldg(static_cast<const int32_t*>(ids) + i);
}

// ----------------------------------------------------------------- lookup
constexpr int kLookupRows = 4, kLookupWide = 2;  // rows, and loads of a row, that a thread has in flight

// teams of p.team lanes, a row each
template <typename T, int VEC>
__global__ void __launch_bounds__(256) lookup_kernel(const __grid_constant__ Params p) {
  const int lane = threadIdx.x % p.team, teams = 256 / p.team;
  const T* table = static_cast<const T*>(p.table);
  T* out = static_cast<T*>(p.out);
  const int64_t step = (int64_t)gridDim.x * teams * kLookupRows;
  for (int64_t r0 = ((int64_t)blockIdx.x * teams + threadIdx.x / p.team) * kLookupRows; r0 < p.n; r0 += step) {
    const T* from[kLookupRows];
#pragma unroll
    for (int k = 0; k < kLookupRows; ++k)
      from[k] = table + (r0 + k < p.n ? min(max(id_at(p.ids, p.wide_ids, r0 + k), (int64_t)0), p.V - 1) : 0) * p.ld_table;
    for (int c0 = lane * VEC; c0 < p.D; c0 += p.team * VEC * kLookupWide) {
      Raw<T, VEC> v[kLookupRows][kLookupWide];
#pragma unroll
      for (int k = 0; k < kLookupRows; ++k)
#pragma unroll
        for (int u = 0; u < kLookupWide; ++u)
          if (r0 + k < p.n && c0 + u * p.team * VEC < p.D) v[k][u].load(from[k] + c0 + u * p.team * VEC);
#pragma unroll
      for (int k = 0; k < kLookupRows; ++k)
#pragma unroll
        for (int u = 0; u < kLookupWide; ++u) {
          if (r0 + k >= p.n || c0 + u * p.team * VEC >= p.D) continue;
          float f[VEC];
          v[k][u].widen(f);
#pragma unroll
          for (int i = 0; i < VEC; ++i) f[i] *= p.scale;
          store_as<T, VEC>(out + (r0 + k) * p.ld_out + c0 + u * p.team * VEC, f);
        }
    }
  }
}

// ------------------------------------------------------------------- sort
// A stable radix sort, 8 bits a pass.  A CTA ranks a tile of kTile keys: each warp counts its own 128 in their order
// (lanes with equal digits find each other by eight ballots), then warps and tiles are added up before it.
constexpr int kSortThreads = 512, kPerThread = 4, kTile = kSortThreads * kPerThread, kSortWarps = kSortThreads / 32;
constexpr int kDigits = 256;
// Up to so many tiles a CTA adds up the counts of those before it by itself, above that a kernel does it for all: 20,000
// ids (10 tiles) 30 us and 35, 60,000 36 and 36, 100,000 40 and 38, 400,000 69 and 63.
constexpr int kDirect = 32;

// the last b in [0, n_bags] with bags[b] <= i, 0 where there is none: a warp, 32 probes at once
__device__ __forceinline__ int64_t bag_of(const Params& p, int64_t i) {
  int64_t lo = 0, hi = p.n_bags + 1;
  const int lane = threadIdx.x & 31;
  while (hi - lo > 1) {
    const int64_t step = (hi - lo + 31) / 32, b = lo + (lane + 1) * step;
    const int n = __popc(__ballot_sync(kAll, b < hi && id_at(p.bags, p.wide_ids, b) <= i));
    lo += n * step;
    hi = min(hi, lo + step);
  }
  return lo;
}
// key of id i: the table row, or V for an id that gets nothing
__device__ __forceinline__ int key_of(const Params& p, int64_t i) {
  const int key = (int)min(max(id_at(p.ids, p.wide_ids, i), (int64_t)0), p.V - 1);
  return p.padding >= 0 && key == p.padding ? (int)p.V : key;
}

__device__ __forceinline__ uint32_t peers_of(int digit, bool there) {
  uint32_t same = __ballot_sync(kAll, there);
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    const uint32_t set = __ballot_sync(kAll, (digit >> b) & 1);
    same &= (digit >> b) & 1 ? set : ~set;
  }
  return same;
}

// keys of the tile, warp by warp: thread's item k of its warp's rounds
__device__ __forceinline__ int64_t item_at(int tile, int k) {
  return (int64_t)tile * kTile + (threadIdx.x >> 5) * (32 * kPerThread) + k * 32 + (threadIdx.x & 31);
}

// zeros over the gradient, by CTAs beside those that sort (few of which there are)
__device__ __forceinline__ void zero_fill(const Params& p, int64_t block, int64_t blocks) {
  uint4* to = static_cast<uint4*>(p.out);
  const int64_t n = p.zero_bytes / 16;
  for (int64_t i = block * blockDim.x + threadIdx.x; i < n; i += blocks * blockDim.x) to[i] = make_uint4(0u, 0u, 0u, 0u);
  uint8_t* rest = static_cast<uint8_t*>(p.out);
  if (block == 0 && threadIdx.x < p.zero_bytes % 16) rest[n * 16 + threadIdx.x] = 0;
}

// The rows of grad of the ids [i0, i0 + count) that lie in bags: every bag that starts among them marks its first id (the
// last of several, the others being empty), and a running maximum carries it on.  -1: in no bag.
__device__ __forceinline__ void mark_bags(const Params& p, int64_t i0, int count, int* s_mark, int* s_warp) {
  __shared__ int64_t s_edge[2];
  if (threadIdx.x < 64) {
    const int which = threadIdx.x >> 5;
    const int64_t b = bag_of(p, which ? i0 + count - 1 : i0);
    if ((threadIdx.x & 31) == 0) s_edge[which] = b;
  }
  for (int k = threadIdx.x; k < count; k += blockDim.x) s_mark[k] = -1;
  __syncthreads();
  for (int64_t b = s_edge[0] + threadIdx.x; b <= s_edge[1]; b += blockDim.x) {
    const int64_t at = id_at(p.bags, p.wide_ids, b) - i0;
    if (at < count) atomicMax(&s_mark[max(at, (int64_t)0)], (int)b);
  }
  __syncthreads();
  // a thread's own run of marks, then the runs before it
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per = (count + (int)blockDim.x - 1) / (int)blockDim.x;
  const int k0 = min((int)threadIdx.x * per, count), k1 = min(k0 + per, count);
  int high = -1;
  for (int k = k0; k < k1; ++k) high = max(high, s_mark[k]);
  int x = high;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(kAll, x, o);
    if (lane >= o) x = max(x, y);
  }
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  int before = __shfl_up_sync(kAll, x, 1);
  if (lane == 0) before = -1;
  for (int w = 0; w < warp; ++w) before = max(before, s_warp[w]);
  for (int k = k0; k < k1; ++k) {
    before = max(before, s_mark[k]);
    s_mark[k] = before < p.n_bags ? before : -1;
  }
  __syncthreads();
}

// Counts of a pass's digits in each tile.  FIRST: keys come from the ids and are written in their order with their rows;
// CTAs behind the tiles' fill the gradient with zeros, which few tiles leave most of the GPU free for.
template <bool FIRST>
__global__ void __launch_bounds__(kSortThreads) count_kernel(const __grid_constant__ Params p) {
  __shared__ int s_count[kDigits], s_mark[FIRST ? kTile : 1], s_warp[kSortWarps];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (FIRST && (int)blockIdx.x >= p.tiles) {
    zero_fill(p, blockIdx.x - p.tiles, gridDim.x - p.tiles);
    return;
  }
  const int tile = blockIdx.x;
  const int64_t i0 = (int64_t)tile * kTile;
  const int count = (int)min((int64_t)kTile, p.n - i0);
  if (threadIdx.x < kDigits) s_count[threadIdx.x] = 0;
  if (FIRST && p.bags != nullptr) mark_bags(p, i0, count, s_mark, s_warp);
  else __syncthreads();
  int key[kPerThread];
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    const int64_t i = item_at(tile, k);
    key[k] = i >= p.n ? -1 : FIRST ? key_of(p, i) : p.key[0][i];
  }
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    if (key[k] < 0) continue;
    if (FIRST) {
      const int64_t i = item_at(tile, k);
      int row = (int)i;
      if (p.bags != nullptr) {
        row = s_mark[i - i0];
        if (row < 0) {
          row = 0;
          key[k] = (int)p.V;
        }
      }
      p.key[0][i] = key[k];
      p.row[0][i] = row;
    }
    atomicAdd(&s_count[(key[k] >> p.shift) & (kDigits - 1)], 1);
  }
  __syncthreads();
  if (threadIdx.x >= kDigits) return;
  if (p.scanned) p.counts[(int64_t)threadIdx.x * p.tiles + tile] = s_count[threadIdx.x];
  else p.counts[tile * kDigits + threadIdx.x] = s_count[threadIdx.x];
}

// sums before each of a CTA's values, and their total
__device__ __forceinline__ int block_before(int v, int* s_warp, int& total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(kAll, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  int w = lane < (int)blockDim.x / 32 ? s_warp[lane] : 0;
  const int all = __reduce_add_sync(kAll, w);
  const int before = __reduce_add_sync(kAll, lane < warp ? w : 0);
  total = all;
  return before + x - v;
}

// one CTA a digit: its counts become the sums before them
__global__ void __launch_bounds__(256) scan_kernel(const __grid_constant__ Params p) {
  __shared__ int s_warp[8];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int32_t* mine = p.counts + (int64_t)blockIdx.x * p.tiles;
  int carry = 0;
  for (int t0 = 0; t0 < p.tiles; t0 += 256) {
    const int t = t0 + threadIdx.x, v = t < p.tiles ? mine[t] : 0;
    int total;
    const int before = block_before(v, s_warp, total);
    if (t < p.tiles) mine[t] = carry + before;
    carry += total;
  }
  if (threadIdx.x == 0) p.totals[blockIdx.x] = carry;
}

__global__ void __launch_bounds__(kSortThreads, 3) scatter_kernel(const __grid_constant__ Params p) {
  __shared__ int s_hist[kSortWarps][kDigits];  // 16 KB
  __shared__ int s_warp[kSortWarps], s_mine[kSortThreads / kDigits][kDigits], s_all[kSortThreads / kDigits][kDigits];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  for (int i = threadIdx.x; i < kSortWarps * kDigits; i += kSortThreads) s_hist[0][i] = 0;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tile = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int digit_of = threadIdx.x % kDigits, part = threadIdx.x / kDigits;
  int key[kPerThread], row[kPerThread], rank[kPerThread];
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    const int64_t i = item_at(tile, k);
    key[k] = i < p.n ? p.key[0][i] : -1;
    row[k] = i < p.n ? p.row[0][i] : 0;
  }
  // where each digit's keys of this tile go: two threads a digit add up the tiles
  int mine = 0, all = 0, total;
  if (p.scanned) {
    if (part == 0) {
      mine = p.counts[(int64_t)digit_of * p.tiles + tile];
      all = p.totals[digit_of];
    }
  } else {
#pragma unroll 16
    for (int t = part; t < p.tiles; t += kSortThreads / kDigits) {
      const int c = p.counts[t * kDigits + digit_of];
      if (t < tile) mine += c;
      all += c;
    }
  }
  s_mine[part][digit_of] = mine;
  s_all[part][digit_of] = all;
  __syncthreads();
  mine = all = 0;
  if (threadIdx.x < kDigits) {
#pragma unroll
    for (int q = 0; q < kSortThreads / kDigits; ++q) {
      mine += s_mine[q][threadIdx.x];
      all += s_all[q][threadIdx.x];
    }
  }
  mine += block_before(all, s_warp, total);
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    const bool there = key[k] >= 0;
    const int digit = (key[k] >> p.shift) & (kDigits - 1);
    const uint32_t same = peers_of(digit, there);
    const int before = there ? s_hist[warp][digit] : 0;
    rank[k] = before + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (there && (same >> lane) == 1u) s_hist[warp][digit] = before + __popc(same);
    __syncwarp();
  }
  __syncthreads();
  // the warps before: two threads a digit, eight warps each
  constexpr int kEach = kSortWarps / (kSortThreads / kDigits);
  int sum = 0;
#pragma unroll
  for (int w = 0; w < kEach; ++w) sum += s_hist[part * kEach + w][digit_of];
  s_all[part][digit_of] = sum;
  if (part == 0) s_mine[0][digit_of] = mine;
  __syncthreads();
  int base = s_mine[0][digit_of];
  for (int q = 0; q < part; ++q) base += s_all[q][digit_of];
#pragma unroll
  for (int w = 0; w < kEach; ++w) {
    const int c = s_hist[part * kEach + w][digit_of];
    s_hist[part * kEach + w][digit_of] = base;
    base += c;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    if (key[k] < 0) continue;
    const int to = s_hist[warp][(key[k] >> p.shift) & (kDigits - 1)] + rank[k];
    p.key[1][to] = key[k];
    p.row[1][to] = row[k];
  }
}

// All passes of up to kSmall ids in one CTA, in shared memory: a gradient takes 22 us, with a kernel a pass 30.
constexpr int kSmallThreads = 1024, kSmallPer = 4, kSmall = kSmallThreads * kSmallPer;
struct Small {
  int key[2][kSmall], row[2][kSmall];
  int hist[kSmallThreads / 32][kDigits];
  int warp[32];
};
__global__ void __launch_bounds__(kSmallThreads) small_sort_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(16) uint8_t raw[];
  Small& s = *reinterpret_cast<Small*>(raw);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (blockIdx.x > 0) {
    zero_fill(p, blockIdx.x - 1, gridDim.x - 1);
    return;
  }
  const int n = (int)p.n, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (p.bags != nullptr) mark_bags(p, 0, n, s.row[0], s.warp);
  for (int i = threadIdx.x; i < n; i += kSmallThreads) {
    int key = key_of(p, i), row = i;
    if (p.bags != nullptr) {
      row = s.row[0][i];
      if (row < 0) {
        row = 0;
        key = (int)p.V;
      }
    }
    s.key[0][i] = key;
    s.row[0][i] = row;
  }
  int from = 0;
  for (int shift = 0; shift < p.bits; shift += 8, from ^= 1) {
    for (int d = lane; d < kDigits; d += 32) s.hist[warp][d] = 0;
    __syncthreads();
    int rank[kSmallPer];
#pragma unroll
    for (int k = 0; k < kSmallPer; ++k) {
      const int i = warp * 32 * kSmallPer + k * 32 + lane;
      const bool there = i < n;
      const int digit = there ? (s.key[from][i] >> shift) & (kDigits - 1) : 0;
      const uint32_t same = peers_of(digit, there);
      const int before = there ? s.hist[warp][digit] : 0;
      rank[k] = before + __popc(same & ((1u << lane) - 1u));
      __syncwarp();
      if (there && (same >> lane) == 1u) s.hist[warp][digit] = before + __popc(same);
      __syncwarp();
    }
    __syncthreads();
    int all = 0, total;
    if (threadIdx.x < kDigits)
      for (int w = 0; w < kSmallThreads / 32; ++w) all += s.hist[w][threadIdx.x];
    int mine = block_before(all, s.warp, total);
    if (threadIdx.x < kDigits)
      for (int w = 0; w < kSmallThreads / 32; ++w) {
        const int c = s.hist[w][threadIdx.x];
        s.hist[w][threadIdx.x] = mine;
        mine += c;
      }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSmallPer; ++k) {
      const int i = warp * 32 * kSmallPer + k * 32 + lane;
      if (i >= n) continue;
      const int key = s.key[from][i], to = s.hist[warp][(key >> shift) & (kDigits - 1)] + rank[k];
      s.key[from ^ 1][to] = key;
      s.row[from ^ 1][to] = s.row[from][i];
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < n; i += kSmallThreads) {
    p.key[0][i] = s.key[from][i];
    p.row[0][i] = s.row[from][i];
  }
}

// -------------------------------------------------------------------- sums
// (sparse) how many rows start in each run of sorted ids, a warp a run
__global__ void __launch_bounds__(256) heads_kernel(const __grid_constant__ Params p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int run = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (run >= p.runs) return;
  int n = 0;
  for (int k = lane; k < p.run; k += 32) {
    const int64_t i = (int64_t)run * p.run + k;
    if (i < p.n) {
      const int key = p.key[0][i];
      n += key < p.V && (i == 0 || p.key[0][i - 1] != key);
    }
  }
  n = __reduce_add_sync(kAll, n);
  if (lane == 0) p.heads[run] = n;
}
// ... and how many before it, by one CTA
__global__ void __launch_bounds__(1024) heads_scan_kernel(const __grid_constant__ Params p) {
  __shared__ int s_warp[32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int carry = 0;
  for (int t0 = 0; t0 < p.runs; t0 += 4096) {
    int v[4], sum = 0, total;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int t = t0 + threadIdx.x * 4 + k;
      v[k] = t < p.runs ? p.heads[t] : 0;
      sum += v[k];
    }
    int before = carry + block_before(sum, s_warp, total);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int t = t0 + threadIdx.x * 4 + k;
      if (t < p.runs) p.heads[t] = before;
      before += v[k];
    }
    carry += total;
  }
  if (threadIdx.x == 0) *p.count = carry;
}

constexpr int kSumThreads = 256, kAhead = 4;  // rows of grad that a thread has in flight

// A team of p.team threads takes a run of sorted ids: ids and rows go to shared memory at once, so that the loop waits for
// rows of grad alone, and those are asked for kAhead ahead.
template <typename T, int VEC>
__global__ void __launch_bounds__(kSumThreads) sums_kernel(const __grid_constant__ Params p) {
  extern __shared__ int2 s_runs[];  // [teams][run]: key, row
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int team = threadIdx.x / p.team, lane = threadIdx.x % p.team, run = blockIdx.x * (kSumThreads / p.team) + team;
  const int c = (blockIdx.y * p.team + lane) * VEC;
  const int64_t i0 = (int64_t)run * p.run, i1 = min(p.n, i0 + p.run);
  const int count = run < p.runs ? (int)(i1 - i0) : 0;
  const int32_t* keys = p.key[0];
  int2* mine = s_runs + team * p.run;
  for (int k = lane; k < count; k += p.team) mine[k] = make_int2(keys[i0 + k], p.row[0][i0 + k]);
  int prev = -1, next = -1, rank = 0;
  if (count > 0) {
    if (i0 > 0) prev = keys[i0 - 1];
    if (i1 < p.n) next = keys[i1];
    if (p.sparse) rank = p.heads[run];
  }
  __syncthreads();
  if (count == 0 || c >= p.D) return;
  const T* grad = static_cast<const T*>(p.grad) + c;
  int cur = mine[0].x;
  bool before = prev == cur;
  if (before) --rank;  // of the current row among the touched
  float acc[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) acc[v] = 0.0f;
  auto part = [&](int which) {
    float* to = p.part + ((int64_t)run * 2 + which) * p.D + c;
    store_as<float, VEC>(to, acc);
  };
  auto finish = [&] {
    if (before) return part(0);
    if (p.sparse && c == 0) p.out_ids[rank] = cur;
    store_sums<VEC>(p, p.sparse ? (int64_t)rank : (int64_t)cur, c, acc);
  };
  Raw<T, VEC> g[kAhead];
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
    if (k < count) g[k].load(grad + (int64_t)mine[k].y * p.ld_grad);
  for (int i = 0; i < count; i += kAhead) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (i + k >= count) break;
      const int key = mine[i + k].x;
      if (key != cur) {
        finish();
        cur = key;
        if (cur >= p.V) return;  // (the ids that get nothing are the last)
        before = false;
        ++rank;
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[v] = 0.0f;
      }
      if (cur >= p.V) return;
      g[k].add_to(acc);
      if (i + k + kAhead < count) g[k].load(grad + (int64_t)mine[i + k + kAhead].y * p.ld_grad);
    }
  }
  if (next != cur) return finish();
  part(before ? 0 : 1);
}

// A warp for each run whose last row starts in it and goes on: the partial sums of that row, in their order.  Rows over
// more than kNear runs are left to the CTA: teams take every so manyth partial sum, then the teams are added up.
constexpr int kFar = 32, kNear = 12;  // (3 to 31: the same within 6 %)
template <int VEC>
__global__ void __launch_bounds__(kSumThreads) combine_kernel(const __grid_constant__ Params p) {
  __shared__ float s_sum[kSumThreads * VEC];
  __shared__ int s_last[kSumThreads / 32];  // of a row that is left to the CTA, else -1
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, run0 = blockIdx.x * (kSumThreads / 32);
  const int32_t* keys = p.key[0];
  // the key of the row that starts in run r and goes on, or -1
  auto starts = [&](int r) {
    const int64_t i0 = (int64_t)r * p.run, i1 = i0 + p.run;
    if (i1 >= p.n) return -1;
    const int key = keys[i1 - 1], next = keys[i1], first = keys[i0], prev = i0 > 0 ? keys[i0 - 1] : -1;
    return key < p.V && next == key && !(first == key && prev == key) ? key : -1;  // (else it came from before)
  };
  auto add = [&](int j, int from_run, int c, float* acc) {
    const float* from = p.part + ((int64_t)j * 2 + (j == from_run ? 1 : 0)) * p.D + c;
    if constexpr (VEC == 1) {
      acc[0] += from[0];
    } else if constexpr (VEC == 2) {
      const float2 f = *reinterpret_cast<const float2*>(from);
      acc[0] += f.x;
      acc[1] += f.y;
    } else {
#pragma unroll
      for (int v = 0; v < VEC; v += 4) {
        const float4 f = *reinterpret_cast<const float4*>(from + v);
        acc[v] += f.x;
        acc[v + 1] += f.y;
        acc[v + 2] += f.z;
        acc[v + 3] += f.w;
      }
    }
  };
  auto store = [&](int r, int key, int c, float* acc) {
    int64_t at = key;
    if (p.sparse) {
      at = (int64_t)p.heads[r + 1] - 1;
      if (c == 0) p.out_ids[at] = key;
    }
    store_sums<VEC>(p, at, c, acc);
  };
  const int run = run0 + warp, key = starts(run);
  int last = -1;
  if (key >= 0) {  // the runs behind: how many of them end with the row still going on
    const int64_t end = ((int64_t)run + 2 + lane) * p.run - 1;  // of run + 1 + lane
    const bool on = end + 1 < p.n && keys[end] == key && keys[end + 1] == key;
    const uint32_t off = __ballot_sync(kAll, !on);
    last = run + __ffs(off);
    if (off == 0) {  // the last id of the row, 32 probes at once
      int64_t lo = ((int64_t)run + kFar) * p.run, hi = p.n;
      while (hi - lo > 1) {
        const int64_t step = (hi - lo + 31) / 32, m = lo + (lane + 1) * step;
        const int n = __popc(__ballot_sync(kAll, m < hi && keys[m] == key));
        lo += n * step;
        hi = min(hi, lo + step);
      }
      last = (int)(lo >> p.run_log);
    } else if (last <= run + kNear) {
      for (int c = lane * VEC; c < p.D; c += 32 * VEC) {
        float acc[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[v] = 0.0f;
#pragma unroll 6
        for (int j = run; j <= last; ++j) add(j, run, c, acc);
        store(run, key, c, acc);
      }
      last = -1;
    }
  }
  if (lane == 0) s_last[warp] = last;
  __syncthreads();
  const int teams = kSumThreads / p.team, team = threadIdx.x / p.team, slab = p.team * VEC;
  for (int w = 0; w < kSumThreads / 32; ++w) {
    if (s_last[w] < 0) continue;
    const int from = run0 + w, k = starts(from);
    for (int c0 = 0; c0 < p.D; c0 += slab) {
      const int c = c0 + threadIdx.x % p.team * VEC;
      float acc[VEC];
#pragma unroll
      for (int v = 0; v < VEC; ++v) acc[v] = 0.0f;
      if (c < p.D) {
#pragma unroll 8
        for (int j = from + team; j <= s_last[w]; j += teams) add(j, from, c, acc);
      }
      __syncthreads();
#pragma unroll
      for (int v = 0; v < VEC; ++v) s_sum[threadIdx.x * VEC + v] = acc[v];
      __syncthreads();
      if (team == 0 && c < p.D) {
        for (int t = 1; t < teams; ++t)
#pragma unroll
          for (int v = 0; v < VEC; ++v) acc[v] += s_sum[(t * p.team + threadIdx.x) * VEC + v];
        store(from, k, c, acc);
      }
    }
  }
}

// ------------------------------------------------------------------- host
static int bits_of(int64_t values) {
  int b = 1;
  while (b < 31 && ((int64_t)1 << b) < values) ++b;
  return b;
}
// Sorted ids of a team, 16 to 128: enough teams to fill the GPU (32 of 64 threads an SM), runs as long as that leaves
// them, since every run costs up to two partial sums.  512 values a row, us for 16 | 32 | 64 | 128 | 256 ids: 20,000 ids 58 |
// 63 | 71 | 92 | 134, 400,000 ids 194 | 172 | 163 | 178 | 171, 1.4 million 519 | 429 | 392 | 373 | 395.
static int run_log_of(int64_t n) {
  int log = 4;
  while (log < 7 && (n >> log) > (int64_t)sm_count() * 64) ++log;
  return log;
}
struct Sizes {
  int64_t keys, counts, heads, part, total;
};
static Sizes sizes_of(int64_t n, int D) {
  Sizes z;
  const int64_t tiles = (n + kTile - 1) / kTile, runs = (n >> run_log_of(n)) + 1;
  auto up = [](int64_t b) { return (b + 255) / 256 * 256; };
  z.keys = up(n * 4);
  z.counts = up((tiles + 1) * kDigits * 4);
  z.heads = up((runs + 1) * 4);
  z.part = up(runs * 2 * (int64_t)D * 4);
  z.total = 4 * z.keys + z.counts + z.heads + z.part;
  return z;
}

// Values of a thread's load: 16 bytes, or 8 or 4 or one value where the width, the strides or the addresses are not whole
// multiples of that; calls f with their number as a type.  60,000 rows of 1022 bf16 values, two a load: gradient 188 us,
// lookup 56 (one a load 302 and 85); of 513, one a load, 171 and 42; of 512, eight a load, 77 and 21.
template <typename T, typename F>
static int with_vec(const void* a, int64_t lda, const void* b, int64_t ldb, int b_size, int D, const F& f) {
  auto whole = [&](int v) {
    return D % v == 0 && lda % v == 0 && ldb % v == 0 && aligned(a, v * (int)sizeof(T)) && aligned(b, std::min(v * b_size, 16));
  };
  if (whole(16 / (int)sizeof(T))) return f(std::integral_constant<int, 16 / (int)sizeof(T)>());
  if (sizeof(T) == 2 && whole(4)) return f(std::integral_constant<int, 4>());
  if (whole(2)) return f(std::integral_constant<int, 2>());
  return f(std::integral_constant<int, 1>());
}

template <typename T, int VEC>
static int run_lookup(Params p, cudaStream_t st) {
  const int chunks = (p.D + VEC - 1) / VEC;
  p.team = 1;
  while (p.team < chunks && p.team < 32) p.team *= 2;
  const int64_t rows = (int64_t)(256 / p.team) * kLookupRows;  // of a CTA at a time
  const int64_t blocks = std::min<int64_t>((p.n + rows - 1) / rows, (int64_t)sm_count() * 64);
  lookup_kernel<T, VEC><<<(unsigned)blocks, 256, 0, st>>>(p);
  return check_cuda(cudaGetLastError(), "embedding lookup_kernel launch");
}

// a launch that may start under the one before it (whose results it waits for by itself)
static int chain(const void* kernel, dim3 grid, int threads, int smem, cudaStream_t st, Params& p, const char* what) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  void* args[] = {&p};
  return check_cuda(cudaLaunchKernelExC(&cfg, kernel, args), what);
}

static int sort_ids(Params& p, cudaStream_t st) {
  int rc;
  const int fill = p.zero_bytes > 0 ? (int)std::min<int64_t>(2 * sm_count(), (p.zero_bytes + 65535) / 65536) : 0;
  if (p.n <= kSmall) {
    static std::once_flag once[64];
    int dev = 0;
    cudaGetDevice(&dev);
    cudaError_t e = cudaSuccess;
    std::call_once(once[dev & 63], [&] {
      e = cudaFuncSetAttribute(small_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Small));
    });
    if (e != cudaSuccess) return check_cuda(e, "cudaFuncSetAttribute(embedding small_sort_kernel)");
    small_sort_kernel<<<1 + fill, kSmallThreads, sizeof(Small), st>>>(p);
    return check_cuda(cudaGetLastError(), "embedding small_sort_kernel launch");
  }
  p.tiles = (int)((p.n + kTile - 1) / kTile);
  p.scanned = p.tiles > kDirect;
  for (p.shift = 0; p.shift < p.bits; p.shift += 8) {
    if (p.shift == 0) {
      count_kernel<true><<<p.tiles + fill, kSortThreads, 0, st>>>(p);
      rc = check_cuda(cudaGetLastError(), "embedding count_kernel launch");
    } else {
      rc = chain((const void*)count_kernel<false>, dim3(p.tiles), kSortThreads, 0, st, p, "embedding count_kernel launch");
    }
    if (rc) return rc;
    if (p.scanned && (rc = chain((const void*)scan_kernel, dim3(kDigits), 256, 0, st, p, "embedding scan_kernel launch"))) return rc;
    if ((rc = chain((const void*)scatter_kernel, dim3(p.tiles), kSortThreads, 0, st, p, "embedding scatter_kernel launch"))) return rc;
    std::swap(p.key[0], p.key[1]);
    std::swap(p.row[0], p.row[1]);
  }
  return RB_OK;
}

template <typename T, int VEC>
static int run_sums(Params& p, cudaStream_t st) {
  int rc;
  const int chunks = (p.D + VEC - 1) / VEC;
  p.team = 32;
  while (p.team < chunks && p.team < kSumThreads) p.team *= 2;
  const unsigned slabs = (unsigned)((chunks + p.team - 1) / p.team);
  const int teams = kSumThreads / p.team;
  if (p.sparse) {
    if ((rc = chain((const void*)heads_kernel, dim3((p.runs + 7) / 8), 256, 0, st, p, "embedding heads_kernel launch"))) return rc;
    if ((rc = chain((const void*)heads_scan_kernel, dim3(1), 1024, 0, st, p, "embedding heads_scan_kernel launch"))) return rc;
  }
  if ((rc = chain((const void*)sums_kernel<T, VEC>, dim3((p.runs + teams - 1) / teams, slabs), kSumThreads, teams * p.run * 8, st, p,
                  "embedding sums_kernel launch")))
    return rc;
  if (p.runs == 1) return RB_OK;
  return chain((const void*)combine_kernel<VEC>, dim3((p.runs + 7) / 8), kSumThreads, 0, st, p, "embedding combine_kernel launch");
}

template <typename T>
static int run_backward(Params& p, cudaStream_t st) {
  int rc;
  if ((rc = sort_ids(p, st))) return rc;
  return with_vec<T>(p.grad, p.ld_grad, p.out, p.ld_out, dtype_size(p.out_dtype), p.D,
                     [&](auto v) { return run_sums<T, decltype(v)::value>(p, st); });
}

static int check_shape(int64_t V, int D, int64_t n, int idx_dtype, int dtype) {
  if (V < 0 || D <= 0 || n < 0) return fail(RB_ERR_VALUE, "negative or empty embedding shape");
  if (dtype != RB_BF16 && dtype != RB_F16 && dtype != RB_F32) return fail(RB_ERR_VALUE, "embedding rows are fp32, bf16 or f16");
  if (idx_dtype != RB_I64 && idx_dtype != RB_I32) return fail(RB_ERR_VALUE, "ids must be int64 or int32");
  if (V > 0x7ffffffeLL || n > 1 << 30) return fail(RB_ERR_UNSUPPORTED, "more than 2^31 - 2 rows or 2^30 ids");
  if (n > 0 && V == 0) return fail(RB_ERR_VALUE, "ids of an empty table");
  return RB_OK;
}

static int backward(const void* grad, int dtype, int64_t ld_grad, int D, const void* ids, int idx_dtype, int64_t n, int64_t V,
                    const void* bags, int64_t n_bags, int64_t padding, float scale, int accumulate, void* workspace,
                    int64_t workspace_bytes, void* out, int out_dtype, int64_t ld_out, int64_t* out_ids, int32_t* count,
                    bool sparse, cudaStream_t st) {
  int rc;
  if ((rc = check_shape(V, D, n, idx_dtype, dtype)) || (rc = check_shape(V, D, n, idx_dtype, out_dtype))) return rc;
  if (ld_grad < D || ld_out < D) return fail(RB_ERR_VALUE, "leading dimension smaller than the row");
  if (bags != nullptr && (n_bags < 0 || n_bags > 1 << 30)) return fail(RB_ERR_VALUE, "bad number of bags");
  if (bags != nullptr && n_bags == 0) n = 0;
  if ((n > 0 && (grad == nullptr || ids == nullptr)) || ((sparse ? n : V) > 0 && out == nullptr) ||
      (sparse && (count == nullptr || (n > 0 && out_ids == nullptr))))
    return fail(RB_ERR_VALUE, "null operand");
  const Sizes z = sizes_of(n, D);
  if (n > 0 && (workspace == nullptr || workspace_bytes < z.total || !aligned(workspace, 16)))
    return fail(RB_ERR_VALUE, "workspace of %lld bytes (16-byte aligned) needed, %lld given", (long long)z.total,
                (long long)workspace_bytes);
  if (!device_is_sm100()) return fail(RB_ERR_DEVICE, "the embedding kernels need an sm_100 (B200) device");
  const bool zeros = !sparse && !accumulate && V > 0;
  // (rows apart, or rows off 16 bytes, are filled row by row)
  const bool whole = ld_out == D && aligned(out, 16);
  if (zeros && (n == 0 || !whole)) {
    const size_t e = (size_t)dtype_size(out_dtype);
    if ((rc = check_cuda(cudaMemset2DAsync(out, ld_out * e, 0, D * e, (size_t)V, st), "embedding gradient's zeros"))) return rc;
  }
  if (n == 0) return sparse ? check_cuda(cudaMemsetAsync(count, 0, 4, st), "embedding count") : RB_OK;
  Params p{};
  p.grad = grad;
  p.ids = ids;
  p.bags = bags;
  p.out = out;
  p.out_ids = out_ids;
  p.count = count;
  p.ld_grad = ld_grad;
  p.ld_out = ld_out;
  p.V = V;
  p.n = n;
  p.n_bags = n_bags;
  p.padding = padding;
  p.scale = scale;
  p.D = D;
  p.wide_ids = idx_dtype == RB_I64;
  p.out_dtype = out_dtype;
  p.accumulate = accumulate;
  p.sparse = sparse;
  p.zero_bytes = zeros && whole ? V * D * dtype_size(out_dtype) : 0;
  p.bits = bits_of(V + 1);
  p.run_log = run_log_of(n);
  p.run = 1 << p.run_log;
  p.runs = (int)((n + p.run - 1) >> p.run_log);
  uint8_t* w = static_cast<uint8_t*>(workspace);
  for (int i = 0; i < 2; ++i) {
    p.key[i] = reinterpret_cast<int32_t*>(w);
    w += z.keys;
    p.row[i] = reinterpret_cast<int32_t*>(w);
    w += z.keys;
  }
  p.counts = reinterpret_cast<int32_t*>(w);
  p.totals = p.counts + (int64_t)((n + kTile - 1) / kTile) * kDigits;
  w += z.counts;
  p.heads = reinterpret_cast<int32_t*>(w);
  w += z.heads;
  p.part = reinterpret_cast<float*>(w);
  switch (dtype) {
    case RB_BF16: return run_backward<__nv_bfloat16>(p, st);
    case RB_F16: return run_backward<__half>(p, st);
    default: return run_backward<float>(p, st);
  }
}

template <typename T>
static int lookup(const Params& p, cudaStream_t st) {
  return with_vec<T>(p.table, p.ld_table, p.out, p.ld_out, sizeof(T), p.D,
                     [&](auto v) { return run_lookup<T, decltype(v)::value>(p, st); });
}

}  // namespace embed
}  // namespace rb

using namespace rb;

extern "C" int rb_embed_rows(const void* table, int dtype, int64_t ld, int64_t V, int D, const void* ids, int idx_dtype,
                             int64_t n, float scale, void* out, int64_t ldo, void* stream) {
  using namespace rb::embed;
  int rc;
  if ((rc = check_shape(V, D, n, idx_dtype, dtype))) return rc;
  if (ld < D || ldo < D) return fail(RB_ERR_VALUE, "leading dimension smaller than the row");
  if (n > 0 && (table == nullptr || ids == nullptr || out == nullptr)) return fail(RB_ERR_VALUE, "null operand");
  if (!device_is_sm100()) return fail(RB_ERR_DEVICE, "rb_embed_rows needs an sm_100 (B200) device");
  if (n == 0) return RB_OK;
  Params p{};
  p.table = table;
  p.ids = ids;
  p.out = out;
  p.ld_table = ld;
  p.ld_out = ldo;
  p.V = V;
  p.n = n;
  p.scale = scale;
  p.D = D;
  p.wide_ids = idx_dtype == RB_I64;
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case RB_BF16: return lookup<__nv_bfloat16>(p, st);
    case RB_F16: return lookup<__half>(p, st);
    default: return lookup<float>(p, st);
  }
}

extern "C" int64_t rb_embed_rows_backward_workspace_size(int64_t n, int D) {
  if (n < 0 || n > 1 << 30 || D <= 0) return -1;
  return n == 0 ? 0 : embed::sizes_of(n, D).total;
}

extern "C" int rb_embed_rows_backward(const void* grad, int dtype, int64_t ld_grad, int D, const void* ids, int idx_dtype,
                                      int64_t n, int64_t V, const void* bags, int64_t n_bags, int64_t padding, float scale,
                                      int accumulate, void* workspace, int64_t workspace_bytes, void* out, int out_dtype,
                                      int64_t ld_out, void* stream) {
  return embed::backward(grad, dtype, ld_grad, D, ids, idx_dtype, n, V, bags, n_bags, padding, scale, accumulate != 0, workspace,
                         workspace_bytes, out, out_dtype, ld_out, nullptr, nullptr, false, (cudaStream_t)stream);
}

extern "C" int rb_embed_rows_backward_sparse(const void* grad, int dtype, int64_t ld_grad, int D, const void* ids, int idx_dtype,
                                             int64_t n, int64_t V, const void* bags, int64_t n_bags, int64_t padding, float scale,
                                             void* workspace, int64_t workspace_bytes, int64_t* out_ids, void* out_rows,
                                             int out_dtype, int64_t ld_out, int32_t* count, void* stream) {
  return embed::backward(grad, dtype, ld_grad, D, ids, idx_dtype, n, V, bags, n_bags, padding, scale, 0, workspace,
                         workspace_bytes, out_rows, out_dtype, ld_out, out_ids, count, true, (cudaStream_t)stream);
}

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
// so a row that a tenth of all ids ask for costs no more than its bytes.
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
  int vec;                       // values of a thread's load (16 bytes), or 1
  // workspace
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

// VEC values from memory as fp32
template <typename T, int VEC>
__device__ __forceinline__ void load_values(const T* p, float* v) {
  if constexpr (VEC == 1) {
    v[0] = to_f32(__ldg(p));
  } else {
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, float>::value) {
        v[i] = __uint_as_float(u[i]);
      } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        v[2 * i] = bf16_lo(u[i]);
        v[2 * i + 1] = bf16_hi(u[i]);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
  }
}
// VEC values to memory as T2, whole words where there are several (from an aligned address)
template <typename T2, int VEC>
__device__ __forceinline__ void store_as(T2* p, const float* v) {
  if constexpr (VEC == 1) {
    p[0] = T2(v[0]);
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
    if constexpr (VEC == 4) *reinterpret_cast<uint2*>(p) = make_uint2(u[0], u[1]);
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
constexpr int kRowsAThread = 4;  // loads in flight

template <typename T, int VEC>
__global__ void __launch_bounds__(256) lookup_kernel(const __grid_constant__ Params p) {
  const int chunks = (p.D + VEC - 1) / VEC;
  const int64_t total = p.n * chunks, step = (int64_t)gridDim.x * 256;
  const T* table = static_cast<const T*>(p.table);
  T* out = static_cast<T*>(p.out);
  for (int64_t i0 = (int64_t)blockIdx.x * 256 + threadIdx.x; i0 < total; i0 += step * kRowsAThread) {
    float v[kRowsAThread][VEC];
    int64_t to[kRowsAThread];
#pragma unroll
    for (int k = 0; k < kRowsAThread; ++k) {
      const int64_t i = i0 + k * step;
      to[k] = -1;
      if (i < total) {
        const int64_t r = i / chunks;
        const int c = (int)(i - r * chunks) * VEC;
        const int64_t id = min(max(id_at(p.ids, p.wide_ids, r), (int64_t)0), p.V - 1);
        load_values<T, VEC>(table + id * p.ld_table + c, v[k]);
        to[k] = r * p.ld_out + c;
      }
    }
#pragma unroll
    for (int k = 0; k < kRowsAThread; ++k) {
      if (to[k] < 0) continue;
#pragma unroll
      for (int c = 0; c < VEC; ++c) v[k][c] *= p.scale;
      store_as<T, VEC>(out + to[k], v[k]);
    }
  }
}

// ------------------------------------------------------------------- sort
// A stable radix sort, 8 bits a pass.  A CTA ranks a tile of kTile keys: each warp counts its own 512 in their order
// (lanes with equal digits find each other by eight ballots), then warps and tiles are added up before it.
constexpr int kSortThreads = 256, kPerThread = 16, kTile = kSortThreads * kPerThread;
constexpr int kDigits = 256;
constexpr int kDirect = 64;  // up to so many tiles a CTA adds up the counts of those before it by itself

// the row of grad of id i, or -1: i itself, or its bag, searched in [lo, hi]
__device__ __forceinline__ int bag_of(const Params& p, int64_t i, int64_t lo, int64_t hi) {
  // the last b in [lo, hi] with bags[b] <= i
  while (lo < hi) {
    const int64_t m = (lo + hi + 1) >> 1;
    if (id_at(p.bags, p.wide_ids, m) <= i) lo = m;
    else hi = m - 1;
  }
  return (int)lo;
}
// key (the table row, V for an id that gets nothing) and row of grad of id i
__device__ __forceinline__ void source_of(const Params& p, int64_t i, int64_t lo, int64_t hi, int& key, int& row) {
  const int64_t id = id_at(p.ids, p.wide_ids, i);
  key = (int)min(max(id, (int64_t)0), p.V - 1);
  row = (int)i;
  if (p.bags != nullptr) {
    row = bag_of(p, i, lo, hi);
    if (row >= p.n_bags || i < id_at(p.bags, p.wide_ids, row) || i >= id_at(p.bags, p.wide_ids, row + 1)) key = (int)p.V;
    row = min(row, (int)max(p.n_bags - 1, (int64_t)0));
  }
  if (p.padding >= 0 && key == p.padding) key = (int)p.V;
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

__device__ __forceinline__ void zero_fill(const Params& p, int64_t block, int64_t blocks) {
  uint4* to = static_cast<uint4*>(p.out);
  const int64_t n = p.zero_bytes / 16;
  for (int64_t i = block * kSortThreads + threadIdx.x; i < n; i += blocks * kSortThreads) to[i] = make_uint4(0u, 0u, 0u, 0u);
  uint8_t* rest = static_cast<uint8_t*>(p.out);
  if (block == 0 && threadIdx.x < p.zero_bytes % 16) rest[n * 16 + threadIdx.x] = 0;
}

// Counts of a pass's digits in each tile.  FIRST: keys come from the ids and are written in their order with their rows;
// CTAs behind the tiles' fill the gradient with zeros, which few tiles leave most of the GPU free for.
template <bool FIRST>
__global__ void __launch_bounds__(kSortThreads) count_kernel(const __grid_constant__ Params p) {
  if (FIRST && (int)blockIdx.x >= p.tiles) {
    zero_fill(p, blockIdx.x - p.tiles, gridDim.x - p.tiles);
    return;
  }
  __shared__ int s_count[kDigits];
  __shared__ int64_t s_bag[2];
  s_count[threadIdx.x] = 0;
  const int tile = blockIdx.x;
  if (FIRST && p.bags != nullptr && threadIdx.x < 2) {
    const int64_t i = threadIdx.x ? min(p.n - 1, (int64_t)(tile + 1) * kTile - 1) : (int64_t)tile * kTile;
    s_bag[threadIdx.x] = bag_of(p, i, 0, p.n_bags);
  }
  __syncthreads();
#pragma unroll 4
  for (int k = 0; k < kPerThread; ++k) {
    const int64_t i = item_at(tile, k);
    if (i >= p.n) continue;
    int key;
    if (FIRST) {
      int row;
      source_of(p, i, s_bag[0], s_bag[1], key, row);
      p.key[0][i] = key;
      p.row[0][i] = row;
    } else {
      key = __ldg(p.key[0] + i);
    }
    atomicAdd(&s_count[(key >> p.shift) & (kDigits - 1)], 1);
  }
  __syncthreads();
  if (p.scanned) p.counts[(int64_t)threadIdx.x * p.tiles + tile] = s_count[threadIdx.x];
  else p.counts[tile * kDigits + threadIdx.x] = s_count[threadIdx.x];
}

// sums before each of a CTA's values (256 threads), and their total
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
  int before = 0, all = 0;
  for (int w = 0; w < (int)blockDim.x / 32; ++w) {
    if (w < warp) before += s_warp[w];
    all += s_warp[w];
  }
  total = all;
  return before + x - v;
}

// one CTA a digit: its counts become the sums before them
__global__ void __launch_bounds__(256) scan_kernel(const __grid_constant__ Params p) {
  __shared__ int s_warp[8];
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

__global__ void __launch_bounds__(kSortThreads) scatter_kernel(const __grid_constant__ Params p) {
  __shared__ int s_hist[kSortThreads / 32][kDigits];
  __shared__ int s_warp[8];
  const int tile = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int key[kPerThread], row[kPerThread], rank[kPerThread];
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    const int64_t i = item_at(tile, k);
    key[k] = i < p.n ? __ldg(p.key[0] + i) : -1;
    row[k] = i < p.n ? __ldg(p.row[0] + i) : 0;
  }
  for (int w = 0; w < kSortThreads / 32; ++w) s_hist[w][threadIdx.x] = 0;
  // where each digit's keys of this tile go
  int total, mine = 0, all = 0;
  if (p.scanned) {
    mine = p.counts[(int64_t)threadIdx.x * p.tiles + tile];
    all = p.totals[threadIdx.x];
  } else {
#pragma unroll 8
    for (int t = 0; t < p.tiles; ++t) {
      const int c = p.counts[t * kDigits + threadIdx.x];
      if (t < tile) mine += c;
      all += c;
    }
  }
  mine += block_before(all, s_warp, total);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    const bool there = item_at(tile, k) < p.n;
    const int digit = (key[k] >> p.shift) & (kDigits - 1);
    const uint32_t same = peers_of(digit, there);
    const int before = there ? s_hist[warp][digit] : 0;
    rank[k] = before + __popc(same & ((1u << lane) - 1u));
    __syncwarp();
    if (there && (same >> lane) == 1u) s_hist[warp][digit] = before + __popc(same);
    __syncwarp();
  }
  __syncthreads();
  for (int w = 0; w < kSortThreads / 32; ++w) {
    const int c = s_hist[w][threadIdx.x];
    s_hist[w][threadIdx.x] = mine;
    mine += c;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    if (item_at(tile, k) >= p.n) continue;
    const int to = s_hist[warp][(key[k] >> p.shift) & (kDigits - 1)] + rank[k];
    p.key[1][to] = key[k];
    p.row[1][to] = row[k];
  }
}

// All passes of up to kSmall ids in one CTA, in shared memory.
constexpr int kSmallThreads = 1024, kSmallPer = 4, kSmall = kSmallThreads * kSmallPer;
struct Small {
  int key[2][kSmall], row[2][kSmall];
  int hist[kSmallThreads / 32][kDigits];
  int warp[32];
};
__global__ void __launch_bounds__(kSmallThreads) small_sort_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(16) uint8_t raw[];
  Small& s = *reinterpret_cast<Small*>(raw);
  if (blockIdx.x > 0) {
    uint4* to = static_cast<uint4*>(p.out);
    const int64_t n = p.zero_bytes / 16;
    for (int64_t i = (int64_t)(blockIdx.x - 1) * kSmallThreads + threadIdx.x; i < n; i += (int64_t)(gridDim.x - 1) * kSmallThreads)
      to[i] = make_uint4(0u, 0u, 0u, 0u);
    if (blockIdx.x == 1 && threadIdx.x < p.zero_bytes % 16) static_cast<uint8_t*>(p.out)[n * 16 + threadIdx.x] = 0;
    return;
  }
  const int n = (int)p.n, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < n; i += kSmallThreads) source_of(p, i, 0, p.n_bags, s.key[0][i], s.row[0][i]);
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
  const int run = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (run >= p.runs) return;
  int n = 0;
  for (int k = lane; k < p.run; k += 32) {
    const int64_t i = (int64_t)run * p.run + k;
    if (i < p.n) {
      const int key = __ldg(p.key[0] + i);
      n += key < p.V && (i == 0 || __ldg(p.key[0] + i - 1) != key);
    }
  }
  n = __reduce_add_sync(kAll, n);
  if (lane == 0) p.heads[run] = n;
}
// ... and how many before it, by one CTA
__global__ void __launch_bounds__(1024) heads_scan_kernel(const __grid_constant__ Params p) {
  __shared__ int s_warp[32];
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

template <typename T, int VEC>
__global__ void __launch_bounds__(kSumThreads) sums_kernel(const __grid_constant__ Params p) {
  const int team = threadIdx.x / p.team, run = blockIdx.x * (kSumThreads / p.team) + team;
  const int c = (blockIdx.y * p.team + threadIdx.x % p.team) * VEC;
  if (run >= p.runs || c >= p.D) return;
  const int64_t i0 = (int64_t)run * p.run, i1 = min(p.n, i0 + p.run);
  const T* grad = static_cast<const T*>(p.grad) + c;
  const int32_t* keys = p.key[0];
  int cur = __ldg(keys + i0);
  bool before = i0 > 0 && __ldg(keys + i0 - 1) == cur;
  int64_t rank = p.sparse ? (int64_t)p.heads[run] - (before ? 1 : 0) : 0;  // of the current row among the touched
  float acc[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) acc[v] = 0.0f;
  auto part = [&](int which) {
    float* to = p.part + ((int64_t)run * 2 + which) * p.D + c;
#pragma unroll
    for (int v = 0; v < VEC; ++v) to[v] = acc[v];
  };
  auto finish = [&] {
    if (cur >= p.V) return;
    if (before) return part(0);
    if (p.sparse && c == 0) p.out_ids[rank] = cur;
    store_sums<VEC>(p, p.sparse ? rank : (int64_t)cur, c, acc);
  };
  for (int64_t i = i0; i < i1; i += kAhead) {
    float g[kAhead][VEC];
    int key[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      key[k] = i + k < i1 ? __ldg(keys + i + k) : -1;
      if (key[k] >= 0 && key[k] < p.V) load_values<T, VEC>(grad + (int64_t)__ldg(p.row[0] + i + k) * p.ld_grad, g[k]);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (key[k] < 0 || key[k] >= p.V) {
        if (key[k] >= 0 && key[k] != cur) {
          finish();
          cur = key[k];
        }
        continue;
      }
      if (key[k] != cur) {
        finish();
        cur = key[k];
        before = false;
        ++rank;
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[v] = 0.0f;
      }
#pragma unroll
      for (int v = 0; v < VEC; ++v) acc[v] += g[k][v];
    }
  }
  if (cur >= p.V) return;
  const bool on = i1 < p.n && __ldg(keys + i1) == cur;
  if (!on) return finish();
  part(before ? 0 : 1);
}

// A CTA for each run whose last row starts in it and goes on: the partial sums of that row, in teams that take every so
// manyth of them, then the teams in their order.
template <int VEC>
__global__ void __launch_bounds__(kSumThreads) combine_kernel(const __grid_constant__ Params p) {
  __shared__ float s_sum[kSumThreads * VEC];
  const int run = blockIdx.x;
  const int64_t i0 = (int64_t)run * p.run, i1 = i0 + p.run;
  if (i1 >= p.n) return;
  const int32_t* keys = p.key[0];
  const int key = __ldg(keys + i1 - 1);
  if (key >= p.V || __ldg(keys + i1) != key) return;
  if (__ldg(keys + i0) == key && i0 > 0 && __ldg(keys + i0 - 1) == key) return;  // (it came from before)
  int64_t lo = i1, hi = p.n;  // the first id behind the row
  while (lo < hi) {
    const int64_t m = (lo + hi) >> 1;
    if (__ldg(keys + m) <= key) lo = m + 1;
    else hi = m;
  }
  const int last = (int)((lo - 1) >> p.run_log);
  const int teams = kSumThreads / p.team, team = threadIdx.x / p.team;
  const int c = (blockIdx.y * p.team + threadIdx.x % p.team) * VEC;
  float acc[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) acc[v] = 0.0f;
  if (c < p.D) {
#pragma unroll 4
    for (int j = run + team; j <= last; j += teams) {
      const float* from = p.part + ((int64_t)j * 2 + (j == run ? 1 : 0)) * p.D + c;
#pragma unroll
      for (int v = 0; v < VEC; ++v) acc[v] += from[v];
    }
  }
#pragma unroll
  for (int v = 0; v < VEC; ++v) s_sum[threadIdx.x * VEC + v] = acc[v];
  __syncthreads();
  if (team > 0 || c >= p.D) return;
  for (int t = 1; t < teams; ++t)
#pragma unroll
    for (int v = 0; v < VEC; ++v) acc[v] += s_sum[(t * p.team + threadIdx.x) * VEC + v];
  int64_t at = key;
  if (p.sparse) {
    at = (int64_t)p.heads[run + 1] - 1;
    if (c == 0) p.out_ids[at] = key;
  }
  store_sums<VEC>(p, at, c, acc);
}

// ------------------------------------------------------------------- host
static int bits_of(int64_t values) {
  int b = 1;
  while (b < 31 && ((int64_t)1 << b) < values) ++b;
  return b;
}
// Sorted ids of a team: enough teams to fill the GPU (32 of 64 threads an SM), runs as long as that leaves them, since
// every run costs up to two partial sums.
static int run_log_of(int64_t n) {
  int log = 4;
  while (log < 8 && (n >> log) > (int64_t)sm_count() * 32) ++log;
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

template <typename T>
static int vec_of(const void* a, int64_t lda, const void* b, int64_t ldb, int b_size, int D) {
  const int v = 16 / (int)sizeof(T);
  return D % v == 0 && aligned(a, 16) && lda % v == 0 && aligned(b, 16) && ldb * b_size % 16 == 0 ? v : 1;
}

template <typename T, int VEC>
static int run_lookup(const Params& p, cudaStream_t st) {
  const int64_t total = p.n * ((p.D + VEC - 1) / VEC);
  const int64_t blocks = std::min<int64_t>((total + 255) / 256, (int64_t)sm_count() * 32);
  lookup_kernel<T, VEC><<<(unsigned)blocks, 256, 0, st>>>(p);
  return check_cuda(cudaGetLastError(), "embedding lookup_kernel launch");
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
    if (p.shift == 0) count_kernel<true><<<p.tiles + fill, kSortThreads, 0, st>>>(p);
    else count_kernel<false><<<p.tiles, kSortThreads, 0, st>>>(p);
    if ((rc = check_cuda(cudaGetLastError(), "embedding count_kernel launch"))) return rc;
    if (p.scanned) {
      scan_kernel<<<kDigits, 256, 0, st>>>(p);
      if ((rc = check_cuda(cudaGetLastError(), "embedding scan_kernel launch"))) return rc;
    }
    scatter_kernel<<<p.tiles, kSortThreads, 0, st>>>(p);
    if ((rc = check_cuda(cudaGetLastError(), "embedding scatter_kernel launch"))) return rc;
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
    heads_kernel<<<(p.runs + 7) / 8, 256, 0, st>>>(p);
    if ((rc = check_cuda(cudaGetLastError(), "embedding heads_kernel launch"))) return rc;
    heads_scan_kernel<<<1, 1024, 0, st>>>(p);
    if ((rc = check_cuda(cudaGetLastError(), "embedding heads_scan_kernel launch"))) return rc;
  }
  sums_kernel<T, VEC><<<dim3((p.runs + teams - 1) / teams, slabs), kSumThreads, 0, st>>>(p);
  if ((rc = check_cuda(cudaGetLastError(), "embedding sums_kernel launch"))) return rc;
  if (p.runs > 1) {
    combine_kernel<VEC><<<dim3(p.runs - 1, slabs), kSumThreads, 0, st>>>(p);
    rc = check_cuda(cudaGetLastError(), "embedding combine_kernel launch");
  }
  return rc;
}

template <typename T>
static int run_backward(Params& p, cudaStream_t st) {
  int rc;
  if ((rc = sort_ids(p, st))) return rc;
  if (vec_of<T>(p.grad, p.ld_grad, p.out, p.ld_out, dtype_size(p.out_dtype), p.D) > 1) return run_sums<T, 16 / sizeof(T)>(p, st);
  return run_sums<T, 1>(p, st);
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
  if (vec_of<T>(p.table, p.ld_table, p.out, p.ld_out, sizeof(T), p.D) > 1) return run_lookup<T, 16 / sizeof(T)>(p, st);
  return run_lookup<T, 1>(p, st);
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

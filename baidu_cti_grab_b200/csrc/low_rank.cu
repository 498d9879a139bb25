// low_rank.cu -- low-rank adapters of many requests beside a projection that they
// share: out[t] = y[t] + scale[i] * B_i (A_i x[t]) for token t's adapter i = idx[t]
// (y is the shared projection's output; a token without an adapter keeps y).
//
// Three kernels, by the sizes:
//
// * token kernel: a cluster of CTAs per token, CUDA cores.  Few tokens (or few products
//   in all) are bound by the latency of reading their adapters: the CTAs of a cluster split A's columns,
//   share the partial h = A x through distributed shared memory and split B's rows.
//   Also takes every shape that the tensor maps cannot.
// * tile kernel: 128 tokens a CTA on tcgen05.  The tile's distinct adapters are
//   listed, and taken in groups whose ranks fill 64 (or 128) columns:
//     H [128, 64] = X [128, K] . [A_i ; A_j ; ...]^T   all of the group in one MMA per K step
//     each row keeps its own adapter's columns, the others become zeros
//     out tile = H . [B_i | B_j | ...]^T               the zeros select the adapter
//   so tokens need no sorting and a tile of mixed requests costs MMA work (of which
//   there is plenty), not bytes.  A row is written in the group that has its adapter.
// * the same split in two, H then out, when there is a 128-token tile an SM
//   or fewer: H is split along K (fp32 partials in the workspace, summed in a fixed
//   order), out along N.
//
// What bounds it: HBM from about 20k tokens (x and y read, out written once), the
// two GEMMs being 2 r (K + N) operations a token.  Sums are fp32.  The second product
// takes h in two values of the model type (16 or 22 bits; fp16 rows are brought into
// the type's range first), the second of them from TMEM: the MMAs are twice as many
// and cost nothing that was measured, splitting and storing h costs 2-5 % (103725 x
// 512 83 -> 85 us, 4099 x 14336 48.5 -> 51, 9001 x 1000 50 -> 52).  With h rounded
// to the type, out was 1.25 times as far from the exact sum.  out is rounded once.
//
// Measured on a B200: 64 tokens of their own adapters (512 to 1536, rank 16) 5.5 us,
// a launch, a cluster barrier and three dependent reads; 103725 x 512 to 512, rank 16,
// 85 us (0.57 of HBM: tiles take 17-21 us at the bandwidth, the few with over four
// adapters 40 and end last); 4099 x 14336 to 512, rank 32, 51 us (H by itself 29, 0.6
// of the copy rate in 264 CTAs of 28 K blocks each, of which the start is not hidden;
// out by itself 25 for 8 MB, most of it its start and the partial sums); 9001 x 1000 to
// 1544, rank 8, in runs of 7, 52 us (by themselves, caches cold, H 16 and out 49, in its
// longest tile).  Ranks padded to 16 columns and four warps of rows took 83 us there.
#include "common.cuh"

#include <algorithm>
#include <mutex>
#include <type_traits>

namespace rb {
namespace lowrank {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kMaxRank = 128;

struct Params {
  const void *y, *x, *a, *b, *idx;
  const float* scale;  // [R] or null
  void* out;
  float* part;         // [splits][T][rank] partial h, or null
  int64_t ldy, ldx, ldo, T;
  int K, N, R, rank, idx64;
  int unit;            // columns of B that a copy brings side by side: 64, 32 or 16 (swizzled), 8
  int chunk_io;        // y and out can be moved by whole chunks
  int splits;          // of K (H alone) -- partials to sum (out alone)
  int chunks;          // 64-column chunks of a CTA (out alone)
  int vec_y, vec_out;  // bytes of the loads and stores that rows allow: 32, 16 or 2
};

__device__ __forceinline__ int adapter_of(const Params& p, int64_t t) {
  if (t >= p.T) return -1;
  const int64_t i = p.idx64 ? __ldg(static_cast<const int64_t*>(p.idx) + t)
                            : (int64_t)__ldg(static_cast<const int32_t*>(p.idx) + t);
  return i >= 0 && i < p.R ? (int)i : -1;
}

template <typename T>
__device__ __forceinline__ float to_f32(T v) { return (float)v; }

// eight 16-bit values times eight others, added up
template <typename T>
__device__ __forceinline__ float dot8(uint4 a, uint4 b, float s) {
  const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      s = fmaf(bf16_lo(aw[i]), bf16_lo(bw[i]), s);
      s = fmaf(bf16_hi(aw[i]), bf16_hi(bw[i]), s);
    } else {
      const float2 u = __half22float2(*reinterpret_cast<const __half2*>(&aw[i]));
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&bw[i]));
      s = fmaf(u.x, v.x, s);
      s = fmaf(u.y, v.y, s);
    }
  }
  return s;
}

// ------------------------------------------------------------ token kernel
constexpr int kTokenThreads = 256;

// VEC: 16-byte loads of x, A and B (K and rank multiples of 8, aligned bases and rows).
template <typename T, bool VEC>
__global__ void __launch_bounds__(kTokenThreads) token_kernel(const __grid_constant__ Params p) {
  __shared__ float s_part[kMaxRank], s_h[kMaxRank];
  const uint32_t rank = tc::pair::cluster_rank();
  uint32_t size;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
  const int64_t t = blockIdx.x / size;
  const int i = adapter_of(p, t);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* x = static_cast<const T*>(p.x) + t * p.ldx;
  const T* y = static_cast<const T*>(p.y) + t * p.ldy;
  T* out = static_cast<T*>(p.out) + t * p.ldo;
  const int n0 = (int)((int64_t)p.N * rank / size), n1 = (int)((int64_t)p.N * (rank + 1) / size);
  if (i < 0) {  // the whole cluster alike
    if (out != y)
      for (int n = n0 + threadIdx.x; n < n1; n += kTokenThreads) out[n] = y[n];
    return;
  }
  // this CTA's part of h: eights of K from k0 to k1, a warp for each rank in turn
  const T* a = static_cast<const T*>(p.a) + (int64_t)i * p.rank * p.K;
  const int eights = (p.K + 7) / 8;
  const int k0 = (int)((int64_t)eights * rank / size) * 8;
  const int k1 = min(p.K, (int)((int64_t)eights * (rank + 1) / size) * 8);
  for (int j = warp; j < p.rank; j += kTokenThreads / 32) {
    const T* row = a + (int64_t)j * p.K;
    float s = 0.0f;
    if constexpr (VEC) {
#pragma unroll 4
      for (int k = k0 + lane * 8; k < k1; k += 256)
        s = dot8<T>(__ldg(reinterpret_cast<const uint4*>(row + k)), __ldg(reinterpret_cast<const uint4*>(x + k)), s);
    } else {
      for (int k = k0 + lane; k < k1; k += 32) s = fmaf(to_f32(row[k]), to_f32(x[k]), s);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kAll, s, o);
    if (lane == 0) s_part[j] = s;
  }
  if (size > 1) {
    tc::pair::cluster_sync_all();
    for (int j = threadIdx.x; j < p.rank; j += kTokenThreads) {
      float s = 0.0f;
      for (uint32_t c = 0; c < size; ++c) {
        float v;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(tc::pair::map_rank(smem_u32(&s_part[j]), c)) : "memory");
        s += v;
      }
      s_h[j] = s;
    }
    tc::pair::cluster_sync_all();  // no CTA leaves while another may read its part
  } else {
    __syncthreads();
    for (int j = threadIdx.x; j < p.rank; j += kTokenThreads) s_h[j] = s_part[j];
    __syncthreads();
  }
  const float w = p.scale != nullptr ? __ldg(p.scale + i) : 1.0f;
  const T* b = static_cast<const T*>(p.b) + (int64_t)i * p.N * p.rank;
  for (int n = n0 + threadIdx.x; n < n1; n += kTokenThreads) {
    const T* row = b + (int64_t)n * p.rank;
    const float base = to_f32(y[n]);
    float s = 0.0f;
    if constexpr (VEC) {
      for (int j = 0; j < p.rank; j += 8) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(row + j));
        const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
        for (int q = 0; q < 8; ++q) s = fmaf(to_f32(e[q]), s_h[j + q], s);
      }
    } else {
      for (int j = 0; j < p.rank; ++j) s = fmaf(to_f32(row[j]), s_h[j], s);
    }
    out[n] = T(fmaf(w, s, base));
  }
}

// ------------------------------------------------------------- tile kernel
constexpr int kRows = 128;         // tokens of a tile
constexpr int kChunk = 64;         // columns of an out chunk
constexpr int kRowThreads = 256;   // two warps for each 32 rows (TMEM lanes): the halves of a chunk
constexpr int kTileThreads = 96 + kRowThreads;  // a warp for the copies, one for the MMAs, the rows' warps, the lists' warp
constexpr int kListWarp = 2 + kRowThreads / 32;
constexpr int kXBytes = kRows * 128;  // 64 columns of X (of K), or of y
constexpr int kPiece = kChunk * 16;   // eight columns of B for a chunk
constexpr int kZeroBytes = kPiece;    // what an odd piece of eight columns is paired with

enum Mode : int { kFused = 0, kHOnly = 1, kOutOnly = 2 };

// Two CTAs fit an SM in each form (the fused one 106 KB, H alone 98 KB, out alone 98 KB).
template <int MODE>
struct Tile {
  static constexpr int kCols = MODE == kFused ? 64 : 128;  // of H: the ranks of a group of adapters
  static constexpr int kStages = MODE == kOutOnly ? 2 : 3;  // ring of X (and A) blocks of 64 columns of K, then of y
  static constexpr int kABytes = MODE == kOutOnly ? 0 : kCols * 128;
  static constexpr int kHBytes = MODE == kHOnly ? 0 : (kCols + 63) / 64 * kXBytes;  // 64-column tiles of 16 KB
  static constexpr int kBBytes = MODE == kHOnly ? 0 : kChunk * kCols * 2;
  static constexpr int kSmem = 1024 + kStages * (kXBytes + kABytes) + kHBytes + 2 * kBBytes + kZeroBytes;
  // TMEM: H, then two out chunks, then the rest of what the H tile holds of h (two columns of H to a 32-bit word)
  static constexpr int kHCols = MODE == kOutOnly ? 0 : kCols;
  static constexpr int kRestAt = kHCols + 2 * kChunk;
  static constexpr int kTmemCols = MODE == kHOnly ? 128 : 256;
};

// K-major operand without swizzle: eight rows of 16 bytes are 128 bytes in a row, groups of eight rows follow each
// other, and the second eight columns of K lie `next` bytes on
__device__ __forceinline__ uint64_t plain_desc(uint32_t saddr, uint32_t next) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(next >> 4) << 16) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}
// the same with rows of 32, 64 or 128 bytes under the swizzle of that width
__device__ __forceinline__ uint64_t swizzled_desc(uint32_t saddr, int row_bytes) {
  const uint64_t layout = row_bytes == 128 ? 2 : row_bytes == 64 ? 4 : 6;
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)1 << 16) | ((uint64_t)(8 * row_bytes >> 4) << 32) |
         ((uint64_t)1 << 46) | (layout << 61);
}
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* tm, int c0, int c1, int c2, uint32_t bar,
                                            uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4, %5}], [%2], %6;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "l"(policy)
      : "memory");
}
__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %6, %7, %8}, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc), "r"(0u), "r"(0u), "r"(0u), "r"(0u));
}

// the same with A in TMEM: sixteen columns of a row are eight 32-bit words of its lane, the lower column in the lower half
__device__ __forceinline__ void umma_f16_from_tmem(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(acc), "r"(0u), "r"(0u), "r"(0u), "r"(0u));
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* w) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(w[0]),
               "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t* w) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
      : "r"(taddr)
      : "memory");
}

// whether all threads of the rows' warps say so; they meet here
__device__ __forceinline__ bool rows_all(bool ok) {
  uint32_t every;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(every)
            : "r"((uint32_t)ok), "n"(kRowThreads)
      : "memory");
  return every != 0;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return pack_bf16x2(lo, hi);
  else return pack_f16x2(lo, hi);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) return make_float2(bf16_lo(w), bf16_hi(w));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// h as the second product takes it: two values of the model type, top = h rounded and rest = what is left, rounded.  Their
// sum is off by 2^-18 of h in bf16 and 2^-22 in fp16 (half a step of a half step), where top alone would be off by 2^-9 and
// 2^-11: a token's result would then depend on whether its batch is taken by tokens or by tiles.
template <typename T>
__device__ __forceinline__ void split2(float a, float b, uint32_t& top, uint32_t& rest) {
  top = pack2<T>(a, b);
  const float2 u = unpack2<T>(top);
  rest = pack2<T>(fabsf(u.x) < INFINITY ? a - u.x : 0.0f, fabsf(u.y) < INFINITY ? b - u.y : 0.0f);
}
// The power of two that brings a row of h, whose largest finite magnitude is `peak`, to [2^14, 2^15): in fp16 h itself may
// be out of the type's range (65504), and its last bits are lost below 2^-14.  `down` takes it back.
__device__ __forceinline__ float row_factor(float peak, float& down) {
  const int up = min(14 - ((int)(__float_as_uint(peak) >> 23) - 127), 100);  // at least -113
  down = __uint_as_float((uint32_t)(127 - up) << 23);
  return __uint_as_float((uint32_t)(127 + up) << 23);
}
__device__ __forceinline__ float finite_max(float peak, float v) { return fabsf(v) < INFINITY ? fmaxf(peak, fabsf(v)) : peak; }

// The tile's product adds the other adapters' columns times zeros, and a zero times an infinity or NaN in one of
// THEIR B's is a NaN.  So where a row's 32 sums are not all finite (`redo`) they are taken again from its own adapter alone (h as
// the H tile and, its rest, TMEM hold it): out = y + w * delta for `n` columns from B row `b`, added to column q by `at`
// (which holds copies: captured by reference, what the rows keep in registers went to memory for it, and 103725 x 512
// took 97 us for 83).  Called by whole warps, whose lanes read their rows of TMEM together.
template <typename T, typename At>
__device__ __noinline__ void add_own(bool redo, const T* b, int n, int rank, const uint8_t* h_tile, uint32_t rest_at, int sixteens,
                                     int r, int e0, float w, At at) {
#pragma unroll 1
  for (int q = 0; q < n; ++q) {
    float s = 0.0f;
#pragma unroll 1
    for (int k = 0; k < sixteens; ++k) {
      uint32_t rest[8];
      __syncwarp();
      tmem_ld8(rest_at + (uint32_t)(8 * k), rest);
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        const int e = 2 * k + d, j = e - e0;
        if (!redo || j < 0 || j >= rank / 8) continue;
        const uint4 h = *reinterpret_cast<const uint4*>(h_tile + (e >> 3) * kXBytes + r * 128 + (((e & 7) ^ (r & 7)) << 4));
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(b + (int64_t)q * rank + 8 * j));
        const uint32_t hw[4] = {h.x, h.y, h.z, h.w}, vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 t = unpack2<T>(hw[i]), u = unpack2<T>(rest[4 * d + i]), f = unpack2<T>(vw[i]);
          s = fmaf(f.x, t.x + u.x, s);
          s = fmaf(f.y, t.y + u.y, s);
        }
      }
    }
    if (redo) at(q, w, s);
  }
}
// whether the first n of 32 are finite: their sum times zero is NaN where one is not (columns beyond N hold anything)
__device__ __forceinline__ bool all_finite(const uint32_t* v, int n) {
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (n >= 32) {
#pragma unroll
    for (int q = 0; q < 32; ++q) s[q & 3] = fmaf(__uint_as_float(v[q]), 0.0f, s[q & 3]);
  } else {
#pragma unroll
    for (int q = 0; q < 32; ++q) s[q & 3] = q < n ? fmaf(__uint_as_float(v[q]), 0.0f, s[q & 3]) : s[q & 3];
  }
  const float all = (s[0] + s[1]) + (s[2] + s[3]);
  return all == all;
}

// sixteen values of a row from column c on (0 beyond N) as they lie in memory, and back
template <typename T>
__device__ __forceinline__ void load16(const T* row, int c, int N, int vec, uint32_t* w) {
  if (c + 16 <= N && vec >= 16) {
    if (vec == 32) {
      asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                   : "l"(row + c));
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(row + c), b = *reinterpret_cast<const uint4*>(row + c + 8);
      w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
      w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
    }
    return;
  }
  const uint16_t* u = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t lo = c + 2 * i < N ? u[c + 2 * i] : 0u, hi = c + 2 * i + 1 < N ? u[c + 2 * i + 1] : 0u;
    w[i] = lo | (hi << 16);
  }
}
template <typename T>
__device__ __forceinline__ void store16(T* row, int c, int N, int vec, const uint32_t* w) {
  if (c + 16 <= N && vec >= 16) {
    if (vec == 32) {
      stg_v8(row + c, w);
    } else {
      *reinterpret_cast<uint4*>(row + c) = make_uint4(w[0], w[1], w[2], w[3]);
      *reinterpret_cast<uint4*>(row + c + 8) = make_uint4(w[4], w[5], w[6], w[7]);
    }
    return;
  }
  uint16_t* u = reinterpret_cast<uint16_t*>(row);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (c + 2 * i < N) u[c + 2 * i] = (uint16_t)w[i];
    if (c + 2 * i + 1 < N) u[c + 2 * i + 1] = (uint16_t)(w[i] >> 16);
  }
}

// A position in a ring of S slots: the slot, and the parity of its use.
template <int S>
struct Turn {
  int slot = 0;
  uint32_t parity = 0;
  __device__ void next() {
    if (++slot == S) {
      slot = 0;
      parity ^= 1;
    }
  }
  __device__ void skip(int n) {
    slot += n;
    parity ^= (uint32_t)(slot / S) & 1u;
    slot %= S;
  }
};

// Asks the hardware for the tile of a CTA that has not started yet (cluster launch control); the 16-byte answer
// lands at `to` and completes 16 bytes on `bar`.
__device__ __forceinline__ void ask_tile(uint32_t to, uint32_t bar) {
  mbar_arrive_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(to), "r"(bar)
               : "memory");
}
// The answer: blockIdx.x of the CTA whose work was taken over, or -1.
__device__ __forceinline__ int told_tile(uint32_t from) {
  uint32_t taken, x;
  asm volatile(
      "{\n\t.reg .b128 r;\n\t.reg .pred p;\n\t"
      "ld.shared.b128 r, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "mov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t}"
      : "=r"(taken), "=r"(x)
      : "r"(from)
      : "memory");
  return taken ? (int)x : -1;
}

// One CTA a tile of 128 tokens (blockIdx.x); blockIdx.y: split of K (H alone) or of N (out alone).  A fused CTA goes on
// with the tiles of CTAs that have not started: while the rows' warps finish a tile, the next one's adapters are listed
// and the ring is filled with its X, and a tile of many adapters (several groups, each with X again) leaves its other
// tiles to the rest.  103725 x 512 took 84 us with a CTA a tile (a quarter of it before its first X block had come) and
// with tiles dealt out beforehand (half of the CTAs ended at 64 us, the last at 91).
template <typename T, int MODE>
__global__ void __launch_bounds__(kTileThreads, 2)
    tile_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmA,
                const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmY,
                const __grid_constant__ CUtensorMap tmO, const __grid_constant__ Params p) {
  using C = Tile<MODE>;
  constexpr int kStages = C::kStages, kABytes = C::kABytes, kBBytes = C::kBBytes;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* sX = smem;
  uint8_t* sA = sX + kStages * kXBytes;
  uint8_t* sH = sA + kStages * kABytes;
  uint8_t* sB = sH + C::kHBytes;
  uint8_t* const s_zero = sB + 2 * kBBytes;
  __shared__ __align__(8) uint64_t full[kStages], empty[kStages], hfull, hready, bfull[2], bempty[2], dfull[2], dempty[2], done;
  __shared__ __align__(8) uint64_t lfull[2], lempty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  __shared__ int s_tile[2], s_count[2], s_list[2][kRows], s_slot[2][kRows];  // of this tile and the next; tile -1: no more
  __shared__ float s_peak[2][MODE == kOutOnly ? kRows : 1];  // of a row's h, by its two warps
  __shared__ __align__(16) uint4 s_told;
  __shared__ __align__(8) uint64_t told;
  volatile int* abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr uint32_t kType = std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
  constexpr uint32_t kIdesc = (1u << 4) | kType | ((uint32_t)(kRows >> 4) << 24);  // N is added where it is known

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    mbar_init(smem_u32(&hfull), 1);
    mbar_init(smem_u32(&hready), kRowThreads);
    for (int s = 0; s < 2; ++s) {
      mbar_init(smem_u32(&bfull[s]), 1);
      mbar_init(smem_u32(&bempty[s]), 1);
      mbar_init(smem_u32(&dfull[s]), 1);
      mbar_init(smem_u32(&dempty[s]), kRowThreads);
      mbar_init(smem_u32(&lfull[s]), 1);
      mbar_init(smem_u32(&lempty[s]), kRowThreads + 2);  // the rows' threads, the copies' and the MMAs'
    }
    mbar_init(smem_u32(&done), 1);
    mbar_init(smem_u32(&told), 1);
    abort_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmX)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmA)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmB)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmY)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmO)) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(C::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == 3) {
    for (int i = lane; i < kZeroBytes / 16; i += 32) reinterpret_cast<uint4*>(s_zero)[i] = make_uint4(0u, 0u, 0u, 0u);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = tmem_slot;
  // The out kernel may start while this one's last CTAs run: it lists its tiles and asks for B and y meanwhile, none
  // of which this kernel writes.  Not before this CTA has its TMEM: the out kernel holds its own while it waits for this one.
  if constexpr (MODE == kHOnly) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int group = C::kCols / p.rank;  // adapters of a group
  const int kblocks = (p.K + 63) / 64;
  const int split = MODE == kFused ? 0 : (int)blockIdx.y;
  const int kb0 = MODE == kHOnly ? (int)((int64_t)kblocks * split / p.splits) : 0;
  const int kb1 = MODE == kHOnly ? (int)((int64_t)kblocks * (split + 1) / p.splits) : kblocks;
  const int all_chunks = (p.N + kChunk - 1) / kChunk;
  const int ch0 = MODE == kOutOnly ? split * p.chunks : 0;
  const int ch1 = MODE == kOutOnly ? min(all_chunks, ch0 + p.chunks) : all_chunks;
  const int eights = p.rank / 8;  // pieces of eight columns of an adapter
  // one group (as a rule): y comes and out goes by whole 64-column chunks through the ring
  auto is_whole = [&](int groups) { return MODE != kHOnly && groups == 1 && p.chunk_io != 0; };

  if (warp == 0) {
    if (lane == 0) {
      // ---------------------------------------------------------- copies
      const uint64_t once = tc::policy_evict_first(), keep = tc::policy_evict_last();
      Turn<kStages> ring;
      Turn<2> bt, lt;
      uint32_t issued = 0, issued_phase = 0;  // bits: ring stages, then the two B buffers
      bool ok = true;
      auto note = [&](int bit, uint32_t parity) {
        issued |= 1u << bit;
        issued_phase = (issued_phase & ~(1u << bit)) | (parity << bit);
      };
      while (ok) {
        if (!mbar_wait_bounded(smem_u32(&lfull[lt.slot]), lt.parity, kWaitTimeoutProducer, abort_flag)) break;
        const int tile = s_tile[lt.slot], row0 = tile * kRows;
        if (tile < 0) break;
        const int* list = s_list[lt.slot];
        const int count = s_count[lt.slot], groups = (count + group - 1) / group;
        const bool whole = is_whole(groups);
        for (int g = 0; g < groups && ok; ++g) {
          const int first = g * group, n = min(group, count - first);
          if constexpr (MODE != kOutOnly) {
            for (int kb = kb0; kb < kb1; ++kb) {
              if (!mbar_wait_bounded(smem_u32(&empty[ring.slot]), ring.parity ^ 1, kWaitTimeoutProducer, abort_flag)) {
                ok = false;
                break;
              }
              const uint32_t fb = smem_u32(&full[ring.slot]);
              mbar_arrive_expect_tx(fb, kXBytes + n * p.rank * 128);
              tc::tma_load_2d(smem_u32(sX + ring.slot * kXBytes), &tmX, kb * 64, row0, fb, groups > 1 ? keep : once);
              for (int j = 0; j < n; ++j)
                tc::tma_load_2d(smem_u32(sA + ring.slot * kABytes + j * p.rank * 128), &tmA, kb * 64, list[first + j] * p.rank, fb, keep);
              note(ring.slot, ring.parity);
              ring.next();
            }
          }
          if constexpr (MODE != kHOnly) {
            for (int ch = ch0; ch < ch1 && ok; ++ch) {
              if (!mbar_wait_bounded(smem_u32(&bempty[bt.slot]), bt.parity ^ 1, kWaitTimeoutProducer, abort_flag)) {
                ok = false;
                break;
              }
              const uint32_t fb = smem_u32(&bfull[bt.slot]);
              const int left = min(kChunk, p.N - ch * kChunk);  // rows of B that the chunk has
              mbar_arrive_expect_tx(fb, p.rank == 8 ? n * left * 16 : n * eights * kPiece);
              for (int j = 0; j < n; ++j) {
                const int row = list[first + j] * p.N + ch * kChunk;
                const uint32_t to = smem_u32(sB + bt.slot * kBBytes + j * eights * kPiece);
                if (p.rank == 8) {  // 16 bytes a row: the chunk's rows lie as the operand wants them
                  bulk_copy(to, static_cast<const T*>(p.b) + (int64_t)row * 8, left * 16, fb);
                } else if (p.unit == 8) {
                  tma_load_3d(to, &tmB, 0, row, 0, fb, keep);
                } else {
                  for (int u = 0; u < p.rank; u += p.unit) tc::tma_load_2d(to + u * kChunk * 2, &tmB, u, row, fb, keep);
                }
              }
              note(kStages + bt.slot, bt.parity);
              bt.next();
              if (!whole) continue;
              if (!mbar_wait_bounded(smem_u32(&empty[ring.slot]), ring.parity ^ 1, kWaitTimeoutProducer, abort_flag)) {
                ok = false;
                break;
              }
              const uint32_t fy = smem_u32(&full[ring.slot]);
              mbar_arrive_expect_tx(fy, kXBytes);
              tc::tma_load_2d(smem_u32(sX + ring.slot * kXBytes), &tmY, ch * kChunk, row0, fy, once);
              note(ring.slot, ring.parity);
              ring.next();
            }
          }
        }
        mbar_arrive(smem_u32(&lempty[lt.slot]));
        lt.next();
      }
      // never leave a copy in flight behind an exiting CTA
      for (int s = 0; s < kStages + 2; ++s)
        if (issued >> s & 1)
          mbar_wait_bounded(smem_u32(s < kStages ? &full[s] : &bfull[s - kStages]), (issued_phase >> s) & 1u,
                            kWaitTimeoutProducer, nullptr);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      // --------------------------------------------------------------- MMA
      Turn<kStages> ring;
      Turn<2> bt, lt;
      uint32_t hparity = 0;
      bool ok = true;
      while (ok) {
        if (!mbar_wait_bounded(smem_u32(&lfull[lt.slot]), lt.parity, kWaitTimeoutMma, abort_flag)) break;
        if (s_tile[lt.slot] < 0) break;
        const int count = s_count[lt.slot], groups = (count + group - 1) / group;
        mbar_arrive(smem_u32(&lempty[lt.slot]));
        lt.next();
        for (int g = 0; g < groups && ok; ++g) {
          const int n = min(group, count - g * group);
          if constexpr (MODE != kOutOnly) {
            const uint32_t idesc = kIdesc | ((uint32_t)((n * eights + 1) & ~1) << 17);  // N in eights, an even number
            for (int kb = kb0; kb < kb1; ++kb) {
              if (!mbar_wait_bounded(smem_u32(&full[ring.slot]), ring.parity, kWaitTimeoutMma, abort_flag)) {
                ok = false;
                break;
              }
              tc::tc_fence_after();
              const uint64_t xd = tc::sw128_desc(smem_u32(sX + ring.slot * kXBytes));
              const uint64_t ad = tc::sw128_desc(smem_u32(sA + ring.slot * kABytes));
#pragma unroll
              for (int s = 0; s < 4; ++s) umma_f16(tmem, xd + 2 * s, ad + 2 * s, idesc, (kb > kb0 || s > 0) ? 1u : 0u);
              tc::umma_commit(smem_u32(&empty[ring.slot]));
              ring.next();
            }
            if (!ok) break;
            tc::umma_commit(smem_u32(&hfull));
          }
          // the rows' warps have H in shared memory (and are done with its TMEM columns)
          if (!mbar_wait_bounded(smem_u32(&hready), hparity, kWaitTimeoutMma, abort_flag)) {
            ok = false;
            break;
          }
          hparity ^= 1;
          if constexpr (MODE != kHOnly) {
            tc::tc_fence_after();
            const uint32_t idesc = kIdesc | ((uint32_t)(kChunk >> 3) << 17);
            const uint64_t hd = tc::sw128_desc(smem_u32(sH));
            for (int ch = ch0; ch < ch1; ++ch) {
              if (!mbar_wait_bounded(smem_u32(&bfull[bt.slot]), bt.parity, kWaitTimeoutMma, abort_flag) ||
                  !mbar_wait_bounded(smem_u32(&dempty[bt.slot]), bt.parity ^ 1, kWaitTimeoutMma, abort_flag)) {
                ok = false;
                break;
              }
              tc::tc_fence_after();
              const uint32_t at_b = smem_u32(sB + bt.slot * kBBytes);
              for (int e = 0; e < n * eights; e += 2) {
                const int at = e >> 1;  // sixteen columns of H: four to a 16 KB tile
                uint64_t bd;
                if (p.unit == 8) {
                  const uint32_t from = at_b + (uint32_t)(e * kPiece);
                  bd = plain_desc(from, e + 1 < n * eights ? (uint32_t)kPiece : smem_u32(s_zero) - from);
                } else {  // a box holds `unit` columns
                  const int in_box = (e * 8) & (p.unit - 1);
                  bd = swizzled_desc(at_b + (uint32_t)((e * 8 - in_box) * kChunk * 2), p.unit * 2) + (uint64_t)(in_box >> 3);
                }
                const uint32_t to = tmem + C::kHCols + bt.slot * kChunk;
                umma_f16(to, hd + (uint64_t)((at >> 2) * (kXBytes >> 4) + 2 * (at & 3)), bd, idesc, e > 0 ? 1u : 0u);
                umma_f16_from_tmem(to, tmem + C::kRestAt + 8 * at, bd, idesc, 1u);
              }
              tc::umma_commit(smem_u32(&bempty[bt.slot]));
              tc::umma_commit(smem_u32(&dfull[bt.slot]));
              bt.next();
            }
          }
        }
        if (MODE == kFused && ok && is_whole(groups)) {
          // y's chunks passed through the ring without this thread.  The rows release the last product only after
          // they have seen the last chunk, so from there on every slot's next use is one of X again; to wait for
          // that earlier could take a use two turns back for it (a barrier tells uses by parity alone).
          const int back = bt.slot ^ 1;
          const uint32_t parity = back == 1 ? bt.parity ^ 1 : bt.parity;
          if (!mbar_wait_bounded(smem_u32(&dempty[back]), parity, kWaitTimeoutMma, abort_flag)) break;
          ring.skip(ch1 - ch0);
        }
      }
      tc::umma_commit(smem_u32(&done));
      mbar_wait_bounded(smem_u32(&done), 0, kWaitTimeoutMma, nullptr);
    }
  } else if (warp == kListWarp) {
    // ------------------------------------------------------- the tiles' adapters
    Turn<2> lt;
    uint32_t answers = 0;
    bool asked = false;
    for (int tile = blockIdx.x;;) {
      if (!__all_sync(kAll, mbar_wait_bounded(smem_u32(&lempty[lt.slot]), lt.parity ^ 1, kWaitTimeoutProducer, abort_flag))) break;
      if (tile < 0) {
        if (lane == 0) {
          s_tile[lt.slot] = -1;
          mbar_arrive(smem_u32(&lfull[lt.slot]));
        }
        break;
      }
      // distinct adapters in the order of their first row, and each row's place among them
      int* list = s_list[lt.slot];
      int id[kRows / 32], count = 0;
#pragma unroll
      for (int c = 0; c < kRows / 32; ++c) id[c] = adapter_of(p, (int64_t)tile * kRows + c * 32 + lane);
#pragma unroll
      for (int c = 0; c < kRows / 32; ++c) {
        const int i = id[c];
        const unsigned peers = __match_any_sync(kAll, i);
        const int leader = __ffs(peers) - 1;
        int at = -1;
        if (i >= 0 && lane == leader)
          for (int q = 0; q < count && at < 0; ++q)
            if (list[q] == i) at = q;
        const unsigned fresh = __ballot_sync(kAll, i >= 0 && lane == leader && at < 0);
        if (fresh >> lane & 1) {
          at = count + __popc(fresh & ((1u << lane) - 1u));
          list[at] = i;
        }
        count += __popc(fresh);
        s_slot[lt.slot][c * 32 + lane] = __shfl_sync(kAll, at, leader);  // -1 for rows without an adapter
        __syncwarp();
      }
      if (lane == 0) {
        s_tile[lt.slot] = tile;
        s_count[lt.slot] = count;
        mbar_arrive(smem_u32(&lfull[lt.slot]));
      }
      const Turn<2> mine = lt;
      lt.next();
      tile = -1;
      if (MODE == kFused) {
        // a tile of several groups takes long: its CTA takes over another one only when it is through.  All of its groups' time
        // (N of millions: seconds), so a wait's usual budget for each; the others' waits are for one step of the work.
        const uint64_t budget = kWaitBudgetNs * (uint64_t)((count + group - 1) / group);
        if (count > group &&
            !__all_sync(kAll, mbar_wait_bounded(smem_u32(&lempty[mine.slot]), mine.parity, kWaitTimeoutProducer, abort_flag, budget)))
          break;
        if (lane == 0) ask_tile(smem_u32(&s_told), smem_u32(&told));
        asked = true;
        if (!__all_sync(kAll, mbar_wait_bounded(smem_u32(&told), answers & 1u, kWaitTimeoutProducer, abort_flag))) break;
        asked = false;
        ++answers;
        tile = told_tile(smem_u32(&s_told));
        __syncwarp();
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the answer was read before the next one may land
      }
    }
    // never leave an answer in flight behind an exiting CTA
    if (asked) mbar_wait_bounded(smem_u32(&told), answers & 1u, kWaitTimeoutProducer, nullptr);
  } else {
    // ----------------------------------------------------------- the rows
    const int quarter = warp & 3;  // the TMEM lanes that this warp can read
    const int half = (warp - 2) >> 2;  // its 32 columns of a chunk, and every other sixteen of H
    const int r = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    Turn<kStages> ring;
    Turn<2> bt, lt;
    uint32_t hparity = 0;
    bool ok = true;
    // all of H's partials are written, and x (which out may overlay) is read, before anything is read or written here
    if constexpr (MODE == kOutOnly) asm volatile("griddepcontrol.wait;" ::: "memory");
    // 16-byte pieces of a row of the H tile are swizzled by the row's place in its eight; eight pieces to 16 KB
    auto piece_at = [&](int e) { return reinterpret_cast<uint4*>(sH + (e >> 3) * kXBytes + r * 128 + (((e & 7) ^ (r & 7)) << 4)); };
    while (true) {
      // the rows' threads leave together, since they count on one another at their barrier
      ok = rows_all(ok && mbar_wait_bounded(smem_u32(&lfull[lt.slot]), lt.parity, kWaitTimeoutEpilogue, abort_flag));
      if (!ok) break;
      const int tile = s_tile[lt.slot];
      if (tile < 0) break;
      const int64_t row = (int64_t)tile * kRows + r;
      const bool live = row < p.T;
      const int count = s_count[lt.slot], groups = (count + group - 1) / group, slot = s_slot[lt.slot][r];
      const int adapter = slot >= 0 ? s_list[lt.slot][slot] : 0;
      const float w = MODE != kHOnly && slot >= 0 && p.scale != nullptr ? __ldg(p.scale + adapter) : 1.0f;
      if (groups <= 1) mbar_arrive(smem_u32(&lempty[lt.slot]));
      const Turn<2> held = lt;
      lt.next();
      const bool whole = is_whole(groups);
      const T* y = static_cast<const T*>(p.y) + row * p.ldy;
      T* out = static_cast<T*>(p.out) + row * p.ldo;
      if (MODE != kHOnly && !whole && live && slot < 0 && out != y) {
        for (int c = ch0 * kChunk + half * 16; c < min(p.N, ch1 * kChunk); c += 32) {
          uint32_t v[8];
          load16(y, c, p.N, p.vec_y, v);
          store16(out, c, p.N, p.vec_out, v);
        }
      }
      // a thread that gave up on a wait still meets the others at a whole chunk's barrier
      for (int g = 0; g < groups && (ok || whole); ++g) {
        const int first = g * group, n = min(group, count - first);
        const int mine = slot >= first && slot < first + n ? slot - first : -1;
        if constexpr (MODE != kOutOnly) {
          // a warp gives up on a wait as one, here and below: its lanes wait for each other before they load from TMEM
          ok = __all_sync(kAll, ok && mbar_wait_bounded(smem_u32(&hfull), hparity, kWaitTimeoutEpilogue, abort_flag));
          tc::tc_fence_after();
          ring.skip(kb1 - kb0);
        }
        hparity ^= 1;
        // own adapter's h into this row of the H tile (and its rest into TMEM), zeros into the others' columns: sixteen
        // columns at a time, whose eights may be of two adapters
        const int e0 = mine * eights;  // its first eight
        float wh = w;  // times what the row's factor left to take back
        if constexpr (MODE == kHOnly) {
          for (int c = half * 16; c < n * p.rank; c += 32) {
            uint32_t v[16];
            __syncwarp();
            tc::swp::tmem_ld16(tmem + lanes + (uint32_t)c, v);
#pragma unroll
            for (int d = 0; d < 2; ++d) {
              const int j = c / 8 + d - e0;
              if (mine < 0 || j < 0 || j >= eights) continue;
              float* to = p.part + ((int64_t)split * p.T + row) * p.rank + 8 * j;
#pragma unroll
              for (int q = 0; q < 8; q += 4)
                *reinterpret_cast<float4*>(to + q) =
                    make_float4(__uint_as_float(v[8 * d + q]), __uint_as_float(v[8 * d + q + 1]),
                                __uint_as_float(v[8 * d + q + 2]), __uint_as_float(v[8 * d + q + 3]));
            }
          }
        } else {
          float factor = 1.0f, down = 1.0f, own[2][16];
          int k0 = 0;  // out alone: own[i] are the sums of the row's sixteen columns k0 + 2 i, where those are its own
          if constexpr (MODE == kOutOnly) {
            // its eights, eight at most and then from a multiple of eight on, lie in two of this warp's sixteens at most
            k0 = e0 >> 1;
            if ((k0 & 1) != half) ++k0;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float* s = own[i];
#pragma unroll
              for (int q = 0; q < 16; ++q) s[q] = 0.0f;
              const int j = 2 * (k0 + 2 * i) - e0;
              const bool in[2] = {mine >= 0 && j >= 0 && j < eights, mine >= 0 && j + 1 >= 0 && j + 1 < eights};
              if (!in[0] && !in[1]) continue;
              const float4* from = reinterpret_cast<const float4*>(p.part + row * p.rank + 8 * j);
              // (by 4 and 8, and one eight at a time by those, 0.1 to 2 us a call more: what they load ahead is spilled)
#pragma unroll 2
              for (int k = 0; k < p.splits; ++k, from += p.T * p.rank / 4) {
#pragma unroll
                for (int f = 0; f < 4; ++f) {
                  if (!in[f >> 1]) continue;
                  const float4 v = __ldcg(from + f);
                  s[4 * f] += v.x;
                  s[4 * f + 1] += v.y;
                  s[4 * f + 2] += v.z;
                  s[4 * f + 3] += v.w;
                }
              }
            }
          }
          if constexpr (std::is_same<T, __half>::value) {
            float peak = 0.0f;
            if constexpr (MODE == kOutOnly) {
#pragma unroll
              for (int q = 0; q < 32; ++q) peak = finite_max(peak, own[q >> 4][q & 15]);
              s_peak[half][r] = peak;  // the row's other columns are the other warp's
              ok = rows_all(ok);
              peak = fmaxf(peak, s_peak[half ^ 1][r]);
            } else {
              for (int c = 0; c < n * p.rank; c += 16) {
                uint32_t v[16];
                __syncwarp();
                tc::swp::tmem_ld16(tmem + lanes + (uint32_t)c, v);
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                  const int j = c / 8 + d - e0;
                  if (mine < 0 || j < 0 || j >= eights) continue;
#pragma unroll
                  for (int q = 0; q < 8; ++q) peak = finite_max(peak, __uint_as_float(v[8 * d + q]));
                }
              }
            }
            factor = row_factor(peak, down);
            wh = w * down;
          }
          auto split16 = [&](const float* v, uint32_t* top, uint32_t* rest) {
#pragma unroll
            for (int q = 0; q < 8; ++q) {
              if constexpr (std::is_same<T, __half>::value) split2<T>(v[2 * q] * factor, v[2 * q + 1] * factor, top[q], rest[q]);
              else split2<T>(v[2 * q], v[2 * q + 1], top[q], rest[q]);
            }
          };
          uint32_t tops[MODE == kOutOnly ? 2 : 1][8], rests[MODE == kOutOnly ? 2 : 1][8];
          if constexpr (MODE == kOutOnly) {
            split16(own[0], tops[0], rests[0]);
            split16(own[1], tops[1], rests[1]);
          }
          for (int c = half * 16; c < n * p.rank; c += 32) {
            const int k = c / 16;
            uint32_t top[8], rest[8];
            if constexpr (MODE == kOutOnly) {
#pragma unroll
              for (int q = 0; q < 8; ++q) {
                top[q] = k == k0 ? tops[0][q] : k == k0 + 2 ? tops[1][q] : 0u;
                rest[q] = k == k0 ? rests[0][q] : k == k0 + 2 ? rests[1][q] : 0u;
              }
            } else {
              uint32_t t[16];
              float v[16];
              __syncwarp();
              tc::swp::tmem_ld16(tmem + lanes + (uint32_t)c, t);
#pragma unroll
              for (int d = 0; d < 2; ++d) {
                const int j = 2 * k + d - e0;
                const bool in = mine >= 0 && j >= 0 && j < eights;
#pragma unroll
                for (int q = 8 * d; q < 8 * d + 8; ++q) v[q] = in ? __uint_as_float(t[q]) : 0.0f;
              }
              split16(v, top, rest);
            }
            *piece_at(2 * k) = make_uint4(top[0], top[1], top[2], top[3]);
            *piece_at(2 * k + 1) = make_uint4(top[4], top[5], top[6], top[7]);
            __syncwarp();
            tmem_st8(tmem + lanes + (uint32_t)(C::kRestAt + 8 * k), rest);
          }
          __syncwarp();
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        }
        tc::tc_fence_before();
        if constexpr (MODE != kHOnly) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(smem_u32(&hready));
        if (whole) {
          for (int ch = ch0; ch < ch1; ++ch) {
            ok = ok && mbar_wait_bounded(smem_u32(&full[ring.slot]), ring.parity, kWaitTimeoutEpilogue, abort_flag) &&
                 mbar_wait_bounded(smem_u32(&dfull[bt.slot]), bt.parity, kWaitTimeoutEpilogue, abort_flag);
            tc::tc_fence_after();
            uint8_t* mem = sX + ring.slot * kXBytes + r * 128;
            const uint32_t sums = tmem + lanes + (uint32_t)(C::kHCols + bt.slot * kChunk + half * 32);
            uint32_t v[32];
            __syncwarp();
            tc::tmem_ld32(sums, v);
            const int n0 = ch * kChunk + half * 32;
            const bool redo = mine >= 0 && ok && !all_finite(v, p.N - n0);
            if (__any_sync(kAll, redo)) {
              add_own<T>(redo, static_cast<const T*>(p.b) + ((int64_t)adapter * p.N + n0) * p.rank, min(32, p.N - n0), p.rank, sH,
                         tmem + lanes + C::kRestAt, (n * eights + 1) / 2, r, e0, wh, [=](int q, float k, float d) {
                           T* to = reinterpret_cast<T*>(mem + (((4 * half + (q >> 3)) ^ (r & 7)) << 4)) + (q & 7);
                           *to = T(fmaf(k, d, to_f32(*to)));
                         });
              __syncwarp();
              tc::tmem_ld32(sums, v);  // of the other rows (kept over the call they would go to memory)
            }
            tc::tc_fence_before();
            mbar_arrive(smem_u32(&dempty[bt.slot]));
            if (mine >= 0 && ok && !redo) {
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                uint4* at = reinterpret_cast<uint4*>(mem + (((4 * half + q) ^ (r & 7)) << 4));
                const uint4 f = *at;
                const uint32_t fw[4] = {f.x, f.y, f.z, f.w};
                uint32_t o[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float2 u = unpack2<T>(fw[i]);
                  o[i] = pack2<T>(fmaf(wh, __uint_as_float(v[8 * q + 2 * i]), u.x), fmaf(wh, __uint_as_float(v[8 * q + 2 * i + 1]), u.y));
                }
                *at = make_uint4(o[0], o[1], o[2], o[3]);
              }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            ok = rows_all(ok);
            if (!ok) break;
            if (threadIdx.x == 64) {
              asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                               reinterpret_cast<uint64_t>(&tmO)),
                           "r"(smem_u32(sX + ring.slot * kXBytes)), "r"(ch * kChunk), "r"(tile * kRows)
                           : "memory");
              asm volatile("cp.async.bulk.commit_group;" ::: "memory");
              // free as soon as it is read: at the ring's two or three stages, leaving that to the next chunk held y's
              // requests back by one (9001 x 1000 to 1544: out alone 35 us)
              asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
              mbar_arrive(smem_u32(&empty[ring.slot]));
            }
            ring.next();
            bt.next();
          }
        } else if constexpr (MODE != kHOnly) {
          for (int ch = ch0; ch < ch1; ++ch) {
            const int c0 = ch * kChunk + half * 32;
            uint32_t base[16];
            if (mine >= 0) {  // requested before the wait for the product
#pragma unroll
              for (int c = 0; c < 32; c += 16)
                if (c0 + c < p.N) load16(y, c0 + c, p.N, p.vec_y, base + c / 2);
            }
            ok = __all_sync(kAll, ok && mbar_wait_bounded(smem_u32(&dfull[bt.slot]), bt.parity, kWaitTimeoutEpilogue, abort_flag));
            if (!ok) break;
            tc::tc_fence_after();
            const uint32_t sums = tmem + lanes + (uint32_t)(C::kHCols + bt.slot * kChunk + half * 32);
            uint32_t v[32];
            __syncwarp();
            tc::tmem_ld32(sums, v);
            const bool redo = mine >= 0 && !all_finite(v, p.N - c0);
            if (__any_sync(kAll, redo)) {
              add_own<T>(redo, static_cast<const T*>(p.b) + ((int64_t)adapter * p.N + c0) * p.rank, min(32, p.N - c0), p.rank, sH,
                         tmem + lanes + C::kRestAt, (n * eights + 1) / 2, r, e0, wh,
                         [=](int q, float k, float d) { out[c0 + q] = T(fmaf(k, d, to_f32(y[c0 + q]))); });
              __syncwarp();
              tc::tmem_ld32(sums, v);
            }
            tc::tc_fence_before();
            mbar_arrive(smem_u32(&dempty[bt.slot]));
            if (mine >= 0 && !redo) {
              uint32_t o[16];
#pragma unroll
              for (int q = 0; q < 16; ++q) {
                const float2 f = unpack2<T>(base[q]);
                o[q] = pack2<T>(fmaf(wh, __uint_as_float(v[2 * q]), f.x), fmaf(wh, __uint_as_float(v[2 * q + 1]), f.y));
              }
#pragma unroll
              for (int c = 0; c < 32; c += 16)
                if (c0 + c < p.N) store16(out, c0 + c, p.N, p.vec_out, o + c / 2);
            }
            bt.next();
          }
          ok = rows_all(ok);  // a row's H is written by two threads: the next group's after both are done with this one's
        }
      }
      if (groups > 1) mbar_arrive(smem_u32(&lempty[held.slot]));
    }
    if (threadIdx.x == 64) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmemCols) : "memory");
  }
}

// ------------------------------------------------------------------- host
// how a call runs: tokens (no tile), one fused kernel, or H and out apart
struct Plan {
  int tiles;   // 0: the token kernel
  int splits;  // 1: fused
  int chunks;  // 64-column chunks of a CTA of the out kernel
};
// Tokens are taken one by one where there are few, or where all of their products are few (T rank (K + N) of 2^24):
// the cost grows with the products, while tiles cost a start, and more for each group of adapters.  Token kernel / tiles
// of one or two adapters / tiles of about 11, in us: 512 to 512, rank 8: 256 tokens 4.3 / 13.1 / 16.2, 1024 tokens 8.4 /
// 13.8 / 16.5; 512 to 1536, rank 16: 256 tokens 7.5 / 14.1 / 22.6, 512 tokens 9.4 / 14.4 / 22.6; 512 to 512, rank 64: 256
// tokens 13.2 / 19.6 / 54.  Above it: 14336 to 512, rank 32: 256 tokens 28 / 32 / 59, 512 tokens 48 / 34 / 60.
constexpr int kTokenMax = 96, kTokenMaxOfFewProducts = 1024;
constexpr int64_t kFewProducts = 1 << 24;

static Plan plan_of(int64_t T, int K, int N, int rank) {
  Plan q{};
  if (T <= kTokenMax || rank % 8 != 0 || rank > 64 || K % 8 != 0) return q;
  if (T <= kTokenMaxOfFewProducts && T * rank * ((int64_t)K + N) <= kFewProducts) return q;
  const int64_t tiles = (T + kRows - 1) / kRows;
  const int sms = sm_count();
  q.tiles = (int)tiles;
  q.splits = 1;
  const int kblocks = (K + 63) / 64, chunks = (N + kChunk - 1) / kChunk;
  q.chunks = chunks;
  // Two CTAs an SM are resident: up to a tile an SM the two phases are spread over them.  Apart / fused, in us, in runs of
  // 100 and of 1 token of 32 adapters: 18000 x 14336 to 512, rank 32: 114 and 820 / 217 and 1780; 18000 x 512 to 1536, rank
  // 16: 42 and 125 / 42 and 241; 18000 x 512 to 512, rank 8: 20.9 and 49 / 18.9 and 63.  Above it fused: two parts a tile
  // gained where most rows of a tile have their own adapter and lost where they share them (60000 x 2048 to 2048, rank 32,
  // runs of 1, 100 and 3000: 1170, 224 and 221 / 1700, 226 and 156).
  if (tiles <= sms) {
    const int64_t want = 2 * sms / tiles;
    q.splits = (int)std::max<int64_t>(1, std::min<int64_t>({want, (int64_t)(kblocks + 3) / 4, 16}));
    // every part sums H's partials again: two chunks at least for each
    const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(want, chunks / 2));
    q.chunks = (int)((chunks + parts - 1) / parts);
    if (q.splits == 1 && q.chunks == chunks) return q;
    if (q.splits == 1) q.splits = -1;  // apart, without a split of K
  }
  return q;
}

// b [R * N, rank].  unit 8: pieces of eight columns, a box holds an adapter's 64 rows piece after piece; else boxes of
// 64 rows and `unit` columns under the swizzle of their width (fewer and wider requests).
static int make_b_map(CUtensorMap* tm, const void* b, int64_t rows, int rank, int unit, CUtensorMapDataType dt) {
  auto enc = tc::encode_fn();
  if (enc == nullptr) return fail(RB_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
  const bool pieces = unit == 8;
  cuuint64_t dims[3] = {pieces ? 8 : (cuuint64_t)rank, (cuuint64_t)rows, (cuuint64_t)(rank / 8)};
  cuuint64_t strides[2] = {(cuuint64_t)rank * 2, 16};
  cuuint32_t box[3] = {(cuuint32_t)unit, kChunk, (cuuint32_t)(rank / 8)};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUtensorMapSwizzle sw = unit == 64   ? CU_TENSOR_MAP_SWIZZLE_128B
                                : unit == 32 ? CU_TENSOR_MAP_SWIZZLE_64B
                                : unit == 16 ? CU_TENSOR_MAP_SWIZZLE_32B
                                             : CU_TENSOR_MAP_SWIZZLE_NONE;
  CUresult r = enc(tm, dt, pieces ? 3 : 2, const_cast<void*>(b), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(RB_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return RB_OK;
}

static int vec_bytes(const void* p, int64_t ld) {
  for (int v : {32, 16})
    if (aligned(p, v) && (ld * 2) % v == 0) return v;
  return 2;
}

template <typename T>
static int run_tokens(const Params& p, bool vec, cudaStream_t st) {
  // CTAs of a token: enough for two an SM, and no more than its adapter's bytes are worth (16 KB each)
  const int64_t bytes = (int64_t)p.rank * (p.K + p.N) * 2;
  int c = 1;
  while (c < 8 && p.T * c < 2 * sm_count() && bytes / (2 * c) >= 16 * 1024) c *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.T * c));
  cfg.blockDim = dim3(kTokenThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)c;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = vec ? cudaLaunchKernelEx(&cfg, token_kernel<T, true>, p) : cudaLaunchKernelEx(&cfg, token_kernel<T, false>, p);
  return check_cuda(e, "low-rank token_kernel launch");
}

template <typename T>
static int run_tiles(Params& p, const Plan& q, CUtensorMapDataType dt, cudaStream_t st) {
  static std::once_flag once[64];
  int dev = 0, rc;
  cudaGetDevice(&dev);
  cudaError_t e = cudaSuccess;
  std::call_once(once[dev & 63], [&] {
    e = cudaFuncSetAttribute(tile_kernel<T, kFused>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile<kFused>::kSmem);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(tile_kernel<T, kHOnly>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile<kHOnly>::kSmem);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(tile_kernel<T, kOutOnly>, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile<kOutOnly>::kSmem);
  });
  if (e != cudaSuccess) return check_cuda(e, "cudaFuncSetAttribute(low-rank tile_kernel)");
  CUtensorMap tmX, tmA, tmB, tmY, tmO;
  if ((rc = tc::make_tmap(&tmX, p.x, p.K, p.T, p.ldx * 2, 64, kRows, dt))) return rc;
  if ((rc = tc::make_tmap(&tmA, p.a, p.K, (int64_t)p.R * p.rank, (int64_t)p.K * 2, 64, (uint32_t)p.rank, dt))) return rc;
  if ((rc = make_b_map(&tmB, p.b, (int64_t)p.R * p.N, p.rank, p.unit, dt))) return rc;
  tmY = tmO = tmX;  // not used where rows do not allow whole chunks
  if (p.chunk_io) {
    if ((rc = tc::make_tmap(&tmY, p.y, p.N, p.T, p.ldy * 2, kChunk, kRows, dt))) return rc;
    if ((rc = tc::make_tmap(&tmO, p.out, p.N, p.T, p.ldo * 2, kChunk, kRows, dt))) return rc;
  }
  if (q.splits == 1) {
    tile_kernel<T, kFused><<<q.tiles, kTileThreads, Tile<kFused>::kSmem, st>>>(tmX, tmA, tmB, tmY, tmO, p);
    return check_cuda(cudaGetLastError(), "low-rank tile_kernel launch");
  }
  p.splits = std::max(1, q.splits);
  p.chunks = q.chunks;
  tile_kernel<T, kHOnly><<<dim3(q.tiles, p.splits), kTileThreads, Tile<kHOnly>::kSmem, st>>>(tmX, tmA, tmB, tmY, tmO, p);
  if ((rc = check_cuda(cudaGetLastError(), "low-rank tile_kernel launch (H)"))) return rc;
  const int parts = ((p.N + kChunk - 1) / kChunk + p.chunks - 1) / p.chunks;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(q.tiles, parts);
  cfg.blockDim = dim3(kTileThreads);
  cfg.dynamicSmemBytes = Tile<kOutOnly>::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, tile_kernel<T, kOutOnly>, tmX, tmA, tmB, tmY, tmO, p),
                    "low-rank tile_kernel launch (out)");
}

}  // namespace lowrank
}  // namespace rb

using namespace rb;

extern "C" int64_t rb_low_rank_workspace_size(int64_t T, int K, int N, int rank) {
  if (T < 0 || K <= 0 || N <= 0 || rank <= 0 || rank > lowrank::kMaxRank || T > 0x7fffffffLL) return -1;
  const lowrank::Plan q = lowrank::plan_of(T, K, N, rank);
  return q.tiles == 0 || q.splits == 1 ? 0 : (int64_t)std::max(1, q.splits) * T * rank * 4;
}

extern "C" int rb_low_rank_add(const void* y, int64_t ldy, const void* x, int64_t ldx, int dtype, int64_t T, int K, int N,
                               const void* a, const void* b, int R, int rank, const void* idx, int idx_dtype,
                               const float* scale, void* workspace, int64_t workspace_bytes, void* out, int64_t ldo,
                               void* stream) {
  using namespace rb::lowrank;
  if (T < 0 || K <= 0 || N <= 0 || R <= 0 || rank <= 0) return fail(RB_ERR_VALUE, "negative or empty adapter shape");
  if (dtype != RB_BF16 && dtype != RB_F16) return fail(RB_ERR_UNSUPPORTED, "rb_low_rank_add takes bf16 or f16");
  if (rank > kMaxRank) return fail(RB_ERR_UNSUPPORTED, "ranks above %d", kMaxRank);
  if (idx_dtype != RB_I64 && idx_dtype != RB_I32) return fail(RB_ERR_VALUE, "adapter ids must be int64 or int32");
  if (T > 0x7fffffffLL / 8 || (int64_t)R * N > 0x7fffffffLL || (int64_t)R * rank > 0x7fffffffLL)
    return fail(RB_ERR_UNSUPPORTED, "more than 2^28 tokens, or than 2^31 rows of all adapters");
  if (ldy < N || ldo < N || ldx < K) return fail(RB_ERR_VALUE, "leading dimension smaller than the row");
  if (T > 0 && (y == nullptr || x == nullptr || a == nullptr || b == nullptr || idx == nullptr || out == nullptr))
    return fail(RB_ERR_VALUE, "null operand");
  Plan q = plan_of(T, K, N, rank);
  const bool fit = aligned(x, 16) && (ldx * 2) % 16 == 0 && aligned(a, 16) && aligned(b, 16) && K % 8 == 0 && rank % 8 == 0;
  if (!fit) q.tiles = 0;
  const int64_t need = q.tiles == 0 ? 0 : rb_low_rank_workspace_size(T, K, N, rank);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(RB_ERR_VALUE, "workspace of %lld bytes (16-byte aligned) needed, %lld given", (long long)need,
                (long long)workspace_bytes);
  if (!device_is_sm100()) return fail(RB_ERR_DEVICE, "rb_low_rank_add needs an sm_100 (B200) device");
  if (T == 0) return RB_OK;
  Params p{};
  p.y = y;
  p.x = x;
  p.a = a;
  p.b = b;
  p.idx = idx;
  p.scale = scale;
  p.out = out;
  p.part = static_cast<float*>(workspace);
  p.ldy = ldy;
  p.ldx = ldx;
  p.ldo = ldo;
  p.T = T;
  p.K = K;
  p.N = N;
  p.R = R;
  p.rank = rank;
  p.idx64 = idx_dtype == RB_I64;
  p.splits = 1;
  p.unit = rank % 64 == 0 ? 64 : rank % 32 == 0 ? 32 : rank % 16 == 0 ? 16 : 8;
  p.vec_y = vec_bytes(y, ldy);
  p.vec_out = vec_bytes(out, ldo);
  // (a chunk's store goes by whole 16 bytes: with N off 8 it would write up to seven columns behind a row)
  p.chunk_io = p.vec_y >= 16 && p.vec_out >= 16 && N % 8 == 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (q.tiles == 0)
    return dtype == RB_BF16 ? run_tokens<__nv_bfloat16>(p, fit, st) : run_tokens<__half>(p, fit, st);
  return dtype == RB_BF16 ? run_tiles<__nv_bfloat16>(p, q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, st)
                          : run_tiles<__half>(p, q, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, st);
}

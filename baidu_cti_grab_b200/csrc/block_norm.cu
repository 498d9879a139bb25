// block_norm.cu -- what stands between two blocks of an encoder: the norm after a
// block, its gate and residual scale, and the norm before the next block, with the
// gradients of all of them.  Per row of D values, in fp32:
//
//   n = post(h)   y = x + scale * act(g) * n   z = pre(y)
//
// post and pre are LayerNorm, RMS norm or nothing; g is one gate per channel, per
// row or per element.  With t = dL/dy (everything that reaches y):
//
//   t = dy + pre'(dz)   dx = t   dn = scale act(g) t   dg = scale n t act'(g)   dh = post'(dn)
//   norm'(d) = r (d w - mean(d w [layer only]) - v^ mean(d w v^)),  v^ the normalised values
//   dw = sum over rows of d v^,  db = sum over rows of d
//
// What bounds it: HBM.  Forward reads x, h and writes y, z; backward reads x, h, dy,
// dz, recomputes n and y from the saved means and deviations (reading x costs what
// reading y would, and y is then not rounded) and writes dx, dh.  So:
//   * a team of threads holds a row in registers, each value is read once;
//   * rows come by bulk copies into a ring in shared memory, several rows ahead of
//     the work, which no register has to hold;
//   * the grid is persistent: in backward each thread keeps its columns' sums of the
//     weights' gradients over all of its team's rows; teams and then CTAs are summed
//     in a fixed order (no atomics: the same bits every time).
// A team is a warp for narrow rows (no barrier but the warp's own), a CTA for wide.
#include "common.cuh"

#include <algorithm>
#include <mutex>

namespace rb {
namespace bnorm {

constexpr unsigned kAll = 0xffffffffu;
constexpr int kMaxWidth = 8192;
constexpr int kMaxStages = 4;
enum Kind : int { kNone = RB_NORM_NONE, kLayer = RB_NORM_LAYER, kRms = RB_NORM_RMS };
enum Gate : int { kGateNone = RB_GATE_NONE, kGateChannel = RB_GATE_CHANNEL, kGateRow = RB_GATE_ROW, kGateFull = RB_GATE_FULL };
enum Act : int { kActNone = RB_GATE_ACT_NONE, kActSigmoid = RB_GATE_ACT_SIGMOID };
constexpr int kSums = 5;  // column sums of backward: dw_post, db_post, dw_pre, db_pre, dgate

struct Params {
  const void *x, *h, *gate, *dy, *dz;     // rows (dy, dz: backward only; each may be null)
  const void *w1, *b1, *w2, *b2;          // post and pre affine, or null
  void *out0, *out1, *out2;               // y, z | dx, dh, dgate (rows or elements)
  float* stats;                           // [N, 4]: post mean, 1/deviation, pre mean, 1/deviation
  float* partial;                         // backward: [CTAs][kSums][D]
  int64_t N, ldx, ldh, ldg, ldy, ldz;
  float eps1, eps2, scale;
  int D, post, pre, gate_kind, act, w1_dtype, w2_dtype, gate_dtype;
  int bulk, stages, row_bytes, need_sums;
};

// eight values as they lie in memory
template <typename T>
struct Eight {
  uint4 q[sizeof(T) / 2];
};
__device__ __forceinline__ void widen(const Eight<__nv_bfloat16>& e, float* v) {
  const uint32_t w[4] = {e.q[0].x, e.q[0].y, e.q[0].z, e.q[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = bf16_lo(w[i]);
    v[2 * i + 1] = bf16_hi(w[i]);
  }
}
__device__ __forceinline__ void widen(const Eight<__half>& e, float* v) {
  const uint32_t w[4] = {e.q[0].x, e.q[0].y, e.q[0].z, e.q[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void widen(const Eight<float>& e, float* v) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    v[4 * i] = __uint_as_float(e.q[i].x);
    v[4 * i + 1] = __uint_as_float(e.q[i].y);
    v[4 * i + 2] = __uint_as_float(e.q[i].z);
    v[4 * i + 3] = __uint_as_float(e.q[i].w);
  }
}
__device__ __forceinline__ void narrow(const float* v, Eight<__nv_bfloat16>& e) {
  e.q[0] = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
__device__ __forceinline__ void narrow(const float* v, Eight<__half>& e) {
  e.q[0] = make_uint4(pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]), pack_f16x2(v[4], v[5]), pack_f16x2(v[6], v[7]));
}
__device__ __forceinline__ void narrow(const float* v, Eight<float>& e) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
    e.q[i] = make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]),
                        __float_as_uint(v[4 * i + 3]));
}

// eight parameters from column c (0 beyond D), or `none` where there are none
__device__ __forceinline__ void param8(const void* p, int dtype, int c, int D, float none, float* v) {
  if (p == nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = none;
    return;
  }
  const int size = dtype == RB_F32 ? 4 : 2;
  const char* at = static_cast<const char*>(p) + (int64_t)c * size;
  if (c + 8 <= D && (reinterpret_cast<uintptr_t>(at) & 15) == 0) {
    if (dtype == RB_F32) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(at)), b = __ldg(reinterpret_cast<const float4*>(at) + 1);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else if (dtype == RB_BF16) {
      Eight<__nv_bfloat16> e;
      e.q[0] = __ldg(reinterpret_cast<const uint4*>(at));
      widen(e, v);
    } else {
      Eight<__half> e;
      e.q[0] = __ldg(reinterpret_cast<const uint4*>(at));
      widen(e, v);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = c + i < D ? load_as_f32(p, dtype, c + i) : 0.0f;
}

__device__ __forceinline__ float gate_act(float g, int act) {
  return act == kActSigmoid ? __fdividef(1.0f, 1.0f + expf(-g)) : g;
}

// A team of G threads on a row of up to 8 V G values; thread r of the team holds the eights r, r + G, ...
template <int G>
struct Team {
  static constexpr int kTeams = G == 32 ? 8 : 1;  // teams of a CTA
  static constexpr int kThreads = G * kTeams;
  static constexpr int kWarps = kThreads / 32;
  __device__ static int index() { return G == 32 ? (int)(threadIdx.x >> 5) : 0; }
  __device__ static int rank() { return G == 32 ? (int)(threadIdx.x & 31) : (int)threadIdx.x; }
  __device__ static void sync() {
    if constexpr (G == 32) __syncwarp();
    else __syncthreads();
  }
  __device__ static bool all(bool ok) {
    if constexpr (G == 32) return __all_sync(kAll, ok);
    else return __syncthreads_and(ok) != 0;
  }
  // sums of M values over the team; `room` holds 2 * kWarps * 4 floats, used in turns
  template <int M>
  __device__ static void sum(float (&v)[M], float* room, int& turn) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int m = 0; m < M; ++m) v[m] += __shfl_xor_sync(kAll, v[m], o);
    if constexpr (G > 32) {
      float* at = room + turn * kWarps * 4;
      turn ^= 1;  // the next sum writes the other half, so one barrier per sum is enough
      if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int m = 0; m < M; ++m) at[(threadIdx.x >> 5) * 4 + m] = v[m];
      __syncthreads();
      const int lane = threadIdx.x & 31;
#pragma unroll
      for (int m = 0; m < M; ++m) v[m] = lane < kWarps ? at[lane * 4 + m] : 0.0f;
#pragma unroll
      for (int o = kWarps / 2; o > 0; o >>= 1)
#pragma unroll
        for (int m = 0; m < M; ++m) v[m] += __shfl_xor_sync(kAll, v[m], o);
#pragma unroll
      for (int m = 0; m < M; ++m) v[m] = __shfl_sync(kAll, v[m], 0);
    }
  }
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// The rows of a team's turn it: row = first + it * step.  `src` are the arrays that a row is read from.
template <typename T, int G, int V, int A>
struct Rows {
  const char* src[A];
  int64_t pitch[A];  // bytes
  uint8_t* ring;     // this team's stages
  uint64_t* full;    // this team's barriers
  volatile int* abort_flag;
  int64_t first, step, N;
  int D, stages, row_bytes, bulk;

  __device__ uint8_t* slot(int stage, int a) const { return ring + ((int64_t)stage * A + a) * row_bytes; }
  __device__ void request(int stage, int64_t row) const {  // one thread
    const uint32_t bytes = (uint32_t)(D * (int)sizeof(T));
    uint32_t n = 0;
#pragma unroll
    for (int a = 0; a < A; ++a) n += src[a] != nullptr ? bytes : 0u;
    const uint32_t bar = smem_u32(full + stage);
    mbar_arrive_expect_tx(bar, n);
#pragma unroll
    for (int a = 0; a < A; ++a)
      if (src[a] != nullptr) bulk_load(smem_u32(slot(stage, a)), src[a] + row * pitch[a], bytes, bar);
  }
  __device__ void start() const {
    if (bulk && Team<G>::rank() == 0)
      for (int s = 0; s < stages; ++s)
        if (first + s * step < N) request(s, first + s * step);
  }
  // Row `row`'s eights (zeros beyond D and for absent arrays) into registers; asks for the row `stages` turns on.
  __device__ bool take(int64_t row, int stage, uint32_t phase, Eight<T> (&e)[A][V]) const {
    const int r = Team<G>::rank();
    bool ok = true;
    if (bulk) {
      ok = mbar_wait_bounded(smem_u32(full + stage), phase, kWaitTimeoutProducer, abort_flag);
    } else {
      // rows that no 16-byte copy can fetch: value by value, neighbours by neighbouring threads
#pragma unroll
      for (int a = 0; a < A; ++a) {
        if (src[a] == nullptr) continue;
        const T* from = reinterpret_cast<const T*>(src[a] + row * pitch[a]);
        T* to = reinterpret_cast<T*>(slot(stage, a));
        for (int c = r; c < D; c += G) to[c] = from[c];
      }
      Team<G>::sync();
    }
#pragma unroll
    for (int a = 0; a < A; ++a)
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int c = (v * G + r) * 8;
#pragma unroll
        for (int q = 0; q < (int)(sizeof(T) / 2); ++q) {
          e[a][v].q[q] = make_uint4(0u, 0u, 0u, 0u);
          if (ok && src[a] != nullptr && c < D)
            e[a][v].q[q] = reinterpret_cast<const uint4*>(slot(stage, a) + (int64_t)c * sizeof(T))[q];
        }
        if (c < D && c + 8 > D) {  // a row's last eight may be short
          T* t = reinterpret_cast<T*>(&e[a][v]);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c + i >= D) t[i] = T(0.0f);
        }
      }
    ok = Team<G>::all(ok);
    const int64_t next = row + stages * step;
    if (bulk && ok && next < N && r == 0) {
      // the slot was read through the generic proxy: order those reads before the copy's writes
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      request(stage, next);
    }
    return ok;
  }
  // After a wait that gave up at (row, stage, phase): the copies still in flight land before this CTA leaves.
  __device__ void drain(int64_t row, int stage, uint32_t phase) const {
    if (!bulk || Team<G>::rank() != 0) return;
    for (int s = 0; s < stages && row < N; ++s, row += step) {
      mbar_wait_bounded(smem_u32(full + stage), phase, kWaitTimeoutProducer, nullptr);
      if (++stage == stages) {
        stage = 0;
        phase ^= 1;
      }
    }
  }
  // A row out: straight from registers, or (rows that 16-byte stores do not fit) through this stage's slot a
  __device__ void put(void* out, int64_t row, int stage, int a, const float (&v)[V * 8]) const {
    const int r = Team<G>::rank();
    T* to = static_cast<T*>(out) + row * D;
    if (bulk) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const int c = (k * G + r) * 8;
        if (c >= D) continue;
        Eight<T> e;
        narrow(v + 8 * k, e);
#pragma unroll
        for (int q = 0; q < (int)(sizeof(T) / 2); ++q) reinterpret_cast<uint4*>(to + c)[q] = e.q[q];
      }
      return;
    }
    T* via = reinterpret_cast<T*>(slot(stage, a));
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = (k * G + r) * 8;
      if (c >= D) continue;
      Eight<T> e;
      narrow(v + 8 * k, e);
#pragma unroll
      for (int q = 0; q < (int)(sizeof(T) / 2); ++q) reinterpret_cast<uint4*>(via + c)[q] = e.q[q];
    }
    Team<G>::sync();
    for (int c = r; c < D; c += G) to[c] = via[c];
    Team<G>::sync();
  }
};

// v centred and normalised in place over the team's row; mean and 1 / deviation
template <int G, int V>
__device__ __forceinline__ void normalise(float (&v)[V * 8], int kind, float eps, int D, float* room, int& turn,
                                          float& mean, float& rstd) {
  const int r = Team<G>::rank();
  const float inv = 1.0f / (float)D;
  mean = 0.0f;
  if (kind == kLayer) {
    float s[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < V * 8; ++i) s[0] += v[i];
    Team<G>::sum(s, room, turn);
    mean = s[0] * inv;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = (k * G + r) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[8 * k + i] = c + i < D ? v[8 * k + i] - mean : 0.0f;
    }
  }
  float s[1] = {0.0f};
#pragma unroll
  for (int i = 0; i < V * 8; ++i) s[0] = fmaf(v[i], v[i], s[0]);
  Team<G>::sum(s, room, turn);
  rstd = rsqrtf(fmaf(s[0], inv, eps));
#pragma unroll
  for (int i = 0; i < V * 8; ++i) v[i] *= rstd;
}

template <int G>
__device__ __forceinline__ void init_ring(uint64_t* full, int stages, volatile int* abort_flag) {
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < stages * Team<G>::kTeams; ++s) mbar_init(smem_u32(full + s), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncthreads();
}

template <typename T, int G, int V>
__global__ void __launch_bounds__(Team<G>::kThreads) sandwich_kernel(const __grid_constant__ Params p) {
  using Tm = Team<G>;
  constexpr int kArrays = 3;  // x, h, a gate of every element
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ __align__(8) uint64_t full[kMaxStages * Tm::kTeams];
  __shared__ float room[2 * Tm::kWarps * 4];
  __shared__ int abort_flag;
  init_ring<G>(full, p.stages, &abort_flag);
  const int r = Tm::rank();
  Rows<T, G, V, kArrays> rows;
  rows.src[0] = static_cast<const char*>(p.x);
  rows.src[1] = static_cast<const char*>(p.h);
  rows.src[2] = p.gate_kind == kGateFull ? static_cast<const char*>(p.gate) : nullptr;
  rows.pitch[0] = p.ldx * (int64_t)sizeof(T);
  rows.pitch[1] = p.ldh * (int64_t)sizeof(T);
  rows.pitch[2] = p.ldg * (int64_t)sizeof(T);
  rows.ring = ring + (int64_t)Tm::index() * p.stages * kArrays * p.row_bytes;
  rows.full = full + Tm::index() * p.stages;
  rows.abort_flag = &abort_flag;
  rows.first = (int64_t)blockIdx.x * Tm::kTeams + Tm::index();
  rows.step = (int64_t)gridDim.x * Tm::kTeams;
  rows.N = p.N;
  rows.D = p.D;
  rows.stages = p.stages;
  rows.row_bytes = p.row_bytes;
  rows.bulk = p.bulk;
  rows.start();

  int stage = 0, turn = 0;
  uint32_t phase = 0;
  float next_gate = 1.0f;
  auto ahead = [&](int64_t row) {
    if (p.gate_kind == kGateRow && row < p.N)
      next_gate = gate_act(load_as_f32(p.gate, p.gate_dtype, row * p.ldg), p.act);
  };
  ahead(rows.first);
  for (int64_t row = rows.first; row < p.N; row += rows.step) {
    Eight<T> e[kArrays][V];
    if (!rows.take(row, stage, phase, e)) {
      rows.drain(row, stage, phase);
      break;
    }
    const float row_gate = next_gate;
    ahead(row + rows.step);
    float n[V * 8], y[V * 8];
    float mean1 = 0.0f, rstd1 = 1.0f, mean2 = 0.0f, rstd2 = 1.0f;
#pragma unroll
    for (int k = 0; k < V; ++k) widen(e[1][k], n + 8 * k);
    if (p.post != kNone) normalise<G, V>(n, p.post, p.eps1, p.D, room, turn, mean1, rstd1);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = (k * G + r) * 8;
      float* nk = n + 8 * k;
      if (p.post != kNone) {
        float w[8], b[8];
        param8(p.w1, p.w1_dtype, c, p.D, 1.0f, w);
        param8(p.b1, p.w1_dtype, c, p.D, 0.0f, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) nk[i] = fmaf(nk[i], w[i], b[i]);
      }
      if (p.gate_kind == kGateChannel || p.gate_kind == kGateFull) {
        float g[8];
        if (p.gate_kind == kGateFull) widen(e[2][k], g);
        else param8(p.gate, p.gate_dtype, c, p.D, 1.0f, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) nk[i] *= gate_act(g[i], p.act);
      }
      widen(e[0][k], y + 8 * k);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[8 * k + i] = c + i < p.D ? fmaf(p.scale * row_gate, nk[i], y[8 * k + i]) : 0.0f;
    }
    rows.put(p.out0, row, stage, 0, y);
    if (p.pre != kNone) {
      normalise<G, V>(y, p.pre, p.eps2, p.D, room, turn, mean2, rstd2);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const int c = (k * G + r) * 8;
        float w[8], b[8];
        param8(p.w2, p.w2_dtype, c, p.D, 1.0f, w);
        param8(p.b2, p.w2_dtype, c, p.D, 0.0f, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[8 * k + i] = fmaf(y[8 * k + i], w[i], b[i]);
      }
      rows.put(p.out1, row, stage, 0, y);
    }
    if (p.stats != nullptr && r == 0)
      reinterpret_cast<float4*>(p.stats)[row] = make_float4(mean1, rstd1, mean2, rstd2);
    if (++stage == p.stages) {
      stage = 0;
      phase ^= 1;
    }
  }
}

// LEAN: no biases and no gate per channel, so two of the five column sums.
template <typename T, int G, int V, bool LEAN>
__global__ void __launch_bounds__(Team<G>::kThreads) sandwich_backward_kernel(const __grid_constant__ Params p) {
  using Tm = Team<G>;
  constexpr int kArrays = 5;  // x, h, dy, dz, a gate of every element
  constexpr int NV = V * 8;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ __align__(8) uint64_t full[kMaxStages * Tm::kTeams];
  __shared__ float room[2 * Tm::kWarps * 4];
  __shared__ int abort_flag;
  init_ring<G>(full, p.stages, &abort_flag);
  const int r = Tm::rank();
  Rows<T, G, V, kArrays> rows;
  rows.src[0] = static_cast<const char*>(p.x);
  rows.src[1] = static_cast<const char*>(p.h);
  rows.src[2] = static_cast<const char*>(p.dy);
  rows.src[3] = static_cast<const char*>(p.dz);
  rows.src[4] = p.gate_kind == kGateFull ? static_cast<const char*>(p.gate) : nullptr;
  rows.pitch[0] = p.ldx * (int64_t)sizeof(T);
  rows.pitch[1] = p.ldh * (int64_t)sizeof(T);
  rows.pitch[2] = p.ldy * (int64_t)sizeof(T);
  rows.pitch[3] = p.ldz * (int64_t)sizeof(T);
  rows.pitch[4] = p.ldg * (int64_t)sizeof(T);
  rows.ring = ring + (int64_t)Tm::index() * p.stages * kArrays * p.row_bytes;
  rows.full = full + Tm::index() * p.stages;
  rows.abort_flag = &abort_flag;
  rows.first = (int64_t)blockIdx.x * Tm::kTeams + Tm::index();
  rows.step = (int64_t)gridDim.x * Tm::kTeams;
  rows.N = p.N;
  rows.D = p.D;
  rows.stages = p.stages;
  rows.row_bytes = p.row_bytes;
  rows.bulk = p.bulk;
  rows.start();

  constexpr int kHeld = LEAN ? 2 : kSums;
  float acc[kHeld][NV];  // dw_post, dw_pre, then db_post, db_pre, dgate
#pragma unroll
  for (int a = 0; a < kHeld; ++a)
#pragma unroll
    for (int i = 0; i < NV; ++i) acc[a][i] = 0.0f;

  const float inv = 1.0f / (float)p.D;
  int stage = 0, turn = 0;
  uint32_t phase = 0;
  float4 st = make_float4(0.0f, 1.0f, 0.0f, 1.0f);
  float g_row = 1.0f;
  auto ahead = [&](int64_t row) {  // the next row's scalars
    if (row < p.N) {
      st = __ldg(reinterpret_cast<const float4*>(p.stats) + row);
      if (p.gate_kind == kGateRow) g_row = load_as_f32(p.gate, p.gate_dtype, row * p.ldg);
    }
  };
  ahead(rows.first);
  for (int64_t row = rows.first; row < p.N; row += rows.step) {
    const float4 s = st;
    const float gr = g_row;
    Eight<T> e[kArrays][V];
    if (!rows.take(row, stage, phase, e)) {
      rows.drain(row, stage, phase);
      break;
    }
    ahead(row + rows.step);
    const float a_row = gate_act(gr, p.gate_kind == kGateRow ? p.act : (int)kActNone);
    float hh[NV], yh[NV], t[NV];
    float s12[2] = {0.0f, 0.0f};
    // n and y again; the pre norm's two sums
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = (k * G + r) * 8;
      float w[8], b[8], g[8], x[8], dz[8], w2[8];
      widen(e[1][k], hh + 8 * k);
      widen(e[0][k], x);
      widen(e[3][k], dz);
      if (p.pre != kNone) {
        param8(p.w1, p.w1_dtype, c, p.D, 1.0f, w);
        param8(p.b1, p.w1_dtype, c, p.D, 0.0f, b);
        param8(p.w2, p.w2_dtype, c, p.D, 1.0f, w2);
        if (p.gate_kind == kGateFull) widen(e[4][k], g);
        else if (p.gate_kind == kGateChannel) param8(p.gate, p.gate_dtype, c, p.D, 1.0f, g);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool in = c + i < p.D;
        const float q = in ? (hh[8 * k + i] - s.x) * s.y : 0.0f;
        hh[8 * k + i] = q;
        t[8 * k + i] = 0.0f;
        if (p.pre != kNone) {
          float a = a_row;
          if (p.gate_kind == kGateFull || p.gate_kind == kGateChannel) a = gate_act(g[i], p.act);
          const float y = fmaf(p.scale * a, fmaf(q, w[i], b[i]), x[i]);
          const float f = in ? (y - s.z) * s.w : 0.0f;
          yh[8 * k + i] = f;
          const float u = dz[i] * w2[i];
          t[8 * k + i] = u;
          s12[0] += u;
          s12[1] = fmaf(u, f, s12[1]);
          acc[1][8 * k + i] = fmaf(dz[i], f, acc[1][8 * k + i]);
          if constexpr (!LEAN) acc[3][8 * k + i] += dz[i];
        }
      }
    }
    if (p.pre != kNone) {
      Tm::sum(s12, room, turn);
      if (p.pre == kRms) s12[0] = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i) t[i] = s.w * (t[i] - s12[0] * inv - yh[i] * (s12[1] * inv));
    }
    // t reaches y; its way into h, the gate and the post norm's weights
    float s34[3] = {0.0f, 0.0f, 0.0f};
    float out[NV];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = (k * G + r) * 8;
      float w[8], b[8], g[8], dy[8];
      widen(e[2][k], dy);
      param8(p.w1, p.w1_dtype, c, p.D, 1.0f, w);
      param8(p.b1, p.w1_dtype, c, p.D, 0.0f, b);
      if (p.gate_kind == kGateFull) widen(e[4][k], g);
      else if (p.gate_kind == kGateChannel) param8(p.gate, p.gate_dtype, c, p.D, 1.0f, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = 8 * k + i;
        const bool in = c + i < p.D;
        const float tt = in ? t[j] + dy[i] : 0.0f;
        t[j] = tt;
        float a = a_row;
        if (p.gate_kind == kGateFull || p.gate_kind == kGateChannel) a = gate_act(g[i], p.act);
        const float dn = p.scale * a * tt;
        float da = p.scale * fmaf(hh[j], w[i], b[i]) * tt;
        if (p.act == kActSigmoid) da *= a * (1.0f - a);
        yh[j] = da;  // a gate of every element: its gradient
        s34[2] += da;
        if constexpr (!LEAN) {
          acc[2][j] += dn;
          acc[4][j] += da;
        }
        acc[0][j] = fmaf(dn, hh[j], acc[0][j]);
        const float v = dn * w[i];
        out[j] = v;
        s34[0] += v;
        s34[1] = fmaf(v, hh[j], s34[1]);
      }
    }
    rows.put(p.out0, row, stage, 0, t);
    if (p.gate_kind == kGateFull) rows.put(p.out2, row, stage, 0, yh);
    if (p.post != kNone || p.gate_kind == kGateRow) Tm::sum(s34, room, turn);
    if (p.gate_kind == kGateRow && r == 0) {
      if (p.gate_dtype == RB_F32) static_cast<float*>(p.out2)[row] = s34[2];
      else if (p.gate_dtype == RB_BF16) static_cast<__nv_bfloat16*>(p.out2)[row] = __float2bfloat16_rn(s34[2]);
      else static_cast<__half*>(p.out2)[row] = __float2half_rn(s34[2]);
    }
    if (p.post != kNone) {
      if (p.post == kRms) s34[0] = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i) out[i] = s.y * (out[i] - s34[0] * inv - hh[i] * (s34[1] * inv));
    }
    rows.put(p.out1, row, stage, 0, out);
    if (++stage == p.stages) {
      stage = 0;
      phase ^= 1;
    }
  }

  if (!p.need_sums) return;
  // the CTA's sums: its teams one after another through shared memory, then this CTA's row of `partial`
  constexpr int kPlace[kSums] = {0, 2, 1, 3, 4};  // acc index -> dw_post, db_post, dw_pre, db_pre, dgate
  if constexpr (Tm::kTeams == 1) {
#pragma unroll
    for (int a = 0; a < kHeld; ++a)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const int c = (k * G + r) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c + i < p.D) p.partial[((int64_t)blockIdx.x * kSums + kPlace[a]) * p.D + c + i] = acc[a][8 * k + i];
      }
  } else {
    __syncthreads();  // every team is done with the ring
    float* sums = reinterpret_cast<float*>(ring);
    for (int w = 0; w < Tm::kTeams; ++w) {
      if (Tm::index() == w) {
#pragma unroll
        for (int a = 0; a < kHeld; ++a)
#pragma unroll
          for (int k = 0; k < V; ++k) {
            const int c = (k * G + r) * 8;
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (c + i < p.D) {
                float* at = sums + a * p.D + c + i;
                *at = (w == 0 ? 0.0f : *at) + acc[a][8 * k + i];
              }
          }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < kHeld * p.D; c += Tm::kThreads) {
      const int a = c / p.D;
      p.partial[((int64_t)blockIdx.x * kSums + kPlace[a]) * p.D + (c - a * p.D)] = sums[c];
    }
  }
}

struct SumOut {
  void* out[kSums];
  int dtype[kSums];
};

// out[s][c] = the sum of partial[cta][s][c] over the CTAs, in a fixed order: 32 columns a block, the CTAs in
// eight runs
__global__ void __launch_bounds__(256) column_sums_kernel(const float* __restrict__ partial, int ctas, int D,
                                                          const __grid_constant__ SumOut o) {
  __shared__ float part[8][32];
  const int s = blockIdx.y;
  if (o.out[s] == nullptr) return;
  const int lane = threadIdx.x & 31, run = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float v = 0.0f;
  if (c < D) {
#pragma unroll 8
    for (int b = run; b < ctas; b += 8) v += partial[((int64_t)b * kSums + s) * D + c];
  }
  part[run][lane] = v;
  __syncthreads();
  if (run == 0 && c < D) {
#pragma unroll
    for (int k = 1; k < 8; ++k) v += part[k][lane];
    if (o.dtype[s] == RB_F32) static_cast<float*>(o.out[s])[c] = v;
    else if (o.dtype[s] == RB_BF16) static_cast<__nv_bfloat16*>(o.out[s])[c] = __float2bfloat16_rn(v);
    else static_cast<__half*>(o.out[s])[c] = __float2half_rn(v);
  }
}

// ------------------------------------------------------------------- host
struct Shape {
  int threads, teams, stages, row_bytes, smem, per_sm;
};

// team and ring of a width: as many stages (up to kMaxStages) as fit `budget` bytes of a CTA's shared memory
static Shape shape_of(int team, int arrays, int D, int elt, int budget, int per_sm) {
  Shape s{};
  s.teams = team == 32 ? 8 : 1;
  s.threads = team * s.teams;
  s.row_bytes = (D * elt + 15) / 16 * 16;
  const int64_t stage = (int64_t)s.teams * arrays * s.row_bytes;
  s.stages = (int)std::max<int64_t>(1, std::min<int64_t>(kMaxStages, budget / stage));
  s.smem = (int)(stage * s.stages);
  s.per_sm = per_sm;
  return s;
}

static int forward_team(int D) { return D <= 1024 ? 32 : D <= 2048 ? 128 : D <= 4096 ? 256 : 512; }
static int backward_team(int D) { return D <= 512 ? 32 : D <= 2048 ? 128 : D <= 4096 ? 256 : 512; }

constexpr int kBackwardBudget = 110 * 1024;
static int backward_ctas(int D, int elt, int64_t N) {
  const Shape s = shape_of(backward_team(D), 5, D, elt, kBackwardBudget, 1);
  const int per_sm = s.threads >= 256 ? 1 : 2;
  return (int)std::min<int64_t>((N + s.teams - 1) / s.teams, (int64_t)sm_count() * per_sm);
}

constexpr int kMaxSmem = 225 * 1024;
template <auto Kernel>
static int launch(const Params& p, const Shape& s, int ctas, cudaStream_t st, const char* name) {
  static std::once_flag once[64];
  int dev = 0;
  cudaGetDevice(&dev);
  cudaError_t e = cudaSuccess;
  std::call_once(once[dev & 63], [&] { e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem); });
  if (e != cudaSuccess) return check_cuda(e, name);
  Kernel<<<ctas, s.threads, s.smem, st>>>(p);
  return check_cuda(cudaGetLastError(), name);
}

template <typename T>
static int forward(Params& p, cudaStream_t st) {
  const int team = forward_team(p.D);
  const Shape s = shape_of(team, 3, p.D, (int)sizeof(T), 72 * 1024, 2);
  p.stages = s.stages;
  p.row_bytes = s.row_bytes;
  const int64_t ctas = std::min<int64_t>((p.N + s.teams - 1) / s.teams, (int64_t)sm_count() * (s.smem > 110 * 1024 ? 1 : 3));
  const char* name = "sandwich_kernel launch";
  if (team == 32) {
    if (p.D <= 256) return launch<sandwich_kernel<T, 32, 1>>(p, s, (int)ctas, st, name);
    if (p.D <= 512) return launch<sandwich_kernel<T, 32, 2>>(p, s, (int)ctas, st, name);
    return launch<sandwich_kernel<T, 32, 4>>(p, s, (int)ctas, st, name);
  }
  if (team == 128) return launch<sandwich_kernel<T, 128, 2>>(p, s, (int)ctas, st, name);
  if (team == 256) return launch<sandwich_kernel<T, 256, 2>>(p, s, (int)ctas, st, name);
  return launch<sandwich_kernel<T, 512, 2>>(p, s, (int)ctas, st, name);
}

template <typename T, bool LEAN>
static int backward(Params& p, cudaStream_t st) {
  const int team = backward_team(p.D);
  Shape s = shape_of(team, 5, p.D, (int)sizeof(T), kBackwardBudget, 1);
  p.stages = s.stages;
  p.row_bytes = s.row_bytes;
  if (s.teams > 1) s.smem = std::max(s.smem, kSums * p.D * 4);
  const int ctas = backward_ctas(p.D, (int)sizeof(T), p.N);
  const char* name = "sandwich_backward_kernel launch";
  if (team == 32) return launch<sandwich_backward_kernel<T, 32, 2, LEAN>>(p, s, ctas, st, name);
  if (p.D <= 1024) return launch<sandwich_backward_kernel<T, 128, 1, LEAN>>(p, s, ctas, st, name);
  if (team == 128) return launch<sandwich_backward_kernel<T, 128, 2, LEAN>>(p, s, ctas, st, name);
  if (team == 256) return launch<sandwich_backward_kernel<T, 256, 2, LEAN>>(p, s, ctas, st, name);
  return launch<sandwich_backward_kernel<T, 512, 2, LEAN>>(p, s, ctas, st, name);
}

static bool is_float(int dt) { return dt == RB_F32 || dt == RB_BF16 || dt == RB_F16; }

// rows that 16-byte copies can fetch
static bool rows_fit(const void* p, int64_t ld, int D, int elt) {
  return p == nullptr || (D % 8 == 0 && aligned(p, 16) && (ld * elt) % 16 == 0);
}

static int check(int dtype, int64_t N, int D, int post, int pre, int gate_kind, int act, const void* w1, const void* b1,
                 int w1_dtype, const void* w2, const void* b2, int w2_dtype, const void* gate, int gate_dtype) {
  if (N < 0 || D <= 0) return fail(RB_ERR_VALUE, "negative or empty norm shape");
  if (D > kMaxWidth) return fail(RB_ERR_UNSUPPORTED, "rows wider than %d", kMaxWidth);
  if (!is_float(dtype)) return fail(RB_ERR_UNSUPPORTED, "rows are fp32, bf16 or fp16");
  if (post < 0 || post > 2 || pre < 0 || pre > 2) return fail(RB_ERR_VALUE, "unknown norm kind");
  if (gate_kind < 0 || gate_kind > 3 || act < 0 || act > 1) return fail(RB_ERR_VALUE, "unknown gate kind or activation");
  if ((gate_kind != kGateNone) != (gate != nullptr) && N > 0) return fail(RB_ERR_VALUE, "gate and its kind do not agree");
  if (gate != nullptr && !is_float(gate_dtype)) return fail(RB_ERR_UNSUPPORTED, "the gate is fp32, bf16 or fp16");
  if (gate_kind == kGateFull && gate_dtype != dtype) return fail(RB_ERR_VALUE, "a gate of every element has the rows' type");
  if (((w1 != nullptr || b1 != nullptr) && !is_float(w1_dtype)) || ((w2 != nullptr || b2 != nullptr) && !is_float(w2_dtype)))
    return fail(RB_ERR_UNSUPPORTED, "weights are fp32, bf16 or fp16");
  if ((post == kNone && (w1 != nullptr || b1 != nullptr)) || (pre == kNone && (w2 != nullptr || b2 != nullptr)))
    return fail(RB_ERR_VALUE, "weights without their norm");
  return RB_OK;
}

}  // namespace bnorm
}  // namespace rb

using namespace rb;

extern "C" int rb_sandwich_norm(const void* x, int64_t ldx, const void* h, int64_t ldh, int dtype, int64_t N, int D, int post,
                                const void* w1, const void* b1, int w1_dtype, float eps1, int gate_kind, const void* gate,
                                int gate_dtype, int64_t ldg, int gate_act, float scale, int pre, const void* w2,
                                const void* b2, int w2_dtype, float eps2, void* y, void* z, float* stats, void* stream) {
  using namespace rb::bnorm;
  int rc = check(dtype, N, D, post, pre, gate_kind, gate_act, w1, b1, w1_dtype, w2, b2, w2_dtype, gate, gate_dtype);
  if (rc) return rc;
  if (ldx < D || ldh < D || (gate_kind == kGateFull && ldg < D) || (gate_kind == kGateRow && ldg < 0))
    return fail(RB_ERR_VALUE, "leading dimension smaller than the row");
  if (N > 0 && (x == nullptr || h == nullptr || y == nullptr || (pre != kNone && z == nullptr)))
    return fail(RB_ERR_VALUE, "null operand");
  if (!aligned(stats, 16)) return fail(RB_ERR_VALUE, "stats misaligned (16 bytes)");
  if (!device_is_sm100()) return fail(RB_ERR_DEVICE, "rb_sandwich_norm needs an sm_100 (B200) device");
  if (N == 0) return RB_OK;
  const int elt = dtype_size(dtype);
  Params p{};
  p.x = x;
  p.h = h;
  p.gate = gate;
  p.w1 = w1;
  p.b1 = b1;
  p.w2 = w2;
  p.b2 = b2;
  p.out0 = y;
  p.out1 = z;
  p.stats = stats;
  p.N = N;
  p.ldx = ldx;
  p.ldh = ldh;
  p.ldg = ldg;
  p.eps1 = eps1;
  p.eps2 = eps2;
  p.scale = scale;
  p.D = D;
  p.post = post;
  p.pre = pre;
  p.gate_kind = gate_kind;
  p.act = gate_act;
  p.w1_dtype = w1_dtype;
  p.w2_dtype = w2_dtype;
  p.gate_dtype = gate_dtype;
  p.bulk = rows_fit(x, ldx, D, elt) && rows_fit(h, ldh, D, elt) && rows_fit(y, D, D, elt) && rows_fit(z, D, D, elt) &&
           (gate_kind != kGateFull || rows_fit(gate, ldg, D, elt));
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == RB_BF16 ? forward<__nv_bfloat16>(p, st) : dtype == RB_F16 ? forward<__half>(p, st) : forward<float>(p, st);
}

extern "C" int64_t rb_sandwich_norm_workspace_size(int64_t N, int D, int dtype) {
  const int elt = dtype_size(dtype);
  if (N < 0 || D <= 0 || D > bnorm::kMaxWidth || !bnorm::is_float(dtype)) return -1;
  return (int64_t)bnorm::backward_ctas(D, elt, std::max<int64_t>(N, 1)) * bnorm::kSums * D * 4;
}

extern "C" int rb_sandwich_norm_backward(const void* dy, int64_t ldy, const void* dz, int64_t ldz, const void* x, int64_t ldx,
                                         const void* h, int64_t ldh, const float* stats, int dtype, int64_t N, int D,
                                         int post, const void* w1, const void* b1, int w1_dtype, int gate_kind,
                                         const void* gate, int gate_dtype, int64_t ldg, int gate_act, float scale, int pre,
                                         const void* w2, const void* b2, int w2_dtype, void* workspace,
                                         int64_t workspace_bytes, void* dx, void* dh, void* dgate, void* dw1, void* db1,
                                         void* dw2, void* db2, void* stream) {
  using namespace rb::bnorm;
  int rc = check(dtype, N, D, post, pre, gate_kind, gate_act, w1, b1, w1_dtype, w2, b2, w2_dtype, gate, gate_dtype);
  if (rc) return rc;
  if (ldx < D || ldh < D || (dy != nullptr && ldy < D) || (dz != nullptr && ldz < D) || (gate_kind == kGateFull && ldg < D) ||
      (gate_kind == kGateRow && ldg < 0))
    return fail(RB_ERR_VALUE, "leading dimension smaller than the row");
  if (N > 0 && (x == nullptr || h == nullptr || stats == nullptr || dx == nullptr || dh == nullptr ||
                (gate_kind != kGateNone && dgate == nullptr) || workspace == nullptr))
    return fail(RB_ERR_VALUE, "null operand");
  if (dz != nullptr && pre == kNone) return fail(RB_ERR_VALUE, "a gradient of z without its norm");
  if (!aligned(stats, 16) || !aligned(workspace, 16)) return fail(RB_ERR_VALUE, "stats or workspace misaligned (16 bytes)");
  if (workspace_bytes < rb_sandwich_norm_workspace_size(N, D, dtype))
    return fail(RB_ERR_VALUE, "workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                (long long)rb_sandwich_norm_workspace_size(N, D, dtype));
  if (!device_is_sm100()) return fail(RB_ERR_DEVICE, "rb_sandwich_norm_backward needs an sm_100 (B200) device");
  const int elt = dtype_size(dtype);
  Params p{};
  p.x = x;
  p.h = h;
  p.gate = gate;
  p.dy = dy;
  p.dz = dz;
  p.w1 = w1;
  p.b1 = b1;
  p.w2 = w2;
  p.b2 = b2;
  p.out0 = dx;
  p.out1 = dh;
  p.out2 = gate_kind == kGateChannel ? nullptr : dgate;
  p.stats = const_cast<float*>(stats);
  p.partial = static_cast<float*>(workspace);
  p.N = N;
  p.ldx = ldx;
  p.ldh = ldh;
  p.ldg = ldg;
  p.ldy = ldy;
  p.ldz = ldz;
  p.scale = scale;
  p.D = D;
  p.post = post;
  p.pre = dz == nullptr ? kNone : pre;  // nothing reaches y through its norm
  p.gate_kind = gate_kind;
  p.act = gate_act;
  p.w1_dtype = w1_dtype;
  p.w2_dtype = w2_dtype;
  p.gate_dtype = gate_dtype;
  p.bulk = rows_fit(x, ldx, D, elt) && rows_fit(h, ldh, D, elt) && rows_fit(dy, ldy, D, elt) && rows_fit(dz, ldz, D, elt) &&
           rows_fit(dx, D, D, elt) && rows_fit(dh, D, D, elt) &&
           (gate_kind != kGateFull || (rows_fit(gate, ldg, D, elt) && rows_fit(dgate, D, D, elt)));
  SumOut o{};
  const int gdt = gate_dtype;
  void* outs[kSums] = {dw1, db1, dw2, db2, gate_kind == kGateChannel ? dgate : nullptr};
  const int dts[kSums] = {w1_dtype, w1_dtype, w2_dtype, w2_dtype, gdt};
  for (int s = 0; s < kSums; ++s) {
    o.out[s] = outs[s];
    o.dtype[s] = dts[s];
    p.need_sums |= outs[s] != nullptr;
  }
  cudaStream_t st = (cudaStream_t)stream;
  if (N > 0) {
    const bool lean = outs[1] == nullptr && outs[3] == nullptr && outs[4] == nullptr;
    if (dtype == RB_BF16) rc = lean ? backward<__nv_bfloat16, true>(p, st) : backward<__nv_bfloat16, false>(p, st);
    else if (dtype == RB_F16) rc = lean ? backward<__half, true>(p, st) : backward<__half, false>(p, st);
    else rc = lean ? backward<float, true>(p, st) : backward<float, false>(p, st);
    if (rc) return rc;
  }
  if (!p.need_sums) return RB_OK;
  const int ctas = N > 0 ? backward_ctas(D, elt, N) : 0;  // no rows: sums of nothing
  column_sums_kernel<<<dim3((unsigned)((D + 31) / 32), kSums), 256, 0, st>>>(p.partial, ctas, D, o);
  return check_cuda(cudaGetLastError(), "column_sums_kernel launch");
}

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
//
// Measured on a B200 (6.55 TB/s copy): forward 103725 x 512 bf16, layer norms, channel gate 85 us (0.76 of HBM); both
// directions 24490 x 512 fp16 with a sigmoid gate of every element 96 us (forward 29, backward 60, sums 5; floor 38), 4099 x
// 5000 bf16 RMS 154 us (57, 97, 8; floor 50).  Backward is bound by instructions and the two dependent row sums: 1210
// warp instructions a row at 512, issue slots half used at the 16 warps of an SM that its registers allow; wide rows
// leave one row an SM.  Bounds of single values (rows that are no multiple of 8 wide) in the same loops took 1620 and
// 131 us; five column sums instead of four and one thread asking for all copies 199 us.
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
// column sums of backward, t' = act(g) t with the gates of rows and elements: P = sum t' v^ and Q = sum t' of the
// post norm (from which its weight's, bias's and a channel gate's gradients follow), dw and db of the pre norm
constexpr int kSums = 4;

struct Params {
  const void* src[5];                     // rows read: x, h, then a gate of every element | dy, dz and that gate; null: absent
  int64_t pitch[5];                       // their bytes from row to row
  const void* gate;
  const void *w1, *b1, *w2, *b2;          // post and pre affine, or null
  void *out0, *out1, *out2;               // y, z | dx, dh, dgate (rows or elements)
  float* stats;                           // [N, 4]: post mean, 1/deviation, pre mean, 1/deviation
  float* partial;                         // backward: [CTAs][kSums][D]
  int64_t N, ldg;
  float eps1, eps2, scale;
  int D, post, pre, gate_kind, act, w1_dtype, w2_dtype, gate_dtype;
  int bulk, stages, row_bytes, need_sums, table_at, arrays;  // arrays: of src, those that are there
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

// eight parameters from column c, or `none` where there are none; 0 beyond D in either case
__device__ __forceinline__ void param8(const void* p, int dtype, int c, int D, float none, float* v) {
  if (p == nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < D ? none : 0.0f;
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

template <typename T>
__device__ __forceinline__ void widen2(const Eight<T>& e, F2* v) {
  float f[8];
  widen(e, f);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = f2(f[2 * i], f[2 * i + 1]);
}
template <typename T>
__device__ __forceinline__ void narrow2(const F2* v, Eight<T>& e) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 q = un(v[i]);
    f[2 * i] = q.x;
    f[2 * i + 1] = q.y;
  }
  narrow(f, e);
}
__device__ __forceinline__ float total(F2 v) {
  const float2 f = un(v);
  return f.x + f.y;
}

// What a column's constants come to: out of the post norm, y = x + a (A v^ + B) with A = scale a_c w, B = scale a_c b,
// a_c the channel's gate (1 without one) and a the row's or element's; the pre norm's w and b; zeros beyond D.  A
// thread's columns stay its own for all rows, so they are made once and kept as variables (registers up to 4096 columns of 16
// bits; of the 320-thread forward and 640-thread backward forms above, and of fp32 rows, a part is spilled); where a thread
// has too few registers for them (backward, wider than 5120) they lie in shared memory as fp32, and where that is full too
// they are made for each row.
enum Where : int { kRegisters = 0, kTable = 1, kAgain = 2 };
template <typename T>
__device__ __forceinline__ float gate_act(float g, int act);
template <int WHICH, typename T>
__device__ __forceinline__ void make_column8(const Params& p, int c, float* v) {
  if constexpr (WHICH < 2) {
    param8(WHICH == 0 ? p.w1 : p.b1, p.w1_dtype, c, p.D, WHICH == 0 ? 1.0f : 0.0f, v);
    float g[8];
    if (p.gate_kind == kGateChannel) param8(p.gate, p.gate_dtype, c, p.D, 1.0f, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= p.gate_kind == kGateChannel ? p.scale * gate_act<T>(g[i], p.act) : p.scale;
  } else {
    param8(WHICH == 2 ? p.w2 : p.b2, p.w2_dtype, c, p.D, WHICH == 2 ? 1.0f : 0.0f, v);
  }
}
template <int WHICH, typename T>
__device__ __forceinline__ void column8(const Params& p, int c, F2* v) {
  float f[8];
  make_column8<WHICH, T>(p, c, f);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = f2(f[2 * i], f[2 * i + 1]);
}
__device__ __forceinline__ uint4 ld_shared(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
// eight of a row of the table, from a shared address
__device__ __forceinline__ void table8(uint32_t at, F2* v) {
  const uint4 a = ld_shared(at), b = ld_shared(at + 16);
  v[0] = f2(__uint_as_float(a.x), __uint_as_float(a.y));
  v[1] = f2(__uint_as_float(a.z), __uint_as_float(a.w));
  v[2] = f2(__uint_as_float(b.x), __uint_as_float(b.y));
  v[3] = f2(__uint_as_float(b.z), __uint_as_float(b.w));
}
// the table [3][pitch] of A, B and the pre norm's w, by all threads of the CTA
template <typename T>
__device__ __forceinline__ void fill_table(const Params& p, float* table, int pitch) {
  for (int c = threadIdx.x * 8; c < pitch; c += blockDim.x * 8) {
    make_column8<0, T>(p, c, table + c);
    make_column8<1, T>(p, c, table + pitch + c);
    make_column8<2, T>(p, c, table + 2 * pitch + c);
  }
}

// A sigmoid and its derivative, off by a few units of 2^-24 of themselves: from exp(-|g|), since 1 - a near a = 1 and
// exp(-g) of a large -g would lose those bits.
__device__ __forceinline__ float2 sigmoid_of(float g) {
  const float e = expf(-fabsf(g)), r = __fdividef(1.0f, 1.0f + e), low = e * r;
  return make_float2(g < 0.0f ? low : r, low * r);
}
// What a gate does to rows of type T.  16-bit rows: by the fast exponential and quotient, off by |g| units of 2^-23 where the
// sigmoid is small, far below the rows' rounding to 2^-9 or 2^-11 (the exact form took 0.6 us more for a single row, most
// of it instructions to fetch, and 2 of 96 us at 24490 x 512).
template <typename T>
__device__ __forceinline__ float gate_act(float g, int act) {
  if constexpr (sizeof(T) == 4) return act == kActSigmoid ? sigmoid_of(g).x : g;
  else return act == kActSigmoid ? __fdividef(1.0f, 1.0f + __expf(-g)) : g;
}

// A team of G threads on a row of up to 8 V G values; thread r of the team holds the eights r, r + G, ...
// Teams of one or two warps share a CTA of 256 threads, wider ones are a CTA.
template <int G>
struct Team {
  static constexpr int kTeams = G <= 64 ? 256 / G : 1;  // of a CTA
  static constexpr int kThreads = G * kTeams;
  static constexpr int kWarps = G / 32;  // of a team
  static constexpr int kRoom = 2 * kTeams * kWarps * 4;
  __device__ static int index() { return kTeams == 1 ? 0 : (int)threadIdx.x / G; }
  __device__ static int rank() { return kTeams == 1 ? (int)threadIdx.x : (int)threadIdx.x % G; }
  __device__ static void sync() {
    if constexpr (G == 32) __syncwarp();
    else if constexpr (kTeams == 1) __syncthreads();
    else asm volatile("barrier.cta.sync %0, %1;" ::"r"(1 + index()), "n"(G) : "memory");
  }
  __device__ static bool all(bool ok) {
    if constexpr (G == 32) return __all_sync(kAll, ok);
    else if constexpr (kTeams == 1) return __syncthreads_and(ok) != 0;
    else {
      uint32_t every;
      asm volatile(
          "{\n\t.reg .pred p, q;\n\t"
          "setp.ne.u32 p, %1, 0;\n\t"
          "barrier.cta.red.and.pred q, %2, %3, p;\n\t"
          "selp.u32 %0, 1, 0, q;\n\t}"
          : "=r"(every)
          : "r"((uint32_t)ok), "r"(1 + index()), "n"(G)
          : "memory");
      return every != 0;
    }
  }
  // sums of M values over the team; `room` holds kRoom floats, its halves used in turns
  template <int M>
  __device__ static void sum(float (&v)[M], float* room, int& turn) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int m = 0; m < M; ++m) v[m] += __shfl_xor_sync(kAll, v[m], o);
    if constexpr (G > 32) {
      float* at = room + (turn * kTeams + index()) * kWarps * 4;
      turn ^= 1;  // the next sum writes the other half, so one barrier per sum is enough
      const int lane = threadIdx.x & 31;
      if (lane == 0)
#pragma unroll
        for (int m = 0; m < M; ++m) at[(rank() >> 5) * 4 + m] = v[m];
      sync();
      if constexpr (kWarps <= 4) {
#pragma unroll
        for (int m = 0; m < M; ++m) {
          v[m] = at[m];
#pragma unroll
          for (int w = 1; w < kWarps; ++w) v[m] += at[w * 4 + m];
        }
      } else {
#pragma unroll
        for (int m = 0; m < M; ++m) v[m] = lane < kWarps ? at[lane * 4 + m] : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
          for (int m = 0; m < M; ++m)
            if (o < kWarps) v[m] += __shfl_xor_sync(kAll, v[m], o);
#pragma unroll
        for (int m = 0; m < M; ++m) v[m] = __shfl_sync(kAll, v[m], 0);
      }
    }
  }
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// A team's rows: first, first + step, ...  A arrays each.  BULK: by bulk copies (D a multiple of 8, rows on 16-byte
// boundaries); else value by value through the same shared memory.
template <typename T, int G, int V, int A, bool BULK>
struct Rows {
  const Params& p;
  uint8_t* ring;   // this team's stages
  uint64_t* full;  // this team's barriers
  volatile int* abort_flag;
  int64_t first, step;
  const char* next;   // thread a < A of the team asks for array a: its next row, or null
  int64_t next_step;  // bytes from one of the team's rows to the next

  __device__ uint32_t slot(int stage, int a) const { return smem_u32(ring) + (uint32_t)((stage * A + a) * p.row_bytes); }
  __device__ void request(int stage) {  // the team's first warp
    const int lane = threadIdx.x & 31;
    const uint32_t bytes = (uint32_t)(p.D * (int)sizeof(T));
    const uint32_t bar = smem_u32(full + stage);
    if (lane == 0) mbar_arrive_expect_tx(bar, p.arrays * bytes);
    __syncwarp();
    if (next != nullptr) {
      bulk_load(slot(stage, lane), next, bytes, bar);
      next += next_step;
    }
  }
  __device__ void start() {
    next = nullptr;
    if constexpr (BULK) {
      const int r = Team<G>::rank();
      if (r >= 32) return;
      if (r < A && p.src[r] != nullptr) {
        next = static_cast<const char*>(p.src[r]) + first * p.pitch[r];
        next_step = step * p.pitch[r];
      }
      for (int s = 0; s < p.stages; ++s)
        if (first + s * step < p.N) request(s);
    }
  }
  // Row `row`'s eights (zeros beyond D and for absent arrays) into registers; asks for the row `stages` turns on.
  __device__ bool take(int64_t row, int stage, uint32_t phase, Eight<T> (&e)[A][V]) {
    const int r = Team<G>::rank();
    bool ok = true;
    if constexpr (BULK) {
      ok = mbar_wait_bounded(smem_u32(full + stage), phase, kWaitTimeoutProducer, abort_flag);
    } else {
      // neighbours by neighbouring threads
#pragma unroll
      for (int a = 0; a < A; ++a) {
        if (p.src[a] == nullptr) continue;
        const T* from = reinterpret_cast<const T*>(static_cast<const char*>(p.src[a]) + row * p.pitch[a]);
        T* to = reinterpret_cast<T*>(ring + (stage * A + a) * p.row_bytes);
        for (int c = r; c < p.D; c += G) to[c] = from[c];
      }
      Team<G>::sync();
    }
    const uint32_t base = slot(stage, 0);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int c = (v * G + r) * 8;
      const bool in = ok && c < p.D;
#pragma unroll
      for (int a = 0; a < A; ++a) {
#pragma unroll
        for (int q = 0; q < (int)(sizeof(T) / 2); ++q) {
          e[a][v].q[q] = make_uint4(0u, 0u, 0u, 0u);
          if (in && p.src[a] != nullptr) e[a][v].q[q] = ld_shared(base + (uint32_t)(a * p.row_bytes + c * (int)sizeof(T) + 16 * q));
        }
        if (!BULK && c < p.D && c + 8 > p.D) {  // a row's last eight may be short
          T* t = reinterpret_cast<T*>(&e[a][v]);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c + i >= p.D) t[i] = T(0.0f);
        }
      }
    }
    ok = Team<G>::all(ok);
    if (BULK && ok && r < 32 && row + p.stages * step < p.N) {
      // the slot was read through the generic proxy: order those reads before the copy's writes
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      request(stage);
    }
    return ok;
  }
  // After a wait that gave up at (row, stage, phase): the copies still in flight land before this CTA leaves.
  __device__ void drain(int64_t row, int stage, uint32_t phase) const {
    if constexpr (BULK) {
      if (Team<G>::rank() != 0) return;
      for (int s = 0; s < p.stages && row < p.N; ++s, row += step) {
        mbar_wait_bounded(smem_u32(full + stage), phase, kWaitTimeoutProducer, nullptr);
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
  }
  // A row out: straight from registers, or (rows that 16-byte stores do not fit) through this stage's first slot
  __device__ void put(void* out, int64_t row, int stage, const F2 (&v)[V * 4]) const {
    const int r = Team<G>::rank();
    T* to = static_cast<T*>(out) + row * p.D;
    T* via = BULK ? to : reinterpret_cast<T*>(ring + stage * A * p.row_bytes);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = (k * G + r) * 8;
      if (c >= p.D) continue;
      Eight<T> e;
      narrow2(v + 4 * k, e);
#pragma unroll
      for (int q = 0; q < (int)(sizeof(T) / 2); ++q) reinterpret_cast<uint4*>(via + c)[q] = e.q[q];
    }
    if constexpr (!BULK) {
      Team<G>::sync();
      for (int c = r; c < p.D; c += G) to[c] = via[c];
      Team<G>::sync();
    }
  }
};

// v centred and normalised in place over the team's row (zeros beyond D stay zeros); mean and 1 / deviation
template <int G, int V, bool BULK>
__device__ __forceinline__ void normalise(F2 (&v)[V * 4], int kind, float eps, int D, float* room, int& turn,
                                          float& mean, float& rstd) {
  const int r = Team<G>::rank();
  const float inv = 1.0f / (float)D;
  mean = 0.0f;
  if (kind == kLayer) {
    F2 a = v[0];
#pragma unroll
    for (int i = 1; i < V * 4; ++i) a = add2(a, v[i]);
    float s[1] = {total(a)};
    Team<G>::sum(s, room, turn);
    mean = s[0] * inv;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = (k * G + r) * 8;
      const F2 m = c < D ? f2(-mean, -mean) : f2(0.0f, 0.0f);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[4 * k + i] = add2(v[4 * k + i], m);
        if constexpr (!BULK) {
          const float2 f = un(v[4 * k + i]);
          v[4 * k + i] = f2(c + 2 * i < D ? f.x : 0.0f, c + 2 * i + 1 < D ? f.y : 0.0f);
        }
      }
    }
  }
  F2 a = mul2(v[0], v[0]);
#pragma unroll
  for (int i = 1; i < V * 4; ++i) a = fma2(v[i], v[i], a);
  float s[1] = {total(a)};
  Team<G>::sum(s, room, turn);
  rstd = rsqrtf(fmaf(s[0], inv, eps));
  const F2 q = f2(rstd, rstd);
#pragma unroll
  for (int i = 0; i < V * 4; ++i) v[i] = mul2(v[i], q);
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

template <typename T, int G, int V, bool BULK>
__global__ void __launch_bounds__(Team<G>::kThreads, G == 320 ? 2 : 512 / Team<G>::kThreads)
    sandwich_kernel(const __grid_constant__ Params p) {
  using Tm = Team<G>;
  constexpr int kArrays = 3;  // x, h, a gate of every element
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ __align__(8) uint64_t full[kMaxStages * Tm::kTeams];
  __shared__ float room[Tm::kRoom];
  __shared__ int abort_flag;
  init_ring<G>(full, p.stages, &abort_flag);
  const int r = Tm::rank();
  Rows<T, G, V, kArrays, BULK> rows{p,
                                    ring + Tm::index() * p.stages * kArrays * p.row_bytes,
                                    full + Tm::index() * p.stages,
                                    &abort_flag,
                                    (int64_t)blockIdx.x * Tm::kTeams + Tm::index(),
                                    (int64_t)gridDim.x * Tm::kTeams,
                                    nullptr,
                                    0};
  rows.start();

  F2 A[V * 4], B[V * 4], w2[V * 4], b2[V * 4];  // zeros beyond D
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = (k * G + r) * 8;
    column8<0, T>(p, c, A + 4 * k);
    column8<1, T>(p, c, B + 4 * k);
    column8<2, T>(p, c, w2 + 4 * k);
    column8<3, T>(p, c, b2 + 4 * k);
  }

  int stage = 0, turn = 0;
  uint32_t phase = 0;
  float next_gate = 1.0f;
  auto ahead = [&](int64_t row) {
    if (p.gate_kind == kGateRow && row < p.N)
      next_gate = gate_act<T>(load_as_f32(p.gate, p.gate_dtype, row * p.ldg), p.act);
  };
  ahead(rows.first);
  for (int64_t row = rows.first; row < p.N; row += rows.step) {
    Eight<T> e[kArrays][V];
    if (!rows.take(row, stage, phase, e)) {
      rows.drain(row, stage, phase);
      break;
    }
    const F2 row_gate = f2(next_gate, next_gate);
    ahead(row + rows.step);
    F2 n[V * 4], y[V * 4];
    float mean1 = 0.0f, rstd1 = 1.0f, mean2 = 0.0f, rstd2 = 1.0f;
#pragma unroll
    for (int k = 0; k < V; ++k) widen2(e[1][k], n + 4 * k);
    if (p.post != kNone) normalise<G, V, BULK>(n, p.post, p.eps1, p.D, room, turn, mean1, rstd1);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      F2 x[4], a[4] = {row_gate, row_gate, row_gate, row_gate};
      widen2(e[0][k], x);
      if (p.gate_kind == kGateFull) {
        float g[8];
        widen(e[2][k], g);
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = f2(gate_act<T>(g[2 * i], p.act), gate_act<T>(g[2 * i + 1], p.act));
      }
#pragma unroll
      for (int i = 4 * k; i < 4 * k + 4; ++i) y[i] = fma2(a[i & 3], fma2(n[i], A[i], B[i]), x[i & 3]);
    }
    rows.put(p.out0, row, stage, y);
    if (p.pre != kNone) {
      normalise<G, V, BULK>(y, p.pre, p.eps2, p.D, room, turn, mean2, rstd2);
#pragma unroll
      for (int i = 0; i < V * 4; ++i) y[i] = fma2(y[i], w2[i], b2[i]);
      rows.put(p.out1, row, stage, y);
    }
    if (p.stats != nullptr && r == 0)
      reinterpret_cast<float4*>(p.stats)[row] = make_float4(mean1, rstd1, mean2, rstd2);
    if (++stage == p.stages) {
      stage = 0;
      phase ^= 1;
    }
  }
}

// LEAN: no biases and no gate per channel: the column sums P and dw alone.  FULL: a gate of every element.  WHERE:
// the column constants.  Eight values a thread.
template <typename T, int G, bool BULK, int WHERE, bool LEAN, bool FULL>
__global__ void __launch_bounds__(Team<G>::kThreads, Team<G>::kThreads <= 512 ? 512 / Team<G>::kThreads : 1)
    sandwich_backward_kernel(const __grid_constant__ Params p) {
  using Tm = Team<G>;
  constexpr int kArrays = FULL ? 5 : 4;  // x, h, dy, dz, a gate of every element
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ __align__(8) uint64_t full[kMaxStages * Tm::kTeams];
  __shared__ float room[Tm::kRoom];
  __shared__ int abort_flag;
  init_ring<G>(full, p.stages, &abort_flag);
  const int r = Tm::rank(), c = 8 * r;
  Rows<T, G, 1, kArrays, BULK> rows{p,
                                    ring + Tm::index() * p.stages * kArrays * p.row_bytes,
                                    full + Tm::index() * p.stages,
                                    &abort_flag,
                                    (int64_t)blockIdx.x * Tm::kTeams + Tm::index(),
                                    (int64_t)gridDim.x * Tm::kTeams,
                                    nullptr,
                                    0};
  rows.start();

  // A, B and the pre norm's w are zeros beyond D, as x, h, dy and dz are: what a thread computes there reaches no sum
  const int pitch = (p.D + 7) / 8 * 8;
  F2 A[4], B[4], w2[4];
  uint32_t table = 0;
  if constexpr (WHERE == kTable) {
    fill_table<T>(p, reinterpret_cast<float*>(ring + p.table_at), pitch);
    __syncthreads();
    table = smem_u32(ring + p.table_at) + (c < p.D ? 4 * c : 0);  // a thread beyond D: any columns, its x, h, dy and dz are 0
  }
  auto columns = [&](bool pre) {
    if constexpr (WHERE == kTable) {
      table8(table, A);
      table8(table + 4 * pitch, B);
      if (pre) table8(table + 8 * pitch, w2);
      if (c >= p.D) {
#pragma unroll
        for (int i = 0; i < 4; ++i) A[i] = B[i] = w2[i] = f2(0.0f, 0.0f);
      }
    } else {
      column8<0, T>(p, c, A);
      column8<1, T>(p, c, B);
      if (pre) column8<2, T>(p, c, w2);
    }
  };
  if constexpr (WHERE == kRegisters) columns(true);

  constexpr int kHeld = LEAN ? 2 : kSums;
  F2 acc[kHeld][4];  // P, dw, then Q, db
#pragma unroll
  for (int a = 0; a < kHeld; ++a)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[a][i] = f2(0.0f, 0.0f);

  const float inv1 = p.post == kLayer ? -1.0f / (float)p.D : 0.0f, inv2 = p.pre == kLayer ? -1.0f / (float)p.D : 0.0f;
  const float inv = -1.0f / (float)p.D;
  int stage = 0, turn = 0;
  uint32_t phase = 0;
  float4 st = make_float4(0.0f, 1.0f, 0.0f, 1.0f);
  float g_row = 1.0f;
  auto ahead = [&](int64_t row) {  // the next row's scalars
    if (row < p.N) {
      st = __ldg(reinterpret_cast<const float4*>(p.stats) + row);
      if (!FULL && p.gate_kind == kGateRow) g_row = gate_act<T>(load_as_f32(p.gate, p.gate_dtype, row * p.ldg), p.act);
    }
  };
  ahead(rows.first);
  for (int64_t row = rows.first; row < p.N; row += rows.step) {
    const float4 s = st;
    const float ar = g_row;
    Eight<T> e[kArrays][1];
    if (!rows.take(row, stage, phase, e)) {
      rows.drain(row, stage, phase);
      break;
    }
    ahead(row + rows.step);
    // the gates of this row; without gates of every element one value, in every a[i]
    F2 a[FULL ? 4 : 1];
    if constexpr (FULL) {
      float g[8];
      widen(e[4][0], g);
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = f2(gate_act<T>(g[2 * i], p.act), gate_act<T>(g[2 * i + 1], p.act));
    } else {
      a[0] = f2(ar, ar);
    }
    F2 hh[4], yh[4], t[4];
    widen2(e[1][0], hh);
    {
      const F2 q = f2(s.y, s.y), m = f2(-s.x * s.y, -s.x * s.y);
#pragma unroll
      for (int i = 0; i < 4; ++i) hh[i] = fma2(hh[i], q, m);
    }
    if (p.pre != kNone) {
      // n and y again, and the pre norm's two sums
      const F2 q = f2(s.w, s.w), m = f2(-s.z * s.w, -s.z * s.w);
      F2 s1 = f2(0.0f, 0.0f), s2 = s1, x[4], dz[4];
      if constexpr (WHERE != kRegisters) columns(true);
      widen2(e[0][0], x);
      widen2(e[3][0], dz);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        yh[i] = fma2(fma2(a[FULL ? i : 0], fma2(hh[i], A[i], B[i]), x[i]), q, m);
        t[i] = mul2(dz[i], w2[i]);
        s1 = add2(s1, t[i]);
        s2 = fma2(t[i], yh[i], s2);
        acc[1][i] = fma2(dz[i], yh[i], acc[1][i]);
        if constexpr (!LEAN) acc[3][i] = add2(acc[3][i], dz[i]);
      }
      float s12[2] = {total(s1), total(s2)};
      Tm::sum(s12, room, turn);
      const float c1 = s12[0] * inv2 * s.w, c2 = s12[1] * inv * s.w;
      const F2 k1 = f2(c1, c1), k2 = f2(c2, c2);
      F2 dy[4];
      widen2(e[2][0], dy);
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = add2(fma2(yh[i], k2, fma2(t[i], q, k1)), dy[i]);
    } else {
      widen2(e[2][0], t);
    }
    // t reaches y; its way into h, the gate and the post norm's weights
    rows.put(p.out0, row, stage, t);
    if constexpr (WHERE != kRegisters) columns(false);
    F2 s3 = f2(0.0f, 0.0f), s4 = s3, s5 = s3;
    if (FULL || p.gate_kind == kGateRow) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const F2 ai = a[FULL ? i : 0];
        F2 da = mul2(fma2(hh[i], A[i], B[i]), t[i]);
        if constexpr (FULL) {
          if (p.act == kActSigmoid) {
            if constexpr (sizeof(T) == 4) {
              float g[8];
              widen(e[4][0], g);
              da = mul2(da, f2(sigmoid_of(g[2 * i]).y, sigmoid_of(g[2 * i + 1]).y));
            } else {
              da = mul2(da, fma2(mul2(ai, f2(-1.0f, -1.0f)), ai, ai));
            }
          }
        }
        yh[i] = da;  // of every element: its gradient
        s5 = add2(s5, da);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const F2 tp = mul2(a[FULL ? i : 0], t[i]);
      acc[0][i] = fma2(tp, hh[i], acc[0][i]);
      if constexpr (!LEAN) acc[2][i] = add2(acc[2][i], tp);
      t[i] = mul2(tp, A[i]);
      s3 = add2(s3, t[i]);
      s4 = fma2(t[i], hh[i], s4);
    }
    if constexpr (FULL) rows.put(p.out2, row, stage, yh);
    if (p.post != kNone || (!FULL && p.gate_kind == kGateRow)) {
      float s345[FULL ? 2 : 3];
      s345[0] = total(s3);
      s345[1] = total(s4);
      if constexpr (!FULL) s345[2] = total(s5);
      Tm::sum(s345, room, turn);
      if (!FULL && p.gate_kind == kGateRow && r == 0) {
        float d = s345[FULL ? 0 : 2];
        if (p.act == kActSigmoid) d *= sigmoid_of(load_as_f32(p.gate, p.gate_dtype, row * p.ldg)).y;
        if (p.gate_dtype == RB_F32) static_cast<float*>(p.out2)[row] = d;
        else if (p.gate_dtype == RB_BF16) static_cast<__nv_bfloat16*>(p.out2)[row] = __float2bfloat16_rn(d);
        else static_cast<__half*>(p.out2)[row] = __float2half_rn(d);
      }
      if (p.post != kNone) {
        const float c3 = s345[0] * inv1 * s.y, c4 = s345[1] * inv * s.y;
        const F2 k3 = f2(c3, c3), k4 = f2(c4, c4), q = f2(s.y, s.y);
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = fma2(hh[i], k4, fma2(t[i], q, k3));
      }
    }
    rows.put(p.out1, row, stage, t);
    if (++stage == p.stages) {
      stage = 0;
      phase ^= 1;
    }
  }

  if (!p.need_sums) return;
  // the CTA's sums: its teams one after another through shared memory, then this CTA's row of `partial`
  auto held_sum = [&](int a, int j) {
    const float2 f = un(acc[a][j >> 1]);
    return (j & 1) ? f.y : f.x;
  };
  if constexpr (Tm::kTeams == 1) {
#pragma unroll
    for (int a = 0; a < kHeld; ++a)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (c + i < p.D) p.partial[((int64_t)blockIdx.x * kSums + a) * p.D + c + i] = held_sum(a, i);
  } else {
    __syncthreads();  // every team is done with the ring
    float* sums = reinterpret_cast<float*>(ring);
    for (int w = 0; w < Tm::kTeams; ++w) {
      if (Tm::index() == w) {
#pragma unroll
        for (int a = 0; a < kHeld; ++a)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c + i < p.D) {
              float* at = sums + a * p.D + c + i;
              *at = (w == 0 ? 0.0f : *at) + held_sum(a, i);
            }
      }
      __syncthreads();
    }
    for (int j = threadIdx.x; j < kHeld * p.D; j += Tm::kThreads) {
      const int a = j / p.D;
      p.partial[((int64_t)blockIdx.x * kSums + a) * p.D + (j - a * p.D)] = sums[j];
    }
  }
}

struct SumOut {
  void *dw1, *db1, *dw2, *db2, *dgate;
};

__device__ __forceinline__ void store_param(void* p, int dtype, int c, float v) {
  if (p == nullptr) return;
  if (dtype == RB_F32) static_cast<float*>(p)[c] = v;
  else if (dtype == RB_BF16) static_cast<__nv_bfloat16*>(p)[c] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[c] = __float2half_rn(v);
}

// The CTAs' sums of eight columns, in a fixed order (32 runs of CTAs, then a tree), and what follows from them:
// dw = scale a_c P, db = scale a_c Q, dgate = scale act'(g) (w P + b Q).
constexpr int kSumRuns = 32;
__global__ void __launch_bounds__(8 * kSumRuns) column_sums_kernel(const __grid_constant__ Params p, int ctas, int held,
                                                             const __grid_constant__ SumOut o) {
  __shared__ float part[kSums][kSumRuns][8];
  const int at = threadIdx.x & 7, run = threadIdx.x >> 3, c = blockIdx.x * 8 + at;
  float v[kSums] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (c < p.D) {
#pragma unroll 4
    for (int b = run; b < ctas; b += kSumRuns)
#pragma unroll
      for (int s = 0; s < kSums; ++s)
        if (s < held) v[s] += p.partial[((int64_t)b * kSums + s) * p.D + c];
  }
#pragma unroll
  for (int s = 0; s < kSums; ++s) part[s][run][at] = v[s];
  for (int n = kSumRuns / 2; n > 0; n >>= 1) {
    __syncthreads();
    if (run < n)
#pragma unroll
      for (int s = 0; s < kSums; ++s) part[s][run][at] += part[s][run + n][at];
  }
  if (run != 0 || c >= p.D) return;
  const float P = part[0][0][at], dw = part[1][0][at], Q = part[2][0][at], db = part[3][0][at];
  float k = p.scale;
  if (p.gate_kind == kGateChannel) {
    const float g = load_as_f32(p.gate, p.gate_dtype, c);
    const float w = p.w1 != nullptr ? load_as_f32(p.w1, p.w1_dtype, c) : 1.0f;
    const float b = p.b1 != nullptr ? load_as_f32(p.b1, p.w1_dtype, c) : 0.0f;
    const float2 a = p.act == kActSigmoid ? sigmoid_of(g) : make_float2(g, 1.0f);
    store_param(o.dgate, p.gate_dtype, c, p.scale * a.y * fmaf(w, P, b * Q));
    k *= a.x;
  }
  store_param(o.dw1, p.w1_dtype, c, k * P);
  store_param(o.db1, p.w1_dtype, c, k * Q);
  store_param(o.dw2, p.w2_dtype, c, dw);
  store_param(o.db2, p.w2_dtype, c, db);
}

// ------------------------------------------------------------------- host
constexpr int kMaxSmem = 225 * 1024;
struct Shape {
  int threads, teams, stages, row_bytes, smem, table_at;
};

// A width's team and ring: as many stages (up to kMaxStages) as fit `budget` bytes of a CTA's shared memory, beside
// `table` rows of fp32 column constants where asked for and where they fit.
static Shape shape_of(int team, int arrays, int D, int elt, int64_t budget, int table) {
  Shape s{};
  s.teams = team <= 64 ? 256 / team : 1;
  s.threads = team * s.teams;
  s.row_bytes = (D + 7) / 8 * 8 * elt;  // whole eights: a thread reads and writes them as such
  const int64_t stage = (int64_t)s.teams * arrays * s.row_bytes, columns = (int64_t)table * ((D + 7) / 8 * 8) * 4;
  const bool room = table > 0 && stage + columns <= kMaxSmem;
  if (room) budget -= columns;
  s.stages = (int)std::max<int64_t>(1, std::min<int64_t>(kMaxStages, budget / stage));
  s.table_at = room ? (int)(stage * s.stages) : -1;
  s.smem = (int)(stage * s.stages + (room ? columns : 0));
  return s;
}

// Eight values a thread.  640 threads from 4097 to 5120 columns: with 1024 the constants no longer fit the registers.
// Backward, 20 M bf16 values, layer norms and RMS without biases, 640 / 1024 threads: 4104 wide 163 and 107 / 308 and 204 us,
// 4608 148 and 101 / 288 and 192, 5120 139 and 95 / 263 and 175.
static int team_of(int D) {
  for (int team : {32, 64, 128, 256, 512, 640})
    if (D <= 8 * team) return team;
  return 1024;
}
static int ctas_per_sm(const Shape& s, int threads_per_sm) {
  const int by_smem = 226 * 1024 / (s.smem + 2048);
  return std::max(1, std::min(by_smem, threads_per_sm / s.threads));
}
// bytes of a CTA's ring, where an SM is to hold `threads` threads and 200 KB of rings
static int64_t ring_budget(int team, int threads) {
  const int cta = team <= 64 ? 256 : team;
  return (int64_t)200 * 1024 / std::max(1, threads / cta);
}
constexpr int kForwardThreads = 512, kBackwardThreads = 512;  // an SM's, by the kernels' registers
static Shape backward_shape(int D, int elt, bool full) {
  const int team = team_of(D);
  Shape s = shape_of(team, full ? 5 : 4, D, elt, ring_budget(team, kBackwardThreads), team == 1024 ? 3 : 0);
  if (s.teams > 1) s.smem = std::max(s.smem, kSums * D * 4);
  return s;
}
static int backward_ctas(int D, int elt, int64_t N) {  // the same with and without gates of every element
  const Shape s = backward_shape(D, elt, true);
  return (int)std::min<int64_t>((N + s.teams - 1) / s.teams, (int64_t)sm_count() * ctas_per_sm(s, kBackwardThreads));
}

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
  // Sixteen values a thread: a row's fixed instructions (copies, waits, sums) fall to half the warps, and two rows
  // fit an SM where eight values leave room for one (50 M bf16 values on a B200, layer norms, sixteen against eight a
  // thread when it was chosen: 512 wide 94 / 146 us, 1024 119 / 151, 2048 119 / 174, 4096 133 / 185, 8192 145 / 195).
  // Teams of 320 just above 4096: two rows an SM, where 512 threads of sixteen would be used to half or two thirds.  20 M
  // bf16 values, layer norms and RMS, 320 / 512 threads: 4104 wide 78.9 and 62.5 / 93.9 and 70.8 us, 4608 71.1 and 57.6 /
  // 84.8 and 64.1, 5120 65.8 and 54.4 / 78.0 and 58.8.
  const bool two = p.D > 256;
  const int team = !two ? 32 : p.D <= 4096 ? team_of((p.D + 1) / 2) : p.D <= 5120 ? 320 : 512;
  const Shape s = shape_of(team, 3, p.D, (int)sizeof(T), ring_budget(team, team == 320 ? 640 : kForwardThreads), 0);
  p.stages = s.stages;
  p.row_bytes = s.row_bytes;
  p.table_at = s.table_at;
  const int ctas = (int)std::min<int64_t>((p.N + s.teams - 1) / s.teams, (int64_t)sm_count() * ctas_per_sm(s, team == 320 ? 640 : kForwardThreads));
  const char* name = "sandwich_kernel launch";
#define RB_FORWARD(G, V)                                                      \
  return p.bulk ? launch<sandwich_kernel<T, G, V, true>>(p, s, ctas, st, name) \
                : launch<sandwich_kernel<T, G, V, false>>(p, s, ctas, st, name)
  if (two) {
    switch (team) {
      case 32: RB_FORWARD(32, 2);
      case 64: RB_FORWARD(64, 2);
      case 128: RB_FORWARD(128, 2);
      case 256: RB_FORWARD(256, 2);
      case 320: RB_FORWARD(320, 2);
      default: RB_FORWARD(512, 2);
    }
  }
  RB_FORWARD(32, 1);
#undef RB_FORWARD
}

template <typename T, int G, int WHERE, bool LEAN>
static int backward_of(const Params& p, const Shape& s, int ctas, cudaStream_t st) {
  const char* name = "sandwich_backward_kernel launch";
  const bool full = p.gate_kind == kGateFull;
  if (!p.bulk)
    return full ? launch<sandwich_backward_kernel<T, G, false, WHERE, false, true>>(p, s, ctas, st, name)
                : launch<sandwich_backward_kernel<T, G, false, WHERE, false, false>>(p, s, ctas, st, name);
  return full ? launch<sandwich_backward_kernel<T, G, true, WHERE, LEAN, true>>(p, s, ctas, st, name)
              : launch<sandwich_backward_kernel<T, G, true, WHERE, LEAN, false>>(p, s, ctas, st, name);
}

template <typename T>
static int backward(Params& p, bool lean, cudaStream_t st) {
  const Shape s = backward_shape(p.D, (int)sizeof(T), p.gate_kind == kGateFull);
  p.stages = s.stages;
  p.row_bytes = s.row_bytes;
  p.table_at = s.table_at;
  const int ctas = backward_ctas(p.D, (int)sizeof(T), p.N);
  switch (team_of(p.D)) {
    case 32: return backward_of<T, 32, kRegisters, false>(p, s, ctas, st);
    case 64: return backward_of<T, 64, kRegisters, false>(p, s, ctas, st);
    case 128: return backward_of<T, 128, kRegisters, false>(p, s, ctas, st);
    case 256: return backward_of<T, 256, kRegisters, false>(p, s, ctas, st);
    case 512: return backward_of<T, 512, kRegisters, false>(p, s, ctas, st);
    // wider teams have fewer registers a thread: without biases and channel gates two sums are left out
    case 640:
      return lean ? backward_of<T, 640, kRegisters, true>(p, s, ctas, st) : backward_of<T, 640, kRegisters, false>(p, s, ctas, st);
    default: break;
  }
  if (s.table_at < 0) {  // fp32 rows and gates of every element from 7201 columns on
    if constexpr (sizeof(T) == 4) return backward_of<T, 1024, kAgain, false>(p, s, ctas, st);
    else return fail(RB_ERR_UNSUPPORTED, "no shared memory for the column constants");  // not reached: 16-bit rows leave room
  }
  return lean ? backward_of<T, 1024, kTable, true>(p, s, ctas, st) : backward_of<T, 1024, kTable, false>(p, s, ctas, st);
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
  const void* gates = gate_kind == kGateFull ? gate : nullptr;
  const void* src[3] = {x, h, gates};
  const int64_t ld[3] = {ldx, ldh, ldg};
  for (int a = 0; a < 3; ++a) {
    p.src[a] = src[a];
    p.pitch[a] = ld[a] * elt;
    p.arrays += src[a] != nullptr;
  }
  p.gate = gate;
  p.w1 = w1;
  p.b1 = b1;
  p.w2 = w2;
  p.b2 = b2;
  p.out0 = y;
  p.out1 = z;
  p.stats = stats;
  p.N = N;
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
  const void* gates = gate_kind == kGateFull ? gate : nullptr;
  const void* src[5] = {x, h, dy, dz, gates};
  const int64_t ld[5] = {ldx, ldh, ldy, ldz, ldg};
  for (int a = 0; a < 5; ++a) {
    p.src[a] = src[a];
    p.pitch[a] = ld[a] * elt;
    p.arrays += src[a] != nullptr;
  }
  p.gate = gate;
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
  p.ldg = ldg;
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
  SumOut o{dw1, db1, dw2, db2, gate_kind == kGateChannel ? dgate : nullptr};
  p.need_sums = o.dw1 != nullptr || o.db1 != nullptr || o.dw2 != nullptr || o.db2 != nullptr || o.dgate != nullptr;
  cudaStream_t st = (cudaStream_t)stream;
  // (the narrow teams and rows that no bulk copy fetches keep all sums)
  const bool lean = o.db1 == nullptr && o.db2 == nullptr && o.dgate == nullptr;
  if (N > 0) {
    rc = dtype == RB_BF16 ? backward<__nv_bfloat16>(p, lean, st)
         : dtype == RB_F16 ? backward<__half>(p, lean, st)
                           : backward<float>(p, lean, st);
    if (rc) return rc;
  }
  if (!p.need_sums) return RB_OK;
  const int ctas = N > 0 ? backward_ctas(D, elt, N) : 0;  // no rows: sums of nothing
  column_sums_kernel<<<(unsigned)((D + 7) / 8), 8 * kSumRuns, 0, st>>>(p, ctas, lean ? 2 : kSums, o);
  return check_cuda(cudaGetLastError(), "column_sums_kernel launch");
}

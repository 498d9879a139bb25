// route.cu -- routing to experts: what stands before rb_smoe_experts.  From a
// row of E logits per token, scores s (softmax or sigmoid), choice values
// c = s + bias, the best groups of experts, the k experts of the highest choice
// value, their scores (renormalised to one, times a scale), and the gradient of
// the logits.
//
// A token is held by a sub-warp of L lanes, V logits a lane (E <= L * V), so
// that maxima and sums over its experts are a few shuffles and every logit is
// read once.  The choice takes k rounds: each lane's best, the sub-warp's best,
// and the winner leaves.
//
// The choice must not depend on how exp rounds: experts are ordered by their
// exact choice values, ties to the lowest index.
//   * A 32-bit word holds the leading bits of the choice value's order-preserving
//     fp32 pattern and the value's place in its lane.  16-bit logits without a bias
//     are compared themselves, since the scores rise with them, and lose nothing.
//   * Otherwise (scores, with a bias or in sums, or fp32 logits) two neighbours of
//     the order, or the last kept and the first dropped group, may lie closer than
//     the fp32 error bound.  A single such pair is settled by its two values in
//     fp64, anything else by the token's whole order in fp64.
// Each lane sorts its V words once (a network of minima and maxima), so a round
// is one maximum over the lanes' heads and a shift in the lane that had it.
//
// What bounds it: the launch for small calls (one token 2.1-2.5 us, 103725 x 8 4.2 us),
// instructions for many experts (integer minima, maxima and selects run at half
// rate), never bytes.  16411 x 256 fp32 in groups with a bias (17 MB, 2.8 us of HBM):
// 19.2 M warp instructions, 29 us, of which about 11 are one or two tokens whose
// groups are decided again in fp64, late in the grid; rounds over unsorted lanes and
// 64-bit words took 25.6 M and 40 us.  24490 x 64: 7.3 us forward, 6.2 backward.
// Eight values a lane: with sixteen (half the lanes a token) 16411 x 256 took 22 us
// for 14 (bf16, no bias), and a persistent grid that asked a token ahead 20.
#include "common.cuh"

namespace rb {
namespace route {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxExperts = 512;
constexpr int kMaxK = 32;
constexpr unsigned kAll = 0xffffffffu;

enum ScoreKind : int { kSoftmax = RB_SCORE_SOFTMAX, kSigmoid = RB_SCORE_SIGMOID };

struct Params {
  const void* logits;
  const float* bias;
  void* idx;
  void* score;
  void* probs;
  int32_t* counts;
  int64_t ld, T;
  float scale, lowest;
  int dtype, E, k, kind, groups, gsize, topk_groups, group_top, renorm, idx64, score_dtype, by_logit;
  uint32_t k_inv;  // ceil(2^16 / k): q / k for q < 1024
};

struct BwdParams {
  const void* logits;
  const void* idx;
  const void* grad_score;
  const void* grad_probs;
  void* grad_logits;
  int64_t ld, T;
  float scale, lowest;
  int dtype, E, k, kind, renorm, idx64, grad_dtype, probs_dtype, out_dtype;
};

// order-preserving patterns; NaN is above everything, and no value maps to 0
__device__ __forceinline__ uint32_t order32(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);  // -0 as +0, any NaN as the positive one
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unorder32(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ unsigned long long order64(double v) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);
  if (v != v) return ~0ull;
  return (u >> 63) ? ~u : (u | (1ull << 63));
}
__device__ __forceinline__ double unorder64(unsigned long long o) {
  return __longlong_as_double((long long)((o >> 63) ? (o & ~(1ull << 63)) : ~o));
}

template <int L, typename T>
__device__ __forceinline__ T sub_sum(T v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}
template <int L>
__device__ __forceinline__ float sub_max(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, o));
  return v;
}
template <int L>
__device__ __forceinline__ uint32_t sub_umax(uint32_t v) {
  if constexpr (L == 32) {
    return __reduce_max_sync(kAll, v);
  } else {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(kAll, v, o));
    return v;
  }
}
template <int L>
__device__ __forceinline__ uint32_t sub_umin(uint32_t v) {
  if constexpr (L == 32) {
    return __reduce_min_sync(kAll, v);
  } else {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v = min(v, __shfl_xor_sync(kAll, v, o));
    return v;
  }
}

// index of a lane's i-th value: 8 neighbours per 16-byte (or 32-byte) load, or
// one value per lane side by side where rows are not aligned for that
template <int L, bool VEC>
__device__ __forceinline__ int elem(int sl, int i) {
  return VEC ? ((i >> 3) * L + sl) * 8 + (i & 7) : i * L + sl;
}

__device__ __forceinline__ void unpack8(const void* p, int dtype, float* v) {
  if (dtype == RB_F32) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    return;
  }
  const uint4 w = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (dtype == RB_BF16) {
      v[2 * j] = bf16_lo(ww[j]);
      v[2 * j + 1] = bf16_hi(ww[j]);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&ww[j]));
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
    }
  }
}
__device__ __forceinline__ void pack8(void* p, int dtype, const float* v) {
  if (dtype == RB_F32) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    return;
  }
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    w[j] = dtype == RB_BF16 ? pack_bf16x2(v[2 * j], v[2 * j + 1]) : pack_f16x2(v[2 * j], v[2 * j + 1]);
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ void store_as(void* p, int dtype, int64_t i, float v) {
  if (dtype == RB_F32) {
    reinterpret_cast<float*>(p)[i] = v;
  } else if (dtype == RB_BF16) {
    reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  } else {
    reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
  }
}

// a lane's V values of row t of a [T, E] matrix (row pitch ld), `fill` where there is none
template <int L, int V, bool VEC>
__device__ __forceinline__ void load_row(const void* p, int dtype, int64_t ld, int64_t t, bool live, int E, int sl,
                                         float fill, float* v) {
  if constexpr (VEC) {
    const char* row = static_cast<const char*>(p) + t * ld * (dtype == RB_F32 ? 4 : 2);
#pragma unroll
    for (int j = 0; j < V / 8; ++j) {
      const int e = elem<L, true>(sl, 8 * j);
      if (live && e < E) {
        unpack8(row + (int64_t)e * (dtype == RB_F32 ? 4 : 2), dtype, v + 8 * j);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[8 * j + i] = fill;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = elem<L, false>(sl, i);
      v[i] = live && e < E ? load_as_f32(p, dtype, t * ld + e) : fill;
    }
  }
}
template <int L, int V, bool VEC>
__device__ __forceinline__ void store_row(void* p, int dtype, int64_t t, int E, int sl, const float* v) {
  if constexpr (VEC) {
    char* row = static_cast<char*>(p) + t * (int64_t)E * (dtype == RB_F32 ? 4 : 2);
#pragma unroll
    for (int j = 0; j < V / 8; ++j) {
      const int e = elem<L, true>(sl, 8 * j);
      if (e < E) pack8(row + (int64_t)e * (dtype == RB_F32 ? 4 : 2), dtype, v + 8 * j);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = elem<L, false>(sl, i);
      if (e < E) store_as(p, dtype, t * (int64_t)E + e, v[i]);
    }
  }
}

// a lane's values in a row of shared memory, and back
template <int L, int V, bool VEC>
__device__ __forceinline__ void put_row(float* row, int sl, const float* v) {
#pragma unroll
  for (int i = 0; i < V; i += VEC ? 4 : 1) {
    if constexpr (VEC)
      *reinterpret_cast<float4*>(row + elem<L, VEC>(sl, i)) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    else
      row[elem<L, VEC>(sl, i)] = v[i];
  }
}

// a lane's logits, -inf where masked or where there is none; whether the warp has such
template <int L, int V, bool VEC>
__device__ __forceinline__ bool load_logits(const void* p, int dtype, int64_t ld, int64_t t, bool live, int E, int sl,
                                            float lowest, float* l) {
  load_row<L, V, VEC>(p, dtype, ld, t, live, E, sl, -INFINITY, l);
  float low = l[0];
#pragma unroll
  for (int i = 1; i < V; ++i) low = fminf(low, l[i]);
  const bool some = __any_sync(kAll, low <= lowest);
  if (some) {
#pragma unroll
    for (int i = 0; i < V; ++i) l[i] = l[i] <= lowest ? -INFINITY : l[i];
  }
  return some;
}

// scores of a lane's logits: softmax over the token's unmasked logits, or sigmoid; 0 where masked.
// Returns a bound of the scores.
template <int L, int V>
__device__ __forceinline__ float scores(const float* l, int kind, float* s) {
  if (kind == kSigmoid) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float e = expf(-fabsf(l[i]));  // at most 1: no overflow, and small scores keep their precision
      s[i] = __fdividef(l[i] < 0.0f ? e : 1.0f, 1.0f + e);
    }
    return 1.0f;
  }
  float m = l[0];
#pragma unroll
  for (int i = 1; i < V; ++i) m = fmaxf(m, l[i]);
  m = sub_max<L>(m);
  if (m == -INFINITY) m = 0.0f;  // a token without experts: all scores 0
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    s[i] = expf(l[i] - m);
    sum += s[i];
  }
  sum = sub_sum<L>(sum);
  const float r = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
#pragma unroll
  for (int i = 0; i < V; ++i) s[i] *= r;
  return r;
}

// the pairs (i, j), i < j, of a sorting network of V values: odd-even merges of sorted halves (Batcher)
template <int V, typename F>
__device__ __forceinline__ void sort_network(F&& order) {
#pragma unroll
  for (int p = 1; p < V; p <<= 1) {
#pragma unroll
    for (int q = p; q >= 1; q >>= 1) {
#pragma unroll
      for (int j = q % p; j + q < V; j += 2 * q) {
#pragma unroll
        for (int i = 0; i < q; ++i) {
          if (i + j + q < V && (i + j) / (2 * p) == (i + j + q) / (2 * p)) order(i + j, i + j + q);
        }
      }
    }
  }
}

// an expert's exact choice value: by_logit, or (z = the sum of exp(l - m)) its score and bias
__device__ __forceinline__ double exact_value(const Params& p, float l, int e, double m, double z) {
  if (l <= p.lowest) return -INFINITY;  // also of a logit read as it is
  if (p.by_logit) return (double)l;
  const double v = p.kind == kSoftmax ? exp((double)l - m) / z : 1.0 / (1.0 + exp(-(double)l));
  return p.bias != nullptr ? v + (double)p.bias[e] : v;
}

// the softmax's maximum and sum in fp64
template <int L, int V>
__device__ __forceinline__ void exact_softmax(const float* l, double& m, double& z) {
  float top = l[0];
#pragma unroll
  for (int i = 1; i < V; ++i) top = fmaxf(top, l[i]);
  top = sub_max<L>(top);
  m = top == -INFINITY ? 0.0 : (double)top;
  z = 0.0;
#pragma unroll
  for (int i = 0; i < V; ++i) z += exp((double)l[i] - m);
  z = sub_sum<L>(z);
}

// The choice in fp64, for the tokens of a warp whose fp32 order is in doubt at
// more than single pairs.  `c` and `gv` are the sub-warp's scratch, `picks` its k
// chosen experts.
template <int L, int V, bool VEC>
__device__ __noinline__ void choose_exact(const Params& p, int64_t t, int lane, double* c, unsigned long long* gv,
                                          int* picks) {
  const int sl = lane % L;
  float l[V];
  load_logits<L, V, VEC>(p.logits, p.dtype, p.ld, t, t < p.T, p.E, sl, p.lowest, l);
  double m = 0.0, z = 1.0;
  if (p.kind == kSoftmax && !p.by_logit) exact_softmax<L, V>(l, m, z);
  unsigned long long key[V];
  int id[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = elem<L, VEC>(sl, i);
    id[i] = e;
    key[i] = 0;
    if (e < p.E) {
      c[e] = exact_value(p, l[i], e, m, z);
      key[i] = order64(c[e]);
    }
  }
  if (p.groups > 1) {
    __syncwarp();
    for (int g = sl; g < p.groups; g += L) {
      unsigned long long a = 0, b = 0;
      int j = g % p.gsize;
      for (int n = 0; n < p.gsize; ++n) {
        const unsigned long long o = order64(c[g * p.gsize + j]);
        b = max(b, min(a, o));
        a = max(a, o);
        if (++j == p.gsize) j = 0;
      }
      gv[g] = order64(p.group_top == 2 && p.gsize > 1 ? unorder64(a) + unorder64(b) : unorder64(a));
    }
    __syncwarp();
    for (int g = sl; g < p.groups; g += L) {
      int better = 0;
      for (int q = 0; q < p.groups; ++q) better += gv[q] > gv[g] || (gv[q] == gv[g] && q < g);
      c[g] = better < p.topk_groups ? 1.0 : 0.0;  // the choice values are in the keys
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (id[i] < p.E && c[id[i] / p.gsize] == 0.0) key[i] = 0;
  }
  sort_network<V>([&](int i, int j) {
    const bool swap = key[j] > key[i] || (key[j] == key[i] && id[j] < id[i]);
    const unsigned long long ki = key[i];
    const int di = id[i];
    key[i] = swap ? key[j] : ki;
    id[i] = swap ? id[j] : di;
    key[j] = swap ? ki : key[j];
    id[j] = swap ? di : id[j];
  });
  for (int r = 0; r < p.k; ++r) {
    const uint32_t hi = (uint32_t)(key[0] >> 32), lo = (uint32_t)key[0];
    const bool top = hi == sub_umax<L>(hi);
    const uint32_t best_lo = sub_umax<L>(top ? lo : 0u);  // all lanes take part, whatever `top` says
    const bool tied = top && lo == best_lo;
    const int e = (int)sub_umin<L>(tied ? (uint32_t)id[0] : (uint32_t)kMaxExperts);
    if (tied && id[0] == e) {
      picks[r] = e;
#pragma unroll
      for (int i = 0; i + 1 < V; ++i) {
        key[i] = key[i + 1];
        id[i] = id[i + 1];
      }
      key[V - 1] = 0;
    }
  }
  __syncwarp();
}

// GUARD: the choice is by fp32 values (scores, with a bias or in sums, or fp32
// logits: `by_logit`) whose order may be in doubt; else by 16-bit logits.
template <int L, int V, bool VEC, bool GUARD>
__global__ void __launch_bounds__(kThreads) route_topk_kernel(const __grid_constant__ Params p) {
  constexpr int kTok = 32 / L;  // tokens of a warp
  constexpr int kRow = L * V;   // experts that a token has room for
  constexpr int kPicks = kRow < kMaxK ? kRow : kMaxK;
  // among equal choice values the words' order is the indices': the place in the lane counts in full where a
  // lane's values lie L apart; within a run of eight it comes after the lane
  constexpr uint32_t kLow = V - 1, kCompare = VEC ? ~7u : ~0u;
  __shared__ __align__(16) float s_score[kWarps][kTok][kRow];
  __shared__ int s_pick[kWarps][kTok][kPicks + 2];
  __shared__ uint2 s_next[kWarps][kTok][kPicks + 2];
  __shared__ double s_exact[GUARD ? kWarps : 1][GUARD ? kTok : 1][GUARD ? kRow : 1];
  __shared__ double s_group[kWarps][kTok][kRow];  // groups' values, beside the choice values while those are fp32
  __shared__ int s_count[kMaxExperts];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / L, sl = lane % L;
  const int64_t t0 = ((int64_t)blockIdx.x * kWarps + warp) * kTok;
  const int64_t t = t0 + sub;
  const bool live = t < p.T;
  if (p.counts != nullptr) {
    for (int e = threadIdx.x; e < p.E; e += kThreads) s_count[e] = 0;
    __syncthreads();
  }

  float l[V], s[V];
  const bool masked = load_logits<L, V, VEC>(p.logits, p.dtype, p.ld, t, live, p.E, sl, p.lowest, l);
  const float most = scores<L, V>(l, p.kind, s);
  if (p.probs != nullptr && live) store_row<L, V, VEC>(p.probs, p.score_dtype, t, p.E, sl, s);
  put_row<L, V, VEC>(s_score[warp][sub], sl, s);

  // choice values; an index past the experts has -inf and comes after every expert
  float c[V];
  float mag = 0.0f;  // what the errors of the token's choice values are relative to
#pragma unroll
  for (int i = 0; i < V; ++i) c[i] = l[i];
  if constexpr (GUARD) {
    if (!p.by_logit) {
      float b[V];
      load_row<L, V, VEC>(p.bias, RB_F32, 0, 0, p.bias != nullptr, p.E, sl, 0.0f, b);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        c[i] = s[i] + b[i];
        mag = fmaxf(mag, fabsf(b[i]));
      }
      mag += most;
      if (masked) {
#pragma unroll
        for (int i = 0; i < V; ++i) c[i] = l[i] == -INFINITY ? -INFINITY : c[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) mag = fmaxf(mag, masked && l[i] == -INFINITY ? 0.0f : fabsf(l[i]));
    }
  }
  uint32_t w[V];
#pragma unroll
  for (int i = 0; i < V; ++i) w[i] = order32(c[i]);
  // fp32 errors of a choice value, in units u = 2^-24 of the token's largest |score| + |bias|.  Softmax: l -
  // max and its exp x + 2 where the score is e^-x of the largest, the sum 21 additions and its terms' own
  // errors (at most 8), reciprocal and product 2, the bias added 1: at most 34.  Sigmoid: exp 2, 1 + that 1,
  // the quotient 4, the bias 1: 8.  A word's dropped bits: 2 V.  Values are in doubt within twice the sum; a
  // group's value is two of them added.
  bool doubt = false;
  float eps = 0.0f, eps_group = 0.0f;
  if constexpr (GUARD) {
    const float base = p.by_logit ? 0.0f : p.kind == kSoftmax ? 34.0f : 8.0f;
    mag = sub_max<L>(mag) * 0x1p-24f;
    eps = 2.0f * (base + 2.0f * V) * mag;
    eps_group = 2.0f * (2.0f * base + 1.0f) * mag;
  }

  if (p.groups > 1) {
    const int gl = p.gsize >> 3;  // lanes of a group, where each run of eight values is of one group
    if (VEC && (p.gsize & 7) == 0 && (gl & (gl - 1)) == 0 && gl <= L) {
      constexpr int kRuns = V / 8;
      uint32_t ov[kRuns];
      float val[kRuns];
      int better[kRuns];
#pragma unroll
      for (int n = 0; n < kRuns; ++n) {
        uint32_t a = 0, b = 0;
#pragma unroll
        for (int i = 8 * n; i < 8 * n + 8; ++i) {
          b = max(b, min(a, w[i]));
          a = max(a, w[i]);
        }
        for (int o = 1; o < gl; o <<= 1) {
          const uint32_t a2 = __shfl_xor_sync(kAll, a, o), b2 = __shfl_xor_sync(kAll, b, o);
          b = max(min(a, a2), max(b, b2));
          a = max(a, a2);
        }
        val[n] = p.group_top == 2 ? unorder32(a) + unorder32(b) : unorder32(a);
        ov[n] = order32(val[n]);
        better[n] = 0;
      }
      const int per = L / gl;  // groups of a run over all lanes
      const int g = sl / gl;   // this lane's group in the first run
#pragma unroll
      for (int m = 0; m < kRuns; ++m) {
        for (int q = 0; q < per && m * per + q < p.groups; ++q) {
          const uint32_t ou = __shfl_sync(kAll, ov[m], sub * L + q * gl);
#pragma unroll
          for (int n = 0; n < kRuns; ++n)
            better[n] += ou > ov[n] || (ou == ov[n] && m * per + q < n * per + g);
        }
      }
      float kept = INFINITY, dropped = -INFINITY;
#pragma unroll
      for (int n = 0; n < kRuns; ++n) {
        if (n * per + g >= p.groups) continue;
        if (better[n] >= p.topk_groups) {
          dropped = fmaxf(dropped, val[n]);
#pragma unroll
          for (int i = 8 * n; i < 8 * n + 8; ++i) w[i] = 0;
        } else {
          kept = fminf(kept, val[n]);
        }
      }
      if constexpr (GUARD) {
        kept = -sub_max<L>(-kept);
        dropped = sub_max<L>(dropped);
        doubt = kept - dropped <= eps_group && kept > -INFINITY;
      }
    } else {
      float* cc = reinterpret_cast<float*>(s_group[warp][sub]);
      float* gv = cc + kRow;
#pragma unroll
      for (int i = 0; i < V; ++i) cc[elem<L, VEC>(sl, i)] = c[i];
      __syncwarp();
      for (int g = sl; g < p.groups; g += L) {
        uint32_t a = 0, b = 0;
        int j = g % p.gsize;  // lanes start at different banks
        for (int n = 0; n < p.gsize; ++n) {
          const uint32_t o = order32(cc[g * p.gsize + j]);
          b = max(b, min(a, o));
          a = max(a, o);
          if (++j == p.gsize) j = 0;
        }
        gv[g] = p.group_top == 2 && p.gsize > 1 ? unorder32(a) + unorder32(b) : unorder32(a);
      }
      __syncwarp();
      // a group stays when fewer than topk_groups others come before it; choice values are no longer needed
      // and their room takes 1 for a group that stays, 0 for one that goes
      for (int g = sl; g < p.groups; g += L) {
        const float v = gv[g];
        const uint32_t o = order32(v);
        int better = 0;
        float next = -INFINITY, prev = INFINITY;  // the nearest values after and before this group
        for (int q = 0; q < p.groups; ++q) {
          const uint32_t ou = order32(gv[q]);
          const bool before = ou > o || (ou == o && q < g);
          better += before;
          if (before) prev = fminf(prev, gv[q]);
          else if (q != g) next = fmaxf(next, gv[q]);
        }
        cc[g] = better < p.topk_groups ? 1.0f : 0.0f;
        if constexpr (GUARD) {
          if (better == p.topk_groups) doubt = prev - v <= eps_group && prev > -INFINITY;
        }
      }
      __syncwarp();
      const float inv = 1.0f / (float)p.gsize;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        // e / gsize: e + 1/2 is at least 1/2 from a multiple of gsize, far more than the product's rounding
        const int e = elem<L, VEC>(sl, i);
        if (e < p.E && cc[(int)(((float)e + 0.5f) * inv)] == 0.0f) w[i] = 0;
      }
    }
  }

  // a word: the value's leading bits, and the place in the lane (at most kLow: an expert of a dropped group)
#pragma unroll
  for (int i = 0; i < V; ++i) w[i] = (w[i] & ~kLow) | (kLow - (uint32_t)i);
  sort_network<V>([&](int i, int j) {
    const uint32_t a = w[i], b = w[j];
    w[i] = max(a, b);
    w[j] = min(a, b);
  });
  constexpr unsigned kSub = L == 32 ? kAll : (1u << L) - 1u;
  const int rounds = GUARD ? p.k + 2 : p.k;  // the chosen, and the two that follow
  for (int r = 0; r < rounds; ++r) {
    const uint32_t head = w[0] & kCompare;
    bool won = head == sub_umax<L>(head);
    if constexpr (L > 1) {
      const unsigned with = __ballot_sync(kAll, won) & (kSub << (sub * L));
      won = lane == __ffs(with) - 1;
    }
    if (won) {
      s_next[warp][sub][r] = make_uint2(w[0], (uint32_t)sl);
#pragma unroll
      for (int i = 0; i + 1 < V; ++i) w[i] = w[i + 1];
      w[V - 1] = 0;
    }
  }
  __syncwarp();
  for (int r = sl; r < rounds; r += L) {
    const uint2 n = s_next[warp][sub][r];
    s_pick[warp][sub][r] = elem<L, VEC>((int)n.y, (int)(kLow - (n.x & kLow)));
  }
  __syncwarp();
  if constexpr (GUARD) {
    // Place r of the order is near place r - 1 when fp32 cannot tell which comes first; equal logits under
    // equal biases are a tie in any arithmetic, and stand in the order of their indices.  A near pair whose
    // neighbours are not near is settled in fp64 by one lane, anything else by the whole order in fp64.
    const uint2* next = s_next[warp][sub];
    auto near = [&](int r) {
      if (r < 1 || r >= rounds || next[r].x <= kLow) return false;
      const float v = unorder32(next[r].x & ~kLow);
      return unorder32(next[r - 1].x & ~kLow) - v <= eps && v > -INFINITY;
    };
    uint32_t pairs = 0;  // of this lane's places sl, sl + L, ...
    for (int r = sl, n = 0; r <= p.k; r += L, ++n) {
      if (live && near(r)) {
        const int e = s_pick[warp][sub][r], f = s_pick[warp][sub][r - 1];
        const bool same =
            load_as_f32(p.logits, p.dtype, t * p.ld + e) == load_as_f32(p.logits, p.dtype, t * p.ld + f) &&
            (p.bias == nullptr || p.bias[e] == p.bias[f]);
        if (!same) {
          if (near(r - 1) || near(r + 1)) doubt = true;
          else pairs |= 1u << n;
        }
      }
    }
    if (__any_sync(kAll, pairs != 0)) {
      double m = 0.0, z = 1.0;
      if (p.kind == kSoftmax && !p.by_logit) exact_softmax<L, V>(l, m, z);
      for (int r = sl, n = 0; r <= p.k; r += L, ++n) {
        if (pairs >> n & 1) {
          const int e = s_pick[warp][sub][r], f = s_pick[warp][sub][r - 1];
          const double ve = exact_value(p, load_as_f32(p.logits, p.dtype, t * p.ld + e), e, m, z);
          const double vf = exact_value(p, load_as_f32(p.logits, p.dtype, t * p.ld + f), f, m, z);
          if (ve > vf || (ve == vf && e < f)) {
            s_pick[warp][sub][r - 1] = e;
            s_pick[warp][sub][r] = f;
          }
        }
      }
      __syncwarp();
    }
    if (__any_sync(kAll, doubt && live)) {
      choose_exact<L, V, VEC>(p, t, lane, s_exact[warp][sub],
                              reinterpret_cast<unsigned long long*>(s_group[warp][sub]), s_pick[warp][sub]);
    }
  }

  // weights of the chosen; the warp's outputs are one run of kTok * k
  float total = 0.0f;
  for (int j = sl; j < p.k; j += L) total += s_score[warp][sub][s_pick[warp][sub][j]];
  total = sub_sum<L>(total);
  const float f = p.renorm ? (total == 0.0f ? 0.0f : __fdiv_rn(p.scale, total)) : p.scale;
  const int64_t left = p.T - t0;
  const int n = (int)(left < kTok ? (left < 0 ? 0 : left) : kTok) * p.k;
  for (int q0 = 0; q0 < kTok * p.k; q0 += 32) {
    const int q = q0 + lane;
    const int qs = (int)(((uint32_t)q * p.k_inv) >> 16), j = q - qs * p.k;
    const float ff = __shfl_sync(kAll, f, qs < kTok ? qs * L : 0);
    if (q < n) {
      const int e = s_pick[warp][qs][j];
      const int64_t o = t0 * p.k + q;
      if (p.idx64)
        reinterpret_cast<int64_t*>(p.idx)[o] = e;
      else
        reinterpret_cast<int32_t*>(p.idx)[o] = e;
      store_as(p.score, p.score_dtype, o, s_score[warp][qs][e] * ff);
      if (p.counts != nullptr) atomicAdd(&s_count[e], 1);
    }
  }
  if (p.counts != nullptr) {
    __syncthreads();
    for (int e = threadIdx.x; e < p.E; e += kThreads)
      if (s_count[e] != 0) atomicAdd(p.counts + e, s_count[e]);
  }
}

__device__ __forceinline__ int chosen_expert(const BwdParams& p, int64_t t, int j) {
  const int64_t e = p.idx64 ? reinterpret_cast<const int64_t*>(p.idx)[t * p.k + j]
                            : (int64_t) reinterpret_cast<const int32_t*>(p.idx)[t * p.k + j];
  return e >= 0 && e < p.E ? (int)e : -1;
}

// dl of a token's logits: with g = grad_score * scale at the chosen experts,
// ds = g, or (g - sum(g w)) / total where the weights w were renormalised;
// ds += grad_probs; dl = s (ds - sum(ds s)) or ds s (1 - s).  Masked logits get 0.
template <int L, int V, bool VEC>
__global__ void __launch_bounds__(kThreads) route_backward_kernel(const __grid_constant__ BwdParams p) {
  constexpr int kTok = 32 / L;
  __shared__ __align__(16) float s_row[kWarps][kTok][L * V];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / L, sl = lane % L;
  const int64_t t = ((int64_t)blockIdx.x * kWarps + warp) * kTok + sub;
  const bool live = t < p.T;
  float l[V], s[V], ds[V];
  const bool masked = load_logits<L, V, VEC>(p.logits, p.dtype, p.ld, t, live, p.E, sl, p.lowest, l);
  load_row<L, V, VEC>(p.grad_probs, p.probs_dtype, p.E, t, p.grad_probs != nullptr && live, p.E, sl, 0.0f, ds);
  scores<L, V>(l, p.kind, s);
  if (p.grad_score != nullptr) {
    // the chosen experts' gradients, a lane for each, go to their places through shared memory
    float* row = s_row[warp][sub];
    put_row<L, V, VEC>(row, sl, s);
    __syncwarp();
    float total = 0.0f, dot = 0.0f;
    if (p.renorm) {
      for (int j = sl; live && j < p.k; j += L) {
        const int e = chosen_expert(p, t, j);
        if (e < 0) continue;
        total += row[e];
        dot += load_as_f32(p.grad_score, p.grad_dtype, t * p.k + j) * row[e];
      }
      total = sub_sum<L>(total);
      dot = sub_sum<L>(dot);
    }
    const float r = !p.renorm ? 1.0f : total == 0.0f ? 0.0f : __fdiv_rn(1.0f, total);
    const float less = p.renorm ? dot * r : 0.0f;
    __syncwarp();
    put_row<L, V, VEC>(row, sl, ds);
    __syncwarp();
    for (int j = sl; live && j < p.k; j += L) {
      const int e = chosen_expert(p, t, j);
      const float d = load_as_f32(p.grad_score, p.grad_dtype, t * p.k + j);
      if (e >= 0) atomicAdd(row + e, (d - less) * r * p.scale);  // an expert comes once in a row: no order to keep
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < V; ++i) ds[i] = row[elem<L, VEC>(sl, i)];
  }
  if (masked) {  // whatever gradient reaches a masked expert
#pragma unroll
    for (int i = 0; i < V; ++i) ds[i] = l[i] == -INFINITY ? 0.0f : ds[i];
  }
  if (p.kind == kSigmoid) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float e = expf(-fabsf(l[i])), q = __fdividef(e, 1.0f + e);  // the smaller of s and 1 - s, to its own last bits
      s[i] = ds[i] * q * (1.0f - q);
    }
  } else {
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) dot += ds[i] * s[i];
    dot = sub_sum<L>(dot);
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] *= ds[i] - dot;
  }
  if (live) store_row<L, V, VEC>(p.grad_logits, p.out_dtype, t, p.E, sl, s);
}

static float lowest_of(int dtype) {
  return dtype == RB_F16 ? -65504.0f : dtype == RB_BF16 ? -0x1.fep127f : -0x1.fffffep127f;
}

template <int L>
static unsigned blocks_for(int64_t T) {
  const int64_t per = (int64_t)kWarps * (32 / L);
  return (unsigned)((T + per - 1) / per);
}

template <int L, int V>
static void launch_fwd(const Params& p, bool vec, bool guard, cudaStream_t st) {
  const unsigned g = blocks_for<L>(p.T);
  if (vec) {
    if (guard) route_topk_kernel<L, V, true, true><<<g, kThreads, 0, st>>>(p);
    else route_topk_kernel<L, V, true, false><<<g, kThreads, 0, st>>>(p);
  } else {
    if (guard) route_topk_kernel<L, V, false, true><<<g, kThreads, 0, st>>>(p);
    else route_topk_kernel<L, V, false, false><<<g, kThreads, 0, st>>>(p);
  }
}

template <int L, int V>
static void launch_bwd(const BwdParams& p, bool vec, cudaStream_t st) {
  const unsigned g = blocks_for<L>(p.T);
  if (vec) route_backward_kernel<L, V, true><<<g, kThreads, 0, st>>>(p);
  else route_backward_kernel<L, V, false><<<g, kThreads, 0, st>>>(p);
}

static bool is_float(int dt) { return dt == RB_F32 || dt == RB_BF16 || dt == RB_F16; }

// a row of E values from `p` in steps of `ld` can be moved in 16-byte pieces of 8 (or 2 x 4) values
static bool rows_of_8(const void* p, int dtype, int64_t ld, int E) {
  return p == nullptr || (E % 8 == 0 && aligned(p, 16) && (ld * dtype_size(dtype)) % 16 == 0);
}

}  // namespace route
}  // namespace rb

using namespace rb;

extern "C" int rb_route_topk(const void* logits, int dtype, int64_t ld, int64_t T, int E, const void* bias, int k,
                             int score_kind, int groups, int topk_groups, int group_top, int renormalize, float scale,
                             void* idx, int idx_dtype, void* score, int score_dtype, void* probs, void* counts,
                             void* stream) {
  using namespace rb::route;
  if (T < 0 || E <= 0) return fail(RB_ERR_VALUE, "negative or empty routing shape");
  if (E > route::kMaxExperts) return fail(RB_ERR_UNSUPPORTED, "more than %d experts", route::kMaxExperts);
  if (!is_float(dtype) || !is_float(score_dtype))
    return fail(RB_ERR_UNSUPPORTED, "logits and scores are fp32, bf16 or fp16");
  if (idx_dtype != RB_I64 && idx_dtype != RB_I32) return fail(RB_ERR_VALUE, "idx must be int64 or int32");
  if (score_kind != kSoftmax && score_kind != kSigmoid) return fail(RB_ERR_VALUE, "unknown score function");
  if (groups <= 0 || E % groups != 0) return fail(RB_ERR_VALUE, "%d experts do not split into %d groups", E, groups);
  if (topk_groups <= 0 || topk_groups > groups) return fail(RB_ERR_VALUE, "topk_groups outside [1, groups]");
  if (group_top != 1 && group_top != 2) return fail(RB_ERR_VALUE, "group_top must be 1 or 2");
  if (k <= 0 || k > kMaxK || k > E / groups * topk_groups)
    return fail(RB_ERR_VALUE, "k must be in [1, %d] and at most the experts of the chosen groups", kMaxK);
  if (ld < E) return fail(RB_ERR_VALUE, "leading dimension smaller than the row");
  if (T > (int64_t)1 << 31) return fail(RB_ERR_UNSUPPORTED, "more than 2^31 tokens");
  if (T > 0 && (logits == nullptr || idx == nullptr || score == nullptr)) return fail(RB_ERR_VALUE, "null operand");
  if (!device_is_sm100()) return fail(RB_ERR_DEVICE, "rb_route_topk needs an sm_100 (B200) device");
  cudaStream_t st = (cudaStream_t)stream;
  if (counts != nullptr) {
    const int rc = check_cuda(cudaMemsetAsync(counts, 0, (size_t)E * 4, st), "zeroing the expert counts");
    if (rc) return rc;
  }
  if (T == 0) return RB_OK;
  Params p{};
  p.logits = logits;
  p.bias = static_cast<const float*>(bias);
  p.idx = idx;
  p.score = score;
  p.probs = probs;
  p.counts = static_cast<int32_t*>(counts);
  p.ld = ld;
  p.T = T;
  p.scale = scale;
  p.lowest = lowest_of(dtype);
  p.dtype = dtype;
  p.E = E;
  p.k = k;
  p.kind = score_kind;
  p.groups = topk_groups == groups ? 1 : groups;  // all groups stay: no choice among them
  p.gsize = E / groups;
  p.topk_groups = topk_groups;
  p.group_top = group_top;
  p.renorm = renormalize != 0;
  p.idx64 = idx_dtype == RB_I64;
  p.score_dtype = score_dtype;
  p.k_inv = (uint32_t)((65536 + k - 1) / k);
  p.by_logit = bias == nullptr && !(p.groups > 1 && group_top == 2 && p.gsize > 1);
  const bool guard = !p.by_logit || dtype == RB_F32;
  const bool vec = rows_of_8(logits, dtype, ld, E) && rows_of_8(probs, score_dtype, E, E) &&
                   rows_of_8(bias, RB_F32, E, E);
  if (E <= 8) launch_fwd<1, 8>(p, vec, guard, st);
  else if (E <= 16) launch_fwd<2, 8>(p, vec, guard, st);
  else if (E <= 32) launch_fwd<4, 8>(p, vec, guard, st);
  else if (E <= 64) launch_fwd<8, 8>(p, vec, guard, st);
  else if (E <= 128) launch_fwd<16, 8>(p, vec, guard, st);
  else if (E <= 256) launch_fwd<32, 8>(p, vec, guard, st);
  else launch_fwd<32, 16>(p, vec, guard, st);
  return check_cuda(cudaGetLastError(), "route_topk_kernel launch");
}

extern "C" int rb_route_topk_backward(const void* logits, int dtype, int64_t ld, int64_t T, int E, const void* idx,
                                      int idx_dtype, int k, const void* grad_score, int grad_dtype,
                                      const void* grad_probs, int probs_dtype, int score_kind, int renormalize,
                                      float scale, void* grad_logits, int out_dtype, void* stream) {
  using namespace rb::route;
  if (T < 0 || E <= 0) return fail(RB_ERR_VALUE, "negative or empty routing shape");
  if (E > route::kMaxExperts) return fail(RB_ERR_UNSUPPORTED, "more than %d experts", route::kMaxExperts);
  if (!is_float(dtype) || !is_float(out_dtype) || (grad_score != nullptr && !is_float(grad_dtype)) ||
      (grad_probs != nullptr && !is_float(probs_dtype)))
    return fail(RB_ERR_UNSUPPORTED, "logits and gradients are fp32, bf16 or fp16");
  if (idx_dtype != RB_I64 && idx_dtype != RB_I32) return fail(RB_ERR_VALUE, "idx must be int64 or int32");
  if (score_kind != kSoftmax && score_kind != kSigmoid) return fail(RB_ERR_VALUE, "unknown score function");
  if (k <= 0 || k > kMaxK || k > E) return fail(RB_ERR_VALUE, "k must be in [1, %d] and at most the experts", kMaxK);
  if (ld < E) return fail(RB_ERR_VALUE, "leading dimension smaller than the row");
  if (T > (int64_t)1 << 31) return fail(RB_ERR_UNSUPPORTED, "more than 2^31 tokens");
  if (T > 0 && (logits == nullptr || grad_logits == nullptr || (grad_score != nullptr && idx == nullptr)))
    return fail(RB_ERR_VALUE, "null operand");
  if (!device_is_sm100()) return fail(RB_ERR_DEVICE, "rb_route_topk_backward needs an sm_100 (B200) device");
  if (T == 0) return RB_OK;
  BwdParams p{};
  p.logits = logits;
  p.idx = idx;
  p.grad_score = grad_score;
  p.grad_probs = grad_probs;
  p.grad_logits = grad_logits;
  p.ld = ld;
  p.T = T;
  p.scale = scale;
  p.lowest = lowest_of(dtype);
  p.dtype = dtype;
  p.E = E;
  p.k = k;
  p.kind = score_kind;
  p.renorm = renormalize != 0;
  p.idx64 = idx_dtype == RB_I64;
  p.grad_dtype = grad_dtype;
  p.probs_dtype = probs_dtype;
  p.out_dtype = out_dtype;
  cudaStream_t st = (cudaStream_t)stream;
  const bool vec = rows_of_8(logits, dtype, ld, E) && rows_of_8(grad_probs, probs_dtype, E, E) &&
                   rows_of_8(grad_logits, out_dtype, E, E);
  if (E <= 8) launch_bwd<1, 8>(p, vec, st);
  else if (E <= 16) launch_bwd<2, 8>(p, vec, st);
  else if (E <= 32) launch_bwd<4, 8>(p, vec, st);
  else if (E <= 64) launch_bwd<8, 8>(p, vec, st);
  else if (E <= 128) launch_bwd<16, 8>(p, vec, st);
  else if (E <= 256) launch_bwd<32, 8>(p, vec, st);
  else launch_bwd<32, 16>(p, vec, st);
  return check_cuda(cudaGetLastError(), "route_backward_kernel launch");
}

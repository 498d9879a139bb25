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
//   * Without bias the scores rise with the logits, so the logits are compared
//     (bit for bit).  For 16-bit logits one 32-bit word holds the logit (the 19
//     leading bits of its order-preserving fp32 pattern; the other 13 carry
//     nothing for bf16 and fp16) and the index, so a round is one maximum.
//   * With a bias, or where a group's value is a sum of scores, fp32 values are
//     compared first.  Where two neighbours of the order (or the last kept and
//     the first dropped group) lie closer than the fp32 error bound, the warp's
//     tokens are decided again in fp64.
#include "common.cuh"

#include <type_traits>

namespace rb {
namespace route {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxExperts = 512;
constexpr int kMaxK = 32;
constexpr uint32_t kIdxMask = 8191;  // low bits of a packed 16-bit logit's word
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
  int dtype, E, k, kind, groups, gsize, topk_groups, group_top, renorm, idx64, score_dtype;
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
  const uint32_t u = __float_as_uint(v + 0.0f);  // -0 as +0
  if (v != v) return 0xffffffffu;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
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
__device__ __forceinline__ unsigned long long sub_umax(unsigned long long v) {
  if constexpr (L == 32) {
    const uint32_t hi = (uint32_t)(v >> 32);
    const uint32_t mh = __reduce_max_sync(kAll, hi);
    const uint32_t ml = __reduce_max_sync(kAll, hi == mh ? (uint32_t)v : 0u);
    return ((unsigned long long)mh << 32) | ml;
  } else {
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(kAll, v, o));
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

// scores of a lane's logits: softmax over the token's unmasked logits, or sigmoid; 0 where masked
template <int L, int V>
__device__ __forceinline__ void scores(const float* l, int kind, float lowest, float* s) {
  if (kind == kSigmoid) {
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = l[i] <= lowest ? 0.0f : __fdiv_rn(1.0f, 1.0f + expf(-l[i]));
    return;
  }
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (!(l[i] <= lowest)) m = fmaxf(m, l[i]);
  m = sub_max<L>(m);
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    s[i] = l[i] <= lowest ? 0.0f : expf(l[i] - m);
    sum += s[i];
  }
  sum = sub_sum<L>(sum);
  const float r = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
#pragma unroll
  for (int i = 0; i < V; ++i) s[i] *= r;
}

// The choice in fp64, for the tokens of a warp whose fp32 order is in doubt.
// `c` is the warp's scratch, `picks` the sub-warp's k chosen experts.
template <int L, int V, bool VEC>
__device__ __noinline__ void choose_exact(const Params& p, int64_t t, int sl, double* c, int* picks) {
  float l[V];
  load_row<L, V, VEC>(p.logits, p.dtype, p.ld, t, t < p.T, p.E, sl, -INFINITY, l);
  double s[V], m = -INFINITY, sum = 0.0;
  if (p.kind == kSoftmax) {
    for (int i = 0; i < V; ++i)
      if (!(l[i] <= p.lowest)) m = fmax(m, (double)l[i]);
    for (int o = L / 2; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(kAll, m, o));
    for (int i = 0; i < V; ++i) {
      s[i] = l[i] <= p.lowest ? 0.0 : exp((double)l[i] - m);
      sum += s[i];
    }
    sum = sub_sum<L>(sum);
  }
  unsigned long long key[V];
  for (int i = 0; i < V; ++i) {
    const int e = elem<L, VEC>(sl, i);
    if (e >= p.E) {
      key[i] = 0;
      continue;
    }
    double v = p.kind == kSoftmax ? s[i] / sum : 1.0 / (1.0 + exp(-(double)l[i]));
    if (p.bias != nullptr) v += (double)p.bias[e];
    if (l[i] <= p.lowest) v = -INFINITY;
    key[i] = order64(v);
    c[e] = v;
  }
  if (p.groups > 1) {
    __syncwarp();
    for (int i = 0; i < V; ++i) {
      const int e = elem<L, VEC>(sl, i);
      if (e >= p.E) continue;
      const int g = e / p.gsize;
      unsigned long long mine = 0;
      int better = 0;
      // every group's value, the own one first
      for (int q = -1; q < p.groups; ++q) {
        const int gg = q < 0 ? g : q;
        unsigned long long a = 0, b = 0;
        for (int j = 0; j < p.gsize; ++j) {
          const unsigned long long o = order64(c[gg * p.gsize + j]);
          if (o > a) {
            b = a;
            a = o;
          } else if (o > b) {
            b = o;
          }
        }
        const double v = p.group_top == 2 && p.gsize > 1 ? unorder64(a) + unorder64(b) : unorder64(a);
        const unsigned long long ov = order64(v);
        if (q < 0)
          mine = ov;
        else if (ov > mine || (ov == mine && gg < g))
          ++better;
      }
      if (better >= p.topk_groups) key[i] = 0;
    }
  }
  for (int r = 0; r < p.k; ++r) {
    unsigned long long best = 0;
    int be = kMaxExperts;
    for (int i = 0; i < V; ++i) {
      const int e = elem<L, VEC>(sl, i);
      if (key[i] > best || (key[i] == best && best != 0 && e < be)) {
        best = key[i];
        be = e;
      }
    }
    for (int o = L / 2; o > 0; o >>= 1) {
      const unsigned long long ob = __shfl_xor_sync(kAll, best, o);
      const int oe = __shfl_xor_sync(kAll, be, o);
      if (ob > best || (ob == best && oe < be)) {
        best = ob;
        be = oe;
      }
    }
    if (sl == 0) picks[r] = be;
    for (int i = 0; i < V; ++i)
      if (elem<L, VEC>(sl, i) == be) key[i] = 0;
  }
  __syncwarp();
}

// PACKED: the logits are 16-bit and their order is the choice's.  GUARD: the
// choice values are sums in fp32 whose order may be in doubt.
template <int L, int V, bool VEC, bool PACKED, bool GUARD>
__global__ void __launch_bounds__(kThreads) route_topk_kernel(const __grid_constant__ Params p) {
  constexpr int kTok = 32 / L;  // tokens of a warp
  constexpr int kRow = L * V;   // experts that a token has room for
  constexpr int kPicks = kRow < kMaxK ? kRow : kMaxK;
  using Word = typename std::conditional<PACKED, uint32_t, unsigned long long>::type;
  __shared__ float s_score[kWarps][kTok][kRow];
  __shared__ int s_pick[kWarps][kTok][kPicks];
  __shared__ double s_exact[GUARD ? kWarps : 1][GUARD ? kTok : 1][GUARD ? kRow : 1];
  __shared__ float s_choice[kWarps][kTok][kRow];
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
  load_row<L, V, VEC>(p.logits, p.dtype, p.ld, t, live, p.E, sl, -INFINITY, l);
  scores<L, V>(l, p.kind, p.lowest, s);
  if (p.probs != nullptr && live) store_row<L, V, VEC>(p.probs, p.score_dtype, t, p.E, sl, s);

  // choice values
  float c[V];
  float mag = 0.0f;  // the token's largest |score| + |bias|: what the fp32 errors are relative to
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = elem<L, VEC>(sl, i);
    s_score[warp][sub][e] = s[i];
    if constexpr (GUARD) {
      const float b = p.bias != nullptr && e < p.E ? __ldg(p.bias + e) : 0.0f;
      c[i] = s[i] + b;
      mag = fmaxf(mag, s[i] + fabsf(b));
    } else {
      c[i] = l[i];
    }
    if (l[i] <= p.lowest) c[i] = -INFINITY;
  }
  Word w[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = elem<L, VEC>(sl, i);
    const uint32_t o = order32(c[i]);
    if constexpr (PACKED) {
      w[i] = e < p.E ? (o & ~kIdxMask) | (kIdxMask - (uint32_t)e) : 0u;
    } else {
      w[i] = e < p.E ? ((unsigned long long)o << 32) | (0xffffffffu - (uint32_t)e) : 0ull;
    }
  }
  // fp32 errors of a choice value: the softmax's sum and quotient, expf (2 ulp)
  // of a rounded difference, the bias added -- under 2^-18 of `mag` for E <= 512
  bool doubt = false;
  float eps = 0.0f;
  if constexpr (GUARD) eps = sub_max<L>(mag) * 0x1p-17f;

  if (p.groups > 1) {
#pragma unroll
    for (int i = 0; i < V; ++i) s_choice[warp][sub][elem<L, VEC>(sl, i)] = c[i];
    __syncwarp();
    const float* cc = s_choice[warp][sub];
    float* gv = s_choice[warp][sub];  // group values replace the choice values below
    // a lane's groups: sl, sl + L, ...
    constexpr int kMine = V;  // groups <= E <= L * V
    float mine[kMine];
#pragma unroll
    for (int q = 0; q < kMine; ++q) {
      const int g = sl + q * L;
      mine[q] = 0.0f;
      if (g >= p.groups) continue;
      uint32_t a = 0, b = 0;
      int j = g % p.gsize;  // lanes start at different banks
      for (int n = 0; n < p.gsize; ++n) {
        const uint32_t o = order32(cc[g * p.gsize + j]);
        b = max(b, min(a, o));
        a = max(a, o);
        if (++j == p.gsize) j = 0;
      }
      mine[q] = p.group_top == 2 && p.gsize > 1 ? unorder32(a) + unorder32(b) : unorder32(a);
    }
    __syncwarp();
#pragma unroll
    for (int q = 0; q < kMine; ++q)
      if (sl + q * L < p.groups) gv[sl + q * L] = mine[q];
    __syncwarp();
    // a group stays when fewer than topk_groups others come before it
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = elem<L, VEC>(sl, i);
      if (e >= p.E) continue;
      const int g = e / p.gsize;
      const float v = gv[g];
      const uint32_t o = order32(v);
      int better = 0;
      for (int q = 0; q < p.groups; ++q) {
        const float u = gv[q];
        const uint32_t ou = order32(u);
        better += ou > o || (ou == o && q < g);
      }
      if (better >= p.topk_groups) w[i] = 0;
      if constexpr (GUARD) {
        if (better == p.topk_groups) {  // the first dropped group: any kept one as near as the errors?
          for (int q = 0; q < p.groups; ++q) {
            const float u = gv[q];
            const uint32_t ou = order32(u);
            if ((ou > o || (ou == o && q < g)) && u - v <= 2.0f * eps && u > -INFINITY) doubt = true;
          }
        }
      }
    }
  }

  float last = INFINITY;
  int last_e = -1;
  const int rounds = GUARD ? p.k + 1 : p.k;
  for (int r = 0; r < rounds; ++r) {
    Word best = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) best = max(best, w[i]);
    best = sub_umax<L>(best);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (w[i] == best) w[i] = 0;
    if constexpr (GUARD) {
      const float v = unorder32((uint32_t)((unsigned long long)best >> 32));
      const int e = (int)(0xffffffffu - (uint32_t)best);
      if (best != 0) {
        if (last - v <= eps && v > -INFINITY) {
          // equal logits under equal biases are a tie in any arithmetic
          bool same = false;
          if (last_e >= 0 && live) {
            same = load_as_f32(p.logits, p.dtype, t * p.ld + e) == load_as_f32(p.logits, p.dtype, t * p.ld + last_e) &&
                   (p.bias == nullptr || p.bias[e] == p.bias[last_e]);
          }
          if (!same) doubt = true;
        }
        last = v;
        last_e = e;
      }
    }
    if (r < p.k && sl == 0)
      s_pick[warp][sub][r] = PACKED ? (int)(kIdxMask - ((uint32_t)best & kIdxMask))
                                    : (int)(0xffffffffu - (uint32_t)best);
  }
  __syncwarp();
  if constexpr (GUARD) {
    if (__any_sync(kAll, doubt && live)) {
      choose_exact<L, V, VEC>(p, t, sl, s_exact[warp][sub], s_pick[warp][sub]);
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
    const int qs = q / p.k, j = q % p.k;
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

// dl of a token's logits: with g = grad_score * scale at the chosen experts,
// ds = g, or (g - sum(g w)) / total where the weights w were renormalised;
// ds += grad_probs; dl = s (ds - sum(ds s)) or ds s (1 - s).  Masked logits get 0.
template <int L, int V, bool VEC>
__global__ void __launch_bounds__(kThreads) route_backward_kernel(const __grid_constant__ BwdParams p) {
  constexpr int kTok = 32 / L;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane / L, sl = lane % L;
  const int64_t t = ((int64_t)blockIdx.x * kWarps + warp) * kTok + sub;
  const bool live = t < p.T;
  float l[V], s[V], ds[V];
  load_row<L, V, VEC>(p.logits, p.dtype, p.ld, t, live, p.E, sl, -INFINITY, l);
  if (p.grad_probs != nullptr) {
    load_row<L, V, VEC>(p.grad_probs, p.probs_dtype, p.E, t, live, p.E, sl, 0.0f, ds);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) ds[i] = 0.0f;
  }
  scores<L, V>(l, p.kind, p.lowest, s);
  if (p.grad_score != nullptr) {
    float g[V];
    uint32_t chosen = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) g[i] = 0.0f;
    for (int j = 0; j < p.k; ++j) {
      int64_t e = -1;
      float d = 0.0f;
      if (live) {
        e = p.idx64 ? reinterpret_cast<const int64_t*>(p.idx)[t * p.k + j]
                    : (int64_t) reinterpret_cast<const int32_t*>(p.idx)[t * p.k + j];
        d = load_as_f32(p.grad_score, p.grad_dtype, t * p.k + j) * p.scale;
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (elem<L, VEC>(sl, i) == e) {
          g[i] += d;
          chosen |= 1u << i;
        }
      }
    }
    float total = 0.0f, dot = 0.0f;
    if (p.renorm) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (chosen >> i & 1) total += s[i];
        dot += g[i] * s[i];
      }
      total = sub_sum<L>(total);
      dot = sub_sum<L>(dot);
      const float r = total == 0.0f ? 0.0f : __fdiv_rn(1.0f, total);
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (chosen >> i & 1) ds[i] += (g[i] - dot * r) * r;
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) ds[i] += g[i];
    }
  }
  if (p.kind == kSigmoid) {
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = l[i] <= p.lowest ? 0.0f : ds[i] * s[i] * (1.0f - s[i]);
  } else {
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (!(l[i] <= p.lowest)) dot += ds[i] * s[i];
    dot = sub_sum<L>(dot);
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = l[i] <= p.lowest ? 0.0f : s[i] * (ds[i] - dot);
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
static void launch_fwd(const Params& p, bool vec, bool packed, bool guard, cudaStream_t st) {
  const unsigned g = blocks_for<L>(p.T);
  if (vec) {
    if (guard) route_topk_kernel<L, V, true, false, true><<<g, kThreads, 0, st>>>(p);
    else if (packed) route_topk_kernel<L, V, true, true, false><<<g, kThreads, 0, st>>>(p);
    else route_topk_kernel<L, V, true, false, false><<<g, kThreads, 0, st>>>(p);
  } else {
    if (guard) route_topk_kernel<L, V, false, false, true><<<g, kThreads, 0, st>>>(p);
    else if (packed) route_topk_kernel<L, V, false, true, false><<<g, kThreads, 0, st>>>(p);
    else route_topk_kernel<L, V, false, false, false><<<g, kThreads, 0, st>>>(p);
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
  const bool guard = bias != nullptr || (p.groups > 1 && group_top == 2 && p.gsize > 1);
  const bool packed = dtype != RB_F32;
  const bool vec = rows_of_8(logits, dtype, ld, E) && rows_of_8(probs, score_dtype, E, E);
  if (E <= 8) launch_fwd<1, 8>(p, vec, packed, guard, st);
  else if (E <= 16) launch_fwd<2, 8>(p, vec, packed, guard, st);
  else if (E <= 32) launch_fwd<4, 8>(p, vec, packed, guard, st);
  else if (E <= 64) launch_fwd<8, 8>(p, vec, packed, guard, st);
  else if (E <= 128) launch_fwd<16, 8>(p, vec, packed, guard, st);
  else if (E <= 256) launch_fwd<32, 8>(p, vec, packed, guard, st);
  else launch_fwd<32, 16>(p, vec, packed, guard, st);
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

// clip.cu -- the norm of all gradients of a model, and the clipping by it.
//
//   norm = scale sqrt(sum over all tensors of g^2)     g' = scale g min(1, most / (norm + 1e-6))
//
// over many tensors of mixed types and sizes, of which some may be the touched rows of a table with their number on the
// device.  Bound by HBM: every gradient is read for the norm, and read and written for the clipping, which is left out
// on the device where the factor is 1 and the tensors stay in place.
//
// Two kernels, no atomics, the same bits every time.  The tensors' addresses travel as kernel parameters (kMaxTensors a
// launch), cut into pieces of kPiece values that the CTAs take in turn; a CTA's sum goes to its own place, and every
// CTA of the second kernel adds all of them up in the same order.  A piece's squares are summed in fp32, each thread's
// of at most 32 values; where such a sum is outside [2^-90, 2^120] (a square of a bf16 or fp32 value may be outside
// fp32's range) and not of zeros alone it is taken again in fp64, and everything above it is fp64.
//
// 290 bf16 tensors of 166 MB together: norm 35 us (4.7 TB/s, what L2 held among it), scaling 56 (5.9 TB/s read and written).
#include "common.cuh"

#include <algorithm>
#include <cmath>

namespace rb {
namespace clip {

constexpr int kMaxTensors = 448, kFewTensors = 24;  // (parameters are copied at every launch: few tensors, few bytes)
constexpr int kThreads = 256, kPer = 32, kPiece = kThreads * kPer, kCtas = 4;  // CTAs an SM holds: the grid is one wave

struct Tensor {
  const void* from;
  void* to;
  const int32_t* count;  // rows that count, or null: all
  int64_t n;             // values
  int32_t first;         // piece
  int16_t dtype, vec;    // vec: 16-byte loads and stores
  int32_t width;         // of a row, with `count`
};
template <int N>
struct Params {
  Tensor t[N];
  double* sums;          // of every CTA of every launch
  float* norm;
  int tensors, pieces, slots, first_slot;
  float scale, most;
};
static_assert(sizeof(Params<kMaxTensors>) <= 32 * 1024 - 512, "kernel parameters");

// the tensor that piece i belongs to
template <int N>
__device__ __forceinline__ int tensor_of(const Params<N>& p, int i) {
  int a = 0, b = p.tensors;
  while (b - a > 1) {
    const int m = (a + b) >> 1;
    if (p.t[m].first <= i) a = m;
    else b = m;
  }
  return a;
}
__device__ __forceinline__ int64_t values_of(const Tensor& t) {
  if (t.count == nullptr) return t.n;
  return min(t.n, (int64_t)max(__ldg(t.count), 0) * t.width);
}

// 16 bytes as fp32: 4 or 8 values
template <int DT>
struct Type;
template <>
struct Type<RB_F32> {
  static constexpr int kVec = 4;
  typedef float T;
  static __device__ void widen(uint4 w, float* v) {
    v[0] = __uint_as_float(w.x);
    v[1] = __uint_as_float(w.y);
    v[2] = __uint_as_float(w.z);
    v[3] = __uint_as_float(w.w);
  }
  static __device__ uint4 narrow(const float* v) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
};
template <>
struct Type<RB_BF16> {
  static constexpr int kVec = 8;
  typedef __nv_bfloat16 T;
  static __device__ void widen(uint4 w, float* v) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = bf16_lo(u[i]);
      v[2 * i + 1] = bf16_hi(u[i]);
    }
  }
  static __device__ uint4 narrow(const float* v) {
    return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  }
};
template <>
struct Type<RB_F16> {
  static constexpr int kVec = 8;
  typedef __half T;
  static __device__ void widen(uint4 w, float* v) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
  static __device__ uint4 narrow(const float* v) {
    return make_uint4(pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]), pack_f16x2(v[4], v[5]), pack_f16x2(v[6], v[7]));
  }
};

// this thread's part of the sum of squares of a piece
template <int DT>
__device__ __forceinline__ double squares(const void* from, int64_t at, int64_t n, bool vec) {
  using Y = Type<DT>;
  const typename Y::T* x = static_cast<const typename Y::T*>(from);
  float v[kPer];
  if (vec) {
    uint4 w[kPer / Y::kVec];
#pragma unroll
    for (int k = 0; k < kPer / Y::kVec; ++k) {
      const int64_t i = at + (int64_t)(k * kThreads + threadIdx.x) * Y::kVec;
      w[k] = make_uint4(0u, 0u, 0u, 0u);
      if (i + Y::kVec <= n) {
        w[k] = __ldg(reinterpret_cast<const uint4*>(x + i));
      } else if (i < n) {
        float e[Y::kVec];
#pragma unroll
        for (int c = 0; c < Y::kVec; ++c) e[c] = i + c < n ? (float)x[i + c] : 0.0f;
        w[k] = Y::narrow(e);
      }
    }
#pragma unroll
    for (int k = 0; k < kPer / Y::kVec; ++k) Y::widen(w[k], v + k * Y::kVec);
  } else {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int64_t i = at + k * kThreads + threadIdx.x;
      v[k] = i < n ? (float)x[i] : 0.0f;
    }
  }
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int k = 0; k < kPer; ++k) s[k & 3] = fmaf(v[k], v[k], s[k & 3]);
  const float sum = (s[0] + s[1]) + (s[2] + s[3]);
  if (sum >= 0x1p-90f && sum <= 0x1p120f) return (double)sum;
  if (sum == 0.0f) {  // zeros (rows of a table that no id touched, the threads behind a tensor's end), or all too small
    float most = 0.0f;
#pragma unroll
    for (int k = 0; k < kPer; ++k) most = fmaxf(most, fabsf(v[k]));
    if (most == 0.0f) return 0.0;
  }
  double exact = 0.0;
#pragma unroll 1
  for (int k = 0; k < kPer; ++k) {
    // (the values again, one by one, so that they need not stay in registers by index)
    const int64_t i = vec ? at + (int64_t)((k / Y::kVec) * kThreads + threadIdx.x) * Y::kVec + k % Y::kVec : at + k * kThreads + threadIdx.x;
    const double e = i < n ? (double)(float)x[i] : 0.0;
    exact += e * e;
  }
  return exact;
}

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double s_warp[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) s += s_warp[w];
  return s;
}

// A CTA takes neighbouring pieces: the tensor is searched for once, then stepped to.  The second kernel takes them in the
// opposite order, so that what the first read last, which L2 still holds, is read first.
struct Range {
  int first, last;
};
template <int N>
__device__ __forceinline__ Range pieces_of(const Params<N>& p) {
  return Range{(int)((int64_t)p.pieces * blockIdx.x / gridDim.x), (int)((int64_t)p.pieces * (blockIdx.x + 1) / gridDim.x)};
}

template <int N>
__global__ void __launch_bounds__(kThreads, kCtas) norm_kernel(const __grid_constant__ Params<N> p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  double sum = 0.0;
  const Range q = pieces_of(p);
  int at_tensor = q.first < q.last ? tensor_of(p, q.first) : 0;
  for (int i = q.first; i < q.last; ++i) {
    while (at_tensor + 1 < p.tensors && p.t[at_tensor + 1].first <= i) ++at_tensor;
    const Tensor& t = p.t[at_tensor];
    const int64_t at = (int64_t)(i - t.first) * kPiece, n = values_of(t);
    if (at >= n) continue;
    if (t.dtype == RB_BF16) sum += squares<RB_BF16>(t.from, at, n, t.vec);
    else if (t.dtype == RB_F16) sum += squares<RB_F16>(t.from, at, n, t.vec);
    else sum += squares<RB_F32>(t.from, at, n, t.vec);
  }
  sum = block_sum(sum);
  if (threadIdx.x == 0) p.sums[p.first_slot + blockIdx.x] = sum;
}

template <int DT>
__device__ __forceinline__ void scaled(const void* from, void* to, int64_t at, int64_t n, bool vec, float f) {
  using Y = Type<DT>;
  const typename Y::T* x = static_cast<const typename Y::T*>(from);
  typename Y::T* y = static_cast<typename Y::T*>(to);
  if (vec) {
    constexpr int kBatch = 4;  // loads in flight (more did not fit the registers of four CTAs)
#pragma unroll 1
    for (int k0 = 0; k0 < kPer / Y::kVec; k0 += kBatch) {
      uint4 w[kBatch];
      const int64_t i0 = at + (int64_t)(k0 * kThreads + threadIdx.x) * Y::kVec;
#pragma unroll
      for (int k = 0; k < kBatch; ++k)
        if (i0 + (k * kThreads + 1) * Y::kVec <= n) w[k] = *reinterpret_cast<const uint4*>(x + i0 + k * kThreads * Y::kVec);
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int64_t i = i0 + k * kThreads * Y::kVec;
        if (i + Y::kVec <= n) {
          float v[Y::kVec];
          Y::widen(w[k], v);
#pragma unroll
          for (int c = 0; c < Y::kVec; ++c) v[c] *= f;
          *reinterpret_cast<uint4*>(y + i) = Y::narrow(v);
        }
      }
    }
    // the last values, off the vectors: by the first threads of the CTA that has them
    const int64_t tail = n / Y::kVec * Y::kVec;
    if (tail >= at && tail < at + kPiece && tail + threadIdx.x < n && threadIdx.x < Y::kVec) y[tail + threadIdx.x] = typename Y::T((float)x[tail + threadIdx.x] * f);
  } else {
#pragma unroll 4
    for (int k = 0; k < kPer; ++k) {
      const int64_t i = at + k * kThreads + threadIdx.x;
      if (i < n) y[i] = typename Y::T((float)x[i] * f);
    }
  }
}

// most < 0: the norm alone
template <int N>
__global__ void __launch_bounds__(kThreads, kCtas) scale_kernel(const __grid_constant__ Params<N> p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  double sum = 0.0;
  for (int i = threadIdx.x; i < p.slots; i += kThreads) sum += p.sums[i];
  const float norm = (float)((double)p.scale * sqrt(block_sum(sum)));
  if (blockIdx.x == 0 && threadIdx.x == 0 && p.first_slot == 0) *p.norm = norm;
  if (p.most < 0.0f) return;
  float f = p.most / (norm + 1e-6f);
  f = p.scale * (f < 1.0f || f != f ? f : 1.0f);
  const Range q = pieces_of(p);
  int at_tensor = q.first < q.last ? tensor_of(p, q.last - 1) : 0;
  for (int i = q.last - 1; i >= q.first; --i) {
    while (at_tensor > 0 && p.t[at_tensor].first > i) --at_tensor;
    const Tensor& t = p.t[at_tensor];
    if (f == 1.0f && t.from == t.to) continue;
    const int64_t at = (int64_t)(i - t.first) * kPiece, n = values_of(t);
    if (at >= n) continue;
    if (t.dtype == RB_BF16) scaled<RB_BF16>(t.from, t.to, at, n, t.vec, f);
    else if (t.dtype == RB_F16) scaled<RB_F16>(t.from, t.to, at, n, t.vec, f);
    else scaled<RB_F32>(t.from, t.to, at, n, t.vec, f);
  }
}

// CTAs of a launch, at most
static int grid_of(int64_t pieces) { return (int)std::min<int64_t>(std::max<int64_t>(pieces, 1), (int64_t)sm_count() * kCtas); }

struct List {
  const void* const* from;
  void* const* to;
  const int64_t* values;
  const int* dtypes;
  const void* const* counts;
  const int64_t* widths;
  int tensors;
};

template <int N>
static int run(const List& q, float scale, float most, double* sums, float* norm, cudaStream_t st) {
  const int launches = std::max(1, (q.tensors + N - 1) / N);
  int rc, slots = 0;
  // the norm's kernels first, then the scaling ones, which need all sums
  for (int pass = 0; pass < 2; ++pass) {
    int slot = 0;
    for (int l = 0; l < launches; ++l) {
      Params<N> p;
      p.tensors = 0;
      p.sums = sums;
      p.norm = norm;
      p.scale = scale;
      p.most = most;
      int64_t pieces = 0;
      for (int i = l * N; i < std::min(q.tensors, (l + 1) * N); ++i) {
        if (q.values[i] == 0) continue;
        Tensor& t = p.t[p.tensors++];
        t.from = q.from[i];
        t.to = most >= 0.0f ? q.to[i] : nullptr;
        t.count = q.counts == nullptr ? nullptr : static_cast<const int32_t*>(q.counts[i]);
        t.width = t.count == nullptr ? 0 : (int32_t)q.widths[i];
        t.n = q.values[i];
        t.first = (int32_t)pieces;
        t.dtype = (int16_t)q.dtypes[i];
        t.vec = aligned(t.from, 16) && (t.to == nullptr || aligned(t.to, 16));
        pieces += (q.values[i] + kPiece - 1) / kPiece;
        if (pieces > 0x7fffffff) return fail(RB_ERR_UNSUPPORTED, "too many values");
      }
      p.pieces = (int)pieces;
      p.first_slot = slot;
      p.slots = slots;
      const int grid = grid_of(pieces);
      if (pass == 0) {
        norm_kernel<N><<<grid, kThreads, 0, st>>>(p);
        if ((rc = check_cuda(cudaGetLastError(), "clip norm_kernel launch"))) return rc;
      } else {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(most < 0.0f ? 1 : grid);
        cfg.blockDim = dim3(kThreads);
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = launches == 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        if ((rc = check_cuda(cudaLaunchKernelEx(&cfg, scale_kernel<N>, p), "clip scale_kernel launch"))) return rc;
        if (most < 0.0f) break;
      }
      slot += grid;
    }
    slots = slot;
  }
  return RB_OK;
}

}  // namespace clip
}  // namespace rb

using namespace rb;

extern "C" int64_t rb_grad_norm_workspace_size(int tensors) {
  if (tensors < 0) return -1;
  const int64_t launches = std::max<int64_t>(1, (tensors + clip::kMaxTensors - 1) / clip::kMaxTensors);
  return launches * sm_count() * clip::kCtas * 8;
}

extern "C" int rb_clip_grads(const void* const* from, void* const* to, const int64_t* values, const int* dtypes,
                             const void* const* counts, const int64_t* widths, int tensors, float scale, float most,
                             void* workspace, int64_t workspace_bytes, float* norm, void* stream) {
  using namespace rb::clip;
  if (tensors < 0) return fail(RB_ERR_VALUE, "negative number of tensors");
  if (tensors > 0 && (from == nullptr || values == nullptr || dtypes == nullptr)) return fail(RB_ERR_VALUE, "null list");
  if (norm == nullptr) return fail(RB_ERR_VALUE, "null operand");
  if (!(scale >= 0.0f) || !(scale < INFINITY)) return fail(RB_ERR_VALUE, "scale must be finite and not negative");
  if (most != most) return fail(RB_ERR_VALUE, "the largest norm is not a number");
  if (workspace == nullptr || workspace_bytes < rb_grad_norm_workspace_size(tensors) || !aligned(workspace, 8))
    return fail(RB_ERR_VALUE, "workspace of %lld bytes (8-byte aligned) needed, %lld given",
                (long long)rb_grad_norm_workspace_size(tensors), (long long)workspace_bytes);
  for (int i = 0; i < tensors; ++i) {
    if (values[i] < 0) return fail(RB_ERR_VALUE, "tensor %d has a negative size", i);
    if (dtypes[i] != RB_F32 && dtypes[i] != RB_BF16 && dtypes[i] != RB_F16) return fail(RB_ERR_VALUE, "gradients are fp32, bf16 or f16");
    if (values[i] > 0 && (from[i] == nullptr || (most >= 0.0f && (to == nullptr || to[i] == nullptr)))) return fail(RB_ERR_VALUE, "null operand");
    if (values[i] > (int64_t)1 << 42) return fail(RB_ERR_UNSUPPORTED, "tensors above 2^42 values");
    if (counts != nullptr && counts[i] != nullptr && (widths == nullptr || widths[i] <= 0 || widths[i] > 0x7fffffffLL))
      return fail(RB_ERR_VALUE, "rows that are counted need a width");
  }
  if (!device_is_sm100()) return fail(RB_ERR_DEVICE, "rb_clip_grads needs an sm_100 (B200) device");
  const List q{from, to, values, dtypes, counts, widths, tensors};
  double* sums = static_cast<double*>(workspace);
  if (tensors <= kFewTensors) return run<kFewTensors>(q, scale, most, sums, norm, (cudaStream_t)stream);
  return run<kMaxTensors>(q, scale, most, sums, norm, (cudaStream_t)stream);
}

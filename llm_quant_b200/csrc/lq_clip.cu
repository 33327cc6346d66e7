// lq_clip.cu -- the norm of many gradients together, and their clipping:
// norm = sqrt(sum g^2) over all values of all tensors, out = g min(1, max_norm /
// (norm + 1e-6)).  Two kernels, the second a programmatic dependent of the
// first: a block's stretch of the values is summed and the block's sum left in
// the workspace; then every block adds up all sums, in one order, and scales the
// same stretch from its end to its start, so that what was read last is still
// in L2.
//
// Squares of 8 (fp32: 4) neighbours are added in fp32, and those sums in fp64;
// a sum that leaves [2^-100, 2^100] is taken again from fp64 squares, so that
// neither the greatest nor the smallest values are lost.
#include <math.h>

#include "lq_common.cuh"

namespace lq {
namespace {

constexpr int kClipThreads = 256;
constexpr int kClipVecs = 8;                                  // 16-byte vectors of a thread in a unit
constexpr int kClipUnit = kClipThreads * kClipVecs * 16;      // bytes of a unit
constexpr int kClipMost = 1024;                               // tensors of a launch
constexpr int kClipBlocks = 148 * 4;

// The tensors of one launch, as a kernel's parameters (no copy to the device,
// nothing for a captured graph to lose).  N by what there are: a launch
// carries the whole struct.
template <int N>
struct ClipTable {
  const void* in[N];
  void* out[N];
  int64_t n[N];
  int unit0[N + 1];  // units before the tensor's
  uint8_t dtype[N];
  int count;
};

// Values of a unit.  The vectors begin at the first 16-byte boundary of `at`
// (and one vector later, and end one earlier, where `wide`); what lies before
// them belongs to the tensor's first unit, what is left behind them to its last.
struct Span {
  int64_t lo;     // the first vector's first value
  int vecs;
  int64_t head;   // values 0 .. head - 1 are this unit's too (0: none)
  int64_t tail, end;  // and values tail .. end - 1
};
template <typename T>
__device__ __forceinline__ Span span_of(const void* at, int64_t n, int unit, int units, bool wide) {
  constexpr int size = sizeof(T), per = kClipUnit / size, vec = 16 / size;
  const int edge = wide ? vec : 0;
  const int64_t head = min(n, (int64_t)((16 - ((reinterpret_cast<uintptr_t>(at)) & 15)) & 15) / size + edge);
  const int64_t stop = head + (max(n - edge - head, (int64_t)0) & -(int64_t)vec);  // behind the last vector
  Span s;
  s.lo = min(stop, head + (int64_t)unit * per);
  const int64_t hi = unit == units - 1 ? stop : min(stop, s.lo + per);
  s.vecs = (int)((hi - s.lo) / vec);
  s.head = unit == 0 ? head : 0;
  s.tail = unit == units - 1 ? stop : n;
  s.end = n;
  return s;
}

template <typename T> struct Clip;  // 16 bytes of T: sum of squares, and scaled
template <> struct Clip<float> {
  static constexpr int V = 4;
  __device__ __forceinline__ static void get(const uint32_t* w, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
  }
  __device__ __forceinline__ static void put(const float* f, uint32_t* w) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(f[i]);
  }
};
template <> struct Clip<__half> {
  static constexpr int V = 8;
  __device__ __forceinline__ static void get(const uint32_t* w, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(w + i));
      f[2 * i] = p.x, f[2 * i + 1] = p.y;
    }
  }
  __device__ __forceinline__ static void put(const float* f, uint32_t* w) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 p = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&p);
    }
  }
};
template <> struct Clip<__nv_bfloat16> {
  static constexpr int V = 8;
  __device__ __forceinline__ static void get(const uint32_t* w, float* f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  __device__ __forceinline__ static void put(const float* f, uint32_t* w) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 p = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&p);
    }
  }
};

template <typename T>
__device__ __forceinline__ double squares(const uint32_t* w) {
  constexpr int V = Clip<T>::V;
  float f[V], s = 0.0f;
  Clip<T>::get(w, f);
#pragma unroll
  for (int i = 0; i < V; ++i) s = fmaf(f[i], f[i], s);
  if (s >= 0x1p-100f && s <= 0x1p100f) return s;
  double d = 0.0;
#pragma unroll
  for (int i = 0; i < V; ++i) d = fma((double)f[i], (double)f[i], d);
  return d;
}

template <typename T>
__device__ __forceinline__ double unit_squares(const void* in, int64_t n, int unit, int units) {
  const T* x = static_cast<const T*>(in);
  const Span s = span_of<T>(in, n, unit, units, false);
  const int vecs = s.vecs;
  double d = 0.0;
  const uint4* v = reinterpret_cast<const uint4*>(x + s.lo);
  uint4 w[kClipVecs];
#pragma unroll
  for (int k = 0; k < kClipVecs; ++k) {
    const int i = k * kClipThreads + threadIdx.x;
    w[k] = i < vecs ? v[i] : make_uint4(0u, 0u, 0u, 0u);
  }
#pragma unroll
  for (int k = 0; k < kClipVecs; ++k)
    if (k * kClipThreads + (int)threadIdx.x < vecs) {
      const uint32_t a[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
      d += squares<T>(a);
    }
  // fewer than a vector's values on either side
  const int t = threadIdx.x;
  if (t < s.head) d += (double)Ty<T>::to_f(x[t]) * (double)Ty<T>::to_f(x[t]);
  if (s.tail + t < s.end) d += (double)Ty<T>::to_f(x[s.tail + t]) * (double)Ty<T>::to_f(x[s.tail + t]);
  return d;
}

// Sum over the block, in one order; thread 0 has it.
__device__ __forceinline__ double block_sum(double d, double* part) {
#pragma unroll
  for (int m = 16; m; m >>= 1) d += __shfl_xor_sync(0xffffffffu, d, m);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = d;
  __syncthreads();
  if (threadIdx.x == 0) {
    d = 0.0;
    for (int w = 0; w < kClipThreads / 32; ++w) d += part[w];
  }
  return d;
}

// The block's stretch of units, and the tensor that unit u is of.
template <int N>
__device__ __forceinline__ int tensor_of(const ClipTable<N>& t, int u) {
  int lo = 0, hi = t.count;  // unit0[lo] <= u < unit0[hi]
  while (hi - lo > 1) {
    const int m = (lo + hi) / 2;
    if (t.unit0[m] <= u) lo = m; else hi = m;
  }
  return lo;
}

template <int N>
__global__ void __launch_bounds__(kClipThreads) clip_norm_kernel(const __grid_constant__ ClipTable<N> t, double* __restrict__ sums) {
  __shared__ double part[kClipThreads / 32];
  pdl_wait();
  pdl_trigger();
  const int64_t units = t.unit0[t.count];
  double d = 0.0;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int i = tensor_of(t, (int)u);
    const int k = (int)u - t.unit0[i], units_i = t.unit0[i + 1] - t.unit0[i];
    if (t.dtype[i] == LQ_F32) d += unit_squares<float>(t.in[i], t.n[i], k, units_i);
    else if (t.dtype[i] == LQ_F16) d += unit_squares<__half>(t.in[i], t.n[i], k, units_i);
    else d += unit_squares<__nv_bfloat16>(t.in[i], t.n[i], k, units_i);
  }
  d = block_sum(d, part);
  if (threadIdx.x == 0) sums[blockIdx.x] = d;
}

// 16 bytes from off bytes into two neighbouring vectors (off: not 0).
__device__ __forceinline__ void shift(const uint4& a, const uint4& b, int off, uint32_t* w) {
  const int bits = (off & 3) * 8;
  uint32_t y[5];
  switch (off >> 2) {
    case 0: y[0] = a.x, y[1] = a.y, y[2] = a.z, y[3] = a.w, y[4] = b.x; break;
    case 1: y[0] = a.y, y[1] = a.z, y[2] = a.w, y[3] = b.x, y[4] = b.y; break;
    case 2: y[0] = a.z, y[1] = a.w, y[2] = b.x, y[3] = b.y, y[4] = b.z; break;
    default: y[0] = a.w, y[1] = b.x, y[2] = b.y, y[3] = b.z, y[4] = b.w; break;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(y[i], y[i + 1], bits);
}

// SHIFTED: the result lies on 16 bytes where the source does not.  A lane loads
// the aligned vector that its source begins in; the rest of it is the next lane's.
template <typename T, bool SHIFTED>
__device__ __forceinline__ void scale_vectors(const uint8_t* from, uint4* to, int vecs, int off, float c) {
  constexpr int V = Clip<T>::V;
  const int lane = threadIdx.x & 31;
  uint4 a[kClipVecs];
#pragma unroll
  for (int k = 0; k < kClipVecs; ++k) {
    const int i = k * kClipThreads + threadIdx.x;
    a[k] = make_uint4(0u, 0u, 0u, 0u);
    // the vector behind the last one is inside the tensor too
    if (SHIFTED ? i <= vecs : i < vecs) a[k] = *reinterpret_cast<const uint4*>(from - off + 16 * (int64_t)i);
  }
#pragma unroll
  for (int k = 0; k < kClipVecs; ++k) {
    const int i = k * kClipThreads + threadIdx.x;
    uint32_t w[4] = {a[k].x, a[k].y, a[k].z, a[k].w};
    if (SHIFTED) {
      uint4 b;
      b.x = __shfl_down_sync(0xffffffffu, a[k].x, 1), b.y = __shfl_down_sync(0xffffffffu, a[k].y, 1);
      b.z = __shfl_down_sync(0xffffffffu, a[k].z, 1), b.w = __shfl_down_sync(0xffffffffu, a[k].w, 1);
      if (lane == 31 && i < vecs) b = *reinterpret_cast<const uint4*>(from - off + 16 * (int64_t)(i + 1));
      shift(a[k], b, off, w);
    }
    if (i >= vecs) continue;
    float f[V];
    Clip<T>::get(w, f);
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = __fmul_rn(f[e], c);
    Clip<T>::put(f, w);
    __stcs(to + i, make_uint4(w[0], w[1], w[2], w[3]));
  }
}

template <typename T>
__device__ __forceinline__ void unit_scale(const void* in, void* res, int64_t n, int unit, int units, float c) {
  const T* x = static_cast<const T*>(in);
  T* out = static_cast<T*>(res);
  const int off = (int)((reinterpret_cast<uintptr_t>(in) - reinterpret_cast<uintptr_t>(res)) & 15);  // the same for all vectors
  const Span s = span_of<T>(res, n, unit, units, off != 0);
  const uint8_t* from = reinterpret_cast<const uint8_t*>(x + s.lo);
  uint4* to = reinterpret_cast<uint4*>(out + s.lo);
  // without a vector there may be no boundary either: the tensor may end before the first
  if (s.vecs > 0) {
    if (off) scale_vectors<T, true>(from, to, s.vecs, off, c);
    else scale_vectors<T, false>(from, to, s.vecs, 0, c);
  }
  // fewer than three vectors' values on either side
  const int t = threadIdx.x;
  if (t < s.head) out[t] = Ty<T>::from_f(__fmul_rn(Ty<T>::to_f(x[t]), c));
  if (s.tail + t < s.end) out[s.tail + t] = Ty<T>::from_f(__fmul_rn(Ty<T>::to_f(x[s.tail + t]), c));
}

template <int N>
__global__ void __launch_bounds__(kClipThreads, 4) clip_scale_kernel(const __grid_constant__ ClipTable<N> t,
                                                                  const double* __restrict__ sums, int n_sums,
                                                                  double max_norm, float* __restrict__ norm) {
  __shared__ double part[kClipThreads / 32];
  __shared__ float coef;
  pdl_wait();
  pdl_trigger();
  double d = 0.0;
  for (int i = threadIdx.x; i < n_sums; i += kClipThreads) d += sums[i];
  d = block_sum(d, part);
  if (threadIdx.x == 0) {
    const double total = sqrt(d), c = max_norm / (total + 1e-6);
    coef = c >= 1.0 ? 1.0f : (float)c;  // NaN stays
    if (blockIdx.x == 0 && norm) *norm = (float)total;
  }
  __syncthreads();
  const float c = coef;
  const int64_t units = t.unit0[t.count];
  for (int64_t u = units - 1 - blockIdx.x; u >= 0; u -= gridDim.x) {
    const int i = tensor_of(t, (int)u);
    if (c == 1.0f && t.in[i] == t.out[i]) continue;  // nothing changes
    const int k = (int)u - t.unit0[i], units_i = t.unit0[i + 1] - t.unit0[i];
    if (t.dtype[i] == LQ_F32) unit_scale<float>(t.in[i], t.out[i], t.n[i], k, units_i, c);
    else if (t.dtype[i] == LQ_F16) unit_scale<__half>(t.in[i], t.out[i], t.n[i], k, units_i, c);
    else unit_scale<__nv_bfloat16>(t.in[i], t.out[i], t.n[i], k, units_i, c);
  }
}

int64_t units_of(int64_t n, int dtype) {
  const int64_t bytes = n * dtype_size(dtype);
  return (bytes + kClipUnit - 1) / kClipUnit;
}

template <int N>
int clip_launch(const void* const* in, void* const* out, const int64_t* n, const int* dtype, int count, bool norm_pass,
                int blocks, double max_norm, double* sums, int n_sums, float* norm, cudaStream_t st) {
  ClipTable<N> t;
  int64_t units = 0;
  for (int i = 0; i < count; ++i) {
    t.in[i] = in[i], t.out[i] = out ? out[i] : const_cast<void*>(in[i]);
    t.n[i] = n[i], t.dtype[i] = (uint8_t)dtype[i], t.unit0[i] = (int)units;
    units += units_of(n[i], dtype[i]);
  }
  LQ_REQUIRE(units < (1LL << 31), LQ_ERANGE, "clip: too many values");
  t.unit0[count] = (int)units, t.count = count;
  const cudaError_t e = norm_pass ? launch_pdl(clip_norm_kernel<N>, dim3(blocks), dim3(kClipThreads), 0, st, t, sums)
                                  : launch_pdl(clip_scale_kernel<N>, dim3(blocks), dim3(kClipThreads), 0, st, t,
                                               (const double*)sums, n_sums, max_norm, norm);
  LQ_REQUIRE(e == cudaSuccess, LQ_ECUDA, "clip: launch failed: %s", cudaGetErrorString(e));
  return launched("clip");
}

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" size_t lq_clip_workspace_bytes(int64_t count) {
  if (count < 0) return 0;
  return sizeof(double) * kClipBlocks * (size_t)((count + kClipMost - 1) / kClipMost + 1);
}

extern "C" int lq_clip_grad_norm(const void* const* host_in, void* const* host_out, const int64_t* host_n,
                                 const int* host_dtype, int64_t count, double max_norm, float* norm, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  LQ_REQUIRE(count >= 0 && count < (1 << 24), LQ_EINVAL, "clip: %lld tensors", (long long)count);
  LQ_REQUIRE(count == 0 || (host_in && host_n && host_dtype), LQ_EINVAL, "clip: NULL pointer");
  LQ_REQUIRE(norm, LQ_EINVAL, "clip: NULL norm");
  LQ_REQUIRE(max_norm >= 0, LQ_EINVAL, "clip: max_norm must not be negative or NaN");
  const size_t need = lq_clip_workspace_bytes(count);
  LQ_REQUIRE(workspace && reinterpret_cast<uintptr_t>(workspace) % 8 == 0 && workspace_bytes >= need, LQ_EINVAL,
             "clip: %zu bytes of workspace needed", need);
  for (int64_t i = 0; i < count; ++i) {
    LQ_REQUIRE(is_float_dtype(host_dtype[i]), LQ_EDTYPE, "clip: tensor %lld: unsupported dtype %d", (long long)i, host_dtype[i]);
    const uintptr_t size = dtype_size(host_dtype[i]);
    LQ_REQUIRE(host_n[i] >= 0 && host_n[i] < (1LL << 40), LQ_EINVAL, "clip: tensor %lld: bad size", (long long)i);
    LQ_REQUIRE(host_n[i] == 0 || (host_in[i] && (!host_out || host_out[i])), LQ_EINVAL, "clip: tensor %lld: NULL pointer", (long long)i);
    LQ_REQUIRE(reinterpret_cast<uintptr_t>(host_in[i]) % size == 0 && (!host_out || reinterpret_cast<uintptr_t>(host_out[i]) % size == 0),
               LQ_EALIGN, "clip: tensor %lld: address not a multiple of its type's size", (long long)i);
  }
  double* sums = static_cast<double*>(workspace);
  cudaStream_t st = as_stream(stream);
  int n_sums = 0;
  for (int pass = 0; pass < 2; ++pass) {
    for (int64_t i0 = 0; i0 < count || i0 == 0; i0 += kClipMost) {
      const int c = (int)(count - i0 < kClipMost ? count - i0 : kClipMost);
      int64_t units = 0;
      for (int i = 0; i < c; ++i) units += units_of(host_n[i0 + i], host_dtype[i0 + i]);
      const int blocks = (int)(units < 1 ? 1 : units < kClipBlocks ? units : kClipBlocks);
      const auto f = c <= 32 ? clip_launch<32> : c <= 256 ? clip_launch<256> : clip_launch<kClipMost>;
      LQ_TRY(f(host_in ? host_in + i0 : nullptr, host_out ? host_out + i0 : nullptr, host_n ? host_n + i0 : nullptr,
               host_dtype ? host_dtype + i0 : nullptr, c, pass == 0, blocks, max_norm, pass == 0 ? sums + n_sums : sums, n_sums,
               i0 == 0 ? norm : nullptr, st));
      if (pass == 0) n_sums += blocks;
    }
  }
  return LQ_OK;
}

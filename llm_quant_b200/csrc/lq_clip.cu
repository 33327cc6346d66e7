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
constexpr int kClipVecs = 8;  // 16-byte vectors of a thread in a unit
// Bytes of a unit; where results lie on other bytes of 16 than their source, a
// warp's last lane only serves the one before it.
__host__ __device__ constexpr int clip_unit(bool shifted) { return kClipThreads / 32 * (shifted ? 31 : 32) * kClipVecs * 16; }
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
  uint16_t first[kClipBlocks + 1];  // the tensor that a block's units begin in (a search on the device cost 8 us of 1024)
  int count;
  int moved;  // some result is not in its source's place
};

// Units k0 .. k1 - 1 of a tensor, in bytes from its start.  Vectors lie on 16
// bytes of the result; those of the source are loaded from `off` bytes before,
// where it lies otherwise.  The tensor's first unit has what comes before the
// first vector too, its last one what is left behind the last; with a shifted
// source these edges are a vector wider, so that the vectors to either side of
// a load are inside the tensor.
struct Stretch {
  int64_t lo;             // the first vector
  int64_t vecs;
  int head;               // bytes 0 .. head - 1 too
  int64_t tail, end;      // and bytes tail .. end - 1
};
__device__ __forceinline__ Stretch stretch_of(const void* at, int64_t bytes, int off, int unit, int k0, int k1, int units) {
  const int wide = off ? 16 : 0;
  const int64_t head = min(bytes, (int64_t)((16 - (reinterpret_cast<uintptr_t>(at) & 15)) & 15) + wide);
  const int64_t stop = head + (max(bytes - wide - head, (int64_t)0) & -16);  // behind the last vector
  Stretch s;
  s.lo = min(stop, head + (int64_t)k0 * unit);
  s.vecs = ((k1 == units ? stop : min(stop, head + (int64_t)k1 * unit)) - s.lo) >> 4;
  s.head = k0 == 0 ? (int)head : 0;
  s.tail = stop, s.end = k1 == units ? bytes : stop;
  return s;
}
__device__ __forceinline__ int shift_of(const void* in, const void* out) {
  return (int)((reinterpret_cast<uintptr_t>(in) - reinterpret_cast<uintptr_t>(out)) & 15);
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
__device__ __forceinline__ double stretch_squares(const void* in, const Stretch& s) {
  const uint4* v = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(in) + s.lo) + threadIdx.x;
  double d = 0.0;
  int64_t left = s.vecs - threadIdx.x;
  for (; left > (kClipVecs - 1) * kClipThreads; left -= kClipVecs * kClipThreads, v += kClipVecs * kClipThreads) {
    uint4 w[kClipVecs];
#pragma unroll
    for (int k = 0; k < kClipVecs; ++k) w[k] = v[k * kClipThreads];
#pragma unroll
    for (int k = 0; k < kClipVecs; ++k) {
      const uint32_t a[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
      d += squares<T>(a);
    }
  }
#pragma unroll 4
  for (; left > 0; left -= kClipThreads, v += kClipThreads) {
    const uint4 w = *v;
    const uint32_t a[4] = {w.x, w.y, w.z, w.w};
    d += squares<T>(a);
  }
  // fewer than a vector's values on either side
  const T* x = static_cast<const T*>(in);
  const int t = threadIdx.x;
  if (t * (int)sizeof(T) < s.head) d += (double)Ty<T>::to_f(x[t]) * (double)Ty<T>::to_f(x[t]);
  const int64_t e = s.tail / (int)sizeof(T) + t;
  if (e * (int)sizeof(T) < s.end) d += (double)Ty<T>::to_f(x[e]) * (double)Ty<T>::to_f(x[e]);
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

template <int N>
__global__ void __launch_bounds__(kClipThreads) clip_norm_kernel(const __grid_constant__ ClipTable<N> t, double* __restrict__ sums) {
  __shared__ double part[kClipThreads / 32];
  pdl_wait();
  pdl_trigger();
  const int64_t units = t.unit0[t.count];
  const int u0 = (int)(units * blockIdx.x / gridDim.x), u1 = (int)(units * (blockIdx.x + 1) / gridDim.x);
  double d = 0.0;
  for (int u = u0, i = t.first[blockIdx.x]; u < u1; ++i) {
    const int a = t.unit0[i], b = t.unit0[i + 1], k1 = min(b, u1);
    if (k1 <= u) continue;  // an empty tensor
    const int size = t.dtype[i] == LQ_F32 ? 4 : 2;
    const Stretch s = stretch_of(t.in[i], t.n[i] * size, 0, clip_unit(shift_of(t.in[i], t.out[i]) != 0), u - a, k1 - a, b - a);
    if (t.dtype[i] == LQ_F32) d += stretch_squares<float>(t.in[i], s);
    else if (t.dtype[i] == LQ_F16) d += stretch_squares<__half>(t.in[i], s);
    else d += stretch_squares<__nv_bfloat16>(t.in[i], s);
    u = k1;
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

// A stretch, from its end to its start.  A lane of a shifted one loads the
// aligned vector that its source begins in; the rest of it is the next lane's.
template <typename T, bool SHIFTED>
__device__ __forceinline__ void stretch_scale(const void* in, void* out, const Stretch& s, int off, float c) {
  constexpr int V = Clip<T>::V, W = SHIFTED ? 31 : 32, STEP = kClipThreads / 32 * W;
  const int lane = threadIdx.x & 31, at = (threadIdx.x >> 5) * W + lane;
  const uint4* from = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(in) + s.lo - off);
  uint4* to = reinterpret_cast<uint4*>(static_cast<uint8_t*>(out) + s.lo);
  const int64_t loads = s.vecs == 0 ? 0 : SHIFTED ? s.vecs + 1 : s.vecs;
  const int64_t most = SHIFTED && lane == 31 ? 0 : s.vecs;  // what the lane writes ends here
  float f[V];
  for (int64_t b = (s.vecs - 1) / (STEP * kClipVecs) * (STEP * kClipVecs); b >= 0; b -= STEP * kClipVecs) {
    uint4 a[kClipVecs];
    const int64_t i0 = b + at;
#pragma unroll
    for (int k = 0; k < kClipVecs; ++k)
      a[k] = i0 + k * STEP < loads ? from[i0 + k * STEP] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int k = 0; k < kClipVecs; ++k) {
      uint32_t x[4] = {a[k].x, a[k].y, a[k].z, a[k].w};
      if (SHIFTED) {
        uint4 n;
        n.x = __shfl_down_sync(0xffffffffu, x[0], 1), n.y = __shfl_down_sync(0xffffffffu, x[1], 1);
        n.z = __shfl_down_sync(0xffffffffu, x[2], 1), n.w = __shfl_down_sync(0xffffffffu, x[3], 1);
        shift(a[k], n, off, x);
      }
      Clip<T>::get(x, f);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = __fmul_rn(f[e], c);
      Clip<T>::put(f, x);
      if (i0 + k * STEP < most) __stcs(to + i0 + k * STEP, make_uint4(x[0], x[1], x[2], x[3]));
    }
  }
  // fewer than three vectors' values on either side
  const T* x = static_cast<const T*>(in);
  T* y = static_cast<T*>(out);
  const int t = threadIdx.x;
  if (t * (int)sizeof(T) < s.head) y[t] = Ty<T>::from_f(__fmul_rn(Ty<T>::to_f(x[t]), c));
  const int64_t e = s.tail / (int)sizeof(T) + t;
  if (e * (int)sizeof(T) < s.end) y[e] = Ty<T>::from_f(__fmul_rn(Ty<T>::to_f(x[e]), c));
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
  if (c == 1.0f && !t.moved) return;  // nothing changes
  const int64_t units = t.unit0[t.count];
  const int u0 = (int)(units * blockIdx.x / gridDim.x), u1 = (int)(units * (blockIdx.x + 1) / gridDim.x);
  for (int u = u1, i = t.first[blockIdx.x + 1]; u > u0; --i) {
    const int a = t.unit0[i], b = t.unit0[i + 1], k0 = max(a, u0);
    if (k0 >= u) continue;  // an empty tensor
    const int size = t.dtype[i] == LQ_F32 ? 4 : 2, off = shift_of(t.in[i], t.out[i]);
    const Stretch s = stretch_of(t.out[i], t.n[i] * size, off, clip_unit(off != 0), k0 - a, u - a, b - a);
    if (t.dtype[i] == LQ_F32)
      off ? stretch_scale<float, true>(t.in[i], t.out[i], s, off, c) : stretch_scale<float, false>(t.in[i], t.out[i], s, 0, c);
    else if (t.dtype[i] == LQ_F16)
      off ? stretch_scale<__half, true>(t.in[i], t.out[i], s, off, c) : stretch_scale<__half, false>(t.in[i], t.out[i], s, 0, c);
    else
      off ? stretch_scale<__nv_bfloat16, true>(t.in[i], t.out[i], s, off, c) : stretch_scale<__nv_bfloat16, false>(t.in[i], t.out[i], s, 0, c);
    u = k0;
  }
}

int64_t units_of(const void* in, const void* out, int64_t n, int dtype) {
  const int64_t bytes = n * dtype_size(dtype);
  const int unit = clip_unit(((reinterpret_cast<uintptr_t>(in) - reinterpret_cast<uintptr_t>(out)) & 15) != 0);
  return (bytes + unit - 1) / unit;
}

template <int N>
int clip_launch(const void* const* in, void* const* out, const int64_t* n, const int* dtype, int count, bool norm_pass,
                int blocks, double max_norm, double* sums, int n_sums, float* norm, cudaStream_t st) {
  ClipTable<N> t;
  int64_t units = 0;
  for (int i = 0; i < count; ++i) {
    t.in[i] = in[i], t.out[i] = out ? out[i] : const_cast<void*>(in[i]);
    t.n[i] = n[i], t.dtype[i] = (uint8_t)dtype[i], t.unit0[i] = (int)units;
    units += units_of(t.in[i], t.out[i], n[i], dtype[i]);
  }
  LQ_REQUIRE(units < (1LL << 31), LQ_ERANGE, "clip: too many values");
  t.unit0[count] = (int)units, t.count = count, t.moved = out != nullptr;
  for (int b = 0, i = 0; b <= blocks; ++b) {
    while (i + 1 < count && t.unit0[i + 1] <= units * b / blocks) ++i;
    t.first[b] = (uint16_t)i;
  }
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
      for (int i = 0; i < c; ++i)
        units += units_of(host_in[i0 + i], host_out ? host_out[i0 + i] : host_in[i0 + i], host_n[i0 + i], host_dtype[i0 + i]);
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

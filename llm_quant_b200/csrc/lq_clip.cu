// lq_clip.cu -- the norm of many gradients together, and their clipping:
// norm = sqrt(sum g^2) over all values of all tensors, out = g min(1, max_norm /
// (norm + 1e-6)).  Two kernels, the second a programmatic dependent of the
// first: a block's stretch of the values is summed and the block's sum left in
// the workspace; then every block adds up all sums, in one order, and scales the
// same stretch from its end to its start, so that what was read last is still
// in L2.  Little is done by one cluster of eight blocks, both at once.
//
// Squares of 8 (fp32: 4) neighbours are added in fp32, and those sums in fp64;
// a sum that leaves [2^-100, 2^100] is taken again from fp64 squares, so that
// neither the greatest nor the smallest values are lost.
#include <math.h>

#include "lq_common.cuh"

namespace lq {
namespace {

constexpr int kClipThreads = 256;
constexpr int kClipVecs = 8;  // 16-byte vectors that a thread has on their way
// Bytes of a unit of `grain` vectors to a thread; where results lie on other
// bytes of 16 than their source, a warp's last lane only serves the one before it.
__host__ __device__ constexpr int clip_unit(bool shifted, int grain) { return kClipThreads / 32 * (shifted ? 31 : 32) * grain * 16; }
constexpr int kClipMost = 1024;                               // tensors of a launch
constexpr int kClipBlocks = 148 * 4;
// Up to here (and 256 tensors) one cluster: three fp32 tensors of 60 KB 5.4 us on
// the device, of 200 KB 7.6, of 340 KB 9.5, where two kernels take 7.6 throughout
// and the host another 3 for the second launch.
constexpr int64_t kClipSmall = 640 << 10;
constexpr int kClipCluster = 8;

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
  int grain;  // vectors of a thread in a unit
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

// Two fp32 operations at a time
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 z, x, y, z;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}

template <typename T>
__device__ __forceinline__ double squares(const uint4& v) {
  constexpr int V = Clip<T>::V;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  float f[V];
  Clip<T>::get(w, f);
  float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int i = 0; i < V; i += 2) s = fma2(make_float2(f[i], f[i + 1]), make_float2(f[i], f[i + 1]), s);
  const float all = s.x + s.y;
  if (all >= 0x1p-100f && all <= 0x1p100f) return all;
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
    for (int k = 0; k < kClipVecs; ++k) d += squares<T>(w[k]);
  }
  for (int h = 0; h < kClipVecs && left > 0; h += 4) {
    uint4 w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = k * kClipThreads < left ? v[k * kClipThreads] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k * kClipThreads < left) d += squares<T>(w[k]);
    left -= 4 * kClipThreads, v += 4 * kClipThreads;
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

// Sum of squares of the block's share of the units (thread 0 has it).
template <int N>
__device__ __forceinline__ double share_squares(const ClipTable<N>& t, double* part) {
  const int64_t units = t.unit0[t.count];
  const int u0 = (int)(units * blockIdx.x / gridDim.x), u1 = (int)(units * (blockIdx.x + 1) / gridDim.x);
  double d = 0.0;
  for (int u = u0, i = t.first[blockIdx.x]; u < u1; ++i) {
    const int a = t.unit0[i], b = t.unit0[i + 1], k1 = min(b, u1);
    if (k1 <= u) continue;  // an empty tensor
    const int size = t.dtype[i] == LQ_F32 ? 4 : 2;
    const Stretch s = stretch_of(t.in[i], t.n[i] * size, 0, clip_unit(shift_of(t.in[i], t.out[i]) != 0, t.grain), u - a, k1 - a, b - a);
    if (t.dtype[i] == LQ_F32) d += stretch_squares<float>(t.in[i], s);
    else if (t.dtype[i] == LQ_F16) d += stretch_squares<__half>(t.in[i], s);
    else d += stretch_squares<__nv_bfloat16>(t.in[i], s);
    u = k1;
  }
  return block_sum(d, part);
}

template <int N>
__global__ void __launch_bounds__(kClipThreads, 4) clip_norm_kernel(const __grid_constant__ ClipTable<N> t, double* __restrict__ sums) {
  __shared__ double part[kClipThreads / 32];
  pdl_wait();
  pdl_trigger();
  const double d = share_squares(t, part);
  if (threadIdx.x == 0) sums[blockIdx.x] = d;
}

// 16 bytes from 4 W + bits / 8 bytes into two neighbouring vectors.
template <int W>
__device__ __forceinline__ void shift(const uint4& a, const uint4& b, int bits, uint32_t* w) {
  const uint32_t x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(x[i + W], x[i + W + 1], bits);
}

// A stretch, from its end to its start.  A lane of a shifted one loads the
// aligned vector that its source begins in; the rest of it is the next lane's.
template <typename T, int WORDS>  // WORDS: whole words of the shift, -1: there is none
__device__ __forceinline__ void stretch_scale(const void* in, void* out, const Stretch& s, int off, float c) {
  constexpr bool SHIFTED = WORDS >= 0;
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
        shift<SHIFTED ? WORDS : 0>(a[k], n, (off & 3) * 8, x);
      }
      Clip<T>::get(x, f);
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const float2 y = mul2(make_float2(f[e], f[e + 1]), make_float2(c, c));
        f[e] = y.x, f[e + 1] = y.y;
      }
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

template <typename T>
__device__ __forceinline__ void any_scale(const void* in, void* out, const Stretch& s, int off, float c) {
  if (off == 0) return stretch_scale<T, -1>(in, out, s, 0, c);
  switch (off >> 2) {
    case 0: return stretch_scale<T, 0>(in, out, s, off, c);
    case 1: return stretch_scale<T, 1>(in, out, s, off, c);
    case 2: return stretch_scale<T, 2>(in, out, s, off, c);
    default: return stretch_scale<T, 3>(in, out, s, off, c);
  }
}

// The block's share of the units, times c.
template <int N>
__device__ __forceinline__ void share_scale(const ClipTable<N>& t, float c) {
  if (c == 1.0f && !t.moved) return;  // nothing changes
  const int64_t units = t.unit0[t.count];
  const int u0 = (int)(units * blockIdx.x / gridDim.x), u1 = (int)(units * (blockIdx.x + 1) / gridDim.x);
  for (int u = u1, i = t.first[blockIdx.x + 1]; u > u0; --i) {
    const int a = t.unit0[i], b = t.unit0[i + 1], k0 = max(a, u0);
    if (k0 >= u) continue;  // an empty tensor
    const int size = t.dtype[i] == LQ_F32 ? 4 : 2, off = shift_of(t.in[i], t.out[i]);
    const Stretch s = stretch_of(t.out[i], t.n[i] * size, off, clip_unit(off != 0, t.grain), k0 - a, u - a, b - a);
    if (t.dtype[i] == LQ_F32) any_scale<float>(t.in[i], t.out[i], s, off, c);
    else if (t.dtype[i] == LQ_F16) any_scale<__half>(t.in[i], t.out[i], s, off, c);
    else any_scale<__nv_bfloat16>(t.in[i], t.out[i], s, off, c);
    u = k0;
  }
}
__device__ __forceinline__ float factor_of(double total, double max_norm) {
  const double c = max_norm / (total + 1e-6);
  return c >= 1.0 ? 1.0f : (float)c;  // NaN stays
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
    const double total = sqrt(d);
    coef = factor_of(total, max_norm);
    if (blockIdx.x == 0 && norm) *norm = (float)total;
  }
  __syncthreads();
  share_scale(t, coef);
}

// Both at once: the cluster's blocks find each other's sums in distributed
// shared memory, and add them up in one order.
template <int N>
__global__ void __launch_bounds__(kClipThreads) clip_small_kernel(const __grid_constant__ ClipTable<N> t, double max_norm,
                                                                  float* __restrict__ norm) {
  __shared__ double part[kClipThreads / 32], mine;
  __shared__ float coef;
  pdl_wait();
  pdl_trigger();
  const double d = share_squares(t, part);
  if (threadIdx.x == 0) mine = d;
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
  if (threadIdx.x == 0) {
    double all = 0.0;
    const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(&mine));
#pragma unroll
    for (int i = 0; i < kClipCluster; ++i) {
      uint32_t peer;
      double v;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(at), "r"(i));
      asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(peer) : "memory");
      all += v;
    }
    const double total = sqrt(all);
    coef = factor_of(total, max_norm);
    if (blockIdx.x == 0) *norm = (float)total;
  }
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");  // waited for at the end: others may still read the sum
  __syncthreads();
  share_scale(t, coef);
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

int64_t units_of(const void* in, const void* out, int64_t n, int dtype, int grain) {
  const int64_t bytes = n * dtype_size(dtype);
  const int unit = clip_unit(((reinterpret_cast<uintptr_t>(in) - reinterpret_cast<uintptr_t>(out)) & 15) != 0, grain);
  return (bytes + unit - 1) / unit;
}

// Host arrays of one launch's tensors
struct ClipList {
  const void* const* in;
  void* const* out;
  const int64_t* n;
  const int* dtype;
  int count;
  int grain, blocks;
};

template <int N>
int clip_table(ClipTable<N>& t, const ClipList& l) {
  int64_t units = 0;
  for (int i = 0; i < l.count; ++i) {
    t.in[i] = l.in[i], t.out[i] = l.out ? l.out[i] : const_cast<void*>(l.in[i]);
    t.n[i] = l.n[i], t.dtype[i] = (uint8_t)l.dtype[i], t.unit0[i] = (int)units;
    units += units_of(t.in[i], t.out[i], l.n[i], l.dtype[i], l.grain);
    LQ_REQUIRE(units < (1LL << 31), LQ_ERANGE, "clip: too many values");
  }
  t.unit0[l.count] = (int)units, t.count = l.count, t.grain = l.grain, t.moved = l.out != nullptr;
  for (int b = 0, i = 0; b <= l.blocks; ++b) {
    while (i + 1 < l.count && t.unit0[i + 1] <= units * b / l.blocks) ++i;
    t.first[b] = (uint16_t)i;
  }
  return LQ_OK;
}

// The passes of a launch's tensors: 1 the sums, 2 the scaling, 3 both at once
template <int N>
int clip_launch(const ClipList& l, int pass, double max_norm, double* sums, int n_sums, float* norm, cudaStream_t st) {
  ClipTable<N> t;
  LQ_TRY(clip_table(t, l));
  cudaError_t e;
  if (pass == 1) {
    e = launch_pdl(clip_norm_kernel<N>, dim3(l.blocks), dim3(kClipThreads), 0, st, t, sums);
  } else if (pass == 2) {
    e = launch_pdl(clip_scale_kernel<N>, dim3(l.blocks), dim3(kClipThreads), 0, st, t, (const double*)sums, n_sums, max_norm, norm);
  } else {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kClipCluster);
    cfg.blockDim = dim3(kClipThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = kClipCluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, clip_small_kernel<N>, t, max_norm, norm);
  }
  LQ_REQUIRE(e == cudaSuccess, LQ_ECUDA, "clip: launch failed: %s", cudaGetErrorString(e));
  return launched("clip");
}
int clip_pass(const ClipList& l, int pass, double max_norm, double* sums, int n_sums, float* norm, cudaStream_t st) {
  if (l.count <= 32) return clip_launch<32>(l, pass, max_norm, sums, n_sums, norm, st);
  if (l.count <= 256) return clip_launch<256>(l, pass, max_norm, sums, n_sums, norm, st);
  if (pass == 3) return LQ_EINVAL;
  return clip_launch<kClipMost>(l, pass, max_norm, sums, n_sums, norm, st);
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
  const auto list = [&](int64_t i0, int grain) {
    ClipList l = {};
    l.count = (int)(count - i0 < kClipMost ? count - i0 : kClipMost);
    if (l.count) l.in = host_in + i0, l.out = host_out ? host_out + i0 : nullptr, l.n = host_n + i0, l.dtype = host_dtype + i0;
    l.grain = grain;
    return l;
  };
  int64_t bytes = 0;
  for (int64_t i = 0; i < count && bytes <= kClipSmall; ++i) bytes += host_n[i] * dtype_size(host_dtype[i]);
  if (bytes <= kClipSmall && count <= 256) {
    ClipList l = list(0, 1);
    l.blocks = kClipCluster;
    return clip_pass(l, 3, max_norm, sums, 0, norm, st);
  }
  int n_sums = 0;
  for (int pass = 1; pass <= 2; ++pass) {
    for (int64_t i0 = 0; i0 < count; i0 += kClipMost) {
      ClipList l = list(i0, kClipVecs);
      int64_t units = 0;
      for (int i = 0; i < l.count; ++i) units += units_of(l.in[i], l.out ? l.out[i] : l.in[i], l.n[i], l.dtype[i], l.grain);
      l.blocks = (int)(units < 1 ? 1 : units < kClipBlocks ? units : kClipBlocks);
      LQ_TRY(clip_pass(l, pass, max_norm, pass == 1 ? sums + n_sums : sums, n_sums, i0 == 0 ? norm : nullptr, st));
      if (pass == 1) n_sums += l.blocks;
    }
  }
  return LQ_OK;
}

// lq_adapters_few.cu -- the adapter bank for a few tokens: out = base + B^T (s A x)
// for each token by a cluster of one to eight blocks, in one launch.
//
// A decode step's product is its adapters' weights once through the SMs, and
// its time the length of the chain: load A, sum over K, exchange, load B, add.
// Each block takes its part of K for all ranks, then its part of the
// columns; the partial sums of a rank meet in distributed shared memory (added
// block by block, in order), and the loads of B and of base do not wait
// for that: they are on their way before the exchange.  Everything is fp32
// with one rounding at the end.
#include "lq_adapters.cuh"

namespace lq {
namespace {

constexpr int kFewThreads = 256, kFewWarps = kFewThreads / 32;
constexpr int kFewAhead = 8;  // ranks of B that a thread has on their way before the exchange

__device__ __forceinline__ float ld_peer(const float* p, uint32_t rank) {
  uint32_t ra;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(rank));
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(ra) : "memory");
  return v;
}

template <typename T>
__device__ __forceinline__ void unpack8(const uint4& w, float* f) {
  const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (sizeof(T) == 2 && Ty<T>::code == LQ_BF16) {
      f[2 * i] = __uint_as_float(x[i] << 16), f[2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u);
    } else {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&x[i]));
      f[2 * i] = p.x, f[2 * i + 1] = p.y;
    }
  }
}

// RW: ranks of a warp (the rank, rounded up, over the block's eight warps); C: blocks
// of a token
template <typename T, int RW, int C>
__global__ void __launch_bounds__(kFewThreads, 2)
    ad_few_kernel(const T* __restrict__ x, int64_t x_stride, const T* __restrict__ a, const T* __restrict__ b,
                  const float* __restrict__ scaling, int R, int K, int N, const int* __restrict__ owner, const T* base,
                  int64_t base_stride, T* out, int64_t out_stride) {
  __shared__ float part[kFewWarps * RW];  // this block's share of each rank's sum
  __shared__ float u[kFewWarps * RW];
  __shared__ float more[kFewThreads * 8];  // sums of the threads that share columns
  pdl_wait();
  pdl_trigger();
  const int64_t t = blockIdx.x / C;
  const int blk = blockIdx.x % C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int o = owner[t];
  const int units = N / 8;  // of 8 columns
  const int c0 = units * blk / C, c1 = units * (blk + 1) / C;
  if (o < 0) {  // the whole cluster
    if (base == out) return;
    for (int c = c0 + tid; c < c1; c += kFewThreads) {
      uint4 y = make_uint4(0u, 0u, 0u, 0u);
      if (base) y = *reinterpret_cast<const uint4*>(base + t * base_stride + 8 * c);
      *reinterpret_cast<uint4*>(out + t * out_stride + 8 * c) = y;
    }
    return;
  }
  // columns: as many threads to 8 of them as there are, each with every G-th rank
  int G = 1;
  while (G < kFewWarps && (c1 - c0) * G * 2 <= kFewThreads) G *= 2;
  const int per = kFewThreads / G, g = tid / per, at = tid - g * per;
  const T* bo = b + (int64_t)o * R * N;
  uint4 bw[kFewAhead], y = make_uint4(0u, 0u, 0u, 0u);
  const bool first = c0 + at < c1;
#pragma unroll
  for (int k = 0; k < kFewAhead; ++k) {
    const int r = g + k * G;
    bw[k] = first && r < R ? __ldg(reinterpret_cast<const uint4*>(bo + (int64_t)r * N + 8 * (c0 + at))) : make_uint4(0u, 0u, 0u, 0u);
  }
  if (first && g == 0 && base) y = *reinterpret_cast<const uint4*>(base + t * base_stride + 8 * (c0 + at));
  // sums over this block's part of K
  const int ku = K / 8, k0 = ku * blk / C, k1 = ku * (blk + 1) / C;
  float s[RW];
#pragma unroll
  for (int j = 0; j < RW; ++j) s[j] = 0.0f;
  const T* xo = x + t * x_stride;
  const T* ao = a + ((int64_t)o * R + warp) * K;
#pragma unroll (RW <= 2 ? 4 : RW <= 4 ? 2 : 1)
  for (int k = k0 + lane; k < k1; k += 32) {
    const uint4 xw = *reinterpret_cast<const uint4*>(xo + 8 * k);
    uint4 aw[RW];
#pragma unroll
    for (int j = 0; j < RW; ++j)
      aw[j] = warp + j * kFewWarps < R ? __ldg(reinterpret_cast<const uint4*>(ao + (int64_t)j * kFewWarps * K + 8 * k)) : make_uint4(0u, 0u, 0u, 0u);
    float xf[8];
    unpack8<T>(xw, xf);
#pragma unroll
    for (int j = 0; j < RW; ++j) {
      float af[8];
      unpack8<T>(aw[j], af);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[j] = fmaf(xf[i], af[i], s[j]);
    }
  }
#pragma unroll
  for (int m = 16; m; m >>= 1)
#pragma unroll
    for (int j = 0; j < RW; ++j) s[j] += __shfl_xor_sync(0xffffffffu, s[j], m);
  if (lane == 0)
#pragma unroll
    for (int j = 0; j < RW; ++j) part[warp + j * kFewWarps] = s[j];
  if (C > 1) asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
  else __syncthreads();
  if (tid < R) {
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < C; ++i) v += C > 1 ? ld_peer(&part[tid], i) : part[tid];
    u[tid] = v * scaling[o];
  }
  if (C > 1) asm volatile("barrier.cluster.arrive.release;" ::: "memory");  // waited for at the end: others may still read part
  __syncthreads();
  for (int c = c0; c < c1; c += per) {
    const bool some = c + at < c1;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    if (some) {
      int r = g;
      if (c == c0) {
#pragma unroll
        for (int k = 0; k < kFewAhead; ++k) {
          float f[8];
          unpack8<T>(bw[k], f);
          const float w = g + k * G < R ? u[g + k * G] : 0.0f;
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = fmaf(w, f[i], v[i]);
        }
        r += kFewAhead * G;
      } else if (g == 0 && base) {
        y = *reinterpret_cast<const uint4*>(base + t * base_stride + 8 * (c + at));
      }
#pragma unroll 8
      for (; r < R; r += G) {
        float f[8];
        unpack8<T>(__ldg(reinterpret_cast<const uint4*>(bo + (int64_t)r * N + 8 * (c + at))), f);
        const float w = u[r];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = fmaf(w, f[i], v[i]);
      }
    }
    if (G > 1) {  // threads share columns where one pass has all of them
#pragma unroll
      for (int i = 0; i < 8; ++i) more[i * kFewThreads + tid] = v[i];
      __syncthreads();
    }
    if (some && g == 0) {
      for (int j = 1; j < G; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += more[i * kFewThreads + j * per + at];
      float f[8];
      unpack8<T>(y, f);
      Vec16<T> w;
#pragma unroll
      for (int i = 0; i < 8; ++i) w.v[i] = Ty<T>::from_f(f[i] + v[i]);
      *reinterpret_cast<uint4*>(out + t * out_stride + 8 * (c + at)) = w.u;
    }
  }
  if (C > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

template <typename T, int RW, int C>
int few_c(const AdCall& a, const void* x, int64_t xs, const void* base, int64_t bs, void* out, int64_t os) {
  const lq_adapter_bank& b = *a.bank;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.n * C));
  cfg.blockDim = dim3(kFewThreads);
  cfg.stream = a.st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = C;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, ad_few_kernel<T, RW, C>, static_cast<const T*>(x), xs, static_cast<const T*>(b.a),
                                           static_cast<const T*>(b.b), b.scaling, (int)b.R, (int)b.K, (int)b.N,
                                           (const int*)a.plan.owner, static_cast<const T*>(base), bs, static_cast<T*>(out), os);
  LQ_REQUIRE(e == cudaSuccess, LQ_ECUDA, "ad_few_kernel launch: %s", cudaGetErrorString(e));
  return launched("ad_few_kernel");
}
// As many blocks to a token as are resident at once, two to an SM; an eighth of
// the room stays empty, since a cluster's blocks lie on one of the chip's groups
// of SMs (37 tokens by 8 blocks 7.9 us, by 4 blocks 4.8; 32 tokens of 14336 columns
// by 8 blocks 5.8, by 4 6.4).  (A third block to an SM,
// with 80 registers, made 5.2 us of 64 tokens 6.9 and 11.7 of 777 13.8.)
template <typename T, int RW>
int few_rw(const AdCall& a, const void* x, int64_t xs, const void* base, int64_t bs, void* out, int64_t os) {
  const int64_t room = num_sms() * 7 / 4;
  if (a.n * 8 <= room) return few_c<T, RW, 8>(a, x, xs, base, bs, out, os);
  if (a.n * 4 <= room) return few_c<T, RW, 4>(a, x, xs, base, bs, out, os);
  if (a.n * 2 <= room) return few_c<T, RW, 2>(a, x, xs, base, bs, out, os);
  return few_c<T, RW, 1>(a, x, xs, base, bs, out, os);
}
template <typename T>
int few_t(const AdCall& a, const void* x, int64_t xs, const void* base, int64_t bs, void* out, int64_t os) {
  switch (ad_padded(a.bank->R)) {
    case 16: return few_rw<T, 2>(a, x, xs, base, bs, out, os);
    case 32: return few_rw<T, 4>(a, x, xs, base, bs, out, os);
    case 64: return few_rw<T, 8>(a, x, xs, base, bs, out, os);
    default: return few_rw<T, 16>(a, x, xs, base, bs, out, os);
  }
}

}  // namespace

int ad_few(const AdCall& a, const void* x, int64_t xs, const void* base, int64_t bs, void* out, int64_t os) {
  return a.bank->dtype == LQ_F16 ? few_t<__half>(a, x, xs, base, bs, out, os) : few_t<__nv_bfloat16>(a, x, xs, base, bs, out, os);
}

}  // namespace lq

// lq_kv4_store.cu -- writing, reading out and evicting of the 4-bit KV cache
// (layout: lq_kv4.cuh).  Compiled without contraction: the quantization below
// is a fixed sequence of fp32 operations.
#include <algorithm>

#include "lq_kv4.cuh"

namespace lq {
namespace {

// ---------------------------------------------------------------------------
// Append.  Per token and head, over its D values, in fp32:
//   lo = min(0, min x), hi = max(0, max x), scale = bf16((hi - lo) / 15),
//   zero = clamp(rint(-lo / scale), 0, 15), code = clamp(rint(x / scale) + zero, 0, 15).
// The range always holds 0, so zero fits 4 bits and 0 is stored exactly.  A
// range that is not finite is stored with a NaN scale and codes 0 (the token
// then reads as NaN); a scale below 2^-100 is stored as 0 (the token reads as
// zeros), which keeps the attention kernels' 1 / scale in range.  The scale is
// rounded once, to bf16, and the codes are taken against the rounded one: its
// 2^-9 costs the far end of the range 0.03 of a step and nothing elsewhere.
// ---------------------------------------------------------------------------
struct AppendArgs {
  const void* x[2];
  int64_t sb[2], sh[2], ss[2];
  int S;
  const int32_t* counts;
};

template <typename T>
__device__ __forceinline__ void load4(const T* p, float* x) {
  if constexpr (sizeof(T) == 4) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(p));
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  } else {
    union {
      uint2 u;
      T t[4];
    } v;
    v.u = __ldg(reinterpret_cast<const uint2*>(p));
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = Ty<T>::to_f(v.t[i]);
  }
}

// Codes (4 nibbles, the first lowest) and parameter word of a token from the
// 4 values of each of its LPT lanes.
template <int LPT>
__device__ __forceinline__ uint32_t quant4(const float* x, uint32_t& par) {
  float lo = fmin_nan(fmin_nan(x[0], x[1]), fmin_nan(x[2], x[3]));
  float hi = fmax_nan(fmax_nan(x[0], x[1]), fmax_nan(x[2], x[3]));
#pragma unroll
  for (int m = LPT / 2; m > 0; m >>= 1) {
    lo = fmin_nan(lo, __shfl_xor_sync(0xffffffffu, lo, m));
    hi = fmax_nan(hi, __shfl_xor_sync(0xffffffffu, hi, m));
  }
  lo = fmin_nan(lo, 0.0f);
  hi = fmax_nan(hi, 0.0f);
  const float s = Ty<__nv_bfloat16>::round(__fdiv_rn(__fsub_rn(hi, lo), 15.0f));
  if (!(s < INFINITY)) {  // NaN or infinite
    par = 0x7fc0u;
    return 0;
  }
  if (s < 7.888609052210118e-31f) {  // 2^-100
    par = 0;
    return 0;
  }
  const float z = fminf(rintf(__fdiv_rn(-lo, s)), 15.0f);
  par = __float_as_uint(z) | (__float_as_uint(s) >> 16);
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float c = fminf(fmaxf(__fadd_rn(rintf(__fdiv_rn(x[i], s)), z), 0.0f), 15.0f);
    w |= (uint32_t)c << (4 * i);
  }
  return w;
}

template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_append_kernel(Kv4 kv, AppendArgs a) {
  constexpr int LPT = D / 4, TPB = 256 / LPT, W = D / 32;  // lanes per token, tokens per block
  const int bh = blockIdx.y, b = bh / kv.H, h = bh % kv.H;
  const int i = blockIdx.x * TPB + threadIdx.x / LPT, l = threadIdx.x % LPT;
  const int cnt = a.counts ? min(max(a.counts[b], 0), a.S) : a.S;
  const int len = kv.len[b];
  const int64_t t = (int64_t)len + i;
  const bool live = i < cnt && t < kv.cap;
  uint32_t par[2], w[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (live) load4(static_cast<const T*>(a.x[s]) + b * a.sb[s] + h * a.sh[s] + i * a.ss[s] + 4 * l, x);
    w[s] = quant4<LPT>(x, par[s]);
  }
  // two lanes make a word of K: even values in its low half, odd ones in its high half
  uint32_t kw = ((w[0] & 0xf) | ((w[0] >> 4) & 0xf0) | ((w[0] << 12) & 0xf0000) | ((w[0] << 8) & 0xf00000)) << (8 * (l & 1));
  kw |= __shfl_xor_sync(0xffffffffu, kw, 1);
  if (live) {
    const int64_t row = (int64_t)bh * kv.cap;
    if (!(l & 1)) *reinterpret_cast<uint32_t*>(kv.k + (row + t) * (D / 2) + 2 * l) = kw;
    *reinterpret_cast<uint16_t*>(kv.v + row * (D / 2) + v_unit(t, l, W)) = (uint16_t)w[1];
    if (l == 0) {
      kv.par[row + t] = make_uint2(par[0], par[1]);
      kv.pos[row + t] = kv.next[b] + i;
      kv.mass[row + t] = 0.0f;
    }
  }
  if (last_block(kv.sync, gridDim.x * gridDim.y)) {
    for (int j = threadIdx.x; j < kv.B; j += blockDim.x) {
      const int n = a.counts ? min(max(a.counts[j], 0), a.S) : a.S, room = kv.cap - kv.len[j];
      kv.len[j] += min(n, room);
      kv.next[j] += min(n, room);
      if (n > room) atomicAdd(&kv.sync[1], n - room);
    }
  }
}

// ---------------------------------------------------------------------------
// Read out the first n slots of every head as values (zeros past a sequence's
// length).
// ---------------------------------------------------------------------------
template <typename T, int N>
__device__ __forceinline__ void store_n(T* p, const float* x) {
  union {
    uint4 u[(N * sizeof(T) + 15) / 16];
    T t[N];
  } v;
#pragma unroll
  for (int i = 0; i < N; ++i) v.t[i] = Ty<T>::from_f(x[i]);
#pragma unroll
  for (int i = 0; i < (int)(N * sizeof(T)) / 16; ++i) st_v4(reinterpret_cast<uint4*>(p) + i, v.u[i]);
}

template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_dequant_kernel(Kv4 kv, int n, T* ko, T* vo) {
  // one warp per tile of 16 tokens and head
  constexpr int W = D / 32;
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int64_t tiles = (n + 15) / 16, item = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (item >= tiles * kv.B * kv.H) return;
  const int64_t bh = item / tiles, t0 = (item % tiles) * 16, row = bh * kv.cap;
  const int len = kv.len[bh / kv.H];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    // K: token g of the half, words c W .. c W + W - 1
    int64_t t = t0 + 8 * half + g;
    if (t < n) {
      const uint32_t* p = reinterpret_cast<const uint32_t*>(kv.k + (row + t) * (D / 2)) + c * W;
      const uint32_t par = t < len ? kv.par[row + t].x : 0;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          x[j] = t < len ? __fmul_rn((float)((p[i] >> (4 * (j >> 1) + 16 * (j & 1))) & 15) - par_zero(par), par_scale(par)) : 0.0f;
        store_n<T, 8>(ko + (bh * n + t) * D + (c * W + i) * 8, x);
      }
    }
    // V: tokens 2c, 2c + 1 of the half, units g W .. g W + W - 1
    const uint32_t* p = reinterpret_cast<const uint32_t*>(kv.v + row * (D / 2) + (t0 >> 4) * (W * 256) + half * (W * 128)) + lane * W;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      t = t0 + 8 * half + 2 * c + e;
      if (t >= n) continue;
      const uint32_t par = t < len ? kv.par[row + t].y : 0;
      float x[4 * W];
#pragma unroll
      for (int i = 0; i < W; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          x[4 * i + j] = t < len ? __fmul_rn((float)((p[i] >> (16 * e + 4 * j)) & 15) - par_zero(par), par_scale(par)) : 0.0f;
      store_n<T, 4 * W>(vo + (bh * n + t) * D + g * (4 * W), x);
    }
  }
}

// ---------------------------------------------------------------------------
// Evict.  One block per (b, h): the keep slots with the greatest keys stay,
// equal keys from the lowest slot up; protected tokens have the greatest key
// of all, NaN weights come next.  The holes below `keep` are filled, in order,
// by the kept tokens at or above it, so that only those move (a slot keeps its
// position beside it, so the order of slots means nothing).
// ---------------------------------------------------------------------------
struct EvictArgs {
  int keep, recent, sinks;
  int32_t* moves;  // [B H, 2, n_moves]: holes, then the tokens that fill them
  int64_t n_moves;
};

constexpr int kEvictThreads = 1024;

__device__ __forceinline__ uint32_t evict_key(const Kv4& kv, int64_t i, int from, int sinks) {
  const int p = kv.pos[i];
  if (p >= from || p < sinks) return 0xffffffffu;
  const float m = kv.mass[i];
  return m != m ? 0x7fffffffu : __float_as_uint(fmaxf(m, 0.0f));
}

// Sum over the block of each thread's flag, before it and in all; two barriers.
__device__ __forceinline__ int block_rank(bool f, int* scratch, int& total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t m = __ballot_sync(0xffffffffu, f);
  __syncthreads();
  if (lane == 0) scratch[warp] = __popc(m);
  __syncthreads();
  int mine = scratch[lane], inc = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += y;
  }
  total = __shfl_sync(0xffffffffu, inc, 31);
  const int before = __shfl_sync(0xffffffffu, inc - mine, warp);
  return before + __popc(m & ((1u << lane) - 1));
}

template <int D>
__global__ void __launch_bounds__(kEvictThreads) kv4_evict_kernel(Kv4 kv, EvictArgs a) {
  __shared__ int hist[2048];
  __shared__ int scratch[32];
  __shared__ int s_bin, s_above;
  constexpr int W = D / 32;
  const int bh = blockIdx.x, b = bh / kv.H, tid = threadIdx.x;
  const int64_t row = (int64_t)bh * kv.cap;
  const int n = min(kv.len[b], kv.cap), keep = a.keep;
  if (n > keep) {
    const int from = kv.next[b] - a.recent;
    // the keep-th greatest key, 11 + 11 + 10 bits at a time
    uint32_t prefix = 0, mask = 0;
    int need = keep;  // of the keys that match the prefix so far
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
      for (int i = tid; i < 2048; i += kEvictThreads) hist[i] = 0;
      __syncthreads();
      for (int t = tid; t < n; t += kEvictThreads) {
        const uint32_t k = evict_key(kv, row + t, from, a.sinks);
        if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1);
      }
      __syncthreads();
      // thread i sums the two bins from the top, 2047 - 2i and 2046 - 2i
      const int hi = hist[2047 - 2 * tid], lo = hist[2046 - 2 * tid];
      int inc = hi + lo;
      const int warp = tid >> 5, lane = tid & 31;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += y;
      }
      if (lane == 31) scratch[warp] = inc;
      __syncthreads();
      int w = scratch[lane];
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, w, d);
        if (lane >= d) w += y;
      }
      const int base = __shfl_sync(0xffffffffu, w, warp) - scratch[warp] + inc - hi - lo;  // in the bins above mine
      if (base < need && base + hi >= need) {
        s_bin = 2047 - 2 * tid;
        s_above = base;
      } else if (base + hi < need && base + hi + lo >= need) {
        s_bin = 2046 - 2 * tid;
        s_above = base + hi;
      }
      __syncthreads();
      prefix |= (uint32_t)s_bin << shift;
      mask |= (uint32_t)(bins - 1) << shift;
      need -= s_above;
      __syncthreads();
    }
    // slots in order: which keys equal to the threshold stay, the holes, the tokens that move
    int32_t* holes = a.moves + (int64_t)bh * 2 * a.n_moves;
    int32_t* late = holes + a.n_moves;
    int equal = 0, n_holes = 0, n_late = 0;
#pragma unroll 1
    for (int t0 = 0; t0 < n; t0 += kEvictThreads) {
      const int t = t0 + tid;
      const uint32_t k = t < n ? evict_key(kv, row + t, from, a.sinks) : 0;
      const bool eq = t < n && k == prefix;
      int total;
      const int er = equal + block_rank(eq, scratch, total);
      equal += total;
      const bool kept = t < n && (k > prefix || (eq && er < need));
      const bool hole = t < keep && !kept, moves = t >= keep && kept;
      const int hr = n_holes + block_rank(hole, scratch, total);
      n_holes += total;
      if (hole) holes[hr] = t;
      const int lr = n_late + block_rank(moves, scratch, total);
      n_late += total;
      if (moves) late[lr] = t;
    }
    __threadfence_block();
    __syncthreads();
    // n_late == n_holes: keep slots stay in all.  A warp moves a token.
    const int lane = tid & 31;
    for (int j = tid >> 5; j < n_late; j += kEvictThreads / 32) {
      const int src = late[j], dst = holes[j];
      uint8_t* kc = kv.k + row * (D / 2);
      uint8_t* vc = kv.v + row * (D / 2);
      if (lane < D / 8) {
        reinterpret_cast<uint32_t*>(kc + (int64_t)dst * (D / 2))[lane] = reinterpret_cast<const uint32_t*>(kc + (int64_t)src * (D / 2))[lane];
      }
      if (lane < D / 4)
        *reinterpret_cast<uint16_t*>(vc + v_unit(dst, lane, W)) = *reinterpret_cast<const uint16_t*>(vc + v_unit(src, lane, W));
      if (lane == 0) {
        kv.par[row + dst] = kv.par[row + src];
        kv.pos[row + dst] = kv.pos[row + src];
        kv.mass[row + dst] = kv.mass[row + src];
      }
    }
    __syncthreads();
    for (int t = keep + tid; t < n; t += kEvictThreads) {
      kv.pos[row + t] = -1;
      kv.mass[row + t] = 0.0f;
    }
  }
  if (last_block(kv.sync, gridDim.x))
    for (int j = tid; j < kv.B; j += kEvictThreads)
      if (kv.len[j] > keep) kv.len[j] = keep, kv.sync[2] = 1;
}

__global__ void __launch_bounds__(256) kv4_reset_kernel(Kv4 kv) {
  const int64_t n = (int64_t)kv.B * kv.H * kv.cap / 4, step = (int64_t)gridDim.x * blockDim.x;
  const int64_t i0 = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  for (int64_t i = i0; i < n; i += step) {
    reinterpret_cast<int4*>(kv.pos)[i] = make_int4(-1, -1, -1, -1);
    reinterpret_cast<float4*>(kv.mass)[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  for (int64_t i = i0; i < 2 * kv.B + 4; i += step) kv.len[i] = 0;
}

template <typename T>
int append_t(const Kv4& kv, const AppendArgs& a, cudaStream_t st) {
  const int tpb = kv.D == 128 ? 8 : 16;
  const dim3 grid((unsigned)((a.S + tpb - 1) / tpb), kv.B * kv.H);
  if (kv.D == 128) kv4_append_kernel<T, 128><<<grid, 256, 0, st>>>(kv, a);
  else kv4_append_kernel<T, 64><<<grid, 256, 0, st>>>(kv, a);
  return launched("kv4_append_kernel");
}

template <typename T>
int dequant_t(const Kv4& kv, int64_t n, void* k, void* v, cudaStream_t st) {
  const int64_t items = (n + 15) / 16 * kv.B * kv.H;
  const unsigned grid = (unsigned)((items + 7) / 8);
  if (kv.D == 128) kv4_dequant_kernel<T, 128><<<grid, 256, 0, st>>>(kv, (int)n, static_cast<T*>(k), static_cast<T*>(v));
  else kv4_dequant_kernel<T, 64><<<grid, 256, 0, st>>>(kv, (int)n, static_cast<T*>(k), static_cast<T*>(v));
  return launched("kv4_dequant_kernel");
}

}  // namespace
}  // namespace lq

extern "C" int lq_kv4_append(const lq_kv4_cache* cache, const void* k, const void* v, int dtype, int64_t S,
                             int64_t k_sb, int64_t k_sh, int64_t k_ss, int64_t v_sb, int64_t v_sh, int64_t v_ss,
                             const int32_t* counts, void* stream) {
  using namespace lq;
  LQ_TRY(kv4_check(cache));
  LQ_REQUIRE(is_float_dtype(dtype), LQ_EDTYPE, "float K / V required");
  LQ_REQUIRE(S >= 0 && S <= (1LL << 30), LQ_EINVAL, "bad chunk length");
  if (S == 0) return LQ_OK;
  LQ_REQUIRE(k && v, LQ_EINVAL, "NULL pointer");
  const uintptr_t vec = 4 * dtype_size(dtype);  // a lane loads 4 values at once
  LQ_REQUIRE(((uintptr_t)k | (uintptr_t)v) % vec == 0 && ((k_sb | k_sh | k_ss | v_sb | v_sh | v_ss) & 3) == 0, LQ_EALIGN,
             "K / V rows must start on multiples of 4 elements");
  const Kv4 kv = kv4_of(cache);
  const AppendArgs a{{k, v}, {k_sb, v_sb}, {k_sh, v_sh}, {k_ss, v_ss}, (int)S, counts};
  cudaStream_t st = as_stream(stream);
  switch (dtype) {
    case LQ_F32: return append_t<float>(kv, a, st);
    case LQ_F16: return append_t<__half>(kv, a, st);
    default: return append_t<__nv_bfloat16>(kv, a, st);
  }
}

extern "C" int lq_kv4_dequant(const lq_kv4_cache* cache, int64_t n, int dtype, void* k, void* v, void* stream) {
  using namespace lq;
  LQ_TRY(kv4_check(cache));
  LQ_REQUIRE(is_float_dtype(dtype), LQ_EDTYPE, "float output required");
  LQ_REQUIRE(n >= 0 && n <= cache->cap, LQ_EINVAL, "%lld slots of %lld", (long long)n, (long long)cache->cap);
  if (n == 0) return LQ_OK;
  LQ_REQUIRE(k && v, LQ_EINVAL, "NULL pointer");
  LQ_REQUIRE(aligned16(k) && aligned16(v), LQ_EALIGN, "outputs must be 16-byte aligned");
  const Kv4 kv = kv4_of(cache);
  cudaStream_t st = as_stream(stream);
  switch (dtype) {
    case LQ_F32: return dequant_t<float>(kv, n, k, v, st);
    case LQ_F16: return dequant_t<__half>(kv, n, k, v, st);
    default: return dequant_t<__nv_bfloat16>(kv, n, k, v, st);
  }
}

extern "C" size_t lq_kv4_evict_workspace_bytes(int64_t B, int64_t H, int64_t cap, int64_t keep) {
  if (B <= 0 || H <= 0 || keep <= 0 || keep >= cap) return 0;
  return (size_t)(B * H) * 2 * (keep < cap - keep ? keep : cap - keep) * sizeof(int32_t);
}

extern "C" int lq_kv4_evict(const lq_kv4_cache* cache, int64_t keep, int64_t recent, int64_t sinks, void* workspace,
                            size_t workspace_bytes, void* stream) {
  using namespace lq;
  LQ_TRY(kv4_check(cache));
  LQ_REQUIRE(keep > 0 && recent >= 0 && sinks >= 0 && recent + sinks <= keep, LQ_EINVAL,
             "keep %lld must be positive and hold the %lld recent and %lld first tokens", (long long)keep,
             (long long)recent, (long long)sinks);
  if (keep >= cache->cap) return LQ_OK;
  const size_t need = lq_kv4_evict_workspace_bytes(cache->B, cache->H, cache->cap, keep);
  LQ_REQUIRE(workspace && workspace_bytes >= need, LQ_EINVAL, "workspace of %zu bytes needed", need);
  const Kv4 kv = kv4_of(cache);
  const EvictArgs a{(int)keep, (int)recent, (int)sinks, static_cast<int32_t*>(workspace),
                    std::min(keep, (int64_t)kv.cap - keep)};
  cudaStream_t st = as_stream(stream);
  if (kv.D == 128) kv4_evict_kernel<128><<<kv.B * kv.H, kEvictThreads, 0, st>>>(kv, a);
  else kv4_evict_kernel<64><<<kv.B * kv.H, kEvictThreads, 0, st>>>(kv, a);
  return launched("kv4_evict_kernel");
}

extern "C" int lq_kv4_reset(const lq_kv4_cache* cache, void* stream) {
  using namespace lq;
  LQ_TRY(kv4_check(cache));
  const Kv4 kv = kv4_of(cache);
  const int64_t n = (int64_t)kv.B * kv.H * kv.cap / 4;
  kv4_reset_kernel<<<resident_grid(kv4_reset_kernel, 256, 0, (n + 255) / 256), 256, 0, as_stream(stream)>>>(kv);
  return launched("kv4_reset_kernel");
}

// lq_kv4_store.cu -- writing, reading out and evicting of the 4-bit KV cache
// (layout: lq_kv4.cuh).  Compiled without contraction: the quantization below
// is a fixed sequence of fp32 operations.
#include <algorithm>
#include <type_traits>

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
union Four {  // values as they are loaded
  typename std::conditional<sizeof(T) == 4, uint4, uint2>::type u;
  T t[4];
  __device__ __forceinline__ Four() : u{} {}
  __device__ __forceinline__ void load(const T* p) { u = __ldg(reinterpret_cast<const decltype(u)*>(p)); }
  __device__ __forceinline__ void to(float* x) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = Ty<T>::to_f(t[i]);
  }
};

// x / y, correctly rounded, from inv = 1 / y correctly rounded: a quotient within
// an ulp, its remainder (exact by fma), and one correction (Markstein); for
// quotients, remainders and y far from over- and underflow.
__device__ __forceinline__ float quotient(float x, float y, float inv) {
  const float q = __fmul_rn(x, inv);
  return __fmaf_rn(__fmaf_rn(-q, y, x), inv, q);
}
// Greatest and least value of a group of LPT neighbouring lanes, NaN if there is one.
template <int LPT>
__device__ __forceinline__ void group_range(float& lo, float& hi) {
  if constexpr (LPT == 32) {
    asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(hi) : "f"(hi));
    asm("redux.sync.min.NaN.f32 %0, %1, 0xffffffff;" : "=f"(lo) : "f"(lo));
  } else {
#pragma unroll
    for (int m = LPT / 2; m > 0; m >>= 1) {
      lo = fmin_nan(lo, __shfl_xor_sync(0xffffffffu, lo, m));
      hi = fmax_nan(hi, __shfl_xor_sync(0xffffffffu, hi, m));
    }
  }
}

// Scale, its reciprocal, zero point and parameter word from a token's range.
struct Grid {
  float s, inv;
  int zero;
  uint32_t par;
};
__device__ __forceinline__ Grid grid_of(float lo, float hi) {
  lo = fmin_nan(lo, 0.0f);
  hi = fmax_nan(hi, 0.0f);
  Grid g;
  g.s = Ty<__nv_bfloat16>::round(quotient(__fsub_rn(hi, lo), 15.0f, 0.066666667f));
  g.inv = __frcp_rn(g.s);
  const bool real = g.s < INFINITY, some = g.s >= 7.888609052210118e-31f;  // not NaN or infinite; 2^-100 or more
  // rint by adding 1.5 * 2^23, whose last mantissa bit is 1
  const float z = fminf(__fsub_rn(__fadd_rn(quotient(-lo, g.s, g.inv), 12582912.0f), 12582912.0f), 15.0f);
  g.par = !real ? 0x7fc0u : some ? __float_as_uint(z) | (__float_as_uint(g.s) >> 16) : 0u;
  g.zero = real && some ? (int)z : 0;
  if (!(real && some)) g.s = g.inv = 0.0f;  // codes 0 for finite values, and something for others
  return g;
}
// Codes of 4 values, the first lowest.  They are not below 0, since the zero
// point is the least value's, but the greatest may reach 16.
// 16-bit values have 11 bits at most and the scale has 8, so a quotient that is
// no tie is 2^-12 or more away from one: both 2 x and (2 k + 1) s are multiples
// of 2^-11 s there.  x / s rounded to 2^-13 (by adding 1.5 * 2^10; the
// reciprocal is off by 2^-20 at most) then goes to the same integer as x / s
// itself, ties included, and no exact quotient is needed.
template <typename T>
__device__ __forceinline__ uint32_t codes4(const float* x, const Grid& g) {
  const int off = g.zero - 0x4b400000;
  uint32_t w = 0;
#pragma unroll
  for (int i = 3; i >= 0; --i) {
    float y;  // 1.5 * 2^23 + rint(x / s)
    if constexpr (sizeof(T) == 2) y = __fadd_rn(__fmaf_rn(x[i], g.inv, 1536.0f), 12582912.0f - 1536.0f);
    else y = __fadd_rn(quotient(x[i], g.s, g.inv), 12582912.0f);
    w = w * 16 + (uint32_t)__viaddmin_s32(__float_as_int(y), off, 15);
  }
  return w & 0xffffu;  // a token that is not finite keeps what it gets to itself
}

// A group of D / 4 lanes takes the two tokens that share words of V (slots 2j,
// 2j + 1), so that V is written in whole words too.  The blocks
// of a head go over its pairs in turn: twice as many blocks as the GPU holds, so that
// heads of unequal lengths even out, and no more, since each counts at the ticket
// (64 heads x up to 2048 tokens: 21.6, 18.7, 20.8 us with 1, 2, 3 times as many).
// 64 registers: 4 blocks per SM (20.3 us with 3).
// Bound by instructions (370 to 512 values; 76 % of the issue slots of SMs that have
// work) and, in that case, by heads of unequal lengths (SMs have work for 76 % of the
// time); 48 MB in 18.9 us are 2.5 TB/s.
template <typename T, int D>
__global__ void __launch_bounds__(256, 4) kv4_append_kernel(Kv4 kv, AppendArgs a, int groups) {
  constexpr int LPT = D / 4, PPB = 256 / LPT, W = D / 32;  // lanes per token, pairs per block
  const int l = threadIdx.x % LPT, pair = threadIdx.x / LPT;
  const int bh = blockIdx.y, b = bh / kv.H, h = bh % kv.H;
  const int cnt = a.counts ? min(max(a.counts[b], 0), a.S) : a.S;
  const int len = kv.len[b], next = kv.next[b];
  const int64_t row = (int64_t)bh * kv.cap;
  const int most = min(cnt, kv.cap - len);  // tokens that find room
  const T* from[2];
#pragma unroll
  for (int s = 0; s < 2; ++s) from[s] = static_cast<const T*>(a.x[s]) + b * a.sb[s] + h * a.sh[s] + 4 * l;
  Four<T> raw[2][2];
  auto first_of = [&](int group) { return 2 * (group * PPB + pair) - (len & 1); };  // first token of the pair
  auto fetch = [&](int group) {
    const int i0 = first_of(group);
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (i0 + e >= 0 && i0 + e < most) raw[e][s].load(from[s] + (i0 + e) * a.ss[s]);
  };
  if ((int)blockIdx.x < groups) fetch(blockIdx.x);
  for (int group = blockIdx.x; group < groups; group += gridDim.x) {
    const int i0 = first_of(group);
    if (i0 - 2 * pair >= cnt) break;  // nothing for the whole block any more
    uint32_t w[2][2];
    const bool live[2] = {i0 >= 0 && i0 < most, i0 + 1 < most};
    float x[2][2][4];
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int s = 0; s < 2; ++s) raw[e][s].to(x[e][s]);
    // the next pair's values arrive while this one's are worked on
    if (group + (int)gridDim.x < groups) fetch(group + gridDim.x);
    // the four ranges (token, K or V); a lane makes the grid of one of them
    float lo = 0.0f, hi = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float* y = x[k >> 1][k & 1];
      float l4 = fmin_nan(fmin_nan(y[0], y[1]), fmin_nan(y[2], y[3]));
      float h4 = fmax_nan(fmax_nan(y[0], y[1]), fmax_nan(y[2], y[3]));
      group_range<LPT>(l4, h4);
      if ((l & 3) == k) lo = l4, hi = h4;
    }
    const Grid mine = grid_of(lo, hi);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int src = (threadIdx.x & 31 & ~3) + k;
      Grid g = mine;
      if constexpr (sizeof(T) == 4) g.s = __shfl_sync(0xffffffffu, mine.s, src);
      g.inv = __shfl_sync(0xffffffffu, mine.inv, src);
      g.zero = __shfl_sync(0xffffffffu, mine.zero, src);
      w[k >> 1][k & 1] = codes4<T>(x[k >> 1][k & 1], g);
    }
    // Two lanes make a word of K, even values in its low half, odd ones in its
    // high half: the even lane the first token's, the odd lane the second's.
    uint32_t kw[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t k = w[e][0];
      kw[e] = ((k & 0xf) | ((k >> 4) & 0xf0) | ((k << 12) & 0xf0000) | ((k << 8) & 0xf00000)) << (8 * (l & 1));
    }
    const uint32_t word = (l & 1 ? kw[1] : kw[0]) | __shfl_xor_sync(0xffffffffu, l & 1 ? kw[0] : kw[1], 1);
    const int64_t t0 = row + len + i0;
    if ((l & 1 ? live[1] : live[0])) *reinterpret_cast<uint32_t*>(kv.k + (t0 + (l & 1)) * (D / 2) + 2 * (l & ~1)) = word;
    // lanes 0-3 have the parameters of both tokens' K and V; 4-7 set positions and weights
    if (l < 4 && (l & 2 ? live[1] : live[0])) reinterpret_cast<uint32_t*>(kv.par + t0)[l] = mine.par;
    if (l >= 4 && l < 8 && (l & 1 ? live[1] : live[0]))
      (l < 6 ? kv.pos : reinterpret_cast<int32_t*>(kv.mass))[t0 + (l & 1)] = l < 6 ? next + i0 + (l & 1) : 0;
    uint8_t* v = kv.v + row * (D / 2) + v_unit((int64_t)len + i0, l, W);  // the pair's word
    if (live[0] && live[1]) *reinterpret_cast<uint32_t*>(v) = w[0][1] | (w[1][1] << 16);
    else if (live[0]) *reinterpret_cast<uint16_t*>(v) = (uint16_t)w[0][1];
    else if (live[1]) *reinterpret_cast<uint16_t*>(v + 2) = (uint16_t)w[1][1];
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
// length).  A warp takes 16 tokens; code - zero is exact in 16 bits (bias + code
// less bias + zero), its product with the scale is rounded once.  Bound by the
// bytes written; each lane writes whole 32-byte sectors
// (64 heads x 8192 tokens of D = 128 to fp16: 56 us, 6.0 TB/s).
// ---------------------------------------------------------------------------
template <typename T> struct Out;
template <> struct Out<__nv_bfloat16> {
  static constexpr uint32_t bias = 0x43004300u;  // 128
  // the pair of values of a pair of codes; z: zero point, s: scale (bf16 pairs)
  __device__ __forceinline__ static uint32_t value(uint32_t c, uint32_t z, uint32_t s) {
    c |= bias;
    __nv_bfloat162 v = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&c), *reinterpret_cast<__nv_bfloat162*>(&z));
    v = __hmul2(v, *reinterpret_cast<__nv_bfloat162*>(&s));
    return *reinterpret_cast<uint32_t*>(&v);
  }
};
__device__ __forceinline__ void st_v8(void* p, const uint32_t* r) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// 16 values of a token from 8 pairs of codes: 32 bytes in 16 bits, 64 in 32
template <typename T>
__device__ __forceinline__ void put16(T* p, const uint32_t* c, uint32_t par, bool live) {
  uint32_t r[16];
  if constexpr (sizeof(T) == 2 && Ty<T>::code == LQ_BF16) {
    const uint32_t z = (uint32_t)(int)par_zero(par) * 0x10001u + Out<T>::bias, s = (par & 0xffffu) * 0x10001u;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = live ? Out<T>::value(c[i], z, s) : 0u;
    st_v8(p, r);
  } else {
    const float z = par_zero(par), s = par_scale(par);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = live ? __fmul_rn((float)(c[i] & 0xffffu) - z, s) : 0.0f;
      const float y = live ? __fmul_rn((float)(c[i] >> 16) - z, s) : 0.0f;
      if constexpr (sizeof(T) == 2) {
        const __half2 v = __floats2half2_rn(x, y);
        r[i] = *reinterpret_cast<const uint32_t*>(&v);
      } else {
        r[2 * i] = __float_as_uint(x), r[2 * i + 1] = __float_as_uint(y);
      }
    }
    st_v8(p, r);
    if constexpr (sizeof(T) == 4) st_v8(p + 8, r + 8);
  }
}

template <typename T>  // 8 values, for head dim 64
__device__ __forceinline__ void put8(T* p, const uint32_t* c, uint32_t par, bool live) {
  const float z = par_zero(par), s = par_scale(par);
  union {
    T t[8];
    uint4 u[sizeof(T) / 2];
  } r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r.t[i] = Ty<T>::from_f(live ? __fmul_rn((float)((c[i / 2] >> (16 * (i & 1))) & 0xffffu) - z, s) : 0.0f);
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) st_v4(reinterpret_cast<uint4*>(p) + i, r.u[i]);
}

template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_dequant_kernel(Kv4 kv, int n, T* ko, T* vo) {
  constexpr int W = D / 32;
  const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int64_t tiles = (n + 15) / 16, item = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (item >= tiles * kv.B * kv.H) return;
  const int64_t bh = item / tiles, t0 = (item % tiles) * 16, row = bh * kv.cap;
  const int len = kv.len[bh / kv.H];
  constexpr uint32_t m = 0x000f000fu;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    // K: token g of the half, words c W .. c W + W - 1, 16 values to two words
    const int64_t t = t0 + 8 * half + g;
    if (t < n) {
      const uint32_t* p = reinterpret_cast<const uint32_t*>(kv.k + (row + t) * (D / 2)) + c * W;
      const uint32_t par = t < len ? kv.par[row + t].x : 0u;
#pragma unroll
      for (int i = 0; i < W; i += 2) {
        const uint2 w = *reinterpret_cast<const uint2*>(p + i);
        const uint32_t x[8] = {w.x & m, (w.x >> 4) & m, (w.x >> 8) & m, (w.x >> 12) & m,
                               w.y & m, (w.y >> 4) & m, (w.y >> 8) & m, (w.y >> 12) & m};
        put16<T>(ko + (bh * n + t) * D + (c * W + i) * 8, x, par, t < len);
      }
    }
    // V: tokens 2c, 2c + 1 of the half, units g W .. g W + W - 1, 4 values to a word
    const uint32_t* p = reinterpret_cast<const uint32_t*>(kv.v + row * (D / 2) + (t0 >> 4) * (W * 256) + half * (W * 128)) + lane * W;
    uint32_t w[W];
#pragma unroll
    for (int i = 0; i < W; i += 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(p + i);
      w[i] = v.x, w[i + 1] = v.y;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int64_t tv = t0 + 8 * half + 2 * c + e;
      if (tv >= n) continue;
      const uint32_t par = tv < len ? kv.par[row + tv].y : 0u;
      uint32_t x[2 * W < 8 ? 8 : 2 * W];
#pragma unroll
      for (int i = 0; i < W; ++i) {  // nibbles (0, 1) and (2, 3) of the token's half
        const uint32_t u = (w[i] >> (16 * e)) & 0xffffu;
        x[2 * i] = (u & 0xfu) | ((u & 0xf0u) << 12);
        x[2 * i + 1] = ((u >> 8) & 0xfu) | ((u & 0xf000u) << 4);
      }
      T* out = vo + (bh * n + tv) * D + g * (4 * W);
      if constexpr (W == 4) put16<T>(out, x, par, tv < len);
      else put8<T>(out, x, par, tv < len);
    }
  }
}

// ---------------------------------------------------------------------------
// Evict.  One block per (b, h): the keep slots with the greatest keys stay,
// equal keys from the lowest slot up; protected tokens have the greatest key
// of all, NaN weights come next.  The holes below `keep` are filled, in order,
// by the kept tokens at or above it, so that only those move (a slot keeps its
// position beside it, so the order of slots means nothing).
// Bound by latency: passes over the keys with barriers between them, then moves
// that one block makes for a head (64 heads x 9216 -> 8192 tokens: 39 us; 32
// heads x 1001 -> 1000: 8.5 us).
// ---------------------------------------------------------------------------
struct EvictArgs {
  int keep, recent, sinks;
  int n_keys;      // keys that shared memory holds
  int lists;       // and it holds the lists of the moves too
  int32_t* moves;  // [B H, 2, n_moves]: holes, then the tokens that fill them
  int64_t n_moves;
};

constexpr int kEvictThreads = 1024;
constexpr int kEvictKeys = 48 * 1024;  // 192 KB

__device__ __forceinline__ uint32_t evict_key(const Kv4& kv, int64_t i, int from, int sinks) {
  const int p = kv.pos[i];
  const float m = kv.mass[i];
  if (p >= from || p < sinks) return 0xffffffffu;
  return m != m ? 0x7fffffffu : __float_as_uint(fmaxf(m, 0.0f));
}

// Ranks of each thread's flags in the block, 10 bits and a total of 11 for each
// of three; two barriers.
__device__ __forceinline__ void block_ranks(const bool* f, uint64_t* scratch, int* before, int* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t m[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) m[i] = __ballot_sync(0xffffffffu, f[i]);
  __syncthreads();
  if (lane == 0) scratch[warp] = (uint64_t)__popc(m[0]) | (uint64_t)__popc(m[1]) << 20 | (uint64_t)__popc(m[2]) << 40;
  __syncthreads();
  const uint64_t mine = scratch[lane];
  uint64_t inc = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint64_t y = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += y;
  }
  const uint64_t all = __shfl_sync(0xffffffffu, inc, 31), base = __shfl_sync(0xffffffffu, inc - mine, warp);
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    before[i] = (int)((base >> (20 * i)) & 0xfffff) + __popc(m[i] & ((1u << lane) - 1));
    total[i] = (int)((all >> (20 * i)) & 0xfffff);
  }
}

template <int W>
__device__ __forceinline__ void ld_vec(const uint8_t* p, uint32_t* w) {
  if constexpr (W == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  }
}

template <int D>
__global__ void __launch_bounds__(kEvictThreads) kv4_evict_kernel(Kv4 kv, EvictArgs a) {
  extern __shared__ uint32_t keys[];
  __shared__ int hist[2048];
  __shared__ int scratch[32];
  __shared__ uint64_t scratch3[32];
  __shared__ int s_bin, s_above, s_inside;
  constexpr int W = D / 32;
  const int bh = blockIdx.x, b = bh / kv.H, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t row = (int64_t)bh * kv.cap;
  const int n = min(kv.len[b], kv.cap), keep = a.keep;
  if (n > keep) {
    const int from = kv.next[b] - a.recent;
    auto key_of = [&](int t) { return t < a.n_keys ? keys[t] : evict_key(kv, row + t, from, a.sinks); };
#pragma unroll 4
    for (int t = tid; t < min(n, a.n_keys); t += kEvictThreads) keys[t] = evict_key(kv, row + t, from, a.sinks);
    // the keep-th greatest key, 11 + 11 + 10 bits at a time (a thread reads back
    // the keys that it wrote)
    uint32_t prefix = 0, mask = 0;
    int need = keep;  // of the keys that match the prefix so far
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
      hist[tid] = hist[tid + 1024] = 0;
      __syncthreads();
#pragma unroll 1
      for (int t0 = 0; t0 < n; t0 += kEvictThreads) {
        const int t = t0 + tid;
        const bool in = t < n;
        const uint32_t k = in ? key_of(t) : 0u;
        const bool match = in && (k & mask) == prefix;
        // protected tokens, and those that never got any weight, are many and
        // lie together: one addition for all that a warp has of them
        const uint32_t safe = __ballot_sync(0xffffffffu, match && k == 0xffffffffu);
        const uint32_t none = __ballot_sync(0xffffffffu, match && k == 0u);
        const int bin = (k >> shift) & (bins - 1);
        if (match && k != 0u && k != 0xffffffffu) atomicAdd(&hist[bin], 1);
        if (lane == 0) {
          if (safe) atomicAdd(&hist[bins - 1], __popc(safe));
          if (none) atomicAdd(&hist[0], __popc(none));
        }
      }
      __syncthreads();
      // thread i sums the two bins from the top, 2047 - 2i and 2046 - 2i
      const int hi = hist[2047 - 2 * tid], lo = hist[2046 - 2 * tid];
      int inc = hi + lo;
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
        s_inside = hi;
      } else if (base + hi < need && base + hi + lo >= need) {
        s_bin = 2046 - 2 * tid;
        s_above = base + hi;
        s_inside = lo;
      }
      __syncthreads();
      prefix |= (uint32_t)s_bin << shift;
      mask |= (uint32_t)(bins - 1) << shift;
      need -= s_above;
      if (s_inside == need) break;  // all of the bin stay: what is below it does not matter
      __syncthreads();
    }
    // Keys above the prefix stay, of those that match it the first `need`.  Slots
    // in order: the holes, the tokens that move.
    int32_t* holes = a.lists ? reinterpret_cast<int32_t*>(keys + a.n_keys) : a.moves + (int64_t)bh * 2 * a.n_moves;
    int32_t* late = holes + a.n_moves;
    int seen[3] = {0, 0, 0};  // keys that match, holes, tokens that move
#pragma unroll 1
    for (int t0 = 0; t0 < n; t0 += kEvictThreads) {
      const int t = t0 + tid;
      const uint32_t k = t < n ? key_of(t) & mask : 0u;
      const bool eq = t < n && k == prefix, above = t < n && k > prefix;
      // where a token's fate hangs on its rank, that comes first
      int before[3], total[3];
      bool kept = above || eq;
      if (__syncthreads_count(eq) + seen[0] > need) {
        const bool f[3] = {eq, false, false};
        block_ranks(f, scratch3, before, total);
        kept = above || (eq && seen[0] + before[0] < need);
      }
      const bool f[3] = {eq, t < keep && !kept, t >= keep && kept};
      block_ranks(f, scratch3, before, total);
      if (f[1]) holes[seen[1] + before[1]] = t;
      if (f[2]) late[seen[2] + before[2]] = t;
#pragma unroll
      for (int i = 0; i < 3; ++i) seen[i] += total[i];
    }
    __threadfence_block();
    __syncthreads();
    // As many move as there are holes: keep slots stay in all.  8 lanes move a token.
    const int l8 = tid & 7;
    uint8_t* kc = kv.k + row * (D / 2);
    uint8_t* vc = kv.v + row * (D / 2);
#pragma unroll 2
    for (int j = tid >> 3; j < seen[2]; j += kEvictThreads / 8) {
      const int src = late[j], dst = holes[j];
      if constexpr (D == 128)
        reinterpret_cast<uint2*>(kc + (int64_t)dst * (D / 2))[l8] = reinterpret_cast<const uint2*>(kc + (int64_t)src * (D / 2))[l8];
      else
        reinterpret_cast<uint32_t*>(kc + (int64_t)dst * (D / 2))[l8] = reinterpret_cast<const uint32_t*>(kc + (int64_t)src * (D / 2))[l8];
      // The lane's units of V lie in one vector, in one half of its words; the other
      // half is the neighbouring slot's.  It is written whole (by halves, the
      // stores were half of the kernel's time): with what the neighbour has, or,
      // if that is a hole too, with what it gets, by the group of the even slot.
      const bool odd = dst & 1;
      const int jn = odd ? j - 1 : j + 1;
      const bool both = jn >= 0 && jn < seen[2] && holes[jn] == (dst ^ 1);
      if (!(both && odd)) {
        const int near = both ? late[jn] : dst ^ 1;
        uint32_t u[W], o[W];
        ld_vec<W>(vc + (v_unit(src, l8 * W, W) & ~(int64_t)3), u);
        ld_vec<W>(vc + (v_unit(near, l8 * W, W) & ~(int64_t)3), o);
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const uint32_t x = (u[i] >> (16 * (src & 1))) & 0xffffu, y = (o[i] >> (16 * (near & 1))) & 0xffffu;
          u[i] = odd ? y | x << 16 : x | y << 16;
        }
        uint8_t* to = vc + (v_unit(dst, l8 * W, W) & ~(int64_t)3);
        if constexpr (W == 4) *reinterpret_cast<uint4*>(to) = make_uint4(u[0], u[1], u[2], u[3]);
        else *reinterpret_cast<uint2*>(to) = make_uint2(u[0], u[1]);
      }
      if (l8 == 0) kv.par[row + dst] = kv.par[row + src];
      if (l8 == 1) kv.pos[row + dst] = kv.pos[row + src];
      if (l8 == 2) kv.mass[row + dst] = kv.mass[row + src];
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

template <typename T, int D>
int append_td(const Kv4& kv, const AppendArgs& a, cudaStream_t st) {
  constexpr int PPB = 1024 / D;                 // pairs per block
  const int groups = (a.S / 2 + 1 + PPB - 1) / PPB;  // a chunk may begin at an odd slot
  const int heads = kv.B * kv.H;
  const int grid = resident_grid(kv4_append_kernel<T, D>, 256, 0, (int64_t)groups * heads);
  kv4_append_kernel<T, D><<<dim3(std::max(1, std::min(groups, 2 * grid / heads)), heads), 256, 0, st>>>(kv, a, groups);
  return launched("kv4_append_kernel");
}
template <typename T>
int append_t(const Kv4& kv, const AppendArgs& a, cudaStream_t st) {
  return kv.D == 128 ? append_td<T, 128>(kv, a, st) : append_td<T, 64>(kv, a, st);
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
  LQ_REQUIRE((((uintptr_t)k | (uintptr_t)v) & 31) == 0, LQ_EALIGN, "outputs must be 32-byte aligned");
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
  const int n_keys = (int)std::min<int64_t>(kv.cap, kEvictKeys);
  const int64_t n_moves = std::min(keep, (int64_t)kv.cap - keep);
  const int lists = n_keys + 2 * n_moves <= kEvictKeys;
  const EvictArgs a{(int)keep, (int)recent, (int)sinks, n_keys, lists, static_cast<int32_t*>(workspace), n_moves};
  const int smem = 4 * (n_keys + (lists ? 2 * (int)n_moves : 0));
  cudaStream_t st = as_stream(stream);
  auto kern = kv.D == 128 ? kv4_evict_kernel<128> : kv4_evict_kernel<64>;
  static DeviceOnce once[2];
  LQ_TRY(once[kv.D == 128].allow_smem((const void*)kern, 4 * kEvictKeys, "kv4_evict_kernel"));
  kern<<<kv.B * kv.H, kEvictThreads, smem, st>>>(kv, a);
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

// lq_kv4_attn.cuh -- what the attention kernels of the 4-bit KV cache share:
// the call's arguments, the visible part of a sequence, the split of the work,
// and the arithmetic of scores.
#pragma once

#include "lq_kv4.cuh"

namespace lq {

struct Attn {
  Kv4 kv;
  const uint8_t* q;
  int q_dtype;
  int64_t q_sb, q_sh, q_ss;
  int Hq, G, Sq, rows, rows_pad;
  const int32_t* counts;
  float sm, cap;  // softmax scale; cap 0: none
  const float* slopes;
  const int32_t* prefix;
  int causal, window;
  int bound;      // tokens of the longest sequence as far as the host knows: for grids, nothing else
  uint32_t g_mul; // ceil(2^32 / G), 0 for G = 1
  int q_wide;     // query rows start on multiples of 16 bytes
  int blocks;     // blocks of the split (at most; never more than there are units)
  uint8_t* out;
  float* part;    // [blocks + B H][rows_pad][D] unnormalised O
  float2* ml;     // [blocks + B H][rows_pad] running reference and sum
  int whole;      // a block to a head: blocks = B H
  float* lse;     // [B H][rows_pad] log2 of the softmax denominators (weights collected), or NULL
  float* scores;  // [B H][cap][pitch] scores, instead of lse, or NULL
  int pitch;
};

constexpr int kPromptRows = 256;
// lq_kv4_prompt.cu: 16-bit queries with many rows; rows_pad is a multiple of
// kPromptRows, part and ml hold 2 * blocks times kPromptRows rows.
int kv4_prompt(const Attn& a, cudaStream_t st);

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// r / G of a row: exact for r G < 2^32 (rows are fewer than 2^20, G at most 4096)
__device__ __forceinline__ int div_g(const Attn& a, int r) { return a.g_mul ? (int)__umulhi((uint32_t)r, a.g_mul) : r; }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// y = cap * tanh(x) of N scores of a thread (cap in log2 units); all lanes of a warp.
// |x| <= 3/4: x + x u P(u), u = x^2, P of degree 4 with the least greatest relative
// error of tanh (2^-24.9; fitted by Remez exchange, 2^-23.6 in fp32), so that a
// score keeps its bits however large the cap.  Above: 1 - 2 / (1 + exp 2x), off by
// 2^-22 of the cap or less, 2^-21 of the score (near 0 it would be 2^-22 of the cap
// still, and a score nothing beside it).  The second form takes two of the
// special-function unit's operations and is left out where the warp has no such score.
__device__ __forceinline__ float f32_of(float x) { return x; }
__device__ __forceinline__ float f32_of(uint32_t x) { return __uint_as_float(x); }
__device__ __forceinline__ void put_f32(float& d, float x) { d = x; }
__device__ __forceinline__ void put_f32(uint32_t& d, float x) { d = __float_as_uint(x); }
template <int N, typename T>  // T: float, or its bits
__device__ __forceinline__ void capped(T* v, float cap) {
  constexpr float kSmall = 0.75f;
  float top = 0.0f;
#pragma unroll
  for (int k = 0; k < N; ++k) top = fmaxf(top, fabsf(f32_of(v[k])));
  auto small = [&](float x) {
    const float u = x * x;
    float p = fmaf(-0.0047694904f, u, 0.019664914f);
    p = fmaf(p, u, -0.053390259f);
    p = fmaf(p, u, 0.13326521f);
    p = fmaf(p, u, -0.33333068f);
    return cap * fmaf(x * u, p, x);
  };
  if (!__any_sync(0xffffffffu, top > kSmall)) {
#pragma unroll
    for (int k = 0; k < N; ++k) put_f32(v[k], small(f32_of(v[k])));
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float x = f32_of(v[k]), y = fmaf(-2.0f * cap, rcp(1.0f + ex2(2.0f * kLog2e * x)), cap);
      put_f32(v[k], fabsf(x) > kSmall ? y : small(x));
    }
  }
}
__device__ __forceinline__ uint32_t h2(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ float2 f2(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
__device__ __forceinline__ void st_out(uint8_t* p, int64_t i, int dt, float v) {
  if (dt == LQ_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (dt == LQ_F16) reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
  else reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

__device__ __forceinline__ void st_out4(uint8_t* p, int64_t i, int dt, float4 v, float f) {
  if (dt == LQ_F32) {
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i) = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
  } else if (dt == LQ_F16) {
    *reinterpret_cast<uint2*>(reinterpret_cast<__half*>(p) + i) = make_uint2(h2(v.x * f, v.y * f), h2(v.z * f, v.w * f));
  } else {
    union {
      __nv_bfloat162 b[2];
      uint2 u;
    } r;
    r.b[0] = __floats2bfloat162_rn(v.x * f, v.y * f);
    r.b[1] = __floats2bfloat162_rn(v.z * f, v.w * f);
    *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p) + i) = r.u;
  }
}

constexpr float pow2(int e) { return e < 0 ? 1.0f / (float)(1u << -e) : (float)(1u << e); }


// New queries of sequence b, and the units that they may see: units [0, pre)
// and [pre + gap, pre + gap + ...), `count` in all.  Slots are positions when
// nothing was evicted (ordered); only then can a window leave units out.
struct Seq {
  int n, cnt, first;  // tokens held, new queries, position of the first of them
  int pre, gap, count;
  int ordered;        // nothing was evicted: slots are positions
};
__device__ __forceinline__ Seq seq_of(const Attn& a, int b) {
  Seq s;
  s.n = min(a.kv.len[b], a.kv.cap);
  s.cnt = a.counts ? min(max(a.counts[b], 0), a.Sq) : a.Sq;
  s.first = a.kv.next[b] - s.cnt;
  s.ordered = a.kv.sync[2] == 0;
  s.pre = s.gap = 0;
  s.count = s.cnt > 0 ? (s.n + kUnit - 1) / kUnit : 0;
  if (a.window > 0 && s.ordered && s.count > 0) {
    const int lo = min(max(s.first - a.window + 1, 0) / kUnit, s.count - 1);
    const int pre = a.prefix ? min(max(a.prefix[b], 0), s.n) : 0;
    s.pre = min((pre + kUnit - 1) / kUnit, lo);
    s.gap = lo - s.pre;
    s.count -= s.gap;
  }
  return s;
}

// The row of all heads' units, cut into equal stretches.  (A unit takes 32 D
// bytes, so that their number fits an int on any GPU.)
struct Cut {
  int units, blocks, base, rem;
  __device__ __forceinline__ void set(int u, int most) {
    units = u;
    blocks = max(min(u, most), 1);
    base = units / blocks;
    rem = units % blocks;
  }
  // units * cta / blocks, and the block that unit x falls to
  __device__ __forceinline__ int begin(int cta) const { return cta * base + cta * rem / blocks; }
  __device__ __forceinline__ int owner(int x) const {
    int c = min((int)__fdividef((x + 0.5f) * blocks, (float)units), blocks - 1);  // or a neighbour
    while (begin(c) > x) --c;
    while (begin(c + 1) <= x) ++c;
    return c;
  }
};
__device__ __forceinline__ int warp_sum(int u) {
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) u += __shfl_xor_sync(0xffffffffu, u, m);
  return u;
}
__device__ __forceinline__ int warp_scan(int u) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, u, d);
    if (lane >= d) u += y;
  }
  return u;
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, float* x) {  // p on a multiple of 4 elements
  if constexpr (sizeof(T) == 4) {
    const float4 u = __ldg(reinterpret_cast<const float4*>(p)), v = __ldg(reinterpret_cast<const float4*>(p) + 1);
    x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
  } else {
    union {
      uint2 u[2];
      T t[8];
    } v;
    v.u[0] = __ldg(reinterpret_cast<const uint2*>(p));
    v.u[1] = __ldg(reinterpret_cast<const uint2*>(p) + 1);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = Ty<T>::to_f(v.t[i]);
  }
}

// P is kept up to 2^kHead above 1 and scaled by 2^kHead: the running reference
// of a row is raised only when a probability would pass 2^(2 kHead - 0.1), so
// most units need no maximum across lanes and no rescaling.
constexpr float kHead = 8.0f, kTop = 15.9f;
constexpr float kNone = -1e30f;  // reference of a row that has seen nothing

}  // namespace
}  // namespace lq

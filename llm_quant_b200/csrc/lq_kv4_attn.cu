// lq_kv4_attn.cu -- attention over the 4-bit KV cache for few query rows
// (layout: lq_kv4.cuh).
//
// out[r, :] = sum_t softmax_t(x[r, t]) v[t, :] with x = sm_scale * q_r . k_t,
// optionally capped, biased and masked; rows r are the G * Sq queries of one
// kv head (r = i G + head of the group).  With k = sk (ck - zk), v = sv (cv - zv):
//   q . k = sk (sum_d q_d ck_d - zk sum_d q_d)
//   out_d = sum_t p_t sv_t cv_td - sum_t p_t sv_t zv_t
// so the tensor cores see bare codes and the zero points cost one fp32 FMA per
// score and one per probability.
//
// Tensor cores (mma.sync.m16n8k16, f16 in, fp32 accumulate):
//   S = K q^T: A = 16 tokens x 16 values of codes, B = 8 query rows;
//   O^T += V^T P^T: A = 16 values x 16 tokens of codes, B = P (8 rows), from the
//   S accumulators by movmatrix.
// A nibble in bits b..b+3 of a half, b <= 6, is the f16 subnormal code * 2^(b - 24),
// exactly: see Nibbles for which b is taken where.  q is scaled per row by a power
// of two that puts its largest value into [2^14, 2^15): every f16 or bf16 value
// within 2^-31 of the row's largest is then exact in f16.  An fp32 query is
// taken as f16 hi + lo (two MMAs, 22 bits), and P likewise; with 16-bit queries
// P is rounded once to f16 (2^-11 of each probability, below the output's own
// rounding), and the zero-point sum uses the rounded value.
// P carries sv: p sv = exp2(x + log2 sv - m) with m the running maximum of
// x + log2 sv, so that it is at most 1 whatever the scales (and times 2^15, so
// that what is small beside it stays a normal f16); the denominator sums
// exp2(x - m).
//
// Split: the 32-token units of all (sequence, kv head) pairs lie in one row,
// and each block takes an equal stretch of it (it may begin and end inside a
// head, and cover several), so that sequences of unequal lengths and few heads
// fill the GPU alike.  The lengths are read on the device.  A head that one
// block covers is finished there; partial results of the others are merged by
// kv4_combine_kernel, a programmatic dependent launch.
#include <algorithm>

#include "lq_kv4.cuh"

namespace lq {
namespace {

constexpr int kWarps = 4;
constexpr float kLog2e = 1.4426950408889634f;

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
  int blocks;     // blocks of the split (at most; never more than there are units)
  uint8_t* out;
  float* part;    // [blocks + B H][rows_pad][D] unnormalised O
  float2* ml;     // [blocks + B H][rows_pad] running maximum and sum
  float* lse;     // [B H][rows_pad] log2 of the softmax denominators (weights collected), or NULL
};

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
// tanh from the exponential: the error is about 2^-23 absolute, which is what a
// capped score needs (tanh.approx is only good to 2^-11)
__device__ __forceinline__ float tanh_exp(float x) {
  return 1.0f - __fdividef(2.0f, 1.0f + ex2(2.0f * kLog2e * x));
}
__device__ __forceinline__ uint32_t h2(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ float2 f2(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
__device__ __forceinline__ void mma16(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ float ld_q(const uint8_t* p, int64_t i, int dt) {
  if (dt == LQ_F32) return reinterpret_cast<const float*>(p)[i];
  if (dt == LQ_F16) return __half2float(reinterpret_cast<const __half*>(p)[i]);
  return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void st_out(uint8_t* p, int64_t i, int dt, float v) {
  if (dt == LQ_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (dt == LQ_F16) reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
  else reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// Fragment registers from a word of codes: nibble n of both halves as f16.
// The tensor cores align a subnormal's product by the exponent 2^-14 it would
// have as a normal number, and cut below 24 bits: a code whose unit is 2^(b -
// 24) loses what is under 2^(-14 - b) of that unit, times the largest factor it
// meets.  That is nothing beside a 16-bit output, so V takes nibbles where they
// are with a mask and one shift for two (b = 0 and 4: 5 instructions for 8
// codes); scores decide collected weights in fp32, so K is shifted to b = 4 (7);
// with fp32 queries K and V are shifted to b = 6 (8).
enum Place { kMixed, kFour, kSix };
template <Place P>
struct Nibbles {
  // log2 of the unit of nibble n
  __host__ __device__ static constexpr int unit(int n) { return P == kMixed ? ((n & 1) ? -20 : -24) : P == kFour ? -20 : -18; }
  __device__ __forceinline__ static void take(uint32_t w, uint32_t* r) {
    if constexpr (P == kMixed) {
      const uint32_t v = w >> 8;
      r[0] = w & 0x000f000fu, r[1] = w & 0x00f000f0u, r[2] = v & 0x000f000fu, r[3] = v & 0x00f000f0u;
    } else if constexpr (P == kFour) {
      r[0] = (w << 4) & 0x00f000f0u, r[1] = w & 0x00f000f0u, r[2] = (w >> 4) & 0x00f000f0u, r[3] = (w >> 8) & 0x00f000f0u;
    } else {
      r[0] = (w << 6) & 0x03c003c0u, r[1] = (w << 2) & 0x03c003c0u, r[2] = (w >> 2) & 0x03c003c0u, r[3] = (w >> 6) & 0x03c003c0u;
    }
  }
};
constexpr float pow2(int e) { return e < 0 ? 1.0f / (float)(1u << -e) : (float)(1u << e); }

// W aligned words (16 or 8 bytes) of codes
template <int W>
__device__ __forceinline__ void ld_codes(const uint8_t* p, uint32_t* w) {
  if constexpr (W == 4) {
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "l"(p));
  } else {
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
  }
}

// New queries of sequence b, and the units that they may see: units [0, pre)
// and [pre + gap, pre + gap + ...), `count` in all.  Slots are positions when
// nothing was evicted (ordered); only then can a window leave units out.
struct Seq {
  int n, cnt, first;  // tokens held, new queries, position of the first of them
  int pre, gap, count;
  bool ordered;  // nothing was evicted: slots are positions
};
__device__ __forceinline__ Seq seq_of(const Attn& a, int b) {
  Seq s;
  s.n = min(a.kv.len[b], a.kv.cap);
  s.cnt = a.counts ? min(max(a.counts[b], 0), a.Sq) : a.Sq;
  s.first = a.kv.next[b] - s.cnt;
  s.pre = s.gap = 0;
  s.ordered = a.kv.sync[2] == 0;
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

// Units of all heads; every warp computes it for itself.
__device__ __forceinline__ int64_t all_units(const Attn& a) {
  int64_t u = 0;
  for (int b = threadIdx.x & 31; b < a.kv.B; b += 32) u += seq_of(a, b).count;
#pragma unroll
  for (int m = 16; m > 0; m >>= 1) u += __shfl_xor_sync(0xffffffffu, u, m);
  return u * a.kv.H;
}

// Sequence that holds unit x of the row of units, and where it begins.
__device__ __forceinline__ int seq_at(const Attn& a, int64_t x, int64_t& begin) {
  const int lane = threadIdx.x & 31;
  int64_t base = 0;
  for (int b0 = 0; b0 < a.kv.B; b0 += 32) {
    const int b = b0 + lane;
    int64_t inc = b < a.kv.B ? (int64_t)seq_of(a, b).count * a.kv.H : 0;
    const int64_t own = inc;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += y;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, base + inc > x);
    if (hit) {
      const int src = __ffs(hit) - 1;
      begin = base + __shfl_sync(0xffffffffu, inc - own, src);
      return b0 + src;
    }
    base += __shfl_sync(0xffffffffu, inc, 31);
  }
  begin = base;
  return a.kv.B;
}

// Queries of a block's rows as B fragments, and what each score column needs.
template <int D, int NQ, bool QLO>
struct Rows {
  static constexpr int W = D / 32;
  uint32_t hi[NQ][W][4], lo[QLO ? NQ : 1][QLO ? W : 1][4];
  float sum[NQ][2], fac[NQ][2];  // of columns 2c, 2c + 1: sum of q, factor that undoes the scaling
  float slope[NQ][2];
  int at[NQ][2];                 // position of the query; INT_MIN: no such row

  __device__ __forceinline__ void load(const Attn& a, const Seq& s, int b, int h, int zb, bool gen) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
      const int r = zb * 8 * NQ + 8 * nq + g, i = r / a.G;
      float x[8 * W];
#pragma unroll
      for (int d = 0; d < 8 * W; ++d) x[d] = 0.0f;
      if (r < a.rows && i < s.cnt) {
        const int64_t off = b * a.q_sb + (int64_t)(h * a.G + r % a.G) * a.q_sh + i * a.q_ss + c * (8 * W);
#pragma unroll
        for (int d = 0; d < 8 * W; ++d) x[d] = ld_q(a.q, off + d, a.q_dtype);
      }
      float mx = 0.0f;
#pragma unroll
      for (int d = 0; d < 8 * W; ++d) mx = fmaxf(mx, fabsf(x[d]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      // 2^(14 - exponent of mx), kept a normal number
      const int e = (int)(__float_as_uint(mx) >> 23);
      const int up = mx > 0.0f && e < 255 ? min(268 - e, 254) : 127;
      const float f = __uint_as_float((uint32_t)max(up, 1) << 23);
      float sum = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w)
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // register j: nibbles (n, n + 4), n = 0, 2, 1, 3
          const int n = 8 * w + (j < 2 ? 2 * j : 2 * j - 3);
          const float u = x[n] * f, v = x[n + 4] * f;
          const uint32_t p = h2(u, v);
          const float2 y = f2(p);
          hi[nq][w][j] = p;
          sum += y.x + y.y;
          if constexpr (QLO) {
            lo[nq][w][j] = h2(u - y.x, v - y.y);
            const float2 y2 = f2(lo[nq][w][j]);
            sum += y2.x + y2.y;
          }
        }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      // the accumulators hold `unit` times the true sums
      constexpr float unit = pow2(Nibbles<QLO ? kSix : kFour>::unit(0));
      const float back = a.sm / f * (1.0f / unit);
#pragma unroll
      for (int e2 = 0; e2 < 2; ++e2) {
        const int src = (2 * c + e2) * 4;
        this->sum[nq][e2] = __shfl_sync(0xffffffffu, sum, src) * unit;
        fac[nq][e2] = __shfl_sync(0xffffffffu, back, src) * (gen && a.cap > 0.0f ? 1.0f / a.cap : kLog2e);
        const int rc = zb * 8 * NQ + 8 * nq + 2 * c + e2, ic = rc / a.G;
        at[nq][e2] = rc < a.rows && ic < s.cnt ? s.first + ic : INT_MIN;
        slope[nq][e2] = gen && a.slopes && rc < a.rows ? a.slopes[h * a.G + rc % a.G] * kLog2e : 0.0f;
      }
    }
  }
};

// Scores (in log2 units) of one 16-token tile: x[nq][0..3] = (token g, column
// 2c), (g, 2c + 1), (g + 8, 2c), (g + 8, 2c + 1); -inf where the query does not see the token.
template <int D, int NQ, bool QLO, bool GEN>
__device__ __forceinline__ void tile_scores(const Attn& a, const Rows<D, NQ, QLO>& q, const uint32_t* k0,
                                            const uint32_t* k1, const uint32_t* par, const int* tok, const int* pos,
                                            int n, int pre, float (*x)[4]) {
  constexpr int W = D / 32;
  float s0[NQ][4], s1[NQ][4];
#pragma unroll
  for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
    for (int u = 0; u < 4; ++u) s0[nq][u] = s1[nq][u] = 0.0f;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    uint32_t ka[4], kb[4];
    Nibbles<QLO ? kSix : kFour>::take(k0[w], ka);
    Nibbles<QLO ? kSix : kFour>::take(k1[w], kb);
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
      mma16(s0[nq], ka[0], kb[0], ka[2], kb[2], q.hi[nq][w][0], q.hi[nq][w][1]);
      mma16(s1[nq], ka[1], kb[1], ka[3], kb[3], q.hi[nq][w][2], q.hi[nq][w][3]);
      if constexpr (QLO) {
        mma16(s0[nq], ka[0], kb[0], ka[2], kb[2], q.lo[nq][w][0], q.lo[nq][w][1]);
        mma16(s1[nq], ka[1], kb[1], ka[3], kb[3], q.lo[nq][w][2], q.lo[nq][w][3]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float sk = par_scale(par[j]), zk = par_zero(par[j]);
    const bool in = tok[j] < n;
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int u = 2 * j + e;
        float v = s0[nq][u] + s1[nq][u];
        v = fmaf(-zk, q.sum[nq][e], v) * (sk * q.fac[nq][e]);
        bool sees = in;
        if constexpr (GEN) {
          if (a.cap > 0.0f) v = tanh_exp(v) * (a.cap * kLog2e);
          const int back = q.at[nq][e] - pos[j];
          if (a.slopes) v = fmaf(-q.slope[nq][e], fabsf((float)back), v);
          bool near = true;
          if (a.causal) near = back >= 0;
          if (a.window > 0) near = near && back < a.window;
          sees = in && (near || pos[j] < pre) && q.at[nq][e] != INT_MIN;
        }
        x[nq][u] = sees ? v : -INFINITY;
      }
  }
}

// Positions of a lane's tokens (general masks only).
__device__ __forceinline__ void load_pos(const Attn& a, int64_t row, const int* tok, const Seq& s, int* pos, int count) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < count) pos[j] = s.ordered || tok[j] >= s.n ? tok[j] : a.kv.pos[row + tok[j]];
}

template <int D, int NQ, bool QLO, bool GEN>
__global__ void __launch_bounds__(32 * kWarps, NQ == 1 && !QLO && !GEN ? 4 : 2) kv4_attn_kernel(const Attn a) {
  constexpr int W = D / 32, NR = 8 * NQ;
  using VN = Nibbles<QLO ? kSix : kMixed>;
  __shared__ float ob[kWarps][NR][D + 1];
  __shared__ float2 mlb[kWarps][NR];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int zb = blockIdx.y, cta = blockIdx.x;
  const int64_t units = all_units(a);
  const int64_t blocks = units < a.blocks ? units : a.blocks;
  if (cta >= blocks) return;
  int64_t x0 = cta * units / blocks;
  const int64_t x1 = (cta + 1) * units / blocks;
  int64_t seq_begin;
  int b = seq_at(a, x0, seq_begin);
  Seq s = seq_of(a, b);

  while (x0 < x1) {
    while (x0 >= seq_begin + (int64_t)s.count * a.kv.H) {  // next sequence that has units
      seq_begin += (int64_t)s.count * a.kv.H;
      s = seq_of(a, ++b);
    }
    const int h = (int)((x0 - seq_begin) / s.count);
    const int u0 = (int)((x0 - seq_begin) % s.count);
    const int u1 = (int)min((int64_t)s.count, u0 + (x1 - x0));
    const int bh = b * a.kv.H + h;
    const int64_t row = (int64_t)bh * a.kv.cap;
    const uint8_t* kc = a.kv.k + row * (D / 2);
    const uint8_t* vc = a.kv.v + row * (D / 2);
    const int pre = GEN && a.prefix ? a.prefix[b] : 0;
    Rows<D, NQ, QLO> q;
    q.load(a, s, b, h, zb, GEN);

    float m[NQ][2], l[NQ][2], z[NQ][2], O[NQ][2 * W][4];
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
      for (int e = 0; e < 2; ++e) m[nq][e] = -INFINITY, l[nq][e] = z[nq][e] = 0.0f;
#pragma unroll
      for (int e = 0; e < 2 * W; ++e)
#pragma unroll
        for (int u = 0; u < 4; ++u) O[nq][e][u] = 0.0f;
    }
    uint32_t kw[4][W], vw[4][W];
    uint2 pw[4];
    auto token = [&](int u) { return (u < s.pre ? u : u + s.gap) * kUnit; };
    auto load_k = [&](int t0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ld_codes<W>(kc + (int64_t)(t0 + 8 * j) * (D / 2) + lane * (4 * W), kw[j]);
        pw[j] = __ldg(a.kv.par + row + t0 + 8 * j + g);
      }
    };
    auto load_v = [&](int t0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) ld_codes<W>(vc + (int64_t)(t0 + 8 * j) * (D / 2) + lane * (4 * W), vw[j]);
    };
    int u = u0 + warp;
    if (u < u1) {
      load_k(token(u));
      load_v(token(u));
    }
    for (; u < u1; u += kWarps) {
      const int t0 = token(u), t_next = token(u + kWarps);
      const bool more = u + kWarps < u1;
      int tok[4], pos[4];
      uint32_t kp[4], vp[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) tok[j] = t0 + 8 * j + g, kp[j] = pw[j].x, vp[j] = pw[j].y;
      if constexpr (GEN) load_pos(a, row, tok, s, pos, 4);
      float x[2][NQ][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
        tile_scores<D, NQ, QLO, GEN>(a, q, kw[2 * i], kw[2 * i + 1], kp + 2 * i, tok + 2 * i, pos + 2 * i, s.n, pre, x[i]);
      if (more) load_k(t_next);

      // log2 of the V scales; a scale of 0 has only zeros behind it
      float lv[4], zv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float sv = par_scale(vp[j]);
        lv[j] = sv == 0.0f ? -100.0f : lg2(sv);
        zv[j] = par_zero(vp[j]);
      }
      uint32_t pb[NQ][4], pl[QLO ? NQ : 1][4];
#pragma unroll
      for (int nq = 0; nq < NQ; ++nq) {
        float p[2][4], alpha[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float xs[4], w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            xs[j] = x[j >> 1][nq][2 * (j & 1) + e];
            w[j] = xs[j] == -INFINITY ? -INFINITY : xs[j] + lv[j];
          }
          float mt = fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3]));
          mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 4));
          mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 8));
          mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 16));
          const float mn = fmaxf(m[nq][e], mt), ref = mn == -INFINITY ? 0.0f : mn, ref15 = ref - 15.0f;
          alpha[e] = ex2(m[nq][e] - ref);
          m[nq][e] = mn;
          l[nq][e] *= alpha[e];
          z[nq][e] *= alpha[e];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            l[nq][e] += ex2(xs[j] - ref);
            p[j >> 1][2 * (j & 1) + e] = ex2(w[j] - ref15);
          }
        }
        if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
          for (int d = 0; d < 2 * W; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) O[nq][d][i] *= alpha[i & 1];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float pa = p[j >> 1][2 * (j & 1)], pc = p[j >> 1][2 * (j & 1) + 1];
          const uint32_t r = h2(pa, pc);
          const float2 rf = f2(r);
          // tokens past the end have p = 0, but their zero point may be anything
          const float zj = tok[j] < s.n ? zv[j] : 0.0f;
          if constexpr (QLO) {
            const uint32_t rl = h2(pa - rf.x, pc - rf.y);
            const float2 rlf = f2(rl);
            pl[nq][j] = transposed(rl);
            z[nq][0] = fmaf(rf.x + rlf.x, zj, z[nq][0]);
            z[nq][1] = fmaf(rf.y + rlf.y, zj, z[nq][1]);
          } else {
            z[nq][0] = fmaf(rf.x, zj, z[nq][0]);
            z[nq][1] = fmaf(rf.y, zj, z[nq][1]);
          }
          pb[nq][j] = transposed(r);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int w = 0; w < W; ++w) {
          uint32_t va[4], vb[4];
          VN::take(vw[2 * i][w], va);
          VN::take(vw[2 * i + 1][w], vb);
#pragma unroll
          for (int nq = 0; nq < NQ; ++nq) {
            mma16(O[nq][2 * w], va[0], va[2], vb[0], vb[2], pb[nq][2 * i], pb[nq][2 * i + 1]);
            mma16(O[nq][2 * w + 1], va[1], va[3], vb[1], vb[3], pb[nq][2 * i], pb[nq][2 * i + 1]);
            if constexpr (QLO) {
              mma16(O[nq][2 * w], va[0], va[2], vb[0], vb[2], pl[nq][2 * i], pl[nq][2 * i + 1]);
              mma16(O[nq][2 * w + 1], va[1], va[3], vb[1], vb[3], pl[nq][2 * i], pl[nq][2 * i + 1]);
            }
          }
        }
      if (more) load_v(t_next);
    }

    // ---- merge the warps: O in true units, minus the zero points' share ----
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) {
          l[nq][e] += __shfl_xor_sync(0xffffffffu, l[nq][e], k);
          z[nq][e] += __shfl_xor_sync(0xffffffffu, z[nq][e], k);
        }
        if (g == 0) mlb[warp][8 * nq + 2 * c + e] = make_float2(m[nq][e], l[nq][e]);
      }
#pragma unroll
      for (int d = 0; d < 2 * W; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          ob[warp][8 * nq + 2 * c + (i & 1)][(g * W + d / 2) * 4 + (d & 1) + 2 * (i >> 1)] =
              fmaf(O[nq][d][i], pow2(-VN::unit(d & 1)), -z[nq][i & 1]) * pow2(-15);
    }
    __syncthreads();
    const bool whole = u0 == 0 && u1 == s.count;
    const int64_t slot = ((int64_t)cta + bh) * a.rows_pad;
    for (int i = threadIdx.x; i < NR * D; i += 32 * kWarps) {
      const int r = i / D, d = i % D, qr = zb * NR + r;
      if (qr >= a.rows) break;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) M = fmaxf(M, mlb[w][r].x);
      const float ref = M == -INFINITY ? 0.0f : M;
      float o = 0.0f, L = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = ex2(mlb[w][r].x - ref);
        o = fmaf(f, ob[w][r][d], o);
        L = fmaf(f, mlb[w][r].y, L);
      }
      if (whole) {
        const int iq = qr / a.G, hq = h * a.G + qr % a.G;
        st_out(a.out, (((int64_t)b * a.Hq + hq) * a.Sq + iq) * D + d, a.q_dtype, L == 0.0f ? 0.0f : o / L);
        if (a.lse && d == 0) a.lse[(int64_t)bh * a.rows_pad + qr] = L == 0.0f ? INFINITY : ref + lg2(L);
      } else {
        a.part[(slot + qr) * D + d] = o;
        if (d == 0) a.ml[slot + qr] = make_float2(M, L);
      }
    }
    __syncthreads();
    x0 += u1 - u0;
  }
  if (threadIdx.x == 0) pdl_trigger();
}

// One block per (row, head): merges the partial results of the blocks that
// shared the head; zeros where there is nothing to see.  Heads that one block
// covered are done already.
__global__ void __launch_bounds__(128) kv4_combine_kernel(const Attn a) {
  pdl_wait();
  const int bh = blockIdx.y, b = bh / a.kv.H, h = bh % a.kv.H, qr = blockIdx.x, D = a.kv.D, d = threadIdx.x;
  const int64_t units = all_units(a);
  const int64_t blocks = units < a.blocks ? units : a.blocks;
  const Seq s = seq_of(a, b);
  float o = 0.0f, L = 0.0f, ref = 0.0f;
  if (s.count > 0) {
    int64_t begin = 0;  // units of the sequences before b
    for (int j = threadIdx.x & 31; j < b; j += 32) begin += seq_of(a, j).count;
#pragma unroll
    for (int m = 16; m > 0; m >>= 1) begin += __shfl_xor_sync(0xffffffffu, begin, m);
    begin = begin * a.kv.H + (int64_t)h * s.count;
    const int64_t c0 = ((begin + 1) * blocks - 1) / units, c1 = ((begin + s.count) * blocks - 1) / units;
    if (c0 == c1) return;
    float M = -INFINITY;
    for (int64_t c = c0; c <= c1; ++c) M = fmaxf(M, a.ml[(c + bh) * a.rows_pad + qr].x);
    ref = M == -INFINITY ? 0.0f : M;
    for (int64_t c = c0; c <= c1; ++c) {
      const int64_t i = (c + bh) * a.rows_pad + qr;
      const float2 ml = a.ml[i];
      const float f = ex2(ml.x - ref);
      o = fmaf(f, d < D ? a.part[i * D + d] : 0.0f, o);
      L = fmaf(f, ml.y, L);
    }
  }
  const int iq = qr / a.G, hq = h * a.G + qr % a.G;
  if (d < D) st_out(a.out, (((int64_t)b * a.Hq + hq) * a.Sq + iq) * D + d, a.q_dtype, L == 0.0f ? 0.0f : o / L);
  if (a.lse && d == 0) a.lse[(int64_t)bh * a.rows_pad + qr] = L == 0.0f ? INFINITY : ref + lg2(L);
}

// mass[t] += sum over the rows of exp2(x[r, t] - lse[r]).  A warp owns 16
// tokens and goes over all rows, so that no two threads add to one token and
// the order of the sum is fixed.
template <int D, bool QLO, bool GEN>
__global__ void __launch_bounds__(128) kv4_mass_kernel(const Attn a) {
  constexpr int W = D / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int bh = blockIdx.y, b = bh / a.kv.H, h = bh % a.kv.H;
  const Seq s = seq_of(a, b);
  const int pre = GEN && a.prefix ? a.prefix[b] : 0;
  const int64_t row = (int64_t)bh * a.kv.cap;
  for (int t0 = (blockIdx.x * 4 + warp) * 16; t0 < s.n && s.cnt > 0; t0 += gridDim.x * 64) {
    uint32_t kw[2][W], kp[2];
    int tok[2], pos[4];
    float sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      ld_codes<W>(a.kv.k + (row + t0 + 8 * j) * (D / 2) + lane * (4 * W), kw[j]);
      tok[j] = t0 + 8 * j + g;
      kp[j] = a.kv.par[row + tok[j]].x;
    }
    if constexpr (GEN) load_pos(a, row, tok, s, pos, 2);
    for (int zb = 0; zb * 8 < a.rows; ++zb) {
      Rows<D, 1, QLO> q;
      q.load(a, s, b, h, zb, GEN);
      float x[1][4];
      tile_scores<D, 1, QLO, GEN>(a, q, kw[0], kw[1], kp, tok, pos, s.n, pre, x);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int qr = zb * 8 + 2 * c + e;
        if (qr >= a.rows) continue;
        const float lse = a.lse[(int64_t)bh * a.rows_pad + qr];
        sum[0] += ex2(x[0][e] - lse);
        sum[1] += ex2(x[0][2 + e] - lse);
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 1);
      sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 2);
      if (c == 0 && tok[j] < s.n) a.kv.mass[row + tok[j]] += sum[j];
    }
  }
}

// Rows of a block, and blocks of the split: one wave of 4 blocks per SM over
// all row blocks, and at least one unit per warp.
struct Plan {
  int nq, row_blocks, rows_pad, blocks;
};
Plan plan_of(const Kv4& kv, int64_t rows, int64_t bound) {
  Plan p;
  p.nq = rows <= 8 ? 1 : 2;
  p.row_blocks = (int)((rows + 8 * p.nq - 1) / (8 * p.nq));
  p.rows_pad = p.row_blocks * 8 * p.nq;
  const int64_t units = (int64_t)kv.B * kv.H * ((std::max<int64_t>(bound, 1) + kUnit - 1) / kUnit);
  const int64_t slots = std::max<int64_t>(1, (int64_t)num_sms() * 4 / p.row_blocks);
  p.blocks = (int)std::max<int64_t>(1, std::min<int64_t>(slots, (units + kWarps - 1) / kWarps));
  return p;
}

// part, ml, lse
void spaces(const Kv4& kv, const Plan& p, bool weigh, size_t* bytes) {
  const size_t slots = (size_t)(p.blocks + kv.B * kv.H) * p.rows_pad;
  bytes[0] = slots * kv.D * sizeof(float);
  bytes[1] = slots * sizeof(float2);
  bytes[2] = weigh ? (size_t)kv.B * kv.H * p.rows_pad * sizeof(float) : 0;
}

template <int D, int NQ, bool QLO, bool GEN>
int run_attn(const Attn& a, const Plan& p, cudaStream_t st) {
  kv4_attn_kernel<D, NQ, QLO, GEN><<<dim3(p.blocks, p.row_blocks), 32 * kWarps, 0, st>>>(a);
  LQ_TRY(launched("kv4_attn_kernel"));
  launch_pdl(kv4_combine_kernel, dim3(a.rows, a.kv.B * a.kv.H), dim3(D), 0, st, a);
  LQ_TRY(launched("kv4_combine_kernel"));
  if (a.lse) {
    kv4_mass_kernel<D, QLO, GEN><<<dim3((a.kv.cap + 63) / 64, a.kv.B * a.kv.H), 128, 0, st>>>(a);
    LQ_TRY(launched("kv4_mass_kernel"));
  }
  return LQ_OK;
}
template <int D, bool QLO, bool GEN>
int run_attn_nq(const Attn& a, const Plan& p, cudaStream_t st) {
  return p.nq == 1 ? run_attn<D, 1, QLO, GEN>(a, p, st) : run_attn<D, 2, QLO, GEN>(a, p, st);
}
template <int D>
int run_attn_d(const Attn& a, const Plan& p, bool gen, cudaStream_t st) {
  if (a.q_dtype == LQ_F32) return gen ? run_attn_nq<D, true, true>(a, p, st) : run_attn_nq<D, true, false>(a, p, st);
  return gen ? run_attn_nq<D, false, true>(a, p, st) : run_attn_nq<D, false, false>(a, p, st);
}

}  // namespace
}  // namespace lq

extern "C" size_t lq_kv4_attention_workspace_bytes(const lq_kv4_cache* cache, int q_dtype, int64_t Hq, int64_t Sq,
                                                   int64_t bound, int accumulate) {
  using namespace lq;
  (void)q_dtype;
  if (kv4_check(cache) != LQ_OK || Hq <= 0 || Sq <= 0 || Hq % cache->H) return 0;
  const Kv4 kv = kv4_of(cache);
  size_t b[3];
  spaces(kv, plan_of(kv, Hq / cache->H * Sq, bound), accumulate != 0, b);
  return b[0] + b[1] + b[2];
}

extern "C" int lq_kv4_attention(const lq_kv4_cache* cache, const void* q, int q_dtype, int64_t Hq, int64_t Sq,
                                int64_t q_sb, int64_t q_sh, int64_t q_ss, int64_t bound, const int32_t* counts,
                                float sm_scale, int causal, float softcap, const float* slopes, int64_t window,
                                const int32_t* prefix, int accumulate, void* out, void* workspace,
                                size_t workspace_bytes, void* stream) {
  using namespace lq;
  LQ_TRY(kv4_check(cache));
  LQ_REQUIRE(is_float_dtype(q_dtype), LQ_EDTYPE, "float query required");
  LQ_REQUIRE(Hq > 0 && Hq % cache->H == 0, LQ_EINVAL, "query heads %lld not a multiple of kv heads %lld",
             (long long)Hq, (long long)cache->H);
  LQ_REQUIRE(Sq >= 0 && bound >= 0, LQ_EINVAL, "bad shape");
  LQ_REQUIRE(softcap >= 0.0f, LQ_EINVAL, "softcap must not be negative");
  LQ_REQUIRE(window >= 0 && window <= INT32_MAX, LQ_EINVAL, "bad window");
  const int64_t rows = Hq / cache->H * Sq;
  if (rows == 0) return LQ_OK;
  LQ_REQUIRE(rows <= 16 * 65535, LQ_ERANGE, "too many query rows");
  LQ_REQUIRE(q && out, LQ_EINVAL, "NULL pointer");
  const Kv4 kv = kv4_of(cache);
  const Plan p = plan_of(kv, rows, bound);
  size_t bytes[3];
  spaces(kv, p, accumulate != 0, bytes);
  LQ_REQUIRE(workspace && workspace_bytes >= bytes[0] + bytes[1] + bytes[2], LQ_EINVAL, "workspace of %zu bytes needed",
             bytes[0] + bytes[1] + bytes[2]);
  LQ_REQUIRE(aligned16(workspace), LQ_EALIGN, "workspace must be 16-byte aligned");
  Attn a;
  a.kv = kv;
  a.q = static_cast<const uint8_t*>(q);
  a.q_dtype = q_dtype;
  a.q_sb = q_sb, a.q_sh = q_sh, a.q_ss = q_ss;
  a.Hq = (int)Hq, a.G = (int)(Hq / cache->H), a.Sq = (int)Sq, a.rows = (int)rows, a.rows_pad = p.rows_pad;
  a.counts = counts;
  a.sm = sm_scale, a.cap = softcap;
  a.slopes = slopes, a.prefix = prefix;
  a.causal = causal != 0, a.window = (int)window;
  a.blocks = p.blocks;
  a.out = static_cast<uint8_t*>(out);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.part = reinterpret_cast<float*>(ws);
  a.ml = reinterpret_cast<float2*>(ws + bytes[0]);
  a.lse = accumulate ? reinterpret_cast<float*>(ws + bytes[0] + bytes[1]) : nullptr;
  // a single query sees every token but for a window, a bias or a cap
  const bool gen = (Sq > 1 && (causal || counts)) || softcap > 0.0f || slopes || window > 0;
  cudaStream_t st = as_stream(stream);
  return kv.D == 128 ? run_attn_d<128>(a, p, gen, st) : run_attn_d<64>(a, p, gen, st);
}

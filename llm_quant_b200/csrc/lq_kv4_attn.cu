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
// P carries sv: p sv = exp2(x + log2 sv - m) with m a running reference of
// x + log2 sv, so that it fits f16 whatever the scales; the denominator sums
// exp2(x - m).
//
// Split: the 32-token units of all (sequence, kv head) pairs lie in one row,
// and each block takes an equal stretch of it (it may begin and end inside a
// head, and cover several), so that sequences of unequal lengths and few heads
// fill the GPU alike.  The lengths are read on the device.  A head that one
// block covers is finished there; partial results of the others are merged by
// kv4_combine_kernel, a programmatic dependent launch.
//
// Bound and measured (D = 128): 8 sequences x 8 kv heads x 4 of 8192 tokens 21.9
// us, merge 4.8 (71 MB, 3.3 TB/s); 16 of up to 20011 tokens, groups of 8, 47.7 us,
// merge 5.4 (196 MB, 4.1 TB/s).  The copies alone take 15 and 35.6 us; the rest
// is what mma.sync and the nibbles add (half of the MMAs taken out: -13 %).
#include <algorithm>

#include "lq_kv4_attn.cuh"
#include "lq_tma.cuh"

namespace lq {
namespace {

constexpr int kWarps = 4;
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
// Fragment registers from a word of codes: nibble n of both halves as f16.
// The tensor cores align a subnormal's product by the exponent 2^-14 it would
// have as a normal number, and cut below 24 bits: a code whose unit is 2^(b -
// 24) loses what is under 2^(-14 - b) of that unit, times the largest factor that
// it meets among the 16 of an MMA.  V takes nibbles where they are with a mask and
// one shift for two (b = 0 and 4: 5 instructions for 8 codes): an output then loses
// up to 16 * 2^-14 of the V scale times the probability, as much as P's rounding to
// f16 costs a value of 2 scales.  With all of them at b = 4 (7 instructions) it is
// 2^-14, at 28.7 us instead of 27.0 (8 x 8 heads of 8192 tokens, groups of 4) and
// 55.6 instead of 53.6 (16 of up to 20011, groups of 8): not worth it beside values that
// are off by up to half a scale.  Scores decide collected weights in fp32, so K is
// shifted to b = 4 (7); with fp32 queries K and V are shifted to b = 6 (8).
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

// Units of the sequences before b, and of all; every warp computes it for itself.
__device__ __forceinline__ int units_before(const Attn& a, int b, int& all) {
  int before = 0, sum = 0;
#pragma unroll 1
  for (int j = threadIdx.x & 31; j < a.kv.B; j += 32) {
    const int u = seq_of(a, j).count;
    sum += u;
    if (j < b) before += u;
  }
  all = warp_sum(sum) * a.kv.H;
  return warp_sum(before) * a.kv.H;
}
// Sequence that holds unit x, and the unit it begins at.
__device__ __forceinline__ int seq_at(const Attn& a, int x, int& begin) {
  const int lane = threadIdx.x & 31;
  begin = 0;
#pragma unroll 1
  for (int b0 = 0; b0 < a.kv.B; b0 += 32) {
    const int own = b0 + lane < a.kv.B ? seq_of(a, b0 + lane).count * a.kv.H : 0;
    const int inc = warp_scan(own);
    const uint32_t hit = __ballot_sync(0xffffffffu, begin + inc > x);
    if (hit) {
      const int src = __ffs(hit) - 1;
      begin += __shfl_sync(0xffffffffu, inc - own, src);
      return b0 + src;
    }
    begin += __shfl_sync(0xffffffffu, inc, 31);
  }
  return a.kv.B;
}

// Queries of a block's rows as B fragments, and what each score column needs.
// They are made once per head by the whole block, in shared memory.
template <int D, int NQ, bool QLO>
struct RowsShared {
  static constexpr int NW = D / 8;  // words of a row
  uint4 hi[8 * NQ][NW];             // values (0, 1), (4, 5), (2, 3), (6, 7) of each word
  uint4 lo[QLO ? 8 * NQ : 1][QLO ? NW : 1];
  float sum[8 * NQ], fac[8 * NQ];
};
template <int D, int NQ, bool QLO>
struct Rows {
  static constexpr int W = D / 32, NW = D / 8;
  static constexpr float kUnitK = pow2(Nibbles<QLO ? kSix : kFour>::unit(0));
  const RowsShared<D, NQ, QLO>* sh;
  float sum[NQ][2], fac[NQ][2];  // of columns 2c, 2c + 1: -sum of q, factor that undoes the scaling
  float slope[NQ][2];
  int at[NQ][2];                 // position of the query; INT_MIN: no such row

  // NW neighbouring lanes make a row, 8 values each
  __device__ __forceinline__ static void make(RowsShared<D, NQ, QLO>& sh, const Attn& a, const Seq& s, int b, int h,
                                              int zb, int tid, int threads, bool gen) {
    for (int j = tid; j < 8 * NQ * NW; j += threads) {
      const int lr = j / NW, w = j % NW, r = zb * 8 * NQ + lr, i = r / a.G;
      float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
      if (r < a.rows && i < s.cnt) {
        const int64_t off = b * a.q_sb + (int64_t)(h * a.G + r % a.G) * a.q_sh + i * a.q_ss + 8 * w;
        if constexpr (QLO) load8(reinterpret_cast<const float*>(a.q) + off, x);
        else if (a.q_dtype == LQ_F16) load8(reinterpret_cast<const __half*>(a.q) + off, x);
        else load8(reinterpret_cast<const __nv_bfloat16*>(a.q) + off, x);
      }
      float mx = 0.0f, sum = 0.0f;
#pragma unroll
      for (int d = 0; d < 8; ++d) mx = fmaxf(mx, fabsf(x[d])), sum += x[d];
#pragma unroll
      for (int m = NW / 2; m > 0; m >>= 1) {
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, m));
        sum += __shfl_xor_sync(0xffffffffu, sum, m);
      }
      // 2^(14 - exponent of mx), kept a normal number
      const int e = (int)(__float_as_uint(mx) >> 23);
      const int up = mx > 0.0f && e < 255 ? max(min(268 - e, 254), 1) : 127;
      const float f = __uint_as_float((uint32_t)up << 23);
      uint32_t p[4], q[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {  // register k: nibble n of both halves, n = 0, 2, 1, 3
        const int n = k < 2 ? 2 * k : 2 * k - 3;
        const float u = x[2 * n] * f, v = x[2 * n + 1] * f;
        p[k] = h2(u, v);
        if constexpr (QLO) {
          const float2 y = f2(p[k]);
          q[k] = h2(u - y.x, v - y.y);
        }
      }
      sh.hi[lr][w] = make_uint4(p[0], p[1], p[2], p[3]);
      if constexpr (QLO) sh.lo[lr][w] = make_uint4(q[0], q[1], q[2], q[3]);
      if (w == 0) {
        // the accumulators hold kUnitK * f times the true sums
        sh.sum[lr] = -sum * f * kUnitK;
        sh.fac[lr] = a.sm / f * (1.0f / kUnitK) * (gen && a.cap > 0.0f ? 1.0f / a.cap : kLog2e);
      }
    }
  }
  // fragment registers of word w: read where they are used, they are not worth 16 registers
  __device__ __forceinline__ uint4 hi(int nq, int w) const {
    const int lane = threadIdx.x & 31;
    return sh->hi[8 * nq + (lane >> 2)][(lane & 3) * W + w];
  }
  __device__ __forceinline__ uint4 lo(int nq, int w) const {
    const int lane = threadIdx.x & 31;
    return sh->lo[8 * nq + (lane >> 2)][(lane & 3) * W + w];
  }
  __device__ __forceinline__ void load(const RowsShared<D, NQ, QLO>& sh, const Attn& a, const Seq& s, int h, int zb,
                                       bool gen) {
    const int c = threadIdx.x & 3;
    this->sh = &sh;
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        sum[nq][e] = sh.sum[8 * nq + 2 * c + e];
        fac[nq][e] = sh.fac[8 * nq + 2 * c + e];
        if (gen) {
          const int r = zb * 8 * NQ + 8 * nq + 2 * c + e, i = r / a.G;
          at[nq][e] = r < a.rows && i < s.cnt ? s.first + i : INT_MIN;
          slope[nq][e] = a.slopes && r < a.rows ? a.slopes[h * a.G + r % a.G] * kLog2e : 0.0f;
        }
      }
    }
  }
};

// Products of N tiles of 16 tokens from the codes of rows k[2 N]: x[i][nq][0..3] =
// (token g, column 2c), (g, 2c + 1), (g + 8, 2c), (g + 8, 2c + 1) of tile i, the
// zero points' share taken off beforehand.
template <int N, int D, int NQ, bool QLO>
__device__ __forceinline__ void products(const Rows<D, NQ, QLO>& q, const uint32_t (*k)[D / 32], const uint32_t* par,
                                         float (*x)[NQ][4]) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
      for (int u = 0; u < 4; ++u) x[i][nq][u] = par_zero(par[2 * i + (u >> 1)]) * q.sum[nq][u & 1];
#pragma unroll
  for (int w = 0; w < D / 32; ++w) {
    uint4 hi[NQ], lo[NQ];
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
      hi[nq] = q.hi(nq, w);
      if constexpr (QLO) lo[nq] = q.lo(nq, w);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      uint32_t ka[4], kb[4];
      Nibbles<QLO ? kSix : kFour>::take(k[2 * i][w], ka);
      Nibbles<QLO ? kSix : kFour>::take(k[2 * i + 1][w], kb);
#pragma unroll
      for (int nq = 0; nq < NQ; ++nq) {
        mma16(x[i][nq], ka[0], kb[0], ka[2], kb[2], hi[nq].x, hi[nq].y);
        mma16(x[i][nq], ka[1], kb[1], ka[3], kb[3], hi[nq].z, hi[nq].w);
        if constexpr (QLO) {
          mma16(x[i][nq], ka[0], kb[0], ka[2], kb[2], lo[nq].x, lo[nq].y);
          mma16(x[i][nq], ka[1], kb[1], ka[3], kb[3], lo[nq].z, lo[nq].w);
        }
      }
    }
  }
}

// Score (log2 units) from a scaled and capped product, with bias and masks: -inf
// where the query does not see the token.
template <int D, int NQ, bool QLO>
__device__ __forceinline__ float full_score(const Attn& a, const Rows<D, NQ, QLO>& q, int nq, int e, float v, bool in,
                                            int pos, int pre) {
  const int back = q.at[nq][e] - pos;
  if (a.slopes) v = fmaf(-q.slope[nq][e], fabsf((float)back), v);
  bool near = true;
  if (a.causal) near = back >= 0;
  if (a.window > 0) near = near && back < a.window;
  return in && (near || pos < pre) && q.at[nq][e] != INT_MIN ? v : -INFINITY;
}

// Positions of a lane's tokens (general masks only).
template <int N>
__device__ __forceinline__ void load_pos(const Attn& a, int64_t row, const int* tok, const Seq& s, int* pos) {
#pragma unroll
  for (int j = 0; j < N; ++j) pos[j] = s.ordered || tok[j] >= s.n ? tok[j] : a.kv.pos[row + tok[j]];
}

// Shared memory of a block: each warp has a ring of its own of kStages units,
// filled by bulk copies that one lane issues, so that a unit's bytes are on
// their way while the warp works on the one before and need no registers.
constexpr int kStages = 2;
template <int D>
struct Stage {
  uint32_t k[4][32][D / 32], v[4][32][D / 32];
  uint2 par[kUnit];
  static constexpr uint32_t bytes = kUnit * D + kUnit * 8;
};
template <int D, int NQ, bool QLO>
struct alignas(128) AttnShared {
  Stage<D> ring[kWarps][kStages];
  float o[kWarps][8][D + 4];
  RowsShared<D, NQ, QLO> q;
  float2 ml[kWarps][8 * NQ];
  uint64_t full[kWarps][kStages];
};
template <int W>
__device__ __forceinline__ void lds_codes(const uint32_t* p, uint32_t* w) {
  if constexpr (W == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  }
}

template <int D, int NQ, bool QLO, bool GEN>
__global__ void __launch_bounds__(32 * kWarps, NQ == 1 && !QLO ? 4 : NQ == 1 ? 2 : 1) kv4_attn_kernel(const Attn a) {
  constexpr int W = D / 32;
  using VN = Nibbles<QLO ? kSix : kMixed>;
  extern __shared__ __align__(128) uint8_t smem[];
  AttnShared<D, NQ, QLO>& sh = *reinterpret_cast<AttnShared<D, NQ, QLO>*>(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int zb = blockIdx.y, cta = blockIdx.x;
  Cut cut;
  int x0, x1, b, seq_begin;
  Seq s;
  if (a.whole) {  // a block to a head
    b = cta / a.kv.H;
    s = seq_of(a, b);
    seq_begin = 0;
    x0 = cta % a.kv.H * s.count;
    x1 = x0 + s.count;
  } else {
    int all;
    units_before(a, 0, all);
    cut.set(all, a.blocks);
    if (all == 0 || cta >= cut.blocks) return;
    x0 = cut.begin(cta);
    x1 = cut.begin(cta + 1);
    b = seq_at(a, x0, seq_begin);
    s = seq_of(a, b);
  }
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < kStages; ++i) mbar_init(&sh.full[warp][i], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncwarp();
  int fill = 0, take = 0;  // units that this warp has asked for, and used
  int h = a.whole ? cta % a.kv.H : (x0 - seq_begin) / s.count, u0 = x0 - seq_begin - h * s.count;
  int u1 = min(s.count, u0 + (x1 - x0));
  auto token = [&](int u) { return GEN ? (u < s.pre ? u : u + s.gap) * kUnit : u * kUnit; };
  auto ask = [&](int u) {  // every lane has read what the stage held
    if (u < u1 && fill >= 0) {
      if (lane == 0) {
        Stage<D>& st = sh.ring[warp][fill % kStages];
        uint64_t* bar = &sh.full[warp][fill % kStages];
        const int64_t t = (int64_t)(b * a.kv.H + h) * a.kv.cap + token(u);
        mbar_expect_tx(bar, Stage<D>::bytes);
        bulk_load(st.k, a.kv.k + t * (D / 2), kUnit * (D / 2), bar);
        bulk_load(st.v, a.kv.v + t * (D / 2), kUnit * (D / 2), bar);
        bulk_load(st.par, a.kv.par + t, kUnit * 8, bar);
      }
      ++fill;
    }
  };
#pragma unroll
  for (int i = 0; i < kStages; ++i) ask(u0 + warp + i * kWarps);

  while (true) {  // (a whole head with nothing to see goes through too, and gives zeros)
    const int bh = b * a.kv.H + h;
    const int64_t row = (int64_t)bh * a.kv.cap;
    const int pre = GEN && a.prefix ? a.prefix[b] : 0;
    int u = u0 + warp;
    __syncthreads();  // the last head's queries have been read
    Rows<D, NQ, QLO>::make(sh.q, a, s, b, h, zb, threadIdx.x, 32 * kWarps, GEN);
    __syncthreads();
    Rows<D, NQ, QLO> q;
    q.load(sh.q, a, s, h, zb, GEN);

    float m[NQ][2], l[NQ][2], z[NQ][2], O[NQ][2 * W][4];
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
#pragma unroll
      for (int e = 0; e < 2; ++e) m[nq][e] = kNone, l[nq][e] = z[nq][e] = 0.0f;
#pragma unroll
      for (int e = 0; e < 2 * W; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) O[nq][e][i] = 0.0f;
    }
    for (; u < u1 && fill >= 0; u += kWarps) {
      const int t0 = token(u);
      const Stage<D>& st = sh.ring[warp][take % kStages];
      if (!mbar_wait_warp(&sh.full[warp][take % kStages], (take / kStages) & 1)) {
        // The copy never came (2 s): give up, so that the host learns of it.  Nothing
        // more is asked for (fill < 0), and the block does not end with copies on their way.
        if (lane == 0) a.kv.sync[3] = LQ_ETIMEOUT;
        for (; take < fill; ++take) mbar_wait_warp(&sh.full[warp][take % kStages], (take / kStages) & 1);
        fill = -1;
        break;
      }
      ++take;
      uint32_t kp[4], vp[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint2 p = st.par[8 * j + g];
        kp[j] = p.x, vp[j] = p.y;
      }
      const bool tail = t0 + kUnit > s.n;
      if (tail) {  // what lies past the end may be anything
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (t0 + 8 * j + g >= s.n) kp[j] = vp[j] = 0u;
      }
      float x[2][NQ][4];
      {
        uint32_t k[4][W];
#pragma unroll
        for (int j = 0; j < 4; ++j) lds_codes<W>(st.k[j][lane], k[j]);
        products<2, D, NQ, QLO>(q, k, kp, x);
      }
      // scores
      int tok[4], pos[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) tok[j] = t0 + 8 * j + g;
      if constexpr (GEN) load_pos<4>(a, row, tok, s, pos);
      float lv[4], zv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float sk = par_scale(kp[j]), sv = par_scale(vp[j]);
        lv[j] = (sv == 0.0f ? -100.0f : lg2(sv)) + kHead;  // a scale of 0 has only zeros behind it
        zv[j] = par_zero(vp[j]);
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& v = x[j >> 1][nq][2 * (j & 1) + e];
            v *= sk * q.fac[nq][e];
            if (!GEN && tail && tok[j] >= s.n) v = -INFINITY;
          }
      }
      if constexpr (GEN) {
        if (a.cap > 0.0f) capped<8 * NQ>(&x[0][0][0], a.cap * kLog2e);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int nq = 0; nq < NQ; ++nq)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float& v = x[j >> 1][nq][2 * (j & 1) + e];
              v = full_score<D, NQ, QLO>(a, q, nq, e, v, tok[j] < s.n, pos[j], pre);
            }
      }
      if (a.scores) {
#pragma unroll
        for (int nq = 0; nq < NQ; ++nq)
          if (8 * nq + 2 * c < a.pitch)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              *reinterpret_cast<float2*>(a.scores + (row + tok[j]) * a.pitch + 8 * nq + 2 * c) =
                  make_float2(x[j >> 1][nq][2 * (j & 1)], x[j >> 1][nq][2 * (j & 1) + 1]);
      }
      uint32_t pb[NQ][4], pl[QLO ? NQ : 1][4];
#pragma unroll
      for (int nq = 0; nq < NQ; ++nq) {
        // exponents of P, above the reference; a token that is not seen has none, whatever its scale
        float w[4][2];
        auto exponents = [&] {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float v = x[j >> 1][nq][2 * (j & 1) + e];
              w[j][e] = (v - m[nq][e]) + lv[j];
              if (GEN && v == -INFINITY) w[j][e] = -INFINITY;
            }
        };
        exponents();
        const float w0 = fmaxf(fmaxf(w[0][0], w[1][0]), fmaxf(w[2][0], w[3][0]));
        const float w1 = fmaxf(fmaxf(w[0][1], w[1][1]), fmaxf(w[2][1], w[3][1]));
        if (__any_sync(0xffffffffu, fmaxf(w0, w1) > kTop)) {
          float alpha[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mt = kNone;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float v = x[j >> 1][nq][2 * (j & 1) + e];
              if (!GEN || v != -INFINITY) mt = fmaxf(mt, v + lv[j] - kHead);
            }
            mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 4));
            mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 8));
            mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 16));
            mt = fmaxf(m[nq][e], mt);
            alpha[e] = ex2(m[nq][e] - mt);
            m[nq][e] = mt;
            l[nq][e] *= alpha[e];
            z[nq][e] *= alpha[e];
          }
#pragma unroll
          for (int d = 0; d < 2 * W; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i) O[nq][d][i] *= alpha[i & 1];
          exponents();
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
          for (int e = 0; e < 2; ++e) l[nq][e] += ex2(x[j >> 1][nq][2 * (j & 1) + e] - m[nq][e]);
          const float pa = ex2(w[j][0]), pc = ex2(w[j][1]);
          const uint32_t r = h2(pa, pc);
          const float2 rf = f2(r);
          if constexpr (QLO) {
            const uint32_t rl = h2(pa - rf.x, pc - rf.y);
            const float2 rlf = f2(rl);
            pl[nq][j] = transposed(rl);
            z[nq][0] = fmaf(rf.x + rlf.x, zv[j], z[nq][0]);
            z[nq][1] = fmaf(rf.y + rlf.y, zv[j], z[nq][1]);
          } else {
            z[nq][0] = fmaf(rf.x, zv[j], z[nq][0]);
            z[nq][1] = fmaf(rf.y, zv[j], z[nq][1]);
          }
          pb[nq][j] = transposed(r);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t v0[W], v1[W];
        lds_codes<W>(st.v[2 * i][lane], v0);
        lds_codes<W>(st.v[2 * i + 1][lane], v1);
#pragma unroll
        for (int w = 0; w < W; ++w) {
          uint32_t va[4], vb[4];
          VN::take(v0[w], va);
          VN::take(v1[w], vb);
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
      }
      __syncwarp();
      ask(u + kStages * kWarps);
    }

    // ---- merge the warps: O in true units, minus the zero points' share ----
    const bool whole = u0 == 0 && u1 == s.count;
    const int b_done = b, h_done = h;
    x0 += u1 - u0;
    const bool more = x0 < x1;
    if (more) {  // the next head's first units come while this one is merged
      ++h;
      while (h == a.kv.H || s.count == 0) {
        s = seq_of(a, ++b);
        h = 0;
      }
      u0 = 0;
      u1 = min(s.count, x1 - x0);
#pragma unroll
      for (int i = 0; i < kStages; ++i) ask(warp + i * kWarps);
    }
    const int64_t slot = ((int64_t)cta + bh) * a.rows_pad;
#pragma unroll
    for (int nq = 0; nq < NQ; ++nq) {
      __syncthreads();  // the last round's O has been read
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) {
          l[nq][e] += __shfl_xor_sync(0xffffffffu, l[nq][e], k);
          z[nq][e] += __shfl_xor_sync(0xffffffffu, z[nq][e], k);
        }
        if (g == 0) sh.ml[warp][8 * nq + 2 * c + e] = make_float2(m[nq][e], l[nq][e]);
      }
      // d = 4 (g W + w) + n: nibble n of word w
#pragma unroll
      for (int w = 0; w < W; ++w)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float v[4];
#pragma unroll
          for (int n = 0; n < 4; ++n)
            v[n] = fmaf(O[nq][2 * w + (n & 1)][e + 2 * (n >> 1)], pow2(-VN::unit(n & 1)), -z[nq][e]) * pow2(-(int)kHead);
          *reinterpret_cast<float4*>(&sh.o[warp][2 * c + e][4 * (g * W + w)]) = make_float4(v[0], v[1], v[2], v[3]);
        }
      __syncthreads();
      for (int i = threadIdx.x; i < 2 * D; i += 32 * kWarps) {
        const int r = i / (D / 4), d = 4 * (i % (D / 4)), qr = zb * 8 * NQ + 8 * nq + r;
        if (qr >= a.rows) break;
        float M = kNone;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sh.ml[w][8 * nq + r].x);
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float L = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float2 ml = sh.ml[w][8 * nq + r];
          const float f = ex2(ml.x - M);
          const float4 v = *reinterpret_cast<const float4*>(&sh.o[w][r][d]);
          o.x = fmaf(f, v.x, o.x), o.y = fmaf(f, v.y, o.y), o.z = fmaf(f, v.z, o.z), o.w = fmaf(f, v.w, o.w);
          L = fmaf(f, ml.y, L);
        }
        if (whole) {
          const float inv = L == 0.0f ? 0.0f : 1.0f / L;
          const int iq = qr / a.G, hq = h_done * a.G + qr % a.G;
          st_out4(a.out, (((int64_t)b_done * a.Hq + hq) * a.Sq + iq) * D + d, a.q_dtype, o, inv);
          if (a.lse && d == 0) a.lse[(int64_t)bh * a.rows_pad + qr] = L == 0.0f ? INFINITY : M + lg2(L);
          if (a.scores && d == 0) a.ml[slot + qr] = make_float2(M, L);
        } else {
          *reinterpret_cast<float4*>(a.part + (slot + qr) * D + d) = o;
          if (d == 0) a.ml[slot + qr] = make_float2(M, L);
        }
      }
    }
    if (!more) break;
  }
  if (threadIdx.x == 0) pdl_trigger();
}

// First out_blocks blocks, a warp per (row, head): merges the partial results of
// the blocks that shared the head; zeros where there is nothing to see.  Heads
// that one block covered are done already.
// The blocks behind them, if weights are collected from the scores that the
// attention kernel left: 256 tokens of a head at a time, mass[t] += sum over the rows
// of exp2(x[r, t] - lse[r]), with lse from the same partial results.
// The lengths are older than the kernel before this one, so they are read while
// it still runs.
template <int D, bool WEIGH>
__global__ void __launch_bounds__(128) kv4_combine_kernel(const Attn a, int out_blocks) {
  constexpr int V = D / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const bool spread = WEIGH && (int)blockIdx.x >= out_blocks;
  const int heads = a.kv.B * a.kv.H;
  int bh, qr = 0, t0 = 0;
  if (spread) {
    bh = (blockIdx.x - out_blocks) % heads;
    t0 = (blockIdx.x - out_blocks) / heads * 256;
  } else {
    const int item = blockIdx.x * 4 + warp;
    if (item >= a.rows * heads) return pdl_wait();  // no block ends before the kernel that it waits for
    bh = item / a.rows, qr = item % a.rows;
  }
  const int b = bh / a.kv.H, h = bh % a.kv.H;
  const Seq s = seq_of(a, b);
  if (spread && (s.count == 0 || t0 >= s.n)) return pdl_wait();
  int c0 = bh, c1 = bh;  // the blocks that had a part of the head
  if (!a.whole) {
    int all;
    const int begin = units_before(a, b, all) + h * s.count;
    Cut cut;
    cut.set(all, a.blocks);
    c0 = s.count ? cut.owner(begin) : 0, c1 = s.count ? cut.owner(begin + s.count - 1) : -1;
  }
  pdl_wait();
  if (!spread && s.count && c0 == c1) return;
  const int64_t first = (int64_t)(c0 + bh) * a.rows_pad;
  auto reference = [&](int r) {
    float m = kNone;
    for (int c = c0 + lane; c <= c1; c += 32) m = fmaxf(m, a.ml[first + r + (int64_t)(c - c0) * a.rows_pad].x);
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
    return m;
  };
  if constexpr (WEIGH) if (spread) {
    __shared__ float lse[16];
    for (int r = warp; r < a.rows; r += 4) {
      const float M = reference(r);
      float L = 0.0f;
      for (int c = c0 + lane; c <= c1; c += 32) {
        const float2 ml = a.ml[first + r + (int64_t)(c - c0) * a.rows_pad];
        L = fmaf(ex2(ml.x - M), ml.y, L);
      }
#pragma unroll
      for (int k = 16; k > 0; k >>= 1) L += __shfl_xor_sync(0xffffffffu, L, k);
      if (lane == 0) lse[r] = L == 0.0f ? INFINITY : M + lg2(L);
    }
    __syncthreads();
    // from 256 tokens to the next that no other block has
    const int step = ((int)gridDim.x - out_blocks) / heads * 256;
    for (int64_t t2 = t0; t2 < s.n; t2 += (t2 & 128) ? step - 128 : 128) {
      const int t = (int)t2 + threadIdx.x;
      if (t >= s.n) break;
      const int u = t / kUnit;
      if (u >= s.pre && u < s.pre + s.gap) continue;  // behind the window: no scores were made
      const int64_t i = (int64_t)bh * a.kv.cap + t;
      float sum = 0.0f;
      for (int r = 0; r < a.rows; r += 4) {
        const float4 x = *reinterpret_cast<const float4*>(a.scores + i * a.pitch + r);
        sum += ex2(x.x - lse[r]);
        if (r + 1 < a.rows) sum += ex2(x.y - lse[r + 1]);
        if (r + 2 < a.rows) sum += ex2(x.z - lse[r + 2]);
        if (r + 3 < a.rows) sum += ex2(x.w - lse[r + 3]);
      }
      a.kv.mass[i] += sum;
    }
    return;
  }
  // a lane has the factor of a part: loads of the parts wait for nothing but the wait above
  const float M = reference(qr);
  float L = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
  for (int base = 0; base <= c1 - c0; base += 32) {
    const int64_t i = first + qr + (int64_t)base * a.rows_pad;
    const int n = min(32, c1 - c0 + 1 - base);
    float f = 0.0f;
    if (lane < n) {
      const float2 ml = a.ml[i + (int64_t)lane * a.rows_pad];
      f = ex2(ml.x - M);
      L = fmaf(f, ml.y, L);
    }
    const float* p = a.part + i * D + V * lane;
#pragma unroll 1
    for (int c = 0; c < n; c += 8) {  // behind the last part: that one again, with factor 0
      float v[8][V];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float* from = p + (int64_t)min(c + k, n - 1) * a.rows_pad * D;
        if constexpr (V == 4) *reinterpret_cast<float4*>(v[k]) = *reinterpret_cast<const float4*>(from);
        else *reinterpret_cast<float2*>(v[k]) = *reinterpret_cast<const float2*>(from);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float fc = __shfl_sync(0xffffffffu, f, c + k);
#pragma unroll
        for (int d = 0; d < V; ++d) o[d] = fmaf(fc, v[k][d], o[d]);
      }
    }
  }
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) L += __shfl_xor_sync(0xffffffffu, L, k);
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  const int iq = div_g(a, qr), hq = h * a.G + qr - iq * a.G;
  const int64_t at = (((int64_t)b * a.Hq + hq) * a.Sq + iq) * D + V * lane;
  if constexpr (V == 4) {
    st_out4(a.out, at, a.q_dtype, make_float4(o[0], o[1], o[2], o[3]), inv);
  } else {
    st_out(a.out, at, a.q_dtype, o[0] * inv);
    st_out(a.out, at + 1, a.q_dtype, o[1] * inv);
  }
  if (a.lse && lane == 0) a.lse[(int64_t)bh * a.rows_pad + qr] = L == 0.0f ? INFINITY : M + lg2(L);
}

// mass[t] += sum over the rows of exp2(x[r, t] - lse[r]).  A warp owns 16
// tokens and goes over all rows, so that no two threads add to one token and
// the order of the sum is fixed.
template <int D, bool QLO, bool GEN>
__global__ void __launch_bounds__(128) kv4_mass_kernel(const Attn a) {
  constexpr int W = D / 32;
  __shared__ RowsShared<D, 1, QLO> sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const int bh = blockIdx.y, b = bh / a.kv.H, h = bh % a.kv.H;
  const Seq s = seq_of(a, b);
  const int pre = GEN && a.prefix ? a.prefix[b] : 0;
  const int64_t row = (int64_t)bh * a.kv.cap;
  if (s.cnt == 0) return;
  for (int base = blockIdx.x * 64; base < s.n; base += gridDim.x * 64) {
    const int t0 = base + warp * 16;  // within the capacity, a multiple of 32: the last warps of a block may find
    const bool some = t0 < s.n;       // nothing there, but they help with the queries
    uint32_t kw[2][W] = {}, kp[2] = {0u, 0u};
    int tok[2], pos[2];
    float sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      tok[j] = t0 + 8 * j + g;
      if (some) ld_codes<W>(a.kv.k + (row + t0 + 8 * j) * (D / 2) + lane * (4 * W), kw[j]);
      if (tok[j] < s.n) kp[j] = a.kv.par[row + tok[j]].x;
    }
    if constexpr (GEN) load_pos<2>(a, row, tok, s, pos);
    for (int zb = 0; zb * 8 < a.rows; ++zb) {
      __syncthreads();
      Rows<D, 1, QLO>::make(sh, a, s, b, h, zb, threadIdx.x, 128, GEN);
      __syncthreads();
      Rows<D, 1, QLO> q;
      q.load(sh, a, s, h, zb, GEN);
      float x[1][1][4];
      products<1, D, 1, QLO>(q, kw, kp, x);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[0][0][i] *= par_scale(kp[i >> 1]) * q.fac[0][i & 1];
      if (GEN && a.cap > 0.0f) capped<4>(&x[0][0][0], a.cap * kLog2e);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int qr = zb * 8 + 2 * c + e;
        if (qr >= a.rows) continue;
        const float lse = a.lse[(int64_t)bh * a.rows_pad + qr];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float v = x[0][0][2 * j + e];
          if constexpr (GEN) v = full_score<D, 1, QLO>(a, q, 0, e, v, tok[j] < s.n, pos[j], pre);
          sum[j] += ex2(v - lse);
        }
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

// Rows of a block, and blocks of the split: one wave of resident blocks over
// all row blocks, and at least one unit per warp.
struct Plan {
  int nq, row_blocks, rows_pad, blocks;
  int64_t slots;  // partial results, of rows_pad (prompt: kPromptRows) rows each
  bool prompt;    // lq_kv4_prompt.cu's
  bool whole;     // a block to a head
  int pitch;      // scores kept per token for the collected weight; 0: none are kept
};
// Up to so many units a head is left to one block, and nothing has to be merged.
// One block to a head against cut heads, us (D = 128, groups of 4): 512 tokens 7.1 /
// 8.4 with one head, 7.2 / 8.7 with 8, 7.3 / 11.0 with 128, 12.5 / 19.7 with 512;
// 1024 tokens 10.7 / 8.4, 10.8 / 8.8, 11.0 / 15.2, 20.0 / 26.0.
constexpr int kWholeUnits = 16;
constexpr int64_t kMostScores = 256 << 20;  // bytes of kept scores
// Up to so many query rows a row of the cache is read once by this file's kernel;
// beyond, once per 16 rows, against once per 256 by the prompt kernel.  This against
// that, us (D = 128): 16 rows 17.3 / 26.3 on 8 heads of 8192 tokens, 57.8 / 80.8 on 64
// heads, 26.8 / 34.5 on 128 heads of 1000; 24 rows 22.7 / 26.9, 101 / 81, 42.3 / 35.0.
constexpr int kFewRows = 16;
Plan plan_of(const Kv4& kv, int64_t rows, int64_t bound, bool qlo, bool weigh) {
  Plan p;
  p.whole = false;
  p.pitch = 0;
  p.prompt = !qlo && rows > kFewRows;
  if (p.prompt) {
    p.nq = p.row_blocks = 0;
    p.rows_pad = (int)((rows + kPromptRows - 1) / kPromptRows * kPromptRows);
    p.blocks = num_sms();
    p.slots = 2 * p.blocks;
    return p;
  }
  p.nq = rows <= 8 ? 1 : 2;
  p.row_blocks = (int)((rows + 8 * p.nq - 1) / (8 * p.nq));
  p.rows_pad = p.row_blocks * 8 * p.nq;
  const int64_t per_head = (std::max<int64_t>(bound, 1) + kUnit - 1) / kUnit, units = (int64_t)kv.B * kv.H * per_head;
  if (weigh && p.row_blocks == 1) {
    const int pitch = (int)(rows + 3) / 4 * 4;
    if ((int64_t)kv.B * kv.H * kv.cap * pitch * 4 <= kMostScores) p.pitch = pitch;
  }
  int64_t slots = std::max<int64_t>(1, (int64_t)num_sms() * (p.nq == 1 && !qlo ? 4 : p.nq == 1 ? 2 : 1) / p.row_blocks);
  // the same number of blocks for every head, where that leaves few slots empty:
  // with equal lengths no block then has to change heads
  const int64_t heads = (int64_t)kv.B * kv.H;
  if (slots >= heads && slots % heads * 10 <= slots) slots -= slots % heads;
  p.blocks = (int)std::max<int64_t>(1, std::min<int64_t>(slots, (units + kWarps - 1) / kWarps));
  if (per_head <= kWholeUnits) {
    p.whole = true;
    p.blocks = (int)heads;
  }
  p.slots = p.whole && !p.pitch ? 0 : p.blocks + heads;
  return p;
}

// part, ml, and lse or scores
void spaces(const Kv4& kv, const Plan& p, bool weigh, size_t* bytes) {
  const size_t rows = (size_t)p.slots * (p.prompt ? kPromptRows : p.rows_pad);
  bytes[0] = rows * kv.D * sizeof(float);
  bytes[1] = (rows * sizeof(float2) + 15) / 16 * 16;
  const size_t heads = (size_t)kv.B * kv.H;
  bytes[2] = !weigh ? 0 : p.pitch ? heads * kv.cap * p.pitch * sizeof(float) : heads * p.rows_pad * sizeof(float);
}

template <int D, bool QLO, bool GEN>
int run_mass(const Attn& a, cudaStream_t st) {
  kv4_mass_kernel<D, QLO, GEN><<<dim3((a.bound + 63) / 64, a.kv.B * a.kv.H), 128, 0, st>>>(a);
  return launched("kv4_mass_kernel");
}

template <int D, int NQ, bool QLO, bool GEN>
int run_attn(const Attn& a, const Plan& p, cudaStream_t st) {
  constexpr int smem = sizeof(AttnShared<D, NQ, QLO>);
  auto kern = kv4_attn_kernel<D, NQ, QLO, GEN>;
  static DeviceOnce once;
  LQ_TRY(once.allow_smem((const void*)kern, smem, "kv4_attn_kernel"));
  kern<<<dim3(p.blocks, p.row_blocks), 32 * kWarps, smem, st>>>(a);
  LQ_TRY(launched("kv4_attn_kernel"));
  const int heads = a.kv.B * a.kv.H;
  const int out_blocks = a.whole ? 0 : (int)(((int64_t)a.rows * heads + 3) / 4);
  const int64_t spread_blocks = a.scores ? (int64_t)(a.bound + 255) / 256 * heads : 0;
  if (out_blocks + spread_blocks == 0) return a.lse ? run_mass<D, QLO, GEN>(a, st) : LQ_OK;
  launch_pdl(a.scores ? kv4_combine_kernel<D, true> : kv4_combine_kernel<D, false>, dim3((unsigned)(out_blocks + spread_blocks)), dim3(128), 0, st, a, out_blocks);
  LQ_TRY(launched("kv4_combine_kernel"));
  return a.lse ? run_mass<D, QLO, GEN>(a, st) : LQ_OK;
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

extern "C" size_t lq_kv4_attention_workspace_bytes(const lq_kv4_cache* cache, const lq_kv4_attn* f) {
  using namespace lq;
  if (!f || kv4_check(cache) != LQ_OK || f->Hq <= 0 || f->Sq <= 0 || f->Hq % cache->H) return 0;
  const Kv4 kv = kv4_of(cache);
  size_t b[3];
  spaces(kv, plan_of(kv, f->Hq / cache->H * f->Sq, f->bound, f->q_dtype == LQ_F32, f->accumulate != 0), f->accumulate != 0, b);
  return b[0] + b[1] + b[2];
}

extern "C" int lq_kv4_attention(const lq_kv4_cache* cache, const lq_kv4_attn* f, const void* q, const int32_t* counts,
                                const float* slopes, const int32_t* prefix, void* out, void* workspace,
                                size_t workspace_bytes, void* stream) {
  using namespace lq;
  LQ_TRY(kv4_check(cache));
  LQ_REQUIRE(f, LQ_EINVAL, "NULL form");
  LQ_REQUIRE(is_float_dtype(f->q_dtype), LQ_EDTYPE, "float query required");
  LQ_REQUIRE(f->Hq > 0 && f->Hq % cache->H == 0, LQ_EINVAL, "query heads %lld not a multiple of kv heads %lld",
             (long long)f->Hq, (long long)cache->H);
  LQ_REQUIRE(f->Sq >= 0 && f->bound >= 0, LQ_EINVAL, "bad shape");
  LQ_REQUIRE(f->softcap == 0.0f || (f->softcap >= 1e-20f && f->softcap <= 1e30f), LQ_EINVAL,
             "softcap %g: 0 (none) or 1e-20 to 1e30", (double)f->softcap);
  LQ_REQUIRE(f->window >= 0 && f->window <= (1 << 30), LQ_EINVAL, "window %lld: 0 (none) to 2^30", (long long)f->window);
  const int64_t rows = f->Hq / cache->H * f->Sq;
  if (rows == 0) return LQ_OK;
  LQ_REQUIRE(f->Hq / cache->H <= 4096 && rows <= 16 * 65535 && rows * cache->B * cache->H <= INT32_MAX, LQ_ERANGE, "too many query rows");
  LQ_REQUIRE(q && out, LQ_EINVAL, "NULL pointer");
  LQ_REQUIRE((uintptr_t)q % (4 * dtype_size(f->q_dtype)) == 0 && ((f->q_sb | f->q_sh | f->q_ss) & 3) == 0, LQ_EALIGN,
             "query rows must start on multiples of 4 elements");
  const Kv4 kv = kv4_of(cache);
  const Plan p = plan_of(kv, rows, f->bound, f->q_dtype == LQ_F32, f->accumulate != 0);
  size_t bytes[3];
  spaces(kv, p, f->accumulate != 0, bytes);
  const size_t need = bytes[0] + bytes[1] + bytes[2];
  LQ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), LQ_EINVAL, "workspace of %zu bytes needed", need);
  LQ_REQUIRE(aligned16(workspace) && aligned16(out), LQ_EALIGN, "output and workspace must be 16-byte aligned");
  Attn a;
  a.kv = kv;
  a.q = static_cast<const uint8_t*>(q);
  a.q_dtype = f->q_dtype;
  a.q_sb = f->q_sb, a.q_sh = f->q_sh, a.q_ss = f->q_ss;
  a.Hq = (int)f->Hq, a.G = (int)(f->Hq / cache->H), a.Sq = (int)f->Sq, a.rows = (int)rows, a.rows_pad = p.rows_pad;
  a.counts = counts;
  a.sm = f->sm_scale, a.cap = f->softcap;
  a.slopes = slopes, a.prefix = prefix;
  a.causal = f->causal != 0, a.window = (int)f->window;
  a.bound = (int)std::min<int64_t>(std::max<int64_t>(f->bound, 1), kv.cap);
  a.g_mul = a.G == 1 ? 0u : (uint32_t)(0x100000000ull / a.G) + 1u;
  a.q_wide = (uintptr_t)q % 16 == 0 && ((f->q_sb | f->q_sh | f->q_ss) * dtype_size(f->q_dtype)) % 16 == 0;
  a.blocks = p.blocks;
  a.out = static_cast<uint8_t*>(out);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.part = reinterpret_cast<float*>(ws);
  a.ml = reinterpret_cast<float2*>(ws + bytes[0]);
  float* extra = f->accumulate ? reinterpret_cast<float*>(ws + bytes[0] + bytes[1]) : nullptr;
  a.lse = p.pitch ? nullptr : extra;
  a.scores = p.pitch ? extra : nullptr;
  a.pitch = p.pitch;
  a.whole = p.whole;
  // a single query sees every token but for a window, a bias or a cap
  const bool gen = (f->Sq > 1 && (f->causal || counts)) || f->softcap > 0.0f || slopes || f->window > 0;
  cudaStream_t st = as_stream(stream);
  if (p.prompt) {
    LQ_REQUIRE((int64_t)p.rows_pad / kPromptRows * kv.B * kv.H <= INT32_MAX / ((kv.cap + 127) / 128), LQ_ERANGE,
               "%lld query rows by %d tokens are too many for one call", (long long)rows, kv.cap);
    return kv4_prompt(a, st);
  }
  return kv.D == 128 ? run_attn_d<128>(a, p, gen, st) : run_attn_d<64>(a, p, gen, st);
}

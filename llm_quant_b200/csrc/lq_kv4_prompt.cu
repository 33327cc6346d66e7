// lq_kv4_prompt.cu -- attention over the 4-bit KV cache for many query rows
// (chunks of a prompt), on the 5th-generation tensor cores.  Formulas and
// layouts: lq_kv4.cuh, lq_kv4_attn.cuh.
//
// A block works on 256 rows of one kv head (two tiles of 128; row r = i G +
// head of the group) and goes over the cached tokens in tiles of 128:
//   S = Q (C_k - Z_k)^T      kind::f16, Q and the bare integers of K in Q's type;
//   O += P' (C_v - Z_v)      kind::f16 in f16, P' from tensor memory.
// Code minus zero point is an integer of 5 bits, exact in either type, so the
// products are exact; the scales stay in fp32 outside: K's times the softmax
// scale multiplies a column of S, V's goes into P'.  P' = 2^(x + e - R + 8) sv /
// 2^e with R the row's running reference and e the exponent of the tile's
// largest sv: it fits f16 whatever the scales, and takes one exponential.  R is
// raised only when an exponent passes 15.9 (then the row's O in tensor memory is
// rescaled by the softmax threads themselves; it happens in the first tiles).
//
// Warps: 0-3 and 4-7 softmax of the two row tiles (a thread owns a row), 8-11
// turn packed codes into the two operands in shared memory (swizzled, two
// stages), 12 issues the MMAs, 13 tells the others what to do next.  Tensor memory: S0, S1 (P' lies over S), O0, O1.
// A row tile has two halves of S (64 tokens each): while one is turned into P'
// in place, the MMAs fill the other.
//
// Bound: per 128 x 128 tile of scores the tensor cores need 1024 cycles (D =
// 128) and the 16384 exponentials 1024 on the SM's special-function units; the
// softmax is written with packed fp32 pairs (f32x2) so that its instructions
// stay below that.
//
// Measured: 2048 queries of 8 kv heads x 4 on 8192 tokens, D = 128, causal: 339
// us, merge 16; 0.42 of the bf16 rate.  Issue slots are 43 % used, the tensor pipe
// 34 %, the special-function units 35 %: what holds it is the chain of a half
// tile (S, load, exponentials, store, PV) with two softmax warps to a scheduler.
// (D = 128 spills 112 bytes a thread.)  With cap, window and prefix, 3 x up to 777
// queries of 4 kv heads x 2 on 1500 tokens, D = 64: 30.5 us, merge 7.1.
//
// Split: as in lq_kv4_attn.cu, the (row tile, token tile) pairs that have
// anything to see lie in one row and each block takes an equal stretch;
// kv4_prompt_combine_kernel merges row tiles that were cut.
#include <algorithm>

#include "lq_kv4_attn.cuh"
#include "lq_tc.cuh"

namespace lq {
namespace {

constexpr int kTok = 128;    // tokens of a tile
constexpr int kTile = 128;   // rows of a tile
constexpr int kItem = kPromptRows;  // rows of an item
constexpr int kSoftmaxWarps = 8, kCodeWarps = 4;
// 16 warps of 128 registers at launch; each group of four then takes what its
// role needs: 2 x 168 + 96 + 80 = 4 x 128.
constexpr int kPromptThreads = 512;
template <int N>
__device__ __forceinline__ void more_regs() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void fewer_regs() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
constexpr int kScaleStages = 4;

// The token tiles that the rows of an item may see: tiles [0, pre) and [pre +
// gap, ...), `count` in all.
struct Tiles {
  int n, cnt, first, ordered;
  int pre, gap, count;
};
__device__ __forceinline__ Tiles tiles_of(const Attn& a, int b, int rt) {
  const Seq s = seq_of(a, b);
  Tiles t{s.n, s.cnt, s.first, s.ordered, 0, 0, 0};
  const int i0 = div_g(a, rt * kItem), i1 = min(div_g(a, rt * kItem + kItem - 1), s.cnt - 1);
  if (i0 >= s.cnt || s.n == 0) return t;
  int lo = 0, hi = s.n, pre = 0;
  if (s.ordered) {
    if (a.causal) hi = max(min(s.n, s.first + i1 + 1), 0);
    if (a.window > 0) lo = min(max(s.first + i0 - a.window + 1, 0), hi);
    if (a.prefix) pre = min(max(a.prefix[b], 0), s.n);
  }
  const int lo_t = lo / kTok, hi_t = hi > lo ? (hi + kTok - 1) / kTok : lo_t;
  t.pre = (pre + kTok - 1) / kTok;
  if (t.pre >= lo_t) {
    t.pre = max(t.pre, hi_t);
    t.count = t.pre;
  } else {
    t.gap = lo_t - t.pre;
    t.count = t.pre + hi_t - lo_t;
  }
  return t;
}

// A block's way through the items (sequence, row tile, head) that its stretch
// covers.
struct Walk {
  int x0, x1, j, h, u0, u1;
  Tiles t;
  __device__ __forceinline__ void piece() { u1 = min(t.count, u0 + (x1 - x0)); }
  __device__ __forceinline__ bool next(const Attn& a) {  // to the next piece; false: done
    const int rts = a.rows_pad / kItem;
    x0 += u1 - u0;
    if (x0 >= x1) return false;
    ++h;
#pragma unroll 1
    while (h == a.kv.H || t.count == 0) {
      h = 0;
      ++j;
      t = tiles_of(a, j / rts, j % rts);
    }
    u0 = 0;
    piece();
    return true;
  }
};
// Units of all items, and of those before item group j (a sequence's row tile, all heads).
__device__ __forceinline__ int tiles_before(const Attn& a, int j, int& all) {
  const int rts = a.rows_pad / kItem;
  int before = 0, sum = 0;
#pragma unroll 1
  for (int i = threadIdx.x & 31; i < a.kv.B * rts; i += 32) {
    const int u = tiles_of(a, i / rts, i % rts).count;
    sum += u;
    if (i < j) before += u;
  }
  all = warp_sum(sum) * a.kv.H;
  return warp_sum(before) * a.kv.H;
}
__device__ __forceinline__ bool walk_begin(const Attn& a, int cta, Walk& w) {
  const int rts = a.rows_pad / kItem, lane = threadIdx.x & 31;
  int all;
  tiles_before(a, 0, all);
  Cut cut;
  cut.set(all, a.blocks);
  if (all == 0 || cta >= cut.blocks) return false;
  w.x0 = cut.begin(cta);
  w.x1 = cut.begin(cta + 1);
  int begin = 0;
#pragma unroll 1
  for (int j0 = 0;; j0 += 32) {
    const int own = j0 + lane < a.kv.B * rts ? tiles_of(a, (j0 + lane) / rts, (j0 + lane) % rts).count * a.kv.H : 0;
    const int inc = warp_scan(own);
    const uint32_t hit = __ballot_sync(0xffffffffu, begin + inc > w.x0);
    if (hit) {
      const int src = __ffs(hit) - 1;
      begin += __shfl_sync(0xffffffffu, inc - own, src);
      w.j = j0 + src;
      break;
    }
    begin += __shfl_sync(0xffffffffu, inc, 31);
  }
  w.t = tiles_of(a, w.j / rts, w.j % rts);
  w.h = (w.x0 - begin) / w.t.count;
  w.u0 = (w.x0 - begin) % w.t.count;
  w.piece();
  return true;
}

// A part of an item, in shared memory: one warp goes the way, the others read
// from here what they need (registers are short in all roles).
struct Piece {
  int some;  // 0: there is no more
  int b, h, rt, u0, u1, n, cnt, first, ordered, pre, gap, whole;
  __device__ __forceinline__ int token(int u) const { return (u < pre ? u : u + gap) * kTok; }
};
constexpr int kPieces = 4;

template <int D>
struct PromptShared {
  static constexpr int kHalves = D / 64;             // 64-wide halves of the head dim
  static constexpr int kQ = 2 * kHalves * 16384;     // [row tile][half][128 rows][128 bytes]
  static constexpr int kK = kHalves * 16384;         // a stage: [half][128 tokens][128 bytes]
  static constexpr int kV = 2 * D * 128;             // a stage: [token half][D values][128 bytes]
  static constexpr int off_q = 0, off_k = kQ, off_v = off_k + 2 * kK, off_s = off_v + 2 * kV;
  struct Scales {
    float sk[kScaleStages][kTok], sv[kScaleStages][kTok];
    int pos[kScaleStages][kTok];
    float e[kScaleStages];
    uint32_t zv[2][kTok / 2];   // V zero points as f16 pairs, biased
    float top[2][kCodeWarps];
    Piece piece[kPieces];
    uint64_t piece_full[kPieces], piece_empty[kPieces];
    uint64_t q_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2], t_full[2], s_full[2][2], p_full[2][2], pv_done[2][2], drain;
    uint32_t tmem;
    int fail;
  };
  static constexpr int bytes = off_s + (int)sizeof(Scales) + 1024;  // and room to align
};

__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Bits lo .. hi - 1, as far as there are such.
__device__ __forceinline__ uint32_t bits_of(int lo, int hi) {
  lo = max(lo, 0);
  hi = min(hi, 32);
  return hi <= lo ? 0u : (0xffffffffu >> (32 - hi)) & (0xffffffffu << lo);
}
template <int N>  // products to scores
__device__ __forceinline__ void scaled(uint32_t* y, const float* sk) {
#pragma unroll
  for (int k = 0; k < N; k += 4) {
    const float4 f = *reinterpret_cast<const float4*>(sk + k);
    y[k] = __float_as_uint(__uint_as_float(y[k]) * f.x), y[k + 1] = __float_as_uint(__uint_as_float(y[k + 1]) * f.y);
    y[k + 2] = __float_as_uint(__uint_as_float(y[k + 2]) * f.z), y[k + 3] = __float_as_uint(__uint_as_float(y[k + 3]) * f.w);
  }
}

// Integers of 4 bits as operands: bias + code is exact in the type, and so is
// its difference from bias + zero point.
template <typename T> struct Ints;
template <> struct Ints<__half> {
  static constexpr uint32_t bias = 0x64006400u;  // 1024
  static constexpr int fmt = 0;
  __device__ __forceinline__ static uint32_t sub(uint32_t x, uint32_t z) {
    __half2 h = __hsub2(*reinterpret_cast<__half2*>(&x), *reinterpret_cast<__half2*>(&z));
    return *reinterpret_cast<uint32_t*>(&h);
  }
};
template <> struct Ints<__nv_bfloat16> {
  static constexpr uint32_t bias = 0x43004300u;  // 128
  static constexpr int fmt = 1;
  __device__ __forceinline__ static uint32_t sub(uint32_t x, uint32_t z) {
    __nv_bfloat162 h = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&x), *reinterpret_cast<__nv_bfloat162*>(&z));
    return *reinterpret_cast<uint32_t*>(&h);
  }
};
// The 8 values of a word of K (or 4 of two tokens of V) less their zero points z.
template <typename T>
__device__ __forceinline__ void ints_of(uint32_t w, uint32_t z, uint32_t* r) {
#pragma unroll
  for (int n = 0; n < 4; ++n) r[n] = Ints<T>::sub(((w >> (4 * n)) & 0x000f000fu) | Ints<T>::bias, z);
}

// A tile of 128 query rows on its way into shared memory as a K-major,
// 128-byte-swizzled operand; zeros for what is no row.  128 threads; each waits
// for its own copies with staged().
template <typename T, int D>
__device__ __forceinline__ void stage_rows(uint8_t* dst, const Attn& a, int b, int h, int cnt, int r0, int tid) {
  constexpr int CH = D / 8, STEP = 128 / CH;  // 8 or 16 rows at a time: lr & 7 stays
  const int c = tid % CH, lr = tid / CH;
  uint32_t at = smem_u32(dst) + (c / 8) * 16384 + lr * 128 + (((c % 8) ^ (lr & 7)) << 4);
  // row r = i G + g, and its address, are counted on: a step is di queries and dg heads
  int r = r0 + lr, i = div_g(a, r), g = r - i * a.G;
  const int di = div_g(a, STEP), dg = STEP - di * a.G;
  const T* base = reinterpret_cast<const T*>(a.q) + b * a.q_sb + 8 * c;
  const T* p = base + (int64_t)(h * a.G + g) * a.q_sh + i * a.q_ss;
  const int64_t step = di * a.q_ss + dg * a.q_sh, carry = a.q_ss - a.G * a.q_sh;
#pragma unroll 4
  for (int k = 0; k < CH; ++k) {
    const bool in = r < a.rows && i < cnt;
    const T* from = in ? p : base;
    const int bytes = in ? 16 : 0;  // the rest is filled with zeros
    if (a.q_wide) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(from), "r"(bytes) : "memory");
    } else {
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(at), "l"(from), "r"(bytes / 2) : "memory");
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(at + 8), "l"(from + 4), "r"(bytes / 2) : "memory");
    }
    r += STEP, at += STEP * 128, i += di, g += dg, p += step;
    if (g >= a.G) g -= a.G, ++i, p += carry;
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>  // all but the last N tiles are there, for the MMAs too
__device__ __forceinline__ void staged() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(kPromptThreads, 1) kv4_prompt_kernel(const Attn a) {
  using L = PromptShared<D>;
  constexpr int W = D / 32;
  extern __shared__ __align__(16) uint8_t raw[];
  // aligned without a cast to an integer, after which every access would be generic
  uint8_t* smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  typename L::Scales& sc = *reinterpret_cast<typename L::Scales*>(smem + L::off_s);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rts = a.rows_pad / kItem;
  if (threadIdx.x == 0) {
    sc.fail = 0;
    for (int i = 0; i < kPieces; ++i) {
      mbar_init(&sc.piece_full[i], 1);
      mbar_init(&sc.piece_empty[i], kSoftmaxWarps + kCodeWarps + 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sc.q_full[i], kTile);
      mbar_init(&sc.k_full[i], kCodeWarps);
      mbar_init(&sc.k_empty[i], 1);
      mbar_init(&sc.v_full[i], kCodeWarps);
      mbar_init(&sc.t_full[i], kCodeWarps);
      mbar_init(&sc.v_empty[i], 1);
      // one for each half of S: a row tile's softmax may be a step ahead of the
      // MMAs, and a parity only tells neighbouring phases apart
      for (int h = 0; h < 2; ++h) {
        mbar_init(&sc.s_full[i][h], 1);
        mbar_init(&sc.p_full[i][h], 4);
        mbar_init(&sc.pv_done[i][h], 1);
      }
    }
    mbar_init(&sc.drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == kSoftmaxWarps + kCodeWarps) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sc.tmem)), "r"(512u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sc.tmem;
  // A wait that runs out ends the block: every role leaves its loop, as
  // every wait, this one's aside, is bounded too.  Whole warps agree on it.
  volatile int* fail = &sc.fail;
  auto gone = [&] { return __any_sync(0xffffffffu, *fail != 0); };
  // the k-th piece; its warp's lanes return the slot together
  auto next_piece = [&](int k) {
    if (!wait_warp(&sc.piece_full[k % kPieces], (k / kPieces) & 1)) *fail = 1;
  };
  auto done_with = [&](int k) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&sc.piece_empty[k % kPieces]);
  };

  if (warp < kSoftmaxWarps) {
    // ---------------- softmax: a thread owns a row of its tile ----------------
    more_regs<168>();
    const int wg = warp >> 2, tid = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t O = tmem + lanes + 256 + wg * 128;
    int unit = 0;    // token tiles of this block so far
    int steps = 0;   // half tiles that this row tile has worked on
    for (int k = 0;; ++k) {
      next_piece(k);
      if (gone()) break;
      const Piece& w = sc.piece[k % kPieces];
      if (!w.some) break;
      const int r0 = w.rt * kItem + wg * kTile;
      if (r0 >= a.rows) {
        unit += w.u1 - w.u0;
        done_with(k);
        continue;
      }
      const int r = r0 + tid, i = div_g(a, r);
      const bool valid = r < a.rows && i < w.cnt;
      const int at = w.first + i, n = w.n, n_steps = 2 * (w.u1 - w.u0), ordered = w.ordered;
      const int first_tile = w.u0, pre_tiles = w.pre, gap = w.gap;
      stage_rows<T, D>(smem + L::off_q + wg * (L::kQ / 2), a, w.b, w.h, w.cnt, r0, tid);
      staged<0>();
      mbar_arrive(&sc.q_full[wg]);
      const float slope = a.slopes && r < a.rows ? a.slopes[w.h * a.G + r % a.G] * kLog2e : 0.0f;
      const int pre = a.prefix ? a.prefix[w.b] : 0;
      // positions of the tile's first and last row
      const int qa = w.first + div_g(a, r0), qb = w.first + div_g(a, r0 + kTile - 1);
      // half tiles that begin in here need no masks
      int plain_from = 0, plain_to = n - 64;
      if (a.cap != 0.0f || a.slopes || (!ordered && (a.causal || a.window > 0))) plain_to = -1;
      else {
        if (a.causal) plain_to = min(plain_to, qa - 63);
        if (a.window > 0) plain_from = max(qb - a.window + 1, 0);
      }
      float R = kNone, l = 0.0f;
      for (int j = 0; j < n_steps; ++j, ++steps) {
        const int st = (unit + (j >> 1)) % kScaleStages, u = first_tile + (j >> 1);
        const int t0 = (u < pre_tiles ? u : u + gap) * kTok + 64 * (j & 1);
        const float* sk = sc.sk[st] + 64 * (j & 1);
        const float* sv = sc.sv[st] + 64 * (j & 1);
        const bool plain = t0 >= plain_from && t0 <= plain_to;
        const uint32_t S = tmem + lanes + wg * 128 + 64 * (steps & 1);
        if (!wait_warp(&sc.s_full[wg][steps & 1], (steps >> 1) & 1)) {
          *fail = 1;
          break;
        }
        tc_fence_after();
        const float e = sc.e[st];
        float sum = 0.0f;
        // Raises the row's reference to the greatest score m, and brings O to
        // it once the last PV is complete.  References are whole numbers, so that
        // what is there already, P' in f16 too, is multiplied by powers of two.
        auto raise = [&](float m) {
          m = fmaxf(R, m == -INFINITY ? kNone : ceilf(m + e));
          const float alpha = ex2(R - m);
          l *= alpha;
          sum *= alpha;
          R = m;
          if (j > 0) {
            if (!wait_warp(&sc.pv_done[wg][(steps - 1) & 1], ((steps - 1) >> 1) & 1)) *fail = 1;
            tc_fence_after();
            uint32_t z[16];
#pragma unroll 1
            for (int d = 0; d < D; d += 16) {
              tmem_ld16(O + d, z);
              tmem_wait_ld16(z);
#pragma unroll
              for (int k = 0; k < 16; ++k) z[k] = __float_as_uint(__uint_as_float(z[k]) * alpha);
              tmem_st16(O + d, z);
            }
            tmem_wait_st();  // the step's second half may raise it again
          }
        };
        if (plain) {
          uint32_t y[64], p[32];
          // twice where the reference has to be raised first; one copy of the code
#pragma unroll 1
          for (int pass = 0; pass < 2; ++pass) {
            tmem_ld32(S, y);
            tmem_ld32(S + 32, y + 32);
            tmem_wait_ld32(y);
            tmem_wait_ld32(y + 32);
            if (pass) {
              float m = -INFINITY;
#pragma unroll
              for (int k = 0; k < 64; ++k) m = fmaxf(m, __uint_as_float(y[k]) * sk[k]);
              raise(m);
            }
            const float off = e + kHead - R;
            const uint64_t off2 = pair(off, off);
            float top[2] = {-INFINITY, -INFINITY};
            uint64_t s2[2] = {pair(0.0f, 0.0f), pair(0.0f, 0.0f)};
            // exponentials, sums and conversions in one block, so that the
            // special-function unit is fed while the rest goes on
#pragma unroll
            for (int k = 0; k < 64; k += 4) {
              const float4 f = *reinterpret_cast<const float4*>(sk + k), v = *reinterpret_cast<const float4*>(sv + k);
              const float2 y0 = unpair(fma2(pair(__uint_as_float(y[k]), __uint_as_float(y[k + 1])), pair(f.x, f.y), off2));
              const float2 y1 = unpair(fma2(pair(__uint_as_float(y[k + 2]), __uint_as_float(y[k + 3])), pair(f.z, f.w), off2));
              top[0] = fmaxf(top[0], fmaxf(y0.x, y0.y));
              top[1] = fmaxf(top[1], fmaxf(y1.x, y1.y));
              const uint64_t q0 = pair(ex2(y0.x), ex2(y0.y)), q1 = pair(ex2(y1.x), ex2(y1.y));
              s2[0] = add2(s2[0], q0);
              s2[1] = add2(s2[1], q1);
              const float2 p0 = unpair(mul2(q0, pair(v.x, v.y))), p1 = unpair(mul2(q1, pair(v.z, v.w)));
              p[k / 2] = h2(p0.x, p0.y);
              p[k / 2 + 1] = h2(p1.x, p1.y);
            }
            const float2 x0 = unpair(s2[0]), x1 = unpair(s2[1]);
            sum = (x0.x + x0.y) + (x1.x + x1.y);
            if (!__any_sync(0xffffffffu, fmaxf(top[0], top[1]) > kTop)) break;
          }
          tmem_st16(S, p);  // P' lies over S
          tmem_st16(S + 16, p + 16);
        } else {
#pragma unroll 1
          for (int c = 0; c < 64; c += 32) {
            uint32_t y[32], p[16];
            tmem_ld32(S + c, y);
            tmem_wait_ld32(y);
            // columns that the row sees: between two bounds, or before the prefix
            uint32_t seen;
            const int t = t0 + c;
            if (ordered) {
              seen = bits_of(a.window > 0 ? at - a.window + 1 - t : 0, a.causal ? at + 1 - t : 32) | bits_of(0, pre - t);
            } else {
              const int hi = a.causal ? at : INT_MAX, lo = a.window > 0 ? at - a.window + 1 : INT_MIN;
              const int* pos = sc.pos[st] + 64 * (j & 1) + c;
              seen = 0;
#pragma unroll 8
              for (int k = 0; k < 32; ++k) seen |= ((pos[k] <= hi && pos[k] >= lo) || pos[k] < pre ? 1u : 0u) << k;
            }
            seen &= valid ? bits_of(0, n - t) : 0u;
            scaled<32>(y, sk + c);
            if (a.cap > 0.0f) capped<32>(y, a.cap * kLog2e);
            if (a.slopes) {
              if (ordered) {
                const float d = (float)(at - t);
#pragma unroll
                for (int k = 0; k < 32; ++k) y[k] = __float_as_uint(fmaf(-slope, fabsf(d - (float)k), __uint_as_float(y[k])));
              } else {
                const int* pos = sc.pos[st] + 64 * (j & 1) + c;
#pragma unroll
                for (int k = 0; k < 32; ++k) y[k] = __float_as_uint(fmaf(-slope, fabsf((float)(at - pos[k])), __uint_as_float(y[k])));
              }
            }
            float m = -INFINITY;
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              if (!(seen >> k & 1)) y[k] = 0xff800000u;
              m = fmaxf(m, __uint_as_float(y[k]));
            }
            if (__any_sync(0xffffffffu, m + (e + kHead - R) > kTop)) {
              const float before = R;
              raise(m);
              if (c) {  // the first half's P' is there already
                const float alpha = ex2(before - R);
                tmem_wait_st();  // of P' itself
                tmem_ld16(S, p);
                tmem_wait_ld16(p);
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                  const float2 v = f2(p[k]);
                  p[k] = h2(v.x * alpha, v.y * alpha);
                }
                tmem_st16(S, p);
              }
            }
            const float off = e + kHead - R;
            float s4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
              const float q0 = ex2(__uint_as_float(y[k]) + off), q1 = ex2(__uint_as_float(y[k + 1]) + off);
              const float2 v = *reinterpret_cast<const float2*>(sv + c + k);
              s4[k & 2] += q0;
              s4[(k & 2) + 1] += q1;
              // a token that is not seen has no weight, whatever its scale
              p[k / 2] = h2(seen >> k & 1 ? q0 * v.x : 0.0f, seen >> (k + 1) & 1 ? q1 * v.y : 0.0f);
            }
            sum += (s4[0] + s4[1]) + (s4[2] + s4[3]);
            tmem_st16(S + c / 2, p);
          }
        }
        l = fmaf(sum, ex2(-e - kHead), l);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sc.p_full[wg][steps & 1]);
      }
      unit += n_steps / 2;
      if (gone()) break;
      // ---- the item's rows, or this block's part of them ----
      if (!wait_warp(&sc.pv_done[wg][(steps - 1) & 1], ((steps - 1) >> 1) & 1)) *fail = 1;
      if (gone()) break;
      tc_fence_after();
      if (w.whole) {
        const float inv = !valid || l == 0.0f ? 0.0f : pow2(-(int)kHead) / l;
        T* out = reinterpret_cast<T*>(a.out) + (((int64_t)w.b * a.Hq + w.h * a.G + r % a.G) * a.Sq + i) * D;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t x[32];
          tmem_ld32(O + c, x);
          tmem_wait_ld32(x);
          if (r < a.rows) {
#pragma unroll
            for (int k = 0; k < 32; k += 8) {
              union {
                T t[8];
                uint4 v;
              } y;
#pragma unroll
              for (int d = 0; d < 8; ++d) y.t[d] = Ty<T>::from_f(valid ? __uint_as_float(x[k + d]) * inv : 0.0f);
              st_v4(out + c + k, y.v);
            }
          }
        }
        if (a.lse && r < a.rows)
          a.lse[(int64_t)(w.b * a.kv.H + w.h) * a.rows_pad + r] = !valid || l == 0.0f ? INFINITY : R + lg2(l);
      } else {
        const int64_t row = (int64_t)(2 * blockIdx.x + (k ? 1 : 0)) * kItem + wg * kTile + tid;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t x[32];
          tmem_ld32(O + c, x);
          tmem_wait_ld32(x);
          if (r < a.rows) {
#pragma unroll
            for (int k = 0; k < 32; k += 4)
              *reinterpret_cast<float4*>(a.part + row * D + c + k) =
                  make_float4(__uint_as_float(x[k]), __uint_as_float(x[k + 1]), __uint_as_float(x[k + 2]), __uint_as_float(x[k + 3]));
          }
        }
        if (r < a.rows) a.ml[row] = make_float2(R, valid ? l : 0.0f);
      }
      tc_fence_before();
      done_with(k);
    }
  } else if (warp < kSoftmaxWarps + kCodeWarps) {
    // ---------------- codes to operands ----------------
    fewer_regs<96>();
    const int tid = threadIdx.x - 32 * kSoftmaxWarps, cw = warp - kSoftmaxWarps;
    const int g = tid >> 4, tg = tid & 15;  // V: 16 values (units g W ..) of 8 tokens
    const float fk = a.sm * (a.cap > 0.0f ? 1.0f / a.cap : kLog2e);
    uint32_t kr[2 * W][2], vr[4][W];
    uint2 par = make_uint2(0u, 0u);
    int unit = 0;
    auto fetch_k = [&](const Piece& x, int u) {
      const int t = x.token(u) + tid;
      const int64_t row = (int64_t)(x.b * a.kv.H + x.h) * a.kv.cap;
      par = make_uint2(0u, 0u);
      if (t < x.n) {
        const uint2* p = reinterpret_cast<const uint2*>(a.kv.k + (row + t) * (D / 2));
#pragma unroll
        for (int i = 0; i < 2 * W; ++i) {
          const uint2 v = __ldg(p + i);
          kr[i][0] = v.x, kr[i][1] = v.y;
        }
        par = __ldg(a.kv.par + row + t);
      }
    };
    auto fetch_v = [&](const Piece& x, int u) {
      const int t = x.token(u) + 8 * tg;
      const int64_t row = (int64_t)(x.b * a.kv.H + x.h) * a.kv.cap;
      if (t < x.n) {
        const uint8_t* p = a.kv.v + row * (D / 2) + (int64_t)(t >> 4) * (W * 256) + ((t >> 3) & 1) * (W * 128) + g * (W * 16);
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < W; i += 2) {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(p + c * (W * 4) + i * 4));
            vr[c][i] = v.x, vr[c][i + 1] = v.y;
          }
      }
    };
#pragma unroll
    for (int i = 0; i < 2 * W; ++i) kr[i][0] = kr[i][1] = 0u;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int i = 0; i < W; ++i) vr[c][i] = 0u;
    int k = 0;
    next_piece(0);
    bool more = !gone() && sc.piece[0].some;
    int u = sc.piece[0].u0;
    if (more) {
      fetch_k(sc.piece[0], u);
      fetch_v(sc.piece[0], u);
    }
    while (more) {
      const Piece& w = sc.piece[k % kPieces];
      const int s2 = unit & 1, st = unit % kScaleStages;
      // where the next unit is
      int nk = k, nu = u + 1;
      if (nu == w.u1) {
        nk = k + 1;
        next_piece(nk);
        more = sc.piece[nk % kPieces].some;
        nu = sc.piece[nk % kPieces].u0;
      }
      const Piece& nx = sc.piece[nk % kPieces];
      if (unit >= 2 && !wait_warp(&sc.k_empty[s2], ((unit >> 1) - 1) & 1)) *fail = 1;
      if (gone()) break;
      // ---- K, and the columns' scales ----
      const uint32_t zk = (uint32_t)(int)par_zero(par.x) * 0x10001u + Ints<T>::bias;
      uint8_t* kd = smem + L::off_k + s2 * L::kK + tid * 128;
#pragma unroll
      for (int i = 0; i < 4 * W; ++i) {
        uint32_t r[4];
        ints_of<T>(kr[i >> 1][i & 1], zk, r);
        *reinterpret_cast<uint4*>(kd + (i / 8) * 16384 + (((i % 8) ^ (tid & 7)) << 4)) = make_uint4(r[0], r[1], r[2], r[3]);
      }
      const float sv = par_scale(par.y);
      // a NaN scale (its token reads as NaN) is kept out of the tile's exponent
      const uint32_t top = __reduce_max_sync(0xffffffffu, sv < INFINITY ? __float_as_uint(sv) : 0u);
      if (lane == 0) sc.top[s2][cw] = __uint_as_float(top);
      reinterpret_cast<uint16_t*>(sc.zv[s2])[tid] = (uint16_t)((uint32_t)(int)par_zero(par.y) + 0x6400u);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sc.t_full[s2]);
      if (!wait_warp(&sc.t_full[s2], (unit >> 1) & 1)) *fail = 1;
      if (gone()) break;
      const float big = fmaxf(fmaxf(sc.top[s2][0], sc.top[s2][1]), fmaxf(sc.top[s2][2], sc.top[s2][3]));
      const int e = big > 0.0f ? (int)(__float_as_uint(big) >> 23) - 126 : 0;  // big < 2^e
      sc.sk[st][tid] = par_scale(par.x) * fk;
      sc.sv[st][tid] = sv * __uint_as_float((uint32_t)(127 - e) << 23);
      if (!w.ordered) {
        const int t = w.token(u) + tid;
        sc.pos[st][tid] = t < w.n ? a.kv.pos[(int64_t)(w.b * a.kv.H + w.h) * a.kv.cap + t] : 0;
      }
      if (tid == 0) sc.e[st] = (float)e;
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&sc.k_full[s2]);
      if (more) fetch_k(nx, nu);
      // ---- V^T ----
      if (unit >= 2 && !wait_warp(&sc.v_empty[s2], ((unit >> 1) - 1) & 1)) *fail = 1;
      if (gone()) break;
      const uint4 z = *reinterpret_cast<const uint4*>(&sc.zv[s2][4 * tg]);
      uint8_t* vd = smem + L::off_v + s2 * L::kV + (tg >> 3) * (D * 128);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        uint32_t r[4][4];
        ints_of<__half>(vr[0][i], z.x, r[0]);
        ints_of<__half>(vr[1][i], z.y, r[1]);
        ints_of<__half>(vr[2][i], z.z, r[2]);
        ints_of<__half>(vr[3][i], z.w, r[3]);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int d = 4 * (g * W + i) + n;
          *reinterpret_cast<uint4*>(vd + d * 128 + (((tg & 7) ^ (d & 7)) << 4)) = make_uint4(r[0][n], r[1][n], r[2][n], r[3][n]);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&sc.v_full[s2]);
      if (more) fetch_v(nx, nu);
      if (nk != k) done_with(k);
      k = nk;
      u = nu;
      ++unit;
    }
  } else {
    fewer_regs<80>();
    if (warp == kSoftmaxWarps + kCodeWarps + 1) {
      // ---------------- the way through the items ----------------
      Walk w;
      bool some = walk_begin(a, blockIdx.x, w);
      for (int k = 0;; ++k) {
        if (k >= kPieces && !wait_warp(&sc.piece_empty[k % kPieces], ((k / kPieces) - 1) & 1)) *fail = 1;
        if (gone()) break;
        if (lane == 0) {
          Piece& p = sc.piece[k % kPieces];
          p.some = some;
          if (some) {
            p.b = w.j / rts, p.rt = w.j % rts, p.h = w.h, p.u0 = w.u0, p.u1 = w.u1;
            p.n = w.t.n, p.cnt = w.t.cnt, p.first = w.t.first, p.ordered = w.t.ordered, p.pre = w.t.pre, p.gap = w.t.gap;
            p.whole = w.u0 == 0 && w.u1 == w.t.count;
          }
          mbar_arrive(&sc.piece_full[k % kPieces]);
        }
        if (!some) break;
        some = w.next(a);
      }
    }
    // ---------------- MMA issuer ----------------
    if (warp == kSoftmaxWarps + kCodeWarps) {
      // The whole warp goes the way together and elects the lane that issues, so
      // that descriptors and addresses are warp-uniform values.
      constexpr uint32_t idesc_s = make_idesc(Ints<T>::fmt, 64), idesc_o = make_idesc(0, D);
      const uint32_t base = __reduce_max_sync(0xffffffffu, smem_u32(smem)), tm = __reduce_max_sync(0xffffffffu, tmem);
      int unit = 0, items[2] = {0, 0}, steps[2] = {0, 0};
      bool ok = true;
      for (int k = 0;; ++k) {
        ok = wait_warp(&sc.piece_full[k % kPieces], (k / kPieces) & 1);
        const Piece& w = sc.piece[k % kPieces];
        if (!ok || !w.some) break;
        const int two = __reduce_max_sync(0xffffffffu, w.rt * kItem + kTile < a.rows ? 1 : 0);
        const int n_steps = 2 * __reduce_max_sync(0xffffffffu, w.u1 - w.u0);
        // A slot is the PV of a row tile's half, then an S of the other row tile,
        // which lies where the slot before last had its P' (the MMAs that read it
        // are done by then).  Short code: unrolled further it did not fit the
        // instruction cache, and an MMA took 200 cycles to issue instead of 64.
        auto pv = [&](int wg, int half, int vs, uint32_t fresh) {
          const uint64_t dv = sw128_desc(base + L::off_v) + (uint32_t)((vs * L::kV + half * (D * 128)) >> 4);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_ts(tm + 256 + wg * 128, tm + wg * 128 + 64 * half + 8 * k, dv + ((k * 32) >> 4), idesc_o, k > 0 ? 1u : fresh);
          commit(&sc.pv_done[wg][half]);
        };
        auto qk = [&](int wg, int half, int ks) {
          // a step of 16 along K is 32 bytes of the swizzled rows, 64 are a half
          const uint64_t dq = sw128_desc(base + L::off_q) + (uint32_t)((wg * (L::kQ / 2)) >> 4);
          const uint64_t dk = sw128_desc(base + L::off_k) + (uint32_t)((ks * L::kK + half * 8192) >> 4);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint64_t step = ((k >> 2) * 16384 + (k & 3) * 32) >> 4;
            mma_ss(tm + wg * 128 + 64 * half, dq + step, dk + step, idesc_s, k > 0);
          }
          commit(&sc.s_full[wg][half]);
        };
        // the first S of each half; whichever half comes first is half 0, since a piece has whole tiles
        ok = wait_warp(&sc.k_full[unit & 1], (unit >> 1) & 1) && wait_warp(&sc.q_full[0], items[0]++ & 1);
        if (ok && two) ok = wait_warp(&sc.q_full[1], items[1]++ & 1);
        if (!ok) break;
        tc_fence_after();
        qk(0, 0, unit & 1);
        if (two) qk(1, 0, unit & 1);
        qk(0, 1, unit & 1);
#pragma unroll 1
        for (int t = 0; t < n_steps / 2; ++t) {
          const int u = unit + t, s2 = u & 1, p0 = ((steps[0] >> 1) + t) & 1, p1 = ((steps[1] >> 1) + t) & 1;
          const bool more = t + 1 < n_steps / 2;
          if (!wait_warp(&sc.v_full[s2], (u >> 1) & 1) || !wait_warp(&sc.p_full[0][0], p0)) { ok = false; break; }
          tc_fence_after();
          pv(0, 0, s2, t > 0);
          if (two) qk(1, 1, s2);
          commit(&sc.k_empty[s2]);
          if (two) {
            if (!wait_warp(&sc.p_full[1][0], p1)) { ok = false; break; }
            tc_fence_after();
            pv(1, 0, s2, t > 0);
          }
          if (more) {
            if (!wait_warp(&sc.k_full[s2 ^ 1], ((u + 1) >> 1) & 1)) { ok = false; break; }
            tc_fence_after();
            qk(0, 0, s2 ^ 1);
          }
          if (!wait_warp(&sc.p_full[0][1], p0)) { ok = false; break; }
          tc_fence_after();
          pv(0, 1, s2, 1);
          if (two) {
            if (more) qk(1, 0, s2 ^ 1);
            if (!wait_warp(&sc.p_full[1][1], p1)) { ok = false; break; }
            tc_fence_after();
            pv(1, 1, s2, 1);
          }
          commit(&sc.v_empty[s2]);
          if (more) qk(0, 1, s2 ^ 1);
        }
        if (!ok) break;
        steps[0] += n_steps;
        if (two) steps[1] += n_steps;
        unit += n_steps / 2;
        done_with(k);
      }
      if (!ok) *fail = 1;
      commit(&sc.drain);  // nothing may be in flight when tensor memory is given back
      if (!wait_warp(&sc.drain, 0)) *fail = 1;
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (threadIdx.x == 0) {
    if (*fail) a.kv.sync[3] = LQ_ETIMEOUT;
    pdl_trigger();
  }
  if (warp == kSoftmaxWarps + kCodeWarps)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u));
}

// 8 lanes merge the parts of a row that blocks shared, a block those of 16 rows;
// zeros where there is nothing to see.
constexpr int kMergeRows = 16;
template <int D>
__global__ void __launch_bounds__(128) kv4_prompt_combine_kernel(const Attn a) {
  constexpr int V = D / 32;  // vectors of 4 to a lane
  const int rts = a.rows_pad / kItem, item = blockIdx.x / (kItem / kMergeRows);
  const int j = item / a.kv.H, h = item % a.kv.H, b = j / rts, rt = j % rts;
  const int k = blockIdx.x % (kItem / kMergeRows) * kMergeRows + threadIdx.x / 8, l8 = threadIdx.x & 7, r = rt * kItem + k;
  const Tiles t = tiles_of(a, b, rt);
  int all;
  const int begin = tiles_before(a, j, all) + h * t.count;
  Cut cut;
  cut.set(all, a.blocks);
  const int c0 = t.count ? cut.owner(begin) : 0, c1 = t.count ? cut.owner(begin + t.count - 1) : -1;
  pdl_wait();  // no block ends before the kernel it waits for
  if ((t.count && c0 == c1) || r >= a.rows) return;
  float M = kNone, L = 0.0f;
  float4 o[V];
#pragma unroll
  for (int d = 0; d < V; ++d) o[d] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 2
  for (int c = c0; c <= c1; ++c) {
    const int64_t row = (int64_t)(2 * c + (cut.begin(c) >= begin ? 0 : 1)) * kItem + k;
    const float2 ml = a.ml[row];
    float4 v[V];
#pragma unroll
    for (int d = 0; d < V; ++d) v[d] = *reinterpret_cast<const float4*>(a.part + row * D + 32 * d + 4 * l8);
    const float m = fmaxf(M, ml.x), f = ex2(M - m), g = ex2(ml.x - m);
    M = m;
    L = fmaf(L, f, g * ml.y);
#pragma unroll
    for (int d = 0; d < V; ++d) {
      o[d].x = fmaf(o[d].x, f, g * v[d].x), o[d].y = fmaf(o[d].y, f, g * v[d].y);
      o[d].z = fmaf(o[d].z, f, g * v[d].z), o[d].w = fmaf(o[d].w, f, g * v[d].w);
    }
  }
  const float inv = L == 0.0f ? 0.0f : pow2(-(int)kHead) / L;
  const int i = div_g(a, r), hq = h * a.G + r - i * a.G;
  const int64_t at = (((int64_t)b * a.Hq + hq) * a.Sq + i) * D;
#pragma unroll
  for (int d = 0; d < V; ++d) {
    if (L == 0.0f) o[d] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // padding's O may be anything
    st_out4(a.out, at + 32 * d + 4 * l8, a.q_dtype, o[d], inv);
  }
  if (a.lse && l8 == 0) a.lse[(int64_t)(b * a.kv.H + h) * a.rows_pad + r] = L == 0.0f ? INFINITY : M + lg2(L);
}

// ---------------------------------------------------------------------------
// Collected weight: mass[t] += sum over the rows of exp2(x[r, t] - lse[r]).
//   S^T = (C_k - Z_k) Q^T: 128 tokens (lanes) by 128 rows (columns)
// so that a thread owns a token: it multiplies by its own scale, subtracts the
// rows' log2 denominators and adds up what it has, in a fixed order and with no
// exchange but one at the end between the two groups that take alternate row
// tiles.  A block takes 128 tokens of a head at a time; heads' first tokens come
// first, as with a causal mask they have the most rows.
//
// Warps: 0-3 and 4-7 sums of even and odd row tiles, 8-11 K's codes and the
// query rows to operands, 12 the MMAs.  Bound: 16384 exponentials to a pair of
// tiles, 1024 cycles, beside 512 of the tensor cores.  Measured: 2 x 1024 queries
// of 8 kv heads x 4 on 2048 tokens, D = 128, causal: 74 us (special-function units
// 41 % while an SM has work, which it has for 71 % of the time).
// ---------------------------------------------------------------------------
constexpr int kWeighThreads = 416;
constexpr int kQs = 4;  // stages of query rows; what belongs to rows is kept twice as long, for the sums
template <int D>
struct WeighShared {
  static constexpr int kOp = D / 64 * 16384;  // an operand of 128 rows
  static constexpr int off_k = 0, off_q = kOp, off_s = off_q + kQs * kOp;
  struct Rows {
    float nl[2 * kQs][kTile], slope[2 * kQs][kTile];  // -lse, bias
    int at[2 * kQs][kTile];
    float sk[2][kTok], half[2][kTok];
    int pos[2][kTok];
    // item_done: the eight warps of the sums are through with an item of this parity,
    // whose half, sk and pos may then be another's.  An item of one row tile gives one group
    // nothing to wait for, so that it could be two items ahead of the other.
    uint64_t k_full, k_empty, q_full[kQs], q_empty[kQs], s_full[2], s_empty[2], half_full[2], item_done[2], drain;
    uint32_t tmem;
    int fail;
  };
  static constexpr int bytes = off_s + (int)sizeof(Rows) + 1024;
};
// Tokens t0 .. of head bh, and the row tiles [lo, hi) that may see any of them.
struct WeighItem {
  int b, h, t0, n, cnt, first, ordered, lo, hi;
};
__device__ __forceinline__ WeighItem weigh_item(const Attn& a, int idx) {
  WeighItem w;
  const int heads = a.kv.B * a.kv.H, bh = idx % heads;
  w.b = bh / a.kv.H, w.h = bh % a.kv.H, w.t0 = idx / heads * kTok;
  const Seq s = seq_of(a, w.b);
  w.n = s.n, w.cnt = s.cnt, w.first = s.first, w.ordered = s.ordered;
  w.lo = 0, w.hi = w.t0 < s.n ? (s.cnt * a.G + kTile - 1) / kTile : 0;
  if (s.ordered && !(a.prefix && w.t0 < a.prefix[w.b])) {
    if (a.causal) w.lo = (int)((int64_t)max(w.t0 - s.first, 0) * a.G / kTile);
    if (a.window > 0) {
      const int64_t i = (int64_t)w.t0 + kTok - 1 + a.window - s.first;  // queries from here on are past the window
      w.hi = (int)min((int64_t)w.hi, i <= 0 ? 0 : (i * a.G + kTile - 1) / kTile);
    }
  }
  return w;
}

// CAP apart: its code beside the rest costs calls without a cap 2 % (instruction cache).
template <typename T, int D, bool CAP>
__global__ void __launch_bounds__(kWeighThreads, 1) kv4_weigh_kernel(const Attn a) {
  using L = WeighShared<D>;
  constexpr int W = D / 32;
  extern __shared__ __align__(16) uint8_t raw[];
  uint8_t* smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  typename L::Rows& sc = *reinterpret_cast<typename L::Rows*>(smem + L::off_s);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    sc.fail = 0;
    mbar_init(&sc.k_full, 4);
    mbar_init(&sc.k_empty, 1);
    for (int i = 0; i < kQs; ++i) {
      mbar_init(&sc.q_full[i], 4);
      mbar_init(&sc.q_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sc.s_full[i], 1);
      mbar_init(&sc.s_empty[i], 4);
      mbar_init(&sc.half_full[i], 4);
      mbar_init(&sc.item_done[i], 8);
    }
    mbar_init(&sc.drain, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sc.tmem)), "r"(256u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sc.tmem;
  volatile int* fail = &sc.fail;
  const float fk = a.sm * (CAP ? 1.0f / a.cap : kLog2e);
  int longest = 0;
  for (int b = lane; b < a.kv.B; b += 32) longest = max(longest, min(a.kv.len[b], a.kv.cap));
  const int items = (__reduce_max_sync(0xffffffffu, longest) + kTok - 1) / kTok * a.kv.B * a.kv.H;

  if (warp < 8) {
    const int wg = warp >> 2, tid = threadIdx.x & 127;
    const uint32_t S = tmem + ((uint32_t)((warp & 3) * 32) << 16) + wg * 128;
    int tile = 0, mine = 0, item = 0;  // row tiles so far, of this group, items with any
    bool ok = true;
    for (int idx = blockIdx.x; idx < items && ok; idx += gridDim.x) {
      const WeighItem w = weigh_item(a, idx);
      if (w.lo >= w.hi) continue;
      const int t = w.t0 + tid, pre = a.prefix ? a.prefix[w.b] : 0, odd = (tile + wg) & 1;
      float sum = 0.0f, sk = 0.0f;
      int pos = t;
      for (int rt = w.lo + odd; rt < w.hi; rt += 2, ++mine) {
        const int st = (tile + rt - w.lo) % (2 * kQs);
        if (!wait_warp(&sc.s_full[wg], mine & 1)) { ok = false; break; }
        tc_fence_after();
        sk = sc.sk[item & 1][tid];
        if (!w.ordered) pos = sc.pos[item & 1][tid];
        const int q0 = w.first + div_g(a, rt * kTile), q1 = w.first + min(div_g(a, rt * kTile + kTile - 1), w.cnt - 1);
        const bool plain = !CAP && !a.slopes &&
                           ((!a.causal && a.window <= 0) ||
                            (w.ordered && (!a.causal || w.t0 + kTok - 1 <= q0) && (a.window <= 0 || q1 - w.t0 < a.window)));
        if (plain) {
          uint64_t s2[2] = {pair(0.0f, 0.0f), pair(0.0f, 0.0f)};
          const uint64_t k2 = pair(sk, sk);
#pragma unroll 1
          for (int c = 0; c < kTile; c += 64) {
            uint32_t y[64];
            tmem_ld32(S + c, y);
            tmem_ld32(S + c + 32, y + 32);
            tmem_wait_ld32(y);
            tmem_wait_ld32(y + 32);
#pragma unroll
            for (int k = 0; k < 64; k += 4) {
              const float4 f = *reinterpret_cast<const float4*>(&sc.nl[st][c + k]);
              const float2 y0 = unpair(fma2(pair(__uint_as_float(y[k]), __uint_as_float(y[k + 1])), k2, pair(f.x, f.y)));
              const float2 y1 = unpair(fma2(pair(__uint_as_float(y[k + 2]), __uint_as_float(y[k + 3])), k2, pair(f.z, f.w)));
              s2[0] = add2(s2[0], pair(ex2(y0.x), ex2(y0.y)));
              s2[1] = add2(s2[1], pair(ex2(y1.x), ex2(y1.y)));
            }
          }
          const float2 x0 = unpair(s2[0]), x1 = unpair(s2[1]);
          sum += (x0.x + x0.y) + (x1.x + x1.y);
        } else {
          // rows that see the token: those between two, or all
          const int64_t hi_r = a.window > 0 ? ((int64_t)pos + a.window - w.first) * a.G - rt * kTile : kTile;
          const int64_t lo_r = a.causal ? ((int64_t)pos - w.first) * a.G - rt * kTile : 0;
          const int lo = (int)max(min(lo_r, (int64_t)kTile), (int64_t)-1), hi = (int)max(min(hi_r, (int64_t)kTile), (int64_t)-1);
          const float d = (float)(pos - w.first);  // and the queries count from 0: positions may pass 2^24
#pragma unroll 1
          for (int c = 0; c < kTile; c += 32) {
            uint32_t y[32];
            tmem_ld32(S + c, y);
            tmem_wait_ld32(y);
            const uint32_t seen = pos < pre ? 0xffffffffu : bits_of(lo - c, hi - c);
#pragma unroll
            for (int k = 0; k < 32; ++k) y[k] = __float_as_uint(__uint_as_float(y[k]) * sk);
            if constexpr (CAP) capped<32>(y, a.cap * kLog2e);
            if (a.slopes) {
#pragma unroll
              for (int k = 0; k < 32; ++k)
                y[k] = __float_as_uint(fmaf(-sc.slope[st][c + k], fabsf((float)sc.at[st][c + k] - d), __uint_as_float(y[k])));
            }
            float s4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              const float p = ex2(__uint_as_float(y[k]) + sc.nl[st][c + k]);
              s4[k & 3] += seen >> k & 1 ? p : 0.0f;
            }
            sum += (s4[0] + s4[1]) + (s4[2] + s4[3]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sc.s_empty[wg]);
      }
      if (!ok) break;
      // the groups' sums, and what the token had
      if (wg == 1) {
        if (item >= 2 && !wait_warp(&sc.item_done[item & 1], ((item >> 1) - 1) & 1)) { ok = false; break; }
        sc.half[item & 1][tid] = sum;
        __syncwarp();
        if (lane == 0) mbar_arrive(&sc.half_full[item & 1]);
      } else {
        if (!wait_warp(&sc.half_full[item & 1], (item >> 1) & 1)) { ok = false; break; }
        if (t < w.n) a.kv.mass[(int64_t)(w.b * a.kv.H + w.h) * a.kv.cap + t] += sum + sc.half[item & 1][tid];
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sc.item_done[item & 1]);
      ++item;
      tile += w.hi - w.lo;
    }
    if (!ok) *fail = 1;
  } else if (warp < 12) {
    const int tid = threadIdx.x - 256;
    int tile = 0, item = 0;
    bool ok = true;
    for (int idx = blockIdx.x; idx < items && ok; idx += gridDim.x) {
      const WeighItem w = weigh_item(a, idx);
      if (w.lo >= w.hi) continue;
      // ---- K ----
      const int t = w.t0 + tid;
      const int64_t row = (int64_t)(w.b * a.kv.H + w.h) * a.kv.cap + t;
      const bool in = t < w.n;
      const uint32_t par = in ? a.kv.par[row].x : 0u;
      if (item > 0 && !wait_warp(&sc.k_empty, (item - 1) & 1)) { ok = false; break; }
      if (item >= 2 && !wait_warp(&sc.item_done[item & 1], ((item >> 1) - 1) & 1)) { ok = false; break; }
      const uint32_t zk = (uint32_t)(int)par_zero(par) * 0x10001u + Ints<T>::bias;
      uint8_t* kd = smem + L::off_k + tid * 128;
#pragma unroll 2
      for (int i = 0; i < 4 * W; i += 2) {
        const uint2 v = in ? __ldg(reinterpret_cast<const uint2*>(a.kv.k + row * (D / 2)) + i / 2) : make_uint2(0u, 0u);
        uint32_t r[4];
        ints_of<T>(v.x, zk, r);
        *reinterpret_cast<uint4*>(kd + (i / 8) * 16384 + (((i % 8) ^ (tid & 7)) << 4)) = make_uint4(r[0], r[1], r[2], r[3]);
        ints_of<T>(v.y, zk, r);
        *reinterpret_cast<uint4*>(kd + (i / 8) * 16384 + (((i % 8 + 1) ^ (tid & 7)) << 4)) = make_uint4(r[0], r[1], r[2], r[3]);
      }
      sc.sk[item & 1][tid] = par_scale(par) * fk;
      if (!w.ordered) sc.pos[item & 1][tid] = in ? a.kv.pos[row] : 0;
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&sc.k_full);
      // ---- query rows, two tiles on their way while another arrives ----
      const float* lse = a.lse + (int64_t)(w.b * a.kv.H + w.h) * a.rows_pad;
      auto lse_of = [&](int rt) {
        const int r = rt * kTile + tid;
        return r < a.rows && div_g(a, r) < w.cnt ? -__ldcg(lse + r) : -INFINITY;
      };
      float nl = lse_of(w.lo);
      for (int rt = w.lo; rt < w.hi; ++rt, ++tile) {
        const int qs = tile % kQs, st = tile % (2 * kQs);
        if (tile >= kQs && !wait_warp(&sc.q_empty[qs], (tile / kQs - 1) & 1)) { ok = false; break; }
        stage_rows<T, D>(smem + L::off_q + qs * L::kOp, a, w.b, w.h, w.cnt, rt * kTile, tid);
        sc.nl[st][tid] = nl;
        if (rt + 1 < w.hi) nl = lse_of(rt + 1);
        const int r = rt * kTile + tid, i = div_g(a, r);
        sc.at[st][tid] = i;
        if (a.slopes) sc.slope[st][tid] = r < a.rows ? a.slopes[w.h * a.G + r - i * a.G] * kLog2e : 0.0f;
        if (rt >= w.lo + 2) {
          staged<2>();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sc.q_full[(tile - 2) % kQs]);
        }
      }
      if (!ok) break;
      if (w.hi >= w.lo + 2) {
        staged<1>();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sc.q_full[(tile - 2) % kQs]);
      }
      staged<0>();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sc.q_full[(tile - 1) % kQs]);
      ++item;
    }
    if (!ok) *fail = 1;
    staged<0>();  // nothing on its way when the block ends, after a failed wait too
  } else {
    constexpr uint32_t idesc = make_idesc(Ints<T>::fmt, kTile);
    const uint32_t base = __reduce_max_sync(0xffffffffu, smem_u32(smem)), tm = __reduce_max_sync(0xffffffffu, tmem);
    int tile = 0, item = 0, used[2] = {0, 0};
    bool ok = true;
    for (int idx = blockIdx.x; idx < items && ok; idx += gridDim.x) {
      const WeighItem w = weigh_item(a, idx);
      const int tiles = __reduce_max_sync(0xffffffffu, max(w.hi - w.lo, 0));
      if (tiles == 0) continue;
      if (!wait_warp(&sc.k_full, item & 1)) { ok = false; break; }
      // row tile `tile` goes to group tile % 2, whichever item it is of
#pragma unroll 1
      for (int i = 0; i < tiles; ++i, ++tile) {
        const int qs = tile % kQs, wg = tile & 1;
        if (!wait_warp(&sc.q_full[qs], (tile / kQs) & 1)) { ok = false; break; }
        if (used[wg] > 0 && !wait_warp(&sc.s_empty[wg], (used[wg] - 1) & 1)) { ok = false; break; }
        ++used[wg];
        tc_fence_after();
        const uint64_t dk = sw128_desc(base + L::off_k), dq = sw128_desc(base + L::off_q + qs * L::kOp);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint64_t step = ((k >> 2) * 16384 + (k & 3) * 32) >> 4;
          mma_ss(tm + wg * 128, dk + step, dq + step, idesc, k > 0);
        }
        commit(&sc.s_full[wg]);
        commit(&sc.q_empty[qs]);
      }
      commit(&sc.k_empty);
      ++item;
    }
    if (!ok) *fail = 1;
    commit(&sc.drain);
    if (!wait_warp(&sc.drain, 0)) *fail = 1;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (threadIdx.x == 0 && *fail) a.kv.sync[3] = LQ_ETIMEOUT;
  if (warp == 12)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256u));
}

template <typename T, int D, bool CAP>
int run_weigh(const Attn& a, cudaStream_t st) {
  constexpr int smem = WeighShared<D>::bytes;
  auto kern = kv4_weigh_kernel<T, D, CAP>;
  static DeviceOnce once;
  LQ_TRY(once.allow_smem((const void*)kern, smem, "kv4_weigh_kernel"));
  const int64_t items = (int64_t)((a.kv.cap + kTok - 1) / kTok) * a.kv.B * a.kv.H;
  LQ_REQUIRE(items <= INT32_MAX, LQ_ERANGE, "cache too large to collect weights");
  kern<<<(int)std::min<int64_t>(items, num_sms()), kWeighThreads, smem, st>>>(a);
  return launched("kv4_weigh_kernel");
}

template <typename T, int D>
int run_prompt(const Attn& a, cudaStream_t st) {
  constexpr int smem = PromptShared<D>::bytes;
  static_assert(smem <= 227 * 1024, "shared memory per block");
  auto kern = kv4_prompt_kernel<T, D>;
  static DeviceOnce once;
  LQ_TRY(once.allow_smem((const void*)kern, smem, "kv4_prompt_kernel"));
  kern<<<a.blocks, kPromptThreads, smem, st>>>(a);
  LQ_TRY(launched("kv4_prompt_kernel"));
  launch_pdl(kv4_prompt_combine_kernel<D>, dim3((unsigned)(a.rows_pad / kMergeRows * a.kv.B * a.kv.H)), dim3(128), 0, st, a);
  LQ_TRY(launched("kv4_prompt_combine_kernel"));
  if (!a.lse) return LQ_OK;
  return a.cap > 0.0f ? run_weigh<T, D, true>(a, st) : run_weigh<T, D, false>(a, st);
}

}  // namespace

int kv4_prompt(const Attn& a, cudaStream_t st) {
  if (a.q_dtype == LQ_F16) return a.kv.D == 128 ? run_prompt<__half, 128>(a, st) : run_prompt<__half, 64>(a, st);
  return a.kv.D == 128 ? run_prompt<__nv_bfloat16, 128>(a, st) : run_prompt<__nv_bfloat16, 64>(a, st);
}

}  // namespace lq

// lq_adapters_mm.cu -- the three products of the adapter bank for batches of
// many tokens, over tiles of up to 128 tokens of one adapter:
//   ad_down    u = s A x      [128 tokens x K] by [K x rank], tcgen05
//   ad_up      y = base + B^T u   [128 tokens x rank] by [rank x 256], mma.sync
//   ad_outer   dA = sum v x^T  [256 columns x tokens] by [tokens x rank], tcgen05
// All three are bound by memory (2 R flops to 2 bytes of x): the point is to
// read x, dy and base once, and to keep the loads coming.
//
// u and v are fp32.  Where they meet a 16-bit factor they go in as two 16-bit
// values, hi = round(u) and lo = round(u - hi), and two products: u is then off
// by 2^-16 of itself (bf16; 2^-22 in fp16), far below the rounding of the
// output, where one 16-bit value would be off as much as that.  fp16 has too
// small a range for values nobody scaled: a row of u (an adapter's rows of v)
// goes in times a power of two that puts its greatest below 2^13, which is
// taken back from the fp32 sum.
#include "lq_adapters.cuh"
#include "lq_tc.cuh"

namespace lq {
namespace {

template <typename T> struct Half16;
template <> struct Half16<__half> {
  static constexpr int fmt = 0;
  static constexpr bool scaled = true;
  __device__ __forceinline__ static uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ __forceinline__ static float2 unpack(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
  __device__ __forceinline__ static void mma(float* d, const uint4& a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
  }
};
template <> struct Half16<__nv_bfloat16> {
  static constexpr int fmt = 1;
  static constexpr bool scaled = false;
  __device__ __forceinline__ static uint32_t pack(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ __forceinline__ static float2 unpack(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  __device__ __forceinline__ static void mma(float* d, const uint4& a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
  }
};

constexpr float kInf = __builtin_huge_valf();

// Two fp32 values as two 16-bit pairs that add up to them.
template <typename T>
__device__ __forceinline__ void split(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = Half16<T>::pack(a, b);
  const float2 h = Half16<T>::unpack(hi);
  // nothing is left of what went to infinity (infinity less itself is NaN)
  lo = Half16<T>::pack(fabsf(h.x) < kInf ? a - h.x : 0.0f, fabsf(h.y) < kInf ? b - h.y : 0.0f);
}
// The power of two that brings values of magnitude m (finite) below 2^13.
__device__ __forceinline__ int scale_exp(float m) {
  if (m == 0.0f) return 0;
  return 12 - max((int)(__float_as_uint(m) >> 23) - 127, -113);
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
__device__ __forceinline__ float finite_mag(float v) {
  v = fabsf(v);
  return v < kInf ? v : 0.0f;
}

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool some) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(some ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ float4 ld_cluster_v4(uint32_t addr, uint32_t rank) {
  uint32_t ra;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(addr), "r"(rank));
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(ra) : "memory");
  return v;
}

__device__ __forceinline__ int token_of(const AdPlan& p, const AdTile& d, int row) {
  return d.run >= 0 ? d.run + row : p.order[d.first + row];
}

// ---------------------------------------------------------------------------
// u = s f x over one tile: D [128 tokens x NP] += X [128 x 64] F^T [64 x NP] in
// steps of 64 k.  A cluster of `split` blocks shares a tile's K and adds its
// partial sums up through distributed shared memory, block by block.
// ---------------------------------------------------------------------------
template <int NP>
struct DownShared {
  static constexpr int stages = NP <= 32 ? 5 : NP <= 64 ? 4 : 3;
  static constexpr int stage = 16384 + NP * 128;
  static constexpr int pitch = NP + 4;  // of the partial sums: rows 16 bytes apart in the banks
  static constexpr int bytes = stages * stage + 1024;
  static_assert(stages * stage >= 128 * pitch * 4, "partial sums take the stages' place");
};

template <typename T, int NP>
__global__ void __launch_bounds__(160, 2) ad_down_kernel(const T* __restrict__ x, int64_t stride, const T* __restrict__ f,
                                                         const float* __restrict__ scaling, int R, int pitch, int K, AdPlan p,
                                                         int L, float* __restrict__ u, int split) {
  using S = DownShared<NP>;
  constexpr int NS = S::stages, LAG = NS - 2;
  constexpr uint32_t kCols = NP < 32 ? 32 : NP;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[NS], empty[NS], done;
  __shared__ uint32_t tmem_at;
  __shared__ int failed;
  pdl_wait();
  pdl_trigger();
  const int tile = blockIdx.x / split, rank = blockIdx.x - tile * split;
  if (tile >= p.tile_of[L]) return;  // the whole cluster
  const AdTile d = p.tiles[tile];
  const int tid = threadIdx.x, warp = tid >> 5;
  const uint32_t base = (smem_u32(raw) + 1023) & ~1023u;
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) mbar_init(&full[i], 128), mbar_init(&empty[i], 1);
    mbar_init(&done, 1);
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    proxy_fence();
  }
  if (warp == 4) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_at)), "r"(kCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_at;
  const int all = (K + 63) / 64, s0 = (int)((int64_t)all * rank / split), n = (int)((int64_t)all * (rank + 1) / split) - s0;
  if (warp < 4) {
    const int c = tid & 7, r0 = tid >> 3;
    const T* xr[8];
    const T* fr[NP / 16];
#pragma unroll
    for (int i = 0; i < 8; ++i) xr[i] = r0 + 16 * i < d.rows ? x + (int64_t)token_of(p, d, r0 + 16 * i) * stride : nullptr;
#pragma unroll
    for (int i = 0; i < NP / 16; ++i) fr[i] = r0 + 16 * i < R ? f + ((int64_t)d.owner * R + r0 + 16 * i) * K : nullptr;
    const uint32_t at = base + r0 * 128 + ((c ^ (r0 & 7)) << 4);
    for (int i = 0; i < n + LAG; ++i) {
      if (i < n) {
        const int slot = i % NS;
        if (i >= NS && !mbar_wait(&empty[slot], (i / NS - 1) & 1)) failed = 1;
        if (*(volatile int*)&failed) break;
        const int k = (s0 + i) * 64 + c * 8;
        const bool some = k < K;  // behind K: zeros in both factors
        const int kk = some ? k : 0;
        const uint32_t to = at + slot * S::stage;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (xr[j]) cp16(to + j * 2048, xr[j] + kk, some);
#pragma unroll
        for (int j = 0; j < NP / 16; ++j)
          if (fr[j]) cp16(to + 16384 + j * 2048, fr[j] + kk, some);
      }
      cp_commit();
      if (i >= LAG) {
        cp_wait<LAG>();
        proxy_fence();
        mbar_arrive(&full[(i - LAG) % NS]);
      }
    }
    cp_wait<0>();
  } else {
    constexpr uint32_t idesc = make_idesc(Half16<T>::fmt, NP);
    for (int i = 0; i < n; ++i) {
      const int slot = i % NS;
      if (!wait_warp(&full[slot], (i / NS) & 1)) {
        failed = 1;
        break;
      }
      tc_fence_after();
      const uint64_t da = sw128_desc(base + slot * S::stage), db = sw128_desc(base + slot * S::stage + 16384);
#pragma unroll
      for (int k = 0; k < 4; ++k) mma_ss(tmem, da + 2 * k, db + 2 * k, idesc, (i | k) > 0);
      commit(&empty[slot]);
    }
    commit(&done);
  }
  const float s = scaling[d.owner];
  const bool ok = mbar_wait_warp(&done, 0);
  if (!ok) failed = 1;
  tc_fence_after();
  if (warp < 4) {
    const int row = tid;
    const bool mine = split == 1 && row < d.rows;
    float* to = mine ? u + (int64_t)token_of(p, d, row) * pitch : nullptr;
#pragma unroll
    for (int c = 0; c < NP; c += 16) {
      uint32_t v[16];
      tmem_ld16(tmem + ((uint32_t)warp << 21) + c, v);
      tmem_wait_ld16(v);
#pragma unroll
      for (int q = 0; q < 16; q += 4) {
        float4 w = make_float4(__uint_as_float(v[q]), __uint_as_float(v[q + 1]), __uint_as_float(v[q + 2]), __uint_as_float(v[q + 3]));
        if (split == 1) {
          if (mine && c + q < pitch) {  // ranks behind R: rows of F that nobody loaded
            w.x = c + q < R ? w.x * s : 0.0f, w.y = c + q + 1 < R ? w.y * s : 0.0f;
            w.z = c + q + 2 < R ? w.z * s : 0.0f, w.w = c + q + 3 < R ? w.w * s : 0.0f;
            *reinterpret_cast<float4*>(to + c + q) = w;
          }
        } else {
          asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(base + (row * S::pitch + c + q) * 4), "f"(w.x), "f"(w.y), "f"(w.z), "f"(w.w) : "memory");
        }
      }
    }
    tc_fence_before();
  }
  if (split > 1) {
    cluster_arrive();
    cluster_wait();
    if (warp < 4) {
      const int rows = 128 / split;
      for (int e = tid; e < rows * (NP / 4); e += 128) {
        const int row = rank * rows + e / (NP / 4), r = e % (NP / 4) * 4;
        if (row >= d.rows || r >= pitch) continue;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int b = 0; b < split; ++b) {
          const float4 w = ld_cluster_v4(base + (row * S::pitch + r) * 4, b);
          v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
        }
        v.x = r < R ? v.x * s : 0.0f, v.y = r + 1 < R ? v.y * s : 0.0f;
        v.z = r + 2 < R ? v.z * s : 0.0f, v.w = r + 3 < R ? v.w * s : 0.0f;
        *reinterpret_cast<float4*>(u + (int64_t)token_of(p, d, row) * pitch + r) = v;
      }
    }
    cluster_arrive();
    cluster_wait();  // no block leaves while others read its sums
  }
  __syncthreads();
  if (tid == 0 && failed) *p.status = LQ_ETIMEOUT;
  if (warp == 4) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols));
}

// ---------------------------------------------------------------------------
// out = base + u f over one tile and 256 columns.  A warp has 32 columns: its
// part of F stays in registers as B operands while the tile's 8 groups of 16
// rows pass.  A lane's 8 values of an output row are neighbours: F's columns are
// dealt out to the four 8-column operands so (column 8 p + 2 j + e goes to
// operand j, place 2 p + e), so that base and out move in whole 16-byte pieces
// between global memory and registers.
// ---------------------------------------------------------------------------
template <int NP>
struct UpShared {
  static constexpr int row = 512 + 16;  // bytes of a rank's 256 columns: 8 rows' pieces in all banks
  static constexpr int off_u = NP * row;
  static constexpr int bytes = off_u + NP * 512;
};

template <typename T, int NP>
__global__ void __launch_bounds__(256, NP <= 64 ? 2 : 1)
    ad_up_kernel(const float* __restrict__ u, int pitch, const T* __restrict__ f, int R, int N, AdPlan p, int L,
                 const T* base, int64_t base_stride, T* out, int64_t out_stride, int chunks) {
  using S = UpShared<NP>;
  using H = Half16<T>;
  extern __shared__ __align__(16) uint8_t raw[];
  __shared__ int64_t tok[kAdTile];
  __shared__ float back[kAdTile];
  pdl_wait();
  pdl_trigger();
  const int tile = blockIdx.x / chunks, col0 = (blockIdx.x - tile * chunks) * 256;
  if (tile >= p.tile_of[L + 1]) return;
  const AdTile d = p.tiles[tile];
  if (d.owner < 0 && base == out) return;  // nothing changes
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  if (tid < kAdTile) tok[tid] = tid < d.rows ? token_of(p, d, tid) : -1;
  const uint32_t at = smem_u32(raw);
  if (d.owner >= 0) {
    // F: 64 bytes of a row at a time, as a 4 x 4 transpose of words
    for (int e = tid; e < NP * 8; e += 256) {
      const int r = e >> 3, q = e & 7;
      uint32_t w[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int col = col0 + q * 32 + i * 8;
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (r < R && col < N) v = __ldg(reinterpret_cast<const uint4*>(f + ((int64_t)d.owner * R + r) * N + col));
        w[i][0] = v.x, w[i][1] = v.y, w[i][2] = v.z, w[i][3] = v.w;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + r * S::row + q * 64 + j * 16), "r"(w[0][j]), "r"(w[1][j]), "r"(w[2][j]), "r"(w[3][j]) : "memory");
    }
  }
  __syncthreads();
  if (d.owner >= 0) {
    // u: warp w makes the A operands of rows 16 w .. 16 w + 15
    const int64_t t0 = tok[16 * warp + g], t1 = tok[16 * warp + g + 8];
    float v[NP / 16][8];
    float m0 = 0.0f, m1 = 0.0f;
#pragma unroll
    for (int k = 0; k < NP / 16; ++k) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = 16 * k + 8 * h + 2 * c;
        const float2 a = t0 >= 0 && r < pitch ? *reinterpret_cast<const float2*>(u + t0 * pitch + r) : make_float2(0.0f, 0.0f);
        const float2 b = t1 >= 0 && r < pitch ? *reinterpret_cast<const float2*>(u + t1 * pitch + r) : make_float2(0.0f, 0.0f);
        v[k][4 * h] = a.x, v[k][4 * h + 1] = a.y, v[k][4 * h + 2] = b.x, v[k][4 * h + 3] = b.y;
        if (H::scaled) {
          m0 = fmaxf(m0, fmaxf(finite_mag(a.x), finite_mag(a.y)));
          m1 = fmaxf(m1, fmaxf(finite_mag(b.x), finite_mag(b.y)));
        }
      }
    }
    float f0 = 1.0f, f1 = 1.0f;
    if (H::scaled) {
#pragma unroll
      for (int i = 1; i < 4; i <<= 1) {
        m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, i));
        m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, i));
      }
      const int e0 = scale_exp(m0), e1 = scale_exp(m1);
      f0 = exp2i(e0), f1 = exp2i(e1);
      if (c == 0) back[16 * warp + g] = exp2i(-e0), back[16 * warp + g + 8] = exp2i(-e1);
    }
#pragma unroll
    for (int k = 0; k < NP / 16; ++k) {
      uint4 hi, lo;
      split<T>(v[k][0] * f0, v[k][1] * f0, hi.x, lo.x);
      split<T>(v[k][2] * f1, v[k][3] * f1, hi.y, lo.y);
      split<T>(v[k][4] * f0, v[k][5] * f0, hi.z, lo.z);
      split<T>(v[k][6] * f1, v[k][7] * f1, hi.w, lo.w);
      uint4* to = reinterpret_cast<uint4*>(raw + S::off_u) + ((warp * (NP / 16) + k) * 2) * 32 + lane;
      to[0] = hi, to[32] = lo;
    }
  }
  __syncthreads();
  const int col = col0 + warp * 32 + c * 8;
  if (col0 + warp * 32 >= N) return;
  const bool in = col < N;
  uint32_t b[NP / 16][8];
  if (d.owner >= 0) {
#pragma unroll
    for (int k = 0; k < NP / 16; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        // lanes 0..15: the 16 ranks of operand 2 h, lanes 16..31: of operand 2 h + 1
        const uint32_t a = at + (16 * k + (lane & 15)) * S::row + warp * 64 + (2 * h + (lane >> 4)) * 16;
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(b[k][4 * h]), "=r"(b[k][4 * h + 1]), "=r"(b[k][4 * h + 2]), "=r"(b[k][4 * h + 3])
                     : "r"(a));
      }
  }
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  constexpr int AHEAD = 4;  // groups of 16 rows whose base is on its way
  uint4 y[AHEAD][2];
  auto fetch = [&](int mt) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t t = tok[16 * mt + 8 * h + g];
      y[mt % AHEAD][h] = base && in && t >= 0 ? *reinterpret_cast<const uint4*>(base + t * base_stride + col) : zero;
    }
  };
#pragma unroll
  for (int mt = 0; mt < AHEAD; ++mt) fetch(mt);
#pragma unroll
  for (int mt = 0; mt < 8; ++mt) {
    if (16 * mt >= d.rows) break;
    float acc[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = 0.0f;
    if (d.owner >= 0) {
      const uint4* from = reinterpret_cast<const uint4*>(raw + S::off_u) + mt * (NP / 16) * 64 + lane;
#pragma unroll
      for (int k = 0; k < NP / 16; ++k) {
        const uint4 hi = from[64 * k], lo = from[64 * k + 32];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          H::mma(acc[j], lo, b[k][2 * j], b[k][2 * j + 1]);
          H::mma(acc[j], hi, b[k][2 * j], b[k][2 * j + 1]);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = 16 * mt + 8 * h + g;
      const int64_t t = tok[row];
      const float w = H::scaled && d.owner >= 0 ? back[row] : 1.0f;
      const uint4 z = y[mt % AHEAD][h];
      uint32_t o[4] = {z.x, z.y, z.z, z.w};
      if (d.owner >= 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 q = H::unpack(o[j]);
          o[j] = H::scaled ? H::pack(fmaf(acc[j][2 * h], w, q.x), fmaf(acc[j][2 * h + 1], w, q.y))
                           : H::pack(q.x + acc[j][2 * h], q.y + acc[j][2 * h + 1]);
        }
      }
      if (in && t >= 0) *reinterpret_cast<uint4*>(out + t * out_stride + col) = make_uint4(o[0], o[1], o[2], o[3]);
    }
    if (mt + AHEAD < 8) fetch(mt + AHEAD);
  }
}

// ---------------------------------------------------------------------------
// Sums of outer products over an adapter's tokens, g[l][r][c] = sum v[t][r]
// x[t][c]: D [256 columns x 2 NP] += X^T [256 x 64 tokens] V [64 x 2 NP], with X
// as its rows lie in memory (the operand's M runs along them) and V^T's hi and lo
// parts beside each other, added when they leave tensor memory.  A block has
// 256 columns and a group of tiles, which may be of several adapters (a run
// each).  A run that is all of its adapter goes straight to the gradient; one
// that goes on in another group leaves a partial sum (place 0 if it began
// before the group, else 1), which ad_sum adds up in order.
// ---------------------------------------------------------------------------
constexpr int kOuterLoaders = 256;
template <int NP>
struct OuterShared {
  static constexpr int stages = NP <= 16 ? 3 : NP <= 64 ? 4 : 3;
  static constexpr int blocks = NP <= 16 ? 2 : 1;  // resident on an SM
  static constexpr int off_v = 32768;
  static constexpr int stage = off_v + 2 * NP * 128;
  static constexpr int bytes = stages * stage + 1024;
};

// Whether any loader found that a wait ran out: they leave together, at a run's
// start, since they meet at barriers that have no limit.
__device__ __forceinline__ bool any_loader(int fail) {
  int r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.s32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, %2, p;\n\t"
      "selp.s32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(fail), "n"(kOuterLoaders)
      : "memory");
  return r != 0;
}

// One of the two problems of a launch: (v, x, dA) and (u, dy, dB).
template <typename T>
struct OuterSide {
  const float* v;
  const T* x;
  int64_t stride;
  int K, chunks;
  void* g;
  float* part;
};

template <typename T, int NP, typename G>
__global__ void __launch_bounds__(kOuterLoaders + 32, OuterShared<NP>::blocks)
    ad_outer_kernel(const OuterSide<T> one, const OuterSide<T> two, int R, int pitch, AdPlan p, int L) {
  using S = OuterShared<NP>;
  using H = Half16<T>;
  constexpr int NS = S::stages, LAG = NS - 2, VI = NP * 8 / kOuterLoaders > 0 ? NP * 8 / kOuterLoaders : 1;
  constexpr uint32_t kCols = 4 * NP;  // two tiles of 128 columns, hi and lo
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[NS], empty[NS], done, free_, drain;
  __shared__ uint32_t tmem_at;
  __shared__ int failed;
  __shared__ float top[kOuterLoaders / 32];
  pdl_wait();
  pdl_trigger();
  const bool first_side = (int)blockIdx.x < one.chunks;
  const OuterSide<T>& q = first_side ? one : two;
  const int col0 = ((int)blockIdx.x - (first_side ? 0 : one.chunks)) * 256;
  const int n_tiles = p.tile_of[L], per = (n_tiles + gridDim.y - 1) / gridDim.y;
  const int t_lo = blockIdx.y * per, t_hi = min(t_lo + per, n_tiles);
  if (t_lo >= t_hi) return;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = (smem_u32(raw) + 1023) & ~1023u;
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) mbar_init(&full[i], kOuterLoaders), mbar_init(&empty[i], 1);
    mbar_init(&done, 1);
    mbar_init(&free_, kOuterLoaders);
    mbar_init(&drain, 1);
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    proxy_fence();
  }
  if (warp == kOuterLoaders / 32) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_at)), "r"(kCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_at;
  volatile int* fail = &failed;
  int step = 0, run = 0;  // 64-token steps and runs so far: the barriers' phases
  if (warp < kOuterLoaders / 32) {
    const int c = tid & 15, r0 = tid >> 4;
    const int col = col0;
    const uint32_t at = base + r0 * 128 + (((c & 7) ^ (r0 & 7)) << 4) + (c >> 3) * 8192;
    const bool c0 = col + c * 8 < q.K, c1 = col + 128 + c * 8 < q.K;
    for (int t0 = t_lo; !any_loader(*fail) && t0 < t_hi; ++run) {
      const int owner = p.tiles[t0].owner;
      const int first = p.tiles[t0].first, last = min(p.tile_of[owner + 1], t_hi) - 1;
      const int rows = p.tiles[last].first + p.tiles[last].rows - first;  // of the whole run, one behind the other in `order`
      float f = 1.0f, back = 1.0f;
      if (H::scaled) {
        // fp16: the run's greatest value of v
        float m = 0.0f;
        for (int e = tid; e < rows * (pitch / 4); e += kOuterLoaders) {
          const int row = e / (pitch / 4);
          const float4 w = *reinterpret_cast<const float4*>(q.v + (int64_t)p.order[first + row] * pitch + (e - row * (pitch / 4)) * 4);
          m = fmaxf(m, fmaxf(fmaxf(finite_mag(w.x), finite_mag(w.y)), fmaxf(finite_mag(w.z), finite_mag(w.w))));
        }
#pragma unroll
        for (int i = 16; i; i >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, i));
        if (lane == 0) top[warp] = m;
        asm volatile("bar.sync 1, %0;" ::"n"(kOuterLoaders) : "memory");
        for (int i = 0; i < kOuterLoaders / 32; ++i) m = fmaxf(m, top[i]);
        asm volatile("bar.sync 1, %0;" ::"n"(kOuterLoaders) : "memory");
        const int e = scale_exp(m);
        f = exp2i(e), back = exp2i(-e);
      }
      const int n = (rows + 63) / 64;
      float v[VI][8];
      // the next step's part of V: 8 tokens of one rank to a lane
      auto fetch = [&](int i) {
#pragma unroll
        for (int j = 0; j < VI; ++j) {
          const int e = tid + j * kOuterLoaders, r = e % NP, tk = i * 64 + e / NP * 8;
#pragma unroll
          for (int k = 0; k < 8; ++k)
            v[j][k] = e < NP * 8 && r < R && tk + k < rows ? q.v[(int64_t)p.order[first + tk + k] * pitch + r] : 0.0f;
        }
      };
      fetch(0);
      for (int i = 0; i < n + LAG; ++i) {
        if (i < n) {
          const int slot = (step + i) % NS;
          if (step + i >= NS && !mbar_wait(&empty[slot], ((step + i) / NS - 1) & 1)) *fail = 1;
          if (*fail) break;
          const uint32_t to = at + slot * S::stage;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int row = i * 64 + r0 + 16 * j;
            const bool some = row < rows;  // behind the run: zeros in both factors
            const T* from = q.x + (some ? (int64_t)p.order[first + row] * q.stride : 0);
            cp16(to + j * 2048, c0 ? from + col + c * 8 : q.x, some && c0);
            cp16(to + j * 2048 + 16384, c1 ? from + col + 128 + c * 8 : q.x, some && c1);
          }
          const uint32_t vt = base + slot * S::stage + S::off_v;
#pragma unroll
          for (int j = 0; j < VI; ++j) {
            const int e = tid + j * kOuterLoaders, r = e % NP, k8 = e / NP;
            if (e >= NP * 8) continue;
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) split<T>(v[j][2 * k] * f, v[j][2 * k + 1] * f, hi[k], lo[k]);
            const uint32_t a = vt + r * 128 + ((k8 ^ (r & 7)) << 4);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(hi[0]), "r"(hi[1]), "r"(hi[2]), "r"(hi[3]) : "memory");
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a + NP * 128), "r"(lo[0]), "r"(lo[1]), "r"(lo[2]), "r"(lo[3]) : "memory");
          }
          if (i + 1 < n) fetch(i + 1);
        }
        cp_commit();
        if (i >= LAG) {
          cp_wait<LAG>();
          proxy_fence();
          mbar_arrive(&full[(step + i - LAG) % NS]);
        }
      }
      step += n;
      cp_wait<0>();
      if (!mbar_wait(&done, run & 1)) *fail = 1;
      __syncwarp();
      tc_fence_after();
      const int mt = warp >> 2, my = col0 + mt * 128 + (warp & 3) * 32 + lane;
      const uint32_t from = tmem + ((uint32_t)(warp & 3) << 21) + mt * 2 * NP;
      const bool starts = p.tile_of[owner] == t0, ends = p.tile_of[owner + 1] == last + 1;
      float* part = q.part + ((int64_t)blockIdx.y * 2 + (starts ? 1 : 0)) * R * q.K;
#pragma unroll
      for (int r = 0; r < NP; r += 16) {
        uint32_t hi[16], lo[16];
        tmem_ld16(from + r, hi);
        tmem_ld16(from + NP + r, lo);
        tmem_wait_ld16(hi);
        tmem_wait_ld16(lo);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          if (r + k >= R || my >= q.K) continue;
          const float w = (__uint_as_float(hi[k]) + __uint_as_float(lo[k])) * back;
          if (starts && ends) static_cast<G*>(q.g)[((int64_t)owner * R + r + k) * q.K + my] = Ty<G>::from_f(w);
          else part[(int64_t)(r + k) * q.K + my] = w;
        }
      }
      tc_fence_before();
      mbar_arrive(&free_);
      t0 = last + 1;
    }
    cp_wait<0>();
  } else {
    constexpr uint32_t idesc = make_idesc(H::fmt, 2 * NP) | kMajorA;
    for (int t0 = t_lo; t0 < t_hi && !*fail; ++run) {
      const int owner = p.tiles[t0].owner;
      const int last = min(p.tile_of[owner + 1], t_hi) - 1;
      const int rows = p.tiles[last].first + p.tiles[last].rows - p.tiles[t0].first, n = (rows + 63) / 64;
      if (run && !wait_warp(&free_, (run - 1) & 1)) *fail = 1;
      tc_fence_after();
      for (int i = 0; i < n && !*fail; ++i) {
        const int slot = (step + i) % NS;
        if (!wait_warp(&full[slot], ((step + i) / NS) & 1)) {
          *fail = 1;
          break;
        }
        tc_fence_after();
        const uint32_t s = base + slot * S::stage;
        const uint64_t db = sw128_desc(s + S::off_v);
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          const uint64_t da = sw128_mn_desc(s + mt * 16384, 8192);
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_ss(tmem + mt * 2 * NP, da + 128 * k, db + 2 * k, idesc, (i | k) > 0);
        }
        commit(&empty[slot]);
      }
      commit(&done);
      step += n;
      t0 = last + 1;
    }
    if (*fail) {  // the products that were begun end before their memory goes
      commit(&drain);
      wait_warp(&drain, 0);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (tid == 0 && failed) *p.status = LQ_ETIMEOUT;
  if (warp == kOuterLoaders / 32) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols));
}

// What several groups left of an adapter, added in order, and zeros for
// adapters without tokens.  A block to 2048 values of an adapter's [R, K].
template <typename T, typename G>
__global__ void __launch_bounds__(256) ad_sum_kernel(const OuterSide<T> one, const OuterSide<T> two, int R, AdPlan p, int L,
                                                     int groups, int blocks_one) {
  pdl_wait();
  pdl_trigger();
  const bool first_side = (int)blockIdx.x < blocks_one;
  const OuterSide<T>& q = first_side ? one : two;
  const int l = blockIdx.y, a = p.tile_of[l], b = p.tile_of[l + 1];
  const int per = max(1, (p.tile_of[L] + groups - 1) / groups);
  const int ga = a / per, gb = (b - 1) / per;
  if (a < b && ga == gb) return;
  const int64_t size = (int64_t)R * q.K;
  const int64_t i = ((int64_t)((int)blockIdx.x - (first_side ? 0 : blocks_one)) * 256 + threadIdx.x) * 8;
  if (i >= size) return;
  float s[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) s[k] = 0.0f;
  for (int j = ga; a < b && j <= gb; ++j) {
    const float4* w = reinterpret_cast<const float4*>(q.part + ((int64_t)j * 2 + (j == ga ? 1 : 0)) * size + i);
    const float4 x = w[0], y = w[1];
    s[0] += x.x, s[1] += x.y, s[2] += x.z, s[3] += x.w, s[4] += y.x, s[5] += y.y, s[6] += y.z, s[7] += y.w;
  }
  G* g = static_cast<G*>(q.g) + (int64_t)l * size + i;
#pragma unroll
  for (int k = 0; k < 8; ++k) g[k] = Ty<G>::from_f(s[k]);
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
// Once for each kernel and device.
template <auto Kern>
int more_shared(int bytes) {
  static std::atomic<uint64_t> known{0};
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (known.load(std::memory_order_relaxed) & bit) return LQ_OK;
  const cudaError_t e = cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  LQ_REQUIRE(e == cudaSuccess, LQ_ECUDA, "adapters: %d bytes of shared memory: %s", bytes, cudaGetErrorString(e));
  known.fetch_or(bit, std::memory_order_relaxed);
  return LQ_OK;
}

template <typename T, int NP>
int down_np(const AdCall& a, const void* x, int64_t stride, bool is_a, float* u) {
  using S = DownShared<NP>;
  const lq_adapter_bank& b = *a.bank;
  const int K = (int)(is_a ? b.K : b.N), steps = (K + 63) / 64;
  const int64_t tiles = ad_max_tiles(a.n, b.L);
  int split = 1;
  while (split < 8 && tiles * split * 2 <= 2 * num_sms() && split * 4 <= steps) split *= 2;
  constexpr auto kern = ad_down_kernel<T, NP>;
  LQ_TRY(more_shared<kern>(S::bytes));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * split));
  cfg.blockDim = dim3(160);
  cfg.dynamicSmemBytes = S::bytes;
  cfg.stream = a.st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, static_cast<const T*>(x), stride, static_cast<const T*>(is_a ? b.a : b.b),
                                           b.scaling, (int)b.R, ad_pitch(b.R), K, a.plan, (int)b.L, u, split);
  LQ_REQUIRE(e == cudaSuccess, LQ_ECUDA, "ad_down_kernel launch: %s", cudaGetErrorString(e));
  return launched("ad_down_kernel");
}

template <typename T, int NP>
int up_np(const AdCall& a, const float* u, bool is_a, const void* base, int64_t bs, void* out, int64_t os) {
  using S = UpShared<NP>;
  const lq_adapter_bank& b = *a.bank;
  const int N = (int)(is_a ? b.K : b.N), chunks = (N + 255) / 256;
  const int64_t grid = ad_max_tiles(a.n, b.L) * chunks;
  LQ_REQUIRE(grid < (1LL << 31), LQ_ERANGE, "adapters: too many tokens for %d features", N);
  constexpr auto kern = ad_up_kernel<T, NP>;
  LQ_TRY(more_shared<kern>(S::bytes));
  const cudaError_t e = launch_pdl(kern, dim3((unsigned)grid), dim3(256), S::bytes, a.st, u, ad_pitch(b.R),
                                   static_cast<const T*>(is_a ? b.a : b.b), (int)b.R, N, a.plan, (int)b.L,
                                   static_cast<const T*>(base), bs, static_cast<T*>(out), os, chunks);
  LQ_REQUIRE(e == cudaSuccess, LQ_ECUDA, "ad_up_kernel launch: %s", cudaGetErrorString(e));
  return launched("ad_up_kernel");
}

template <typename T, int NP, typename G>
int outer_np(const AdCall& a, const AdOuter& o) {
  using S = OuterShared<NP>;
  const lq_adapter_bank& b = *a.bank;
  const int64_t groups = ad_outer_groups(b, a.n);
  OuterSide<T> one = {}, two = {};
  if (o.da) one = {o.v, static_cast<const T*>(o.x), o.x_stride, (int)b.K, (int)(b.K + 255) / 256, o.da, o.part};
  if (o.db) two = {o.u, static_cast<const T*>(o.dy), o.dy_stride, (int)b.N, (int)(b.N + 255) / 256, o.db, o.part + 2 * groups * b.R * b.K};
  constexpr auto kern = ad_outer_kernel<T, NP, G>;
  LQ_TRY(more_shared<kern>(S::bytes));
  cudaError_t e = launch_pdl(kern, dim3((unsigned)(one.chunks + two.chunks), (unsigned)groups), dim3(kOuterLoaders + 32), S::bytes,
                             a.st, one, two, (int)b.R, ad_pitch(b.R), a.plan, (int)b.L);
  LQ_REQUIRE(e == cudaSuccess, LQ_ECUDA, "ad_outer_kernel launch: %s", cudaGetErrorString(e));
  LQ_TRY(launched("ad_outer_kernel"));
  const int64_t b1 = o.da ? (b.R * b.K + 2047) / 2048 : 0, b2 = o.db ? (b.R * b.N + 2047) / 2048 : 0;
  e = launch_pdl(ad_sum_kernel<T, G>, dim3((unsigned)(b1 + b2), (unsigned)b.L), dim3(256), 0, a.st, one, two, (int)b.R, a.plan,
                 (int)b.L, (int)groups, (int)b1);
  LQ_REQUIRE(e == cudaSuccess, LQ_ECUDA, "ad_sum_kernel launch: %s", cudaGetErrorString(e));
  return launched("ad_sum_kernel");
}

// NP: the rank, rounded up to what the kernels are made for
#define AD_BY_RANK(call)                          \
  const int64_t r = a.bank->R;                    \
  if (r <= 16) return call(16);                   \
  if (r <= 32) return call(32);                   \
  if (r <= 64) return call(64);                   \
  return call(128)

template <typename T>
int down_t(const AdCall& a, const void* x, int64_t stride, bool is_a, float* u) {
#define AD_CALL(np) (down_np<T, np>(a, x, stride, is_a, u))
  AD_BY_RANK(AD_CALL);
#undef AD_CALL
}
template <typename T>
int up_t(const AdCall& a, const float* u, bool is_a, const void* base, int64_t bs, void* out, int64_t os) {
#define AD_CALL(np) (up_np<T, np>(a, u, is_a, base, bs, out, os))
  AD_BY_RANK(AD_CALL);
#undef AD_CALL
}
template <typename T>
int outer_t(const AdCall& a, const AdOuter& o) {
  if (o.grad_dtype == LQ_F32) {
#define AD_CALL(np) (outer_np<T, np, float>(a, o))
    AD_BY_RANK(AD_CALL);
#undef AD_CALL
  }
#define AD_CALL(np) (outer_np<T, np, T>(a, o))
  AD_BY_RANK(AD_CALL);
#undef AD_CALL
}

}  // namespace

int ad_down(const AdCall& a, const void* x, int64_t stride, bool is_a, float* u) {
  return a.bank->dtype == LQ_F16 ? down_t<__half>(a, x, stride, is_a, u) : down_t<__nv_bfloat16>(a, x, stride, is_a, u);
}
int ad_up(const AdCall& a, const float* u, bool is_a, const void* base, int64_t bs, void* out, int64_t os) {
  return a.bank->dtype == LQ_F16 ? up_t<__half>(a, u, is_a, base, bs, out, os) : up_t<__nv_bfloat16>(a, u, is_a, base, bs, out, os);
}
int ad_outer(const AdCall& a, const AdOuter& o) {
  return a.bank->dtype == LQ_F16 ? outer_t<__half>(a, o) : outer_t<__nv_bfloat16>(a, o);
}

}  // namespace lq

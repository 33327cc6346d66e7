// lq_adapters_mm.cu -- the three products of the adapter bank for batches of
// many tokens, over tiles of up to 128 tokens of one adapter, on tcgen05:
//   ad_down    u = s A x          [128 tokens x K] by [K x rank]
//   ad_up      y = base + B^T u   [128 tokens x rank] by [rank x 128 columns]
//   ad_outer   dA = sum v x^T     [256 columns x tokens] by [tokens x rank]
// All three are bound by memory (2 R flops to 2 bytes of x): the point is to
// read x, dy and base once, and to keep the loads coming.  With 16384 tokens,
// 14336 columns and rank 64 in bf16, each launch by itself and nothing in L2 (events,
// to 2 us): ad_down 82 us (470 MB, 5.7 TB/s), ad_up 160 (940 MB read and written,
// 5.9 TB/s), ad_outer of 4096 and 14336 columns with ad_sum 117 (604 MB, 5.2 TB/s); a
// copy reaches 6.4 TB/s.  In fp16 86, 158 and 119.
//
// u and v are fp32 sums.  Where they meet a 16-bit factor they go in as two
// 16-bit values, hi = round(u) and lo = round(u - hi), and two products: u is then
// off by 2^-16 of itself (bf16; 2^-22 in fp16), far below the rounding of the
// output, where one 16-bit value would be off as much as that.  fp16 has too
// small a range for values nobody scaled: a row of u (an adapter's rows of v)
// goes in times a power of two that puts its greatest in [2^12, 2^13), which is
// taken back from the fp32 sum.  A value 2^-15 of the greatest or less has a lo
// below fp16's normal numbers, and is off by half of their step, 2^-25, which is
// 2^-37 of the greatest at most (measured against 64 bits in the tests).
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
};

constexpr float kInf = __builtin_huge_valf();

// Two fp32 values as two 16-bit pairs that add up to them.
template <typename T>
__device__ __forceinline__ void split16(float a, float b, uint32_t& hi, uint32_t& lo) {
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
// A bounded wait of a thread by itself (as wait_warp: no timer is read)
__device__ __forceinline__ bool wait_lane(uint64_t* bar, uint32_t parity) {
  bool ok = false;
#pragma unroll 1
  for (int i = 0; i < (1 << 20) && !ok; ++i) ok = mbar_try_sleep(bar, parity, 10000u);
  return ok;
}
__device__ __forceinline__ void cp_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// Arrives at the barrier once all of the thread's copies so far are there.  The
// proxy fence that the tensor cores' reads need is the reader's.
__device__ __forceinline__ void cp_arrive(uint64_t* b) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(b)) : "memory");
}
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

// Sums of 8 values over the blocks of a cluster, in order; all loads first.
template <int BLOCKS>
__device__ __forceinline__ void cluster_sum(uint32_t addr, float (&v)[8]) {
  float4 a[BLOCKS], z[BLOCKS];
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b) a[b] = ld_cluster_v4(addr, b), z[b] = ld_cluster_v4(addr + 16, b);
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = 0.0f;
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
    v[0] += a[b].x, v[1] += a[b].y, v[2] += a[b].z, v[3] += a[b].w, v[4] += z[b].x, v[5] += z[b].y, v[6] += z[b].z, v[7] += z[b].w;
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
__device__ __forceinline__ void bulk_load_at(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
               "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
// A box of a tensor map; what lies outside of the tensor reads as zeros.
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
// Rows of a call as tensor maps, where the rows lie one behind the other (ok:
// else the rows are copied by threads); always 64 columns, 128 bytes, wide, on a
// multiple of 64, with the 128-byte swizzle that the operands have.
struct RowsMap {
  CUtensorMap map;
  int ok;
};
__device__ __forceinline__ int lane_id() { return threadIdx.x & 31; }
__device__ __forceinline__ int token_of(const AdPlan& p, const AdTile& d, int row) {
  return d.run >= 0 ? d.run + row : p.order[d.first + row];
}

// Whether a wait ran out for any of the `threads` that meet at a named barrier:
// they leave together, since such a barrier has no limit.
template <int THREADS>
__device__ __forceinline__ bool any_failed(int barrier, int fail) {
  int r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.s32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, %3, %2, p;\n\t"
      "selp.s32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(fail), "n"(THREADS), "r"(barrier)
      : "memory");
  return r != 0;
}

// ---------------------------------------------------------------------------
// The low-rank rows of a call (u or v), as ad_down leaves them for each tile:
//   image  the two 16-bit parts as the K-major operand that ad_up copies into
//          shared memory as it is: rows of hi (NP) | lo (NP), in panels of 64 values
//          with the 128-byte swizzle (NP = 16: 32 values, 64-byte swizzle)
//   back   fp16: what each row of the image is to be multiplied with
//   turned fp32 [NP][128 tokens], for ad_outer
//   top    fp16: greatest magnitude in the tile, by parts
// ---------------------------------------------------------------------------
struct Low {
  uint8_t* image;
  float* back;
  float* turned;  // NULL: nobody reads it
  float* top;
};
template <int NP>
__host__ __device__ inline Low low_at(void* p, int64_t tiles, bool turned) {
  Low l;
  l.image = static_cast<uint8_t*>(p);
  l.back = reinterpret_cast<float*>(l.image + tiles * (128 * NP * 4));
  l.top = l.back + tiles * 128;
  l.turned = turned ? l.top + tiles * 8 : nullptr;
  return l;
}
template <int NP>
__device__ __forceinline__ uint32_t image_offset(int row, int k) {  // of value k (a multiple of 8) of a row
  if (NP == 16) return row * 64 + (((k >> 3) ^ ((row >> 1) & 3)) << 4);
  return (k >> 6) * 16384 + row * 128 + ((((k >> 3) & 7) ^ (row & 7)) << 4);
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
__global__ void __launch_bounds__(160, 2) ad_down_kernel(const __grid_constant__ RowsMap xm, const __grid_constant__ CUtensorMap fm,
                                                         const T* __restrict__ x, int64_t stride, const T* __restrict__ f,
                                                         const float* __restrict__ scaling, int R, int K, AdPlan p, int L,
                                                         Low low, int split) {
  using S = DownShared<NP>;
  constexpr int NS = S::stages;
  constexpr uint32_t kCols = NP < 32 ? 32 : NP;
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[NS], empty[NS], done;
  __shared__ uint32_t tmem_at;
  __shared__ int failed, row_top[128];
  using H = Half16<T>;
  if (threadIdx.x == 0 && xm.ok) prefetch_map(&xm.map), prefetch_map(&fm);
  pdl_wait();
  const int tile = blockIdx.x / split, rank = blockIdx.x - tile * split;
  const AdTile d = p.tiles[tile];  // (there is room for every tile of the grid: both loads at once)
  if (tile >= p.tile_of[L]) return;  // the whole cluster
  const float s = scaling[d.owner];
  const int tid = threadIdx.x, warp = tid >> 5;
  const uint32_t base = (smem_u32(raw) + 1023) & ~1023u;
  // a tile whose tokens follow each other comes by TMA (rows of others behind its
  // own do no harm: each row of D is its own), any other by threads
  const bool tma = xm.ok && d.run >= 0;
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) mbar_init(&full[i], tma ? 1 : 128), mbar_init(&empty[i], 1);
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
  // only now: a block of the next kernel that took its tensor memory on this SM
  // first would wait for this one, and this one for it
  pdl_trigger();
  const uint32_t tmem = tmem_at;
  const int all = (K + 63) / 64, s0 = (int)((int64_t)all * rank / split), n = (int)((int64_t)all * (rank + 1) / split) - s0;
  if (warp < 4 && tma) {
    for (int i = 0; i < n && warp == 0; ++i) {
      const int slot = i % NS;
      if (i >= NS && !wait_warp(&empty[slot], (i / NS - 1) & 1)) failed = 1;
      if (*(volatile int*)&failed) break;
      if (tid == 0) {
        const uint32_t to = base + slot * S::stage;
        mbar_expect_tx(&full[slot], S::stage);
        tma_2d(to, &xm.map, (s0 + i) * 64, d.run, &full[slot]);
        tma_3d(to + 16384, &fm, (s0 + i) * 64, 0, d.owner, &full[slot]);
      }
      __syncwarp();
    }
  } else if (warp < 4) {
    const int c = tid & 7, r0 = tid >> 3;
    const T* xr[8];
    const T* fr[NP / 16];
#pragma unroll
    for (int i = 0; i < 8; ++i) xr[i] = r0 + 16 * i < d.rows ? x + (int64_t)token_of(p, d, r0 + 16 * i) * stride : nullptr;
#pragma unroll
    for (int i = 0; i < NP / 16; ++i) fr[i] = r0 + 16 * i < R ? f + ((int64_t)d.owner * R + r0 + 16 * i) * K : nullptr;
    const uint32_t at = base + r0 * 128 + ((c ^ (r0 & 7)) << 4);
    for (int i = 0; i < n; ++i) {
      const int slot = i % NS;
      if (i >= NS && !wait_lane(&empty[slot], (i / NS - 1) & 1)) failed = 1;
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
      cp_arrive(&full[slot]);
    }
    cp_wait_all();
  } else {
    constexpr uint32_t idesc = make_idesc(Half16<T>::fmt, NP);
    for (int i = 0; i < n; ++i) {
      const int slot = i % NS;
      if (!wait_warp(&full[slot], (i / NS) & 1)) {
        failed = 1;
        // what may still be on its way
        for (int j = i + 1; j < min(n, i + NS); ++j) wait_warp(&full[j % NS], (j / NS) & 1);
        break;
      }
      proxy_fence();
      tc_fence_after();
      const uint64_t da = sw128_desc(base + slot * S::stage), db = sw128_desc(base + slot * S::stage + 16384);
#pragma unroll
      for (int k = 0; k < 4; ++k) mma_ss(tmem, da + 2 * k, db + 2 * k, idesc, (i | k) > 0);
      commit(&empty[slot]);
    }
    commit(&done);
  }
  const bool ok = wait_warp(&done, 0);
  if (!ok) failed = 1;
  tc_fence_after();
  if (warp < 4) {
#pragma unroll
    for (int c = 0; c < NP; c += 16) {
      uint32_t v[16];
      tmem_ld16(tmem + ((uint32_t)warp << 21) + c, v);
      tmem_wait_ld16(v);
#pragma unroll
      for (int q = 0; q < 16; q += 4)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(base + (tid * S::pitch + c + q) * 4), "r"(v[q]), "r"(v[q + 1]), "r"(v[q + 2]), "r"(v[q + 3]) : "memory");
    }
    tc_fence_before();
  }
  if (tid < 128) row_top[tid] = 0;
  cluster_arrive();
  cluster_wait();
  // The block's share of the tile's rows, a lane to a row and 8 ranks.  fp16: once
  // for the rows' greatest values, and again.
  const int rows = 128 / split;
#pragma unroll
  for (int pass = H::scaled ? 0 : 1; pass < 2; ++pass) {
    for (int e = tid; warp < 4 && e < rows * (NP / 8); e += 128) {
      const int row = rank * rows + e % rows, r = e / rows * 8;
      if (row >= d.rows) continue;
      float v[8];
      const uint32_t from = base + (row * S::pitch + r) * 4;
      if (split == 8) cluster_sum<8>(from, v);
      else if (split == 4) cluster_sum<4>(from, v);
      else if (split == 2) cluster_sum<2>(from, v);
      else cluster_sum<1>(from, v);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = r + k < R ? v[k] * s : 0.0f;  // behind R: rows of F that nobody loaded
      if (pass == 0) {
        float m = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) m = fmaxf(m, finite_mag(v[k]));
        atomicMax(&row_top[row], __float_as_int(m));  // not negative: ordered as integers, whoever comes first
        continue;
      }
      float f = 1.0f;
      if (H::scaled) {
        const int x2 = scale_exp(__int_as_float(row_top[row]));
        f = exp2i(x2);
        if (r == 0) low.back[(int64_t)tile * 128 + row] = exp2i(-x2);
      }
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) split16<T>(v[2 * k] * f, v[2 * k + 1] * f, hi[k], lo[k]);
      uint8_t* to = low.image + (int64_t)tile * (128 * NP * 4);
      *reinterpret_cast<uint4*>(to + image_offset<NP>(row, r)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      *reinterpret_cast<uint4*>(to + image_offset<NP>(row, NP + r)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      if (low.turned) {
#pragma unroll
        for (int k = 0; k < 8; ++k) low.turned[((int64_t)tile * NP + r + k) * 128 + row] = v[k];
      }
    }
    if (pass == 0) {
      __syncthreads();
      if (low.turned && warp == 0) {
        int m = 0;
        for (int i = lane_id(); i < rows; i += 32) m = max(m, row_top[rank * rows + i]);
#pragma unroll
        for (int i = 16; i; i >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, i));
        if (tid == 0)
          for (int i = rank; i < 8; i += split) low.top[(int64_t)tile * 8 + i] = __int_as_float(m);
      }
    }
  }
  cluster_arrive();
  cluster_wait();  // no block leaves while others read its sums
  __syncthreads();
  if (tid == 0 && failed) *p.status = LQ_ETIMEOUT;
  if (warp == 4) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols));
}

// ---------------------------------------------------------------------------
// out = base + u f, a unit of one tile and 128 columns at a time: D [128 tokens
// x 128] = (hi + lo) [128 x NP] F [NP x 128], F as its rows lie in memory.  A
// block has a stretch of units.  Base and F come by TMA (base whose tokens do not
// follow each other by cp.async, a row of 256 bytes to half a warp); the thread that
// has a row of D adds it to the row of base in shared memory, and half a warp of
// others takes each row out again.  (A lane that loads its own part of base, as
// mma.sync deals D out, touches eight lines of 64 bytes each at a time: L1 was busy
// 4 cycles of 5, and a call of eight prompts of up to 2048 tokens, 4096 to 14336
// features, rank 64, took 289 us where it takes 207 now.  With bulk copies of a row
// each it took 484.)  Two groups of four warps take turns with the units, and two
// teams of two with bringing base.
// ---------------------------------------------------------------------------
// Blocks that go along a tile's rows side by side, so that 1024 bytes of a row are
// asked for at a time: a call of 16384 tokens, rank 64, takes 194.7 us with four and
// 198.1 with one at 14336 columns, 80.3 and 81.3 at 4096, 59.8 and 59.7 at 2048
// (runs lie 0.3 us apart).  A group's share is rounded up to whole rounds of it, which
// narrow rows are fewer than: 48.3 and 45.2 us at 1032 columns, 34.9 and 31.4 at 64.
constexpr int kUpBeside = 2, kUpBesideFrom = 32;  // 1 << 2 blocks; chunks of 128 columns
constexpr int kUpThreads = 704;  // 8 warps add, 8 take out, 4 bring base, 1 F, 1 has the products
template <int NP>
struct UpShared {
  // Two stages of base are being added to, two taken out, the others on their way
  // (with three in all, each with its F, the 16384 tokens above took 226 us where they
  // took 157 with four and F by itself).  An even number: a stage then is always the
  // same team's and the same group's, who see each of its phases (a barrier's parity
  // tells a phase from the next one only, and nothing else keeps the teams abreast).
  static constexpr int stages = NP <= 32 ? 6 : 4;
  static constexpr int stage = 32768;                   // two halves of 64 columns, rows of 128 bytes, swizzled
  static constexpr int fs = NP <= 64 ? 2 : 1;           // stages of F
  static constexpr int f_bytes = NP * 256;
  static constexpr int images = NP == 16 || NP == 64 ? 2 : 1;
  static constexpr int image = 128 * NP * 4;
  static constexpr int off_f = stages * stage, off_image = off_f + fs * f_bytes;
  static constexpr int bytes = off_image + images * image + 1024;
  static_assert(stages % 2 == 0, "a stage to a team");
  static_assert(bytes <= 232448 && f_bytes % 1024 == 0, "shared memory; operands are swizzled in pieces of 1024 bytes");
};
// 16 bytes of a row of a stage
__device__ __forceinline__ uint32_t up_at(int row, int c16) { return (c16 >> 3) * 16384 + row * 128 + (((c16 & 7) ^ (row & 7)) << 4); }

template <typename T, int NP>
__global__ void __launch_bounds__(kUpThreads, 1)
    ad_up_kernel(const __grid_constant__ RowsMap bm, const __grid_constant__ CUtensorMap fm, const Low low, int N, AdPlan p, int L,
                 const T* base, int64_t base_stride, T* out, int64_t out_stride, int chunks, int beside_log2) {
  using S = UpShared<NP>;
  using H = Half16<T>;
  constexpr int NS = S::stages, NF = S::fs, NI = S::images;
  extern __shared__ uint8_t raw[];
  // full: base is there; added: D too; empty: the unit was taken out; f_, i_, d_: the same of F, of images and of D
  __shared__ uint64_t full[NS], added[NS], empty[NS], f_full[NF], f_empty[NF], i_full[NI], i_empty[NI], d_full[2], d_empty[2], drain;
  __shared__ uint32_t tmem_at;
  __shared__ int failed;
  // Started while ad_down (or ad_sum) still runs, which began only when all before
  // it had ended: base, F and the plan are there, and only the low-rank rows are
  // waited for, by the warps that read them.  Nothing is written before them.
  // tokens without an adapter: nothing to do where out is base
  const int beside = 1 << beside_log2, wide = (chunks + beside - 1) & -beside;  // of a tile; what is behind the columns is empty
  const int64_t units = (int64_t)p.tile_of[base == out ? L : L + 1] * (wide >> beside_log2);  // of each block of a group
  const int64_t group = blockIdx.x >> beside_log2, groups = gridDim.x >> beside_log2;
  const int64_t u0 = units * group / groups, u1 = units * (group + 1) / groups;
  const int n = (int)(u1 - u0);
  if (n == 0) return;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t at = (smem_u32(raw) + 1023) & ~1023u;
  if (tid == 0) {
    prefetch_map(&fm);
    if (bm.ok) prefetch_map(&bm.map);
    for (int i = 0; i < NS; ++i) mbar_init(&full[i], 64), mbar_init(&added[i], 128), mbar_init(&empty[i], 128);
    for (int i = 0; i < NF; ++i) mbar_init(&f_full[i], 1), mbar_init(&f_empty[i], 1);
    for (int i = 0; i < NI; ++i) mbar_init(&i_full[i], 1), mbar_init(&i_empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&d_full[i], 1), mbar_init(&d_empty[i], 128);
    mbar_init(&drain, 1);
    failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    proxy_fence();
  }
  if (warp == 21) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_at)), "r"(256u));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();
  const uint32_t tmem = tmem_at;
  volatile int* fail = &failed;
  int tile = (int)(u0 * beside / wide), chunk = (int)(u0 * beside - (int64_t)tile * wide + (blockIdx.x & (beside - 1)));
  if (warp < 8) {
    // ---- add: a thread to a row ----
    pdl_wait();
    const int e = warp >> 2, row = (warp & 3) * 32 + lane;
    float back = 1.0f;
    bool some = false;
    int known = -1;
    for (int i = 0; i < n; ++i, chunk += beside) {
      if (chunk >= wide) chunk -= wide, ++tile;
      if ((i & 1) != e) continue;
      const int slot = i % NS;
      if (tile != known) {
        const AdTile d = p.tiles[tile];
        some = d.owner >= 0;
        if (H::scaled) back = some && row < d.rows ? low.back[(int64_t)tile * 128 + row] : 1.0f;
        known = tile;
      }
      if (!wait_lane(&full[slot], (i / NS) & 1) || !wait_lane(&d_full[e], (i >> 1) & 1)) *fail = 1;
      __syncwarp();
      if (*fail) break;
      tc_fence_after();
      const uint32_t stage = at + slot * S::stage, from = tmem + ((uint32_t)(warp & 3) << 21) + e * 128;
      if (some) {
        // the next 32 columns leave tensor memory while these are added
        uint32_t v[2][32];
        tmem_ld32(from, v[0]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t* w = v[c & 1];
          uint4 y[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) y[q] = base ? lds_v4(stage + up_at(row, 4 * c + q)) : make_uint4(0u, 0u, 0u, 0u);
          tmem_wait_ld32(w);
          if (c < 3) tmem_ld32(from + c * 32 + 32, v[(c + 1) & 1]);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t o[4] = {y[q].x, y[q].y, y[q].z, y[q].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 b = H::unpack(o[k]);
              const float v0 = __uint_as_float(w[8 * q + 2 * k]), v1 = __uint_as_float(w[8 * q + 2 * k + 1]);
              o[k] = H::scaled ? H::pack(fmaf(v0, back, b.x), fmaf(v1, back, b.y)) : H::pack(b.x + v0, b.y + v1);
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + up_at(row, 4 * c + q)), "r"(o[0]), "r"(o[1]), "r"(o[2]), "r"(o[3]) : "memory");
          }
        }
      }
      tc_fence_before();
      mbar_arrive(&d_empty[e]);
      mbar_arrive(&added[slot]);
    }
  } else if (warp < 16) {
    // ---- take out: half a warp to a row, a team every other unit ----
    pdl_wait();
    const int team = (warp - 8) >> 2;
    const int c16 = lane & 15, row0 = (warp & 3) * 2 + (lane >> 4);  // its 16 bytes, and the first of its rows, 8 apart
    AdTile d = {};
    int tok = -1;  // lane k: of row (warp & 3) * 2 + k / 16 + 8 (k % 16)
    int known = -1;
    for (int i = 0; i < n; ++i, chunk += beside) {
      if (chunk >= wide) chunk -= wide, ++tile;
      if ((i & 1) != team) continue;
      const int slot = i % NS;
      if (tile != known) {
        d = p.tiles[tile];
        const int r = row0 + 8 * c16;
        tok = r < d.rows ? token_of(p, d, r) : -1;
        known = tile;
      }
      if (!wait_lane(&added[slot], (i / NS) & 1)) *fail = 1;
      __syncwarp();
      if (*fail) break;
      const uint32_t from = at + slot * S::stage + up_at(row0, c16);  // 8 rows on: the same place of the swizzle
      T* to = out + chunk * 128 + c16 * 8;
      const bool in = chunk * 128 + c16 * 8 < N, some = d.owner >= 0 || base;
#pragma unroll
      for (int j0 = 0; j0 < 16; j0 += 8) {
        uint4 y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = lds_v4(from + (j0 + j) * 1024);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int t = __shfl_sync(0xffffffffu, tok, (lane & 16) + j0 + j);
          if (in && t >= 0) *reinterpret_cast<uint4*>(to + (int64_t)t * out_stride) = some ? y[j] : make_uint4(0u, 0u, 0u, 0u);
        }
      }
      mbar_arrive(&empty[slot]);
    }
  } else if (warp < 20) {
    // ---- base: a team brings every other unit ----
    const int team = (warp - 16) >> 1, w2 = warp & 1, c16 = lane & 15, row0 = w2 * 2 + (lane >> 4);
    AdTile d = {};
    int tok[2] = {-1, -1};  // lane k: of rows row0(k) + 4 (k % 16), and 64 later
    int known = -1, sent = 0;
    for (int i = 0; i < n; ++i, chunk += beside) {
      if (chunk >= wide) chunk -= wide, ++tile;
      if ((i & 1) != team) continue;
      const int slot = i % NS;
      if (tile != known) {
        d = p.tiles[tile];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int r = row0 + 4 * c16 + 64 * k;
          tok[k] = r < d.rows ? token_of(p, d, r) : -1;
        }
        known = tile;
      }
      if (i >= NS && !wait_lane(&empty[slot], (i / NS - 1) & 1)) *fail = 1;
      __syncwarp();
      if (*fail) break;
      sent = i + 1;
      const uint32_t stage = at + slot * S::stage;
      const int col = chunk * 128 + c16 * 8;
      const bool in = col < N;
      if (base && bm.ok && d.run >= 0) {
        // rows of other tiles behind the tile's own are not taken out
        if (w2 == 0 && lane == 0) {
          proxy_fence();  // the sums that were written here come before the box
          mbar_expect_tx(&full[slot], S::stage);
          tma_2d(stage, &bm.map, chunk * 128, d.run, &full[slot]);
          tma_2d(stage + 16384, &bm.map, chunk * 128 + 64, d.run, &full[slot]);
        } else {
          mbar_arrive(&full[slot]);
        }
        __syncwarp();
        continue;
      }
      if (base) {
        const T* from = base + (in ? col : 0);
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const int t = __shfl_sync(0xffffffffu, tok[j >> 4], (lane & 16) + (j & 15));
          if (in && t >= 0) cp16(stage + up_at(row0 + 4 * j, c16), from + (int64_t)t * base_stride, true);
        }
      }
      cp_arrive(&full[slot]);
    }
    cp_wait_all();
    if (*fail)  // boxes that were sent for arrive before their memory goes
      for (int i = max(sent - NS, 0); i < sent; ++i)
        if ((i & 1) == team) wait_lane(&full[i % NS], (i / NS) & 1);
  } else if (warp == 20) {
    // ---- F: 128 columns of the adapter's rows, zeros behind the rank (they meet zeros of the image) ----
    int known = -1, owner = -1, sent = 0;
    for (int i = 0; i < n; ++i, chunk += beside) {
      if (chunk >= wide) chunk -= wide, ++tile;
      if (tile != known) owner = p.tiles[tile].owner, known = tile;
      if (owner < 0) continue;
      const int fs = sent % NF;
      if (sent >= NF && !wait_warp(&f_empty[fs], (sent / NF - 1) & 1)) *fail = 1;
      if (*fail) break;
      if (lane == 0) {
        const uint32_t to = at + S::off_f + fs * S::f_bytes;
        mbar_expect_tx(&f_full[fs], S::f_bytes);
        tma_3d(to, &fm, chunk * 128, 0, owner, &f_full[fs]);
        tma_3d(to + NP * 128, &fm, chunk * 128 + 64, 0, owner, &f_full[fs]);
      }
      __syncwarp();
      ++sent;
    }
    if (*fail)  // what was sent for arrives before its memory goes
      for (int k = max(sent - NF, 0); k < sent; ++k) wait_warp(&f_full[k % NF], (k / NF) & 1);
  } else {
    // ---- images and products ----
    pdl_wait();
    constexpr uint32_t idesc = make_idesc(H::fmt, 128) | kMajorB;
    // the tile's image, and the next one where there is room for two
    int known = -1, images = 0, sent = 0, b = 0, used = 0;
    int next = tile;  // the next tile whose image was not asked for
    const int last = (int)((u1 - 1) * beside / wide);
    bool some = false;
    for (int i = 0; i < n && !*fail; ++i, chunk += beside) {
      if (chunk >= wide) chunk -= wide, ++tile;
      const int fs = used % NF, e = i & 1;
      if (tile != known) {
        some = p.tiles[tile].owner >= 0;
        known = tile;
        while (next <= last && (next <= tile || (NI > 1 && next == tile + 1))) {
          if (p.tiles[next].owner >= 0) {
            const int k = sent % NI;
            if (sent >= NI && !wait_warp(&i_empty[k], (sent / NI - 1) & 1)) *fail = 1;
            if (*fail) break;
            if (lane == 0) {
              mbar_expect_tx(&i_full[k], S::image);
              bulk_load_at(at + S::off_image + k * S::image, low.image + (int64_t)next * S::image, S::image, &i_full[k]);
            }
            __syncwarp();
            ++sent;
          }
          ++next;
        }
        if (*fail) break;
        if (some) {
          b = images % NI;
          if (!wait_warp(&i_full[b], (images / NI) & 1)) *fail = 1;
          ++images;
        }
      }
      if ((some && !wait_warp(&f_full[fs], (used / NF) & 1)) || (i >= 2 && !wait_warp(&d_empty[e], ((i >> 1) - 1) & 1))) *fail = 1;
      if (*fail) break;
      proxy_fence();
      tc_fence_after();
      if (some) {
        const uint32_t im = at + S::off_image + b * S::image;
        const uint64_t df = sw128_mn_desc(at + S::off_f + fs * S::f_bytes, NP * 128);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int k = 0; k < NP / 16; ++k) {
            const int v = h * NP + 16 * k;  // value of the image's row
            const uint64_t da = NP == 16 ? sw64_desc(im + v * 2) : sw128_desc(im + (v >> 6) * 16384 + (v & 63) * 2);
            mma_ss(tmem + e * 128, da, df + 128 * k, idesc, (h | k) > 0);
          }
        commit(&d_full[e]);
        commit(&f_empty[fs]);
        ++used;
        if (i + 1 == n || chunk + beside >= wide) commit(&i_empty[b]);
      } else if (lane == 0) {
        mbar_arrive(&d_full[e]);
      }
      __syncwarp();
    }
    if (*fail) {  // what was begun, or sent for, ends before its memory goes
      commit(&drain);
      wait_warp(&drain, 0);
      for (int k = max(images - 1, 0); k < sent; ++k) wait_warp(&i_full[k % NI], (k / NI) & 1);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (tid == 0 && failed) *p.status = LQ_ETIMEOUT;
  if (warp == 21) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256u));
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
constexpr int kOuterX = 128, kOuterV = 256, kOuterLoaders = kOuterX + kOuterV;
template <int NP>
struct OuterShared {
  static constexpr int stages = NP <= 16 ? 6 : NP <= 32 ? 5 : NP <= 64 ? 4 : 3;
  static constexpr int off_v = 32768;
  static constexpr int stage = off_v + 2 * NP * 128;
  static constexpr int bytes = stages * stage + 1024;
};

// One of the two problems of a launch: (v, x, dA) and (u, dy, dB).
template <typename T>
struct OuterSide {
  Low v;
  const T* x;
  int64_t stride;
  int K, chunks;
  void* g;
  float* part;
};

template <typename T, int NP, typename G>
__global__ void __launch_bounds__(kOuterLoaders + 32, 1)
    ad_outer_kernel(const __grid_constant__ RowsMap one_m, const __grid_constant__ RowsMap two_m, const OuterSide<T> one,
                    const OuterSide<T> two, int R, AdPlan p, int L, int early) {
  using S = OuterShared<NP>;
  using H = Half16<T>;
  constexpr int NS = S::stages, VI = NP <= 32 ? 1 : NP / 32;  // 8 tokens of a rank, of a lane that brings V
  constexpr uint32_t kCols = 4 * NP;  // two tiles of 128 columns, hi and lo
  extern __shared__ uint8_t raw[];
  __shared__ uint64_t full[NS], empty[NS], done, free_, drain;
  __shared__ uint32_t tmem_at;
  __shared__ int failed;
  // behind ad_down (early), as ad_up: x, dy, u and the plan are there, v is waited
  // for by those who read it.  Behind any other kernel dy may be that one's.
  if (!early) pdl_wait();
  const bool first_side = (int)blockIdx.x < one.chunks;
  const OuterSide<T>& q = first_side ? one : two;
  const RowsMap& xm = first_side ? one_m : two_m;
  const int col0 = ((int)blockIdx.x - (first_side ? 0 : one.chunks)) * 256;
  const int n_tiles = p.tile_of[L], per = (n_tiles + gridDim.y - 1) / gridDim.y;
  const int t_lo = blockIdx.y * per, t_hi = min(t_lo + per, n_tiles);
  if (t_lo >= t_hi) return;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = (smem_u32(raw) + 1023) & ~1023u;
  if (tid == 0) {
    if (xm.ok) prefetch_map(&xm.map);
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
  pdl_trigger();
  const uint32_t tmem = tmem_at;
  volatile int* fail = &failed;
  int step = 0, run = 0;  // 64-token steps and runs so far: the barriers' phases
  if (warp < kOuterLoaders / 32) {
    // warps 0 .. 3 bring X, by TMA or a row of 512 bytes at a time; the others V
    const bool brings_x = warp < 4;
    if (H::scaled || !brings_x) pdl_wait();
    const uint32_t at = base + (lane >> 3) * 8192;
    const bool in = col0 + lane * 8 < q.K;
    for (int t0 = t_lo; !any_failed<kOuterLoaders>(1, *fail) && t0 < t_hi; ++run) {
      const int owner = p.tiles[t0].owner;
      const int first = p.tiles[t0].first, last = min(p.tile_of[owner + 1], t_hi) - 1;
      const int rows = p.tiles[last].first + p.tiles[last].rows - first;  // of the whole run, one behind the other in `order`
      float f = 1.0f, back = 1.0f;
      if (H::scaled) {  // fp16: by the run's greatest value of v
        float m = 0.0f;
        for (int e = lane; e < (last - t0 + 1) * 8; e += 32) m = fmaxf(m, q.v.top[(int64_t)t0 * 8 + e]);
#pragma unroll
        for (int i = 16; i; i >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, i));
        const int e = scale_exp(m);
        f = exp2i(e), back = exp2i(-e);
      }
      const int n = (rows + 63) / 64;
      if (brings_x) {
        // lane k has the token of the warp's k-th row of the next step
        auto token = [&](int i) {
          const int row = i * 64 + warp + 4 * lane;
          return lane < 16 && row < rows ? p.order[first + row] : -1;
        };
        // the token of a step's first row if all its 64 rows are there and follow each other: it comes by TMA
        auto whole = [&](int i) {
          const AdTile d = p.tiles[t0 + (i >> 1)];
          const int r = (i & 1) * 64;
          return xm.ok && d.run >= 0 && r + 64 <= d.rows ? d.run + r : -1;
        };
        int next = token(0), next_box = whole(0);
        for (int i = 0; i < n; ++i) {
          const int slot = (step + i) % NS, now = next, box = next_box;
          if (i + 1 < n) next = token(i + 1), next_box = whole(i + 1);
          if (step + i >= NS && !wait_lane(&empty[slot], ((step + i) / NS - 1) & 1)) *fail = 1;
          __syncwarp();
          if (*fail) break;
          if (box >= 0) {
            if (tid == 0) {
              proxy_fence();  // rows that threads copied here come before the box
              mbar_expect_tx(&full[slot], 32768);
#pragma unroll
              for (int j = 0; j < 4; ++j) tma_2d(base + slot * S::stage + j * 8192, &xm.map, col0 + j * 64, box, &full[slot]);
            } else {
              mbar_arrive(&full[slot]);
            }
            __syncwarp();
            continue;
          }
          const uint32_t to = at + slot * S::stage;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int row = warp + 4 * j, tok = __shfl_sync(0xffffffffu, now, j);
            const bool some = in && tok >= 0;  // behind the run: zeros in both factors
            cp16(to + row * 128 + (((lane & 7) ^ (row & 7)) << 4), some ? q.x + (int64_t)tok * q.stride + col0 + lane * 8 : q.x, some);
          }
          cp_arrive(&full[slot]);
        }
      } else {
        const int id = tid - kOuterX, k8 = id & 7, r0 = id >> 3;
        float v[2][VI][8];
        // whole pieces, the ones behind the run too (a tile's rows are all there, if
        // nobody wrote them): loads under a condition, whose value is looked at before
        // the next one, cost a trip to L2 each (a training step of 16384 tokens, rank 64,
        // 741 us, without them 573).  Two steps are on their way: with one, and half of
        // the warps, the trip was the step's time (the sums 140 us, with two 105)
        auto fetch = [&](int i, float (&w)[VI][8]) {
          const float* from = q.v.turned + (int64_t)(t0 + (i >> 1)) * NP * 128 + (i & 1) * 64 + k8 * 8;
#pragma unroll
          for (int j = 0; j < VI; ++j) {
            if (r0 + 32 * j >= NP) continue;  // (NP = 16: half of the warps)
#pragma unroll
            for (int k = 0; k < 8; k += 4) {
              const float4 a = *reinterpret_cast<const float4*>(from + (r0 + 32 * j) * 128 + k);
              w[j][k] = a.x, w[j][k + 1] = a.y, w[j][k + 2] = a.z, w[j][k + 3] = a.w;
            }
          }
        };
        auto put = [&](int i, float (&w)[VI][8]) {
          const int slot = (step + i) % NS;
          if (step + i >= NS && !wait_lane(&empty[slot], ((step + i) / NS - 1) & 1)) *fail = 1;
          if (*fail) return false;
          const uint32_t vt = base + slot * S::stage + S::off_v;
          const int left = rows - i * 64 - k8 * 8;  // tokens of the run from here on
          if (left < 8) {
#pragma unroll
            for (int j = 0; j < VI; ++j)
#pragma unroll
              for (int k = 0; k < 8; ++k) w[j][k] = k < left ? w[j][k] : 0.0f;
          }
#pragma unroll
          for (int j = 0; j < VI; ++j) {
            const int r = r0 + 32 * j;
            if (r >= NP) continue;
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) split16<T>(w[j][2 * k] * f, w[j][2 * k + 1] * f, hi[k], lo[k]);
            const uint32_t a = vt + r * 128 + ((k8 ^ (r & 7)) << 4);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(hi[0]), "r"(hi[1]), "r"(hi[2]), "r"(hi[3]) : "memory");
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a + NP * 128), "r"(lo[0]), "r"(lo[1]), "r"(lo[2]), "r"(lo[3]) : "memory");
          }
          proxy_fence();
          mbar_arrive(&full[slot]);
          if (i + 2 < n) fetch(i + 2, w);
          return true;
        };
        fetch(0, v[0]);
        if (n > 1) fetch(1, v[1]);
        for (int i = 0; i < n; i += 2) {
          if (!put(i, v[0])) break;
          if (i + 1 < n && !put(i + 1, v[1])) break;
        }
      }
      step += n;
      cp_wait_all();
      if (!wait_lane(&done, run & 1)) *fail = 1;
      __syncwarp();
      tc_fence_after();
      if (warp >= 8) {  // eight warps have the 256 columns
        mbar_arrive(&free_);
        t0 = last + 1;
        continue;
      }
      const int mt = warp >> 2, my = col0 + mt * 128 + (warp & 3) * 32 + lane;
      const uint32_t from = tmem + ((uint32_t)(warp & 3) << 21) + mt * 2 * NP;
      const bool starts = p.tile_of[owner] == t0, ends = p.tile_of[owner + 1] == last + 1;
      float* part = q.part + ((int64_t)blockIdx.y * 2 + (starts ? 1 : 0)) * R * q.K;
      bool nan = false;
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
          nan |= w != w;
          if (starts && ends) static_cast<G*>(q.g)[((int64_t)owner * R + r + k) * q.K + my] = Ty<G>::from_f(w);
          else part[(int64_t)(r + k) * q.K + my] = w;
        }
      }
      if (nan) *p.nan = 1;
      tc_fence_before();
      mbar_arrive(&free_);
      t0 = last + 1;
    }
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
        proxy_fence();
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
    if (*fail) {  // the products that were begun, and boxes on their way, end before their memory goes
      commit(&drain);
      wait_warp(&drain, 0);
      for (int i = 0; i < NS; ++i) wait_warp(&full[i], 0), wait_warp(&full[i], 1);
    }
  }
  pdl_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (tid == 0 && failed) *p.status = LQ_ETIMEOUT;
  if (warp == kOuterLoaders / 32) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols));
}

// Sums of one rank and 8 columns over an adapter's tokens in fp32, or until all are no numbers.
template <typename T>
__device__ __forceinline__ void sum_again(const OuterSide<T>& q, const AdPlan& p, int l, int np, int r, int c, float (&s)[8]) {
  constexpr int AHEAD = 8;  // tokens on their way
#pragma unroll
  for (int k = 0; k < 8; ++k) s[k] = 0.0f;
  const int first = p.start[l], rows = p.start[l + 1] - first;
  const float* v = q.v.turned + ((int64_t)p.tile_of[l] * np + r) * 128;
  for (int i0 = 0; i0 < rows; i0 += AHEAD) {
    const float* u = v + (int64_t)(i0 >> 7) * np * 128 + (i0 & 127);
    Vec16<T> x[AHEAD];
    float w[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      const bool some = i0 + j < rows;
      x[j].u = make_uint4(0u, 0u, 0u, 0u);
      if (some) x[j].u = *reinterpret_cast<const uint4*>(q.x + p.order[first + i0 + j] * q.stride + c);
      w[j] = some ? u[j] : 0.0f;
    }
    bool some = false;  // a sum that may still be one
#pragma unroll
    for (int k = 0; k < 8; ++k) {
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) s[k] = fmaf(w[j], Ty<T>::to_f(x[j].v[k]), s[k]);
      some |= s[k] == s[k];
    }
    if (!some) return;
  }
}

// What several groups left of an adapter, added in order, and zeros for
// adapters without tokens.  A block to 2048 values of an adapter's [R, K].
//
// Where x is infinite, v's parts give no number although v itself may: 0 times it
// where lo is 0, infinities of both signs where lo's sign is not hi's.  Sums that are
// no numbers are taken again, then, from v as it is; a call without any reads one word.
// A backward pass of 16384 tokens, 4096 to 14336 features, rank 64, of 0.32 ms takes 1.6
// with one infinite value in x and 2.1 with a token of dy infinite (by the number of
// loads on their way: with a token at a time 3.8 and 4.0).
template <typename T, typename G>
__global__ void __launch_bounds__(256) ad_sum_kernel(const OuterSide<T> one, const OuterSide<T> two, int R, AdPlan p, int L,
                                                     int groups, int blocks_one, int np) {
  pdl_wait();
  pdl_trigger();
  const bool first_side = (int)blockIdx.x < blocks_one, odd = *p.nan != 0;
  const OuterSide<T>& q = first_side ? one : two;
  const int l = blockIdx.y, a = p.tile_of[l], b = p.tile_of[l + 1];
  const int per = max(1, (p.tile_of[L] + groups - 1) / groups);
  const int ga = a / per, gb = (b - 1) / per;
  const bool there = a < b && ga == gb;  // in the gradient
  if (there && !odd) return;
  const int64_t size = (int64_t)R * q.K;
  const int64_t i = ((int64_t)((int)blockIdx.x - (first_side ? 0 : blocks_one)) * 256 + threadIdx.x) * 8;
  if (i >= size) return;
  G* g = static_cast<G*>(q.g) + (int64_t)l * size + i;
  float s[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) s[k] = there ? Ty<G>::to_f(g[k]) : 0.0f;
  for (int j = ga; !there && a < b && j <= gb; ++j) {
    const float4* w = reinterpret_cast<const float4*>(q.part + ((int64_t)j * 2 + (j == ga ? 1 : 0)) * size + i);
    const float4 x = w[0], y = w[1];
    s[0] += x.x, s[1] += x.y, s[2] += x.z, s[3] += x.w, s[4] += y.x, s[5] += y.y, s[6] += y.z, s[7] += y.w;
  }
  if (odd && a < b) {
    bool nan = false;
#pragma unroll
    for (int k = 0; k < 8; ++k) nan |= s[k] != s[k];
    if (nan) {
      float w[8];
      const int r = (int)(i / q.K);
      sum_again(q, p, l, np, r, (int)(i - (int64_t)r * q.K), w);
#pragma unroll
      for (int k = 0; k < 8; ++k) s[k] = s[k] != s[k] ? w[k] : s[k];
    } else if (there) {
      return;
    }
  }
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

// The encoder needs a current context, which a thread that made no call of the
// runtime yet (autograd's, at its first backward pass) does not have.
template <typename... Args>
CUresult encode(Args... args) {
  const EncodeTiledFn enc = encode_fn();
  if (!enc) return CUDA_ERROR_NOT_FOUND;
  CUresult r = enc(args...);
  if (r == CUDA_ERROR_INVALID_CONTEXT) {
    int dev = 0;
    if (cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess) r = enc(args...);
  }
  return r;
}

// [rows, width] of 16-bit values as boxes of 64 columns and `box` rows
template <typename T>
int map_rows(RowsMap* m, const void* p, int64_t rows, int64_t width, int64_t stride, int box) {
  m->ok = 0;
  if (!p || (rows > 1 && stride < width)) return LQ_OK;  // rows that share memory: not a tensor map's
  const cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)(rows > 1 ? stride : width) * 2};
  const cuuint32_t boxes[2] = {64, (cuuint32_t)box}, ones[2] = {1, 1};
  const CUresult r = encode(&m->map, Half16<T>::fmt ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                         const_cast<void*>(p), dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  LQ_REQUIRE(r == CUDA_SUCCESS, LQ_ECUDA, "adapters: a tensor map of %lld rows of %lld values failed (%d)", (long long)rows,
             (long long)width, (int)r);
  m->ok = 1;
  return LQ_OK;
}
// A bank's factor [L, R, width], boxes of one adapter's ranks
template <typename T, int NP>
int map_factor(CUtensorMap* m, const lq_adapter_bank& b, bool is_a) {
  const int64_t width = is_a ? b.K : b.N;
  const cuuint64_t dims[3] = {(cuuint64_t)width, (cuuint64_t)b.R, (cuuint64_t)b.L};
  const cuuint64_t strides[2] = {(cuuint64_t)width * 2, (cuuint64_t)(b.R * width) * 2};
  const cuuint32_t boxes[3] = {64, NP, 1}, ones[3] = {1, 1, 1};
  const CUresult r = encode(m, Half16<T>::fmt ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                         const_cast<void*>(is_a ? b.a : b.b), dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  LQ_REQUIRE(r == CUDA_SUCCESS, LQ_ECUDA, "adapters: a tensor map of the bank failed (%d)", (int)r);
  return LQ_OK;
}

template <typename T, int NP>
int down_np(const AdCall& a, const void* x, int64_t stride, bool is_a, void* low, bool turned) {
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
  RowsMap xm;
  CUtensorMap fm;
  LQ_TRY(map_rows<T>(&xm, x, a.n, K, stride, 128));
  LQ_TRY((map_factor<T, NP>(&fm, b, is_a)));
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, xm, fm, static_cast<const T*>(x), stride, static_cast<const T*>(is_a ? b.a : b.b),
                                           b.scaling, (int)b.R, K, a.plan, (int)b.L, low_at<NP>(low, tiles, turned), split);
  LQ_REQUIRE(e == cudaSuccess, LQ_ECUDA, "ad_down_kernel launch: %s", cudaGetErrorString(e));
  return launched("ad_down_kernel");
}

template <typename T, int NP>
int up_np(const AdCall& a, void* low, bool is_a, const void* base, int64_t bs, void* out, int64_t os) {
  using S = UpShared<NP>;
  const lq_adapter_bank& b = *a.bank;
  const int N = (int)(is_a ? b.K : b.N), chunks = (N + 127) / 128;
  const int beside_log2 = chunks < kUpBesideFrom ? 0 : kUpBeside, beside = 1 << beside_log2;
  const int64_t tiles = ad_max_tiles(a.n, b.L), units = tiles * ((chunks + beside - 1) / beside);
  const int64_t groups = units < num_sms() / beside ? units : num_sms() / beside;
  constexpr auto kern = ad_up_kernel<T, NP>;
  LQ_TRY(more_shared<kern>(S::bytes));
  RowsMap bm;
  CUtensorMap fm;
  LQ_TRY(map_rows<T>(&bm, base, a.n, N, bs, 128));
  LQ_TRY((map_factor<T, NP>(&fm, b, is_a)));
  const cudaError_t e = launch_pdl(kern, dim3((unsigned)(groups * beside)), dim3(kUpThreads), S::bytes, a.st, bm, fm,
                                   low_at<NP>(low, tiles, false), N, a.plan, (int)b.L, static_cast<const T*>(base), bs, static_cast<T*>(out), os, chunks, beside_log2);
  LQ_REQUIRE(e == cudaSuccess, LQ_ECUDA, "ad_up_kernel launch: %s", cudaGetErrorString(e));
  return launched("ad_up_kernel");
}

template <typename T, int NP, typename G>
int outer_np(const AdCall& a, const AdOuter& o) {
  using S = OuterShared<NP>;
  const lq_adapter_bank& b = *a.bank;
  const int64_t groups = ad_outer_groups(b, a.n), tiles = ad_max_tiles(a.n, b.L);
  OuterSide<T> one = {}, two = {};
  if (o.da) one = {low_at<NP>(o.v, tiles, true), static_cast<const T*>(o.x), o.x_stride, (int)b.K, (int)(b.K + 255) / 256, o.da, o.part};
  if (o.db) two = {low_at<NP>(o.u, tiles, true), static_cast<const T*>(o.dy), o.dy_stride, (int)b.N, (int)(b.N + 255) / 256, o.db,
                   o.part + 2 * groups * b.R * b.K};
  constexpr auto kern = ad_outer_kernel<T, NP, G>;
  LQ_TRY(more_shared<kern>(S::bytes));
  RowsMap one_m, two_m;
  LQ_TRY(map_rows<T>(&one_m, one.x, a.n, b.K, one.stride, 64));
  LQ_TRY(map_rows<T>(&two_m, two.x, a.n, b.N, two.stride, 64));
  cudaError_t e = launch_pdl(kern, dim3((unsigned)(one.chunks + two.chunks), (unsigned)groups), dim3(kOuterLoaders + 32), S::bytes,
                             a.st, one_m, two_m, one, two, (int)b.R, a.plan, (int)b.L, (int)o.behind_down);
  LQ_REQUIRE(e == cudaSuccess, LQ_ECUDA, "ad_outer_kernel launch: %s", cudaGetErrorString(e));
  LQ_TRY(launched("ad_outer_kernel"));
  const int64_t b1 = o.da ? (b.R * b.K + 2047) / 2048 : 0, b2 = o.db ? (b.R * b.N + 2047) / 2048 : 0;
  e = launch_pdl(ad_sum_kernel<T, G>, dim3((unsigned)(b1 + b2), (unsigned)b.L), dim3(256), 0, a.st, one, two, (int)b.R, a.plan,
                 (int)b.L, (int)groups, (int)b1, NP);
  LQ_REQUIRE(e == cudaSuccess, LQ_ECUDA, "ad_sum_kernel launch: %s", cudaGetErrorString(e));
  return launched("ad_sum_kernel");
}

// NP: the rank, rounded up to what the kernels are made for
#define AD_BY_RANK(rank, call)                  \
  (ad_padded(rank) == 16   ? call(16)           \
   : ad_padded(rank) == 32 ? call(32)           \
   : ad_padded(rank) == 64 ? call(64)           \
                           : call(128))

template <typename T>
int down_t(const AdCall& a, const void* x, int64_t stride, bool is_a, void* low, bool turned) {
#define AD_CALL(np) (down_np<T, np>(a, x, stride, is_a, low, turned))
  return AD_BY_RANK(a.bank->R, AD_CALL);
#undef AD_CALL
}
template <typename T>
int up_t(const AdCall& a, void* low, bool is_a, const void* base, int64_t bs, void* out, int64_t os) {
#define AD_CALL(np) (up_np<T, np>(a, low, is_a, base, bs, out, os))
  return AD_BY_RANK(a.bank->R, AD_CALL);
#undef AD_CALL
}
template <typename T, typename G>
int outer_t(const AdCall& a, const AdOuter& o) {
#define AD_CALL(np) (outer_np<T, np, G>(a, o))
  return AD_BY_RANK(a.bank->R, AD_CALL);
#undef AD_CALL
}

}  // namespace

size_t ad_low_bytes(const lq_adapter_bank& b, int64_t n, bool turned) {
  const int np = ad_padded(b.R);
  return (size_t)ad_max_tiles(n, b.L) * (128 * np * 4 + 128 * 4 + 8 * 4 + (turned ? 128 * np * 4 : 0));
}
int ad_down(const AdCall& a, const void* x, int64_t stride, bool is_a, void* low, bool turned) {
  return a.bank->dtype == LQ_F16 ? down_t<__half>(a, x, stride, is_a, low, turned)
                                 : down_t<__nv_bfloat16>(a, x, stride, is_a, low, turned);
}
int ad_up(const AdCall& a, void* low, bool is_a, const void* base, int64_t bs, void* out, int64_t os) {
  return a.bank->dtype == LQ_F16 ? up_t<__half>(a, low, is_a, base, bs, out, os)
                                 : up_t<__nv_bfloat16>(a, low, is_a, base, bs, out, os);
}
int ad_outer(const AdCall& a, const AdOuter& o) {
  if (o.grad_dtype == LQ_F32)
    return a.bank->dtype == LQ_F16 ? outer_t<__half, float>(a, o) : outer_t<__nv_bfloat16, float>(a, o);
  return a.bank->dtype == LQ_F16 ? outer_t<__half, __half>(a, o) : outer_t<__nv_bfloat16, __nv_bfloat16>(a, o);
}

}  // namespace lq

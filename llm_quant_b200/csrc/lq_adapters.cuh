// lq_adapters.cuh -- what the kernels of the adapter bank share: the plan that
// says which tokens use which adapter, and the arguments of a call.
#pragma once

#include "lq_common.cuh"

namespace lq {

constexpr int kAdTile = 128;        // tokens of a tile
constexpr int kAdMaxAdapters = 8192;
constexpr int kAdMaxRank = 128;

// A tile: up to 128 tokens of one adapter (owner -1: of none), at places first
// .. first + rows - 1 of `order`; run is the first one's token if all follow
// each other, else -1.
struct AdTile {
  int owner, first, rows, run;
};

// One buffer of int32.  Tokens in `order` are sorted by adapter, those without
// one last, and keep their order within each; adapter l has the places start[l]
// .. start[l + 1] - 1 and the tiles tile_of[l] .. tile_of[l + 1] - 1, the
// tokens without an adapter the tiles from tile_of[L] up to tile_of[L + 1].
struct AdPlan {
  int* owner;    // [T]
  int* order;    // [T]
  int* start;    // [L + 2]
  int* tile_of;  // [L + 2]
  AdTile* tiles;
  int* status;   // an lq_status: LQ_ETIMEOUT if a wait on the device ran out
  int* nan;      // whether ad_outer left a sum that is no number, since the plan was made
};

__host__ __device__ inline int64_t ad_round4(int64_t n) { return (n + 3) / 4 * 4; }
// No batch of T tokens has more tiles: each group of tokens ends in at most one
// that is not full, and there are min(L + 1, T) groups at most.
__host__ __device__ inline int64_t ad_max_tiles(int64_t T, int64_t L) {
  const int64_t groups = L + 1 < T ? L + 1 : T;
  const int64_t n = (T + (kAdTile - 1) * groups) / kAdTile;
  return n < T ? n : T;
}
__host__ __device__ inline int64_t ad_plan_ints(int64_t T, int64_t L) {
  return 4 + 2 * ad_round4(T) + 2 * ad_round4(L + 2) + 4 * ad_max_tiles(T, L);
}
__host__ __device__ inline AdPlan ad_plan(void* p, int64_t T, int64_t L) {
  AdPlan a;
  a.status = static_cast<int*>(p);
  a.nan = a.status + 1;
  a.owner = a.status + 4;
  a.order = a.owner + ad_round4(T);
  a.start = a.order + ad_round4(T);
  a.tile_of = a.start + ad_round4(L + 2);
  a.tiles = reinterpret_cast<AdTile*>(a.tile_of + ad_round4(L + 2));
  return a;
}

// The rank, rounded up to what the kernels are made for.
inline int ad_padded(int64_t R) { return R <= 16 ? 16 : R <= 32 ? 32 : R <= 64 ? 64 : 128; }

// What every launch of a call has.
struct AdCall {
  const lq_adapter_bank* bank;
  AdPlan plan;
  int64_t n;
  cudaStream_t st;
};

// The sums of outer products: da = sum v x^T and db = sum u dy^T, either NULL.
struct AdOuter {
  void* v;
  const void* x;
  int64_t x_stride;
  void* da;
  void* u;
  const void* dy;
  int64_t dy_stride;
  void* db;
  int grad_dtype;
  float* part;  // two partial sums of each side's [R, K], [R, N] for each group
  bool behind_down;  // ad_down is the launch before
};
// Groups that the tiles of a call are dealt out to: with all column chunks of
// both sides, one wave of blocks, one to an SM.  Chunks are whole, so that it goes by
// the features how many SMs have one: of 16384 tokens, rank 64, ad_outer and ad_sum
// take 117 us with 4096 and 14336 columns (144 blocks of 148 SMs, 5.2 TB/s), 115 with
// 8192 twice (128 blocks, 4.7), but 211 with 3584 and 18944 and with 8192 and 14336
// (88 blocks, 3.5).
inline int64_t ad_outer_groups(const lq_adapter_bank& b, int64_t n) {
  const int64_t chunks = (b.K + 255) / 256 + (b.N + 255) / 256, tiles = ad_max_tiles(n, b.L);
  int64_t g = (int64_t)num_sms() / chunks;
  g = g < tiles ? g : tiles;
  return g > 1 ? g : 1;
}
inline size_t ad_outer_part_bytes(const lq_adapter_bank& b, int64_t n) {
  return sizeof(float) * 2 * (size_t)ad_outer_groups(b, n) * b.R * (b.K + b.N);
}

// lq_adapters_few.cu: out = base + B^T (s A x), in fp32, a cluster of blocks to a
// token.
int ad_few(const AdCall& a, const void* x, int64_t x_stride, const void* base, int64_t base_stride, void* out,
           int64_t out_stride);

// lq_adapters_mm.cu.  ad_down: low = s A x (is_a) or s B dy, of the tokens with
// an adapter, ad_low_bytes in the forms that the others read (`turned`: ad_outer
// too); ad_up: out = base + A^T low (is_a) or base + B^T low; ad_outer as above.
size_t ad_low_bytes(const lq_adapter_bank& b, int64_t n, bool turned);
int ad_down(const AdCall& a, const void* x, int64_t stride, bool is_a, void* low, bool turned);
int ad_up(const AdCall& a, void* low, bool is_a, const void* base, int64_t base_stride, void* out, int64_t out_stride);
int ad_outer(const AdCall& a, const AdOuter& o);

}  // namespace lq

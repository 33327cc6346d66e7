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
  return 2 * ad_round4(T) + 2 * ad_round4(L + 2) + 4 * ad_max_tiles(T, L);
}
__host__ __device__ inline AdPlan ad_plan(void* p, int64_t T, int64_t L) {
  AdPlan a;
  a.owner = static_cast<int*>(p);
  a.order = a.owner + ad_round4(T);
  a.start = a.order + ad_round4(T);
  a.tile_of = a.start + ad_round4(L + 2);
  a.tiles = reinterpret_cast<AdTile*>(a.tile_of + ad_round4(L + 2));
  return a;
}

}  // namespace lq

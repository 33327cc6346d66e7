// lq_adapters.cu -- low-rank adapters of many requests beside one shared
// projection: y_t = base_t + s_i B_i^T (A_i x_t) with i the adapter of token t,
// and the gradients of x, A and B.  A is [L, R, K], B is [L, R, N] (each
// adapter's lora_B transposed), so that both directions are the same three
// products: rows times a factor (u = s A x, v = s B dy), a low-rank row times a
// factor (y = B^T u, dx = A^T v) and sums of outer products over an adapter's
// tokens (dA = v x^T, dB = u dy^T).
//
// This file: the plan and the entry points; the products are in
// lq_adapters_few.cu and lq_adapters_mm.cu.
#include "lq_adapters.cuh"

namespace lq {
namespace {

// ---------------------------------------------------------------------------
// The plan.  A block to an adapter (block L: the tokens without one) counts all
// requests' tokens by adapter in shared memory (integers: no order of atomics
// shows), adds up the counts below its own, and writes its tokens, in order, by
// sums over the block.  Every block counts for itself: the requests are read
// from L2 L + 1 times, and there is no second launch.  8 requests of 2048 tokens
// with 8 adapters 5.1 us, 16384 tokens by themselves with 64 25 us, 64 requests of
// 16384 with 64 108 us.
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 512;
constexpr int kPlanShort = 32;  // requests of up to so many tokens are a thread's, four at a time; longer ones the block's

struct Share {  // of a request's tokens, the ones that belong to a block
  int from, n;
};
// Tokens 0 .. live - 1 of a request are its adapter's, the others nobody's.
template <typename I>
__device__ __forceinline__ Share share_of(const I* ids, const int* counts, int seq, int L, int r, int me) {
  const int64_t id = static_cast<int64_t>(ids[r]);
  const int live = id < 0 || id >= L ? 0 : counts ? min(max(counts[r], 0), seq) : seq;
  Share s;
  s.from = me == L ? live : 0;
  s.n = me == L ? seq - live : id == me ? live : 0;
  return s;
}

template <typename I>
__global__ void __launch_bounds__(kPlanThreads) ad_plan_kernel(const I* __restrict__ ids, const int* __restrict__ counts,
                                                               int seq, int requests, int L, AdPlan p) {
  extern __shared__ int hist[];  // [L + 1]
  __shared__ int part[2][kPlanThreads / 32];
  __shared__ int base[2], listed;
  __shared__ int4 list[kPlanThreads];  // requests of the block: first token, number, place
  const int me = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i <= L; i += kPlanThreads) hist[i] = 0;
  __syncthreads();
  for (int r = tid; r < requests; r += kPlanThreads) {
    const int64_t id = static_cast<int64_t>(ids[r]);
    const int live = id < 0 || id >= L ? 0 : counts ? min(max(counts[r], 0), seq) : seq;
    if (live) atomicAdd(&hist[static_cast<int>(id)], live);
    if (live < seq) atomicAdd(&hist[L], seq - live);
  }
  __syncthreads();
  int before = 0, tiles = 0;
  for (int i = tid; i < me; i += kPlanThreads) before += hist[i], tiles += (hist[i] + kAdTile - 1) / kAdTile;
#pragma unroll
  for (int m = 16; m; m >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, m);
    tiles += __shfl_xor_sync(0xffffffffu, tiles, m);
  }
  if (lane == 0) part[0][warp] = before, part[1][warp] = tiles;
  __syncthreads();
  if (tid < 2) {
    int s = 0;
    for (int w = 0; w < kPlanThreads / 32; ++w) s += part[tid][w];
    base[tid] = s;
  }
  __syncthreads();
  const int first = base[0], tile = base[1], n = hist[me], n_tiles = (n + kAdTile - 1) / kAdTile;
  if (tid == 0) {
    p.start[me] = first, p.tile_of[me] = tile;
    if (me == L) p.start[L + 1] = first + n, p.tile_of[L + 1] = tile + n_tiles, *p.status = LQ_OK, *p.nan = 0;
  }
  const int owner = me == L ? -1 : me, each = seq <= kPlanShort ? 4 : 1;  // requests of a thread at a time
  int at = first;
  for (int r0 = 0; r0 < requests && at < first + n; r0 += each * kPlanThreads) {
    Share s[4];
    int mine = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = r0 + tid * each + k;
      s[k] = k < each && r < requests ? share_of(ids, counts, seq, L, r, me) : Share{0, 0};
      mine += s[k].n;
    }
    int upto = mine;  // of the warp's threads up to this one
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, upto, m);
      if (lane >= m) upto += x;
    }
    __syncthreads();  // part and list were read
    if (lane == 31) part[0][warp] = upto;
    if (tid == 0) listed = 0;
    __syncthreads();
    int place = at + upto - mine, all = 0;
    for (int w = 0; w < kPlanThreads / 32; ++w) {
      place += w < warp ? part[0][w] : 0;
      all += part[0][w];
    }
    if (each > 1) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int t = (r0 + tid * each + k) * seq + s[k].from;
        for (int i = 0; i < s[k].n; ++i, ++place) p.order[place] = t + i, p.owner[t + i] = owner;
      }
    } else {
      if (mine) list[atomicAdd(&listed, 1)] = make_int4((r0 + tid) * seq + s[0].from, mine, place, 0);
      __syncthreads();
      for (int e = 0; e < listed; ++e) {
        const int4 q = list[e];
        for (int i = tid; i < q.y; i += kPlanThreads) p.order[q.z + i] = q.x + i, p.owner[q.x + i] = owner;
      }
    }
    at += all;
  }
  __syncthreads();  // the block's own order, read back below
  for (int i = tid; i < n_tiles; i += kPlanThreads) {
    AdTile d;
    d.owner = owner;
    d.first = first + i * kAdTile;
    d.rows = min(kAdTile, n - i * kAdTile);
    const int a = p.order[d.first], z = p.order[d.first + d.rows - 1];
    d.run = z - a == d.rows - 1 ? a : -1;
    p.tiles[tile + i] = d;
  }
}

int check_bank(const lq_adapter_bank* b, const void* plan, int64_t n) {
  LQ_REQUIRE(b && b->a && b->b && b->scaling, LQ_EINVAL, "adapters: NULL bank");
  LQ_REQUIRE(b->dtype == LQ_F16 || b->dtype == LQ_BF16, LQ_EDTYPE, "adapters: fp16 or bf16 (got dtype %d)", b->dtype);
  LQ_REQUIRE(b->L >= 1 && b->L <= kAdMaxAdapters, LQ_ERANGE, "adapters: %lld adapters outside [1, %d]", (long long)b->L,
             kAdMaxAdapters);
  LQ_REQUIRE(b->R >= 1 && b->R <= kAdMaxRank, LQ_ERANGE, "adapters: rank %lld outside [1, %d]", (long long)b->R, kAdMaxRank);
  LQ_REQUIRE(b->K >= 8 && b->N >= 8 && b->K <= (1 << 22) && b->N <= (1 << 22), LQ_ERANGE, "adapters: features outside [8, 2^22]");
  LQ_REQUIRE(b->K % 8 == 0 && b->N % 8 == 0, LQ_EALIGN, "adapters: features must be multiples of 8");
  LQ_REQUIRE(aligned16(b->a) && aligned16(b->b), LQ_EALIGN, "adapters: weights must be 16-byte aligned");
  LQ_REQUIRE(n >= 0 && n <= (1 << 24), LQ_ERANGE, "adapters: %lld tokens outside [0, 2^24]", (long long)n);
  LQ_REQUIRE(n == 0 || (plan && aligned16(plan)), LQ_EINVAL, "adapters: the plan is NULL or not 16-byte aligned");
  return LQ_OK;
}
int check_rows(const char* what, const void* p, int64_t stride, int64_t width, bool wide) {
  LQ_REQUIRE(p && aligned16(p) && stride % 8 == 0, LQ_EALIGN, "adapters: %s must be on 16 bytes, its rows too", what);
  LQ_REQUIRE(stride >= (wide ? width : 0), LQ_EINVAL, "adapters: rows of %s overlap", what);
  return LQ_OK;
}

bool sizes_ok(const lq_adapter_bank& b, int64_t n) {
  return n >= 0 && n <= (1 << 24) && b.L >= 1 && b.L <= kAdMaxAdapters && b.R >= 1 && b.R <= kAdMaxRank && b.K >= 8 && b.N >= 8;
}
size_t v_bytes(const lq_adapter_bank& b, int64_t n) { return (ad_low_bytes(b, n, true) + 255) / 256 * 256; }

}  // namespace
}  // namespace lq

using namespace lq;

extern "C" size_t lq_adapter_plan_bytes(int64_t n, int64_t L) {
  if (n < 0 || n > (1 << 24) || L < 1 || L > kAdMaxAdapters) return 0;
  return 4 * (size_t)ad_plan_ints(n, L);
}

extern "C" int lq_adapter_plan(const void* ids, int ids_dtype, int64_t n_ids, int64_t seq_len, const int32_t* counts,
                               int64_t L, void* plan, void* stream) {
  LQ_REQUIRE(ids_dtype == LQ_I32 || ids_dtype == LQ_I64, LQ_EDTYPE, "adapters: ids must be int32 or int64");
  LQ_REQUIRE(L >= 1 && L <= kAdMaxAdapters, LQ_ERANGE, "adapters: %lld adapters outside [1, %d]", (long long)L, kAdMaxAdapters);
  LQ_REQUIRE(n_ids >= 0 && n_ids <= (1 << 24) && seq_len >= 0 && seq_len <= (1 << 24) && n_ids * seq_len <= (1 << 24),
             LQ_ERANGE, "adapters: tokens outside [0, 2^24]");
  const int64_t n = n_ids * seq_len;
  LQ_REQUIRE(n == 0 || (ids && plan && aligned16(plan)), LQ_EINVAL, "adapters: NULL ids, or a plan not on 16 bytes");
  if (n == 0) return LQ_OK;
  const AdPlan p = ad_plan(plan, n, L);
  const size_t smem = 4 * (size_t)(L + 1);
  cudaStream_t st = as_stream(stream);
  if (ids_dtype == LQ_I32)
    ad_plan_kernel<int32_t><<<(unsigned)L + 1, kPlanThreads, smem, st>>>(static_cast<const int32_t*>(ids), counts, (int)seq_len, (int)n_ids, (int)L, p);
  else
    ad_plan_kernel<int64_t><<<(unsigned)L + 1, kPlanThreads, smem, st>>>(static_cast<const int64_t*>(ids), counts, (int)seq_len, (int)n_ids, (int)L, p);
  return launched("ad_plan_kernel");
}

// Whether a call takes ad_few, where every token reads its adapter's weights,
// through L2 where tokens share them, or the tiles, where an adapter's tokens
// share a read but two launches and a tile's fixed costs stand against it.  How
// many adapters a call's tokens use is not known here: as many as there can be.
// Measured (us on the device, ad_few / tiles, weights from memory, `users` adapters
// in the bank and in use), over 420 shapes of ranks 16 to 128, 4096 to 14336 features
// and 4 to 256 tokens, of which the choice below is over 5 % slower than the other in
// 10, by 23 % at most.  B costs ad_few some three times what A does:
//   rank  features     users  tokens
//     16   4096  4096      1      64   4.5 / 10    256   7.9 / 11
//     64   4096  4096      1      64   9.8 / 13     96    16 / 15    256    30 / 16
//     64   4096  4096    all      64    16 / 30     96    25 / 42    256    50 / 91
//     64   4096 14336      1      24    13 / 13     48    23 / 13     96    44 / 15
//     64  14336  4096      1      48    18 / 20     64    18 / 20     96    32 / 22
//    128  14336 14336      8      16    35 / 37     32    37 / 37     64    66 / 37
//    128  14336 14336    all      16    40 / 49     64    88 / 139   256   312 / 534
// and, where a block's columns of so many ranks are a longer chain than the tiles':
//    128   4096 14336      1       1    25 / 13     16    22 / 15
//    128   4096 14336      4       4    25 / 22
//    128   4096 14336      8       8    26 / 28
static bool few_tokens(const lq_adapter_bank& b, const lq_adapter_form* f) {
  if (f->keep || f->n > 1024) return false;
  const int64_t cost = b.R * (b.K + 3 * b.N), users = f->n < b.L ? f->n : b.L;
  if (users <= 4 && 2 * b.R * b.N > (3 << 20)) return false;
  return f->n * cost <= (112 << 20) + users * cost * 3 / 2;
}

extern "C" size_t lq_adapter_low_bytes(const lq_adapter_bank* bank, const lq_adapter_form* form) {
  if (!bank || !form || !sizes_ok(*bank, form->n) || few_tokens(*bank, form)) return 0;
  return ad_low_bytes(*bank, form->n, form->keep != 0);
}

extern "C" int lq_adapter_forward(const lq_adapter_bank* bank, const lq_adapter_form* form, void* plan, const void* x,
                                  const void* base, void* out, void* low, size_t low_bytes, void* stream) {
  LQ_REQUIRE(form, LQ_EINVAL, "adapters: NULL form");
  const int64_t n = form->n;
  LQ_TRY(check_bank(bank, plan, n));
  if (n == 0) return LQ_OK;
  LQ_TRY(check_rows("x", x, form->x_stride, bank->K, false));
  LQ_TRY(check_rows("out", out, form->out_stride, bank->N, n > 1));
  if (base) LQ_TRY(check_rows("base", base, form->base_stride, bank->N, false));
  LQ_REQUIRE(base != out || form->base_stride == form->out_stride, LQ_EINVAL, "adapters: out is base, with other rows");
  const size_t need = lq_adapter_low_bytes(bank, form);
  LQ_REQUIRE(need == 0 || (low && aligned16(low) && low_bytes >= need), LQ_EINVAL, "adapters: low must have %zu bytes, on 16", need);
  const AdCall a = {bank, ad_plan(plan, n, bank->L), n, as_stream(stream)};
  if (few_tokens(*bank, form)) return ad_few(a, x, form->x_stride, base, form->base_stride, out, form->out_stride);
  LQ_TRY(ad_down(a, x, form->x_stride, true, low, form->keep != 0));
  return ad_up(a, low, false, base, form->base_stride, out, form->out_stride);
}

extern "C" size_t lq_adapter_backward_workspace_bytes(const lq_adapter_bank* bank, int64_t n) {
  if (!bank || !sizes_ok(*bank, n)) return 0;
  return v_bytes(*bank, n) + ad_outer_part_bytes(*bank, n);
}

extern "C" int lq_adapter_backward(const lq_adapter_bank* bank, const lq_adapter_form* form, void* plan, const void* x,
                                   const void* dy, void* low, size_t low_bytes, void* dx, void* da, void* db, int grad_dtype,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  LQ_REQUIRE(form, LQ_EINVAL, "adapters: NULL form");
  const int64_t n = form->n;
  LQ_TRY(check_bank(bank, plan, n));
  LQ_REQUIRE(grad_dtype == LQ_F32 || grad_dtype == bank->dtype, LQ_EDTYPE, "adapters: gradients in fp32 or the bank's type");
  cudaStream_t st = as_stream(stream);
  if (n == 0) {
    const size_t size = bank->L * bank->R * (grad_dtype == LQ_F32 ? 4 : 2);
    LQ_REQUIRE(!da || cudaMemsetAsync(da, 0, size * bank->K, st) == cudaSuccess, LQ_ECUDA, "adapters: memset failed");
    LQ_REQUIRE(!db || cudaMemsetAsync(db, 0, size * bank->N, st) == cudaSuccess, LQ_ECUDA, "adapters: memset failed");
    return LQ_OK;
  }
  LQ_TRY(check_rows("dy", dy, form->out_stride, bank->N, false));
  if (da) LQ_TRY(check_rows("x", x, form->x_stride, bank->K, false));
  LQ_REQUIRE(!dx || aligned16(dx), LQ_EALIGN, "adapters: dx must be 16-byte aligned");
  LQ_REQUIRE(!db || (form->keep && low && aligned16(low) && low_bytes >= ad_low_bytes(*bank, n, true)), LQ_EINVAL,
             "adapters: low must be what a forward call with `keep` left");
  const size_t need = lq_adapter_backward_workspace_bytes(bank, n);
  LQ_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= need, LQ_EINVAL, "adapters: %zu bytes of workspace needed", need);
  const AdCall a = {bank, ad_plan(plan, n, bank->L), n, st};
  void* v = workspace;
  float* part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + v_bytes(*bank, n));
  if (dx || da) LQ_TRY(ad_down(a, dy, form->out_stride, false, v, da != nullptr));
  if (da || db) LQ_TRY(ad_outer(a, {v, x, form->x_stride, da, low, dy, form->out_stride, db, grad_dtype, part, dx || da}));
  if (dx) LQ_TRY(ad_up(a, v, true, nullptr, 0, dx, bank->K));
  return LQ_OK;
}

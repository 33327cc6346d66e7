// lq_kv4.cuh -- layout of the 4-bit KV cache (lq_kv4_cache) and the pieces
// its kernels share.
//
// One token of one kv head holds, for K and for V each, D codes of 4 bits and
// one parameter word: value = (code - zero) * scale, scale in bf16 (low half
// of the word), zero (an integer 0..15) as bf16 (high half).  Both halves
// become fp32 with one shift or mask.  The words of K and V of a token lie
// side by side (uint2), [B, H, cap].
//
// K codes [B, H, cap, D / 2]: value d in 32-bit word d / 8 of the token's row,
// nibble (d % 8) / 2 of its low half for even d and of its high half for odd d:
// a mask (after a shift by whole nibbles) leaves two neighbouring values.
//
// V codes [B, H, cap / 16, 8 D]: tiles of 16 tokens, laid out as the A
// fragments of mma.m16n8k16 for O^T = V^T P^T: the 16-bit unit u of token t
// (values 4u .. 4u+3, lowest nibble first) lies in the tile at byte
//   half * (W * 128) + lane * (W * 4) + i * 4 + (t & 1) * 2
// with W = D / 32, half = t % 16 / 8, lane = 4 (u / W) + t % 8 / 2, i = u % W.
// A lane's words are then one aligned vector, the warp's are contiguous, and
// a word holds the same values of two neighbouring tokens in its two halves,
// which is what a fragment register wants.
//
// Conversion: a nibble in bits 0..3 of an f16 is the subnormal code * 2^-24,
// one in bits 4..7 is code * 2^-20, exactly.  So `word & 0x000f000f` is a
// fragment register of two codes, with no addition and no magic number; the
// powers of two and the zero points are applied to the fp32 accumulators.
#pragma once

#include "lq_common.cuh"

namespace lq {

struct Kv4 {
  uint8_t* k;
  uint8_t* v;
  uint2* par;
  int32_t* pos;
  float* mass;
  int32_t* len;   // [B] tokens held
  int32_t* next;  // [B] position of the next token
  int32_t* sync;  // [0] ticket of the running call, [1] tokens dropped for want of room, [2] something was evicted, [3] a wait on the device ran out
  int B, H, cap, D;
};

namespace {

constexpr int kUnit = 32;  // tokens that a warp takes at a time (two tiles of 16)

// Dynamic shared memory of a kernel, asked for once on each device (the call
// takes as long as a small launch): one of these beside each kernel.
struct DeviceOnce {
  std::atomic<uint64_t> done{0};
  int allow_smem(const void* kernel, int bytes, const char* what) {
    int dev = 0;
    cudaGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_relaxed) & bit) return LQ_OK;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) {
      set_error("%s: %d bytes of shared memory: %s", what, bytes, cudaGetErrorString(e));
      cudaGetLastError();
      return LQ_ECUDA;
    }
    if (dev < 64) done.fetch_or(bit, std::memory_order_relaxed);
    return LQ_OK;
  }
};

inline Kv4 kv4_of(const lq_kv4_cache* c) {
  Kv4 k;
  k.k = static_cast<uint8_t*>(c->k_codes);
  k.v = static_cast<uint8_t*>(c->v_codes);
  k.par = static_cast<uint2*>(c->params);
  k.pos = c->positions;
  k.mass = c->mass;
  k.len = c->state;
  k.next = c->state + c->B;
  k.sync = c->state + 2 * c->B;
  k.B = (int)c->B;
  k.H = (int)c->H;
  k.cap = (int)c->cap;
  k.D = (int)c->D;
  return k;
}

inline int kv4_check(const lq_kv4_cache* c) {
  LQ_REQUIRE(c, LQ_EINVAL, "NULL cache");
  LQ_REQUIRE(c->B > 0 && c->H > 0 && c->cap > 0, LQ_EINVAL, "bad cache shape");
  LQ_REQUIRE(c->D == 64 || c->D == 128, LQ_EINVAL, "head dim %lld: 64 or 128 supported", (long long)c->D);
  LQ_REQUIRE(c->cap % kUnit == 0, LQ_EINVAL, "capacity %lld must be a multiple of %d", (long long)c->cap, kUnit);
  LQ_REQUIRE(c->cap <= (1LL << 30) && c->B * c->H <= 65535, LQ_ERANGE, "cache too large");
  LQ_REQUIRE(c->k_codes && c->v_codes && c->params && c->positions && c->mass && c->state, LQ_EINVAL, "NULL pointer");
  LQ_REQUIRE(aligned16(c->k_codes) && aligned16(c->v_codes) && aligned16(c->params) && aligned16(c->positions) &&
                 aligned16(c->mass),
             LQ_EALIGN,
             "cache buffers must be 16-byte aligned");
  return LQ_OK;
}

// Byte of unit u of token t inside a head's V codes (see above).
__device__ __forceinline__ int64_t v_unit(int64_t t, int u, int W) {
  const int r = (int)(t & 15);
  return (t >> 4) * (W * 256) + (r >> 3) * (W * 128) + (4 * (u / W) + ((r & 7) >> 1)) * (W * 4) + (u % W) * 4 + (r & 1) * 2;
}

__device__ __forceinline__ float par_scale(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float par_zero(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

// The block that finishes last may change what all blocks have read: every
// block calls this after its last read of the cache's lengths, and all threads
// of one block get true.  The counter is zero again afterwards, so that the
// next call (or the next replay of a graph) finds it as this one did.
__device__ __forceinline__ bool last_block(int32_t* ticket, int blocks) {
  __shared__ bool last;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(ticket, 1) == blocks - 1;
    if (last) *ticket = 0;
  }
  __syncthreads();
  return last;
}

}  // namespace
}  // namespace lq

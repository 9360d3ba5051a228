// int8_tile.h — operand pieces, LDS loads and epilogue functions of the int8 products (linear_int8.hip,
// expert_linear.hip).
#pragma once

#include "decoder_common.h"
#include "mfma_frag.h"

namespace rxmet {
namespace dec {

__device__ __forceinline__ float activate(float v, int act) {
  switch (act) {
    case RXMET_ACT_RELU: return v < 0.0f ? 0.0f : v;
    case RXMET_ACT_SILU: return v / (1.0f + expf(-v));
    case RXMET_ACT_GELU: return 0.5f * v * (1.0f + erff(v * 0.70710678118654752440f));
    default: return v;
  }
}

// Bytes k..k+15 of a row of K; those past its end are 0.
__device__ __forceinline__ uint4 load_piece(const int8_t *row, int k, int K) {
  uint4 v = {0, 0, 0, 0};
  if (k + 16 <= K) {
    __builtin_memcpy(&v, row + k, 16);
  } else {
    unsigned u[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (k + e < K) u[e / 4] |= static_cast<unsigned>(static_cast<uint8_t>(row[k + e])) << (8 * (e % 4));
    v = make_uint4(u[0], u[1], u[2], u[3]);
  }
  return v;
}

__device__ __forceinline__ v4i as_v4i(uint4 u) { return __builtin_bit_cast(v4i, u); }

// The sum times such a row scale may leave fp32 where the result does not: the weight's scale goes first.
__device__ __forceinline__ bool is_large(float sx) { return fabsf(sx) > 0x1p90f; }

constexpr int kStep = 64;

typedef int v16i __attribute__((ext_vector_type(16)));

// f of a weight row and of a token row
__device__ __forceinline__ int turn_w(int row) { return (row >> 2 & 1) | (row >> 3 & 2); }
__device__ __forceinline__ int turn_x(int row) { return row >> 2 & 3; }

// 16 bytes of each lane's address to LDS at `lds` + 16 * lane, in flight until vmcnt says so.
__device__ __forceinline__ void load_to_lds(const int8_t *p, int8_t *lds) {
  __builtin_amdgcn_global_load_lds(
      (const __attribute__((address_space(1))) void *)p,
      (__attribute__((address_space(3))) void *)lds, 16, 0, 0);
}
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
// A barrier that lets loads to LDS stay in flight (__syncthreads waits for them).  What this wave
// wrote to or read from LDS before it is done.
__device__ __forceinline__ void meet() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
}

}  // namespace dec
}  // namespace rxmet

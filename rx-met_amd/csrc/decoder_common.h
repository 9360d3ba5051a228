// decoder_common.h — element types, vectors of eight and the int8 grid of the 8-bit decoder
// operators (rms_quant.hip, linear_int8.hip, kv_cache.hip, kv_attention.hip).
#pragma once

#include "../../include/rxmet_decoder.h"
#include "../../include/rxmet_qdq.h"
#include "rxmet_common.h"

namespace rxmet {
namespace dec {

typedef _Float16 f16;
typedef __bf16 bf16;

// Least magnitude that a scale is made from: 127 / 2^-112 and the scale itself stay normal.
constexpr float kFloor = 0x1p-112f;
constexpr float kInv127 = static_cast<float>(1.0 / 127.0);

__device__ __forceinline__ float nanf32() { return __builtin_nanf(""); }

// Eight consecutive elements as fp32.  Rows of odd length start at any element, so the access is
// declared with the element's alignment; gfx950 takes such 16-byte accesses in one instruction.
template <typename T>
struct Vec8 {
  T v[8];
};

template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&f)[8]) {
  Vec8<T> u;
  __builtin_memcpy(&u, p, sizeof(u));
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = static_cast<float>(u.v[e]);
}

// The first n < 8 of them; the others become 0.
template <typename T>
__device__ __forceinline__ void load8_part(const T *p, int n, float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = e < n ? static_cast<float>(p[e]) : 0.0f;
}

template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&f)[8]) {
  Vec8<T> u;
#pragma unroll
  for (int e = 0; e < 8; ++e) u.v[e] = static_cast<T>(f[e]);
  __builtin_memcpy(p, &u, sizeof(u));
}

template <typename T>
__device__ __forceinline__ void store8_part(T *p, int n, const float (&f)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < n) p[e] = static_cast<T>(f[e]);
}

// The code of v, |v| < 2^22, in the low byte: adding 1.5 * 2^23 rounds half to even into the last
// bits of the sum.  A NaN gives 0.
__device__ __forceinline__ unsigned code_byte(float v) {
  return __builtin_bit_cast(unsigned, v + 12582912.0f) & 0xffu;
}

__device__ __forceinline__ unsigned code_bytes4(float a, float b, float c, float d) {
  return code_byte(a) | code_byte(b) << 8 | code_byte(c) << 16 | code_byte(d) << 24;
}

// Byte k of a word as a signed code.
__device__ __forceinline__ float code_value(unsigned w, int k) {
  return static_cast<float>(static_cast<int>(w << (24 - 8 * k)) >> 24);
}

// Runs f(T{}) for an element type of the ABI; false for another one.
template <typename F>
bool with_type(int32_t dtype, F &&f) {
  switch (dtype) {
    case RXMET_QDQ_F32: f(float{}); return true;
    case RXMET_QDQ_F16: f(f16{}); return true;
    case RXMET_QDQ_BF16: f(bf16{}); return true;
    default: return false;
  }
}

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace dec
}  // namespace rxmet

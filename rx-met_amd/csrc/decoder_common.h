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

// store8 past the caches' usual order, for outputs as large as the inputs that go through
// the caches beside them ([8192, 4096] bf16, norm forward and backward: 124 -> 110 us; loads of
// this kind bring 4 us more there and cost 2 to 6 us where rows are short or not aligned).
typedef int v4i_any __attribute__((ext_vector_type(4), aligned(2)));
template <typename T>
__device__ __forceinline__ void stream_out8(T *p, const float (&f)[8]) {
  Vec8<T> u;
#pragma unroll
  for (int e = 0; e < 8; ++e) u.v[e] = static_cast<T>(f[e]);
#pragma unroll
  for (int k = 0; k < static_cast<int>(sizeof(u) / 16); ++k) {
    v4i_any w;
    __builtin_memcpy(&w, reinterpret_cast<const char *>(&u) + 16 * k, 16);
    __builtin_nontemporal_store(w, reinterpret_cast<v4i_any *>(p) + k);
  }
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
// bits of the sum.  A NaN gives a byte of its payload: groups that hold one are cleared with `keep` of
// code_bytes4, 0 there and ~0 elsewhere.
__device__ __forceinline__ unsigned code_word(float v) {
  return __builtin_bit_cast(unsigned, v + 12582912.0f);
}

__device__ __forceinline__ unsigned code_bytes4(float a, float b, float c, float d, unsigned keep = ~0u) {
  const unsigned lo = __builtin_amdgcn_perm(code_word(b), code_word(a), 0x0c0c0400u);
  return (lo | __builtin_amdgcn_perm(code_word(d), code_word(c), 0x04000c0cu)) & keep;
}

// The largest magnitude as an integer: without their signs, floats are ordered as their bits are,
// infinity above all numbers and NaN above infinity, so that a maximum of bits keeps a NaN.
__device__ __forceinline__ unsigned magnitude(float v) {
  return __builtin_bit_cast(unsigned, v) & 0x7fffffffu;
}
__device__ __forceinline__ unsigned wave_max_bits(unsigned v) {
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) {
    const unsigned o = __shfl_xor(v, off, kWave);
    v = o > v ? o : v;
  }
  return v;
}

// Largest magnitude of vectors of eight, as fp32 bits once asked for: two 16-bit values a step.
template <typename T>
struct Peak {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  u16x2 top = {0, 0};
  __device__ __forceinline__ void add(const Vec8<T> &v) {
    unsigned w[4];
    __builtin_memcpy(w, &v, 16);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[k] & 0x7fff7fffu));
  }
  __device__ __forceinline__ unsigned bits() const {
    const unsigned short t = top[0] > top[1] ? top[0] : top[1];
    return magnitude(static_cast<float>(__builtin_bit_cast(T, t)));
  }
};
template <>
struct Peak<float> {
  unsigned top = 0;
  __device__ __forceinline__ void add(const Vec8<float> &v) {
#pragma unroll
    for (int k = 0; k < 8; ++k) top = __builtin_elementwise_max(top, magnitude(v.v[k]));
  }
  __device__ __forceinline__ unsigned bits() const { return top; }
};

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

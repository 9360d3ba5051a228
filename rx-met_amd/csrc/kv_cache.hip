// kv_cache.hip — the paged int8 cache of keys and values: new tokens in, values out.
//
// One scale covers a page's tokens of one head.  A page that new tokens enter gets the scale
// s' = max(max|new| / 127, s), s its scale so far if it holds older tokens of the sequence; where s' > s
// the older codes are moved to the new grid, rint(c * s / s').  Keys lie token by token, values
// dimension by dimension (each dimension's tokens side by side): both are what a lane of the
// attention's matrix instructions reads as 16 consecutive bytes.
//
// A workgroup owns a page's keys or values of one head.  No two workgroups write the same bytes, and the
// older codes are read only where they move or share 16 bytes with a new token.
//
// Bound: HBM traffic for prompts (each new token read once, its codes written), the launch and three dependent
// reads (length, page, codes) for single tokens.  Measured, bf16, 8 heads of 128, pages of 64: 28098
// tokens of 8 prompts in 45 us (173 MB, 3.8 TB/s, the tokens in no cache), read back in 31 us (172 MB,
// 5.5 TB/s); one token for each of 64 sequences 6.0 us, their open pages read back in 7.2 us.
// Neighbouring workgroups have neighbouring heads, so that those at work together read whole rows of the
// tokens (pages first: 50, 30, 6.8 and 9.4 us; 20 sequences of 500 to 1000 tokens, 3 heads of 64, pages of 16:
// 24 and 13.5 us then, 20.5 and 12.4 so).
#include <type_traits>

#include "kv_cache.h"

namespace rxmet {
namespace dec {
namespace {

struct AppendArgs {
  Pages g;
  const int32_t *lengths, *cu;
  int64_t tokens;
  const void *x[2];  // key, value
  int64_t stride_t[2], stride_h[2];
};

__device__ __forceinline__ float block_max(unsigned v) {
  __shared__ unsigned s[4];
  v = wave_max_bits(v);
  __syncthreads();  // the last page's maxima have been read
  if (threadIdx.x % kWave == 0) s[threadIdx.x / kWave] = v;
  __syncthreads();
  const unsigned a = s[0] > s[1] ? s[0] : s[1], b = s[2] > s[3] ? s[2] : s[3];
  return __builtin_bit_cast(float, a > b ? a : b);
}

// Four codes of an old page on its new grid.
__device__ __forceinline__ unsigned move_codes(unsigned w, float ratio) {
  return code_bytes4(code_value(w, 0) * ratio, code_value(w, 1) * ratio, code_value(w, 2) * ratio,
                     code_value(w, 3) * ratio);
}

// A thread holds units of four tokens x eight dimensions in registers between the maximum and the
// codes, so that the tokens are read once; values are turned in LDS, where a unit gives one word (four
// tokens) for each dimension.
template <typename T, int D, int P>
__global__ __launch_bounds__(256) void kv_append(const AppendArgs a) {
  constexpr int C = D / 8;                              // chunks of eight dimensions
  constexpr int units = P / 4 * C, NU = (units + 255) / 256;
  constexpr int pitch = P / 4 + 1;                      // words of a dimension in LDS
  __shared__ unsigned s_v[D * pitch];
  const int tid = threadIdx.x, heads = a.g.c.heads, b = blockIdx.z;
  const int which = static_cast<int>(blockIdx.x) >= heads;  // 0: keys, 1: values
  const int head = blockIdx.x - which * heads;
  const int64_t start = a.lengths[b];
  const int64_t row0 = a.cu ? a.cu[b] : b;
  int64_t count = a.cu ? a.cu[b + 1] - row0 : 1;
  if (start < 0 || row0 < 0) return;
  if (count > a.tokens - row0) count = a.tokens - row0;
  if (count <= 0) return;
  const int64_t first = start / P, last = (start + count - 1) / P;
  int8_t *pool = which ? a.g.c.v : a.g.c.k;
  float *scales = which ? a.g.c.v_scale : a.g.c.k_scale;
  const int64_t stride = a.stride_t[which];
  const T *x = static_cast<const T *>(a.x[which]) + head * a.stride_h[which];
  for (int64_t p = first + blockIdx.y; p <= last; p += gridDim.y) {
    const int64_t page = page_of(a.g, b, p);
    if (page < 0) continue;
    // new tokens stand in slots s0..s1-1, older ones below s0
    const int s0 = static_cast<int>(p == first ? start - p * P : 0);
    const int s1 = static_cast<int>(p == last ? start + count - p * P : P);
    const int64_t row = row0 + p * P - start;  // of slot 0 (may lie before the rows)
    const int64_t at = page * a.g.c.heads + head;
    int8_t *codes = pool + at * P * D;
    const float was = s0 > 0 ? scales[at] : 0.0f;
    Vec8<T> u[NU][4];
    Peak<T> peak;
#pragma unroll
    for (int j = 0; j < NU; ++j) {
      const int i = tid + 256 * j, c = i % C, q = i / C * 4;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        u[j][e] = {};
        if (q + e >= s0 && q + e < s1)  // false past the last unit, where q >= P
          __builtin_memcpy(&u[j][e], x + (row + q + e) * stride + 8 * c, sizeof(Vec8<T>));
      }
    }
#pragma unroll
    for (int j = 0; j < NU; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) peak.add(u[j][e]);
    const float top = block_max(peak.bits());
    // block_max's barriers stand between every thread's read of the old scale and this write
    const bool good = top <= 3.402823466e38f && was == was;
    const float fresh = fmaxf(top, kFloor) * kInv127;
    const float scale = good ? fmaxf(fresh, was) : nanf32();
    const float inv = good ? 1.0f / scale : 0.0f;
    const float ratio = good ? was * inv : 0.0f;
    const unsigned keep = good ? ~0u : 0u;
    const bool moves = s0 > 0 && !(scale == was);
    if (tid == 0) scales[at] = scale;
    if (which == 0) {
#pragma unroll
      for (int j = 0; j < NU; ++j) {
        const int i = tid + 256 * j, c = i % C, q = i / C * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (q + e < s0 || q + e >= s1) continue;
          unsigned w[2];
#pragma unroll
          for (int k = 0; k < 2; ++k)
            w[k] = code_bytes4(static_cast<float>(u[j][e].v[4 * k]) * inv,
                               static_cast<float>(u[j][e].v[4 * k + 1]) * inv,
                               static_cast<float>(u[j][e].v[4 * k + 2]) * inv,
                               static_cast<float>(u[j][e].v[4 * k + 3]) * inv, keep);
          *reinterpret_cast<uint2 *>(codes + (q + e) * D + 8 * c) = make_uint2(w[0], w[1]);
        }
      }
      if (moves) {
        for (int i = tid; i < s0 * (D / 16); i += 256) {
          uint4 w = *reinterpret_cast<const uint4 *>(codes + i * 16);
          w = make_uint4(move_codes(w.x, ratio), move_codes(w.y, ratio), move_codes(w.z, ratio),
                         move_codes(w.w, ratio));
          *reinterpret_cast<uint4 *>(codes + i * 16) = w;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < NU; ++j) {
        const int i = tid + 256 * j, c = i % C, q = i / C;
        if (i < units) {
#pragma unroll
          for (int d = 0; d < 8; ++d)
            s_v[(8 * c + d) * pitch + q] = code_bytes4(
                static_cast<float>(u[j][0].v[d]) * inv, static_cast<float>(u[j][1].v[d]) * inv,
                static_cast<float>(u[j][2].v[d]) * inv, static_cast<float>(u[j][3].v[d]) * inv, keep);
        }
      }
      __syncthreads();
      // pieces of 16 slots of a dimension: those with a new token, and those whose codes move
      const int from = moves ? 0 : s0 / 16, to = (s1 + 15) / 16;
      for (int i = tid; i < (to - from) * D; i += 256) {
        const int g = from + i % (to - from), d = i / (to - from), old = s0 - 16 * g;
        uint4 *place = reinterpret_cast<uint4 *>(codes + d * P + 16 * g);
        const unsigned *n = s_v + d * pitch + 4 * g;
        unsigned w[4] = {n[0], n[1], n[2], n[3]};
        if (old > 0) {  // the older codes of the piece
          unsigned o[4];
          __builtin_memcpy(o, place, 16);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (moves) o[k] = move_codes(o[k], ratio);
            const int keep = old - 4 * k;  // of this word's bytes
            const unsigned mask = keep <= 0 ? 0u : keep >= 4 ? ~0u : (1u << (8 * keep)) - 1;
            w[k] = (o[k] & mask) | (w[k] & ~mask);
          }
        }
        *place = make_uint4(w[0], w[1], w[2], w[3]);
      }
      __syncthreads();  // the next page's codes take the LDS
    }
  }
}

struct ReadArgs {
  Pages g;
  const int32_t *first, *cu;
  int64_t tokens;
  void *out[2];
};

template <typename T, int D, int P>
__global__ __launch_bounds__(256) void kv_read(const ReadArgs a) {
  const int tid = threadIdx.x, heads = a.g.c.heads, b = blockIdx.z;
  const int which = static_cast<int>(blockIdx.x) >= heads;  // 0: keys, 1: values
  const int head = blockIdx.x - which * heads;
  const int64_t start = a.first[b], row0 = a.cu[b];
  int64_t count = a.cu[b + 1] - row0;
  if (row0 < 0) return;
  if (count > a.tokens - row0) count = a.tokens - row0;
  if (count <= 0) return;
  // pages of tokens before 0 have no place in the table: their values are NaN
  const int64_t first = start >= 0 ? start / P : -((-start + P - 1) / P);
  const int64_t end = start + count, last = end > 0 ? (end - 1) / P : -((-end + P) / P);
  const int64_t pitch = static_cast<int64_t>(a.g.c.heads) * D;
  T *out = static_cast<T *>(a.out[which]) + head * D;
  for (int64_t p = first + blockIdx.y; p <= last; p += gridDim.y) {
    const int64_t page = page_of(a.g, b, p);
    const int s0 = static_cast<int>(p == first ? start - p * P : 0);
    const int s1 = static_cast<int>(p == last ? end - p * P : P);
    const int64_t at = (page < 0 ? 0 : page) * a.g.c.heads + head;
    const int8_t *codes = (which ? a.g.c.v : a.g.c.k) + at * P * D;
    const float scale = page < 0 ? nanf32() : (which ? a.g.c.v_scale : a.g.c.k_scale)[at];
    T *q = out + (row0 + p * P - start) * pitch;  // slot 0's row (may lie before the rows)
    if (which == 0) {
      constexpr int C = D / 16;
#pragma unroll 4
      for (int i = s0 * C + tid; i < s1 * C; i += 256) {
        const uint4 u = *reinterpret_cast<const uint4 *>(codes + i * 16);
        const unsigned w[4] = {u.x, u.y, u.z, u.w};
        T *o = q + i / C * pitch + i % C * 16;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float f[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = code_value(w[2 * k + e / 4], e % 4) * scale;
          store8(o + 8 * k, f);
        }
      }
    } else {
      // a thread takes 16 slots of two dimensions, so that a wave writes 128 or 256 bytes of a row
      const int from = s0 / 16, groups = (s1 + 15) / 16 - from;
      for (int i = tid; i < groups * (D / 2); i += 256) {
        const int d = i % (D / 2) * 2, lo = (from + i / (D / 2)) * 16;
        const uint4 u0 = *reinterpret_cast<const uint4 *>(codes + d * P + lo);
        const uint4 u1 = *reinterpret_cast<const uint4 *>(codes + (d + 1) * P + lo);
        const unsigned w0[4] = {u0.x, u0.y, u0.z, u0.w}, w1[4] = {u1.x, u1.y, u1.z, u1.w};
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if (lo + e < s0 || lo + e >= s1) continue;
          struct {
            T v[2];
          } o = {{static_cast<T>(code_value(w0[e / 4], e % 4) * scale),
                  static_cast<T>(code_value(w1[e / 4], e % 4) * scale)}};
          __builtin_memcpy(q + (lo + e) * pitch + d, &o, sizeof(o));
        }
      }
    }
  }
}

// Runs f(dim, page size) for a cache that check_cache has passed.
template <typename F>
void with_page_shape(const rxmet_kv_cache &c, F &&f) {
  auto sized = [&](auto d) {
    switch (c.page_size) {
      case 16: f(d, std::integral_constant<int, 16>{}); break;
      case 32: f(d, std::integral_constant<int, 32>{}); break;
      case 64: f(d, std::integral_constant<int, 64>{}); break;
      default: f(d, std::integral_constant<int, 128>{}); break;
    }
  };
  switch (c.dim) {
    case 64: sized(std::integral_constant<int, 64>{}); break;
    case 128: sized(std::integral_constant<int, 128>{}); break;
    case 192: sized(std::integral_constant<int, 192>{}); break;
    default: sized(std::integral_constant<int, 256>{}); break;
  }
}

}  // namespace

int check_cache(const rxmet_kv_cache *c, const rxmet_kv_table *t) {
  RXMET_CHECK_ARG(c && t, "cache and table are needed");
  RXMET_CHECK_ARG(c->dim == 64 || c->dim == 128 || c->dim == 192 || c->dim == 256,
                  "head dimension must be 64, 128, 192 or 256");
  RXMET_CHECK_ARG(c->page_size == 16 || c->page_size == 32 || c->page_size == 64 ||
                      c->page_size == 128,
                  "page size must be 16, 32, 64 or 128");
  RXMET_CHECK_ARG(c->heads >= 1 && c->heads <= 16384, "heads must be between 1 and 16384");
  RXMET_CHECK_ARG(c->pages >= 1 && c->pages <= INT32_MAX, "pages must be between 1 and 2^31 - 1");
  RXMET_CHECK_ARG(c->k && c->v && c->k_scale && c->v_scale, "the cache has a null pointer");
  RXMET_CHECK_ARG((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) % 16 == 0,
                  "the cache's codes must be aligned to 16 bytes");
  RXMET_CHECK_ARG(t->seqs >= 0 && t->seqs <= 65535, "at most 65535 sequences");
  // a tensor without elements has no address: no sequences need no ids
  RXMET_CHECK_ARG(t->cols >= 1 && (t->ids || t->seqs == 0), "the block table is empty");
  return 0;
}

}  // namespace dec
}  // namespace rxmet

using namespace rxmet;
using namespace rxmet::dec;

extern "C" int rxmet_kv_append(const rxmet_kv_cache *cache, const rxmet_kv_table *table,
                               const int32_t *lengths, const int32_t *cu_new, int64_t tokens,
                               int64_t max_new, const void *key, int64_t key_stride_t,
                               int64_t key_stride_h, const void *value, int64_t value_stride_t,
                               int64_t value_stride_h, int32_t dtype, void *stream) {
  if (int rc = check_cache(cache, table)) return rc;
  RXMET_CHECK_ARG(dtype == RXMET_QDQ_F32 || dtype == RXMET_QDQ_F16 || dtype == RXMET_QDQ_BF16,
                  "element type must be fp32, fp16 or bf16");
  RXMET_CHECK_ARG(tokens >= 0 && max_new >= 0, "tokens and max_new must be >= 0");
  RXMET_CHECK_ARG(cu_new || tokens == table->seqs, "without cu_new there is one token a sequence");
  if (tokens == 0 || table->seqs == 0) return 0;
  RXMET_CHECK_ARG(lengths && key && value, "lengths, key and value are needed");
  const AppendArgs a{{*cache, *table}, lengths, cu_new, tokens, {key, value},
                     {key_stride_t, value_stride_t}, {key_stride_h, value_stride_h}};
  // n >= 1 tokens touch at most (n + P - 2) / P + 1 pages
  const int64_t pages = (max_new + cache->page_size - 2) / cache->page_size + 1;
  const dim3 grid(2 * cache->heads, static_cast<unsigned>(pages < 65535 ? pages : 65535),
                  table->seqs);
  auto st = static_cast<hipStream_t>(stream);
  prof::Scope scope("kv_append", st);
  with_type(dtype, [&](auto t) {
    with_page_shape(*cache, [&](auto d, auto p) {
      kv_append<decltype(t), d.value, p.value><<<grid, 256, 0, st>>>(a);
    });
  });
  RXMET_CHECK_LAUNCH();
  return 0;
}

extern "C" int rxmet_kv_read(const rxmet_kv_cache *cache, const rxmet_kv_table *table,
                             const int32_t *first, const int32_t *cu, int64_t tokens,
                             int64_t max_tokens, void *key, void *value, int32_t dtype,
                             void *stream) {
  if (int rc = check_cache(cache, table)) return rc;
  RXMET_CHECK_ARG(dtype == RXMET_QDQ_F32 || dtype == RXMET_QDQ_F16 || dtype == RXMET_QDQ_BF16,
                  "element type must be fp32, fp16 or bf16");
  RXMET_CHECK_ARG(tokens >= 0 && max_tokens >= 0, "tokens and max_tokens must be >= 0");
  if (tokens == 0 || table->seqs == 0) return 0;
  RXMET_CHECK_ARG(first && cu && key && value, "first, cu, key and value are needed");
  const ReadArgs a{{*cache, *table}, first, cu, tokens, {key, value}};
  const int64_t pages = (max_tokens + cache->page_size - 2) / cache->page_size + 1;
  const dim3 grid(2 * cache->heads, static_cast<unsigned>(pages < 65535 ? pages : 65535),
                  table->seqs);
  auto st = static_cast<hipStream_t>(stream);
  prof::Scope scope("kv_read", st);
  with_type(dtype, [&](auto t) {
    with_page_shape(*cache, [&](auto d, auto p) {
      kv_read<decltype(t), d.value, p.value><<<grid, 256, 0, st>>>(a);
    });
  });
  RXMET_CHECK_LAUNCH();
  return 0;
}

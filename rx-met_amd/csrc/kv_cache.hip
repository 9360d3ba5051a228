// kv_cache.hip — the paged int8 cache of keys and values: new tokens in, values out.
//
// One scale covers a page's tokens of one head.  A page that new tokens enter gets the scale
// s' = max(max|new| / 127, s), s its scale so far if it holds older tokens of the sequence; where s' > s
// the older codes are moved to the new grid, rint(c * s / s').  Keys lie token by token, values
// dimension by dimension (each dimension's tokens side by side): both are what a lane of the
// attention's matrix instructions reads as 16 consecutive bytes.
//
// A workgroup owns a page's keys or values of one head, in pieces of 16 bytes: 16 dimensions of a
// token, or 16 tokens of a dimension.  No two workgroups write the same bytes, and the older codes are
// read only where they move or share a piece with a new token.
//
// Bound: HBM traffic for prompts (each new token read, its codes written); for single tokens the
// launch and two dependent reads.
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

__device__ __forceinline__ float block_max(float v) {
  __shared__ float s[4];
  v = wave_max(v);
  __syncthreads();  // the last page's maxima have been read
  if (threadIdx.x % kWave == 0) s[threadIdx.x / kWave] = v;
  __syncthreads();
  return nan_max(nan_max(s[0], s[1]), nan_max(s[2], s[3]));
}

template <typename T>
__global__ __launch_bounds__(256) void kv_append(const AppendArgs a) {
  const int P = a.g.c.page_size, D = a.g.c.dim, b = blockIdx.y;
  const int which = blockIdx.z & 1, head = blockIdx.z >> 1;
  const int64_t start = a.lengths[b];
  const int64_t row0 = a.cu ? a.cu[b] : b;
  int64_t count = a.cu ? a.cu[b + 1] - row0 : 1;
  if (start < 0 || row0 < 0) return;
  if (count > a.tokens - row0) count = a.tokens - row0;
  if (count <= 0) return;
  const int64_t first = start / P, last = (start + count - 1) / P;
  int8_t *pool = which ? a.g.c.v : a.g.c.k;
  float *scales = which ? a.g.c.v_scale : a.g.c.k_scale;
  const T *x = static_cast<const T *>(a.x[which]) + head * a.stride_h[which];
  for (int64_t p = first + blockIdx.x; p <= last; p += gridDim.x) {
    const int64_t page = page_of(a.g, b, p);
    if (page < 0) continue;
    // new tokens stand in slots s0..s1-1, older ones below s0
    const int s0 = static_cast<int>(p == first ? start - p * P : 0);
    const int s1 = static_cast<int>(p == last ? start + count - p * P : P);
    const T *xp = x + (row0 + p * P - start) * a.stride_t[which];  // slot 0's token (may lie before x)
    const int64_t at = page * a.g.c.heads + head;
    int8_t *codes = pool + at * P * D;
    const int vecs = (s1 - s0) * (D / 8);
    float top = 0.0f;
    for (int i = threadIdx.x; i < vecs; i += 256) {
      float f[8];
      load8(xp + (s0 + i / (D / 8)) * a.stride_t[which] + i % (D / 8) * 8, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) top = nan_max(top, fabsf(f[e]));
    }
    const float was = s0 > 0 ? scales[at] : 0.0f;
    top = block_max(top);
    // block_max's barriers stand between every thread's read of the old scale and this write
    const bool good = top <= 3.402823466e38f && was == was;
    const float fresh = fmaxf(top, kFloor) * kInv127;
    const float scale = good ? fmaxf(fresh, was) : nanf32();
    const float inv = good ? 1.0f / scale : 0.0f;
    const float ratio = good ? was * inv : 0.0f;
    const bool moves = s0 > 0 && !(scale == was);
    if (threadIdx.x == 0) scales[at] = scale;
    // pieces: keys (slot, 16 dimensions), values (16 slots, dimension)
    const int pieces = P * D / 16;
    for (int i = threadIdx.x; i < pieces; i += 256) {
      int lo, hi, off;  // slots of the piece, its bytes' place
      if (which == 0) {
        lo = i / (D / 16), hi = lo + 1, off = i * 16;
      } else {
        const int d = i % D, g = i / D;
        lo = g * 16, hi = lo + 16, off = d * P + lo;
      }
      const bool has_new = lo < s1 && hi > s0, has_old = lo < s0;
      if (!(has_new || (has_old && moves))) continue;
      unsigned w[4] = {};
      if (has_old) {
        __builtin_memcpy(w, codes + off, 16);
        if (moves) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            w[k] = code_bytes4(code_value(w[k], 0) * ratio, code_value(w[k], 1) * ratio,
                               code_value(w[k], 2) * ratio, code_value(w[k], 3) * ratio);
        }
      }
      if (has_new) {
        if (which == 0) {
          const T *q = xp + lo * a.stride_t[0] + i % (D / 16) * 16;
          float f[8];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            load8(q + 8 * k, f);
            w[2 * k] = code_bytes4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
            w[2 * k + 1] = code_bytes4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv);
          }
        } else {
          const T *q = xp + i % D;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int s = lo + e;
            if (s >= s0 && s < s1) {
              const float f = static_cast<float>(q[s * a.stride_t[1]]);
              const int sh = 8 * (e % 4);
              w[e / 4] = (w[e / 4] & ~(0xffu << sh)) | code_byte(f * inv) << sh;
            }
          }
        }
      }
      __builtin_memcpy(codes + off, w, 16);
    }
  }
}

struct ReadArgs {
  Pages g;
  const int32_t *first, *cu;
  int64_t tokens;
  void *out[2];
};

template <typename T>
__global__ __launch_bounds__(256) void kv_read(const ReadArgs a) {
  const int P = a.g.c.page_size, D = a.g.c.dim, b = blockIdx.y;
  const int which = blockIdx.z & 1, head = blockIdx.z >> 1;
  const int64_t start = a.first[b], row0 = a.cu[b];
  int64_t count = a.cu[b + 1] - row0;
  if (row0 < 0) return;
  if (count > a.tokens - row0) count = a.tokens - row0;
  if (count <= 0) return;
  const int64_t first = start >= 0 ? start / P : -((-start + P - 1) / P);
  const int64_t last = (start + count - 1) / P;
  const int64_t row = static_cast<int64_t>(a.g.c.heads) * D;
  for (int64_t p = first + blockIdx.x; p <= last; p += gridDim.x) {
    const int64_t page = page_of(a.g, b, p);
    const int s0 = static_cast<int>(p == first ? start - p * P : 0);
    const int s1 = static_cast<int>(p == last ? start + count - p * P : P);
    const int64_t at = (page < 0 ? 0 : page) * a.g.c.heads + head;
    const int8_t *codes = (which ? a.g.c.v : a.g.c.k) + at * P * D;
    const float scale = page < 0 ? nanf32() : (which ? a.g.c.v_scale : a.g.c.k_scale)[at];
    T *out = static_cast<T *>(a.out[which]) + head * D;
    for (int i = threadIdx.x; i < P * D / 16; i += 256) {
      const int lo = which == 0 ? i / (D / 16) : i / D * 16;
      if (lo >= s1 || lo + (which == 0 ? 1 : 16) <= s0) continue;
      unsigned w[4] = {};
      if (page >= 0)
        __builtin_memcpy(w, codes + (which == 0 ? i * 16 : i % D * P + lo), 16);
      if (which == 0) {
        T *q = out + (row0 + p * P + lo - start) * row + i % (D / 16) * 16;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float f[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = code_value(w[2 * k + e / 4], e % 4) * scale;
          store8(q + 8 * k, f);
        }
      } else {
        T *q = out + (row0 + p * P - start) * row + i % D;
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (lo + e >= s0 && lo + e < s1)
            q[(lo + e) * row] = static_cast<T>(code_value(w[e / 4], e % 4) * scale);
      }
    }
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
  RXMET_CHECK_ARG(t->cols >= 1 && t->ids, "the block table is empty");
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
  const dim3 grid(static_cast<unsigned>(pages < 65536 ? pages : 65536), table->seqs,
                  2 * cache->heads);
  auto st = static_cast<hipStream_t>(stream);
  prof::Scope scope("kv_append", st);
  with_type(dtype, [&](auto t) { kv_append<decltype(t)><<<grid, 256, 0, st>>>(a); });
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
  const dim3 grid(static_cast<unsigned>(pages < 65536 ? pages : 65536), table->seqs,
                  2 * cache->heads);
  auto st = static_cast<hipStream_t>(stream);
  prof::Scope scope("kv_read", st);
  with_type(dtype, [&](auto t) { kv_read<decltype(t)><<<grid, 256, 0, st>>>(a); });
  RXMET_CHECK_LAUNCH();
  return 0;
}

// kv_cache.h — pages of the int8 cache as kernels see them (kv_cache.hip, kv_attention.hip).
#pragma once

#include "decoder_common.h"

namespace rxmet {
namespace dec {

struct Pages {
  rxmet_kv_cache c;
  rxmet_kv_table t;
};

// Page of the sequence's p-th page of tokens, or -1 where there is none.
__device__ __forceinline__ int64_t page_of(const Pages &g, int b, int64_t p) {
  if (p < 0 || p >= g.t.cols) return -1;
  const int32_t id = g.t.ids[b * g.t.stride + p];
  return id >= 0 && id < g.c.pages ? id : -1;
}

// Refuses what the kernels do not take; 0 or a negative status with a message.
int check_cache(const rxmet_kv_cache *c, const rxmet_kv_table *t);

}  // namespace dec
}  // namespace rxmet

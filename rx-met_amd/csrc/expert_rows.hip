// expert_rows.hip — the entries in the experts' order, a token's rows added up, and the gradient of that.
#include "../../include/rxmet_experts.h"
#include "decoder_common.h"

namespace rxmet {
namespace dec {
namespace {

// ---------------------------------------------------------------------------------------------
// Order by expert: a counting sort that keeps the entries' order.  A workgroup has kChunk entries; its
// counts go to memory, and a second launch adds up the counts of the chunks before, ranks the entries of
// its chunk and writes both directions.  Up to kAlone entries one workgroup does it all in one launch;
// above kFewChunks chunks, whose counts every chunk would read, a launch in between adds them up once.
// Bound: launches and trips to memory behind each other ([16384, 8] of 256 experts: 11 us, 2.4 + 9.2 of kernels,
// 1.6 MB; [16, 8]: 3.6 us of kernel; 2^26 entries 1.8 ms).
struct GroupArgs {
  const int32_t *experts;
  int64_t count;
  int E, chunks;
  int32_t *offsets, *entries, *places;
  int32_t *counts;  // [chunks + 1, E + 1]; added up: of the chunks before, and of all in the last row
};

constexpr int kChunk = 1024, kGroupWaves = kChunk / kWave;
constexpr int64_t kAlone = 4096;
constexpr int64_t kFewChunks = 128;
constexpr int kBins = RXMET_EXPERTS_MAX + 1;  // the last one: entries of no expert

__device__ __forceinline__ int bin_of(const GroupArgs &a, int64_t i) {
  const int32_t e = a.experts[i];
  return e >= 0 && e < a.E ? e : a.E;
}

__global__ __launch_bounds__(kChunk) void group_count(const GroupArgs a) {
  __shared__ int s_count[kBins];
  for (int b = threadIdx.x; b <= a.E; b += kChunk) s_count[b] = 0;
  __syncthreads();
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kChunk + threadIdx.x;
  if (i < a.count) atomicAdd(&s_count[bin_of(a, i)], 1);
  __syncthreads();
  for (int b = threadIdx.x; b <= a.E; b += kChunk)
    a.counts[static_cast<int64_t>(blockIdx.x) * (a.E + 1) + b] = s_count[b];
}

// The counts of each bin's chunks before every chunk: 64 bins a workgroup, 16 threads a bin, each with
// a run of the chunks.
__global__ __launch_bounds__(1024) void group_sum(const GroupArgs a) {
  __shared__ int s_run[16][64];
  const int bins = a.E + 1, b = blockIdx.x * 64 + threadIdx.x % 64, r = threadIdx.x / 64;
  const int share = (a.chunks + 15) / 16, from = r * share, to = from + share < a.chunks ? from + share : a.chunks;
  int n = 0;
  if (b < bins)
#pragma unroll 8
    for (int c = from; c < to; ++c) n += a.counts[c * bins + b];
  s_run[r][threadIdx.x % 64] = n;
  __syncthreads();
  int before = 0;
  for (int v = 0; v < r; ++v) before += s_run[v][threadIdx.x % 64];
  if (b >= bins) return;
#pragma unroll 8
  for (int c = from; c < to; ++c) {
    const int m = a.counts[c * bins + b];
    a.counts[c * bins + b] = before;
    before += m;
  }
  if (r == 15) a.counts[a.chunks * bins + b] = before;
}

// ALONE: one workgroup has all entries and counts them first.  SUMMED: the chunks' counts are added up.
template <bool ALONE, bool SUMMED>
__global__ __launch_bounds__(kChunk) void group_place(const GroupArgs a) {
  __shared__ int s_all[kBins], s_at[kBins];  // entries of a bin; where its next one goes
  __shared__ unsigned short s_wave[kGroupWaves][kBins];
  __shared__ int s_sum[kGroupWaves];
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave, bins = a.E + 1;
  for (int b = tid; b < bins; b += kChunk) s_all[b] = s_at[b] = 0;
  __syncthreads();
  if (ALONE) {
    for (int64_t i = tid; i < a.count; i += kChunk) atomicAdd(&s_all[bin_of(a, i)], 1);
  } else if (SUMMED) {
    for (int b = tid; b < bins; b += kChunk) {
      s_all[b] = a.counts[a.chunks * bins + b];
      s_at[b] = a.counts[static_cast<int>(blockIdx.x) * bins + b];
    }
  } else {
    // each bin's column of counts by as many threads as there are
    const int columns = bins < kChunk ? bins : kChunk, share = kChunk / columns;
    if (tid < columns * share)
      for (int b = tid % columns; b < bins; b += columns) {
        int all = 0, mine = 0;
#pragma unroll 8
        for (int c = tid / columns; c < a.chunks; c += share) {
          const int n = a.counts[c * bins + b];
          all += n;
          mine += c < static_cast<int>(blockIdx.x) ? n : 0;
        }
        atomicAdd(&s_all[b], all);
        atomicAdd(&s_at[b], mine);
      }
  }
  __syncthreads();
  // places before each bin; bins beyond the threads go around again
  int before = 0;
  for (int base = 0; base < bins; base += kChunk) {
    const int b = base + tid, n = b < bins ? s_all[b] : 0;
    int up = n;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int o = __shfl_up(up, d, kWave);
      if (lane >= d) up += o;
    }
    if (lane == kWave - 1) s_sum[wave] = up;
    __syncthreads();
    int first = before + up - n;
    for (int v = 0; v < kGroupWaves; ++v) {
      if (v < wave) first += s_sum[v];
      before += s_sum[v];
    }
    if (b < bins) {
      s_at[b] += first;
      if (blockIdx.x == 0) a.offsets[b] = first;  // of the last bin: where the experts' entries end
    }
    __syncthreads();
  }
  const int64_t from = static_cast<int64_t>(blockIdx.x) * kChunk, to = ALONE ? a.count : from + 1;
  for (int64_t base = from; base < to; base += kChunk) {
    for (int b = lane; b < bins; b += kWave) s_wave[wave][b] = 0;
    const int64_t i = base + tid;
    const int bin = i < a.count ? bin_of(a, i) : bins;  // lanes behind the end stand apart
    // lanes of the same bin
    unsigned long long same = ~0ull;
    for (int bit = 1; bit <= bins; bit <<= 1) {
      const unsigned long long set = __ballot((bin & bit) != 0);
      same &= bin & bit ? set : ~set;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    __syncthreads();
    if (bin < bins && rank == 0) s_wave[wave][bin] = static_cast<unsigned short>(__popcll(same));
    __syncthreads();
    for (int b = tid; b < bins; b += kChunk) {  // counts of the waves before; the bin moves on
      int n = 0;
      int c[kGroupWaves];
#pragma unroll
      for (int v = 0; v < kGroupWaves; ++v) c[v] = s_wave[v][b];
#pragma unroll
      for (int v = 0; v < kGroupWaves; ++v) {
        s_wave[v][b] = static_cast<unsigned short>(n);
        n += c[v];
      }
      s_all[b] = s_at[b];
      s_at[b] += n;
    }
    __syncthreads();
    if (bin < bins) {
      const int place = s_all[bin] + s_wave[wave][bin] + rank;
      a.entries[place] = static_cast<int32_t>(i);
      a.places[i] = bin < a.E ? place : -1;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------
// Rows added up: a run of threads has a token's row, eight columns a thread, and adds the rows of
// its entries in fp32 in their order.  Bound: the rows' bytes.  PAST: y is larger than the memory's 256 MB
// cache and is read past it ([65536, 2048]: 71 us, 76 through the caches; 25.6 us become 31.9 for 67 MB).
struct CombineArgs {
  const int32_t *entries, *places;
  int64_t tokens, rows;
  int top_k;
  const void *y, *res, *d_out;
  int64_t y_stride, res_stride, d_stride;
  const float *weights;
  void *out, *d_y;
  float *d_weights;
  int64_t N;
  int shift;  // 2^shift threads have a row
  unsigned blocks;  // workgroups of the tokens; those behind them clear rows of the gradient
};

template <typename T>
__device__ __forceinline__ void load_any(const T *p, int64_t left, float (&f)[8]) {
  if (left >= 8)
    load8(p, f);
  else
    load8_part(p, static_cast<int>(left), f);
}
// load8 of what is read once and does not stay in the caches
template <typename T>
__device__ __forceinline__ void load8_past(const T *p, float (&f)[8]) {
  Vec8<T> u;
#pragma unroll
  for (int k = 0; k < static_cast<int>(sizeof(u) / 16); ++k) {
    const v4i_any w = __builtin_nontemporal_load(reinterpret_cast<const v4i_any *>(p) + k);
    __builtin_memcpy(reinterpret_cast<char *>(&u) + 16 * k, &w, 16);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = static_cast<float>(u.v[e]);
}
template <typename T>
__device__ __forceinline__ void store_any(T *p, int64_t left, const float (&f)[8]) {
  if (left >= 8)
    store8(p, f);
  else
    store8_part(p, static_cast<int>(left), f);
}

template <typename T, bool PAST>
__global__ __launch_bounds__(256) void combine_rows(const CombineArgs a) {
  const int width = 1 << a.shift, lane = threadIdx.x & (width - 1);
  const int64_t t = static_cast<int64_t>(blockIdx.x) * (256 >> a.shift) + (threadIdx.x >> a.shift);
  if (t >= a.tokens) return;
  const int32_t *place = a.places + t * a.top_k;
  const float *w = a.weights + t * a.top_k;
  for (int64_t n = 8 * lane; n < a.N; n += 8 * width) {
    const int64_t left = a.N - n;
    float sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 4
    for (int j = 0; j < a.top_k; ++j) {
      const int64_t p = place[j];
      if (p < 0 || p >= a.rows) continue;
      float v[8];
      const T *row = static_cast<const T *>(a.y) + p * a.y_stride + n;
      if (PAST && left >= 8)
        load8_past(row, v);
      else
        load_any(row, left, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] = __builtin_fmaf(w[j], v[e], sum[e]);
    }
    if (a.res) {
      float v[8];
      load_any(static_cast<const T *>(a.res) + t * a.res_stride + n, left, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e] += v[e];
    }
    store_any(static_cast<T *>(a.out) + t * a.N + n, left, sum);
  }
}

// The gradient: the threads of a token read its gradient once for up to TOGETHER of its rows, write theirs
// and add up their products with y.  Rows that no entry has as its place (behind the experts' last, or taken away by
// the caller) are cleared.  Such a row's entry of `entries` is not placed there.  Up to kScan rows, where a launch
// costs most (2 to 4 us of a pass that the host bounds), waves of the same launch clear those that no place names; above,
// where that would read all places too often, a launch ahead clears all whose entry is placed elsewhere, and what is
// placed there against `entries` is written after.  Bound: the rows' bytes, read and
// written ([65536, 2041] bf16, a tenth of no expert: 7 + 125 us, 541 MB, 4.1 TB/s).
constexpr int kScan = 4096;
constexpr int kClearRows = 16;  // rows that a wave looks at, far from each other: those to clear lie together

// Whether no entry that `entries` knows of has row i as its place.
__device__ __forceinline__ bool unplaced(const CombineArgs &a, int64_t i) {
  const int64_t entry = a.entries[i];
  return entry < 0 || entry >= a.rows || a.places[entry] != i;
}

template <typename T>
__device__ __forceinline__ void clear_row(const CombineArgs &a, int64_t i, int lane) {
  T *row = static_cast<T *>(a.d_y) + i * a.N;
  // 16 bytes at a time from where memory's lines are cut, the ends by element (from the row's start: 12 us)
  const int64_t lead = (16 - reinterpret_cast<uintptr_t>(row) % 16) % 16 / sizeof(T), first = lead < a.N ? lead : a.N;
  const int64_t pieces = (a.N - first) * static_cast<int64_t>(sizeof(T)) / 16, last = first + pieces * 16 / sizeof(T);
  const v4i_any none = {0, 0, 0, 0};
  for (int64_t n = lane; n < pieces; n += kWave) __builtin_memcpy(reinterpret_cast<char *>(row + first) + 16 * n, &none, 16);
  if (lane < first) row[lane] = static_cast<T>(0.0f);
  if (last + lane < a.N) row[last + lane] = static_cast<T>(0.0f);
}

template <typename T>
__global__ __launch_bounds__(256) void clear_rows(const CombineArgs a) {
  const int64_t waves = (a.rows + kClearRows - 1) / kClearRows;
  const int64_t wave = static_cast<int64_t>(blockIdx.x) * (256 / kWave) + threadIdx.x / kWave;
  const int lane = threadIdx.x % kWave;
  if (wave >= waves) return;
  const int64_t i = wave + waves * lane;
  const bool clear = lane < kClearRows && i < a.rows && unplaced(a, i);
  for (unsigned long long left = __ballot(clear); left != 0; left &= left - 1)
    clear_row<T>(a, wave + waves * (__ffsll(left) - 1), lane);
}

template <typename T, int TOGETHER>
__global__ __launch_bounds__(256) void combine_backward(const CombineArgs a) {
  __shared__ float s_dot[4][TOGETHER];
  const int width = 1 << a.shift, at = threadIdx.x & (width - 1), wave = threadIdx.x / kWave;
  if (blockIdx.x >= a.blocks) {  // a wave a row
    const int64_t i = static_cast<int64_t>(blockIdx.x - a.blocks) * (256 / kWave) + wave;
    const int lane = threadIdx.x % kWave;
    if (i >= a.rows || !unplaced(a, i)) return;
    bool named = false;
#pragma unroll 8
    for (int64_t x = lane; x < a.rows; x += kWave) named |= a.places[x] == i;
    if (!__any(named)) clear_row<T>(a, i, lane);
    return;
  }
  const int64_t wanted = static_cast<int64_t>(blockIdx.x) * (256 >> a.shift) + (threadIdx.x >> a.shift);
  const int64_t t = wanted < a.tokens ? wanted : a.tokens - 1;  // (all threads meet below)
  const int32_t *place = a.places + t * a.top_k;
  // written past the caches only where rows start on 16 bytes ([65536, 2041]: 273 us so, 257 otherwise)
  const bool whole = (a.N * sizeof(T) | reinterpret_cast<uintptr_t>(a.d_y)) % 16 == 0;
  for (int j0 = 0; j0 < a.top_k; j0 += TOGETHER) {
    int64_t p[TOGETHER];
    float w[TOGETHER], dot[TOGETHER];
#pragma unroll
    for (int j = 0; j < TOGETHER; ++j) {
      p[j] = j0 + j < a.top_k && wanted < a.tokens ? place[j0 + j] : -1;
      if (p[j] >= a.rows) p[j] = -1;
      w[j] = j0 + j < a.top_k ? a.weights[t * a.top_k + j0 + j] : 0.0f;
      dot[j] = 0;
    }
    for (int64_t n = 8 * at; n < a.N; n += 8 * width) {
      const int64_t left = a.N - n;
      float g[8];
      load_any(static_cast<const T *>(a.d_out) + t * a.d_stride + n, left, g);
#pragma unroll
      for (int j = 0; j < TOGETHER; ++j) {
        if (p[j] < 0) continue;
        if (a.d_weights) {
          float v[8];
          load_any(static_cast<const T *>(a.y) + p[j] * a.y_stride + n, left, v);
#pragma unroll
          for (int e = 0; e < 8; ++e) dot[j] = __builtin_fmaf(g[e], v[e], dot[j]);
        }
        if (a.d_y) {
          float d[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) d[e] = w[j] * g[e];
          T *out = static_cast<T *>(a.d_y) + p[j] * a.N + n;
          if (left < 8)
            store8_part(out, static_cast<int>(left), d);
          else if (whole)
            stream_out8(out, d);
          else
            store8(out, d);
        }
      }
    }
    if (!a.d_weights) continue;
#pragma unroll
    for (int j = 0; j < TOGETHER; ++j)
      for (int d = (width < kWave ? width : kWave) / 2; d > 0; d >>= 1) dot[j] += __shfl_xor(dot[j], d, kWave);
    if (width > kWave) {  // a token's waves
      __syncthreads();
      if (threadIdx.x % kWave == 0)
#pragma unroll
        for (int j = 0; j < TOGETHER; ++j) s_dot[wave][j] = dot[j];
      __syncthreads();
#pragma unroll
      for (int j = 0; j < TOGETHER; ++j) {
        dot[j] = 0;
        for (int v = wave & ~(width / kWave - 1), n = 0; n < width / kWave; ++n) dot[j] += s_dot[v + n][j];
      }
    }
    if (at == 0 && wanted < a.tokens)
#pragma unroll
      for (int j = 0; j < TOGETHER; ++j)
        if (j0 + j < a.top_k) a.d_weights[t * a.top_k + j0 + j] = dot[j];
  }
}

// Threads of a row, as a power of two: eight columns each, at most `most`.
int shift_for(int64_t N, int most) {
  int shift = 0;
  while (shift < most && (8LL << shift) < N) ++shift;
  return shift;
}

int check_groups(const rxmet_expert_groups *g, int64_t N, int32_t dtype) {
  RXMET_CHECK_ARG(g != nullptr, "the groups are missing");
  RXMET_CHECK_ARG(g->experts >= 1 && g->experts <= RXMET_EXPERTS_MAX, "there must be 1 to 1024 experts");
  RXMET_CHECK_ARG(g->top_k >= 1 && g->top_k <= RXMET_TOP_K_MAX, "top_k must be between 1 and 64");
  RXMET_CHECK_ARG(g->tokens >= 0 && g->tokens <= 1 << 23, "there must be at most 2^23 tokens");
  RXMET_CHECK_ARG(N >= 1 && N <= 1 << 24, "N must be between 1 and 2^24");
  RXMET_CHECK_ARG(dtype == RXMET_QDQ_F32 || dtype == RXMET_QDQ_F16 || dtype == RXMET_QDQ_BF16,
                  "element type must be fp32, fp16 or bf16");
  return 0;
}

}  // namespace
}  // namespace dec
}  // namespace rxmet

using namespace rxmet;
using namespace rxmet::dec;

extern "C" int64_t rxmet_group_experts_workspace_bytes(int64_t count, int32_t num_experts) {
  if (count <= kAlone || num_experts < 1) return 0;
  return (cdiv(count, kChunk) + 1) * (num_experts + 1) * 4;
}

extern "C" int rxmet_group_experts(const int32_t *experts, int64_t count, int32_t num_experts,
                                   int32_t *offsets, int32_t *entries, int32_t *places,
                                   void *workspace, void *stream) {
  RXMET_CHECK_ARG(num_experts >= 1 && num_experts <= RXMET_EXPERTS_MAX, "there must be 1 to 1024 experts");
  RXMET_CHECK_ARG(count >= 0 && count <= 1 << 26, "there must be at most 2^26 entries");
  RXMET_CHECK_ARG(offsets != nullptr, "offsets are needed");
  RXMET_CHECK_ARG(count == 0 || (experts && entries && places), "experts, entries and places are needed");
  RXMET_CHECK_ARG(count <= kAlone || workspace, "this call needs a workspace");
  RXMET_CHECK_ARG(reinterpret_cast<uintptr_t>(workspace) % 4 == 0, "the workspace must be aligned to 4 bytes");
  auto st = static_cast<hipStream_t>(stream);
  prof::Scope scope("group_experts", st);
  const int chunks = static_cast<int>(cdiv(count, kChunk));
  const GroupArgs a{experts, count, num_experts, chunks, offsets, entries, places,
                    static_cast<int32_t *>(workspace)};
  if (count <= kAlone) {
    group_place<true, false><<<1, kChunk, 0, st>>>(a);
  } else {
    group_count<<<chunks, kChunk, 0, st>>>(a);
    if (chunks <= kFewChunks) {
      group_place<false, false><<<chunks, kChunk, 0, st>>>(a);
    } else {
      group_sum<<<static_cast<unsigned>(cdiv(num_experts + 1, 64)), 1024, 0, st>>>(a);
      group_place<false, true><<<chunks, kChunk, 0, st>>>(a);
    }
  }
  RXMET_CHECK_LAUNCH();
  return 0;
}

extern "C" int rxmet_experts_combine(const rxmet_expert_groups *g, const void *y, int64_t y_stride,
                                     const float *weights, const void *residual,
                                     int64_t residual_stride, void *out, int64_t N, int32_t dtype,
                                     void *stream) {
  if (const int rc = check_groups(g, N, dtype)) return rc;
  if (g->tokens == 0) return 0;
  RXMET_CHECK_ARG(g->places && y && weights && out, "places, y, weights and out are needed");
  const int shift = shift_for(N, 8);
  const CombineArgs a{g->entries, g->places, g->tokens, g->tokens * g->top_k, g->top_k, y,
                      residual, nullptr, y_stride, residual_stride, 0, weights, out, nullptr, nullptr, N, shift, 0};
  auto st = static_cast<hipStream_t>(stream);
  prof::Scope scope("experts_combine", st);
  with_type(dtype, [&](auto t) {
    using T = decltype(t);
    const unsigned grid = static_cast<unsigned>(cdiv(g->tokens, 256 >> shift));
    if (a.rows * N * static_cast<int64_t>(sizeof(T)) >= 256LL << 20)
      combine_rows<T, true><<<grid, 256, 0, st>>>(a);
    else
      combine_rows<T, false><<<grid, 256, 0, st>>>(a);
  });
  RXMET_CHECK_LAUNCH();
  return 0;
}

extern "C" int rxmet_experts_combine_backward(const rxmet_expert_groups *g, const void *d_out,
                                              int64_t d_out_stride, const void *y, int64_t y_stride,
                                              const float *weights, void *d_y, float *d_weights,
                                              int64_t N, int32_t dtype, void *stream) {
  if (const int rc = check_groups(g, N, dtype)) return rc;
  if (g->tokens == 0 || (!d_y && !d_weights)) return 0;
  RXMET_CHECK_ARG(g->places && d_out && weights, "places, d_out and weights are needed");
  RXMET_CHECK_ARG(!d_y || g->entries, "d_y needs the groups' entries");
  RXMET_CHECK_ARG(!d_weights || y, "d_weights needs y");
  // a wave has a token, so that its sums over N meet without a barrier ([8192, 2041] x 8: 225 us, a workgroup
  // 271); a workgroup where tokens are few ([2048, 8192] x 8: 167 us, a wave 217)
  const int shift = shift_for(N, g->tokens >= 4096 ? 6 : 8);
  const CombineArgs a{g->entries, g->places, g->tokens, g->tokens * g->top_k, g->top_k, y,
                      nullptr, d_out, y_stride, 0, d_out_stride, weights, nullptr, d_y, d_weights, N, shift,
                      static_cast<unsigned>(cdiv(g->tokens, 256 >> shift))};
  auto st = static_cast<hipStream_t>(stream);
  prof::Scope scope("experts_combine_backward", st);
  with_type(dtype, [&](auto t) {
    using T = decltype(t);
    if (d_y && a.rows > kScan)
      clear_rows<T><<<static_cast<unsigned>(cdiv(cdiv(a.rows, kClearRows), 256 / kWave)), 256, 0, st>>>(a);
    const unsigned grid = a.blocks + (d_y && a.rows <= kScan ? static_cast<unsigned>(cdiv(a.rows, 256 / kWave)) : 0);
    if (g->top_k <= 2)
      combine_backward<T, 2><<<grid, 256, 0, st>>>(a);
    else if (g->top_k <= 4)
      combine_backward<T, 4><<<grid, 256, 0, st>>>(a);
    else
      combine_backward<T, 8><<<grid, 256, 0, st>>>(a);
  });
  RXMET_CHECK_LAUNCH();
  return 0;
}

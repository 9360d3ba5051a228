// expert_linear.hip — int8 product with a weight for each expert, rows gathered or in the experts' order.
//
// Mathematics.  Of place i of expert e, with r its row of codes: acc[n] = sum_k x[r, k] w[e, n, k] exact in
// int32, y[i, n] = act(acc * sx[r] * sw[e, n] + b[e, n]); gated: act(gate) * value, the gate from weight
// row n and the value from row N + n, both in the same lane's hands.  The epilogue is fp32 and rounds once.
//
// The experts' rows are known on the device alone: a launch is sized for the most tiles that the entries
// can need, and each workgroup finds its tile in the offsets.
//
// Bound and measured.  Few rows: the weights' bytes (16 tokens of 8 of 64 experts, gated [2048, 2048]: 268 MB
// of which 56 experts' are read, 46 us warm, 5.1 TB/s; 57 with other inputs in between).  Many: [65536, 2048] of 32
// experts' [2048, 2048] 327 us warm, 1.68 POP/s, gated [4096, 2048] 628 us, 1.75 POP/s; the matrix unit is
// busy for 35 and 41 % of that.  Over K alone (2048 to 4096) the loop runs at 2.0 POP/s, where the library's
// product of 8192^3 without an epilogue reaches 2.1: without its loads it would at 2.9, and they are 64 KB a step and
// CU on their way while one step is multiplied, which LDS has no room to do further ahead.  The rest is
// the tiles' start and end, when the outputs' bytes (268 MB) are written with little to multiply.
#include <type_traits>

#include "../../include/rxmet_experts.h"
#include "../../include/rxmet_selftest.h"
#include "int8_tile.h"

namespace rxmet {
namespace dec {
namespace {

struct ExpertArgs {
  const int32_t *offsets, *entries;
  int64_t tokens, rows;  // rows: places, tokens * top_k
  int top_k, experts, grouped;
  const int8_t *x, *w;
  int64_t x_stride, w_stride, e_stride;
  const float *sx, *sw;
  const void *bias;
  void *y;
  int64_t N;
  int K, gated, act, dtype, past;  // past: y is written past the caches
};

// The places of expert e, kept inside the rows whatever the offsets hold.
__device__ __forceinline__ void places_of(const ExpertArgs &a, int e, int64_t &from, int64_t &to) {
  const int64_t lo = a.offsets[e], hi = a.offsets[e + 1];
  from = lo < 0 ? 0 : lo < a.rows ? lo : a.rows;
  to = hi < from ? from : hi < a.rows ? hi : a.rows;
}

// The row of codes of place i.
__device__ __forceinline__ int64_t row_of(const ExpertArgs &a, int64_t i) {
  if (a.grouped) return i;
  const int64_t t = a.entries[i] / a.top_k;
  return t < 0 ? 0 : t < a.tokens ? t : a.tokens - 1;
}

// silu of outputs in 16 bits: v / (1 + exp(-v)) by the hardware's exponential and reciprocal, 5 instructions instead of
// activate()'s 25 (gated [65536, 2048] of 32 experts: 670 us, 738).  The exponential's argument is rounded to fp32, so
// the result is off by up to |v| + 4 half steps of fp32: below 1 / 100 of the half step of fp16 that it is rounded by.
__device__ __forceinline__ float silu16(float v) {
  return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.44269504088896340736f));
}

// silu of outputs in fp32, off by at most 7 half steps: v u / (1 + u) or v / (1 + u) with u = exp(-|v|), which neither
// overflows nor leaves (0, 1].  u = 2^t (1 + c): t = -|v| / ln 2 rounded, c = -|v| - t ln 2 what that left, ln 2 in two
// parts.  The hardware's 2^t is within 2 half steps, u 3; v u, 1 + u, its reciprocal (an estimate and one step of Newton's
// rule) and the last product take one each.  Below -87 the result may be 0.  14 instructions (the same product: 720 us; by
// activate() 765, by silu16 698).
__device__ __forceinline__ float silu32(float v) {
  const float m = fminf(fabsf(v), 120.0f), t = m * -1.44269504088896340736f;
  const float c = __builtin_fmaf(t, 1.9046542121259336e-9f, __builtin_fmaf(t, -0.693147182464599609375f, -m));
  float u = __builtin_amdgcn_exp2f(t);
  u = __builtin_fmaf(u, c, u);
  const float d = 1.0f + u;
  float q = __builtin_amdgcn_rcpf(d);
  q = __builtin_fmaf(__builtin_fmaf(-d, q, 1.0f), q, q);
  return (v < 0.0f ? v * u : v) * q;
}

// The activation of an output of type T; both kernels take the same, so that a row's result does not go by how
// many there are.
template <typename T>
__device__ __forceinline__ float activated(float v, int act) {
  if (act != RXMET_ACT_SILU) return activate(v, act);
  return std::is_same<T, float>::value ? silu32(v) : silu16(v);
}

// f of a weight row and of a row of codes
__device__ __forceinline__ int wide_turn_w(int row) { return (row >> 1 & 3) | (row >> 2 & 4); }
__device__ __forceinline__ int wide_turn_x(int row) { return row >> 1 & 7; }

// Finishes and writes C consecutive n of place i; v: the sums of the values where gated.
template <typename T, int C>
__device__ __forceinline__ void finish(const ExpertArgs &a, int e, int64_t i, float sx, int64_t n0,
                                       const int (&acc)[C], const int (&val)[C]) {
  const int64_t first = static_cast<int64_t>(e) * a.N * (1 + a.gated) + n0;
  const float *sw = a.sw + first;
  const T *bias = a.bias ? static_cast<const T *>(a.bias) + first : nullptr;
  T *y = static_cast<T *>(a.y) + i * a.N + n0;
  const bool large = is_large(sx);
  auto scaled = [&](int acc, float w, T b) {
    const float v = static_cast<float>(acc) * (large ? w : sx) * (large ? sx : w);
    return bias ? v + static_cast<float>(b) : v;
  };
  struct Vec {
    T v[C];
  };
  if (n0 + C <= a.N) {
    Vec out, b = {}, bv = {};
    float w[C], wv[C];
    __builtin_memcpy(w, sw, sizeof(w));
    if (bias) __builtin_memcpy(&b, bias, sizeof(b));
    if (a.gated) {
      __builtin_memcpy(wv, sw + a.N, sizeof(wv));
      if (bias) __builtin_memcpy(&bv, bias + a.N, sizeof(bv));
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float v = activated<T>(scaled(acc[c], w[c], b.v[c]), a.act);
      if (a.gated) v *= scaled(val[c], wv[c], bv.v[c]);
      out.v[c] = static_cast<T>(v);
    }
    __builtin_memcpy(y, &out, sizeof(out));
  } else {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (n0 + c < a.N) {
        float v = activated<T>(scaled(acc[c], sw[c], bias ? bias[c] : static_cast<T>(0.0f)), a.act);
        if (a.gated) v *= scaled(val[c], sw[a.N + c], bias ? bias[a.N + c] : static_cast<T>(0.0f));
        y[c] = static_cast<T>(v);
      }
  }
}

// f(T{}) for an element type that the host has checked.
template <typename F>
__device__ __forceinline__ void with_type_of(int dtype, F &&f) {
  if (dtype == RXMET_QDQ_BF16)
    f(bf16{});
  else if (dtype == RXMET_QDQ_F16)
    f(f16{});
  else
    f(float{});
}

constexpr int kWide = 128;  // bytes of K in a step: a whole line of each row

// ---------------------------------------------------------------------------------------------
// Few rows of an expert: WK waves have 32 weight rows of one expert (gated: 16 gates and their 16
// values), each every WK-th step of K, and multiply 16 places at a time on mfma 16x16x64.  A wave's steps go memory
// -> LDS without registers, some steps ahead in a ring of its own, so that waves wait for memory and not
// for each other; their sums meet in LDS at the end.  Rows that do not start on 16 bytes (ALIGNED
// false) go from memory into the matrix instruction.
constexpr int kFewRows = 32, kFewPlaces = 16;

template <int WK, bool ALIGNED>
__global__ __launch_bounds__(64 * WK) void experts_few(const ExpertArgs a) {
  constexpr int depth = 4;
  constexpr int bytes = (kFewRows + kFewPlaces) * kWide, loads = bytes / 1024;
  __shared__ __attribute__((aligned(16))) int8_t s[WK][ALIGNED ? depth * bytes : 2048];
  const int width = a.gated ? kFewRows / 2 : kFewRows;
  const int tiles = static_cast<int>((a.N + width - 1) / width);
  const int e = blockIdx.x / tiles;
  int64_t from, to;
  places_of(a, e, from, to);
  if (from >= to) return;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int col = lane % 16, g = lane / 16;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x % tiles) * width;
  auto weight_row = [&](int row) {
    const int64_t n = n0 + (a.gated ? row % 16 : row);
    return a.w + e * a.e_stride + ((n < a.N ? n : a.N - 1) + (a.gated && row >= 16 ? a.N : 0)) * a.w_stride;
  };
  const int whole = a.K / kWide;
  for (int64_t m0 = from; m0 < to; m0 += kFewPlaces) {
    auto code_row = [&](int row) { return a.x + row_of(a, m0 + row < to ? m0 + row : to - 1) * a.x_stride; };
    v4i acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    if constexpr (ALIGNED) {
      // a load takes eight rows; piece p of row r lies at p ^ (r / 2 % 8), for the banks
      const int8_t *src[loads];
#pragma unroll
      for (int j = 0; j < loads; ++j) {
        const int row = 8 * j + lane / 8;
        src[j] = (8 * j < kFewRows ? weight_row(row) : code_row(row - kFewRows)) + (lane % 8 ^ (row >> 1 & 7)) * 16;
      }
      auto issue = [&](int step, int slot) {
#pragma unroll
        for (int j = 0; j < loads; ++j) load_to_lds(src[j] + step * kWide, &s[wave][slot * bytes + 1024 * j]);
      };
      const int mine = whole > wave ? (whole - wave + WK - 1) / WK : 0;
#pragma unroll
      for (int i = 0; i < depth; ++i)
        if (i < mine) issue(wave + i * WK, i);
      int slot = 0;
      for (int i = 0; i < mine; ++i) {
        if (i + depth <= mine)
          wait_loads<(depth - 1) * loads>();
        else
          wait_loads<0>();
        const int8_t *buf = &s[wave][slot * bytes];
        v4i wf[2][2], xf[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int at = col * kWide + ((4 * c + g) ^ (col >> 1 & 7)) * 16;
          wf[0][c] = *reinterpret_cast<const v4i *>(buf + at);
          wf[1][c] = *reinterpret_cast<const v4i *>(buf + 16 * kWide + at);
          xf[c] = *reinterpret_cast<const v4i *>(buf + kFewRows * kWide + at);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");  // read before it is written again
        if (i + depth < mine) issue(wave + (i + depth) * WK, slot);
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int f = 0; f < 2; ++f) acc[f] = mfma_i8(wf[f][c], xf[c], acc[f]);
        slot = slot + 1 == depth ? 0 : slot + 1;
      }
    } else {
      const int8_t *w[2] = {weight_row(col), weight_row(16 + col)}, *x = code_row(col);
      auto steps = [&](auto N, int k0) {  // N of them, all their loads before the first product
        v4i wf[N.value][2][2], xf[N.value][2];
#pragma unroll
        for (int i = 0; i < N.value; ++i)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int k = (k0 + WK * i) * kWide + 64 * c + 16 * g;
            __builtin_memcpy(&wf[i][0][c], w[0] + k, 16);
            __builtin_memcpy(&wf[i][1][c], w[1] + k, 16);
            __builtin_memcpy(&xf[i][c], x + k, 16);
          }
#pragma unroll
        for (int i = 0; i < N.value; ++i)
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int f = 0; f < 2; ++f) acc[f] = mfma_i8(wf[i][f][c], xf[i][c], acc[f]);
      };
      int k = wave;
      for (; k + 3 * WK < whole; k += 4 * WK) steps(std::integral_constant<int, 4>{}, k);
      for (; k < whole; k += WK) steps(std::integral_constant<int, 1>{}, k);
    }
    if (whole * kWide < a.K && whole % WK == wave) {  // the step that K ends in
      const int8_t *w[2] = {weight_row(col), weight_row(16 + col)}, *x = code_row(col);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int k = whole * kWide + 64 * c + 16 * g;
        const v4i xf = as_v4i(load_piece(x, k, a.K));
#pragma unroll
        for (int f = 0; f < 2; ++f) acc[f] = mfma_i8(as_v4i(load_piece(w[f], k, a.K)), xf, acc[f]);
      }
    }
    if (WK > 1) {
      v4i *sums = reinterpret_cast<v4i *>(&s[wave][0]);
      sums[lane] = acc[0];
      sums[kWave + lane] = acc[1];
      __syncthreads();
      if (wave == 0)
#pragma unroll
        for (int v = 1; v < WK; ++v)
#pragma unroll
          for (int f = 0; f < 2; ++f) acc[f] += reinterpret_cast<const v4i *>(&s[v][0])[kWave * f + lane];
    }
    if (wave == 0 && m0 + col < to) {
      const float sx = a.sx[row_of(a, m0 + col)];
      const int p[4] = {acc[0][0], acc[0][1], acc[0][2], acc[0][3]}, q[4] = {acc[1][0], acc[1][1], acc[1][2], acc[1][3]};
      with_type_of(a.dtype, [&](auto t) {
        using T = decltype(t);
        if (n0 + 4 * g < a.N) finish<T, 4>(a, e, m0 + col, sx, n0 + 4 * g, p, q);
        if (!a.gated && n0 + 16 + 4 * g < a.N) finish<T, 4>(a, e, m0 + col, sx, n0 + 16 + 4 * g, q, q);
      });
    }
    if (WK > 1) __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------
// Tiles of TN weight rows x TM places of one expert on mfma 32x32x32; WN x WM waves take equal parts.
// Where gated, a wave's weight rows are gates in their first half and the same columns' values in the
// second, so that a lane holds both.
//
// K goes through LDS in steps of 128 bytes, whole lines of memory (of 64 bytes: 306 us for each 2048 of K
// against 260), memory -> LDS without registers, one step ahead.  A row's
// eight 16-byte pieces lie at the places piece ^ f(row), so that 16 lanes that read one piece of 16 rows meet
// 16 different bank groups.  Row i of a wave's 32 weight rows stands for n = 16 * (i / 4 % 2) + 4 * (i / 8) +
// i % 4: a lane holds 16 consecutive n of one place.  Rows that do not start on 16 bytes (ALIGNED
// false) go through registers.  Scales and bias wait in LDS for the end.
template <int TN, int TM, int WN, int WM, bool GATED, bool ALIGNED>
__global__ __launch_bounds__(64 * WN * WM, TN * TM > 128 * 64 ? 2 : 3) void experts_tile(const ExpertArgs a) {
  constexpr int threads = 64 * WN * WM;
  constexpr int FN = TN / WN / 32, FM = TM / WM / 32;
  constexpr int bytes = (TN + TM) * kWide;
  constexpr int ring = 2;
  constexpr int loads = bytes / 16 / threads;  // pieces of a thread in a step
  constexpr int wide = GATED ? TN / 2 : TN;    // columns of y
  constexpr int FI = GATED ? FN / 2 : FN;      // 32 columns each of a wave
  static_assert(loads * 16 * threads == bytes, "a step is whole pieces of all threads");
  static_assert(!GATED || FN % 2 == 0, "a wave has gates and values");
  static_assert(WN * WM * 4096 <= ring * bytes, "the epilogue fits the ring");
  static_assert(RXMET_EXPERTS_MAX * 4 + 64 <= ring * bytes, "the experts' tiles fit the ring");
  __shared__ __attribute__((aligned(16))) int8_t s[ring][bytes];
  __shared__ __attribute__((aligned(16))) float s_sw[TN], s_bias[TN], s_sx[TM];
  const int tid = threadIdx.x, lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int col = lane % 32, h = lane / 32;
  const int tiles_n = static_cast<int>((a.N + wide - 1) / wide);

  // tiles of the experts before each one
  int *first = reinterpret_cast<int *>(&s[0][0]), *sums = first + RXMET_EXPERTS_MAX;
  int before = 0;
  for (int base = 0; base < a.experts; base += threads) {
    const int e = base + tid;
    int n = 0;
    if (e < a.experts) {
      int64_t lo, hi;
      places_of(a, e, lo, hi);
      n = static_cast<int>((hi - lo + TM - 1) / TM);
    }
    int up = n;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const int o = __shfl_up(up, d, kWave);
      if (lane >= d) up += o;
    }
    if (lane == kWave - 1) sums[wave] = up;
    __syncthreads();
    int add = before;
#pragma unroll
    for (int v = 0; v < WN * WM; ++v) {
      const int t = sums[v];
      if (v < wave) add += t;
      before += t;
    }
    if (e < a.experts) first[e] = add + up - n;
    __syncthreads();
  }
  // Workgroups go to the eight XCDs in turn: each XCD gets a run of the tiles' order, in which bands of
  // four tiles of places go through the weights together, so that its L2 holds what they share.
  const int64_t total = static_cast<int64_t>(before) * tiles_n;
  const int xcd = blockIdx.x % 8;
  const int64_t per = total / 8, rest = total % 8, at = blockIdx.x / 8;
  if (at >= per + (xcd < rest)) return;
  const int64_t id = xcd * per + (xcd < rest ? xcd : rest) + at;
  const int band = static_cast<int>(id / (4 * tiles_n)) * 4, in = static_cast<int>(id - static_cast<int64_t>(band) * tiles_n);
  const int high = before - band < 4 ? before - band : 4;
  const int tm = band + in % high, tn = in / high;
  int e = 0;
  for (int d = RXMET_EXPERTS_MAX / 2; d > 0; d >>= 1)
    if (e + d < a.experts && first[e + d] <= tm) e += d;
  e = __builtin_amdgcn_readfirstlane(e);
  int64_t m0, end;
  places_of(a, e, m0, end);
  const int within = tm - __builtin_amdgcn_readfirstlane(first[e]);
  m0 += static_cast<int64_t>(within) * TM;
  if (within < 0 || m0 >= end) return;  // offsets that do not rise
  const int64_t n0 = static_cast<int64_t>(tn) * wide;
  __syncthreads();

  // the weight row of a tile's row, for one past the columns the last
  constexpr int part = 32 * FN;  // weight rows of a wave
  auto weight_row = [&](int row) {
    const int64_t n = GATED ? n0 + row / part * (part / 2) + row % (part / 2) : n0 + row;
    return (n < a.N ? n : a.N - 1) + (GATED && row % part >= part / 2 ? a.N : 0);
  };
  // piece j of a thread lies at place tid + threads * j of the step, which holds this piece of a row
  const int8_t *src[loads];
  auto piece_at = [&](int j) {
    const int p = tid + threads * j, row = p / 8;
    return (p % 8) ^ (row < TN ? wide_turn_w(row) : wide_turn_x(row - TN));
  };
#pragma unroll
  for (int j = 0; j < loads; ++j) {
    const int row = (tid + threads * j) / 8;
    if (row < TN) {
      src[j] = a.w + e * a.e_stride + weight_row(row) * a.w_stride;
    } else {
      const int64_t i = m0 + row - TN;
      src[j] = a.x + row_of(a, i < end ? i : end - 1) * a.x_stride;
    }
  }
  {
    const int64_t row0 = static_cast<int64_t>(e) * a.N * (GATED ? 2 : 1);
    for (int r = tid; r < TN; r += threads) {
      const int64_t n = row0 + weight_row(r);
      s_sw[r] = a.sw[n];
      float b = 0;
      if (a.bias)
        with_type_of(a.dtype, [&](auto t) { b = static_cast<float>(static_cast<const decltype(t) *>(a.bias)[n]); });
      s_bias[r] = b;
    }
    for (int r = tid; r < TM; r += threads) s_sx[r] = a.sx[row_of(a, m0 + r < end ? m0 + r : end - 1)];
  }
  v16i acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
  const int wn = wave % WN * (TN / WN), wm = wave / WN * (TM / WM);
  // 32 rows on, a row has the same f: one place for each quarter of a step
  int wat[4], xat[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int w = wn + 16 * (col >> 2 & 1) + 4 * (col >> 3) + (col & 3), x = wm + col;
    wat[c] = w * kWide + ((2 * c + h) ^ wide_turn_w(w)) * 16;
    xat[c] = (TN + x) * kWide + ((2 * c + h) ^ wide_turn_x(x)) * 16;
  }
  struct Quarter {  // the operands of a quarter of a step
    v4i w[FN], x[FM];
  };
  auto load = [&](Quarter &f, const int8_t *buf, int c) {
#pragma unroll
    for (int i = 0; i < FN; ++i) f.w[i] = *reinterpret_cast<const v4i *>(buf + wat[c] + 32 * i * kWide);
#pragma unroll
    for (int j = 0; j < FM; ++j) f.x[j] = *reinterpret_cast<const v4i *>(buf + xat[c] + 32 * j * kWide);
  };
  auto multiply = [&](const Quarter &f) {
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int j = 0; j < FM; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.w[i], f.x[j], acc[i][j], 0, 0, 0);
  };
  const int whole = a.K / kWide;
  if constexpr (ALIGNED) {
    auto issue = [&](int step, int slot) {
#pragma unroll
      for (int j = 0; j < loads; ++j)
        load_to_lds(src[j] + piece_at(j) * 16 + step * kWide, &s[slot][wave * 1024 + j * threads * 16]);
    };
    if (whole > 0) {
      // past the end a step is read once more, so that the count of loads in flight holds
      issue(0, 0);
      issue(whole > 1 ? 1 : 0, 1);
      wait_loads<loads>();
      meet();
      // each quarter's operands are read from LDS while the quarter before is multiplied
      Quarter even, odd;
      load(even, s[0], 0);
      for (int k = 0; k < whole; ++k) {
        const int slot = k & 1;
        load(odd, s[slot], 1);
        multiply(even);
        load(even, s[slot], 2);
        multiply(odd);
        load(odd, s[slot], 3);
        multiply(even);
        wait_loads<0>();
        meet();  // step k + 1 is there for all, and step k has been read by all
        load(even, s[slot ^ 1], 0);
        issue(k + 2 < whole ? k + 2 : k, slot);
        multiply(odd);
      }
      wait_loads<0>();
    }
  } else {
    uint4 piece[loads];
    auto fetch = [&](int step) {
#pragma unroll
      for (int j = 0; j < loads; ++j) {
        uint4 v;
        __builtin_memcpy(&v, src[j] + piece_at(j) * 16 + step * kWide, 16);
        piece[j] = v;
      }
    };
    auto put = [&](int slot) {
#pragma unroll
      for (int j = 0; j < loads; ++j) *reinterpret_cast<uint4 *>(&s[slot][16 * (tid + threads * j)]) = piece[j];
    };
    if (whole > 0) {
      fetch(0);
      put(0);
      __syncthreads();
    }
    for (int k = 0; k < whole; ++k) {
      if (k + 1 < whole) fetch(k + 1);
      Quarter f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        load(f, s[k % 2], c);
        multiply(f);
      }
      if (k + 1 < whole) put((k + 1) % 2);
      __syncthreads();
    }
  }
  __syncthreads();
  if (whole * kWide < a.K) {  // the step that K ends in
#pragma unroll
    for (int j = 0; j < loads; ++j)
      *reinterpret_cast<uint4 *>(&s[0][16 * (tid + threads * j)]) =
          load_piece(src[j], whole * kWide + 16 * piece_at(j), a.K);
    __syncthreads();
    Quarter f;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      load(f, s[0], c);
      multiply(f);
    }
    __syncthreads();
  }

  // A lane finishes its 16 consecutive columns of a place; 128 bytes of 32 places at a time (64 of gated outputs in
  // 16 bits) go through the wave's part of the LDS, from where neighbouring lanes write what lies side by side.
  // The activation is chosen once: asked for at each element, the code that is jumped over falls out
  // of the instruction cache.
  uint4 *out = reinterpret_cast<uint4 *>(&s[0][0]) + wave * 256;
  auto put = [&](auto type, int first, int chunks, const float (&v)[16]) {
    using T = decltype(type);
    T y[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) y[r] = static_cast<T>(v[r]);
#pragma unroll
    for (int c = 0; c < static_cast<int>(sizeof(T)); ++c) {
      uint4 w;
      __builtin_memcpy(&w, &y[c * 16 / sizeof(T)], 16);
      out[col * chunks + ((first + c) ^ (col >> 1 & (chunks - 1)))] = w;
    }
  };
  auto flush = [&](int j, int n, int chunks, int size) {
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    for (int p = lane; p < 32 * chunks; p += kWave) {
      const int m = p / chunks, c = p % chunks;
      const uint4 w = out[m * chunks + (c ^ (m >> 1 & (chunks - 1)))];
      const int64_t i = m0 + wm + 32 * j + m, n1 = n + c * 16 / size;
      if (i >= end || n1 >= a.N) continue;
      char *y = static_cast<char *>(a.y) + (i * a.N + n1) * size;
      const int64_t left = (a.N - n1) * size;
      if (left >= 16) {
        if (a.past) {
          v4i_any v;
          __builtin_memcpy(&v, &w, 16);
          __builtin_nontemporal_store(v, reinterpret_cast<v4i_any *>(y));
        } else {
          __builtin_memcpy(y, &w, 16);
        }
      } else {
        const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int b = 0; b < 16; b += 2)
          if (b < left) *reinterpret_cast<unsigned short *>(y + b) = static_cast<unsigned short>(u[b / 4] >> (8 * (b % 4)));
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");  // read before it is written again
  };
  bool general = a.bias != nullptr;  // or some row's scale is large
  for (int r = lane; r < TM / WM; r += kWave) general |= is_large(s_sx[wm + r]);
  general = __any(general);
  auto finish_tile = [&](auto act, auto type, auto GENERAL) {
    constexpr int pair = FI < 2 || GATED ? 1 : 2;
    // keeps apart what the copies have in common: done ahead of the choice it would take all registers
    asm volatile("; activation %0 %1" : : "n"(2 * decltype(act)::value + GENERAL.value), "n"(sizeof(type)));
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const float sx = s_sx[wm + 32 * j + col];
      const float lead = GENERAL.value && is_large(sx) ? 1.0f : sx, rest = is_large(sx) ? sx : 1.0f;
#pragma unroll
      for (int i0 = 0; i0 < FI; i0 += pair) {
        float y[pair][16];
#pragma unroll
        for (int d = 0; d < pair; ++d) {
          // the sum of fragment i's column 4 q + r of the lane, scaled
          auto scaled = [&](int i, int q, int up, float (&v)[4]) {
            const int r0 = wn + 32 * (i0 + d) + 16 * h + 4 * q + up;
            const f4 w = *reinterpret_cast<const f4 *>(&s_sw[r0]);
            f4 b;
            if (GENERAL.value) b = *reinterpret_cast<const f4 *>(&s_bias[r0]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              v[r] = static_cast<float>(acc[i][j][4 * q + r]) * lead * w[r];
              if (GENERAL.value) v[r] = v[r] * rest + b[r];
            }
          };
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            float v[4];
            scaled(i0 + d, q, 0, v);
#pragma unroll
            for (int r = 0; r < 4; ++r) y[d][4 * q + r] = activated<decltype(type)>(v[r], decltype(act)::value);
            if (GATED) {
              scaled(FI + i0 + d, q, part / 2, v);
#pragma unroll
              for (int r = 0; r < 4; ++r) y[d][4 * q + r] *= v[r];
            }
            if (decltype(act)::value == RXMET_ACT_GELU) __builtin_amdgcn_sched_barrier(0);
          }
          __builtin_amdgcn_sched_barrier(0);  // scales of 16 columns at a time, for the registers
        }
        const int n = static_cast<int>(n0) + (GATED ? wn / 2 : wn) + 32 * i0;
        if (a.dtype == RXMET_QDQ_F32) {
#pragma unroll
          for (int d = 0; d < pair; ++d) {
            put(float{}, 4 * h, 8, y[d]);
            flush(j, n + 32 * d, 8, 4);
          }
        } else {
#pragma unroll
          for (int d = 0; d < pair; ++d) {
            if (a.dtype == RXMET_QDQ_BF16)
              put(bf16{}, 4 * d + 2 * h, 4 * pair, y[d]);
            else
              put(f16{}, 4 * d + 2 * h, 4 * pair, y[d]);
          }
          flush(j, n, 4 * pair, 2);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  using std::integral_constant;
  auto finish_as = [&](auto act, auto type) {  // type: float or one of 16 bits, for the activation alone
    if (general)
      finish_tile(act, type, std::true_type{});
    else
      finish_tile(act, type, std::false_type{});
  };
  switch (a.act) {
    case RXMET_ACT_RELU: finish_as(integral_constant<int, RXMET_ACT_RELU>{}, float{}); break;
    case RXMET_ACT_SILU:
      if (a.dtype == RXMET_QDQ_F32)
        finish_as(integral_constant<int, RXMET_ACT_SILU>{}, float{});
      else
        finish_as(integral_constant<int, RXMET_ACT_SILU>{}, bf16{});
      break;
    case RXMET_ACT_GELU: finish_as(integral_constant<int, RXMET_ACT_GELU>{}, float{}); break;
    default: finish_as(integral_constant<int, RXMET_ACT_NONE>{}, float{});
  }
}

// Whether the rows can be read in aligned pieces of 16 bytes.
bool aligned(const ExpertArgs &a) {
  return (reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.w) |
          static_cast<uintptr_t>(a.x_stride) | static_cast<uintptr_t>(a.w_stride) |
          static_cast<uintptr_t>(a.e_stride)) % 16 == 0;
}

template <int TN, int TM, int WN, int WM, bool GATED>
void launch_tile(const ExpertArgs &a, hipStream_t st) {
  // an expert's last tile may be partly filled; a run of an XCD is rounded up
  const int64_t tiles_m = a.rows / TM + (a.experts < a.rows ? a.experts : a.rows);
  const int64_t tiles = cdiv(a.N, GATED ? TN / 2 : TN) * tiles_m;
  const unsigned grid = static_cast<unsigned>(cdiv(tiles, 8) * 8);
  if (aligned(a))
    experts_tile<TN, TM, WN, WM, GATED, true><<<grid, 64 * WN * WM, 0, st>>>(a);
  else
    experts_tile<TN, TM, WN, WM, GATED, false><<<grid, 64 * WN * WM, 0, st>>>(a);
}

template <int WK>
void launch_few(const ExpertArgs &a, int64_t grid, hipStream_t st) {
  const unsigned n = static_cast<unsigned>(grid);
  if (aligned(a))
    experts_few<WK, true><<<n, 64 * WK, 0, st>>>(a);
  else
    experts_few<WK, false><<<n, 64 * WK, 0, st>>>(a);
}

// How a call is run, by how many rows an expert has (R / E) and how much weight there is to stream.
//
// Up to 16 rows each: the smallest tiles where there are three for two CUs ([64 x 2048, 2048] gated weights of 64
// experts, 128 rows: 45.8 us, 5.2 TB/s; experts_few 48.1), else experts_few, whose waves are more (16
// experts of [2048, 2048], 16 rows: 11.9 us against 16.0), and where those are fewer than 128, four waves
// for each 32 weight rows (4 experts of [512, 4096]: 8.0 us, one wave 11.0).  Experts that have rows are
// at most as many as rows.
//
// More: a tile size costs its rounds of tiles over the CUs (half a round more, for the last one is not
// full) times what a round takes; of 32 experts with [2048, 2048], [R / E: 256 x 256, 128 x 128, 128 x 64]
// 64: 40 28 29 us; 256: 72 67 65; 384: 105 91 97; 512: 108 116 118; 2048: 388 441 481.
//
// R counts entries of no expert too, as how many there are stands on the device alone: with nine of ten such, 8192 x 8
// of them take 61 us (as many rows in a call of their own 84), 2048 x 8 48 us (45).
enum Shape { kFewShared, kFewOne, k128x64, k128x128, k256x256 };

Shape shape_for(int64_t rows, int64_t experts, int64_t out_rows) {
  const int64_t busy = rows < experts ? rows : experts;
  if (rows <= 16 * experts && busy * cdiv(out_rows, 128) < 384)
    return busy * cdiv(out_rows, 32) < 128 ? kFewShared : kFewOne;
  // tiles of an expert's rows, the last one half full; relative time of a round, tiles that a CU holds
  auto cost = [&](int64_t tn, int64_t tm, double round, int held) {
    const double tiles = static_cast<double>(cdiv(out_rows, tn)) * (static_cast<double>(rows) / tm + busy / 2.0);
    return (tiles / (256 * held) + 0.5) * round;
  };
  const double small = cost(128, 64, 22, 3), middle = cost(128, 128, 26, 2), large = cost(256, 256, 43, 1);
  return small <= middle && small <= large ? k128x64 : middle <= large ? k128x128 : k256x256;
}

template <bool GATED>
void launch(const ExpertArgs &a, hipStream_t st) {
  const int64_t few = cdiv(a.N, GATED ? kFewRows / 2 : kFewRows) * a.experts;
  switch (shape_for(a.rows, a.experts, GATED ? 2 * a.N : a.N)) {
    case kFewShared: launch_few<4>(a, few, st); break;
    case kFewOne: launch_few<1>(a, few, st); break;
    case k128x64: launch_tile<128, 64, 2, 2, GATED>(a, st); break;
    case k128x128: launch_tile<128, 128, 2, 2, GATED>(a, st); break;
    case k256x256: launch_tile<256, 256, 2, 4, GATED>(a, st); break;
  }
}

}  // namespace
}  // namespace dec
}  // namespace rxmet

using namespace rxmet;
using namespace rxmet::dec;

extern "C" int rxmet_selftest_experts_form(int64_t rows, int64_t experts, int64_t weight_rows) {
  RXMET_CHECK_ARG(rows >= 1 && experts >= 1 && weight_rows >= 1, "sizes must be positive");
  return shape_for(rows, experts, weight_rows);
}

extern "C" int rxmet_experts_linear_int8(const rxmet_expert_groups *g, int32_t grouped,
                                         const int8_t *codes, int64_t codes_stride,
                                         const float *scales, const int8_t *weight,
                                         int64_t weight_stride, int64_t expert_stride,
                                         const float *weight_scales, const void *bias, void *y,
                                         int64_t N, int64_t K, int32_t gated, int32_t activation,
                                         int32_t dtype, void *stream) {
  RXMET_CHECK_ARG(g != nullptr, "the groups are missing");
  RXMET_CHECK_ARG(g->experts >= 1 && g->experts <= RXMET_EXPERTS_MAX, "there must be 1 to 1024 experts");
  RXMET_CHECK_ARG(g->top_k >= 1 && g->top_k <= RXMET_TOP_K_MAX, "top_k must be between 1 and 64");
  RXMET_CHECK_ARG(g->tokens >= 0 && g->tokens <= 1 << 24, "there must be at most 2^24 tokens");
  RXMET_CHECK_ARG(N >= 1 && N <= 1 << 24 && K >= 1 && K <= RXMET_LINEAR_INT8_K_MAX,
                  "N must be between 1 and 2^24 and K between 1 and 131071");
  RXMET_CHECK_ARG(activation >= RXMET_ACT_NONE && activation <= RXMET_ACT_GELU, "unknown activation");
  RXMET_CHECK_ARG(dtype == RXMET_QDQ_F32 || dtype == RXMET_QDQ_F16 || dtype == RXMET_QDQ_BF16,
                  "element type must be fp32, fp16 or bf16");
  const int64_t rows = g->tokens * g->top_k;
  if (rows == 0) return 0;
  RXMET_CHECK_ARG(g->offsets && (grouped || g->entries), "the groups' offsets and entries are needed");
  RXMET_CHECK_ARG(codes && scales && weight && weight_scales && y,
                  "codes, weight, their scales and y are needed");
  // An output of whole 16-byte pieces that would push codes and weights out of the memory's 256 MB cache is
  // written past it, also where the next call reads it (us through the caches and past them, in brackets with
  // quantize_rows behind: 32 experts' [2048, 2048] weights, bf16, 64 MB of output 122 and 115 [141, 140], 128 MB 204
  // and 185 [238, 236], 256 MB 364 and 335 [451, 434]; below, 32 MB, 84 and 75 [95, 97]).  Gated ones, with twice the
  // products to an output, gain and lose up to 2 % (128 MB 374 and 380 [418, 425], 256 MB 688 and 688 [778, 775], other
  // inputs in turn 690 and 685).
  const int64_t size = dtype == RXMET_QDQ_F32 ? 4 : 2;
  const bool past = rows * N * size >= 64LL << 20 && (N * size | reinterpret_cast<uintptr_t>(y)) % 16 == 0;
  const ExpertArgs a{g->offsets, g->entries, g->tokens, rows, g->top_k, g->experts, grouped != 0,
                     codes, weight, codes_stride, weight_stride, expert_stride, scales, weight_scales,
                     bias, y, N, static_cast<int>(K), gated != 0, activation, dtype, past};
  const int64_t few = cdiv(N, gated ? kFewRows / 2 : kFewRows) * g->experts;
  RXMET_CHECK_ARG(rows < 1 << 26 && few < 1 << 22 &&
                      cdiv(N, gated ? 64 : 128) * (rows / 64 + g->experts) < 1 << 22,
                  "too many outputs for one call");
  auto st = static_cast<hipStream_t>(stream);
  prof::Scope scope("experts_linear_int8", st);
  if (a.gated)
    launch<true>(a, st);
  else
    launch<false>(a, st);
  RXMET_CHECK_LAUNCH();
  return 0;
}

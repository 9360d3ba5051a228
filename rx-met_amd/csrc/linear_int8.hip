// linear_int8.hip — product of int8 codes with int8 weights and its epilogue.
//
// Mathematics.  y[m, n] = act(acc * sx[m] * sw[n] + b[n]) + r[m, n] with acc = sum_k x[m, k] w[n, k] exact in
// int32 (|acc| <= 2^14 K).  The epilogue is fp32 and rounds once.
//
// Layout.  The matrix instruction's rows are weight rows (n), its columns are token rows (m), so
// that a lane holds several consecutive n of one m and writes them as one vector: row i of tile t
// of a wave's 64 weight rows stands for n = 16 * (i / 4) + 4 t + i % 4, which gives a lane 16
// consecutive n.
#include <type_traits>

#include "decoder_common.h"
#include "mfma_frag.h"

namespace rxmet {
namespace dec {
namespace {

struct LinArgs {
  const int8_t *x, *w;
  int64_t x_stride, w_stride;
  const float *sx, *sw;
  const void *bias, *res;
  int64_t res_stride;
  void *y;
  int64_t M, N;
  int K, act;
};

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

// Writes C consecutive n of row m.
template <typename T, int C>
__device__ __forceinline__ void finish(const LinArgs &a, int64_t m, int64_t n0, const int (&acc)[C]) {
  if (m >= a.M || n0 >= a.N) return;
  const float sx = a.sx[m];
  const T *bias = static_cast<const T *>(a.bias);
  const T *res = a.res ? static_cast<const T *>(a.res) + m * a.res_stride + n0 : nullptr;
  T *y = static_cast<T *>(a.y) + m * a.N + n0;
  struct Run {
    T v[C];
  } out, r;
  const int left = a.N - n0 < C ? static_cast<int>(a.N - n0) : C;
  if (res) {
    if (left == C) {
      __builtin_memcpy(&r, res, sizeof(r));
    } else {
#pragma unroll
      for (int e = 0; e < C; ++e)
        if (e < left) r.v[e] = res[e];
    }
  }
#pragma unroll
  for (int e = 0; e < C; ++e) {
    if (e >= left) continue;
    float v = static_cast<float>(acc[e]) * sx * a.sw[n0 + e];
    if (bias) v += static_cast<float>(bias[n0 + e]);
    v = activate(v, a.act);
    if (res) v += static_cast<float>(r.v[e]);
    out.v[e] = static_cast<T>(v);
  }
  if (left == C) {
    __builtin_memcpy(y, &out, sizeof(out));
  } else {
#pragma unroll
    for (int e = 0; e < C; ++e)
      if (e < left) y[e] = out.v[e];
  }
}

// Few rows of x: a workgroup takes 16 weight rows and all of K, its eight waves take runs of 128
// of K in turn; the weights go from memory into the matrix instruction with no stop in LDS.
constexpr int kFewWaves = 8;

template <typename T, int MT>
__global__ __launch_bounds__(64 * kFewWaves) void linear_few(const LinArgs a) {
  __shared__ int s[kFewWaves][MT * 16][20];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int col = lane % 16, g = lane / 16;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16;
  const int64_t nrow = n0 + col < a.N ? n0 + col : a.N - 1;
  const int8_t *w = a.w + nrow * a.w_stride;
  const int8_t *x[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int64_t m = t * 16 + col < a.M ? t * 16 + col : a.M - 1;
    x[t] = a.x + m * a.x_stride;
  }
  v4i acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = v4i{0, 0, 0, 0};
#pragma unroll 4
  for (int k0 = wave * 128; k0 < a.K; k0 += kFewWaves * 128) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int k = k0 + 64 * c + 16 * g;
      const v4i wf = as_v4i(load_piece(w, k, a.K));
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[t] = mfma_i8(wf, as_v4i(load_piece(x[t], k, a.K)), acc[t]);
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) s[wave][t * 16 + col][4 * g + r] = acc[t][r];
  __syncthreads();
  for (int i = threadIdx.x; i < MT * 16 * 4; i += 64 * kFewWaves) {
    const int m = i / 4, n = i % 4 * 4;
    int sum[4] = {0, 0, 0, 0};
#pragma unroll
    for (int v = 0; v < kFewWaves; ++v)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += s[v][m][n + e];
    finish<T, 4>(a, m, n0 + n, sum);
  }
}

// Tiles of 128 weight rows x 128 token rows, 128 of K at a time through LDS; four waves take
// 64 x 64 each.  A row's eight 16-byte pieces lie at the places (piece ^ f(row)), so that the 16 lanes that
// read one piece of 16 rows find it in 16 different bank groups.
constexpr int kTile = 128, kStep = 128;

__device__ __forceinline__ int place_w(int row, int piece) {
  return (row * 8 + (piece ^ ((row >> 1 & 1) | (row >> 4 & 3) << 1))) * 16;
}
__device__ __forceinline__ int place_x(int row, int piece) {
  return (row * 8 + (piece ^ (row >> 1 & 7))) * 16;
}

template <typename T>
__global__ __launch_bounds__(256) void linear_tile(const LinArgs a) {
  __shared__ __attribute__((aligned(16))) int8_t s[2][2][kTile * kStep];
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int col = lane % 16, g = lane / 16;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * kTile, m0 = static_cast<int64_t>(blockIdx.y) * kTile;
  // staging: thread takes piece tid % 8 of rows tid / 8 + 32 j
  const int8_t *wp[4], *xp[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int r = tid / 8 + 32 * j;
    wp[j] = a.w + (n0 + r < a.N ? n0 + r : a.N - 1) * a.w_stride;
    xp[j] = a.x + (m0 + r < a.M ? m0 + r : a.M - 1) * a.x_stride;
  }
  uint4 wr[4], xr[4];
  auto fetch = [&](int k0) {
    const int k = k0 + 16 * (tid % 8);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      wr[j] = load_piece(wp[j], k, a.K);
      xr[j] = load_piece(xp[j], k, a.K);
    }
  };
  auto put = [&](int buf) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = tid / 8 + 32 * j;
      *reinterpret_cast<uint4 *>(&s[buf][0][place_w(r, tid % 8)]) = wr[j];
      *reinterpret_cast<uint4 *>(&s[buf][1][place_x(r, tid % 8)]) = xr[j];
    }
  };
  v4i acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = v4i{0, 0, 0, 0};
  const int wn = wave % 2 * 64, wm = wave / 2 * 64;
  fetch(0);
  put(0);
  __syncthreads();
  int buf = 0;
  for (int k0 = 0; k0 < a.K; k0 += kStep, buf ^= 1) {
    const bool more = k0 + kStep < a.K;
    if (more) fetch(k0 + kStep);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      v4i wf[4], xf[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int r = wn + 16 * (col >> 2) + 4 * t + (col & 3);
        wf[t] = as_v4i(*reinterpret_cast<const uint4 *>(&s[buf][0][place_w(r, 4 * c + g)]));
        xf[t] = as_v4i(*reinterpret_cast<const uint4 *>(&s[buf][1][place_x(wm + 16 * t + col, 4 * c + g)]));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = mfma_i8(wf[i], xf[j], acc[i][j]);
    }
    if (more) put(buf ^ 1);
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    int v[16];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) v[4 * i + r] = acc[i][j][r];
    finish<T, 16>(a, m0 + wm + 16 * j + col, n0 + wn + 16 * g, v);
  }
}

}  // namespace
}  // namespace dec
}  // namespace rxmet

using namespace rxmet;
using namespace rxmet::dec;

extern "C" int64_t rxmet_linear_int8_workspace_bytes(int64_t, int64_t, int64_t) { return 0; }

extern "C" int rxmet_linear_int8(const int8_t *codes, int64_t codes_stride, const float *scales,
                                 const int8_t *weight, int64_t weight_stride,
                                 const float *weight_scales, const void *bias,
                                 const void *residual, int64_t residual_stride, void *y, int64_t M,
                                 int64_t N, int64_t K, int32_t activation, int32_t dtype,
                                 void *workspace, void *stream) {
  (void)workspace;
  RXMET_CHECK_ARG(M >= 0 && N >= 1 && K >= 1 && K <= RXMET_LINEAR_INT8_K_MAX,
                  "M must be >= 0, N >= 1 and K between 1 and 131071");
  RXMET_CHECK_ARG(M <= INT32_MAX && N <= INT32_MAX, "M and N must be below 2^31");
  RXMET_CHECK_ARG(activation >= RXMET_ACT_NONE && activation <= RXMET_ACT_GELU,
                  "unknown activation");
  RXMET_CHECK_ARG(dtype == RXMET_QDQ_F32 || dtype == RXMET_QDQ_F16 || dtype == RXMET_QDQ_BF16,
                  "element type must be fp32, fp16 or bf16");
  if (M == 0) return 0;
  RXMET_CHECK_ARG(codes && scales && weight && weight_scales && y,
                  "codes, weight, their scales and y are needed");
  const LinArgs a{codes, weight, codes_stride, weight_stride, scales, weight_scales, bias,
                  residual, residual_stride, y, M, N, static_cast<int>(K), activation};
  auto st = static_cast<hipStream_t>(stream);
  prof::Scope scope("linear_int8", st);
  with_type(dtype, [&](auto t) {
    using T = decltype(t);
    if (M <= 64) {
      const unsigned grid = static_cast<unsigned>(cdiv(N, 16));
      if (M <= 16) linear_few<T, 1><<<grid, 64 * kFewWaves, 0, st>>>(a);
      else if (M <= 32) linear_few<T, 2><<<grid, 64 * kFewWaves, 0, st>>>(a);
      else linear_few<T, 4><<<grid, 64 * kFewWaves, 0, st>>>(a);
    } else {
      const dim3 grid(static_cast<unsigned>(cdiv(N, kTile)), static_cast<unsigned>(cdiv(M, kTile)));
      linear_tile<T><<<grid, 256, 0, st>>>(a);
    }
  });
  RXMET_CHECK_LAUNCH();
  return 0;
}

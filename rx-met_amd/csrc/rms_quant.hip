// rms_quant.hip — root-mean-square norm of x + residual with int8 output and a scale per row, the
// same without the norm, and the gradient of the fake-quantised training form.
//
// Mathematics.  With h = round(x + r), rstd = 1 / sqrt(mean(h^2) + eps) and u = h * w, the
// normalised row is n = u * rstd and its symmetric grid has the scale max|n| / 127.  rstd is positive, so
// it cancels out of n / scale = u * 127 / max|u|: the codes follow from u alone (bit for bit, whatever the
// order in which the mean was summed), and rstd enters the scale only.  The sum and the maximum are
// taken in one pass over a row that stays in registers.  Rows whose squares leave fp32's range are
// summed again in 64 bits.
//
// Bound: HBM traffic, one read of each input and one write of each output, and for few rows the launch and one
// trip to memory.  A workgroup of 256 threads has a row of up to 8192 elements (a wave up to 1024, 1024
// threads above); the next rows' loads are other workgroups'.  Measured, bf16: [8192, 4096] with a
// residual, forward (h and the values out) 268 MB in 50 us and backward 268 MB and 17 MB of partial sums in 53
// us; [3001, 4099], whose rows start at any two bytes, with h and codes out 86 MB in 22 us; [16, 4096]
// 4.4 us.
#include <type_traits>

#include "decoder_common.h"

namespace rxmet {
namespace dec {
namespace {

struct RowArgs {
  const void *x, *res, *w;
  int64_t x_stride, res_stride;
  void *h;
  int8_t *codes;
  void *y;
  float *scales, *rstd;
  int64_t rows, row0;  // row0: of the tensors, where a launch takes a part of the rows
  int cols;
  float eps;
};

// Sum, and maximum of magnitudes as bits, over the TPR threads of a row.
template <int TPR>
__device__ __forceinline__ void row_reduce(float &sum, unsigned &top) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, kWave);
  top = wave_max_bits(top);
  if constexpr (TPR > kWave) {
    constexpr int waves = TPR / kWave;
    __shared__ float s_sum[waves];
    __shared__ unsigned s_top[waves];
    const int wave = threadIdx.x / kWave;
    if (threadIdx.x % kWave == 0) s_sum[wave] = sum, s_top[wave] = top;
    __syncthreads();
    sum = s_sum[0], top = s_top[0];
#pragma unroll
    for (int k = 1; k < waves; ++k) {
      sum += s_sum[k];
      top = s_top[k] > top ? s_top[k] : top;
    }
  }
}

constexpr float kLargest = 3.402823466e38f;

// 1 / sqrt(mean(h^2) + eps) in 64 bits, of rows whose squares leave fp32's range.  One element at a time,
// those that the thread has written itself: it is rare, and the usual rows need the registers.
template <typename T, int TPR, int NV>
__device__ __forceinline__ double rstd_beyond_range(const T *h, int cols, float eps) {
  double sum = 0.0;
#pragma unroll 1
  for (int i = 0; i < 8 * NV; ++i) {
    const int c = (i / 8 * TPR + threadIdx.x % TPR) * 8 + i % 8;
    if (c < cols) {
      const double v = static_cast<double>(static_cast<float>(h[c]));
      sum += v * v;
    }
  }
#pragma unroll 1
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, kWave);
  if constexpr (TPR > kWave) {
    constexpr int waves = TPR / kWave;
    __shared__ double s_sum[waves];
    if (threadIdx.x % kWave == 0) s_sum[threadIdx.x / kWave] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll 1
    for (int k = 0; k < waves; ++k) sum += s_sum[k];
  }
  return 1.0 / sqrt(sum / cols + eps);
}

template <typename T, typename W, int TPR, int NV>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rms_forward(const RowArgs a) {
  constexpr int block = TPR < 256 ? 256 : TPR;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * (block / TPR) + threadIdx.x / TPR;
  const int tid = threadIdx.x % TPR;
  if (at >= a.rows) return;  // whole waves (TPR = 64) or none: no barrier follows for them
  const int64_t row = a.row0 + at;
  const T *x = static_cast<const T *>(a.x) + row * a.x_stride;
  const T *res = a.res ? static_cast<const T *>(a.res) + row * a.res_stride : nullptr;
  const W *w = static_cast<const W *>(a.w);
  float u[NV][8];
  float sum = 0.0f;
  unsigned bits = 0;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = (v * TPR + tid) * 8, n = a.cols - c;
    if (n >= 8) {
      load8(x + c, u[v]);
      if (res) {
        float r[8];
        load8(res + c, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) u[v][e] = static_cast<float>(static_cast<T>(u[v][e] + r[e]));
        stream_out8(static_cast<T *>(a.h) + row * a.cols + c, u[v]);
      }
    } else {
      load8_part(x + c, n, u[v]);
      if (res) {
        float r[8];
        load8_part(res + c, n, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) u[v][e] = static_cast<float>(static_cast<T>(u[v][e] + r[e]));
        store8_part(static_cast<T *>(a.h) + row * a.cols + c, n, u[v]);
      }
    }
    if (w) {
      float f[8];
      if (n >= 8)
        load8(w + c, f);
      else
        load8_part(w + c, n, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sum += u[v][e] * u[v][e];
        u[v][e] *= f[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) bits = __builtin_elementwise_max(bits, magnitude(u[v][e]));
  }
  row_reduce<TPR>(sum, bits);
  const float top = __builtin_bit_cast(float, bits);
  const bool good = top <= kLargest;
  const float peak = fmaxf(top, kFloor);
  const float mean = sum / static_cast<float>(a.cols) + a.eps;
  float rstd = w ? 1.0f / sqrtf(mean) : 1.0f, scale = peak * kInv127 * rstd;
  // squares below 2^-126 lose bits, which count where they are the mean; all threads of a row agree
  if (w && (mean > kLargest || mean < 0x1p-100f)) {
    const double r = rstd_beyond_range<T, TPR, NV>(
        res ? static_cast<const T *>(a.h) + row * a.cols : x, a.cols, a.eps);
    rstd = static_cast<float>(r);
    scale = static_cast<float>(static_cast<double>(peak) / 127.0 * r);
  }
  if (!good) scale = nanf32();
  const float inv = good ? 127.0f / peak : 0.0f;
  const unsigned keep = good ? ~0u : 0u;
  if (tid == 0) {
    a.scales[row] = scale;
    if (a.rstd) a.rstd[row] = rstd;
  }
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = (v * TPR + tid) * 8, n = a.cols - c;
    if (n <= 0) continue;
    if (a.codes) {
      unsigned b[2];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        b[k] = code_bytes4(u[v][4 * k] * inv, u[v][4 * k + 1] * inv, u[v][4 * k + 2] * inv,
                           u[v][4 * k + 3] * inv, keep);
      int8_t *p = a.codes + row * a.cols + c;
      if (n >= 8) {
        __builtin_memcpy(p, b, 8);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < n) p[e] = static_cast<int8_t>(b[e / 4] >> (8 * (e % 4)));
      }
    }
    if (a.y) {
      float q[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = rintf(u[v][e] * inv) * scale;
      T *p = static_cast<T *>(a.y) + row * a.cols + c;
      if (n >= 8)
        stream_out8(p, q);
      else
        store8_part(p, n, q);
    }
  }
}

struct BackArgs {
  const void *dy, *dh, *h, *w;
  int64_t dy_stride, dh_stride, h_stride;
  const float *rstd;
  void *dx;
  float *part;  // [blocks, cols] sums of dy * n, or null
  int64_t rows;
  int cols;
};

// A block takes the rows blockIdx.x, + gridDim.x, ... and keeps its columns' weight gradient in
// registers over all of them.
template <typename T, typename W, int TPR, int NV>
__global__ __launch_bounds__(TPR) void rms_backward(const BackArgs a) {
  const int tid = threadIdx.x;
  const W *w = static_cast<const W *>(a.w);
  float dw[NV][8] = {};
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float rstd = a.rstd[row];
    float n[NV][8], dn[NV][8];
    float dot = 0.0f;
    unsigned none = 0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * TPR + tid) * 8, m = a.cols - c;
      const T *dy = static_cast<const T *>(a.dy) + row * a.dy_stride + c;
      const T *h = static_cast<const T *>(a.h) + row * a.h_stride + c;
      float f[8];
      if (m >= 8) {
        load8(dy, dn[v]);
        load8(h, n[v]);
        load8(w + c, f);
      } else {
        load8_part(dy, m, dn[v]);
        load8_part(h, m, n[v]);
        load8_part(w + c, m, f);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        n[v][e] *= rstd;
        dw[v][e] += dn[v][e] * n[v][e];
        dn[v][e] *= f[e];
        dot += dn[v][e] * n[v][e];
      }
    }
    row_reduce<TPR>(dot, none);
    const float mean = dot / static_cast<float>(a.cols);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * TPR + tid) * 8, m = a.cols - c;
      if (m <= 0) continue;
      float g[8] = {};
      if (a.dh) {
        const T *dh = static_cast<const T *>(a.dh) + row * a.dh_stride + c;
        if (m >= 8)
          load8(dh, g);
        else
          load8_part(dh, m, g);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] = rstd * (dn[v][e] - n[v][e] * mean) + g[e];
      T *dx = static_cast<T *>(a.dx) + row * a.cols + c;
      if (m >= 8)
        stream_out8(dx, g);
      else
        store8_part(dx, m, g);
    }
    __syncthreads();  // the reduction's LDS is written again for the next row
  }
  if (a.part) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * TPR + tid) * 8, m = a.cols - c;
      float *p = a.part + static_cast<int64_t>(blockIdx.x) * a.cols + c;
      if (m >= 8)
        store8(p, dw[v]);
      else
        store8_part(p, m, dw[v]);
    }
  }
}

// d_weight[c] = sum over the blocks' partial sums, in a fixed order: a workgroup has 16 columns
// and 64 threads for each, of which each adds every 64th partial; then the 64 sums are added up.
// 16 columns and not 64, because 4096 columns are then 256 workgroups (17 us -> 7 us).
constexpr int kGradCols = 16, kGradLanes = 64;

template <typename W>
__global__ __launch_bounds__(kGradCols * kGradLanes) void rms_weight_grad(const float *part,
                                                                          int blocks, int cols,
                                                                          W *dw) {
  __shared__ float s[kGradLanes][kGradCols];
  const int lane = threadIdx.x % kGradCols, k = threadIdx.x / kGradCols;
  const int c = blockIdx.x * kGradCols + lane;
  float sum = 0.0f;
  if (c < cols) {
#pragma unroll 4
    for (int b = k; b < blocks; b += kGradLanes) sum += part[static_cast<int64_t>(b) * cols + c];
  }
  s[k][lane] = sum;
  __syncthreads();
  if (k == 0 && c < cols) {
#pragma unroll
    for (int j = 1; j < kGradLanes; ++j) sum += s[j][lane];
    dw[c] = static_cast<W>(sum);
  }
}

// Runs f(threads per row, vectors of eight per thread) for rows of `cols` elements.
template <typename F>
void with_row_shape(int64_t cols, F &&f) {
  using std::integral_constant;
  if (cols <= 512) f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  else if (cols <= 1024) f(integral_constant<int, 64>{}, integral_constant<int, 2>{});
  else if (cols <= 2048) f(integral_constant<int, 256>{}, integral_constant<int, 1>{});
  else if (cols <= 4096) f(integral_constant<int, 256>{}, integral_constant<int, 2>{});
  else if (cols <= 8192) f(integral_constant<int, 256>{}, integral_constant<int, 4>{});
  else if (cols <= 16384) f(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
  else if (cols <= 32768) f(integral_constant<int, 1024>{}, integral_constant<int, 4>{});
  else f(integral_constant<int, 1024>{}, integral_constant<int, 8>{});
}

template <typename F>
bool with_weight_type(int32_t dtype, int32_t weight_f32, F &&f) {
  return with_type(dtype, [&](auto t) {
    if (weight_f32)
      f(t, float{});
    else
      f(t, t);
  });
}

// Blocks of the backward pass: enough to fill the GPU, few enough that their partial sums of the
// weight's gradient stay small beside the rows.
int64_t backward_blocks(int64_t rows) { return rows < 1024 ? rows : 1024; }

int check_rows(int64_t rows, int64_t cols) {
  RXMET_CHECK_ARG(rows >= 0 && cols >= 1 && cols <= RXMET_ROW_MAX,
                  "rows must be >= 0 and cols between 1 and 65536");
  RXMET_CHECK_ARG(rows < (1LL << 31), "too many rows");
  return 0;
}

}  // namespace
}  // namespace dec
}  // namespace rxmet

using namespace rxmet;
using namespace rxmet::dec;

extern "C" int rxmet_rms_quantize_forward(const void *x, int64_t x_stride, const void *residual,
                                          int64_t residual_stride, const void *weight,
                                          int32_t weight_f32, void *h, int8_t *codes, void *y,
                                          float *scales, float *rstd, int64_t rows, int64_t cols,
                                          int32_t dtype, float eps, void *stream) {
  if (int rc = check_rows(rows, cols)) return rc;
  RXMET_CHECK_ARG(dtype == RXMET_QDQ_F32 || dtype == RXMET_QDQ_F16 || dtype == RXMET_QDQ_BF16,
                  "element type must be fp32, fp16 or bf16");
  if (rows == 0) return 0;
  RXMET_CHECK_ARG(x && scales && (codes || y), "x, scales and codes or y are needed");
  RXMET_CHECK_ARG(!residual || (weight && h), "a residual needs a weight and h");
  const RowArgs a{x, residual, weight, x_stride, residual_stride, h, codes, y, scales, rstd,
                  rows, 0, static_cast<int>(cols), eps};
  auto st = static_cast<hipStream_t>(stream);
  prof::Scope scope("rms_quantize_forward", st);
  with_weight_type(dtype, weight_f32, [&](auto t, auto w) {
    with_row_shape(cols, [&](auto tpr, auto nv) {
      constexpr int block = tpr.value < 256 ? 256 : tpr.value;
      constexpr int64_t most = 1 << 21;  // rows of a launch, whose threads number below 2^32
      for (int64_t r = 0; r < rows; r += most) {
        RowArgs part = a;
        part.rows = rows - r < most ? rows - r : most;
        part.row0 = r;
        const unsigned grid = static_cast<unsigned>(cdiv(part.rows, block / tpr.value));
        rms_forward<decltype(t), decltype(w), tpr.value, nv.value><<<grid, block, 0, st>>>(part);
      }
    });
  });
  RXMET_CHECK_LAUNCH();
  return 0;
}

extern "C" int64_t rxmet_rms_quantize_backward_workspace_bytes(int64_t rows, int64_t cols) {
  return rows <= 0 || cols <= 0 ? 0 : backward_blocks(rows) * cols * 4;
}

extern "C" int rxmet_rms_quantize_backward(const void *dy, int64_t dy_stride, const void *dh,
                                           int64_t dh_stride, const void *h, int64_t h_stride,
                                           const void *weight, int32_t weight_f32,
                                           const float *rstd, void *dx, void *d_weight,
                                           int64_t rows, int64_t cols, int32_t dtype,
                                           void *workspace, void *stream) {
  if (int rc = check_rows(rows, cols)) return rc;
  RXMET_CHECK_ARG(dtype == RXMET_QDQ_F32 || dtype == RXMET_QDQ_F16 || dtype == RXMET_QDQ_BF16,
                  "element type must be fp32, fp16 or bf16");
  auto st = static_cast<hipStream_t>(stream);
  const int64_t blocks = backward_blocks(rows);
  if (rows > 0) {
    RXMET_CHECK_ARG(dy && h && weight && rstd && dx, "dy, h, weight, rstd and dx are needed");
    RXMET_CHECK_ARG(!d_weight || workspace, "the weight's gradient needs a workspace");
    const BackArgs a{dy, dh, h, weight, dy_stride, dh_stride, h_stride, rstd, dx,
                     d_weight ? static_cast<float *>(workspace) : nullptr, rows,
                     static_cast<int>(cols)};
    prof::Scope scope("rms_quantize_backward", st);
    with_weight_type(dtype, weight_f32, [&](auto t, auto w) {
      with_row_shape(cols, [&](auto tpr, auto nv) {
        rms_backward<decltype(t), decltype(w), tpr.value, nv.value>
            <<<static_cast<unsigned>(blocks), tpr.value, 0, st>>>(a);
      });
    });
    RXMET_CHECK_LAUNCH();
  }
  if (d_weight) {
    const unsigned grid = static_cast<unsigned>(cdiv(cols, kGradCols));
    with_weight_type(dtype, weight_f32, [&](auto, auto w) {
      using W = decltype(w);
      rms_weight_grad<W><<<grid, kGradCols * kGradLanes, 0, st>>>(static_cast<const float *>(workspace),
                                                static_cast<int>(blocks), static_cast<int>(cols),
                                                static_cast<W *>(d_weight));
    });
    RXMET_CHECK_LAUNCH();
  }
  return 0;
}

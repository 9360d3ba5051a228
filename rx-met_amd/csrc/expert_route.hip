// expert_route.hip — the experts of each token, their weights and the gradient of those.
//
// Mathematics.  s_e = exp(l_e - m) / sum_i exp(l_i - m) or 1 / (1 + exp(-l_e)).  The choice goes by
// c_e = fl32(s_e) + b_e, with the score computed in 64 bits, so that its rounding to fp32 does not go
// by the order of a sum or the function's last bit: the score is off by a few 2^-53 of itself (at most one for each
// of the up to 22 additions that one passes through, and some four of exp and the quotient), which changes the
// rounding of one in some 2^26 scores.
// Without a bias the logits themselves are the order.  Weights of the chosen are computed in 64 bits too (k of them,
// against E scores).
//
// Layout.  L lanes have a token, each V consecutive experts, 64 / L tokens a wave.  A candidate is
// one double in [1, 2) whose 52 bits hold the ordered bits of c_e and, below them, 1023 - e: one maximum
// compares both, and ties go to the lowest index.  Lanes sort theirs, then the best of the lanes'
// heads is taken k times.
//
// Bound: instructions, half of them for the scores and the sort ([16384, 256] fp32, bias, 8 groups, k = 8:
// 21 us, 17 MB; without groups 17, without bias and groups 11).  One lane values a group, so few large ones cost
// most: [4096, 1024] in 2 groups 52 us, in 8 27, in 64 25, without groups 18.  A few tokens: one wave's way through all
// steps (7.4 us).  Backward ([16384, 128] bf16, softmax as it is): 7.8 us.
#include "../../include/rxmet_experts.h"
#include "decoder_common.h"

namespace rxmet {
namespace dec {
namespace {

// exp(v) for v in [-700, 700], a value outside taken for the nearest: v = n ln 2 + r with ln 2 in two parts, the first
// of few bits, so that what is taken off is exact (Cody and Waite's reduction), and the series of exp(r),
// |r| <= ln(2) / 2, up to r^13 (what follows is below 2^-57 of it; up to r^11 it was 2^-46, and scores next to a border
// of fp32 fell on its other side).  The factors come as scalars: as literals each of them costs two moves where it is
// used.
struct Series {
  double ln2, ln2_rest;
  double c[12];  // 1 / 2! .. 1 / 13!
};
__device__ __forceinline__ double exp_series(double v, const Series &s) {
  v = fmin(fmax(v, -700.0), 700.0);
  const double n = __builtin_rint(v * 1.4426950408889634);
  const double r = __builtin_fma(-n, s.ln2_rest, __builtin_fma(-n, s.ln2, v));
  double p = s.c[11];
#pragma unroll
  for (int i = 10; i >= 0; --i) p = __builtin_fma(p, r, s.c[i]);
  p = __builtin_fma(__builtin_fma(p, r, 1.0), r, 1.0);
  return __builtin_ldexp(p, static_cast<int>(n));
}

// 1 / v for v in [1, 2^1020]: the hardware's estimate and two steps of Newton's rule.
__device__ __forceinline__ double inverse(double v) {
  double q = __builtin_amdgcn_rcp(v);
  q = __builtin_fma(__builtin_fma(-v, q, 1.0), q, q);
  return __builtin_fma(__builtin_fma(-v, q, 1.0), q, q);
}

struct RouteArgs {
  rxmet_router r;
  const void *logits;
  int64_t stride, tokens;
  const float *bias;
  int32_t *experts;
  float *weights;
  const float *d_weights;
  void *d_logits;
  Series series;
};

// Sums and maxima over the L lanes of a token, in all of them.
template <int L, typename F, typename S>
__device__ __forceinline__ S over_lanes(S v, F f) {
#pragma unroll
  for (int d = L / 2; d > 0; d >>= 1) v = f(v, __shfl_xor(v, d, kWave));
  return v;
}

// Lane i of 16 gets lane i + R's (in a ring) of its own 16.
template <int R>
__device__ __forceinline__ double from_lane(double v) {
  const auto b = __builtin_bit_cast(uint64_t, v);
  const unsigned lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(b), 0x120 + R, 0xf, 0xf, true);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(b >> 32), 0x120 + R, 0xf, 0xf, true);
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

template <int L>
__device__ __forceinline__ double best_of_lanes(double v) {
  v = fmax(v, from_lane<8>(v));
  v = fmax(v, from_lane<4>(v));
  v = fmax(v, from_lane<2>(v));
  v = fmax(v, from_lane<1>(v));
#pragma unroll
  for (int d = 16; d < L; d <<= 1) v = fmax(v, __shfl_xor(v, d, kWave));
  return v;
}

// fp32 bits in the order of the numbers; -0 like 0, NaN like -infinity.
__device__ __forceinline__ unsigned ordered(float v) {
  const unsigned b = __builtin_bit_cast(unsigned, v != v ? -INFINITY : v + 0.0f);
  return b >> 31 ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ double candidate(unsigned key, int e) {
  return __builtin_bit_cast(double, 0x3ffull << 52 | static_cast<uint64_t>(key) << 10 |
                                        static_cast<unsigned>(RXMET_EXPERTS_MAX - 1 - e));
}
__device__ __forceinline__ int expert_of(double c) {
  return RXMET_EXPERTS_MAX - 1 - static_cast<int>(__builtin_bit_cast(uint64_t, c) & 1023);
}

// Falling order by exchanges of (i, i ^ stride) in the order of a bitonic sort.
template <int V>
__device__ __forceinline__ void sort_falling(double (&c)[V]) {
#pragma unroll
  for (int run = 2; run <= V; run <<= 1)
#pragma unroll
    for (int d = run / 2; d > 0; d >>= 1)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int j = i ^ d;
        if (j <= i) continue;
        const double hi = fmax(c[i], c[j]), lo = fmin(c[i], c[j]);
        const bool falling = (i & run) == 0;
        c[i] = falling ? hi : lo;
        c[j] = falling ? lo : hi;
      }
}

template <typename T, int V>
__device__ __forceinline__ void load_logits(const T *p, int left, float (&x)[V]) {
  if (left >= V) {
    T u[V];
    __builtin_memcpy(u, p, sizeof(u));
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = static_cast<float>(u[v]);
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = v < left ? static_cast<float>(p[v]) : -INFINITY;
  }
}

constexpr double kNan = __builtin_nan("");

// exp(x - top) of a row's logit, top its largest and a number; rows of -infinity have no scores.
__device__ __forceinline__ double above(float x, float top, const Series &s) {
  return top == -INFINITY ? 0.0 : exp_series(static_cast<double>(x) - top, s);
}
__device__ __forceinline__ double sigmoid(float x, const Series &s) {
  return inverse(1.0 + exp_series(-static_cast<double>(x), s));
}

// Weight of a chosen logit x where all weights over the sum of the chosen are asked for: each up to the
// factor that the sum takes out.  top: the largest chosen logit.
__device__ __forceinline__ double share(int score, float x, float top, const Series &s) {
  if (x != x) return kNan;
  if (top == -INFINITY) return 0.0;
  const double d = x, t = top;
  if (score == RXMET_SCORE_SOFTMAX) return exp_series(d - t, s);
  // 1 / (1 + exp(-x)) = exp(min(x, 0)) / (1 + exp(-|x|)): relative to the largest none underflows
  return exp_series((d < 0 ? d : 0.0) - (t < 0 ? t : 0.0), s) * inverse(1.0 + exp_series(-fabs(d), s));
}

template <typename T, int L, int V>
__global__ __launch_bounds__(kWave) void route_forward(const RouteArgs a) {
  constexpr int per = kWave / L, most = L * V;
  __shared__ float s_logit[per][most], s_choice[per][most];
  __shared__ float s_value[per][RXMET_EXPERT_GROUPS_MAX];
  __shared__ int s_pick[per][RXMET_TOP_K_MAX];
  const int lane = threadIdx.x % L, slot = threadIdx.x / L;
  const int E = a.r.experts, k = a.r.top_k, G = a.r.groups;
  const bool softmax = a.r.score == RXMET_SCORE_SOFTMAX;
  const int64_t wanted = static_cast<int64_t>(blockIdx.x) * per + slot;
  const int64_t t = wanted < a.tokens ? wanted : a.tokens - 1;
  const int e0 = lane * V;
  float x[V];
  load_logits(static_cast<const T *>(a.logits) + t * a.stride + e0, E - e0, x);
  bool bad = false;  // a softmax row with a NaN or +infinity has no weights
  float top = -INFINITY;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    s_logit[slot][e0 + v] = x[v];
    bad |= !(x[v] < INFINITY);
    top = fmaxf(top, x[v]);
  }
  const auto mask = __ballot(bad) >> (threadIdx.x / L * L);
  bad = softmax && (mask & (L == 64 ? ~0ull : (1ull << L) - 1)) != 0;
  double total = 1;
  if (softmax) top = over_lanes<L>(top, [](float p, float q) { return fmaxf(p, q); });

  float c[V];  // what the choice goes by
  const bool scored = a.bias || (G > 1 && a.r.group_best == 2);
  if (scored) {
    double s[V], sum = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      s[v] = softmax ? above(x[v], top, a.series) : sigmoid(x[v], a.series);
      sum += s[v];
    }
    if (softmax) {
      total = over_lanes<L>(sum, [](double p, double q) { return p + q; });
      const double part = total != 0 ? inverse(total) : 0.0;
#pragma unroll
      for (int v = 0; v < V; ++v) s[v] *= part;
    }
    float b[V];
    if (a.bias) load_logits(a.bias + e0, E - e0, b);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      c[v] = bad || x[v] != x[v] ? static_cast<float>(kNan) : static_cast<float>(s[v]);
      if (a.bias) c[v] += b[v];
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) c[v] = x[v];
    if (softmax && !a.r.renormalize) {
      double sum = 0;
#pragma unroll
      for (int v = 0; v < V; ++v) sum += above(x[v], top, a.series);
      total = over_lanes<L>(sum, [](double p, double q) { return p + q; });
    }
  }
  unsigned long long open = ~0ull;  // groups that are chosen from
  const int size = E / G;
  if (G > 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) s_choice[slot][e0 + v] = c[v] != c[v] ? -INFINITY : c[v];
    __syncthreads();
    for (int g = lane; g < G; g += L) {
      float one = -INFINITY, two = -INFINITY;
      int at = lane % size;  // lanes start apart, for the banks
#pragma unroll 4
      for (int i = 0; i < size; ++i) {
        const float q = s_choice[slot][g * size + at];
        at = at + 1 == size ? 0 : at + 1;
        two = fmaxf(two, fminf(one, q));
        one = fmaxf(one, q);
      }
      s_value[slot][g] = a.r.group_best == 2 && size > 1 ? one + two : one;
    }
    __syncthreads();
    open = 0;
    for (int g = lane; g < G; g += L) {
      const unsigned mine = ordered(s_value[slot][g]);
      int ahead = 0;
      for (int o = 0; o < G; ++o) {
        const unsigned other = ordered(s_value[slot][o]);
        ahead += other > mine || (other == mine && o < g);
      }
      if (ahead < a.r.top_groups) open |= 1ull << g;
    }
    open = over_lanes<L>(open, [](unsigned long long p, unsigned long long q) { return p | q; });
  }
  double head[V];
  {
    int g = G > 1 ? e0 / size : 0, at = G > 1 ? e0 - g * size : 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const bool in = e0 + v < E;
      // without a bias the logits are the order, whatever the groups go by
      const unsigned key = in && (open >> (g & 63) & 1) ? ordered(a.bias ? c[v] : x[v]) : 0;
      head[v] = in ? candidate(key, e0 + v) : 1.0;
      if (G > 1 && ++at == size) at = 0, ++g;
    }
  }
  sort_falling(head);
  for (int j = 0; j < k; ++j) {
    const double best = best_of_lanes<L>(head[0]);
    if (head[0] == best) {
      s_pick[slot][j] = expert_of(best);
#pragma unroll
      for (int v = 0; v + 1 < V; ++v) head[v] = head[v + 1];
      head[V - 1] = 1.0;
    }
  }
  __syncthreads();
  float first = -INFINITY;  // largest chosen logit
  for (int j = lane; j < k; j += L) first = fmaxf(first, s_logit[slot][s_pick[slot][j]]);
  first = over_lanes<L>(first, [](float p, float q) { return fmaxf(p, q); });
  if (a.r.renormalize) {
    double sum = 0;
    for (int j = lane; j < k; j += L) sum += share(a.r.score, s_logit[slot][s_pick[slot][j]], first, a.series);
    total = over_lanes<L>(sum, [](double p, double q) { return p + q; });
  }
  if (wanted >= a.tokens) return;
  for (int j = lane; j < k; j += L) {
    const int e = s_pick[slot][j];
    const float l = s_logit[slot][e];
    double w;
    if (a.r.renormalize)
      w = total == 0 ? 0.0 : share(a.r.score, l, first, a.series) / total;
    else if (softmax)
      w = total != 0 ? above(l, top, a.series) / total : 0.0;
    else
      w = l != l ? kNan : sigmoid(l, a.series);
    a.experts[t * k + j] = e;
    a.weights[t * k + j] = static_cast<float>(bad ? kNan : w * a.r.scale);
  }
}

// In 64 bits, rounded once: where one expert has nearly all of the weight, its gradient is the difference of
// numbers that are nearly the same (in fp32 that left no digit of it: softmax as it is, logits of deviation 8).
template <typename T, int L, int V>
__global__ __launch_bounds__(kWave) void route_backward(const RouteArgs a) {
  constexpr int per = kWave / L, most = L * V;
  __shared__ float s_logit[per][most], s_grad[per][most];
  const int lane = threadIdx.x % L, slot = threadIdx.x / L;
  const int E = a.r.experts, k = a.r.top_k;
  const bool softmax = a.r.score == RXMET_SCORE_SOFTMAX;
  const int64_t wanted = static_cast<int64_t>(blockIdx.x) * per + slot;
  const int64_t t = wanted < a.tokens ? wanted : a.tokens - 1;
  const int e0 = lane * V;
  float x[V];
  load_logits(static_cast<const T *>(a.logits) + t * a.stride + e0, E - e0, x);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    s_logit[slot][e0 + v] = x[v];
    s_grad[slot][e0 + v] = 0;
  }
  const int32_t *experts = a.experts + t * k;
  const float *dw = a.d_weights + t * k;
  __syncthreads();
  auto expert = [&](int j) {
    const int e = experts[j];
    return e >= 0 && e < E ? e : -1;
  };
  auto most_of = [](float p, float q) { return fmaxf(p, q); };
  const bool dense = softmax && !a.r.renormalize;
  double p[V], inner = 0;
  float top = -INFINITY;
  bool bad = false;  // as in the forward pass: the weights are NaN, and so are their gradients
#pragma unroll
  for (int v = 0; v < V; ++v) {
    top = fmaxf(top, x[v]);
    bad |= softmax && !(x[v] < INFINITY);
  }
  bad = over_lanes<L>(static_cast<int>(bad), [](int p, int q) { return p | q; });
  auto plus = [](double p, double q) { return p + q; };
  if (dense) {
    double total = 0;
    top = over_lanes<L>(top, most_of);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      p[v] = above(x[v], top, a.series);
      total += p[v];
    }
    total = over_lanes<L>(total, plus);
    const double part = bad ? kNan : total != 0 ? inverse(total) : 0.0;
#pragma unroll
    for (int v = 0; v < V; ++v) p[v] *= part;
    for (int j = lane; j < k; j += L) {
      const int e = expert(j);
      if (e < 0) continue;
      inner += dw[j] * (above(s_logit[slot][e], top, a.series) * part);
      s_grad[slot][e] = dw[j];
    }
    inner = over_lanes<L>(inner, plus);
  } else {
    top = -INFINITY;
    double total = 0, mean = 0;
    if (a.r.renormalize) {
      for (int j = lane; j < k; j += L)
        if (expert(j) >= 0) top = fmaxf(top, s_logit[slot][expert(j)]);
      top = over_lanes<L>(top, most_of);
      for (int j = lane; j < k; j += L)
        if (expert(j) >= 0) {
          const double s = share(a.r.score, s_logit[slot][expert(j)], top, a.series);
          total += s;
          mean += s * dw[j];
        }
      total = over_lanes<L>(total, plus);
      mean = over_lanes<L>(mean, plus);
      if (total != 0) mean /= total;
    }
    for (int j = lane; j < k; j += L) {
      const int e = expert(j);
      if (e < 0) continue;
      const float l = s_logit[slot][e];
      const double rest = l != l ? kNan : sigmoid(-l, a.series);  // 1 - sigmoid(l)
      double g = 0;
      if (!a.r.renormalize)
        g = dw[j] * sigmoid(l, a.series) * rest;
      else if (total != 0)
        g = share(a.r.score, l, top, a.series) / total * (dw[j] - mean) * (softmax ? 1.0 : rest);
      s_grad[slot][e] = static_cast<float>(bad ? kNan : g * a.r.scale);
    }
  }
  __syncthreads();
  if (wanted >= a.tokens) return;
  T *out = static_cast<T *>(a.d_logits) + t * E + e0;
  float g[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    g[v] = s_grad[slot][e0 + v];
    if (dense) g[v] = static_cast<float>(p[v] * (g[v] - inner) * a.r.scale);
  }
  if (e0 + V <= E) {
    T u[V];
#pragma unroll
    for (int v = 0; v < V; ++v) u[v] = static_cast<T>(g[v]);
    __builtin_memcpy(out, u, sizeof(u));
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (e0 + v < E) out[v] = static_cast<T>(g[v]);
  }
}

// Lanes of a token and experts of a lane.  Few lanes with many experts each spend least on a token, for
// the maxima over lanes are taken for 64 / L tokens at once ([16384, 256] with groups: 16 lanes 22 us, 64 lanes
// 38); where tokens are few, a whole wave for each is done sooner ([16, 256]: 7.7 us and 11.1).
template <typename F>
void by_experts(int64_t tokens, int E, F &&f) {
  using std::integral_constant;
  auto as = [&](auto L, auto V) { f(L, V); };
  constexpr integral_constant<int, 64> whole{};
  if (tokens <= 1024 && E <= 64)
    as(whole, integral_constant<int, 1>{});
  else if (tokens <= 1024 && E <= 128)
    as(whole, integral_constant<int, 2>{});
  else if (tokens <= 1024 && E <= 256)
    as(whole, integral_constant<int, 4>{});
  else if (tokens <= 1024 && E <= 512)
    as(whole, integral_constant<int, 8>{});
  else if (E <= 64)
    as(integral_constant<int, 16>{}, integral_constant<int, 4>{});
  else if (E <= 128)
    as(integral_constant<int, 16>{}, integral_constant<int, 8>{});
  else if (E <= 256)
    as(integral_constant<int, 16>{}, integral_constant<int, 16>{});
  else if (E <= 512)
    as(integral_constant<int, 32>{}, integral_constant<int, 16>{});
  else
    as(whole, integral_constant<int, 16>{});
}

Series series() {
  constexpr long double ln2 = 0.693147180559945309417232121458176568L;
  Series s;
  s.ln2 = std::ldexp(std::floor(std::ldexp(static_cast<double>(ln2), 32)), -32);
  s.ln2_rest = static_cast<double>(ln2 - s.ln2);
  double f = 1;
  for (int i = 0; i < 12; ++i) s.c[i] = 1 / (f *= i + 2);
  return s;
}

int check_router(const rxmet_router *r, int64_t stride, int64_t tokens, int32_t dtype) {
  RXMET_CHECK_ARG(r != nullptr, "the router is missing");
  RXMET_CHECK_ARG(r->experts >= 1 && r->experts <= RXMET_EXPERTS_MAX, "there must be 1 to 1024 experts");
  RXMET_CHECK_ARG(r->score == RXMET_SCORE_SOFTMAX || r->score == RXMET_SCORE_SIGMOID, "unknown score");
  RXMET_CHECK_ARG(r->groups >= 1 && r->groups <= RXMET_EXPERT_GROUPS_MAX && r->experts % r->groups == 0,
                  "there must be 1 to 64 groups of equal length");
  RXMET_CHECK_ARG(r->top_groups >= 1 && r->top_groups <= r->groups, "top_groups must be between 1 and groups");
  RXMET_CHECK_ARG(r->group_best == 1 || r->group_best == 2, "group_best must be 1 or 2");
  RXMET_CHECK_ARG(r->top_k >= 1 && r->top_k <= RXMET_TOP_K_MAX &&
                      r->top_k <= r->top_groups * (r->experts / r->groups),
                  "top_k must be between 1 and 64 and at most the experts of the chosen groups");
  RXMET_CHECK_ARG(tokens >= 0 && tokens <= 1 << 24, "there must be at most 2^24 tokens");
  RXMET_CHECK_ARG(stride >= 0, "the rows' stride must not be negative");
  RXMET_CHECK_ARG(dtype == RXMET_QDQ_F32 || dtype == RXMET_QDQ_F16 || dtype == RXMET_QDQ_BF16,
                  "element type must be fp32, fp16 or bf16");
  return 0;
}

}  // namespace
}  // namespace dec
}  // namespace rxmet

using namespace rxmet;
using namespace rxmet::dec;

extern "C" int rxmet_route_forward(const rxmet_router *r, const void *logits, int64_t stride,
                                   const float *bias, int32_t *experts, float *weights,
                                   int64_t tokens, int32_t dtype, void *stream) {
  if (const int rc = check_router(r, stride, tokens, dtype)) return rc;
  if (tokens == 0) return 0;
  RXMET_CHECK_ARG(logits && experts && weights, "logits, experts and weights are needed");
  auto st = static_cast<hipStream_t>(stream);
  prof::Scope scope("route_forward", st);
  const RouteArgs a{*r, logits, stride, tokens, bias, experts, weights, nullptr, nullptr, series()};
  with_type(dtype, [&](auto t) {
    using T = decltype(t);
    by_experts(tokens, r->experts, [&](auto L, auto V) {
      route_forward<T, L.value, V.value><<<static_cast<unsigned>(cdiv(tokens, kWave / L.value)), kWave, 0, st>>>(a);
    });
  });
  RXMET_CHECK_LAUNCH();
  return 0;
}

extern "C" int rxmet_route_backward(const rxmet_router *r, const void *logits, int64_t stride,
                                    const int32_t *experts, const float *d_weights, void *d_logits,
                                    int64_t tokens, int32_t dtype, void *stream) {
  if (const int rc = check_router(r, stride, tokens, dtype)) return rc;
  if (tokens == 0) return 0;
  RXMET_CHECK_ARG(logits && experts && d_weights && d_logits,
                  "logits, experts and both gradients are needed");
  auto st = static_cast<hipStream_t>(stream);
  prof::Scope scope("route_backward", st);
  const RouteArgs a{*r, logits, stride, tokens, nullptr, const_cast<int32_t *>(experts), nullptr,
                    d_weights, d_logits, series()};
  with_type(dtype, [&](auto t) {
    using T = decltype(t);
    by_experts(tokens, r->experts, [&](auto L, auto V) {
      route_backward<T, L.value, V.value><<<static_cast<unsigned>(cdiv(tokens, kWave / L.value)), kWave, 0, st>>>(a);
    });
  });
  RXMET_CHECK_LAUNCH();
  return 0;
}

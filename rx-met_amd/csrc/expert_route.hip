// expert_route.hip — the experts of each token, their weights and the gradient of those.
//
// Mathematics.  s_e = exp(l_e - m) / sum_i exp(l_i - m) or 1 / (1 + exp(-l_e)).  The choice goes by
// c_e = fl32(s_e) + b_e, with the score computed in 64 bits, so that its rounding to fp32 does not go
// by the order of a sum or the function's last bit, and any evaluation that is good to a few 2^-53
// chooses the same experts.  Without a bias the logits themselves are the order.  Weights of the chosen
// are computed in 64 bits too (k of them, against E scores).
//
// Layout.  L lanes have a token, each V consecutive experts, 64 / L tokens a wave.  A candidate is
// one double in [1, 2) whose 52 bits hold the ordered bits of c_e and, below them, 1023 - e: one maximum
// compares both, and ties go to the lowest index.  Lanes sort theirs, then the best of the lanes'
// heads is taken k times.
#include "../../include/rxmet_experts.h"
#include "decoder_common.h"

namespace rxmet {
namespace dec {
namespace {

struct RouteArgs {
  rxmet_router r;
  const void *logits;
  int64_t stride, tokens;
  const float *bias;
  int32_t *experts;
  float *weights;
  const float *d_weights;
  void *d_logits;
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

// exp(x - top) of a row's logit, top its largest; rows of -infinity have no scores.
__device__ __forceinline__ double above(float x, float top) {
  const double d = x;
  return top == -INFINITY ? (x != x ? kNan : 0.0) : exp(d - top);
}

// Weight of a chosen logit x over `total` where all weights over the sum of the chosen are asked for:
// each up to the factor that the sum takes out.  top: the largest chosen logit.
__device__ __forceinline__ double share(int score, float x, float top) {
  if (top == -INFINITY) return x != x ? kNan : 0.0;
  const double d = x, t = top;
  if (score == RXMET_SCORE_SOFTMAX) return exp(d - t);
  // 1 / (1 + exp(-x)) = exp(min(x, 0)) / (1 + exp(-|x|)): relative to the largest none underflows
  return exp((d < 0 ? d : 0.0) - (t < 0 ? t : 0.0)) / (1 + exp(-fabs(d)));
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
      const double d = x[v];
      s[v] = softmax ? above(x[v], top) : 1 / (1 + exp(-d));
      sum += s[v];
    }
    if (softmax) {
      total = over_lanes<L>(sum, [](double p, double q) { return p + q; });
#pragma unroll
      for (int v = 0; v < V; ++v) s[v] = total != 0 ? s[v] / total : 0.0;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      c[v] = static_cast<float>(s[v]);
      if (a.bias && e0 + v < E) c[v] += a.bias[e0 + v];
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) c[v] = x[v];
    if (softmax && !a.r.renormalize) {
      double sum = 0;
#pragma unroll
      for (int v = 0; v < V; ++v) sum += above(x[v], top);
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
      for (int i = 0; i < size; ++i) {
        int at = i + lane;  // lanes start apart, for the banks
        at = g * size + (at < size ? at : at % size);
        const float q = s_choice[slot][at];
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
#pragma unroll
      for (int v = 0; v + 1 < V; ++v) head[v] = head[v + 1];
      head[V - 1] = 1.0;
      s_pick[slot][j] = expert_of(best);
    }
  }
  __syncthreads();
  float first = -INFINITY;  // largest chosen logit
  for (int j = lane; j < k; j += L) first = fmaxf(first, s_logit[slot][s_pick[slot][j]]);
  first = over_lanes<L>(first, [](float p, float q) { return fmaxf(p, q); });
  if (a.r.renormalize) {
    double sum = 0;
    for (int j = lane; j < k; j += L) sum += share(a.r.score, s_logit[slot][s_pick[slot][j]], first);
    total = over_lanes<L>(sum, [](double p, double q) { return p + q; });
  }
  if (wanted >= a.tokens) return;
  for (int j = lane; j < k; j += L) {
    const int e = s_pick[slot][j];
    const float l = s_logit[slot][e];
    double w;
    if (a.r.renormalize)
      w = total == 0 ? 0.0 : share(a.r.score, l, first) / total;
    else if (softmax)
      w = total != 0 ? above(l, top) / total : 0.0;
    else
      w = 1 / (1 + exp(-static_cast<double>(l)));
    a.experts[t * k + j] = e;
    a.weights[t * k + j] = static_cast<float>(bad ? kNan : w * a.r.scale);
  }
}

// One token of L lanes: the chosen experts' parts in 64 bits, the others' (softmax as it is) in fp32.
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
  float top = -INFINITY;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    s_logit[slot][e0 + v] = x[v];
    s_grad[slot][e0 + v] = 0;
    top = fmaxf(top, x[v]);
  }
  const int32_t *experts = a.experts + t * k;
  const float *dw = a.d_weights + t * k;
  const double scale = a.r.scale;
  __syncthreads();
  auto expert = [&](int j) {
    const int e = experts[j];
    return e >= 0 && e < E ? e : -1;
  };
  auto plus = [](double p, double q) { return p + q; };
  const bool dense = softmax && !a.r.renormalize;
  double total = 0, inner = 0;
  if (dense) {
    top = over_lanes<L>(top, [](float p, float q) { return fmaxf(p, q); });
#pragma unroll
    for (int v = 0; v < V; ++v) total += above(x[v], top);
    total = over_lanes<L>(total, plus);
    for (int j = lane; j < k; j += L) {
      const int e = expert(j);
      if (e < 0) continue;
      if (total != 0) inner += dw[j] * above(s_logit[slot][e], top) / total;
      s_grad[slot][e] = dw[j];
    }
  } else if (a.r.renormalize) {
    top = -INFINITY;
    for (int j = lane; j < k; j += L)
      if (expert(j) >= 0) top = fmaxf(top, s_logit[slot][expert(j)]);
    top = over_lanes<L>(top, [](float p, float q) { return fmaxf(p, q); });
    for (int j = lane; j < k; j += L)
      if (expert(j) >= 0) total += share(a.r.score, s_logit[slot][expert(j)], top);
    total = over_lanes<L>(total, plus);
    for (int j = lane; j < k; j += L)
      if (expert(j) >= 0 && total != 0) inner += dw[j] * share(a.r.score, s_logit[slot][expert(j)], top) / total;
  }
  inner = over_lanes<L>(inner, plus);
  if (!dense)
    for (int j = lane; j < k; j += L) {
      const int e = expert(j);
      if (e < 0) continue;
      const double l = s_logit[slot][e], s = 1 / (1 + exp(-l));
      double g;
      if (a.r.renormalize) {
        g = total != 0 ? share(a.r.score, s_logit[slot][e], top) / total * (dw[j] - inner) : 0.0;
        if (!softmax) g /= 1 + exp(l);
      } else {
        g = dw[j] * s / (1 + exp(l));
      }
      s_grad[slot][e] = static_cast<float>(g * scale);
    }
  __syncthreads();
  if (wanted >= a.tokens) return;
  T *out = static_cast<T *>(a.d_logits) + t * E + e0;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (e0 + v >= E) break;
    float g = s_grad[slot][e0 + v];
    if (dense)
      g = static_cast<float>(
          (total != 0 ? above(x[v], top) / total : 0.0) * (g - inner) * scale);
    out[v] = static_cast<T>(g);
  }
}

// Lanes and experts of a lane by the number of experts.
template <typename T, typename F>
void by_experts(int E, F &&f) {
  using std::integral_constant;
  if (E <= 64)
    f(integral_constant<int, 16>{}, integral_constant<int, 4>{});
  else if (E <= 128)
    f(integral_constant<int, 16>{}, integral_constant<int, 8>{});
  else if (E <= 256)
    f(integral_constant<int, 16>{}, integral_constant<int, 16>{});
  else if (E <= 512)
    f(integral_constant<int, 32>{}, integral_constant<int, 16>{});
  else
    f(integral_constant<int, 64>{}, integral_constant<int, 16>{});
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
  const RouteArgs a{*r, logits, stride, tokens, bias, experts, weights, nullptr, nullptr};
  with_type(dtype, [&](auto t) {
    using T = decltype(t);
    by_experts<T>(r->experts, [&](auto L, auto V) {
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
                    d_weights, d_logits};
  with_type(dtype, [&](auto t) {
    using T = decltype(t);
    by_experts<T>(r->experts, [&](auto L, auto V) {
      route_backward<T, L.value, V.value><<<static_cast<unsigned>(cdiv(tokens, kWave / L.value)), kWave, 0, st>>>(a);
    });
  });
  RXMET_CHECK_LAUNCH();
  return 0;
}

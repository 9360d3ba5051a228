// kv_attention.hip — attention over the paged int8 cache.
//
// Mathematics.  For a query row q of head g (cache head g / (q_heads / heads)) and the cached
// tokens t that it sees: s_t = (q . k_t) * ks * scale, out = sum_t softmax(s)_t * vs * v_t, with the codes k_t, v_t and
// their pages' scales ks, vs.  One pass over the tokens keeps the running maximum m, the sum l of
// 2^(s - m) (log2 e is part of the scale) and the weighted sum of the value codes; m, l and the
// sums are fp32.
//
// Precision.  An int8 code is exact in fp16, so both products run on the fp16 matrix instruction
// with the codes themselves and the scales stay outside.  A query row is brought to [-2, 2) by a power
// of two and keeps all bits of the elements down to 2^-14 of its largest.  What fp16 drops of smaller
// ones decides nothing but where the keys' codes are 0 at the large ones; where it could change a score
// by more than 2^-14, an eighth of the weights' rounding, the tokens are taken again with further products
// that add it (Rest).  The weights are rounded to fp16 (11 bits) once, with their value
// scales in them: as 2^(s - m) vs / 2^d, where 2^d is a running reference of the row's own, like m, that
// follows the largest 2^(s - m) vs which the row has seen.  It never falls below what the sums hold, so
// that they stay finite beside pages of any scale (a page of zeros has 2^-119), and pages that the
// row does not see do not move it.  The heaviest weight is a power of two so, and not rounded: fp16 results are
// 3 to 11 % further from 64 bits than fp32 weights leave them, with 2^d a whole power 24 to 84 %.  The weighted
// sums are in units of 2^d, l in units of 1.
// Weights and l carry a common power of two (kLift): without it a weight 2^-25 of its
// row's largest would round to 0 in fp16, and many such beside one large one make a sum that counts.
//
// Layout.  With mfma 16x16x32 (lane = (col, g), col = lane % 16, g = lane / 16) the first product is
// taken as S^T = K Q^T on 64 tokens: row i of tile t stands for token 16 * (i / 4) + 4 t + i % 4, so that
// lane (col, g) gets the scores of query col for the 16 consecutive tokens 16 g..16 g + 15.  The second
// product is O^T = V^T P^T; its operand from P is what the lane holds already, and its operand
// from V is 16 consecutive bytes, as values lie dimension by dimension.  Nothing crosses lanes but the row maximum.
//
// Bound and measured (bf16 queries, dim 128, pages of 64).  attn_rows: HBM, the cache's bytes: 64 sequences
// of 0 to 16384 tokens, 8 heads, 64 query heads: 1356 MB in 283 us (4.8 TB/s; a copy of 2 GiB reaches 4.9); two
// of 32768 and 16679 tokens, 32 query heads: 101 MB in 25 us and 4.7 us for the join of 64 chunks.  attn_tile: the issue of a
// SIMD's two waves: counted over the whole launch, its ends with it, the matrix unit is busy for 35 % and the
// vector unit (exponentials, conversions) for 46 % of the time: 204 GFLOP in 237 to 258 us by card, 860 to 790
// TFLOP/s, where a large library product reaches 1385.  64 rows a wave (half the LDS reads) spill and take 512 us;
// waves half a turn apart, a higher priority for the products, and products placed among the
// exponentials by hand change nothing or cost 4 to 6 %; weights as two fp16 numbers, which keep 22 bits, cost
// 32 % (and 2 % in attn_rows).
#include <type_traits>
#include <utility>

#include "kv_cache.h"
#include "mfma_frag.h"

namespace rxmet {
namespace dec {
namespace {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

constexpr int kRows = 16;   // query rows of a workgroup: one column of the matrix instruction each
constexpr int kGroup = 64;  // tokens that a wave takes at a time
constexpr int kWaves = 4;
// log2 of the weights' factor: the largest is 2^15 (attn_tile's may be 2^8 above its reference).
constexpr float kLiftRows = 15.0f, kLiftTile = 7.0f;
// Least reference d, below log2 of every scale, and the least log2(vs) - d that is told apart: with it a
// weight's rounding gives 0, and l, which takes the factor out again, keeps its bits.
constexpr float kLeast = -200.0f, kApart = -48.0f;

struct AttnArgs {
  Pages g;
  const int32_t *lengths, *cu;
  int queries;
  const void *q;
  int64_t stride_t, stride_h;
  int q_heads, group;  // group = q_heads / heads
  float scale;         // with log2 e
  int causal;
  int window, chunk, splits, row_tiles, cap;
  void *out;
  float *part, *stats;  // [splits, queries * q_heads, D] and [.., 2]: averages, maxima and l, where splits > 1
};

// Eight codes (two words) as fp16: 0x6400 | u is 1024 + u, and u is the code + 128.
__device__ __forceinline__ v8h codes_f16(unsigned w0, unsigned w1) {
  union {
    unsigned u[4];
    v2h h[4];
    v8h v;
  } r;
  w0 ^= 0x80808080u;
  w1 ^= 0x80808080u;
  r.u[0] = __builtin_amdgcn_perm(0x64646464u, w0, 0x04010400u);
  r.u[1] = __builtin_amdgcn_perm(0x64646464u, w0, 0x04030402u);
  r.u[2] = __builtin_amdgcn_perm(0x64646464u, w1, 0x04010400u);
  r.u[3] = __builtin_amdgcn_perm(0x64646464u, w1, 0x04030402u);
  const v2h bias = {static_cast<_Float16>(1152.0f), static_cast<_Float16>(1152.0f)};
#pragma unroll
  for (int k = 0; k < 4; ++k) r.h[k] -= bias;
  return r.v;
}

__device__ __forceinline__ v4f mfma_f16(v8h a, v8h b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// The wave's number, known to be the same for all of its lanes.
__device__ __forceinline__ int wave_id() {
  return __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
}

// Over the four lanes that share a column.
__device__ __forceinline__ float col_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, kWave));
  return fmaxf(v, __shfl_xor(v, 32, kWave));
}
__device__ __forceinline__ float col_sum(float v) {
  v += __shfl_xor(v, 16, kWave);
  return v + __shfl_xor(v, 32, kWave);
}

// Most tokens of a sequence and most query rows of a call: sums of two of them stay in int32.
constexpr int kMost = 1 << 29;

// Tokens [lo, hi) that query i of n sees.  Of tokens past `cap` (the table's end) one is kept: it
// has no page, and makes the row NaN.
struct Seen {
  int lo, hi;
};
__device__ __forceinline__ Seen seen_by(const AttnArgs &a, int length, int n, int i) {
  const int pos = length - n + i;
  Seen s{0, length};
  if (a.causal && pos + 1 < s.hi) s.hi = pos + 1;
  if (a.window > 0 && pos >= a.window) s.lo = pos - a.window + 1;
  if (s.hi > a.cap + 1) {
    if (s.lo > a.cap) s.lo = a.cap;
    s.hi = a.cap + 1;
  }
  return s;
}

// The sequence of a workgroup: its query rows (n queries of `group` heads) and its tokens.
struct Sequence {
  int length, q0, n, rows;
};
__device__ __forceinline__ Sequence sequence_of(const AttnArgs &a, int b) {
  Sequence s;
  s.length = a.lengths[b];
  s.q0 = a.cu ? a.cu[b] : b;
  s.n = a.cu ? a.cu[b + 1] - s.q0 : 1;
  if (s.q0 < 0 || s.q0 >= a.queries) s.n = 0;
  if (s.n > a.queries - s.q0) s.n = a.queries - s.q0;
  s.rows = s.n > 0 ? s.n * a.group : 0;
  return s;
}

// What a workgroup computes.  Neighbouring workgroups have neighbouring heads (of eight heads each
// stays on one XCD, whose L2 then holds its pages), then chunks, then row tiles, and the longest
// sequences come first, so that short ones fill the end of the launch ([2048 + 1226 queries], 256-row tiles:
// 281 us by sequence and head, 235 us so).  Up to 64 sequences are ranked; more even out by themselves.
struct Job {
  int head, split, slot, b;
};
__device__ __forceinline__ Job job_of(const AttnArgs &a) {
  Job j;
  unsigned i = blockIdx.x;
  j.head = i % a.g.c.heads;
  i /= a.g.c.heads;
  j.split = i % a.splits;
  i /= a.splits;
  j.slot = i % a.row_tiles;
  j.b = i / a.row_tiles;
  const int seqs = a.g.t.seqs;
  if (seqs > 1 && seqs <= kWave) {
    const int lane = threadIdx.x % kWave;
    const int mine = lane < seqs ? a.lengths[lane] : INT32_MIN;
    int rank = 0;  // sequences before this lane's
    for (int k = 0; k < seqs; ++k) {
      const int other = __builtin_amdgcn_readlane(mine, k);
      rank += other > mine || (other == mine && k < lane);
    }
    j.b = __builtin_ctzll(__ballot(lane < seqs && rank == j.b));
  }
  return j;
}

// The id of the page that holds token t, as it stands in the table; -1 past the table, and 0 past
// `end`, where nothing is seen and any page may be read.
__device__ __forceinline__ int page_id(const AttnArgs &a, const int32_t *ids, int t, int end, int shift) {
  if (t >= end) return 0;
  const int p = t >> shift;
  return p < a.g.t.cols ? ids[p] : -1;
}
__device__ __forceinline__ bool in_cache(const AttnArgs &a, int id) {
  return static_cast<unsigned>(id) < static_cast<unsigned>(a.g.c.pages);
}

// Pieces of a query row (eight elements each, `at(i)` the place of piece i) as operands of the
// matrix instruction, brought to [-2, 2) by 2^-e; e returned.  A row with a NaN or an infinity is NaN throughout.
// `join` takes the NaN-keeping maximum over the lanes that share the row.
template <typename T, int N, typename At, typename Join>
__device__ __forceinline__ int load_query(const T *q, bool valid, At at, Join join, v8h (&out)[N]) {
  float f[N][8];
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (valid) {
      load8(q + at(i), f[i]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[i][e] = 0.0f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) top = nan_max(top, fabsf(f[i][e]));
  }
  top = join(top);
  const bool good = top <= 3.402823466e38f;
  const int e2 = good && top > 0.0f ? __builtin_amdgcn_frexp_expf(top) - 1 : 0;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      out[i][e] = static_cast<_Float16>(good ? __builtin_amdgcn_ldexpf(f[i][e], -e2) : nanf32());
  return e2;
}

// What fp16 drops of query rows.  A pass over the tokens keeps the largest factor f from products to
// scores; only if it could matter with f is it found what the rows did lose, and only if that does are the
// tokens taken a second time, with the lost part as further products: in levels, each at 2^24 times the size
// of the one before, so that four of them reach 2^-121 of a row's largest element.  The rows and, for attn_rows, the
// codes are read again for it: it is rare, and registers are not.
template <typename T, int D>
struct Rest {
  static constexpr float kMissed = 0x1p-14f;  // log2 units of a score
  static constexpr int kLevels = 4, kStep = 24;
  static constexpr float kUnit = 1 << kStep;

  // Whether scores of up to f times a product need it.  q: pieces of the lane's row at at(c), c < n;
  // join: as in load_query, over `sharing` lanes.
  template <typename At, typename Join>
  __device__ __forceinline__ static bool counts(float f, const T *q, int e2, bool valid, int n, At at, int sharing,
                                                Join join) {
    if (!__any(127.0f * D * 0x1p-25f * f > kMissed)) return false;  // D subnormal elements
    float lost = 0.0f;
#pragma unroll 1
    for (int c = 0; c < n; ++c) {
      float x[8];
      load8(q + at(c), x);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float v = __builtin_amdgcn_ldexpf(x[e], -e2);
        lost += fabsf(v - static_cast<float>(static_cast<_Float16>(v)));
      }
    }
    // a row that is not finite has NaN here, and NaN in its products
    return __any(valid && 127.0f * sharing * join(lost) * f > kMissed);
  }

  // How many levels a group of tokens needs: an element leaves at most 2^-25 of the last level's unit.
  __device__ __forceinline__ static int levels(float f) {
    int level = 0;
    while (level < kLevels && __any(__builtin_amdgcn_ldexpf(127.0f * D * f, -25 - kStep * level) > kMissed)) ++level;
    return level;
  }

  // Eight elements at q as the operand of a level; level 0: the row as load_query gives it.
  __device__ __forceinline__ static v8h operand(const T *q, int e2, int level) {
    float f[8];
    load8(q, f);
    v8h r;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float v = __builtin_amdgcn_ldexpf(f[e], -e2);
      v += 0.0f * v;  // an infinity becomes NaN
#pragma unroll 1
      for (int k = 0; k < level; ++k)
        v = (v - static_cast<float>(static_cast<_Float16>(v))) * kUnit;
      r[e] = static_cast<_Float16>(v);
    }
    return r;
  }
};

// Sixteen query rows of one cache head, one chunk of their tokens.  The waves take groups of 64
// tokens in turn and join their sums in LDS.
template <typename T, int D>
__global__ __launch_bounds__(256, D <= 64 ? 4 : D <= 128 ? 3 : 2) void attn_rows(const AttnArgs a) {
  constexpr int NC = D / 64, NU = D / 16, pitch = D + 4;
  __shared__ float s_acc[kWaves][kRows][pitch];
  __shared__ float s_m[kWaves][kRows], s_l[kWaves][kRows];
  const int lane = threadIdx.x % kWave, wave = wave_id();
  const int col = lane % 16, g = lane / 16;
  const Job job = job_of(a);
  const int split = job.split, head = job.head;
  const int P = a.g.c.page_size, shift = __builtin_ctz(P), H = a.g.c.heads, G = a.group;
  const Sequence seq = sequence_of(a, job.b);
  const int rows = seq.rows;
  const int32_t *ids = a.g.t.ids + job.b * a.g.t.stride;
  for (int rt = job.slot; rt * kRows < rows; rt += a.row_tiles) {
    const int row = rt * kRows + col;
    const bool valid = row < rows;
    const Seen me = seen_by(a, seq.length, seq.n, valid ? row / G : seq.n - 1);
    const Seen top = seen_by(a, seq.length, seq.n, rt * kRows / G);  // the tile's first and last query
    const int last = rt * kRows + kRows - 1 < rows ? rt * kRows + kRows - 1 : rows - 1;
    const Seen bot = seen_by(a, seq.length, seq.n, last / G);
    const unsigned wide = me.hi > me.lo ? me.hi - me.lo : 0;
    const int begin = (top.lo & ~(kGroup - 1)) + split * a.chunk;
    const int end = split == a.splits - 1 || bot.hi < begin + a.chunk ? bot.hi : begin + a.chunk;

    v8h q[2 * NC];
    const T *qp = static_cast<const T *>(a.q) + (seq.q0 + (valid ? row / G : 0)) * a.stride_t +
                  (head * G + (valid ? row % G : 0)) * a.stride_h;
    const int e2 = load_query(
        qp, valid, [&](int i) { return 64 * (i / 2) + 16 * g + 8 * (i % 2); },
        [](float v) {
          v = nan_max(v, __shfl_xor(v, 16, kWave));
          return nan_max(v, __shfl_xor(v, 32, kWave));
        },
        q);
    const float q_scale = __builtin_amdgcn_ldexpf(a.scale, e2);

    v4f acc[NU];
    float m, l, d;  // maximum, sum, and log2 of the largest weight times scale, relative to m
    float f_most;  // largest factor from products to scores
    auto rest_at = [](int c) { return 32 * (c & ~1) + 8 * (c & 1); };

    auto step = [&](auto all_bits, int t0, int ik, int iv) {  // one group of 64 tokens
      const int tk = t0 + 16 * (col >> 2), tv = t0 + 16 * g;
      const int64_t kat = static_cast<int64_t>(in_cache(a, ik) ? ik : 0) * H + head;
      const int64_t vat = static_cast<int64_t>(in_cache(a, iv) ? iv : 0) * H + head;
      const int8_t *kp = a.g.c.k + kat * P * D + ((tk & (P - 1)) + (col & 3)) * D + 16 * g;
      const int8_t *vp = a.g.c.v + vat * P * D + col * P + (tv & (P - 1));
      uint4 kw[4][NC], vw[NU];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int c = 0; c < NC; ++c)
          kw[t][c] = *reinterpret_cast<const uint4 *>(kp + 4 * t * D + 64 * c);
      float ks = a.g.c.k_scale[vat], vs = a.g.c.v_scale[vat];
#pragma unroll
      for (int u = 0; u < NU; ++u) vw[u] = *reinterpret_cast<const uint4 *>(vp + 16 * u * P);
      if (!in_cache(a, iv)) ks = vs = nanf32();
      if (tv >= bot.hi) ks = vs = 0.0f;

      const float f = ks * q_scale;
      v4f s[4];
#pragma unroll
      for (int t = 0; t < 4; ++t) s[t] = v4f{0, 0, 0, 0};
      if constexpr (all_bits.value) {
        const int levels = Rest<T, D>::levels(fabsf(f));
#pragma unroll 1
        for (int level = 0; level <= levels; ++level) {
#pragma unroll
          for (int t = 0; t < 4; ++t) s[t] *= Rest<T, D>::kUnit;
#pragma unroll 1
          for (int c = 0; c < 2 * NC; ++c) {
            const v8h r = Rest<T, D>::operand(qp + 16 * g + rest_at(c), e2, level);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              const uint2 w = *reinterpret_cast<const uint2 *>(kp + 4 * t * D + rest_at(c));
              s[t] = mfma_f16(codes_f16(w.x, w.y), r, s[t]);
            }
          }
        }
#pragma unroll 1
        for (int level = 1; level <= levels; ++level)
#pragma unroll
          for (int t = 0; t < 4; ++t) s[t] *= 1.0f / Rest<T, D>::kUnit;
      } else {
        f_most = fmaxf(f_most, fabsf(f));
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            s[t] = mfma_f16(codes_f16(kw[t][c].x, kw[t][c].y), q[2 * c], s[t]);
            s[t] = mfma_f16(codes_f16(kw[t][c].z, kw[t][c].w), q[2 * c + 1], s[t]);
          }
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) s[t] *= f;
      if (t0 < bot.lo || t0 + kGroup > top.hi) {  // some row does not see all 64
        asm volatile("");  // stays a branch: few groups need it
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int tok = tv + 4 * t + r;
            s[t][r] = static_cast<unsigned>(tok - me.lo) < wide ? s[t][r] : -INFINITY;
          }
        if (tv + 16 <= me.lo || tv >= me.hi) vs = 0.0f;  // 0 times a hidden page's NaN is no 0
      }
      const float lv = __builtin_amdgcn_logf(fabsf(vs));  // the lane's 16 tokens lie in one page
      float own = -INFINITY;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) own = fmaxf(own, s[t][r]);
      if (__any(own > m || (own - m) + lv > d)) {  // a row's maximum or reference moves
        const float high = fmaxf(m, col_max(own));
        const float base = high == -INFINITY ? 0.0f : high, delta = m - base;
        m = high;
        const float next = fmaxf(fmaxf(d + delta, col_max((own - base) + lv)), kLeast);
        const float fix = exp2f((d - next) + delta);
        d = next;
        l *= exp2f(delta);
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[u][r] *= fix;
      }
      float part = lv - d;
      part = part < kApart ? kApart : part;  // a NaN stays one
      const float lifted = (m == -INFINITY ? 0.0f : m) - (kLiftRows + part);
      float sum = 0.0f;
      v8h p[2];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float e = __builtin_amdgcn_exp2f(s[t][r] - lifted);
          sum += e;
          p[t / 2][4 * (t % 2) + r] = static_cast<_Float16>(e);
        }
      l += sum * __builtin_amdgcn_exp2f(-part);
      if (__any(vs < 0.0f)) {  // such scales come from elsewhere than the append
        if (vs < 0.0f) p[0] = -p[0], p[1] = -p[1];
      }
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        acc[u] = mfma_f16(codes_f16(vw[u].x, vw[u].y), p[0], acc[u]);
        acc[u] = mfma_f16(codes_f16(vw[u].z, vw[u].w), p[1], acc[u]);
      }
    };
    auto pass = [&](auto all_bits) {
#pragma unroll
      for (int u = 0; u < NU; ++u) acc[u] = v4f{0, 0, 0, 0};
      m = -INFINITY;
      l = f_most = 0.0f;
      d = kLeast;
      // the ids of a group's pages are on their way while the group before is computed
      const int t_first = begin + wave * kGroup;
      int ik = page_id(a, ids, t_first + 16 * (col >> 2), end, shift);
      int iv = page_id(a, ids, t_first + 16 * g, end, shift);
      for (int t0 = t_first; t0 < end; t0 += kWaves * kGroup) {
        const int t1 = t0 + kWaves * kGroup;
        const int nk = page_id(a, ids, t1 + 16 * (col >> 2), end, shift);
        const int nv = page_id(a, ids, t1 + 16 * g, end, shift);
        step(all_bits, t0, ik, iv);
        ik = nk;
        iv = nv;
      }
    };
    pass(std::false_type{});
    if (Rest<T, D>::counts(f_most, qp + 16 * g, e2, valid, 2 * NC, rest_at, 4, [](float v) { return col_max(v); }))
      pass(std::true_type{});

    // The four waves' sums on one maximum, as averages: each sum is divided by the row's whole l before
    // anything is added to it, because values near the type's largest have no room for more.
    l = col_sum(l);
    if (g == 0) s_m[wave][col] = m, s_l[wave][col] = l;
    __syncthreads();
    float all = s_m[0][col], total = 0.0f;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) all = fmaxf(all, s_m[w][col]);
    const float base = all == -INFINITY ? 0.0f : all;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += s_l[w][col] * __builtin_amdgcn_exp2f(s_m[w][col] - base);
    const float unit = fmaxf(d + (m - base), -1000.0f);  // log2 of what this wave's sums count
    // of row r's values in `out` or, for this chunk, in `part` and `stats`
    auto place_of = [&](int r) {
      return static_cast<int64_t>(seq.q0 + r / G) * a.q_heads + head * G + r % G;
    };
    const int64_t chunk0 = static_cast<int64_t>(split) * a.queries * a.q_heads;
    if (a.splits > 1 && wave == 0 && g == 0 && valid) {
      float *stats = a.stats + 2 * (chunk0 + place_of(row));
      stats[0] = all, stats[1] = total;
    }
    const float whole = rintf(unit);
    const float mine = total == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(unit - whole) / total;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      v4f o = acc[u] * mine;
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = __builtin_amdgcn_ldexpf(o[r], static_cast<int>(whole));
      *reinterpret_cast<v4f *>(&s_acc[wave][col][16 * u + 4 * g]) = o;
    }
    __syncthreads();
    constexpr int per = D / 16;  // elements of a thread: 16 threads a row
    const int r = threadIdx.x / 16, d0 = threadIdx.x % 16 * per;
    const int orow = rt * kRows + r;
    if (orow < rows) {
      const int64_t place = place_of(orow);
      float o[per];
#pragma unroll
      for (int e = 0; e < per; ++e)
        o[e] = s_acc[0][r][d0 + e] + s_acc[1][r][d0 + e] + s_acc[2][r][d0 + e] +
               s_acc[3][r][d0 + e];
      if (a.splits == 1) {
        T *out = static_cast<T *>(a.out) + place * D + d0;
#pragma unroll
        for (int e = 0; e < per; ++e) out[e] = static_cast<T>(o[e]);
      } else if (begin < end) {
        float *part = a.part + (chunk0 + place) * D + d0;
#pragma unroll
        for (int e = 0; e < per; ++e) part[e] = o[e];
      }
    }
    __syncthreads();  // the next tile writes the LDS again
  }
}

// ---------------------------------------------------------------------------------------------
// Many query rows: 32 W rows of one cache head, 32 to a wave, on mfma 32x32x16 (lane = (col, h),
// col = lane % 32, h = lane / 32).  The workgroup brings 64 tokens at a time into LDS as fp16, so that the
// codes are converted once for all the rows, while the next 64 are on their way.  As above,
// S^T = K Q^T with row i of tile t standing for token 32 t + 16 * (i / 4 % 2) + 4 * (i / 8) + i % 4, so that a lane holds
// 16 consecutive tokens of one page a tile, and the weights are the second product's operand
// where they are.  The weights are 2^(s f - m + log2(vs) - d): vs costs nothing for each weight, and l takes
// it out again once for 16 of them.  The references m and d follow the largest only when that is more
// than 8 above them, which leaves weights below 2^8 and spares most rescalings of the sums.
typedef float v16f __attribute__((ext_vector_type(16)));

__device__ __forceinline__ v16f mfma32_f16(v8h a, v8h b, v16f c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Waves of a SIMD, least and most: with room for more the compiler saves registers that buy nothing.
constexpr int tile_waves(int dim) { return dim <= 64 ? 3 : dim <= 128 ? 2 : 1; }

// Products, each with an operand from LDS that is read AHEAD products before: load(i) and multiply(i, operand),
// i a constant.  The order is pinned: left to itself the compiler reads, waits and multiplies one by one where
// the rest of a kernel needs many registers ([2048 + 1226 queries]: 257 us, so 237).
template <int AHEAD, int... I, typename Load, typename Multiply>
__device__ __forceinline__ void feed_products(std::integer_sequence<int, I...>, Load load, Multiply multiply) {
  v8h next[AHEAD];
  auto fill = [&](auto i) {
    if constexpr (i.value < static_cast<int>(sizeof...(I))) next[i.value % AHEAD] = load(i);
  };
  (((void)(I < AHEAD ? (fill(std::integral_constant<int, I>{}), 0) : 0)), ...);
  ((multiply(std::integral_constant<int, I>{}, next[I % AHEAD]), fill(std::integral_constant<int, I + AHEAD>{}),
    __builtin_amdgcn_sched_barrier(0)), ...);
}

template <typename T, int D, int W, bool WIDE>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(tile_waves(D), tile_waves(D)))) void attn_tile(
    const AttnArgs a) {
  constexpr int tile = 32 * W, threads = 64 * W;
  constexpr int KC = D / 16, NU = D / 32;   // steps of the first product, tiles of the second
  constexpr int kp = kGroup + 1, vp = D + 1;  // pitches in units of 16 bytes
  constexpr int all = D * kGroup / 16;        // pieces of 16 codes of the keys, and of the values
  constexpr int pieces = (all + threads - 1) / threads;
  constexpr int ahead = D <= 64 ? 2 : 4;      // operands that are read before they are needed
  struct Stage {
    uint4 k[D / 8 * kp];  // [8 dimensions][row of the tiles]
    uint4 v[8 * vp];      // [8 tokens][dimension]
    float ks[4], lv[4];   // of 16 tokens each: key scale, log2 of the value scale
  };
  __shared__ Stage stage[2];
  __shared__ int s_again[W];
  const int tid = threadIdx.x, lane = tid % kWave, wave = wave_id();
  const int col = lane % 32, h = lane / 32;
  const Job job = job_of(a);
  const int split = job.split, head = job.head;
  const int P = a.g.c.page_size, shift = __builtin_ctz(P), H = a.g.c.heads, G = a.group;
  const Sequence seq = sequence_of(a, job.b);
  const int rows = seq.rows;
  const int32_t *ids = a.g.t.ids + job.b * a.g.t.stride;
  // where a thread's pieces lie in a page: keys of token i / (D / 16), values of tokens 16 * (i % 4)
  const int page_bytes = H * P * D;
  unsigned kat[pieces], vat[pieces];
#pragma unroll
  for (int j = 0; j < pieces; ++j) {
    const int i = tid + threads * j;
    kat[j] = head * P * D + (i / (D / 16) & (P - 1)) * D + i % (D / 16) * 16;
    vat[j] = head * P * D + i / 4 * P + (i % 4 * 16 & (P - 1));
  }
  // the last rows see the most tokens: they go first
  for (int rt = a.row_tiles - 1 - job.slot; rt * tile < rows; rt += a.row_tiles) {
    const int r0 = rt * tile, w0 = r0 + wave * 32;
    auto seen = [&](int r) { return seen_by(a, seq.length, seq.n, (r < rows ? r : rows - 1) / G); };
    const Seen top = seen(r0), bot = seen(r0 + tile - 1), wtop = seen(w0), wbot = seen(w0 + 31);
    const int row = w0 + col;
    const bool valid = row < rows;
    const Seen me = seen(row);
    const unsigned wide = me.hi > me.lo ? me.hi - me.lo : 0;
    const int begin = (top.lo & ~(kGroup - 1)) + split * a.chunk;
    const int end = split == a.splits - 1 || bot.hi < begin + a.chunk ? bot.hi : begin + a.chunk;

    v8h q[KC];
    const T *qp = static_cast<const T *>(a.q) + (seq.q0 + (valid ? row / G : 0)) * a.stride_t +
                  (head * G + (valid ? row % G : 0)) * a.stride_h;
    const int e2 = load_query(
        qp, valid, [&](int i) { return 16 * i + 8 * h; },
        [](float v) { return nan_max(v, __shfl_xor(v, 32, kWave)); }, q);
    if (a.scale < 0.0f) {  // the maximum is taken before the scale
#pragma unroll
      for (int c = 0; c < KC; ++c) q[c] = -q[c];
    }
    const float q_scale = __builtin_amdgcn_ldexpf(fabsf(a.scale), e2);

    v16f acc[NU];
    float m, l, d, f_most;  // as in attn_rows
    auto rest_at = [](int c) { return 16 * c; };

    // Staging.  Piece i = tid + threads * j.
    uint4 kw[pieces], vw[pieces];
    float ks = 0.0f, vs = 0.0f;
    int ik[pieces], iv;
    auto look_up = [&](int t0) __attribute__((always_inline)) {
      if constexpr (WIDE) {
        iv = page_id(a, ids, t0, end, shift);
      } else {
#pragma unroll
        for (int j = 0; j < pieces; ++j)
          ik[j] = page_id(a, ids, t0 + (tid + threads * j) / (D / 16), end, shift);
        iv = page_id(a, ids, t0 + tid % 4 * 16, end, shift);
      }
    };
    auto fetch = [&](int t0) __attribute__((always_inline)) {
      const int in = t0 & (P - 1);
      if constexpr (WIDE) iv = __builtin_amdgcn_readfirstlane(iv);
      const int64_t pv = in_cache(a, iv) ? iv : 0;
      const int8_t *kpage = a.g.c.k + pv * page_bytes + in * D;
      const int8_t *vpage = a.g.c.v + pv * page_bytes + in;
#pragma unroll
      for (int j = 0; j < pieces; ++j) {
        if (all % threads == 0 || tid + threads * j < all) {
          if constexpr (!WIDE)
            kpage = a.g.c.k + static_cast<int64_t>(in_cache(a, ik[j]) ? ik[j] : 0) * page_bytes;
          kw[j] = *reinterpret_cast<const uint4 *>(kpage + kat[j]);
          vw[j] = *reinterpret_cast<const uint4 *>(vpage + vat[j]);
        }
      }
      if (tid < 4) {
        ks = a.g.c.k_scale[pv * H + head];
        vs = a.g.c.v_scale[pv * H + head];
        if (!in_cache(a, iv)) ks = vs = nanf32();
        if (t0 + 16 * tid >= end) ks = vs = 0.0f;
      }
    };
    auto put = [&](Stage &s) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < pieces; ++j) {
        const int i = tid + threads * j;
        if (all % threads == 0 || i < all) {
          const int t = i / (D / 16), dk = i % (D / 16) * 2;
          const int r = (t & 32) + (t >> 4 & 1) * 4 + (t >> 2 & 3) * 8 + (t & 3);
          s.k[dk * kp + r] = __builtin_bit_cast(uint4, codes_f16(kw[j].x, kw[j].y));
          s.k[(dk + 1) * kp + r] = __builtin_bit_cast(uint4, codes_f16(kw[j].z, kw[j].w));
          const int c = i % 4 * 2, dv = i / 4;
          s.v[c * vp + dv] = __builtin_bit_cast(uint4, codes_f16(vw[j].x, vw[j].y));
          s.v[(c + 1) * vp + dv] = __builtin_bit_cast(uint4, codes_f16(vw[j].z, vw[j].w));
        }
      }
      if (tid < 4) s.ks[tid] = ks, s.lv[tid] = __builtin_amdgcn_logf(vs);
    };

    v16f st[2];
    auto scores = [&](auto all_bits, const Stage &s) __attribute__((always_inline)) {  // one group of 64 tokens
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) st[t][r] = 0.0f;
      auto keys = [&](int c, int t) {
        return __builtin_bit_cast(v8h, s.k[(2 * c + h) * kp + 32 * t + col]);
      };
      if constexpr (all_bits.value) {
        const int levels = Rest<T, D>::levels(fmaxf(s.ks[h], s.ks[2 + h]) * q_scale);
#pragma unroll 1
        for (int level = 0; level <= levels; ++level) {
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) st[t][r] *= Rest<T, D>::kUnit;
#pragma unroll 1
          for (int c = 0; c < KC; ++c) {
            v8h r = Rest<T, D>::operand(qp + 8 * h + rest_at(c), e2, level);
            if (a.scale < 0.0f) r = -r;
#pragma unroll
            for (int t = 0; t < 2; ++t) st[t] = mfma32_f16(keys(c, t), r, st[t]);
          }
        }
#pragma unroll 1
        for (int level = 1; level <= levels; ++level)
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) st[t][r] *= 1.0f / Rest<T, D>::kUnit;
      } else {
        // neighbouring products do not wait for each other's sums
        feed_products<ahead>(
            std::make_integer_sequence<int, 2 * KC>{},
            [&](auto i) { return keys(i.value / 2, i.value % 2); },
            [&](auto i, v8h k) { st[i.value % 2] = mfma32_f16(k, q[i.value / 2], st[i.value % 2]); });
      }
    };
    auto weigh = [&](int t0, const Stage &s) __attribute__((always_inline)) {
      float f[2], v[2], x[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        f[t] = s.ks[2 * t + h] * q_scale;
        f[t] = f[t] < 0x1p-126f ? 0x1p-126f : f[t];  // so that -inf stays -inf
        v[t] = s.lv[2 * t + h];
      }
      f_most = fmaxf(f_most, fmaxf(f[0], f[1]));
      if (t0 < wbot.lo || t0 + kGroup > wtop.hi) {  // some row does not see all 64
        asm volatile("");  // stays a branch: few groups need it
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int t1 = t0 + 32 * t + 16 * h;
#pragma unroll
          for (int r = 0; r < 16; ++r)
            st[t][r] = static_cast<unsigned>(t1 + r - me.lo) < wide ? st[t][r] : -INFINITY;
          if (t1 + 16 <= me.lo || t1 >= me.hi) f[t] = 1.0f, v[t] = 0.0f;  // a hidden page's may be NaN
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        x[t] = st[t][0];
#pragma unroll
        for (int r = 1; r < 16; ++r) x[t] = fmaxf(x[t], st[t][r]);
        x[t] *= f[t];
      }
      if (__any(fmaxf(x[0], x[1]) > m + 8.0f || fmaxf((x[0] - m) + v[0], (x[1] - m) + v[1]) > d + 8.0f)) {
        float high = fmaxf(x[0], x[1]);
        high = fmaxf(m, fmaxf(high, __shfl_xor(high, 32, kWave)));
        const float base = high == -INFINITY ? 0.0f : high, delta = m - base;
        m = high;
        float up = fmaxf((x[0] - base) + v[0], (x[1] - base) + v[1]);
        up = fmaxf(up, __shfl_xor(up, 32, kWave));
        const float next = fmaxf(fmaxf(d + delta, up), kLeast);
        const float fix = exp2f((d - next) + delta);
        d = next;
        l *= exp2f(delta);
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[u][r] *= fix;
      }
      const float base = (m == -INFINITY ? 0.0f : m) - kLiftTile;
      v8h p[4];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float part = v[t] - d;
        part = part < kApart ? kApart : part;  // a NaN stays one
        const float c = part - base;
        float sum = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float x = __builtin_fmaf(st[t][r], f[t], c);
          const float e = __builtin_amdgcn_exp2f(x);
          sum += e;
          p[2 * t + r / 8][r % 8] = static_cast<_Float16>(e);
        }
        l += sum * __builtin_amdgcn_exp2f(-part);
      }
      // weights c: tokens 32 (c / 2) + 16 h + 8 (c % 2) + 0..7
      feed_products<ahead>(
          std::make_integer_sequence<int, 4 * NU>{},
          [&](auto i) {
            constexpr int c = i.value / NU;
            const int chunk = 4 * (c / 2) + 2 * h + c % 2;
            return __builtin_bit_cast(v8h, s.v[chunk * vp + 32 * (i.value % NU) + col]);
          },
          [&](auto i, v8h v) { acc[i.value % NU] = mfma32_f16(v, p[i.value / NU], acc[i.value % NU]); });
    };
    auto pass = [&](auto all_bits) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[u][r] = 0.0f;
      m = -INFINITY;
      l = f_most = 0.0f;
      d = kLeast;
      if (begin < end) {
        look_up(begin);
        fetch(begin);
        look_up(begin + kGroup);
        put(stage[0]);
      }
      __syncthreads();
      int now = 0;
      for (int t0 = begin; t0 < end; t0 += kGroup, now ^= 1) {
        const bool more = t0 + kGroup < end;
        if (more) {
          fetch(t0 + kGroup);
          look_up(t0 + 2 * kGroup);
        }
        if (t0 < wbot.hi && t0 + kGroup > wtop.lo && w0 < rows) {
          scores(all_bits, stage[now]);
          weigh(t0, stage[now]);
        }
        if (more) put(stage[now ^ 1]);
        __syncthreads();
      }
    };
    pass(std::false_type{});
    const bool again = Rest<T, D>::counts(f_most, qp + 8 * h, e2, valid, KC, rest_at, 2,
                                          [](float v) { return fmaxf(v, __shfl_xor(v, 32, kWave)); });
    if (lane == 0) s_again[wave] = again;
    __syncthreads();
    bool any = false;  // the waves of a workgroup stay together
#pragma unroll
    for (int w = 0; w < W; ++w) any |= s_again[w] != 0;
    if (any) pass(std::true_type{});

    l += __shfl_xor(l, 32, kWave);  // its lift is that of the sums
    const float unit = rintf(d);
    if (valid) {
      const int64_t place = static_cast<int64_t>(seq.q0 + row / G) * a.q_heads + head * G + row % G;
      const int64_t at = static_cast<int64_t>(split) * a.queries * a.q_heads + place;
      const float f = l == 0.0f ? 0.0f : exp2f(d - unit) / l;
      if (a.splits > 1 && h == 0) a.stats[2 * at] = m, a.stats[2 * at + 1] = l;
      if (a.splits == 1 || begin < end) {
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int d = 32 * u + 8 * k + 4 * h;
            struct {
              T v[4];
            } o;
            v4f w;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              w[e] = __builtin_amdgcn_ldexpf(acc[u][4 * k + e] * f, static_cast<int>(unit));
              o.v[e] = static_cast<T>(w[e]);
            }
            if (a.splits > 1)
              *reinterpret_cast<v4f *>(a.part + at * D + d) = w;
            else
              __builtin_memcpy(static_cast<T *>(a.out) + place * D + d, &o, sizeof(o));
          }
      }
    }
  }
}

// Joins the chunks of a row, averages with their maxima and sums l, in the chunks' order: W waves take
// every W-th chunk, lane by lane of the row.  A chunk in which the row sees nothing has l = 0 and its
// averages were never written.
template <typename T, int D, int W>
__global__ __launch_bounds__(256) void attn_join(const AttnArgs a) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x % kWave, wave = wave_id();
  const int64_t rows = static_cast<int64_t>(a.queries) * a.q_heads;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kWaves / W) + (W == 1 ? wave : 0);
  if (row >= rows) return;  // whole workgroups where they meet at a barrier
  float best = -INFINITY, total = 0.0f;
  for (int s = lane; s < a.splits; s += kWave) best = fmaxf(best, a.stats[2 * (s * rows + row)]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) best = fmaxf(best, __shfl_xor(best, off, kWave));
  const float base = best == -INFINITY ? 0.0f : best;
  for (int s = lane; s < a.splits; s += kWave) {
    const float *st = a.stats + 2 * (s * rows + row);
    total += st[1] * exp2f(st[0] - base);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off, kWave);
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  float o[E] = {};
#pragma unroll 4
  for (int s = W == 1 ? 0 : wave; s < a.splits; s += W) {
    const int64_t at = s * rows + row;
    const float l = a.stats[2 * at + 1], f = l * exp2f(a.stats[2 * at] - base) * inv;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float v = a.part[at * D + 64 * e + lane];
      o[e] += l == 0.0f ? 0.0f : v * f;
    }
  }
  if constexpr (W > 1) {
    __shared__ float s_o[W][D];
#pragma unroll
    for (int e = 0; e < E; ++e) s_o[wave][64 * e + lane] = o[e];
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int w = 1; w < W; ++w) o[e] += s_o[w][64 * e + lane];
  }
  T *out = static_cast<T *>(a.out) + row * D + lane;
#pragma unroll
  for (int e = 0; e < E; ++e) out[64 * e] = static_cast<T>(o[e]);
}

struct Plan {
  int64_t row_tiles, chunk;
  int splits;
  int waves;  // of attn_tile; 0: attn_rows
};

// Workgroups of a launch, whose threads number below 2^32.
constexpr int64_t kMostJobs = (1 << 23) - 1;

// Chunks of the token axis: for attn_rows eight workgroups for each of 256 CUs, so that ragged
// lengths even out (64 sequences of up to 16384 tokens, 8 heads: 286 us, with four 297, with sixteen 284),
// each with at least 512 tokens, eight groups, so that its start and its sums' join stay small
// beside them; for attn_tile as many as are resident at once, with at least 256 tokens (385 queries
// of three heads over 3256 tokens, dim 256: 51 us with 512, 40 with 256).
//
// From 64 query rows on attn_tile runs, which reads and converts each token once for 128 or 256 rows:
// 8 heads, 6144 and 2217 tokens, 2048 and 1226 queries of 4 heads each: 235 us, attn_rows 741. 256 rows take turns
// in eight waves where there are 256 such workgroups: 281 us against 292 with 128 rows.
Plan plan_for(int32_t heads, int32_t seqs, int32_t group, int64_t queries, int64_t max_query,
              int64_t max_length, int64_t window, int32_t dim) {
  if (max_query > queries) max_query = queries;
  if (max_length > kMost) max_length = kMost;
  Plan p;
  const int64_t rows = (max_query < 1 ? 1 : max_query) * group;
  p.waves = rows < 64 ? 0 : dim <= 128 && cdiv(rows, 256) * heads * seqs >= 256 ? 8 : 4;
  p.row_tiles = cdiv(rows, p.waves ? 32 * p.waves : kRows);
  int64_t span = max_length;
  if (window > 0 && window + max_query + kGroup < span) span = window + max_query + kGroup;
  const int64_t tiles = p.row_tiles * heads * seqs;
  int64_t splits = cdiv(p.waves ? 2048 / p.waves : 2048, tiles < 1 ? 1 : tiles);
  const int64_t least = p.waves ? 256 : 512;
  if (splits > cdiv(span, least)) splits = cdiv(span, least);
  // rows that fill the GPU by themselves; the join's threads stay below 2^32 so
  if (splits < 1 || queries * group * heads >= 1 << 24) splits = 1;
  p.chunk = cdiv(cdiv(span, splits), kWaves * kGroup) * (kWaves * kGroup);
  if (p.chunk < 1) p.chunk = kWaves * kGroup;
  p.splits = static_cast<int>(span < 1 ? 1 : cdiv(span, p.chunk));
  // max_query may be all rows of many sequences: a workgroup takes several row tiles then
  const int64_t others = static_cast<int64_t>(heads) * seqs * p.splits;
  if (p.row_tiles * others > kMostJobs) p.row_tiles = kMostJobs / others > 1 ? kMostJobs / others : 1;
  return p;
}

}  // namespace
}  // namespace dec
}  // namespace rxmet

using namespace rxmet;
using namespace rxmet::dec;

extern "C" int64_t rxmet_kv_attention_workspace_bytes(const rxmet_kv_cache *cache, int32_t seqs,
                                                      int64_t queries, int32_t q_heads,
                                                      int64_t max_query, int64_t max_length,
                                                      int64_t window) {
  if (!cache || cache->heads < 1 || q_heads < cache->heads || queries <= 0 || seqs <= 0) return 0;
  const Plan p = plan_for(cache->heads, seqs, q_heads / cache->heads, queries, max_query,
                          max_length, window, cache->dim);
  return p.splits == 1 ? 0 : p.splits * queries * q_heads * (cache->dim + 2) * 4;
}

extern "C" int rxmet_kv_attention(const rxmet_kv_cache *cache, const rxmet_kv_table *table,
                                  const int32_t *lengths, const int32_t *cu_query, int64_t queries,
                                  int64_t max_query, int64_t max_length, const void *query,
                                  int64_t query_stride_t, int64_t query_stride_h, int32_t q_heads,
                                  float scale, int32_t causal, int64_t window, void *out,
                                  int32_t dtype, void *workspace, void *stream) {
  if (int rc = check_cache(cache, table)) return rc;
  RXMET_CHECK_ARG(dtype == RXMET_QDQ_F16 || dtype == RXMET_QDQ_BF16,
                  "queries must be fp16 or bf16");
  RXMET_CHECK_ARG(q_heads >= cache->heads && q_heads % cache->heads == 0,
                  "query heads must be a multiple of the cache's heads");
  RXMET_CHECK_ARG(queries >= 0 && max_query >= 0 && max_length >= 0 && window >= 0,
                  "queries, max_query, max_length and window must be >= 0");
  RXMET_CHECK_ARG(max_query <= INT32_MAX && max_length <= INT32_MAX && queries <= INT32_MAX,
                  "lengths must be below 2^31");
  RXMET_CHECK_ARG(queries * q_heads <= kMost, "too many query rows for one call");
  RXMET_CHECK_ARG(cu_query || queries == table->seqs,
                  "without cu_query there is one query a sequence");
  if (queries == 0 || table->seqs == 0) return 0;
  RXMET_CHECK_ARG(lengths && query && out, "lengths, query and out are needed");
  const int group = q_heads / cache->heads;
  int64_t cap = static_cast<int64_t>(table->cols) * cache->page_size;
  if (cap > kMost) cap = kMost;
  const Plan p = plan_for(cache->heads, table->seqs, group, queries, max_query, max_length, window,
                          cache->dim);
  if (window > INT32_MAX) window = 0;  // hides nothing
  RXMET_CHECK_ARG(p.splits == 1 || workspace, "this call needs a workspace");
  const int64_t jobs = p.row_tiles * p.splits * cache->heads;
  RXMET_CHECK_ARG(jobs * table->seqs <= kMostJobs, "too many sequences and heads for one call");
  const int64_t rows = queries * q_heads;
  float *part = static_cast<float *>(workspace);
  const AttnArgs a{{*cache, *table}, lengths, cu_query, static_cast<int>(queries), query,
                   query_stride_t, query_stride_h, q_heads, group,
                   scale * 1.44269504088896340736f, causal, static_cast<int>(window),
                   static_cast<int>(p.chunk), p.splits, static_cast<int>(p.row_tiles),
                   static_cast<int>(cap), out, part,
                   part ? part + p.splits * rows * cache->dim : nullptr};
  auto st = static_cast<hipStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(jobs * table->seqs);
  prof::Scope scope("kv_attention", st);
  auto launch = [&](auto t, auto dim) {
    using T = decltype(t);
    const bool wide = cache->page_size >= kGroup;
    if (p.waves == 4) {
      if (wide) attn_tile<T, dim.value, 4, true><<<grid, 256, 0, st>>>(a);
      else attn_tile<T, dim.value, 4, false><<<grid, 256, 0, st>>>(a);
    } else if (p.waves == 8) {
      if constexpr (dim.value <= 128) {
        if (wide) attn_tile<T, dim.value, 8, true><<<grid, 512, 0, st>>>(a);
        else attn_tile<T, dim.value, 8, false><<<grid, 512, 0, st>>>(a);
      }
    } else {
      attn_rows<T, dim.value><<<grid, 256, 0, st>>>(a);
    }
    if (p.splits > 8)
      attn_join<T, dim.value, kWaves><<<static_cast<unsigned>(rows), 256, 0, st>>>(a);
    else if (p.splits > 1)
      attn_join<T, dim.value, 1><<<static_cast<unsigned>(cdiv(rows, kWaves)), 256, 0, st>>>(a);
  };
  auto with_dim = [&](auto t) {
    switch (cache->dim) {
      case 64: launch(t, std::integral_constant<int, 64>{}); break;
      case 128: launch(t, std::integral_constant<int, 128>{}); break;
      case 192: launch(t, std::integral_constant<int, 192>{}); break;
      default: launch(t, std::integral_constant<int, 256>{}); break;
    }
  };
  if (dtype == RXMET_QDQ_F16)
    with_dim(f16{});
  else
    with_dim(bf16{});
  RXMET_CHECK_LAUNCH();
  return 0;
}

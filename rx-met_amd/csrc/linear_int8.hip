// linear_int8.hip — product of int8 codes with int8 weights and its epilogue.
//
// Mathematics.  y[m, n] = act(acc * sx[m] * sw[n] + b[n]) + r[m, n] with acc = sum_k x[m, k] w[n, k] exact in
// int32 (|acc| <= 2^14 K).  The epilogue is fp32 and rounds once.
//
// Layout.  The matrix instruction's rows are weight rows (n), its columns are token rows (m), so
// that a lane holds several consecutive n of one m.
//
// Bound and measured.  Few rows: the weights' bytes ([16, 4096] x [4096, 4096] 6.9 us, [16, 8192] x
// [8192, 8192] 19 us = 3.5 TB/s).  Many: the matrix unit, which is busy for 51 % of the time: [8192, 8192] x [8192, 8192] 568 to 650 us by
// card, 1.94 to 1.69 POP/s, where the library's int8 product without an epilogue reaches 2.1.
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
  int *part;        // [splits, M, N] sums of a part of K each, where splits > 1
  int splits, run;  // run: steps of K of a part
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

// The sum times such a row scale may leave fp32 where the result does not: the weight's scale goes first.
__device__ __forceinline__ bool is_large(float sx) { return fabsf(sx) > 0x1p90f; }

// Finishes and writes C consecutive n of row m: as vectors, and one by one at N's end.  LARGE: some rows
// may be large (asked for each output, that costs 1.5 % of [8192, 8192] x [8192, 8192]).
template <typename T, int C, bool LARGE = true>
__device__ __forceinline__ void finish(const LinArgs &a, int64_t m, int64_t n0, const int (&acc)[C]) {
  if (m >= a.M || n0 >= a.N) return;
  const float sx = a.sx[m];
  const T *bias = a.bias ? static_cast<const T *>(a.bias) + n0 : nullptr;
  const T *res = a.res ? static_cast<const T *>(a.res) + m * a.res_stride + n0 : nullptr;
  T *y = static_cast<T *>(a.y) + m * a.N + n0;
  const bool large = LARGE && is_large(sx);
  auto value = [&](int acc, float sw, T b, T r) {
    float v = static_cast<float>(acc) * (large ? sw : sx) * (large ? sx : sw);
    if (bias) v += static_cast<float>(b);
    v = activate(v, a.act);
    if (res) v += static_cast<float>(r);
    return static_cast<T>(v);
  };
  if (n0 + C <= a.N) {
    struct {
      T v[C];
    } out, b = {}, r = {};
    float sw[C];
    __builtin_memcpy(sw, a.sw + n0, sizeof(sw));
    if (bias) __builtin_memcpy(&b, bias, sizeof(b));
    if (res) __builtin_memcpy(&r, res, sizeof(r));
#pragma unroll
    for (int e = 0; e < C; ++e) out.v[e] = value(acc[e], sw[e], b.v[e], r.v[e]);
    __builtin_memcpy(y, &out, sizeof(out));
  } else {
#pragma unroll
    for (int e = 0; e < C; ++e)
      if (n0 + e < a.N)
        y[e] = value(acc[e], a.sw[n0 + e], bias ? bias[e] : static_cast<T>(0.0f),
                     res ? res[e] : static_cast<T>(0.0f));
  }
}

// ---------------------------------------------------------------------------------------------
// At most 16 rows of x: a workgroup takes 16 weight rows and all of K, its eight waves take runs
// of 128 of K in turn; the weights go from memory into the matrix instruction with no stop in
// LDS.  The eight sums meet in LDS, so there is one launch.
//
// Bound: the weights' bytes, and below some 20 MB the launch and one trip to memory.  [16, 4096] x
// [4096, 4096]: 7.0 us (17 MB: 3.4 us at the copy rate); 32 or 64 weight rows a workgroup, which read x
// less often, 8.8 and 11.5 us; tiles of 64 x 32 with K in four parts 8.9 us.
constexpr int kFewRows = 16, kFewWaves = 8;

template <typename T>
__global__ __launch_bounds__(64 * kFewWaves) void linear_few(const LinArgs a) {
  __shared__ int s[kFewWaves][kFewRows][20];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int col = lane % 16, g = lane / 16;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16;
  const int8_t *w = a.w + (n0 + col < a.N ? n0 + col : a.N - 1) * a.w_stride;
  const int8_t *x = a.x + (col < a.M ? col : a.M - 1) * a.x_stride;
  v4i acc = {0, 0, 0, 0};
  constexpr int turn = kFewWaves * 128;  // from a wave's run of K to its next
  auto runs = [&](auto N, int k0) {      // N of them, all their loads before the first product
    v4i wf[N.value][2], xf[N.value][2];
#pragma unroll
    for (int i = 0; i < N.value; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int k = k0 + turn * i + 64 * c + 16 * g;
        __builtin_memcpy(&wf[i][c], w + k, 16);
        __builtin_memcpy(&xf[i][c], x + k, 16);
      }
#pragma unroll
    for (int i = 0; i < N.value; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c) acc = mfma_i8(wf[i][c], xf[i][c], acc);
  };
  int k0 = wave * 128;
  for (; k0 + 3 * turn + 128 <= a.K; k0 += 4 * turn) runs(std::integral_constant<int, 4>{}, k0);
  for (; k0 + 128 <= a.K; k0 += turn) runs(std::integral_constant<int, 1>{}, k0);
  if (k0 < a.K) {  // K ends in this run
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int k = k0 + 64 * c + 16 * g;
      acc = mfma_i8(as_v4i(load_piece(w, k, a.K)), as_v4i(load_piece(x, k, a.K)), acc);
    }
  }
  *reinterpret_cast<v4i *>(&s[wave][col][4 * g]) = acc;
  __syncthreads();
  if (threadIdx.x < kFewRows * 4) {
    const int m = threadIdx.x / 4, n = threadIdx.x % 4 * 4;
    v4i sum = *reinterpret_cast<const v4i *>(&s[0][m][n]);
#pragma unroll
    for (int v = 1; v < kFewWaves; ++v) sum += *reinterpret_cast<const v4i *>(&s[v][m][n]);
    const int r[4] = {sum[0], sum[1], sum[2], sum[3]};
    finish<T, 4>(a, m, n0 + n, r);
  }
}

// ---------------------------------------------------------------------------------------------
// Tiles of TN weight rows x TM token rows on mfma 32x32x32; WN x WM waves take equal parts.
//
// K goes through LDS in steps of 64 bytes, memory -> LDS without registers, three steps ahead in
// a ring of four.  A row's four 16-byte pieces lie at the places piece ^ f(row), so that 16 lanes
// that read one piece of 16 rows meet 16 different bank groups (none of the 256 x 256
// tiles' LDS accesses counts a conflict, 9 % of the 64 x 64 ones' do).  Row i of a wave's
// 32 weight rows stands for n = 16 * (i / 4 % 2) + 4 * (i / 8) + i % 4: a lane holds 16 consecutive n of
// one m.  Rows have to start on 16 bytes; others are copied first (linear_align).  Twice the ring for the
// smallest tiles, or two steps of them to a barrier, changes nothing.
constexpr int kStep = 64;

typedef int v16i __attribute__((ext_vector_type(16)));

// f of a weight row and of a token row
__device__ __forceinline__ int turn_w(int row) { return (row >> 2 & 1) | (row >> 3 & 2); }
__device__ __forceinline__ int turn_x(int row) { return row >> 2 & 3; }

// 16 bytes of each lane's address to LDS at `lds` + 16 * lane, in flight until vmcnt says so.
__device__ __forceinline__ void load_to_lds(const int8_t *p, int8_t *lds) {
  __builtin_amdgcn_global_load_lds(
      (const __attribute__((address_space(1))) void *)p,
      (__attribute__((address_space(3))) void *)lds, 16, 0, 0);
}
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}
// A barrier that lets loads to LDS stay in flight (__syncthreads waits for them).  What this wave
// wrote to or read from LDS before it is done.
__device__ __forceinline__ void meet() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
}

template <typename T, int TN, int TM, int WN, int WM>
__global__ __launch_bounds__(64 * WN * WM) void linear_tile(const LinArgs a) {
  constexpr int threads = 64 * WN * WM;
  constexpr int FN = TN / WN / 32, FM = TM / WM / 32;
  constexpr int bytes = (TN + TM) * kStep;
  constexpr int ring = 4;
  constexpr int loads = bytes / 16 / threads;  // pieces of a thread in a step
  constexpr int CH = 8 * FN;                   // chunks of four n in a wave's row (epilogue)
  static_assert(loads * 16 * threads == bytes, "a step is whole pieces of all threads");
  static_assert(WN * WM * 32 * CH * 16 <= ring * bytes, "the epilogue fits the ring");
  __shared__ __attribute__((aligned(16))) int8_t s[ring][bytes];
  const int tid = threadIdx.x, lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int col = lane % 32, h = lane / 32;
  const int tiles_n = static_cast<int>((a.N + TN - 1) / TN);
  const int tiles_m = static_cast<int>((a.M + TM - 1) / TM);
  int tn = blockIdx.x % tiles_n, tm = blockIdx.x / tiles_n;
  if constexpr (TN * TM >= 256 * 128) {
    // Workgroups go to the eight XCDs in turn: each XCD gets a run of the tiles' order, in which
    // bands of four tiles of x go through the weights together, so that its L2 holds what they share
    // (8192^3: 598 us then; row by row, over all XCDs: 624 us).
    const int total = tiles_n * tiles_m, per = total / 8, rest = total % 8;
    const int xcd = blockIdx.x % 8;
    const int id = xcd * per + (xcd < rest ? xcd : rest) + blockIdx.x / 8;
    const int first = id / (4 * tiles_n) * 4, in = id - first * tiles_n;
    const int high = tiles_m - first < 4 ? tiles_m - first : 4;
    tm = first + in % high;
    tn = in / high;
  }
  const int64_t n0 = static_cast<int64_t>(tn) * TN, m0 = static_cast<int64_t>(tm) * TM;
  // the steps of this part of K; the last part also takes the one that K ends in
  const int split = blockIdx.y, from = split * a.run;
  const bool last = split == a.splits - 1;
  const int all = a.K / kStep, whole = last ? all - from : a.run;

  // piece j of a thread lies at place tid + threads * j of the step, which holds this piece of a row
  const int8_t *src[loads];
  auto piece_at = [&](int j) {
    const int at = tid + threads * j, row = at / 4;
    return (at % 4) ^ (row < TN ? turn_w(row) : turn_x(row - TN));
  };
#pragma unroll
  for (int j = 0; j < loads; ++j) {
    const int row = (tid + threads * j) / 4;
    if (row < TN) {
      const int64_t n = n0 + row < a.N ? n0 + row : a.N - 1;
      src[j] = a.w + n * a.w_stride;
    } else {
      const int64_t m = m0 + row - TN < a.M ? m0 + row - TN : a.M - 1;
      src[j] = a.x + m * a.x_stride;
    }
    src[j] += piece_at(j) * 16 + from * kStep;
  }
  v16i acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
  const int wn = wave % WN * (TN / WN), wm = wave / WN * (TM / WM);
  int wat[FN][2], xat[FM][2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
#pragma unroll
    for (int i = 0; i < FN; ++i) {
      const int row = wn + 32 * i + 16 * (col >> 2 & 1) + 4 * (col >> 3) + (col & 3);
      wat[i][c] = row * kStep + ((2 * c + h) ^ turn_w(row)) * 16;
    }
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const int row = wm + 32 * j + col;
      xat[j][c] = (TN + row) * kStep + ((2 * c + h) ^ turn_x(row)) * 16;
    }
  }
  struct Half {  // the operands of half a step
    v4i w[FN], x[FM];
  };
  auto load = [&](Half &f, const int8_t *buf, int c) {
#pragma unroll
    for (int i = 0; i < FN; ++i) f.w[i] = *reinterpret_cast<const v4i *>(buf + wat[i][c]);
#pragma unroll
    for (int j = 0; j < FM; ++j) f.x[j] = *reinterpret_cast<const v4i *>(buf + xat[j][c]);
  };
  auto multiply = [&](const Half &f) {
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int j = 0; j < FM; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.w[i], f.x[j], acc[i][j], 0, 0, 0);
  };
  auto issue = [&](int step, int slot) {
#pragma unroll
    for (int j = 0; j < loads; ++j)
      load_to_lds(src[j] + step * kStep, &s[slot][wave * 1024 + j * threads * 16]);
  };
  if (whole > 0) {
    // past the end a step is read once more, so that the count of loads in flight holds
#pragma unroll
    for (int k = 0; k < ring; ++k) issue(k < whole ? k : 0, k);
    wait_loads<(ring - 1) * loads>();
    meet();
    // each half's operands are read from LDS while the half before is multiplied
    Half even, odd;
    load(even, s[0], 0);
    for (int k = 0; k < whole; ++k) {
      load(odd, s[k % ring], 1);
      multiply(even);
      wait_loads<(ring - 2) * loads>();
      meet();  // step k + 1 is there for all, and step k has been read by all
      issue(k + ring < whole ? k + ring : k, k % ring);
      load(even, s[(k + 1) % ring], 0);
      multiply(odd);
    }
    wait_loads<0>();
  }
  __syncthreads();
  if (last && all * kStep < a.K) {
#pragma unroll
    for (int j = 0; j < loads; ++j) {
      const int k = whole * kStep + 16 * piece_at(j);  // from this part's first byte
      *reinterpret_cast<uint4 *>(&s[0][16 * (tid + threads * j)]) =
          load_piece(src[j] + whole * kStep - k, k, a.K - from * kStep);
    }
    __syncthreads();
    Half f;
    load(f, s[0], 0);
    multiply(f);
    load(f, s[0], 1);
    multiply(f);
    __syncthreads();
  }

  // 32 rows of x at a time the wave's sums go through its own part of the LDS, from where eight
  // consecutive n of a row are finished by a lane and neighbouring lanes write what lies side by
  // side.  Chunk c of row m lies at c ^ turn, for the banks.
  auto turn = [](int m) { return CH >= 16 ? m & 15 : m >> 1 & 7; };
  v4i *part = reinterpret_cast<v4i *>(&s[0][0]) + wave * 32 * CH;
  bool large = false;
  for (int r = lane; r < TM / WM; r += kWave) large |= m0 + wm + r < a.M && is_large(a.sx[m0 + wm + r]);
  large = __any(large);
#pragma unroll
  for (int j = 0; j < FM; ++j) {
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        part[col * CH + ((8 * i + 4 * h + k) ^ turn(col))] =
            v4i{acc[i][j][4 * k], acc[i][j][4 * k + 1], acc[i][j][4 * k + 2], acc[i][j][4 * k + 3]};
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
#pragma unroll 1
    for (int at = lane; at < 32 * CH / 2; at += kWave) {
      const int r = at / (CH / 2), c = at % (CH / 2) * 2;
      const v4i lo = part[r * CH + (c ^ turn(r))], hi = part[r * CH + ((c + 1) ^ turn(r))];
      const int v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      const int64_t m = m0 + wm + 32 * j + r, n = n0 + wn + 4 * c;
      if (a.splits == 1) {
        if (large)
          finish<T, 8, true>(a, m, n, v);
        else
          finish<T, 8, false>(a, m, n, v);
      } else if (m < a.M) {
        int *p = a.part + (split * a.M + m) * a.N + n;
        if (n + 8 <= a.N) {
          __builtin_memcpy(p, v, sizeof(v));
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (n + e < a.N) p[e] = v[e];
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");  // read before it is written again
  }
}

// Rows that do not start on 16 bytes, copied to rows of whole steps with zeros behind them: M rows
// of x, then N of the weights.  One launch and the bytes twice, against loads of 16 bytes at any
// address in the tiles' loop ([777, 1025] x [2051, 1025]: 15.6 us and 13.5 us with words moved
// into place).
struct AlignArgs {
  const int8_t *x, *w;
  int64_t x_stride, w_stride;
  int8_t *out;
  int64_t M, rows;
  int K, pitch;
};

__global__ __launch_bounds__(256) void linear_align(const AlignArgs a) {
  const unsigned pieces = a.pitch / 16, i = blockIdx.x * 256 + threadIdx.x;  // below 2^32
  if (i >= a.rows * pieces) return;
  const int64_t row = i / pieces;
  const int k = i % pieces * 16;
  const int8_t *p = row < a.M ? a.x + row * a.x_stride : a.w + (row - a.M) * a.w_stride;
  *reinterpret_cast<uint4 *>(a.out + row * a.pitch + k) = load_piece(p, k, a.K);
}

// Adds the parts of K up and finishes four n of a row.
template <typename T>
__global__ __launch_bounds__(256) void linear_join(const LinArgs a) {
  const int64_t quads = (a.N + 3) / 4;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= a.M * quads) return;
  const int64_t m = i / quads, n = i % quads * 4;
  const int left = a.N - n < 4 ? static_cast<int>(a.N - n) : 4;
  int v[4] = {0, 0, 0, 0};
  for (int s = 0; s < a.splits; ++s) {
    const int *p = a.part + (s * a.M + m) * a.N + n;
    int u[4] = {0, 0, 0, 0};
    if (left == 4) {
      __builtin_memcpy(u, p, 16);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) u[e] = p[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += u[e];
  }
  finish<T, 4>(a, m, n, v);
}

// How a call is run: linear_few up to 16 rows; else the largest tile of which there is one for
// each of 256 CUs, because a step costs much the same for every tile ([1024, 4096] x [4096, 4096]: 128 x 128
// 32 us, 64 x 128 36, 256 x 256 79; [512, ..]: 64 x 128 20 us, 128 x 128 29; [256, ..]: 64 x 64 13 us,
// 64 x 128 18; [2048, ..]: 256 x 128 48 us, 128 x 128 54); where even the smallest tiles are fewer, K is cut
// into parts of at least 16 steps ([64, 4096] x [4096, 12288]: four parts 19 us, one 42).
enum Shape { kFew, k64x32, k64x64, k64x128, k128x128, k256x128, k256x256 };

struct Plan {
  Shape shape;
  int splits, run;
};

Plan plan_for(int64_t M, int64_t N, int64_t K) {
  if (M <= kFewRows) return {kFew, 1, 0};
  auto tiles = [&](int64_t tn, int64_t tm) { return cdiv(N, tn) * cdiv(M, tm); };
  if (M > 64) {
    if (tiles(256, 256) >= 256) return {k256x256, 1, 0};
    if (tiles(256, 128) >= 256) return {k256x128, 1, 0};
    if (tiles(128, 128) >= 256) return {k128x128, 1, 0};
    if (tiles(64, 128) >= 256) return {k64x128, 1, 0};
  }
  Plan p{M <= 32 ? k64x32 : k64x64, 1, 0};
  const int64_t steps = K / kStep;
  int64_t splits = 256 / tiles(64, p.shape == k64x32 ? 32 : 64);
  if (splits > steps / 16) splits = steps / 16;
  if (splits > 1) {
    p.run = static_cast<int>(cdiv(steps, splits));
    p.splits = static_cast<int>(cdiv(steps, p.run));
  }
  return p;
}

// Whether the rows can be read in aligned pieces of 16 bytes.
bool aligned(const void *codes, int64_t codes_stride, const void *weight, int64_t weight_stride) {
  return (reinterpret_cast<uintptr_t>(codes) | reinterpret_cast<uintptr_t>(weight) |
          static_cast<uintptr_t>(codes_stride) | static_cast<uintptr_t>(weight_stride)) % 16 == 0;
}

int64_t pitch_of(int64_t K) { return cdiv(K, kStep) * kStep; }

// Bytes of the parts' sums, behind which the copied rows lie.
int64_t part_bytes(const Plan &p, int64_t M, int64_t N) {
  return p.splits > 1 ? cdiv(p.splits * M * N * 4, 256) * 256 : 0;
}

template <typename T, int TN, int TM, int WN, int WM>
void launch_tile(const LinArgs &a, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(cdiv(a.N, TN) * cdiv(a.M, TM)), a.splits);
  linear_tile<T, TN, TM, WN, WM><<<grid, 64 * WN * WM, 0, st>>>(a);
}

}  // namespace
}  // namespace dec
}  // namespace rxmet

using namespace rxmet;
using namespace rxmet::dec;

extern "C" int64_t rxmet_linear_int8_workspace_bytes(const int8_t *codes, int64_t codes_stride,
                                                     const int8_t *weight, int64_t weight_stride,
                                                     int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const Plan p = plan_for(M, N, K);
  int64_t bytes = part_bytes(p, M, N);
  if (p.shape != kFew && !aligned(codes, codes_stride, weight, weight_stride))
    bytes += (M + N) * pitch_of(K);
  return bytes;
}

extern "C" int rxmet_linear_int8(const int8_t *codes, int64_t codes_stride, const float *scales,
                                 const int8_t *weight, int64_t weight_stride,
                                 const float *weight_scales, const void *bias,
                                 const void *residual, int64_t residual_stride, void *y, int64_t M,
                                 int64_t N, int64_t K, int32_t activation, int32_t dtype,
                                 void *workspace, void *stream) {
  RXMET_CHECK_ARG(M >= 0 && N >= 1 && K >= 1 && K <= RXMET_LINEAR_INT8_K_MAX,
                  "M must be >= 0, N >= 1 and K between 1 and 131071");
  RXMET_CHECK_ARG(M <= 1 << 26 && N <= 1 << 26, "M and N must be at most 2^26");
  RXMET_CHECK_ARG(activation >= RXMET_ACT_NONE && activation <= RXMET_ACT_GELU,
                  "unknown activation");
  RXMET_CHECK_ARG(dtype == RXMET_QDQ_F32 || dtype == RXMET_QDQ_F16 || dtype == RXMET_QDQ_BF16,
                  "element type must be fp32, fp16 or bf16");
  if (M == 0) return 0;
  RXMET_CHECK_ARG(codes && scales && weight && weight_scales && y,
                  "codes, weight, their scales and y are needed");
  RXMET_CHECK_ARG(cdiv(M, 32) * cdiv(N, 64) < 1 << 23, "too many outputs for one call");
  const Plan p = plan_for(M, N, K);
  const bool copy = p.shape != kFew && !aligned(codes, codes_stride, weight, weight_stride);
  RXMET_CHECK_ARG((p.splits == 1 && !copy) || workspace, "this call needs a workspace");
  RXMET_CHECK_ARG(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "the workspace must be aligned to 16 bytes");
  RXMET_CHECK_ARG(!copy || (M + N) * (pitch_of(K) / 16) < 1LL << 32, "too many rows to copy");
  LinArgs a{codes, weight, codes_stride, weight_stride, scales, weight_scales, bias,
            residual, residual_stride, y, M, N, static_cast<int>(K), activation,
            static_cast<int *>(workspace), p.splits, p.run};
  auto st = static_cast<hipStream_t>(stream);
  prof::Scope scope("linear_int8", st);
  if (copy) {
    const int64_t pitch = pitch_of(K);
    int8_t *rows = static_cast<int8_t *>(workspace) + part_bytes(p, M, N);
    const AlignArgs c{codes, weight, codes_stride, weight_stride, rows, M, M + N,
                      static_cast<int>(K), static_cast<int>(pitch)};
    linear_align<<<static_cast<unsigned>(cdiv((M + N) * (pitch / 16), 256)), 256, 0, st>>>(c);
    a.x = rows;
    a.w = rows + M * pitch;
    a.x_stride = a.w_stride = pitch;
    a.K = static_cast<int>(pitch);  // p was made for K: its last part takes what K's end adds
  }
  with_type(dtype, [&](auto t) {
    using T = decltype(t);
    switch (p.shape) {
      case kFew:
        linear_few<T><<<static_cast<unsigned>(cdiv(N, 16)), 64 * kFewWaves, 0, st>>>(a);
        break;
      case k64x32: launch_tile<T, 64, 32, 2, 1>(a, st); break;
      case k64x64: launch_tile<T, 64, 64, 2, 2>(a, st); break;
      case k64x128: launch_tile<T, 64, 128, 2, 2>(a, st); break;
      case k128x128: launch_tile<T, 128, 128, 2, 2>(a, st); break;
      case k256x128: launch_tile<T, 256, 128, 4, 2>(a, st); break;
      case k256x256: launch_tile<T, 256, 256, 2, 4>(a, st); break;
    }
    if (p.splits > 1)
      linear_join<T><<<static_cast<unsigned>(cdiv(M * cdiv(N, 4), 256)), 256, 0, st>>>(a);
  });
  RXMET_CHECK_LAUNCH();
  return 0;
}

// Norms before and after a block, fused with its scale, shift, gate and residual, one row
// (token) of the residual stream at a time:
//   r = x + gate * post(branch)                 post: none, RMS norm or LayerNorm
//   y = norm(r) * (1 + scale) + shift           norm: none, RMS norm or LayerNorm
// without a branch r = x.  Sums and products are fp32 (of rows that do not fit the registers, sums
// in 64 bits); r and y are each rounded once, to their own type, and y is taken from the
// unrounded r.
//
// Bound by memory: 4 to 16 bytes and 2 to 15 flop an element, and by counters the kernels move
// those bytes and no more.  A copy kernel that goes past the caches reaches 6.5 TB/s; here 360 MB
// of bf16 with a gate (720p, 118,800 x 1536) take 169 us, 6.5 TB/s; gate and norm (480p,
// 32,760 x 1536) 66 us, 6.1; gate and norm with a norm of the branch (118,800 x 2048) 321 us, 6.1.
// What the rest goes to: the loads of the row's vectors, which hit the caches, and with a norm of
// the branch the second sum and the four waves a SIMD that its registers leave.
//
// One row per wave and one pass per row, because a wave that walks rows waits for each row's
// stores before the next row's loads (their counter is one): 4, 8 and 16 rows a wave took 188, 200
// and 216 us where one takes 175.  Vectors staged in LDS for a workgroup's rows were slower too
// (480p: 83 us against 72): their barrier holds four waves together.
#include <algorithm>
#include <type_traits>

#include "kernels.hpp"
#include "rows.hpp"

namespace recap {
namespace {

constexpr int kThreads = 256;

// One value of an fp32 or T vector, by a flag that is uniform over the launch.
template <class T>
__device__ inline float load_one(const void* p, bool wide, int64_t i) {
  return wide ? load_elem<F32>(p, i) : load_elem<T>(p, i);
}

// Sum over the workgroup, in every thread: lanes by a butterfly, waves in order.
__device__ inline double block_sum(double v, double* part) {
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  __syncthreads();  // the previous sum's readers are done with `part`
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = part[0];
  for (int w = 1; w < kThreads / 64; ++w) s += part[w];
  return s;
}

struct RowStats {
  double mean;
  float inv;
};

// Mean (LayerNorm only) and reciprocal deviation of value(0 .. width - 1), in 64 bits: a thread
// adds up to 2^16 terms in order, which in fp32 puts a row of equal values off by 8e-4, and the
// squares of 2^24 values pass fp32's range from 4.5e15 on.
template <class V>
__device__ RowStats row_stats(int kind, int width, float eps, double* part, V value) {
  RowStats s{0.0, 1.0f};
  if (kind == kNormNone) return s;
  if (kind == kNormLayer) {
    double sum = 0.0;
    for (int c = threadIdx.x; c < width; c += kThreads) sum += (double)value(c);
    s.mean = block_sum(sum, part) / (double)width;
  }
  double sq = 0.0;
  for (int c = threadIdx.x; c < width; c += kThreads) {
    const double d = (double)value(c) - s.mean;
    sq = fma(d, d, sq);
  }
  s.inv = (float)(1.0 / sqrt(block_sum(sq, part) / (double)width + (double)eps));
  return s;
}

// Rows under a chunk or too wide for the registers of 1024 lanes: one workgroup per row, and
// every pass reads the row again (norm_modulate of 2,000 rows of 40,001: 549 us, sums in fp32 541;
// a million rows of 5: 2.5 ms).
template <class X, class T>
__global__ __launch_bounds__(kThreads) void residual_rows_kernel(ResidualArgs a) {
  __shared__ double part[kThreads / 64];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t b = row / a.tokens, n = row - b * a.tokens;
    const int64_t xo = b * a.x.b + n * a.x.n, bo = b * a.branch.b + n * a.branch.n,
                  go = b * a.gate.b + n * a.gate.n, so = b * a.scale.b + n * a.scale.n,
                  ho = b * a.shift.b + n * a.shift.n;
    const auto added = [&](int c) { return load_elem<T>(a.branch.p, bo + c); };
    RowStats post{0.0, 1.0f};
    if (a.branch.p) post = row_stats(a.post, a.width, a.eps, part, added);
    const auto value = [&](int c) {
      float r = load_elem<X>(a.x.p, xo + c);
      if (a.branch.p) {
        float f = (float)((double)added(c) - post.mean) * post.inv;
        if (a.branch_weight) f *= load_one<T>(a.branch_weight, a.wide_weight, c);
        if (a.branch_bias) f += load_one<T>(a.branch_bias, a.wide_weight, c);
        r = a.gate.p ? fmaf(load_one<T>(a.gate.p, a.wide_mod, go + c), f, r) : r + f;
      }
      return r;
    };
    RowStats s{0.0, 1.0f};
    if (a.y.p) s = row_stats(a.norm, a.width, a.eps, part, value);
    const int64_t ro = b * a.r.b + n * a.r.n, yo = b * a.y.b + n * a.y.n;
    __syncthreads();  // an output may be an input: the row's statistics are all taken
    for (int c = threadIdx.x; c < a.width; c += kThreads) {
      const float r = value(c);
      if (a.y.p) {
        float y = (float)((double)r - s.mean) * s.inv;
        if (a.weight) y *= load_one<T>(a.weight, a.wide_weight, c);
        if (a.bias) y += load_one<T>(a.bias, a.wide_weight, c);
        if (a.scale.p) y *= 1.0f + load_one<T>(a.scale.p, a.wide_mod, so + c);
        if (a.shift.p) y += load_one<T>(a.shift.p, a.wide_mod, ho + c);
        store_elem<T>(const_cast<void*>(a.y.p), yo + c, y);
      }
      if (a.r.p) store_elem<X>(const_cast<void*>(a.r.p), ro + c, r);
    }
  }
}

// ---------------------------------------------------------------------------------------
// Rows in registers: one pass over the data.  `lanes` lanes (a power of two) share a row in
// chunks of 16 bytes of the stream, chunk c in lane c % lanes, so a lane holds CHUNKS chunks;
// rows of more than 64 lanes join their waves' sums through LDS.  Loads are as wide as a chunk at
// any alignment.  The row's last chunk is loaded so that it ends with the row, its elements
// before the chunk's own (`skip` of them) left out of sums and stores; lanes past the row load
// it too.

template <class X>
constexpr int kChunk = X::code == 3 ? 4 : 8;  // 16 bytes of the stream

enum ResidualKind { kPre, kGate, kBoth };

struct Stats {
  float mean, inv;
};

template <int CHUNKS, int N>
__device__ Stats chunk_stats(int kind, const float (&v)[CHUNKS][N], int skip, int width, float eps,
                             int lanes, float* part) {
  Stats s{0.0f, 1.0f};
  if (kind == kNormNone) return s;
  if (kind == kNormLayer) {
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j)
#pragma unroll
      for (int e = 0; e < N; ++e) sum += j < CHUNKS - 1 || e >= skip ? v[j][e] : 0.0f;
    // A division: the mean of equal values whose sum is exact is then that value, and the row 0.
    // (The product with a rounded 1 / width misses it by 6e-8 of the value, which at 1000 and
    // eps 1e-6 is a row of 0.06.)  The time is the same.
    s.mean = row_sum(sum, lanes, part) / (float)width;
  }
  float sq = 0.0f;
#pragma unroll
  for (int j = 0; j < CHUNKS; ++j)
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float d = j < CHUNKS - 1 || e >= skip ? v[j][e] - s.mean : 0.0f;
      sq = fmaf(d, d, sq);
    }
  s.inv = 1.0f / sqrtf(row_sum(sq, lanes, part) * (1.0f / (float)width) + eps);
  return s;
}

// Combines a vector of fp32 or T values with the rows that share it, all of its loads sent out
// together.
template <class T, int ROWS, int CHUNKS, int N, class F>
__device__ inline void combine(const void* p, bool wide, int64_t base,
                               const unsigned (&at)[CHUNKS], float (&v)[ROWS][CHUNKS][N], F f) {
  if (p == nullptr) return;
  float w[CHUNKS][N];
  if (wide) {
    const void* row = row_of<F32>(p, base);
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) load_chunk<F32>(row, at[j], w[j]);
  } else {
    const void* row = row_of<T>(p, base);
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) load_chunk<T>(row, at[j], w[j]);
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i)
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j)
#pragma unroll
      for (int e = 0; e < N; ++e) v[i][j][e] = f(v[i][j][e], w[j][e]);
}

// Each row's norm, before its weight and bias.
template <int ROWS, int CHUNKS, int N>
__device__ inline void normalise(int kind, int skip, int width, float eps, int lanes, float* part,
                                 float (&v)[ROWS][CHUNKS][N]) {
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const Stats s = chunk_stats(kind, v[i], skip, width, eps, lanes, part);
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j)
#pragma unroll
      for (int e = 0; e < N; ++e) v[i][j][e] = (v[i][j][e] - s.mean) * s.inv;
  }
}

// Two rows of three chunks of 8 and a branch take more than the 128 registers that workgroups of
// 1024 leave a lane.
template <class X, int ROWS, int CHUNKS, int KIND>
constexpr bool kWideRows = ROWS > 1 && CHUNKS == 3 && KIND == kBoth && kChunk<X> == 8;
template <class X, int ROWS, int CHUNKS, int KIND>
constexpr int kMaxThreads = kWideRows<X, ROWS, CHUNKS, KIND> ? kThreads : 1024;

// Every level below is a kernel of its own, 300 with the types: 44 s of compiling on one core, the
// longest of the library's sources.
// ROWS > 1: rows of one sample (`per_sample` workgroups each) that share gate, scale and shift.
// STREAM: 1 loads the rows past the caches, 2 also stores the normalised ones past them.
template <class X, class T, int ROWS, int CHUNKS, int KIND, int STREAM>
__global__ __launch_bounds__((kMaxThreads<X, ROWS, CHUNKS, KIND>)) void residual_kernel(
    ResidualArgs a, int lanes, int64_t first, int per_sample) {
  constexpr int N = kChunk<X>;
  __shared__ float part[16];
  const int shift = 31 - __clz(lanes);
  int group = threadIdx.x >> shift;
  if (CHUNKS > 1) group = __builtin_amdgcn_readfirstlane(group);  // 64 lanes or more
  const int lane = threadIdx.x & (lanes - 1), per_block = blockDim.x >> shift;
  unsigned at[CHUNKS];
#pragma unroll
  for (int j = 0; j < CHUNKS; ++j) at[j] = N * (lane + lanes * j);
  const int last = a.width - N, skip = min(max((int)at[CHUNKS - 1] - last, 0), N);
  at[CHUNKS - 1] = min((int)at[CHUNKS - 1], last);

  int64_t b, n[ROWS];
  bool live[ROWS];
  if constexpr (ROWS == 1) {
    const int64_t row = (first + blockIdx.x) * per_block + group;
    live[0] = row < a.rows;
    const unsigned r32 = (unsigned)(live[0] ? row : a.rows - 1);
    b = r32 / (unsigned)a.tokens;
    n[0] = r32 - (unsigned)b * (unsigned)a.tokens;
  } else {
    const unsigned block = (unsigned)first + blockIdx.x;
    b = block / (unsigned)per_sample;
    const int64_t n0 = (int64_t)(block - (unsigned)b * (unsigned)per_sample) * per_block * ROWS;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      n[i] = n0 + i * per_block + group;
      live[i] = n[i] < a.tokens;
      n[i] = live[i] ? n[i] : a.tokens - 1;
    }
  }
  const auto times = [](float x, float w) { return x * w; };
  const auto plus = [](float x, float w) { return x + w; };
  const auto scaled = [](float x, float w) { return fmaf(x, w, x); };
  float v[ROWS][CHUNKS][N], f[KIND == kPre ? 1 : ROWS][CHUNKS][N];
  Rounded<X, N> r[ROWS][CHUNKS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const void* x = row_of<X>(a.x.p, b * a.x.b + n[i] * a.x.n);
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) load_chunk<X, (STREAM > 0)>(x, at[j], v[i][j]);
  }
  if constexpr (KIND != kPre) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const void* added = row_of<T>(a.branch.p, b * a.branch.b + n[i] * a.branch.n);
#pragma unroll
      for (int j = 0; j < CHUNKS; ++j) load_chunk<T, (STREAM > 0)>(added, at[j], f[i][j]);
    }
    if (a.post != kNormNone) normalise(a.post, skip, a.width, a.eps, lanes, part, f);
    combine<T>(a.branch_weight, a.wide_weight, 0, at, f, times);
    combine<T>(a.branch_bias, a.wide_weight, 0, at, f, plus);
    combine<T>(a.gate.p, a.wide_mod, b * a.gate.b + n[0] * a.gate.n, at, f, times);
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
      for (int j = 0; j < CHUNKS; ++j) {
#pragma unroll
        for (int e = 0; e < N; ++e) v[i][j][e] += f[i][j][e];
        r[i][j].set(v[i][j]);
      }
  }
  if constexpr (KIND != kGate) {
    normalise(a.norm, skip, a.width, a.eps, lanes, part, v);
    combine<T>(a.weight, a.wide_weight, 0, at, v, times);
    combine<T>(a.bias, a.wide_weight, 0, at, v, plus);
    combine<T>(a.scale.p, a.wide_mod, b * a.scale.b + n[0] * a.scale.n, at, v, scaled);
    combine<T>(a.shift.p, a.wide_mod, b * a.shift.b + n[0] * a.shift.n, at, v, plus);
  }
  // Stores last: a load behind a store would have to wait for it.  The new residual goes past
  // the caches (the next half's block comes first), the normalised rows to their next reader,
  // the next projection, unless there are more than the caches hold.
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    if (!live[i]) continue;
    void* ro = const_cast<void*>(row_of<X>(a.r.p, b * a.r.b + n[i] * a.r.n));
    void* yo = const_cast<void*>(row_of<T>(a.y.p, b * a.y.b + n[i] * a.y.n));
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) {
      const int from = j < CHUNKS - 1 ? 0 : skip;
      if constexpr (KIND != kPre) r[i][j].template store<true>(ro, at[j], from);
      if constexpr (KIND != kGate) {
        Rounded<T, N> y;
        y.set(v[i][j]);
        y.template store<(STREAM > 1)>(yo, at[j], from);
      }
    }
  }
}

// Widths that 1024 lanes of four chunks hold: up to 16,384 channels of an fp32 stream, 32,768 of a
// 16-bit one.  There norm_modulate at 3,000 x 32,768 takes 95 us, gated_residual_norm 169; a
// workgroup that reads the row again for each sum takes 534 and 1,134.
constexpr int kMinWidth = 8;
template <class X>
constexpr int kMaxWidth = 4 * 1024 * kChunk<X>;
constexpr int64_t kAllLanes = 256 * 2048;  // that the chip holds at once

// Normalised rows of this many bytes or more go past the caches.  The chain of kStreamBytes in us,
// through them -> past them: 101 MB of rows 583 -> 605, 201 MB 1,156 -> 1,188, 276 MB
// 1,747 -> 1,753, 365 MB 2,317 -> 2,310, 487 MB 3,087 -> 3,049, 730 MB 4,578 -> 4,547; the call
// alone, 487 MB (118,800 x 2048), 335 -> 321.
constexpr int64_t kPastBytes = int64_t(320) << 20;

template <class X, class T, int ROWS, int CHUNKS, int KIND>
hipError_t launch_rows(const ResidualArgs& a, int lanes, int threads, hipStream_t s) {
  const int64_t per_block = threads / lanes;
  const int64_t sample = (a.tokens + per_block * ROWS - 1) / (per_block * ROWS);
  const int64_t all =
      ROWS > 1 ? sample * (a.rows / a.tokens) : (a.rows + per_block - 1) / per_block;
  const int64_t bytes = a.rows * a.width *
                        (KIND == kPre    ? kBytes<X> + kBytes<T>
                         : KIND == kGate ? 2 * kBytes<X> + kBytes<T>
                                         : 2 * kBytes<X> + 2 * kBytes<T>);
  const bool past = KIND != kGate && a.rows * a.width * kBytes<T> >= kPastBytes;
  for (int64_t first = 0; first < all; first += kMaxBlocks) {
    const dim3 grid((unsigned)std::min(all - first, kMaxBlocks)), block((unsigned)threads);
    const auto launch = [&](auto stream) {
      residual_kernel<X, T, ROWS, CHUNKS, KIND, decltype(stream)::value>
          <<<grid, block, 0, s>>>(a, lanes, first, (int)sample);
    };
    if (past) {
      launch(std::integral_constant<int, KIND != kGate ? 2 : 1>());
    } else if (bytes >= kStreamBytes) {
      launch(std::integral_constant<int, 1>());
    } else {
      launch(std::integral_constant<int, 0>());
    }
  }
  return hipGetLastError();
}

// Rows a lane holds where they share their vectors.  A row's vectors are up to six times its own
// bytes, and their loads, though they hit the caches, are what bounds one row a lane.  Measured
// at 400 MB a call, us, one row -> several: norm_modulate at widths 256 / 768 / 2560 / 8192
// 101 -> 77 / 100 -> 81 / 93 -> 79 / 99 -> 80 (bf16), 88 -> 73 / 75 -> 72 / 90 -> 76 / 83 -> 76
// (fp32); gated_residual_norm 79 -> 69 / 81 -> 72 (bf16), 77 -> 68 at 4096 (fp32 stream).  A gate
// alone gains nothing from more than two chunks of 8 (720p: 169 -> 176), and four of them and a
// branch spill (gate_norm at 2048: 321 -> 596).
template <class X, int CHUNKS, int KIND>
constexpr int kRows = CHUNKS == 1                                               ? 4
                      : CHUNKS == 2                                             ? 2
                      : KIND == kPre || kChunk<X> == 4                          ? 2
                      : KIND == kBoth && CHUNKS == 3                            ? 2
                                                                                : 1;

template <class X, class T, int CHUNKS, int KIND>
hipError_t launch_chunks(const ResidualArgs& a, int lanes, hipStream_t s) {
  constexpr int ROWS = kRows<X, CHUNKS, KIND>;
  const int threads = lanes > kThreads ? lanes : kThreads;
  if constexpr (ROWS > 1) {
    // Where there are vectors, enough rows to fill the chip all the same, and samples long enough
    // that their last workgroups' idle rows do not count.
    bool several = a.branch_weight || a.branch_bias || a.gate.p || a.weight || a.bias ||
                   a.scale.p || a.shift.p;
    several = several && a.gate.n == 0 && a.scale.n == 0 && a.shift.n == 0 &&
              a.rows * lanes >= ROWS * kAllLanes && a.tokens >= 8 * ROWS * (threads / lanes);
    // These leave a lane's registers to three waves a SIMD: worth it for fp32 vectors, twice the
    // loads (480p: 72 -> 66), not for 16-bit ones (63 -> 65).
    if (kWideRows<X, ROWS, CHUNKS, KIND>) several = several && a.wide_mod && threads == kThreads;
    if (several) return launch_rows<X, T, ROWS, CHUNKS, KIND>(a, lanes, threads, s);
  }
  return launch_rows<X, T, 1, CHUNKS, KIND>(a, lanes, threads, s);
}

template <class X, class T, int KIND>
hipError_t launch_kind(const ResidualArgs& a, hipStream_t s) {
  constexpr int N = kChunk<X>;
  const int chunks = (a.width + N - 1) / N;
  int lanes = 1;
  while (lanes < chunks && lanes < 64) lanes *= 2;
  while (lanes * 4 < chunks) lanes *= 2;  // up to 4 chunks a lane, then more waves a row
  switch ((chunks + lanes - 1) / lanes) {
    case 1: return launch_chunks<X, T, 1, KIND>(a, lanes, s);
    case 2: return launch_chunks<X, T, 2, KIND>(a, lanes, s);
    case 3: return launch_chunks<X, T, 3, KIND>(a, lanes, s);
    default: return launch_chunks<X, T, 4, KIND>(a, lanes, s);
  }
}

template <class X, class T>
hipError_t launch(const ResidualArgs& a, hipStream_t s) {
  if (a.width >= kMinWidth && a.width <= kMaxWidth<X>) {
    if (!a.branch.p) return launch_kind<X, T, kPre>(a, s);
    return a.y.p ? launch_kind<X, T, kBoth>(a, s) : launch_kind<X, T, kGate>(a, s);
  }
  const int64_t grid = std::min(a.rows, kMaxBlocks);
  residual_rows_kernel<X, T><<<dim3((unsigned)grid), dim3(kThreads), 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t run_residual(const ResidualArgs& a, int x_dtype, int dtype, hipStream_t s) {
  if (x_dtype == dtype) {
    if (dtype == F32::code) return launch<F32, F32>(a, s);
    return dtype == BF16::code ? launch<BF16, BF16>(a, s) : launch<F16, F16>(a, s);
  }
  return dtype == BF16::code ? launch<F32, BF16>(a, s) : launch<F32, F16>(a, s);
}

}  // namespace recap

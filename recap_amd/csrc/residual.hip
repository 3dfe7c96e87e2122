// Norms before and after a block, fused with its scale, shift, gate and residual, one row
// (token) of the residual stream at a time:
//   r = x + gate * post(branch)                 post: none, RMS norm or LayerNorm
//   y = norm(r) * (1 + scale) + shift           norm: none, RMS norm or LayerNorm
// without a branch r = x.  Statistics, sums and products are fp32; r and y are each rounded
// once, to their own type, and y is taken from the unrounded r.
#include "kernels.hpp"
#include "rows.hpp"

namespace recap {
namespace {

constexpr int kThreads = 256;

// A vector of fp32 or T values, by a flag that is uniform over the launch.
template <class T>
__device__ inline float load_either(const void* p, bool wide, int64_t i) {
  return wide ? load_elem<F32>(p, i) : load_elem<T>(p, i);
}

// Sum over the workgroup, in every thread: lanes by a butterfly, waves in order.
__device__ inline float block_sum(float v, float* part) {
  v = wave_sum(v);
  __syncthreads();  // the previous sum's readers are done with `part`
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = part[0];
  for (int w = 1; w < kThreads / 64; ++w) s += part[w];
  return s;
}

struct Stats {
  float mean, inv;
};

// Mean (LayerNorm only) and reciprocal deviation of value(0 .. width - 1).
template <class V>
__device__ Stats row_stats(int kind, int width, float eps, float* part, V value) {
  Stats s{0.0f, 1.0f};
  if (kind == kNormNone) return s;
  if (kind == kNormLayer) {
    float sum = 0.0f;
    for (int c = threadIdx.x; c < width; c += kThreads) sum += value(c);
    s.mean = block_sum(sum, part) / (float)width;
  }
  float sq = 0.0f;
  for (int c = threadIdx.x; c < width; c += kThreads) {
    const float d = value(c) - s.mean;
    sq = fmaf(d, d, sq);
  }
  s.inv = 1.0f / sqrtf(block_sum(sq, part) / (float)width + eps);
  return s;
}

// One workgroup per row; every pass reads the row again.
template <class X, class T>
__global__ __launch_bounds__(kThreads) void residual_rows_kernel(ResidualArgs a) {
  __shared__ float part[kThreads / 64];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t b = row / a.tokens, n = row - b * a.tokens;
    const int64_t xo = b * a.x.b + n * a.x.n, bo = b * a.branch.b + n * a.branch.n,
                  go = b * a.gate.b + n * a.gate.n, so = b * a.scale.b + n * a.scale.n,
                  ho = b * a.shift.b + n * a.shift.n;
    const auto added = [&](int c) { return load_elem<T>(a.branch.p, bo + c); };
    Stats post{0.0f, 1.0f};
    if (a.branch.p) post = row_stats(a.post, a.width, a.eps, part, added);
    const auto value = [&](int c) {
      float r = load_elem<X>(a.x.p, xo + c);
      if (a.branch.p) {
        float f = (added(c) - post.mean) * post.inv;
        if (a.branch_weight) f *= load_either<T>(a.branch_weight, a.wide_weight, c);
        if (a.branch_bias) f += load_either<T>(a.branch_bias, a.wide_weight, c);
        r = a.gate.p ? fmaf(load_either<T>(a.gate.p, a.wide_mod, go + c), f, r) : r + f;
      }
      return r;
    };
    Stats s{0.0f, 1.0f};
    if (a.y.p) s = row_stats(a.norm, a.width, a.eps, part, value);
    const int64_t ro = b * a.r.b + n * a.r.n, yo = b * a.y.b + n * a.y.n;
    __syncthreads();  // an output may be an input: the row's statistics are all taken
    for (int c = threadIdx.x; c < a.width; c += kThreads) {
      const float r = value(c);
      if (a.y.p) {
        float y = (r - s.mean) * s.inv;
        if (a.weight) y *= load_either<T>(a.weight, a.wide_weight, c);
        if (a.bias) y += load_either<T>(a.bias, a.wide_weight, c);
        if (a.scale.p) y *= 1.0f + load_either<T>(a.scale.p, a.wide_mod, so + c);
        if (a.shift.p) y += load_either<T>(a.shift.p, a.wide_mod, ho + c);
        store_elem<T>(const_cast<void*>(a.y.p), yo + c, y);
      }
      if (a.r.p) store_elem<X>(const_cast<void*>(a.r.p), ro + c, r);
    }
  }
}

// ---------------------------------------------------------------------------------------
// Rows in registers: one pass over the data.  `lanes` lanes (a power of two) share a row in
// chunks of 8 elements, chunk c in lane c % lanes, so a lane holds CHUNKS chunks; rows of more
// than 64 lanes join their waves' sums through LDS.  Loads are 16 bytes wide at any alignment.
// The row's last chunk is loaded from its last 8 elements, its elements before the chunk's
// own (`skip` of them) left out of sums and stores; lanes past the row load it too.

enum ResidualKind { kPre, kGate, kBoth };

template <int CHUNKS>
__device__ Stats chunk_stats(int kind, const float (&v)[CHUNKS][8], int skip, int width, float eps,
                             int lanes, float* part) {
  Stats s{0.0f, 1.0f};
  if (kind == kNormNone) return s;
  const float per = 1.0f / (float)width;
  if (kind == kNormLayer) {
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += j < CHUNKS - 1 || e >= skip ? v[j][e] : 0.0f;
    s.mean = row_sum(sum, lanes, part) * per;
  }
  float sq = 0.0f;
#pragma unroll
  for (int j = 0; j < CHUNKS; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = j < CHUNKS - 1 || e >= skip ? v[j][e] - s.mean : 0.0f;
      sq = fmaf(d, d, sq);
    }
  s.inv = 1.0f / sqrtf(row_sum(sq, lanes, part) * per + eps);
  return s;
}

template <class X, class T, int CHUNKS, int KIND>
__global__ __launch_bounds__(1024) void residual_kernel(ResidualArgs a, int lanes) {
  __shared__ float part[16];
  const int shift = 31 - __clz(lanes);
  int group = threadIdx.x >> shift;
  if (CHUNKS > 1) group = __builtin_amdgcn_readfirstlane(group);  // 64 lanes or more
  const int lane = threadIdx.x & (lanes - 1), per_block = blockDim.x >> shift;
  int at[CHUNKS];
#pragma unroll
  for (int j = 0; j < CHUNKS; ++j) at[j] = 8 * (lane + lanes * j);
  const int skip = min(max(at[CHUNKS - 1] - (a.width - 8), 0), 8);
  at[CHUNKS - 1] = min(at[CHUNKS - 1], a.width - 8);

  const int64_t row = (int64_t)blockIdx.x * per_block + group;
  const bool live = row < a.rows;
  const unsigned r32 = (unsigned)(live ? row : a.rows - 1);
  const int64_t b = r32 / (unsigned)a.tokens, n = r32 - (unsigned)b * (unsigned)a.tokens;
  float v[CHUNKS][8];
  {
    const int64_t base = b * a.x.b + n * a.x.n;
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) load8<X>(a.x.p, base + at[j], v[j]);
  }
  if constexpr (KIND != kPre) {
    float f[CHUNKS][8];
    const int64_t base = b * a.branch.b + n * a.branch.n, go = b * a.gate.b + n * a.gate.n;
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) load8<T>(a.branch.p, base + at[j], f[j]);
    const Stats s = chunk_stats<CHUNKS>(a.post, f, skip, a.width, a.eps, lanes, part);
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) {
      float w[8];
      if (a.post != kNormNone) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[j][e] = (f[j][e] - s.mean) * s.inv;
        if (a.branch_weight) {
          load8_either<T>(a.branch_weight, a.wide_weight, at[j], w);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[j][e] *= w[e];
        }
        if (a.branch_bias) {
          load8_either<T>(a.branch_bias, a.wide_weight, at[j], w);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[j][e] += w[e];
        }
      }
      if (a.gate.p) {
        load8_either<T>(a.gate.p, a.wide_mod, go + at[j], w);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] = fmaf(w[e], f[j][e], v[j][e]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] += f[j][e];
      }
    }
    const int64_t ro = b * a.r.b + n * a.r.n;
    if (live) {
#pragma unroll
      for (int j = 0; j < CHUNKS; ++j)
        store8<X>(const_cast<void*>(a.r.p), ro + at[j], v[j], j < CHUNKS - 1 ? 0 : skip);
    }
  }
  if constexpr (KIND != kGate) {
    const Stats s = chunk_stats<CHUNKS>(a.norm, v, skip, a.width, a.eps, lanes, part);
    const int64_t yo = b * a.y.b + n * a.y.n, so = b * a.scale.b + n * a.scale.n,
                  ho = b * a.shift.b + n * a.shift.n;
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) {
      float w[8], y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = (v[j][e] - s.mean) * s.inv;
      if (a.weight) {
        load8_either<T>(a.weight, a.wide_weight, at[j], w);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] *= w[e];
      }
      if (a.bias) {
        load8_either<T>(a.bias, a.wide_weight, at[j], w);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] += w[e];
      }
      if (a.scale.p) {
        load8_either<T>(a.scale.p, a.wide_mod, so + at[j], w);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = fmaf(y[e], w[e], y[e]);
      }
      if (a.shift.p) {
        load8_either<T>(a.shift.p, a.wide_mod, ho + at[j], w);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] += w[e];
      }
      if (live)
        store8<T>(const_cast<void*>(a.y.p), yo + at[j], y, j < CHUNKS - 1 ? 0 : skip);
    }
  }
}

constexpr int kMinWidth = 8, kMaxWidth = 8 * 1024 * 4;

template <class X, class T, int CHUNKS, int KIND>
hipError_t launch_rows(const ResidualArgs& a, int lanes, hipStream_t s) {
  const int threads = lanes > kThreads ? lanes : kThreads;
  const int64_t per_block = threads / lanes;
  const int64_t grid = (a.rows + per_block - 1) / per_block;
  residual_kernel<X, T, CHUNKS, KIND>
      <<<dim3((unsigned)grid), dim3((unsigned)threads), 0, s>>>(a, lanes);
  return hipGetLastError();
}

template <class X, class T, int KIND>
hipError_t launch_kind(const ResidualArgs& a, hipStream_t s) {
  const int chunks = (a.width + 7) / 8;
  int lanes = 1;
  while (lanes < chunks && lanes < 64) lanes *= 2;
  while (lanes * 4 < chunks) lanes *= 2;  // up to 4 chunks a lane, then more waves a row
  switch ((chunks + lanes - 1) / lanes) {
    case 1: return launch_rows<X, T, 1, KIND>(a, lanes, s);
    case 2: return launch_rows<X, T, 2, KIND>(a, lanes, s);
    case 3: return launch_rows<X, T, 3, KIND>(a, lanes, s);
    default: return launch_rows<X, T, 4, KIND>(a, lanes, s);
  }
}

template <class X, class T>
hipError_t launch(const ResidualArgs& a, hipStream_t s) {
  if (a.width >= kMinWidth && a.width <= kMaxWidth) {
    if (!a.branch.p) return launch_kind<X, T, kPre>(a, s);
    return a.y.p ? launch_kind<X, T, kBoth>(a, s) : launch_kind<X, T, kGate>(a, s);
  }
  const int64_t grid = a.rows < (1 << 20) ? a.rows : (1 << 20);
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

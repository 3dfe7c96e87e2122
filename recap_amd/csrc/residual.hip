// Norms before and after a block, fused with its scale, shift, gate and residual, one row
// (token) of the residual stream at a time:
//   r = x + gate * post(branch)                 post: none, RMS norm or LayerNorm
//   y = norm(r) * (1 + scale) + shift           norm: none, RMS norm or LayerNorm
// without a branch r = x.  Statistics, sums and products are fp32; r and y are each rounded
// once, to their own type, and y is taken from the unrounded r.
#include "kernels.hpp"

namespace recap {
namespace {

constexpr int kThreads = 256;

struct F32 {
  static constexpr int code = 3;
};

template <class T>
__device__ inline float load_elem(const void* p, int64_t i) {
  if constexpr (T::code == 3) {
    return static_cast<const float*>(p)[i];
  } else {
    return T::to_f(static_cast<const uint16_t*>(p)[i]);
  }
}

template <class T>
__device__ inline void store_elem(void* p, int64_t i, float v) {
  if constexpr (T::code == 3) {
    static_cast<float*>(p)[i] = v;
  } else {
    static_cast<uint16_t*>(p)[i] = T::from_f(v);
  }
}

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

template <class X, class T>
hipError_t launch(const ResidualArgs& a, hipStream_t s) {
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

// Queries and keys of an attention call from their projections: an optional norm of each
// head's channels (RMS norm or LayerNorm) or of all heads' (RMS norm), and the rotation of
// the video tokens by their (time, height, width) positions.
//   frequency i of d/2 belongs to the axis whose section holds it and has the (cos, sin) of
//   that axis's table at the token's position on it;
//   its channels (p, q), 2i and 2i + 1 or i and i + d/2, become (p c - q s, q c + p s).
// Statistics and products are fp32, rounded once.
#include "kernels.hpp"

namespace recap {
namespace {

constexpr int kWaves = 4;

// One workgroup per token of q or k, one wave per head in turn, one lane per pair.
template <class T, int D>
__global__ __launch_bounds__(64 * kWaves) void rotary_kernel(RotaryArgs a) {
  constexpr int kPairs = D / 2;
  __shared__ float part[kWaves];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int which = blockIdx.y;
  const RotaryTensor& t = a.x[which];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t b = row / a.tokens, n = row - b * a.tokens;
    const int64_t v = n - a.offset;
    const bool video = v >= 0 && v < a.video, live = lane < kPairs;
    float c = 1.0f, s = 0.0f;
    if (video && live) {
      const int64_t plane = (int64_t)a.axis[1].length * a.axis[2].length;
      const int64_t pos[3] = {v / plane, v / a.axis[2].length % a.axis[1].length,
                              v % a.axis[2].length};
      int first = 0;
      for (int i = 0; i < 3; ++i) {
        const int pairs = a.axis[i].pairs;
        if (lane >= first && lane < first + pairs) {
          const float* e = a.axis[i].table + 2 * (pos[i] * pairs + lane - first);
          c = e[0];
          s = e[1];
        }
        first += pairs;
      }
    }
    const int i0 = a.halves ? lane : 2 * lane, i1 = a.halves ? lane + kPairs : 2 * lane + 1;
    const uint16_t* src = t.in + b * t.in_b + n * t.in_n;
    uint16_t* dst = t.out + b * t.out_b + n * t.out_n;
    const auto load = [&](int h, float& p, float& q) {
      p = live ? T::to_f(src[h * t.in_h + i0]) : 0.0f;
      q = live ? T::to_f(src[h * t.in_h + i1]) : 0.0f;
    };
    float inv = 1.0f;
    if (a.norm == kRotaryRmsAll) {
      float sq = 0.0f, p, q;
      for (int h = wave; h < t.heads; h += kWaves) {
        load(h, p, q);
        sq += p * p + q * q;
      }
      sq = wave_sum(sq);
      __syncthreads();
      if (lane == 0) part[wave] = sq;
      __syncthreads();
      sq = 0.0f;
      for (int w = 0; w < kWaves; ++w) sq += part[w];
      inv = 1.0f / sqrtf(sq / (float)(t.heads * D) + a.eps);
    }
    for (int h = wave; h < t.heads; h += kWaves) {
      float p, q;
      load(h, p, q);
      if (a.norm == kRotaryLayer) {
        const float mean = wave_sum(p + q) / (float)D;
        p = live ? p - mean : 0.0f;
        q = live ? q - mean : 0.0f;
      }
      if (a.norm == kRotaryRms || a.norm == kRotaryLayer)
        inv = 1.0f / sqrtf(wave_sum(p * p + q * q) / (float)D + a.eps);
      p *= inv;
      q *= inv;
      if (!live) continue;
      const int w = a.norm == kRotaryRmsAll ? h * D : 0;
      if (t.weight) {
        p *= a.wide_weight ? ((const float*)t.weight)[w + i0]
                           : T::to_f(((const uint16_t*)t.weight)[w + i0]);
        q *= a.wide_weight ? ((const float*)t.weight)[w + i1]
                           : T::to_f(((const uint16_t*)t.weight)[w + i1]);
      }
      if (t.bias) {
        p += a.wide_weight ? ((const float*)t.bias)[w + i0]
                           : T::to_f(((const uint16_t*)t.bias)[w + i0]);
        q += a.wide_weight ? ((const float*)t.bias)[w + i1]
                           : T::to_f(((const uint16_t*)t.bias)[w + i1]);
      }
      dst[h * t.out_h + i0] = T::from_f(p * c - q * s);
      dst[h * t.out_h + i1] = T::from_f(q * c + p * s);
    }
  }
}

template <class T>
hipError_t launch(const RotaryArgs& a, int dim, hipStream_t s) {
  const dim3 grid((unsigned)(a.rows < (1 << 20) ? a.rows : (1 << 20)), a.tensors);
  if (dim == 128) {
    rotary_kernel<T, 128><<<grid, dim3(64 * kWaves), 0, s>>>(a);
  } else {
    rotary_kernel<T, 64><<<grid, dim3(64 * kWaves), 0, s>>>(a);
  }
  return hipGetLastError();
}

}  // namespace

hipError_t run_rotary(const RotaryArgs& a, int dtype, int dim, hipStream_t s) {
  return dtype == BF16::code ? launch<BF16>(a, dim, s) : launch<F16>(a, dim, s);
}

}  // namespace recap

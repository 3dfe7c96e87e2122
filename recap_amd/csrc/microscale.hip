// Rows to their microscaled form and back (microscale.hpp has the formats), one pass over the data.
//
// Bound by memory: 2 or 4 bytes a value on one side, 0.53 (fp4) or 1.03 (int8) on the other.  A lane
// holds 8 values (16 bytes of a 16-bit type), the four lanes of a block take its largest magnitude by
// two lane exchanges, and each lane sends kChunks loads out before it uses the first.  Rows without
// gaps whose width needs no filling are one long row.
#include <algorithm>

#include "kernels.hpp"
#include "microscale.hpp"

namespace recap {
namespace {

constexpr int kThreads = 256;
constexpr int kChunks = 4;  // of 8 values a lane

// Where a thread's chunks lie: `lanes` lanes (a power of two, at least a block's four) share a row.
struct Place {
  int64_t row;
  int64_t chunk[kChunks];
  bool live[kChunks];
};

__device__ inline Place place_of(const MxRowsArgs& a, int lanes, unsigned segments, unsigned first) {
  const int shift = 31 - __clz(lanes);
  const unsigned block = first + blockIdx.x;
  const unsigned group = block / segments;
  const int64_t segment = block - group * segments;
  Place p;
  p.row = (int64_t)group * (kThreads >> shift) + (threadIdx.x >> shift);
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    p.chunk[j] = segment * lanes * kChunks + (int64_t)j * lanes + (threadIdx.x & (lanes - 1));
    p.live[j] = p.row < a.rows && p.chunk[j] < a.chunks;
  }
  return p;
}

template <class T, int FORMAT>
__global__ __launch_bounds__(kThreads) void quantise_kernel(MxRowsArgs a, int lanes,
                                                            unsigned segments, unsigned first) {
  const Place p = place_of(a, lanes, segments, first);
  float v[kChunks][8];
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    const int64_t at = 8 * p.chunk[j], left = a.width - at;
    const int64_t from = p.row * a.stride + at;
    if (p.live[j] && left >= 8) {
      load_chunk<T>(row_of<T>(a.values, from), 0, v[j]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        v[j][e] = p.live[j] && e < left ? load_elem<T>(a.values, from + e) : 0.0f;
    }
  }
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    const unsigned s = mx_scale<FORMAT>(quad_max(magnitude_bits(v[j])));
    if (!p.live[j]) continue;
    const int64_t to = p.row * a.chunks + p.chunk[j];
    if constexpr (FORMAT == kMxFp4) {
      static_cast<unsigned*>(a.codes)[to] = mx_fp4_codes(v[j], s);
    } else {
      static_cast<u32x2*>(a.codes)[to] = mx_int8_codes(v[j], s);
    }
    if ((threadIdx.x & 3) == 0) a.scales[to >> 2] = (uint8_t)s;
  }
}

template <class T, int FORMAT>
__global__ __launch_bounds__(kThreads) void dequantise_kernel(MxRowsArgs a, int lanes,
                                                              unsigned segments, unsigned first) {
  const Place p = place_of(a, lanes, segments, first);
  u32x2 w[kChunks] = {};
  unsigned s[kChunks] = {};
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    if (!p.live[j]) continue;
    const int64_t from = p.row * a.chunks + p.chunk[j];
    if constexpr (FORMAT == kMxFp4) {
      w[j][0] = static_cast<const unsigned*>(a.codes)[from];
    } else {
      w[j] = static_cast<const u32x2*>(a.codes)[from];
    }
    s[j] = a.scales[from >> 2];
  }
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    const int64_t at = 8 * p.chunk[j], left = a.width - at;
    if (!p.live[j] || left <= 0) continue;
    float v[8];
    if constexpr (FORMAT == kMxFp4) {
      mx_fp4_values(w[j][0], s[j], v);
    } else {
      mx_int8_values(w[j], s[j], v);
    }
    const int64_t to = p.row * a.stride + at;
    if (left >= 8) {
      Rounded<T, 8> r;
      r.set(v);
      r.template store<false>(const_cast<void*>(row_of<T>(a.values, to)), 0, 0);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < left) store_elem<T>(a.values, to + e, v[e]);
    }
  }
}

template <class T, int FORMAT>
hipError_t launch(MxRowsArgs a, bool read, hipStream_t s) {
  if (a.stride == a.width && a.width % mx_fill(FORMAT) == 0) {
    a.width *= a.rows;
    a.stride = a.width;
    a.rows = 1;
  }
  a.chunks = mx_filled(FORMAT, a.width) / 8;
  int lanes = 4;
  while (lanes < kThreads && lanes * kChunks < a.chunks) lanes *= 2;
  const int64_t segments = (a.chunks + lanes * kChunks - 1) / (lanes * kChunks);
  const int64_t per_block = kThreads / lanes;
  const int64_t all = (a.rows + per_block - 1) / per_block * segments;
  for (int64_t first = 0; first < all; first += kMaxBlocks) {
    const dim3 grid((unsigned)std::min(all - first, kMaxBlocks));
    if (read) {
      dequantise_kernel<T, FORMAT>
          <<<grid, dim3(kThreads), 0, s>>>(a, lanes, (unsigned)segments, (unsigned)first);
    } else {
      quantise_kernel<T, FORMAT>
          <<<grid, dim3(kThreads), 0, s>>>(a, lanes, (unsigned)segments, (unsigned)first);
    }
  }
  return hipGetLastError();
}

template <int FORMAT>
hipError_t launch_type(const MxRowsArgs& a, int dtype, bool read, hipStream_t s) {
  if (dtype == F32::code) return launch<F32, FORMAT>(a, read, s);
  return dtype == BF16::code ? launch<BF16, FORMAT>(a, read, s) : launch<F16, FORMAT>(a, read, s);
}

hipError_t run(const MxRowsArgs& a, int dtype, int format, bool read, hipStream_t s) {
  return format == kMxFp4 ? launch_type<kMxFp4>(a, dtype, read, s)
                          : launch_type<kMxInt8>(a, dtype, read, s);
}

}  // namespace

hipError_t run_mx_quantise(const MxRowsArgs& a, int dtype, int format, hipStream_t s) {
  return run(a, dtype, format, false, s);
}

hipError_t run_mx_dequantise(const MxRowsArgs& a, int dtype, int format, hipStream_t s) {
  return run(a, dtype, format, true, s);
}

}  // namespace recap

// Rows to their microscaled form and back (microscale.hpp has the formats), one pass over the data.
//
// Bound by memory: 2 or 4 bytes a value on one side, 0.53 (fp4) or 1.03 (int8) on the other.  A lane
// holds 8 values (16 bytes of a 16-bit type), the four lanes of a block take its largest magnitude by
// two lane exchanges, and each lane sends kChunks loads out before it uses the first.  fp4 codes, four
// bytes a lane, change places within the four lanes, so that a lane stores a whole block (118,800 x
// 2,048: 145 us with 4-byte stores through the caches, 149 with whole blocks, 101 with those past the
// caches, 6.1 TB/s).  2.85 million rows of 128 into int8 192 us, 5.8 TB/s, and back 176, 6.3 (through
// the caches 212 and 185).  Rows without gaps whose width needs no filling are one long row.
#include <algorithm>
#include <type_traits>

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

// Words w[j] of the four lanes of a block exchanged: lane q's w[i] becomes lane i's w[q].
__device__ inline void quad_transpose(unsigned (&w)[4]) {
  const bool b0 = threadIdx.x & 1, b1 = threadIdx.x & 2;
  const auto swap = [](unsigned& lo, unsigned& hi, bool upper, auto from) {
    const unsigned got = from(upper ? lo : hi);
    lo = upper ? got : lo;
    hi = upper ? hi : got;
  };
  const auto lane1 = [](unsigned x) {
    return (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xf, 0xf, false);
  };
  const auto lane2 = [](unsigned x) {
    return (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xf, 0xf, false);
  };
  swap(w[0], w[1], b0, lane1);
  swap(w[2], w[3], b0, lane1);
  swap(w[0], w[2], b1, lane2);
  swap(w[1], w[3], b1, lane2);
}

// The block a lane stores or loads whole: the one of its chunk `threadIdx.x % 4`.
__device__ inline int64_t own_block(const MxRowsArgs& a, const Place& p, bool* live) {
  const int q = threadIdx.x & 3;
  int64_t chunk = p.chunk[0];
  *live = p.live[0];
#pragma unroll
  for (int j = 1; j < kChunks; ++j) {
    chunk = q == j ? p.chunk[j] : chunk;
    *live = q == j ? p.live[j] : *live;
  }
  return (p.row * a.chunks + chunk) >> 2;
}

template <class T, int FORMAT, bool STREAM>
__global__ __launch_bounds__(kThreads) void quantise_kernel(MxRowsArgs a, int lanes,
                                                            unsigned segments, unsigned first) {
  const Place p = place_of(a, lanes, segments, first);
  float v[kChunks][8];
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    const int64_t at = 8 * p.chunk[j], left = a.width - at;
    const int64_t from = p.row * a.stride + at;
    if (p.live[j] && left >= 8) {
      load_chunk<T, STREAM>(row_of<T>(a.values, from), 0, v[j]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        v[j][e] = p.live[j] && e < left ? load_elem<T>(a.values, from + e) : 0.0f;
    }
  }
  // Codes: 8 bytes a lane of int8 as they are; of fp4, whose four bytes a lane make poor stores, and
  // of the scales the lane's own block.
  unsigned w[kChunks], own = 0;
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    const unsigned s = mx_scale<FORMAT>(quad_max(magnitude_bits(v[j])));
    own = (threadIdx.x & 3) == j ? s : own;
    if constexpr (FORMAT == kMxFp4) {
      w[j] = mx_fp4_codes(v[j], s);
    } else if (p.live[j]) {
      const int64_t to = p.row * a.chunks + p.chunk[j];
      store_words2<STREAM>(static_cast<u32x2*>(a.codes) + to, mx_int8_codes(v[j], s));
    }
  }
  if constexpr (FORMAT == kMxFp4) quad_transpose(w);
  bool live;
  const int64_t block = own_block(a, p, &live);
  if (!live) return;
  if constexpr (FORMAT == kMxFp4)
    store_words4<STREAM>(static_cast<u32x4*>(a.codes) + block, u32x4{w[0], w[1], w[2], w[3]});
  a.scales[block] = (uint8_t)own;
}

// The 32 fp32 values of a block to memory, its four lanes side by side: each lane's own two halves would
// leave gaps of 16 bytes in a store (us so -> side by side: fp4 4,000 x 4,096 15.7 -> 12.9, 5.8 TB/s,
// 60,000 x 2,048 111 -> 101; int8 16.0 -> 13.7 and 125 -> 127).
template <bool STREAM>
__device__ inline void store_block(void* block, const float (&v)[8]) {
  const bool odd = threadIdx.x & 1;
  u32x4 near, far;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int lo = (int)__float_as_uint(v[e]), hi = (int)__float_as_uint(v[4 + e]);
    const unsigned lo0 = (unsigned)__builtin_amdgcn_mov_dpp(lo, 0x50, 0xf, 0xf, false);  // lanes 0 0 1 1
    const unsigned hi0 = (unsigned)__builtin_amdgcn_mov_dpp(hi, 0x50, 0xf, 0xf, false);
    const unsigned lo1 = (unsigned)__builtin_amdgcn_mov_dpp(lo, 0xFA, 0xf, 0xf, false);  // 2 2 3 3
    const unsigned hi1 = (unsigned)__builtin_amdgcn_mov_dpp(hi, 0xFA, 0xf, 0xf, false);
    near[e] = odd ? hi0 : lo0;
    far[e] = odd ? hi1 : lo1;
  }
  const int at = 4 * (threadIdx.x & 3);
  store_words4<STREAM>(place<F32>(block, at), near);
  store_words4<STREAM>(place<F32>(block, 16 + at), far);
}

template <class T, int FORMAT, bool STREAM>
__global__ __launch_bounds__(kThreads) void dequantise_kernel(MxRowsArgs a, int lanes,
                                                              unsigned segments, unsigned first) {
  const Place p = place_of(a, lanes, segments, first);
  bool live;
  const int64_t block = own_block(a, p, &live);
  unsigned own = 0;
  u32x2 w[kChunks] = {};
  if constexpr (FORMAT == kMxFp4) {
    unsigned x[kChunks] = {};
    if (live) {
      const u32x4 c = load_words4<STREAM>(static_cast<const u32x4*>(a.codes) + block);
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = c[i];
    }
    quad_transpose(x);
#pragma unroll
    for (int j = 0; j < kChunks; ++j) w[j][0] = x[j];
  } else {
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
      if (p.live[j])
        w[j] = load_words2<STREAM>(static_cast<const u32x2*>(a.codes) + p.row * a.chunks + p.chunk[j]);
  }
  if (live) own = a.scales[block];
  const unsigned s[kChunks] = {
      (unsigned)__builtin_amdgcn_mov_dpp((int)own, 0x00, 0xf, 0xf, false),
      (unsigned)__builtin_amdgcn_mov_dpp((int)own, 0x55, 0xf, 0xf, false),
      (unsigned)__builtin_amdgcn_mov_dpp((int)own, 0xAA, 0xf, 0xf, false),
      (unsigned)__builtin_amdgcn_mov_dpp((int)own, 0xFF, 0xf, 0xf, false)};
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
    if constexpr (T::code == F32::code) {
      const int before = 8 * (threadIdx.x & 3);  // in the block
      if (left + before >= kMxBlock) {
        store_block<STREAM>(const_cast<void*>(row_of<T>(a.values, to - before)), v);
        continue;
      }
    }
    if (left >= 8) {
      Rounded<T, 8> r;
      r.set(v);
      r.template store<STREAM>(const_cast<void*>(row_of<T>(a.values, to)), 0, 0);
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
  // The lanes of a row: the fewest workgroups, weighted by what the short stretches of memory cost
  // that few lanes reach at once.  us by 8, 16, 32, 64 and 128 lanes, bf16: 118,800 rows of 1,155 into
  // fp4 80, 72, 86, 96, 132 and back 91, 84, 116, 81, 107; 40,000 of 2,283 48, 45, 43, 54, 49 and 43,
  // 41, 39, 45, 37; 311,850 of 37 27, 47, 87, ... and 16, 21, 36, ...  At these and five more sizes in
  // both formats the rule's choice takes up to 7% longer than the best number; of fp32, 8% (once 14:
  // 118,800 x 1,155 into int8 137 with 16 lanes, 120 with 128).
  const auto blocks = [&](int64_t n) {
    const int64_t per_block = kThreads / n;
    return (a.rows + per_block - 1) / per_block * ((a.chunks + n * kChunks - 1) / (n * kChunks));
  };
  const auto cost = [&](int64_t n) {
    const double weight = read ? (n >= 64 ? 1.0 : n == 32 ? 1.2 : n == 16 ? 1.55 : n == 8 ? 1.9 : 2.6)
                               : (n >= 32 ? 1.0 : n == 16 ? 1.15 : n == 8 ? 1.45 : 1.9);
    return weight * (double)blocks(n);
  };
  int lanes = kThreads;
  for (int n = kThreads / 2; n >= 4; n /= 2)
    if (cost(n) < cost(lanes)) lanes = n;
  const int64_t segments = (a.chunks + lanes * kChunks - 1) / (lanes * kChunks), all = blocks(lanes);
  // Past the caches only whole lines: fp32 values read back are stored half a line at a time and never
  // go past them, and rows off 16 bytes share their ends (us through them -> past them: 118,800 x 2,048
  // 112 -> 100, 60,000 x 2,048 of fp32 read back 101 -> 152, 118,800 x 1,155 82 -> 98).
  const bool past = a.rows * a.width * (kBytes<T> + 1) >= kStreamBytes &&
                    (reinterpret_cast<uintptr_t>(a.values) | a.stride * kBytes<T>) % 16 == 0;
  for (int64_t first = 0; first < all; first += kMaxBlocks) {
    const dim3 grid((unsigned)std::min(all - first, kMaxBlocks));
    const auto launch = [&](auto stream) {
      constexpr bool STREAM = decltype(stream)::value;
      if (read) {
        dequantise_kernel<T, FORMAT, STREAM && T::code != F32::code>
            <<<grid, dim3(kThreads), 0, s>>>(a, lanes, (unsigned)segments, (unsigned)first);
      } else {
        quantise_kernel<T, FORMAT, STREAM>
            <<<grid, dim3(kThreads), 0, s>>>(a, lanes, (unsigned)segments, (unsigned)first);
      }
    };
    if (past) {
      launch(std::integral_constant<bool, true>());
    } else {
      launch(std::integral_constant<bool, false>());
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

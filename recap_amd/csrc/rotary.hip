// Queries and keys of an attention call from their projections: an optional norm of each
// head's channels (RMS norm or LayerNorm) or of all heads' (RMS norm), and the rotation of
// the video tokens by their (time, height, width) positions.
//   frequency i of d/2 belongs to the axis whose section holds it and has the (cos, sin) of
//   that axis's table at the token's position on it;
//   its channels (p, q), 2i and 2i + 1 or i and i + d/2, become (p c - q s, q c + p s).
// Statistics and products are fp32, rounded once.
//
// A lane holds 16 channels of a (token, head) row in two 16-byte chunks, u and u + d/16, so
// that both pairings stay within the lane; d/16 lanes hold the row.  A wave takes `side` heads
// of each of its tokens at once (side a power of two) and walks the others, so a token's
// (cos, sin) are looked up once per wave.
//
// Bound by memory: 4 bytes and 3 to 10 flop an element; by counters the kernel moves Q and K once
// in and once out.  24 heads of 128 at 119,056 tokens with RMS norm take 474 us, 6.2 TB/s of the
// 6.5 that a copy kernel reaches past the caches (495 us where the outputs are put head by head);
// 12 heads with a norm over all of them at 32,760 tokens 68 us, 5.9; 48 heads of 64 at 45,106
// tokens with LayerNorm 192 us, 5.8: a load covers half a line of a head of 64, so those go
// through the caches.  One head alone (90 us for 400 MB) leaves too few loads in flight.
#include <algorithm>
#include <type_traits>

#include "kernels.hpp"
#include "rows.hpp"

namespace recap {
namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 4;  // head rows in flight per lane

template <class T>
__device__ inline void load16(const void* p, bool wide, unsigned i, unsigned half,
                              float (&v)[16]) {
  float lo[8], hi[8];
  if (wide) {
    load_chunk<F32>(p, i, lo);
    load_chunk<F32>(p, i + half, hi);
  } else {
    load_chunk<T>(p, i, lo);
    load_chunk<T>(p, i + half, hi);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    v[e] = lo[e];
    v[8 + e] = hi[e];
  }
}

template <class T, int D, bool HALVES, int NORM, bool STREAM>
__global__ __launch_bounds__(kThreads) void rotary_kernel(RotaryArgs a, int64_t first_block) {
  constexpr int kLanes = D / 16, kRows = 64 / kLanes;
  const RotaryTensor& t = a.x[blockIdx.y];
  const int side = t.side;
  const int lane = threadIdx.x & 63, u = lane & (kLanes - 1), g = lane / kLanes;
  const int hl = g & (side - 1), tokens = kRows / side, tl = g / side;
  const int64_t wave = (first_block + blockIdx.x) * (kThreads / 64) + (threadIdx.x >> 6);
  if (wave * tokens >= a.rows) return;  // q and k need not take the same number of waves
  const int64_t row = wave * tokens + tl;
  const bool live = row < a.rows;
  const unsigned r32 = (unsigned)(live ? row : a.rows - 1);
  const unsigned b = r32 / (unsigned)a.tokens, n = r32 - b * (unsigned)a.tokens;

  // (cos, sin) of the lane's 8 frequencies at a token of the video.
  float c[8], s[8];
  const int64_t v64 = (int64_t)n - a.offset;
  const bool turned = v64 >= 0 && v64 < a.video;
  if (turned) {
    const unsigned v = (unsigned)v64, wd = a.axis[2].length, ht = a.axis[1].length;
    const unsigned line = v / wd, x = v - line * wd, z = line / ht, y = line - z * ht;
    const int p0 = a.axis[0].pairs, p1 = p0 + a.axis[1].pairs;
    const float* t0 = a.axis[0].table + (int64_t)z * (2 * a.axis[0].pairs);
    const float* t1 = a.axis[1].table + ((int64_t)y * a.axis[1].pairs - p0) * 2;
    const float* t2 = a.axis[2].table + ((int64_t)x * a.axis[2].pairs - p1) * 2;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = HALVES ? 8 * u + e : (e < 4 ? 4 * u + e : D / 4 + 4 * u + e - 4);
      const float* q = i < p0 ? t0 : i < p1 ? t1 : t2;
      const float2 cs = *reinterpret_cast<const float2*>(q + 2 * i);
      c[e] = cs.x;
      s[e] = cs.y;
    }
  }

  float w[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    w[e] = 1.0f;
  }
  if (NORM == kRotaryRms || NORM == kRotaryLayer) {
    if (t.weight) load16<T>(t.weight, a.wide_weight, 8 * u, D / 2, w);
  }

  // In the last step a lane's head may be past the heads: it loads the last one and stores none.
  const int steps = (t.heads + side - 1) / side, left = t.heads - (steps - 1) * side;
  const int hl_last = min(hl, left - 1);
  const uint16_t* src = t.in + b * t.in_b + n * t.in_n + 8 * u;
  const uint16_t* src_last = src + hl_last * t.in_h;
  src += hl * t.in_h;
  uint16_t* dst = t.out + b * t.out_b + n * t.out_n + hl * t.out_h + 8 * u;
  const auto there = [&](int step) { return step < steps - 1 || hl < left; };
  u32x4 raw[kBatch][2];
  const auto fetch = [&](int first, auto past) {  // past: past the caches
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (first + j < steps) {
        const uint16_t* p = (first + j < steps - 1 ? src : src_last) +
                            (int64_t)(first + j) * side * t.in_h;
        raw[j][0] = load_words4<decltype(past)::value>(p);
        raw[j][1] = load_words4<decltype(past)::value>(p + D / 2);
      }
  };
  const std::bool_constant<STREAM && D == 128> past;
  const auto widen = [&](int j, float (&x)[16]) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[8 * k + 2 * e] = T::to_f((uint16_t)raw[j][k][e]);
        x[8 * k + 2 * e + 1] = T::to_f((uint16_t)(raw[j][k][e] >> 16));
      }
  };
  float all = 1.0f;
  if (NORM == kRotaryRmsAll) {
    // A lane's squares are added over a power of two no smaller than the heads, which changes no
    // bit of the mean but keeps the sum in range: up to 2^16 heads of values up to about 1e17.
    const float down = __uint_as_float((unsigned)(127 - (32 - __clz(t.heads - 1))) << 23);
    float sq = 0.0f;
    for (int first = 0; first < steps; first += kBatch) {
      if (steps > kBatch) {
        fetch(first, std::false_type());  // read again below, from the caches
      } else {
        fetch(first, past);
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (first + j < steps) {
          float x[16];
          widen(j, x);
          float part = 0.0f;
#pragma unroll
          for (int e = 0; e < 16; ++e) part = fmaf(x[e], x[e], part);
          sq = fmaf(there(first + j) ? part : 0.0f, down, sq);
        }
    }
    all = 1.0f / sqrtf(row_sum(sq, kLanes * side, nullptr) / ((float)(t.heads * D) * down) + a.eps);
  }
  for (int first = 0; first < steps; first += kBatch) {
    if (NORM != kRotaryRmsAll || steps > kBatch) fetch(first, past);
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (first + j >= steps) break;
      float x[16], y[16];
      widen(j, x);
      float inv = all;
      if (NORM == kRotaryLayer) {
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) sum += x[e];
        const float mean = row_sum(sum, kLanes, nullptr) * (1.0f / D);
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] -= mean;
      }
      if (NORM == kRotaryRms || NORM == kRotaryLayer) {
        float sq = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) sq = fmaf(x[e], x[e], sq);
        inv = 1.0f / sqrtf(row_sum(sq, kLanes, nullptr) * (1.0f / D) + a.eps);
      }
      // The head's place in the weights: those over a head's channels are the same for all.
      const unsigned at =
          8 * u + (NORM == kRotaryRmsAll
                       ? (unsigned)((first + j) * side + (there(first + j) ? hl : hl_last)) * D
                       : 0);
      if (NORM == kRotaryRmsAll && t.weight) load16<T>(t.weight, a.wide_weight, at, D / 2, w);
      if (NORM != kRotaryNone) {
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = x[e] * inv * w[e];
        if (t.bias) {
          float bias[16];
          load16<T>(t.bias, a.wide_weight, at, D / 2, bias);
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] += bias[e];
        }
      }
      // The others keep their values, also beside an infinity.
#pragma unroll
      for (int e = 0; e < 16; ++e) y[e] = x[e];
      if (turned) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int p = HALVES ? e : 2 * e, q = HALVES ? e + 8 : 2 * e + 1;
          y[p] = x[p] * c[e] - x[q] * s[e];
          y[q] = x[q] * c[e] + x[p] * s[e];
        }
      }
      u32x4 lo, hi;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        lo[e] = pack2<T>(y[2 * e], y[2 * e + 1]);
        hi[e] = pack2<T>(y[8 + 2 * e], y[8 + 2 * e + 1]);
      }
      if (live && there(first + j)) {
        uint16_t* o = dst + (int64_t)(first + j) * side * t.out_h;
        store_words4<STREAM>(o, lo);
        store_words4<STREAM>(o + D / 2, hi);
      }
    }
  }
}

template <class T, int D, bool HALVES, int NORM>
hipError_t launch(const RotaryArgs& a, hipStream_t s) {
  constexpr int kRows = 64 / (D / 16);
  RotaryArgs b = a;
  int64_t waves = 1, values = 0;  // rows of d
  for (int i = 0; i < a.tensors; ++i) {
    // Each tensor by its own heads, so that q's sums do not depend on k's.
    // Heads side by side read long pieces of a projection, steps in flight together keep a wave
    // busy: as many side by side as leave three steps and no more than an eighth of the lanes
    // without a head.  At 400 MB a call, us: 24 heads of 128 by 8 / by 4 65 / 70, 48 of 64 by
    // 16 / by 8 70 / 76, 15 of 64 by 16 / by 8 / by 4 / by 1 102 / 73 / 71 / 86.
    const int heads = a.x[i].heads;
    const auto steps = [&](int n) { return (heads + n - 1) / n; };
    int side = kRows;
    while (side > 1 && (steps(side) < 3 || steps(side) * side * 8 > heads * 9)) side /= 2;
    b.x[i].side = side;
    values += a.rows * a.x[i].heads;
    waves = std::max(waves, (a.rows + kRows / side - 1) / (kRows / side));
  }
  constexpr int kWaves = kThreads / 64;
  const int64_t blocks = (waves + kWaves - 1) / kWaves;
  // Past the caches from kStreamBytes on, loads (of heads of 128) and stores, though Q and K are
  // read next: what they would push out, V and the projections' other outputs, is read as well.
  // Three projections, this call, then recap_kv_pack and recap_pool_blocks in us, heads of 128,
  // stores through the caches -> past them: 101 MB a call 147.5 -> 150.9, 203 MB 279.1 -> 277.3,
  // 302 MB 431.0 -> 423.9, 403 MB 519.2 -> 514.0, 2,926 MB 6,170 -> 6,118; heads of 64, 331 MB
  // 722.8 -> 722.1, 1,109 MB 2,307 -> 2,290.  With the whole sparse call behind them the same way
  // or even (403 MB 1,987 -> 1,975).
  for (int64_t first = 0; first < blocks; first += kMaxBlocks) {
    const dim3 grid((unsigned)std::min(blocks - first, kMaxBlocks), a.tensors);
    if (4 * D * values >= kStreamBytes) {
      rotary_kernel<T, D, HALVES, NORM, true><<<grid, dim3(kThreads), 0, s>>>(b, first);
    } else {
      rotary_kernel<T, D, HALVES, NORM, false><<<grid, dim3(kThreads), 0, s>>>(b, first);
    }
  }
  return hipGetLastError();
}

template <class T, int D, bool HALVES>
hipError_t by_norm(const RotaryArgs& a, hipStream_t s) {
  switch (a.norm) {
    case kRotaryNone: return launch<T, D, HALVES, kRotaryNone>(a, s);
    case kRotaryRms: return launch<T, D, HALVES, kRotaryRms>(a, s);
    case kRotaryLayer: return launch<T, D, HALVES, kRotaryLayer>(a, s);
    default: return launch<T, D, HALVES, kRotaryRmsAll>(a, s);
  }
}

template <class T>
hipError_t by_shape(const RotaryArgs& a, int dim, hipStream_t s) {
  if (dim == 128) return a.halves ? by_norm<T, 128, true>(a, s) : by_norm<T, 128, false>(a, s);
  return a.halves ? by_norm<T, 64, true>(a, s) : by_norm<T, 64, false>(a, s);
}

}  // namespace

hipError_t run_rotary(const RotaryArgs& a, int dtype, int dim, hipStream_t s) {
  return dtype == BF16::code ? by_shape<BF16>(a, dim, s) : by_shape<F16>(a, dim, s);
}

}  // namespace recap

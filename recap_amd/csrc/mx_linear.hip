// Product of fp4 rows: out[m][n] = sum_k x[m][k] w[n][k] + bias[n], both operands in blocks of 32
// along k with power-of-two scales (microscale.hpp), on v_mfma_scale_f32_32x32x64_f8f6f4.
//
// One matrix instruction multiplies 32 rows by 32 rows over two blocks of each: lane l holds the 16
// bytes of row l % 32, block l / 32, and that block's scale byte, which the instruction applies to
// the block's sum.  Products of codes are exact; sums are fp32, the bias is added to the whole sum in
// fp32, and that is rounded to the output's type.  Weight rows are the A operand, so that a lane ends
// with consecutive outputs of one row of x.
//
// Bound by power, then by the copies: from registers the instruction reaches 6.5 PFLOP/s on random
// codes (10.0 on zeros); 8,192^3 takes 256 us on one card and 278 on another, 4.3 and 3.95 PFLOP/s, and
// on the latter 215 us, 5.1, without the copies into LDS.  118,800 x 2,048 to 8,192 outputs: 1,109-1,137
// us in a loop, 3.5-3.6 PFLOP/s, up to 1,260 among other calls.  (A library's bf16 product of 8,192^3:
// 1.2 PFLOP/s.)
#include <algorithm>
#include <type_traits>

#include "kernels.hpp"
#include "microscale.hpp"

namespace recap {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
constexpr int kFp4 = 4;          // operand format of the instruction
constexpr int kStepBytes = 128;  // 256 values of a row
constexpr int kStepScales = 8;

// acc += A B^T over one block pair; byte S of each scale word is the scale.
template <int S>
__device__ inline f32x16 mfma_fp4(u32x4 a, u32x4 b, f32x16 c, unsigned sa, unsigned sb) {
  const i32x8 x = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8 y = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(x, y, c, kFp4, kFp4, S, (int)sa, S, (int)sb);
}

// All of this wave's copies into LDS and LDS reads done, then every wave's.
__device__ inline void step_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x7 << 4);
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Copies 16 bytes a lane (4: copy_to_lds4) of a buffer of `bytes` bytes, from `at` (of the lane) +
// `offset` on, into LDS from `dst` on, lane after lane.
__device__ inline void copy_to_lds(const uint8_t* base, int bytes, char* dst, int at, int offset) {
  const __amdgpu_buffer_rsrc_t r =
      __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, bytes, kBufferRsrcWord3);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)dst, 16, at, offset, 0, 0);
}
__device__ inline void copy_to_lds4(const uint8_t* base, int bytes, char* dst, int at, int offset) {
  const __amdgpu_buffer_rsrc_t r =
      __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, bytes, kBufferRsrcWord3);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)dst, 4, at, offset, 0, 0);
}

__device__ inline float load_bias(const MxProductArgs& a, int n) {
  if (a.bias_dtype == F32::code) return load_elem<F32>(a.bias, n);
  return a.bias_dtype == BF16::code ? load_elem<BF16>(a.bias, n) : load_elem<F16>(a.bias, n);
}

// A workgroup computes BN outputs of BM rows, waves WN x WM of them.  PAST: stored past the caches.
template <class O, int BM, int BN, int WM, int WN, bool PAST>
__global__ __launch_bounds__(64 * WM * WN) void product_kernel(MxProductArgs a, int tiles_m,
                                                               int tiles_n) {
  constexpr int kThreads = 64 * WM * WN;
  constexpr int FM = BM / WM / 32, FN = BN / WN / 32;  // fragments of 32 rows a wave
  __shared__ __attribute__((aligned(16))) char x0[BM * kStepBytes];
  __shared__ __attribute__((aligned(16))) char x1[BM * kStepBytes];
  __shared__ __attribute__((aligned(16))) char w0[BN * kStepBytes];
  __shared__ __attribute__((aligned(16))) char w1[BN * kStepBytes];
  __shared__ __attribute__((aligned(16))) char s0[(BM + BN) * kStepScales];  // of x, then of w
  __shared__ __attribute__((aligned(16))) char s1[(BM + BN) * kStepScales];
  __shared__ __attribute__((aligned(16))) float bias[BN];

  const int t = threadIdx.x, lane = t & 63, g = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm = wave % WM, wn = wave / WM;
  // An XCD's workgroups take neighbouring tiles, kBand rows of tiles deep: those in flight on it read
  // few distinct rows of either operand, which its L2 holds.
  constexpr int kBand = 8;
  const int item = xcd_linear(blockIdx.x, tiles_m * tiles_n);
  const int band = item / (kBand * tiles_n), place = item - band * kBand * tiles_n;
  const int deep = min(kBand, tiles_m - band * kBand);
  const int tn = place / deep, tm = band * kBand + place - tn * deep;
  const int m0 = tm * BM, n0 = tn * BN;
  const int pitch = a.steps * kStepBytes, spitch = a.steps * kStepScales;

  // Copies into LDS go 16 bytes a lane (4 for scales) in lane order, 8 rows (32) an instruction.  A
  // row's 8 chunks are exchanged by row, so that the lanes of a fragment read distinct banks.  Rows
  // past the last are copies of it and not stored.
  constexpr int kWaves = kThreads / 64, CX = BM / 8 / kWaves, CW = BN / 8 / kWaves;
  static_assert(BM % (8 * kWaves) == 0 && BN % (8 * kWaves) == 0 && kWaves % 2 == 0, "tile");
  const int mrows = min(BM, a.rows - m0), nrows = min(BN, a.outputs - n0);
  const int first = 8 * wave + (lane >> 3), chunk = 16 * ((lane & 7) ^ TileGeom<64>::swz(first, 8));
  int x_at[CX], w_at[CW];
#pragma unroll
  for (int i = 0; i < CX; ++i) x_at[i] = min(first + 8 * kWaves * i, mrows - 1) * pitch + chunk;
#pragma unroll
  for (int i = 0; i < CW; ++i) w_at[i] = min(first + 8 * kWaves * i, nrows - 1) * pitch + chunk;
  const uint8_t* const xb = a.x + (int64_t)m0 * pitch;
  const uint8_t* const wb = a.w + (int64_t)n0 * pitch;
  const uint8_t* const xsb = a.x_scales + (int64_t)m0 * spitch;
  const uint8_t* const wsb = a.w_scales + (int64_t)n0 * spitch;
  const auto fetch = [&](char* x, char* w, char* scales, int step) {
#pragma unroll
    for (int i = 0; i < CX; ++i)
      copy_to_lds(xb, mrows * pitch, x + 1024 * (wave + kWaves * i), x_at[i], step * kStepBytes);
#pragma unroll
    for (int i = 0; i < CW; ++i)
      copy_to_lds(wb, nrows * pitch, w + 1024 * (wave + kWaves * i), w_at[i], step * kStepBytes);
#pragma unroll
    for (int i = 0; i < (BM + BN) / 32; i += kWaves) {
      const int at = i + wave;  // 32 rows of scales
      if (at < (BM + BN) / 32) {
        const bool of_x = at < BM / 32;
        const int rows = of_x ? mrows : nrows;
        const int row = min(32 * (of_x ? at : at - BM / 32) + (lane >> 1), rows - 1);
        copy_to_lds4(of_x ? xsb : wsb, rows * spitch, scales + 256 * at,
                     row * spitch + (lane & 1) * 4, step * kStepScales);
      }
    }
  };

  // The reduction goes block pair by block pair, four a step; the fragments of the next pair are read
  // from LDS while this one's are multiplied, over the barrier between two steps too.
  f32x16 acc[FN][FM];
  u32x4 fx[2][FM], fw[2][FN];
  unsigned sx[2][FM], sw[2][FN];
  const int row_x = wm * FM * 32 + l32, row_w = wn * FN * 32 + l32;
  const int swz = TileGeom<64>::swz(l32, 8);
  const auto read = [&](int set, const char* x, const char* w, int s) {
    const int at = ((4 * g + s) ^ swz) << 4;
#pragma unroll
    for (int j = 0; j < FN; ++j) fw[set][j] = lds_load16(w, (row_w + 32 * j) * kStepBytes + at);
#pragma unroll
    for (int i = 0; i < FM; ++i) fx[set][i] = lds_load16(x, (row_x + 32 * i) * kStepBytes + at);
  };
  const auto read_scales = [&](int set, const char* scales) {
    const auto word = [&](int row) {
      return *reinterpret_cast<const unsigned*>(scales + row * kStepScales + 4 * g);
    };
#pragma unroll
    for (int j = 0; j < FN; ++j) sw[set][j] = word(BM + row_w + 32 * j);
#pragma unroll
    for (int i = 0; i < FM; ++i) sx[set][i] = word(row_x + 32 * i);
  };
  const auto multiply = [&](auto s, int scales) {
    constexpr int S = decltype(s)::value;
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int i = 0; i < FM; ++i)
        acc[j][i] = mfma_fp4<S>(fw[S & 1][j], fx[S & 1][i], acc[j][i], sw[scales][j], sx[scales][i]);
  };
  // One step from the buffers (x, w), its first pair already read; then the next step's is.  The
  // scheduler would put a pair's reads behind the products they are to run beside.
  const auto advance = [&](char* x, char* w, char* scales, const char* next_x, const char* next_w,
                           const char* next_scales, int set, int step) {
    const auto pair = [&](auto s) {
      read(1 - (decltype(s)::value & 1), x, w, decltype(s)::value + 1);
      __builtin_amdgcn_sched_barrier(0);
      multiply(s, set);
      __builtin_amdgcn_sched_barrier(0);
    };
    pair(std::integral_constant<int, 0>());
    pair(std::integral_constant<int, 1>());
    pair(std::integral_constant<int, 2>());
    // Opaque: the compiler otherwise moves all products behind the branch below, their fragments
    // kept in registers until then.
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int i = 0; i < FM; ++i) asm volatile("" : "+v"(acc[j][i]));
    step_barrier();
    read_scales(1 - set, next_scales);
    read(0, next_x, next_w, 0);
    __builtin_amdgcn_sched_barrier(0);
    if (step + 2 < a.steps) fetch(x, w, scales, step + 2);
    __builtin_amdgcn_sched_barrier(0);
    multiply(std::integral_constant<int, 3>(), set);
    __builtin_amdgcn_sched_barrier(0);
  };

  // The bias is fetched behind the first step, which it would hold up, and added to the whole sums: one
  // rounding at its size, where sums that start from it would round at that size all along (us so -> now:
  // 118,800 x 2,048 to 8,192 1,128 -> 1,137, 4,600 x 2,048 to 2,048 18.2 -> 18.4).
  const auto fetch_bias = [&]() {
    for (int i = t; i < BN; i += kThreads)
      bias[i] = a.bias != nullptr && n0 + i < a.outputs ? load_bias(a, n0 + i) : 0.0f;
  };
  const auto start = [&]() {
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int i = 0; i < FM; ++i) acc[j][i] = f32x16{};
  };

  // An odd step comes first, through the second buffer: behind the loop its sums would need
  // registers of their own.
  const int odd = a.steps & 1;
  if (odd) {
    fetch(x1, w1, s1, 0);
    fetch_bias();
    step_barrier();
    start();
    if (a.steps > 1) fetch(x0, w0, s0, 1);
    read_scales(1, s1);
    read(0, x1, w1, 0);
    advance(x1, w1, s1, x0, w0, s0, 1, 0);
  } else {
    fetch(x0, w0, s0, 0);
    fetch_bias();
    step_barrier();
    start();
    fetch(x1, w1, s1, 1);
    read_scales(0, s0);
    read(0, x0, w0, 0);
  }
  for (int step = odd; step < a.steps; step += 2) {
    advance(x0, w0, s0, x1, w1, s1, 0, step);
    advance(x1, w1, s1, x0, w0, s0, 1, step + 1);
  }

  // Lane (g, l32) of fragment (j, i) holds outputs 8 q + 4 g .. + 3 of row l32: stored from there, a
  // line of memory would be written in eight parts.  The wave passes its part of the tile, 128 bytes
  // of every row at a time, through LDS of its own (its chunks exchanged by row as above), and stores
  // whole lines.
  constexpr int kSize = kBytes<O>, kFrags = 4 / kSize;  // fragments in 128 bytes
  static_assert(FN % kFrags == 0, "passes");
  constexpr int kRegion = FM * 32 * 128;
  constexpr int kInX = BM * kStepBytes / kRegion, kInW = BN * kStepBytes / kRegion;
  static_assert(2 * (kInX + kInW) >= kWaves, "room");
  char* const region = wave < kInX            ? x0 + wave * kRegion
                       : wave < 2 * kInX      ? x1 + (wave - kInX) * kRegion
                       : wave < 2 * kInX + kInW ? w0 + (wave - 2 * kInX) * kRegion
                                              : w1 + (wave - 2 * kInX - kInW) * kRegion;
#pragma unroll
  for (int pass = 0; pass < FN / kFrags; ++pass) {
    f32x4 b[kFrags][4];  // before the first write, which the compiler does not move reads over
#pragma unroll
    for (int f = 0; f < kFrags; ++f)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        b[f][q] =
            *reinterpret_cast<const f32x4*>(bias + (wn * FN + pass * kFrags + f) * 32 + 8 * q + 4 * g);
#pragma unroll
    for (int f = 0; f < kFrags; ++f)
#pragma unroll
      for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int i = 0; i < FM; ++i) {
          const f32x16& s = acc[pass * kFrags + f][i];
          f32x4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = s[4 * q + e] + b[f][q][e];
          const int row = 32 * i + l32;
          if constexpr (kSize == 2) {
            const int at = row * 128 + (((4 * f + q) ^ swz) << 4) + 8 * g;
            *reinterpret_cast<u32x2*>(region + at) =
                u32x2{pack2<O>(v[0], v[1]), pack2<O>(v[2], v[3])};
          } else {
            const int at = row * 128 + (((2 * q + g) ^ swz) << 4);
            *reinterpret_cast<f32x4*>(region + at) = v;
          }
        }
    asm volatile("" ::: "memory");
    const int n = n0 + (wn * FN + pass * kFrags) * 32 + (lane & 7) * (16 / kSize);
#pragma unroll
    for (int r = 0; r < FM * 32; r += 8) {
      const int row = r + (lane >> 3), m = m0 + wm * FM * 32 + row;
      const u32x4 v = lds_load16(region, row * 128 + (((lane & 7) ^ TileGeom<64>::swz(row, 8)) << 4));
      if (m >= a.rows || n >= a.outputs) continue;
      const int64_t to = m * a.stride + n;
      if (n + 16 / kSize <= a.outputs) {
        store_words4<PAST>(const_cast<void*>(row_of<O>(a.out, to)), v);
      } else {
#pragma unroll
        for (int e = 0; e < 16 / kSize; ++e)
          if (n + e < a.outputs) {
            if constexpr (kSize == 2) {
              static_cast<uint16_t*>(a.out)[to + e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
            } else {
              static_cast<unsigned*>(a.out)[to + e] = v[e];
            }
          }
      }
    }
    asm volatile("" ::: "memory");
  }
}

// ---------------------------------------------------------------------------------------
// A few rows of x (a token, a timestep): the weight is read once, straight into registers, and
// that is what takes the time.  A workgroup computes 32 outputs of every row; its waves take the
// steps of the sum in turn, and their parts are added in that order.  x is brought into LDS by every
// workgroup, as codes or, of few values, from the values themselves (X not Codes), which saves the
// launch that would make its codes.
constexpr int kFewRows = 16, kFewWaves = 8, kFewThreads = 64 * kFewWaves;
constexpr int kBatch = 4;        // steps a wave requests before it uses the first
constexpr int kPartPitch = 36;   // floats of a row of a wave's part
constexpr int kFewLds = 64 * 1024;
__host__ __device__ constexpr int few_code_pitch(int steps) { return steps * kStepBytes + 16; }
__host__ __device__ constexpr int few_scale_pitch(int steps) { return steps * kStepScales + 4; }
__host__ __device__ constexpr int64_t few_bytes(int64_t rows, int64_t steps) {
  return rows * (few_code_pitch((int)steps) + few_scale_pitch((int)steps));
}

struct Codes {};

template <class O, class X>
__global__ __launch_bounds__(kFewThreads) void few_rows_kernel(MxProductArgs a, const void* values,
                                                               int64_t value_stride, int width) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int t = threadIdx.x, lane = t & 63, g = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int n0 = blockIdx.x * 32, n = min(n0 + l32, a.outputs - 1);
  const uint8_t* wrow = a.w + (int64_t)n * a.steps * kStepBytes + 64 * g;
  const uint8_t* wscale = a.w_scales + (int64_t)n * a.steps * kStepScales + 4 * g;
  u32x4 fw[kBatch][4];
  unsigned sw[kBatch];
  const auto request = [&](int first) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int step = first + kFewWaves * i;
      if (step >= a.steps) continue;
#pragma unroll
      for (int s = 0; s < 4; ++s)
        fw[i][s] = *reinterpret_cast<const u32x4*>(wrow + step * kStepBytes + 16 * s);
      sw[i] = *reinterpret_cast<const unsigned*>(wscale + step * kStepScales);
    }
  };
  request(wave);

  const int pitch = few_code_pitch(a.steps), spitch = few_scale_pitch(a.steps);
  char* const scales = lds + a.rows * pitch;
  const unsigned words = (unsigned)a.steps * (kStepBytes / 4);  // 8 values each
  for (unsigned c = t; c < a.rows * words; c += kFewThreads) {
    const unsigned row = c / words, word = c - row * words;
    unsigned code, scale = 0;
    if constexpr (std::is_same_v<X, Codes>) {
      code = reinterpret_cast<const unsigned*>(a.x)[c];
      if ((word & 3) == 0) scale = a.x_scales[c >> 2];
    } else {
      const int at = 8 * word, left = width - at;
      const int64_t from = row * value_stride + at;
      float v[8];
      if (left >= 8) {
        load_chunk<X>(row_of<X>(values, from), 0, v);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < left ? load_elem<X>(values, from + e) : 0.0f;
      }
      scale = mx_scale<kMxFp4>(quad_max(magnitude_bits(v)));
      code = mx_fp4_codes(v, scale);
    }
    *reinterpret_cast<unsigned*>(lds + row * pitch + 4 * word) = code;
    if ((word & 3) == 0) scales[row * spitch + (word >> 2)] = (char)scale;
  }
  __syncthreads();

  f32x16 acc = {};
  const char* xrow = lds + min(l32, a.rows - 1) * pitch + 64 * g;
  const char* xscale = scales + min(l32, a.rows - 1) * spitch + 4 * g;
  for (int first = wave; first < a.steps; first += kFewWaves * kBatch) {
    if (first != wave) request(first);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int step = first + kFewWaves * i;
      if (step >= a.steps) continue;
      const unsigned sx = *reinterpret_cast<const unsigned*>(xscale + step * kStepScales);
      const auto pair = [&](auto s) {
        constexpr int S = decltype(s)::value;
        acc = mfma_fp4<S>(fw[i][S], lds_load16(xrow, step * kStepBytes + 16 * S), acc, sw[i], sx);
      };
      pair(std::integral_constant<int, 0>());
      pair(std::integral_constant<int, 1>());
      pair(std::integral_constant<int, 2>());
      pair(std::integral_constant<int, 3>());
    }
  }
  __syncthreads();  // x is read: its room takes the waves' parts

  float* const part = reinterpret_cast<float*>(lds);
  if (l32 < a.rows)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      *reinterpret_cast<f32x4*>(part + (wave * kFewRows + l32) * kPartPitch + 8 * q + 4 * g) =
          f32x4{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
  __syncthreads();
  const int m = t >> 3, at = n0 + 4 * (t & 7);
  if (m >= a.rows || at >= a.outputs) return;
  f32x4 sum = {};
  for (int w = 0; w < min(kFewWaves, a.steps); ++w) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(part + (w * kFewRows + m) * kPartPitch + 4 * (t & 7));
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += v[e];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (at + e < a.outputs)
      store_elem<O>(a.out, m * a.stride + at + e,
                    sum[e] + (a.bias != nullptr ? load_bias(a, at + e) : 0.0f));
}

template <class O, class X>
hipError_t launch_few(const MxProductArgs& a, const void* values, int64_t value_stride, int width,
                      hipStream_t s) {
  const int64_t bytes = std::max<int64_t>(few_bytes(a.rows, a.steps),
                                          kFewWaves * kFewRows * kPartPitch * 4);
  few_rows_kernel<O, X><<<dim3((unsigned)((a.outputs + 31) / 32)), dim3(kFewThreads), (size_t)bytes,
                          s>>>(a, values, value_stride, width);
  return hipGetLastError();
}

// Where that beats tiles of 64; us, few rows / tiles, the launch that makes the codes of x with both where
// it is needed.  Values: 1 row x 1,536 to 9,216 outputs 5.1 / 8.6, 8 rows 6.6 / 8.7; 1 x 8,192 to 8,192
// 10.7 / 29.6; 8 x 8,192 to 2,048 14.2 / 21.5; 16 x 4,096 to 2,048 11.6 / 13.8.  More than 65,536 values,
// which have that launch here too: 8 x 14,336 to 2,048 27.7 / 33.4, 10 x 8,192 20.3 / 21.6, but 12 x 8,192
// 22.8 / 21.7 and 16 x 5,120 18.4 / 15.3.  8 x 2,048 to 20,000 11.3 / 10.8: x is brought into LDS too
// often.  Codes go the way of values, so that both have the same sums: 1 x 8,192 to 8,192 13.8 / 29.6,
// 8 x 8,192 to 2,048 18.5 / 21.5, 8 x 1,536 to 9,216 8.7 / 8.7, 8 x 256 to 1,024 5.8 / 5.6, 16 x 4,096 to
// 2,048 15.9 / 13.8; 16 x 1,536 to 1,536, 9.2 / 8.3 (values 5.7 / 8.4), is left to the tiles.
bool few(const MxProductArgs& a) {
  const int most = a.steps < 16 ? 8 : a.steps * kFewRows <= 256 ? kFewRows : std::max(10, 256 / a.steps);
  return a.rows <= most && a.outputs <= 320 * 32 && few_bytes(a.rows, a.steps) <= kFewLds;
}

template <class O, int BM, int BN, int WM, int WN, bool PAST = false>
hipError_t launch(const MxProductArgs& a, hipStream_t s) {
  const int64_t tiles_m = (a.rows + BM - 1) / BM, tiles_n = (a.outputs + BN - 1) / BN;
  product_kernel<O, BM, BN, WM, WN, PAST><<<dim3((unsigned)(tiles_m * tiles_n)), dim3(64 * WM * WN), 0, s>>>(
      a, (int)tiles_m, (int)tiles_n);
  return hipGetLastError();
}

// The largest tile whose rounds over the 256 CUs are worth its size.  A tile of 256 x 256 takes as
// long as 2.9 of 128 x 128 (two of which a CU holds at once) where it would take four by its work;
// us at 8 steps, rows x outputs, 256 / 128 / 64 wide: 118,800 x 8,192 1,174 / 1,419 / -;
// 4,600 x 2,048 (144 tiles of 256) 18.9 / 20.7 / 26.9; 19,200 x 1,024 (300) 35.3 / 31.3 / 46.8;
// 3,000 x 2,048 (96) 17.1 / 13.4 / 18.5; 1,500 x 2,048 15.7 / 8.6 / 9.7; 256 x 2,048
// 15.0 / 7.6 / 6.6; 512 x 2,048 at 32 steps 47.4 / 29.5 / 20.8.
template <class O>
hipError_t launch_type(const MxProductArgs& a, hipStream_t s) {
  if (few(a)) return launch_few<O, Codes>(a, nullptr, 0, 0, s);
  const auto tiles = [&](int64_t side) {
    return ((a.rows + side - 1) / side) * ((a.outputs + side - 1) / side);
  };
  const auto rounds = [&](int64_t side) { return (double)((tiles(side) + 255) / 256); };
  if (a.rows <= 64 || a.outputs <= 64 || tiles(64) <= 512) return launch<O, 64, 64, 2, 1>(a, s);
  if (2.9 * rounds(256) < rounds(128) + 0.4) {
    // Outputs that cannot stay in the caches, in whole lines, go past them and leave them to the
    // operands, us through -> past: 118,800 x 8,192 outputs 1,167 -> 1,116, x 2,048 329 -> 292,
    // 60,000 x 2,048 171 -> 153; but 32,760 x 1,536 49.4 -> 50.4, and rows of 999 18.5 -> 32.
    const bool past = a.rows * (int64_t)a.outputs * kBytes<O> >= kStreamBytes &&
                      (reinterpret_cast<uintptr_t>(a.out) | a.stride * kBytes<O>) % 128 == 0;
    return past ? launch<O, 256, 256, 4, 2, true>(a, s) : launch<O, 256, 256, 4, 2>(a, s);
  }
  return launch<O, 128, 128, 4, 2>(a, s);
}

}  // namespace

hipError_t run_mx_product(const MxProductArgs& a, int dtype, hipStream_t s) {
  if (dtype == F32::code) return launch_type<F32>(a, s);
  return dtype == BF16::code ? launch_type<BF16>(a, s) : launch_type<F16>(a, s);
}

// Every workgroup makes the codes of x anew, which for up to 16 chunks of 8 values a thread saves the
// launch that would (2 x 1,536 to 9,216, a call among others: 13.1 -> 10.6 us).
bool mx_product_takes_values(const MxProductArgs& a, int64_t width) {
  return few(a) && a.rows * width <= 16 * 8 * kFewThreads;
}

template <class O>
static hipError_t few_values(const MxProductArgs& a, const void* x, int x_dtype, int64_t stride,
                             int width, hipStream_t s) {
  if (x_dtype == F32::code) return launch_few<O, F32>(a, x, stride, width, s);
  return x_dtype == BF16::code ? launch_few<O, BF16>(a, x, stride, width, s)
                               : launch_few<O, F16>(a, x, stride, width, s);
}

hipError_t run_mx_product_values(const MxProductArgs& a, int dtype, const void* x, int x_dtype,
                                 int64_t stride, int64_t width, hipStream_t s) {
  if (dtype == F32::code) return few_values<F32>(a, x, x_dtype, stride, (int)width, s);
  return dtype == BF16::code ? few_values<BF16>(a, x, x_dtype, stride, (int)width, s)
                             : few_values<F16>(a, x, x_dtype, stride, (int)width, s);
}

}  // namespace recap

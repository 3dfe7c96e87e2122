// Product of fp4 rows: out[m][n] = sum_k x[m][k] w[n][k] + bias[n], both operands in blocks of 32
// along k with power-of-two scales (microscale.hpp), on v_mfma_scale_f32_32x32x64_f8f6f4.
//
// One matrix instruction multiplies 32 rows by 32 rows over two blocks of each: lane l holds the 16
// bytes of row l % 32, block l / 32, and that block's scale byte, which the instruction applies to
// the block's sum.  Products of codes are exact; sums are fp32 and rounded once, after the bias.
// Weight rows are the A operand, so that a lane ends with consecutive outputs of one row of x.
#include <algorithm>

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

__device__ inline float load_bias(const MxProductArgs& a, int n) {
  if (a.bias_dtype == F32::code) return load_elem<F32>(a.bias, n);
  return a.bias_dtype == BF16::code ? load_elem<BF16>(a.bias, n) : load_elem<F16>(a.bias, n);
}

// A workgroup computes BN outputs of BM rows, waves WN x WM of them.
template <class O, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void product_kernel(MxProductArgs a, int tiles_m,
                                                               int tiles_n) {
  constexpr int kThreads = 64 * WM * WN;
  constexpr int FM = BM / WM / 32, FN = BN / WN / 32;  // fragments of 32 rows a wave
  __shared__ __attribute__((aligned(16))) char x0[BM * kStepBytes];
  __shared__ __attribute__((aligned(16))) char x1[BM * kStepBytes];
  __shared__ __attribute__((aligned(16))) char w0[BN * kStepBytes];
  __shared__ __attribute__((aligned(16))) char w1[BN * kStepBytes];
  __shared__ __attribute__((aligned(16))) char xs0[BM * kStepScales];
  __shared__ __attribute__((aligned(16))) char xs1[BM * kStepScales];
  __shared__ __attribute__((aligned(16))) char ws0[BN * kStepScales];
  __shared__ __attribute__((aligned(16))) char ws1[BN * kStepScales];

  const int t = threadIdx.x, lane = t & 63, g = lane >> 5, l32 = lane & 31;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm = wave % WM, wn = wave / WM;
  const int item = xcd_linear(blockIdx.x, tiles_m * tiles_n);
  const int tn = item % tiles_n, tm = item / tiles_n;
  const int m0 = tm * BM, n0 = tn * BN;
  const int pitch = a.steps * kStepBytes, spitch = a.steps * kStepScales;

  // Copies into LDS go 16 bytes a lane (4 for scales) in lane order; rows are 8 chunks whose order
  // is exchanged by row, so that the lanes of a fragment read distinct banks.
  const auto resource = [](const uint8_t* base, int64_t row, int rows, int pitch) {
    return __builtin_amdgcn_make_buffer_rsrc((void*)(base + row * pitch), 0, rows * pitch,
                                             kBufferRsrcWord3);
  };
  const int mrows = min(BM, a.rows - m0), nrows = min(BN, a.outputs - n0);
  const __amdgpu_buffer_rsrc_t xr = resource(a.x, m0, mrows, pitch);
  const __amdgpu_buffer_rsrc_t wr = resource(a.w, n0, nrows, pitch);
  const __amdgpu_buffer_rsrc_t xsr = resource(a.x_scales, m0, mrows, spitch);
  const __amdgpu_buffer_rsrc_t wsr = resource(a.w_scales, n0, nrows, spitch);

  const auto copy = [&](const __amdgpu_buffer_rsrc_t& r, char* dst, int rows, int live, int step) {
    for (int i = wave; i < rows / 8; i += kThreads / 64) {
      const int row = 8 * i + (lane >> 3);
      const int chunk = (lane & 7) ^ TileGeom<64>::swz(row, 8);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(dst + i * 1024), 16,
                                               min(row, live - 1) * pitch + chunk * 16,
                                               step * kStepBytes, 0, 0);
    }
  };
  const auto copy_scales = [&](const __amdgpu_buffer_rsrc_t& r, char* dst, int rows, int live,
                               int step) {
    for (int i = wave; i < rows / 32; i += kThreads / 64) {
      const int row = 32 * i + (lane >> 1);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_void*)(dst + i * 256), 4,
                                               min(row, live - 1) * spitch + (lane & 1) * 4,
                                               step * kStepScales, 0, 0);
    }
  };

  f32x16 acc[FN][FM] = {};
  const auto multiply = [&](const char* x, const char* w, const char* xs, const char* ws) {
    unsigned sx[FM], sw[FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
      sx[i] = *reinterpret_cast<const unsigned*>(xs + ((wm * FM + i) * 32 + l32) * kStepScales + 4 * g);
#pragma unroll
    for (int j = 0; j < FN; ++j)
      sw[j] = *reinterpret_cast<const unsigned*>(ws + ((wn * FN + j) * 32 + l32) * kStepScales + 4 * g);
    const auto fragment = [&](const char* base, int first, int s) {
      const int row = first + l32;
      return lds_load16(base, row * kStepBytes + (((4 * g + s) ^ TileGeom<64>::swz(row, 8)) << 4));
    };
    const auto block = [&](auto s) {
      constexpr int S = decltype(s)::value;
      u32x4 fx[FM], fw[FN];
#pragma unroll
      for (int j = 0; j < FN; ++j) fw[j] = fragment(w, (wn * FN + j) * 32, S);
#pragma unroll
      for (int i = 0; i < FM; ++i) fx[i] = fragment(x, (wm * FM + i) * 32, S);
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int i = 0; i < FM; ++i) acc[j][i] = mfma_fp4<S>(fw[j], fx[i], acc[j][i], sw[j], sx[i]);
    };
    block(std::integral_constant<int, 0>());
    block(std::integral_constant<int, 1>());
    block(std::integral_constant<int, 2>());
    block(std::integral_constant<int, 3>());
  };
  const auto fetch0 = [&](int step) {
    copy(xr, x0, BM, mrows, step);
    copy(wr, w0, BN, nrows, step);
    copy_scales(xsr, xs0, BM, mrows, step);
    copy_scales(wsr, ws0, BN, nrows, step);
  };
  const auto fetch1 = [&](int step) {
    copy(xr, x1, BM, mrows, step);
    copy(wr, w1, BN, nrows, step);
    copy_scales(xsr, xs1, BM, mrows, step);
    copy_scales(wsr, ws1, BN, nrows, step);
  };

  fetch0(0);
  for (int step = 0; step < a.steps; step += 2) {
    step_barrier();
    if (step + 1 < a.steps) fetch1(step + 1);
    multiply(x0, w0, xs0, ws0);
    if (step + 1 >= a.steps) break;
    step_barrier();
    if (step + 2 < a.steps) fetch0(step + 2);
    multiply(x1, w1, xs1, ws1);
  }

  // Lane (g, l32) of fragment (j, i) holds outputs 8 q + 4 g .. + 3 of row l32.
#pragma unroll
  for (int j = 0; j < FN; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int n = n0 + (wn * FN + j) * 32 + 8 * q + 4 * g;
      float b[4] = {};
      if (a.bias != nullptr)
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = n + e < a.outputs ? load_bias(a, n + e) : 0.0f;
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int m = m0 + (wm * FM + i) * 32 + l32;
        if (m >= a.rows) continue;
        const int64_t to = m * a.stride + n;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[j][i][4 * q + e] + b[e];
        if (n + 4 <= a.outputs) {
          Rounded<O, 4> r;
          r.set(v);
          r.template store<false>(const_cast<void*>(row_of<O>(a.out, to)), 0, 0);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < a.outputs) store_elem<O>(a.out, to + e, v[e]);
        }
      }
    }
}

template <class O, int BM, int BN, int WM, int WN>
hipError_t launch(const MxProductArgs& a, hipStream_t s) {
  const int64_t tiles_m = (a.rows + BM - 1) / BM, tiles_n = (a.outputs + BN - 1) / BN;
  product_kernel<O, BM, BN, WM, WN><<<dim3((unsigned)(tiles_m * tiles_n)), dim3(64 * WM * WN), 0, s>>>(
      a, (int)tiles_m, (int)tiles_n);
  return hipGetLastError();
}

template <class O>
hipError_t launch_type(const MxProductArgs& a, hipStream_t s) {
  return launch<O, 128, 128, 2, 2>(a, s);
}

}  // namespace

hipError_t run_mx_product(const MxProductArgs& a, int dtype, hipStream_t s) {
  if (dtype == F32::code) return launch_type<F32>(a, s);
  return dtype == BF16::code ? launch_type<BF16>(a, s) : launch_type<F16>(a, s);
}

}  // namespace recap

// Stage 4 at a refresh: capture the refinement of the tail (recap/kernels/detail_cache.py:
// 64-186, 304-379).  For video rows r < R, with the dense output / LSE read at the native
// row rowmap[r] (= video_offset + permutation[r]):
//   ratio = min(exp(min(lh - lf, 0)), 1 - 1e-6)
//   D     = clamp((of - ratio oh) / (1 - ratio) - go, +-6e4), 0 where ratio > 1 - 1e-3
//   DL    = clamp(lf + ln(1 - ratio) - gl, +-30)
// With a previous refinement it first rebuilds the sparse output that refinement gives
// (drift weight included) and accumulates sum (old - of)^2 and sum of^2.  The reference
// adds them with float atomics; here each workgroup writes a partial pair and sum_pairs
// adds them in a fixed order.  Elementwise, HBM-bound, 16-byte accesses.
//
// The refinement is kept as fp16 or as int8 with a scale for every 32 channels (microscale.hpp): the
// four lanes that hold a block take its largest magnitude and D is rounded once, from fp32, to its
// codes.  There 1 - ratio is -expm1(lh - lf), D = (of - oh) / (1 - ratio) + oh - go and DL =
// (lf - gl) + ln(1 - ratio), which keep the digits that the difference of two near values in fp32
// loses (a row whose head holds all but 4e-4 of the mass: DL 1.5e-4 off against 1e-7).
#include <mutex>

#include "kernels.hpp"
#include "microscale.hpp"

namespace recap {

// Rows of a thread, all of whose loads are sent out first.  At 24 heads x 118,800 x 128 the int8
// capture takes 516 us with one row through the caches, 489 past them and 447 with two (5.8 TB/s).
// It goes past the caches at every size.  us past / through them, alone in a loop, and between the three
// writes of its inputs and a reading back of the bank: 4 MB in all 3.7 / 3.7 and 13.5 / 13.1, 63 MB
// 14.1 / 15.7 and 42.7 / 42.2, 127 MB 25.7 / 26.0 and 78 / 85, 335 MB 63 / 67 and 200 / 210, 2.4 GB
// 447 / 476 and 1,440 / 1,508.
template <bool MX>
constexpr int kRowsEach = MX ? 2 : 1;

template <class T, int D, bool MX>
__global__ __launch_bounds__(256) void capture_kernel(CaptureArgs a) {
  constexpr int TPR = D / 8, RPB = 256 / TPR, ROWS = kRowsEach<MX>;
  __shared__ float red[ROWS][2][4];
  const int blocks = a.rows / (ROWS * RPB);
  const int bank = blockIdx.x / blocks, blk = blockIdx.x % blocks;
  const int b = bank / a.heads, h = bank % a.heads;
  const int t = threadIdx.x, c = t % TPR;
  int64_t ri[ROWS];
  float lf[ROWS], lh[ROWS], glv[ROWS];
  u32x4 ofw[ROWS], ohw[ROWS], gow[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int r = (blk * ROWS + i) * RPB + t / TPR;
    const int nat = a.rowmap[r];
    ri[i] = (int64_t)bank * a.rows + r;
    lf[i] = a.lf[(int64_t)bank * a.n_tokens + nat];
    lh[i] = a.lh[(int64_t)bank * a.n_tokens + r];
    glv[i] = a.gl[ri[i]];
    ofw[i] = load_words4<MX>(a.of + b * a.osB + h * a.osH + (int64_t)nat * a.osN + 8 * c);
    ohw[i] = load_words4<MX>(a.oh + ((int64_t)bank * a.n_tokens + r) * D + 8 * c);
    gow[i] = load_words4<MX>(a.go + ri[i] * D + 8 * c);
  }
  const bool validate = a.glref != nullptr;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    float ratio = expf(fminf(lh[i] - lf[i], 0.0f));
    ratio = fminf(ratio, 1.0f - 1.0e-6f);
    const float den = MX ? fmaxf(-expm1f(lh[i] - lf[i]), 1.0e-6f) : 1.0f - ratio;
    float of[8], oh[8], go[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int sh = (e & 1) * 16;
      of[e] = T::to_f((uint16_t)(ofw[i][e >> 1] >> sh));
      oh[e] = T::to_f((uint16_t)(ohw[i][e >> 1] >> sh));
      go[e] = T::to_f((uint16_t)(gow[i][e >> 1] >> sh));
    }

    if (validate) {
      float before[8];
      if constexpr (MX) {
        mx_int8_values(static_cast<const u32x2*>(a.det)[ri[i] * TPR + c],
                       a.det_scale[(ri[i] * TPR + c) >> 2], before);
      } else {
        load_chunk<F16>(static_cast<const uint16_t*>(a.det) + ri[i] * D, 8 * c, before);
      }
      const float old_dl = a.dl[ri[i]];
      const float admit = expf(-fabsf(glv[i] - a.glref[ri[i]] - a.center[bank]));
      const float cl = glv[i] + old_dl;
      const float tc = fmaxf(glv[i], cl);
      const float sm = (1.0f - admit) * expf(glv[i] - tc);
      const float cm = admit * expf(cl - tc);
      const float tden = fmaxf(sm + cm, 1.0e-30f);
      const float tl = tc + logf(tden);
      const float common = fmaxf(lh[i], tl);
      const float wh = expf(lh[i] - common), wt = expf(tl - common);
      const float mden = fmaxf(wh + wt, 1.0e-30f);
      float err2 = 0.0f, ref2 = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float to = (go[e] * sm + (go[e] + before[e]) * cm) / tden;
        const float old = (oh[e] * wh + to * wt) / mden;
        err2 += (old - of[e]) * (old - of[e]);
        ref2 += of[e] * of[e];
      }
      err2 = wave_sum(err2);
      ref2 = wave_sum(ref2);
      if ((t & 63) == 0) {
        red[i][0][t >> 6] = err2;
        red[i][1][t >> 6] = ref2;
      }
      __syncthreads();  // every old value of these rows is read before any write
    }

    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float tail = MX ? (of[e] - oh[e]) / den + oh[e] : (of[e] - ratio * oh[e]) / den;
      const float cached = fmaxf(fminf(tail - go[e], 6.0e4f), -6.0e4f);
      v[e] = ratio > 1.0f - 1.0e-3f ? 0.0f : cached;
    }
    if constexpr (MX) {
      const unsigned s = mx_scale<kMxInt8>(quad_max(magnitude_bits(v)));
      store_words2<true>(static_cast<u32x2*>(a.det) + ri[i] * TPR + c, mx_int8_codes(v, s));
      if ((c & 3) == 0) a.det_scale[(ri[i] * TPR + c) >> 2] = (uint8_t)s;
    } else {
      Rounded<F16, 8> r;
      r.set(v);
      r.template store<false>(static_cast<uint16_t*>(a.det) + ri[i] * D, 8 * c, 0);
    }
    const float mass = MX ? (lf[i] - glv[i]) + logf(den) : lf[i] + logf(den) - glv[i];
    if (c == 0) a.dl[ri[i]] = fmaxf(fminf(mass, 30.0f), -30.0f);

    if (validate && t == 0) {
      float* out = a.stat_part + 2 * ((int64_t)blockIdx.x * ROWS + i);
      out[0] = ((red[i][0][0] + red[i][0][1]) + red[i][0][2]) + red[i][0][3];
      out[1] = ((red[i][1][0] + red[i][1][1]) + red[i][1][2]) + red[i][1][3];
    }
  }
}

template <class T, int D, bool MX>
static hipError_t launch_rows(const CaptureArgs& a, hipStream_t s) {
  const int per_block = kRowsEach<MX> * 256 / (D / 8);  // divides the 128 rows of a block
  capture_kernel<T, D, MX><<<dim3((unsigned)(a.banks * (a.rows / per_block))), dim3(256), 0, s>>>(a);
  return hipGetLastError();
}

template <class T, int D>
static hipError_t launch_capture(const CaptureArgs& a, int* blocks_per_bank, hipStream_t s) {
  *blocks_per_bank = a.rows / (256 / (D / 8));  // partial pairs
  return a.det_scale != nullptr ? launch_rows<T, D, true>(a, s) : launch_rows<T, D, false>(a, s);
}

hipError_t run_capture(const CaptureArgs& a, int dtype, int dim, int* blocks_per_bank, hipStream_t s) {
  if (dtype == BF16::code)
    return dim == 128 ? launch_capture<BF16, 128>(a, blocks_per_bank, s) : launch_capture<BF16, 64>(a, blocks_per_bank, s);
  return dim == 128 ? launch_capture<F16, 128>(a, blocks_per_bank, s) : launch_capture<F16, 64>(a, blocks_per_bank, s);
}

// ---------------------------------------------------------------------------------------
// Static scratch of the allocation-free capture (recap_refresh_capture_noalloc): the
// per-workgroup validation pairs live in this file-scope device array instead of a caller
// workspace.  Each GPU holds its own copy until the process ends; its address on a device
// is looked up once, with that device current, and kept per device.  In host code the
// array's name is only a host-side stand-in, so kernels and copies get the looked-up
// address, never the name.
__device__ __align__(256) float capture_scratch[2 * kCaptureScratchPairs];

namespace {
constexpr int kMaxDevices = 64;
std::mutex g_scratch_lock;
float* g_scratch_ptr[kMaxDevices] = {};
}  // namespace

hipError_t capture_scratch_pointer(float** out) {
  int device = -1;
  hipError_t e = hipGetDevice(&device);
  if (e != hipSuccess) return e;
  if (device < 0 || device >= kMaxDevices) return hipErrorInvalidDevice;
  std::lock_guard<std::mutex> guard(g_scratch_lock);
  if (g_scratch_ptr[device] == nullptr) {
    void* ptr = nullptr;
    e = hipGetSymbolAddress(&ptr, HIP_SYMBOL(capture_scratch));
    if (e != hipSuccess) return e;
    g_scratch_ptr[device] = static_cast<float*>(ptr);
  }
  *out = g_scratch_ptr[device];
  return hipSuccess;
}

// out2 = fixed-order sums of n (a, b) pairs: thread t adds pairs t, t + 1024, t + 2048, ...
// in turn (coalesced loads), then a fixed tree over the threads.
constexpr int kSumThreads = 1024;

__global__ __launch_bounds__(kSumThreads) void sum_pairs_kernel(const float* part, int n, float* out2) {
  __shared__ float ra[kSumThreads], rb[kSumThreads];
  const int t = threadIdx.x;
  const f32x2* pairs = reinterpret_cast<const f32x2*>(part);
  float sa = 0.0f, sb = 0.0f;
#pragma unroll 8
  for (int i = t; i < n; i += kSumThreads) {
    const f32x2 v = pairs[i];
    sa += v[0];
    sb += v[1];
  }
  ra[t] = sa;
  rb[t] = sb;
  __syncthreads();
  for (int h = kSumThreads / 2; h >= 1; h >>= 1) {
    if (t < h) { ra[t] += ra[t + h]; rb[t] += rb[t + h]; }
    __syncthreads();
  }
  if (t == 0) { out2[0] = ra[0]; out2[1] = rb[0]; }
}

hipError_t run_sum_pairs(const float* part, int n, float* out2, hipStream_t s) {
  hipLaunchKernelGGL(sum_pairs_kernel, dim3(1), dim3(kSumThreads), 0, s, part, n, out2);
  return hipGetLastError();
}

}  // namespace recap

// Element and 8-element chunk accesses at any alignment, and sums over the lanes that share a
// row, for the kernels that hold rows in registers (residual.hip, rotary.hip).
#pragma once

#include "common.hpp"

namespace recap {

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

typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef f32x4 f32x4_any __attribute__((aligned(4)));

template <class T>
__device__ inline void load8(const void* p, int64_t i, float (&v)[8]) {
  if constexpr (T::code == 3) {
    const f32x4_any* q = reinterpret_cast<const f32x4_any*>(static_cast<const float*>(p) + i);
    const f32x4 lo = q[0], hi = q[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = lo[e];
      v[4 + e] = hi[e];
    }
  } else {
    const u32x4 w =
        *reinterpret_cast<const u32x4_any*>(static_cast<const uint16_t*>(p) + i);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = T::to_f((uint16_t)w[e]);
      v[2 * e + 1] = T::to_f((uint16_t)(w[e] >> 16));
    }
  }
}

template <class T>
__device__ inline void load8_either(const void* p, bool wide, int64_t i, float (&v)[8]) {
  if (wide) {
    load8<F32>(p, i, v);
  } else {
    load8<T>(p, i, v);
  }
}

template <class T>
__device__ inline void store8(void* p, int64_t i, const float (&v)[8], int skip) {
  if (skip == 0) {
    if constexpr (T::code == 3) {
      f32x4_any* q = reinterpret_cast<f32x4_any*>(static_cast<float*>(p) + i);
      q[0] = f32x4{v[0], v[1], v[2], v[3]};
      q[1] = f32x4{v[4], v[5], v[6], v[7]};
    } else {
      u32x4 w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = pack2<T>(v[2 * e], v[2 * e + 1]);
      *reinterpret_cast<u32x4_any*>(static_cast<uint16_t*>(p) + i) = w;
    }
  } else if (skip < 8) {
#pragma unroll
    for (int e = 1; e < 8; ++e)
      if (e >= skip) store_elem<T>(p, i + e, v[e]);
  }
}

// Sum over the `lanes` lanes of a row, in each of them: within 64 lanes a butterfly on the
// VALU (both lanes of a pair add the same two values), then the row's waves in order.
__device__ inline float row_sum(float v, int lanes, float* part) {
#define RECAP_DPP_ADD(ctrl) \
  v += __uint_as_float((unsigned)__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), ctrl, 0xf, 0xf, false))
  if (lanes > 1) RECAP_DPP_ADD(0xB1);   // lane ^ 1
  if (lanes > 2) RECAP_DPP_ADD(0x4E);   // lane ^ 2
  if (lanes > 4) RECAP_DPP_ADD(0x141);  // the other 4 of 8
  if (lanes > 8) RECAP_DPP_ADD(0x140);  // the other 8 of 16
#undef RECAP_DPP_ADD
  if (lanes > 16) {
    const auto r =
        __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if (lanes > 32) v = pair_sum(v);
  if (lanes > 64) {
    const int wave = threadIdx.x >> 6, waves = lanes >> 6, first = wave & ~(waves - 1);
    __syncthreads();  // the previous sum's readers are done with `part`
    if ((threadIdx.x & 63) == 0) part[wave] = v;
    __syncthreads();
    v = part[first];
    for (int w = 1; w < waves; ++w) v += part[first + w];
  }
  return v;
}

}  // namespace recap

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

template <class T>
constexpr unsigned kBytes = T::code == 3 ? 4 : 2;

constexpr int64_t kMaxBlocks = 1 << 20;  // of a launch, whose threads have to be under 2^32

// A call that moves this much or more loads its rows past the caches: they cannot stay in the
// 256 MB Infinity Cache beside what comes after.  A chain gated_residual_norm, two projections,
// gated_residual_norm at width 1536 in us, loads through the caches -> past them: 100 MB a call
// 178 -> 182, 151 MB 257 -> 258, 252 MB 385 -> 379, 302 MB 483 -> 471, 403 MB 595 -> 580.
// Rotated queries and keys are also stored past them from there on (rotary.hip).
constexpr int64_t kStreamBytes = int64_t(192) << 20;

// 16 and 8 bytes at any address; STREAM: past the caches, for data that is used once.  (A vector
// type's alignment is lost in a template argument, so the types are named here.)
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef u32x2 u32x2_any __attribute__((aligned(2)));

template <bool STREAM>
__device__ inline u32x4 load_words4(const void* p) {
  const u32x4_any* q = static_cast<const u32x4_any*>(p);
  return STREAM ? __builtin_nontemporal_load(q) : *q;
}
template <bool STREAM>
__device__ inline u32x2 load_words2(const void* p) {
  const u32x2_any* q = static_cast<const u32x2_any*>(p);
  return STREAM ? __builtin_nontemporal_load(q) : *q;
}
template <bool STREAM>
__device__ inline void store_words4(void* p, u32x4 w) {
  u32x4_any* q = static_cast<u32x4_any*>(p);
  if (STREAM) {
    __builtin_nontemporal_store(w, q);
  } else {
    *q = w;
  }
}
template <bool STREAM>
__device__ inline void store_words2(void* p, u32x2 w) {
  u32x2_any* q = static_cast<u32x2_any*>(p);
  if (STREAM) {
    __builtin_nontemporal_store(w, q);
  } else {
    *q = w;
  }
}

// Address of element i of a row: the row's own address is uniform over a wave of 64 lanes a row,
// and a 32-bit byte offset to it is the form the memory instructions take without arithmetic.
template <class T>
__device__ inline const char* place(const void* row, unsigned i) {
  return static_cast<const char*>(row) + i * kBytes<T>;
}
template <class T>
__device__ inline char* place(void* row, unsigned i) {
  return static_cast<char*>(row) + i * kBytes<T>;
}
template <class T>
__device__ inline const void* row_of(const void* p, int64_t i) {
  return static_cast<const char*>(p) + i * kBytes<T>;
}

// N elements (4 or 8) of a row from element i on, as fp32.
template <class T, bool STREAM = false, int N>
__device__ inline void load_chunk(const void* row, unsigned i, float (&v)[N]) {
  if constexpr (T::code == 3) {
#pragma unroll
    for (int k = 0; k < N; k += 4) {
      const u32x4 w = load_words4<STREAM>(place<T>(row, i + k));
#pragma unroll
      for (int e = 0; e < 4; ++e) v[k + e] = __uint_as_float(w[e]);
    }
  } else {
    unsigned w[N / 2];
    if constexpr (N == 8) {
      const u32x4 u = load_words4<STREAM>(place<T>(row, i));
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = u[e];
    } else {
      const u32x2 u = load_words2<STREAM>(place<T>(row, i));
      w[0] = u[0];
      w[1] = u[1];
    }
#pragma unroll
    for (int e = 0; e < N / 2; ++e) {
      v[2 * e] = T::to_f((uint16_t)w[e]);
      v[2 * e + 1] = T::to_f((uint16_t)(w[e] >> 16));
    }
  }
}

// N elements rounded to T, as they go to memory.
template <class T, int N>
struct Rounded {
  static constexpr int kWords = T::code == 3 ? N : N / 2;
  unsigned w[kWords];

  __device__ inline void set(const float (&v)[N]) {
    if constexpr (T::code == 3) {
#pragma unroll
      for (int e = 0; e < N; ++e) w[e] = __float_as_uint(v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < N / 2; ++e) w[e] = pack2<T>(v[2 * e], v[2 * e + 1]);
    }
  }

  // To elements i.. of a row, those from `skip` on.
  template <bool STREAM>
  __device__ inline void store(void* row, unsigned i, int skip) const {
    if (skip == 0) {
      if constexpr (kWords >= 4) {
#pragma unroll
        for (int k = 0; k < kWords; k += 4)
          store_words4<STREAM>(place<T>(row, i) + 4 * k, u32x4{w[k], w[k + 1], w[k + 2], w[k + 3]});
      } else {
        store_words2<STREAM>(place<T>(row, i), u32x2{w[0], w[1]});
      }
    } else if (skip < N) {
#pragma unroll
      for (int e = 1; e < N; ++e)
        if (e >= skip) {
          if constexpr (T::code == 3) {
            *reinterpret_cast<unsigned*>(place<T>(row, i + e)) = w[e];
          } else {
            *reinterpret_cast<uint16_t*>(place<T>(row, i + e)) =
                (uint16_t)(e & 1 ? w[e / 2] >> 16 : w[e / 2]);
          }
        }
    }
  }
};

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

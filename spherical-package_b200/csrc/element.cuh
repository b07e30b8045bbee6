// Element types of the operators around the convolutions (norm, log probabilities, optimizer step): float32, bfloat16 and
// float16 in memory, float32 in registers, one rounding to nearest on the way out; e4m3 for what is held in 8 bits.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"

namespace sph {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// A weight of its own type, float32 or the data's.
template <typename T> __device__ __forceinline__ float load_weight(const void *w, int64_t i, bool f32) {
  return f32 ? __ldg((const float *)w + i) : to_float(((const T *)w)[i]);
}
template <typename T> __device__ __forceinline__ void store_weight(void *w, int64_t i, float v, bool f32) {
  if (f32)
    ((float *)w)[i] = v;
  else
    ((T *)w)[i] = from_float<T>(v);
}

// Values held in 8 bits: e4m3 times a float32 scale, the largest magnitude of a group at e4m3's largest, 448.  A group
// whose values all lie below kTiny (448 / amax would not be finite much below it) is a group of zeros with scale 0.
constexpr float kE4m3Max = 448.f, kTiny = 0x1p-100f;
// (the reciprocals are rounded before they are multiplied, as elementary tensor operations do it)
struct Scale {
  float scale, inverse;
  static __device__ __forceinline__ Scale of(float amax) {
    const bool zero = amax < kTiny;
    return Scale{zero ? 0.f : amax * (1.f / kE4m3Max), zero ? 0.f : __fmul_rn(__frcp_rn(amax), kE4m3Max)};
  }
  // Of values p rstd, most = max |p|: the codes are p `inverse`, without rstd, whose last bit depends on the order in which a
  // kernel has summed; so a norm's codes are the same from every kernel.
  static __device__ __forceinline__ Scale of(float most, float rstd) {
    const Scale r = of(most * rstd);
    return Scale{r.scale, r.inverse > 0.f ? __fmul_rn(__frcp_rn(most), kE4m3Max) : r.inverse};
  }
};
__device__ __forceinline__ __nv_fp8_storage_t to_e4m3(float v) { return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }
__device__ __forceinline__ float from_e4m3(__nv_fp8_storage_t v) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(v, __NV_E4M3)));
}

// max that keeps NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Two float32 operations in one instruction.
__device__ __forceinline__ unsigned long long as_pair(float2 v) { return __builtin_bit_cast(unsigned long long, v); }
__device__ __forceinline__ float2 add_pair(float2 a, float2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(as_pair(a)), "l"(as_pair(b)));
  return __builtin_bit_cast(float2, r);
}
__device__ __forceinline__ float2 mul_pair(float2 a, float2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(as_pair(a)), "l"(as_pair(b)));
  return __builtin_bit_cast(float2, r);
}
__device__ __forceinline__ float2 fma_pair(float2 a, float2 b, float2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(as_pair(a)), "l"(as_pair(b)), "l"(as_pair(c)));
  return __builtin_bit_cast(float2, r);
}

// Sums (or other joins) over the threads of a warp or of a block; every thread gets the same value.
template <class F> __device__ __forceinline__ float warp_join(float v, F f) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
// Over groups of `lanes` neighbouring lanes, a power of two.
template <class F> __device__ __forceinline__ float lanes_join(float v, int lanes, F f) {
  for (int d = lanes >> 1; d > 0; d >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, d));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
  return warp_join(v, [](float a, float b) { return a + b; });
}
// `shared`: one float per warp.
template <class F> __device__ __forceinline__ float block_join(float v, float *shared, F f) {
  v = warp_join(v, f);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (lane == 0) shared[warp] = v;
  __syncthreads();
  float r = shared[0];
  for (int i = 1; i < warps; i++) r = f(r, shared[i]);
  __syncthreads();
  return r;
}

// Asynchronous copies into shared memory.
__device__ __forceinline__ void copy_16(void *to, const void *from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_4(void *to, const void *from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }

// Two 16-bit elements in a word, the first below.
template <typename T> struct TwoOf { using Type = __nv_bfloat162; };
template <> struct TwoOf<__half> { using Type = __half2; };
template <typename T> __device__ __forceinline__ unsigned two_as_word(float2 v) {
  typename TwoOf<T>::Type q;
  if constexpr (std::is_same<T, __half>::value) q = __float22half2_rn(v);
  else q = __float22bfloat162_rn(v);
  return *reinterpret_cast<const unsigned *>(&q);
}
template <typename T> __device__ __forceinline__ typename TwoOf<T>::Type word_as_two(unsigned w) {
  return *reinterpret_cast<const typename TwoOf<T>::Type *>(&w);
}

// 16 bytes of a row at a time.  A row need not start on a 16-byte boundary: vector v holds the elements [v n - shift, v n - shift + n)
// with `shift` the elements between the boundary before the row and its start; the vectors at its two ends are put together
// from single elements.
template <typename T> struct RowVector {
  static constexpr int N = 16 / (int)sizeof(T);
  union {
    uint4 u;
    T t[N];
  };
  static __device__ __forceinline__ int shift_of(const T *row) { return (int)((uintptr_t)row % 16 / sizeof(T)); }
  // Elements outside the row are `outside`.
  __device__ __forceinline__ void load(const T *row, int first, int C, T outside) {
    if (first >= 0 && first + N <= C) {
      u = *(const uint4 *)(row + first);
    } else {
#pragma unroll
      for (int i = 0; i < N; i++) t[i] = first + i >= 0 && first + i < C ? row[first + i] : outside;
    }
  }
  __device__ __forceinline__ void store(T *row, int first, int C) const {
    if (first >= 0 && first + N <= C) {
      *(uint4 *)(row + first) = u;
    } else {
#pragma unroll
      for (int i = 0; i < N; i++)
        if (first + i >= 0 && first + i < C) row[first + i] = t[i];
    }
  }
  __device__ __forceinline__ float at(int i) const { return to_float(t[i]); }
  // An element that is not known at compile time.
  __device__ __forceinline__ float at_any(int i) const {
    float v = 0.f;
#pragma unroll
    for (int j = 0; j < N; j++) v = i == j ? to_float(t[j]) : v;
    return v;
  }
  __device__ __forceinline__ void set_any(int i, float v) {
#pragma unroll
    for (int j = 0; j < N; j++) t[j] = i == j ? from_float<T>(v) : t[j];
  }
  // Elements 2 i and 2 i + 1.
  __device__ __forceinline__ float2 pair(int i) const {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const unsigned w = i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w;
      return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    } else {
      return make_float2(to_float(t[2 * i]), to_float(t[2 * i + 1]));
    }
  }
  __device__ __forceinline__ void set_pair(int i, float2 v) {
    if constexpr (std::is_same<T, float>::value) {
      t[2 * i] = v.x, t[2 * i + 1] = v.y;
    } else {
      (i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w) = two_as_word<T>(v);
    }
  }
};

// Run a statement with T = the element type of a dtype code.
#define SPH_DISPATCH_ELEMENT(dtype, ...)                                \
  switch (dtype) {                                                      \
    case SPH_BF16: { using T = __nv_bfloat16; __VA_ARGS__; break; }     \
    case SPH_F16: { using T = __half; __VA_ARGS__; break; }             \
    default: { using T = float; __VA_ARGS__; break; }                   \
  }
inline bool element_dtype(int dtype) { return dtype == SPH_F32 || dtype == SPH_BF16 || dtype == SPH_F16; }
inline size_t element_size(int dtype) { return dtype == SPH_F32 ? 4 : 2; }

}  // namespace sph

// AdamW step over many tensors in one launch per 'kMaxTensors' of them:
//
//     m = b1 m + (1 - b1) g;   v = b2 v + (1 - b2) g^2;
//     w = w (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Moments in float32, or in e4m3 with one float32 scale for each 256 values of a tensor: m as it is, v as its square root
// (e4m3 spans 2^18 between its smallest and largest value, so the root keeps 2^36 of v) with what is positive never held as
// zero, which would divide m by eps.  Values are rounded to nearest: rounding at random instead would add, every step, a
// noise that the average over 1 / (1 - b2) steps does not forget (at e4m3's steps and b2 = 0.999 about the size of v itself).
// What is not finite is held as NaN, and leaves the other values of its 256 as they are.
#include "element.cuh"

#include <algorithm>

namespace sph {

constexpr int kAdamBlock = 256;  // values behind one scale, and what a warp takes at once: eight a lane

struct AdamTensor {
  void *param;
  const void *grad;
  float *master;
  void *m, *v;
  float *m_scale, *v_scale;
  int64_t n;
};
template <int CAP> struct AdamArgs {
  AdamTensor tensor[CAP];
  int first[CAP + 1];          // first task of each tensor; one past the last behind them
  unsigned char aligned[CAP];  // eight values may be read at once
  int tensors, chunk;          // a task: up to chunk blocks of 256 values
  float lr, beta1, beta2, rest1, rest2, eps, decay, grad_scale;  // rest = 1 - beta, which 1.f - (float)beta is 5e-5 off
  double log_beta1, log_beta2;
  float step_size, root;     // lr / (1 - b1^t), 1 / sqrt(1 - b2^t); from the device's values where there are any
  const float *lr_at, *step_at;
};

// A lane's eight neighbouring values, in stores of up to 32 bytes.
__device__ __forceinline__ void store8(float *p, const float (&v)[8]) {
  asm volatile("st.global.v8.f32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]),
               "f"(v[5]), "f"(v[6]), "f"(v[7]), "l"(p)
               : "memory");
}
template <typename T> __device__ __forceinline__ void store8(T *p, const float (&v)[8]) {
  union { uint4 u; T t[8]; } q;
#pragma unroll
  for (int i = 0; i < 8; i++) q.t[i] = from_float<T>(v[i]);
  *(uint4 *)p = q.u;
}
struct E4m3 {
  __nv_fp8_storage_t v;
};
__device__ __forceinline__ float to_float(E4m3 v) { return from_e4m3(v.v); }
template <> __device__ __forceinline__ E4m3 from_float<E4m3>(float v) { return E4m3{to_e4m3(v)}; }
__device__ __forceinline__ void store8(E4m3 *p, const float (&v)[8]) {
  unsigned q[4];
#pragma unroll
  for (int i = 0; i < 4; i++) q[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i], v[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
  *(uint2 *)p = make_uint2(q[0] | q[1] << 16, q[2] | q[3] << 16);
}

// The same values as they are in memory, in loads of up to 32 bytes.
template <typename T> struct Raw {
  unsigned w[2 * sizeof(T)];
  __device__ __forceinline__ void load(const T *p) {
    if constexpr (sizeof(T) == 4) {
      asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                   : "l"(p));
    } else if constexpr (sizeof(T) == 2) {
      const uint4 q = *(const uint4 *)p;
      w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
    } else {
      const uint2 q = *(const uint2 *)p;
      w[0] = q.x, w[1] = q.y;
    }
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if constexpr (sizeof(T) == 4) {
        v[2 * i] = __uint_as_float(w[2 * i]), v[2 * i + 1] = __uint_as_float(w[2 * i + 1]);
      } else if constexpr (sizeof(T) == 1) {
        const unsigned two = (w[i >> 1] >> (16 * (i & 1))) & 0xffffu;
        const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3)));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      } else if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(word_as_two<T>(w[i]));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      } else {
        v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
};

// A lane's eight of a warp's 256 values: neighbours, or every 32nd where the tensor is not aligned for that or ends inside.
template <typename T> __device__ __forceinline__ void load_lane(const T *p, int lane, bool wide, int n, float (&v)[8]) {
  if (wide) {
    Raw<T> q;
    q.load(p + 8 * lane);
    q.values(v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = lane + 32 * i < n ? to_float(p[lane + 32 * i]) : 0.f;
  }
}
template <typename T> __device__ __forceinline__ void store_lane(T *p, int lane, bool wide, int n, const float (&v)[8]) {
  if (wide) {
    store8(p + 8 * lane, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (lane + 32 * i < n) p[lane + 32 * i] = from_float<T>(v[i]);
  }
}

// Largest magnitude of a warp's 256 values; NaN is passed over, and its code is NaN; infinities become NaN and leave the others
// alone.
__device__ __forceinline__ float largest_of(float (&v)[8]) {
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; i++) amax = fmaxf(amax, fabsf(v[i]));
  amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));
  if (amax == INFINITY) {
    amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
      v[i] = fabsf(v[i]) < INFINITY ? v[i] : NAN;
      amax = fmaxf(amax, fabsf(v[i]));
    }
    amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));
  }
  return amax;
}
// Both moments' scales; their reciprocals are one, in two lanes.
struct Scales {
  float m, m_inverse, u, u_inverse;
  __device__ __forceinline__ Scales(float m_max, float u_max) {
    const Scale s = Scale::of(threadIdx.x & 1 ? u_max : m_max);
    m = __shfl_sync(0xffffffffu, s.scale, 0), m_inverse = __shfl_sync(0xffffffffu, s.inverse, 0);
    u = __shfl_sync(0xffffffffu, s.scale, 1), u_inverse = __shfl_sync(0xffffffffu, s.inverse, 1);
  }
};

// A warp takes up to `chunk` blocks of 256 values of one tensor.  With 8-bit moments, of which fewer bytes are on their way for the
// same work, it fetches the next block while it works on one (332M bf16 weights with masters: 1146 us without, 875 with; through
// asynchronous copies into shared memory, which leave less L1 for what plain loads have on their way, 983; 895 to 907 since the old
// moments' products and the root are rounded by themselves).  It spills up to 32 bytes of its 80 registers.
template <typename P, typename G, bool EIGHT, bool MASTER, int CAP>
__global__ void __launch_bounds__(256, EIGHT ? 3 : 4) adamw_kernel(const __grid_constant__ AdamArgs<CAP> a) {
  using W = typename std::conditional<MASTER, float, P>::type;  // what is updated
  const int lane = threadIdx.x & 31, task = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (task >= a.first[a.tensors]) return;
  int lo = 0, hi = a.tensors;  // the tensor that holds the task: first[lo] <= task < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.first[mid] <= task) lo = mid; else hi = mid;
  }
  const AdamTensor &t = a.tensor[lo];
  const bool aligned = a.aligned[lo];
  const W *weights = MASTER ? (const W *)t.master : (const W *)t.param;
  int64_t b = (int64_t)(task - a.first[lo]) * a.chunk;
  const int count = (int)min((int64_t)a.chunk, (t.n + kAdamBlock - 1) / kAdamBlock - b);
  Raw<W> w_next;
  Raw<G> g_next;
  Raw<E4m3> m_next, v_next;
  float lr = a.lr, step_size = a.step_size, root = a.root;
  const auto fetch = [&](int j) {  // the j-th block from here on
    const int64_t at = (b + j) * kAdamBlock;
    if (j >= count) return;
    if (aligned && at + kAdamBlock <= t.n) {
      w_next.load(weights + at + 8 * lane);
      g_next.load((const G *)t.grad + at + 8 * lane);
      m_next.load((const E4m3 *)t.m + at + 8 * lane);
      v_next.load((const E4m3 *)t.v + at + 8 * lane);
    }
  };
  if (EIGHT) fetch(0);
  if (a.step_at) {
    if (a.lr_at) lr = *a.lr_at;
    const double step = (double)*a.step_at;
    step_size = (float)(lr / -expm1(step * a.log_beta1));
    root = (float)(1.0 / sqrt(-expm1(step * a.log_beta2)));
  }
  const float keep = 1.f - lr * a.decay;
  for (int j = 0; j < count; j++) {
    const int64_t at = (b + j) * kAdamBlock;
    const int n = t.n - at < kAdamBlock ? (int)(t.n - at) : kAdamBlock;
    const bool wide = n == kAdamBlock && aligned;
    float w[8], g[8], m[8], v[8];
    const float ms = EIGHT ? t.m_scale[b + j] : 0.f, vs = EIGHT ? t.v_scale[b + j] : 0.f;
    if (EIGHT && wide) {
      w_next.values(w);
      g_next.values(g);
      m_next.values(m);
      v_next.values(v);
    } else {
      load_lane(weights + at, lane, wide, n, w);
      load_lane((const G *)t.grad + at, lane, wide, n, g);
      if (EIGHT) {
        load_lane((const E4m3 *)t.m + at, lane, wide, n, m);
        load_lane((const E4m3 *)t.v + at, lane, wide, n, v);
      } else {
        load_lane((const float *)t.m + at, lane, wide, n, m);
        load_lane((const float *)t.v + at, lane, wide, n, v);
      }
    }
    if (EIGHT) fetch(j + 1);
    // The old moment's product and the root are rounded by themselves, the new term is fused, as elementary tensor operations do
    // it: codes are cut from these values, and would otherwise depend on what the compiler fuses.
    const auto two = [](float x) { return make_float2(x, x); };
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      float2 gi = make_float2(g[i], g[i + 1]), mi = make_float2(m[i], m[i + 1]), vi = make_float2(v[i], v[i + 1]), wi = make_float2(w[i], w[i + 1]);
      if (EIGHT) {
        mi = mul_pair(mi, two(ms));
        vi = mul_pair(vi, two(vs));
        vi = mul_pair(vi, vi);
      }
      gi = mul_pair(gi, two(a.grad_scale));
      mi = fma_pair(two(a.rest1), gi, mul_pair(two(a.beta1), mi));
      vi = fma_pair(two(a.rest2), mul_pair(gi, gi), mul_pair(two(a.beta2), vi));
      const float2 u = make_float2(sqrtf(vi.x), sqrtf(vi.y)), d = fma_pair(u, two(root), two(a.eps));
      const float2 q = make_float2(__fdividef(mi.x, d.x), __fdividef(mi.y, d.y));
      wi = fma_pair(two(-step_size), q, mul_pair(wi, two(keep)));
      w[i] = wi.x, w[i + 1] = wi.y, m[i] = mi.x, m[i + 1] = mi.y;
      v[i] = EIGHT ? u.x : vi.x, v[i + 1] = EIGHT ? u.y : vi.y;
    }
    if (MASTER) store_lane(t.master + at, lane, wide, n, w);
    store_lane((P *)t.param + at, lane, wide, n, w);
    if (EIGHT) {
      const float m_max = largest_of(m), u_max = largest_of(v);
      const Scales scale(m_max, u_max);
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float2 p = mul_pair(make_float2(m[i], m[i + 1]), two(scale.m_inverse)), q = mul_pair(make_float2(v[i], v[i + 1]), two(scale.u_inverse));
        m[i] = p.x, m[i + 1] = p.y;
        v[i] = q.x > 0.f ? fmaxf(q.x, 0x1p-9f) : q.x;
        v[i + 1] = q.y > 0.f ? fmaxf(q.y, 0x1p-9f) : q.y;
      }
      store_lane((E4m3 *)t.m + at, lane, wide, n, m);
      store_lane((E4m3 *)t.v + at, lane, wide, n, v);
      if (lane == 0) {
        t.m_scale[b + j] = scale.m;
        t.v_scale[b + j] = scale.u;
      }
    } else {
      store_lane((float *)t.m + at, lane, wide, n, m);
      store_lane((float *)t.v + at, lane, wide, n, v);
    }
  }
}
inline bool wide_aligned(const AdamTensor &t, int param_size, int grad_size, int state_size) {
  return ((uintptr_t)t.param % (8 * param_size) | (uintptr_t)t.grad % (8 * grad_size) | (uintptr_t)t.m % (8 * state_size) |
          (uintptr_t)t.v % (8 * state_size) | (uintptr_t)t.master % 32) == 0;
}

template <typename P, typename G, bool EIGHT, bool MASTER, int CAP>
void adamw_launch(const AdamArgs<CAP> &a, cudaStream_t st) {
  adamw_kernel<P, G, EIGHT, MASTER, CAP><<<(unsigned)cdiv(a.first[a.tensors], 8), 256, 0, st>>>(a);
}
template <int CAP> void adamw_dispatch(const AdamArgs<CAP> &a, int dtype, int grad_dtype, bool eight, bool master, cudaStream_t st) {
  SPH_DISPATCH_ELEMENT(dtype, {
    if (grad_dtype == SPH_F32 || dtype == SPH_F32) {
      if (eight && master)
        adamw_launch<T, float, true, true>(a, st);
      else if (eight)
        adamw_launch<T, float, true, false>(a, st);
      else if (master)
        adamw_launch<T, float, false, true>(a, st);
      else
        adamw_launch<T, float, false, false>(a, st);
    } else {
      if (eight && master)
        adamw_launch<T, T, true, true>(a, st);
      else if (eight)
        adamw_launch<T, T, true, false>(a, st);
      else if (master)
        adamw_launch<T, T, false, true>(a, st);
      else
        adamw_launch<T, T, false, false>(a, st);
    }
  });
}

// The tensors [from, to) of a call; kernel parameters hold at most 32,764 bytes.
constexpr int kFewTensors = 32, kMaxTensors = 440;
static_assert(sizeof(AdamArgs<kMaxTensors>) <= 32764, "kernel parameters");

}  // namespace sph

using namespace sph;

template <int CAP>
static int adamw_group(int from, int count, void *const *params, const void *const *grads, float *const *masters, void *const *m,
                       void *const *v, float *const *m_scales, float *const *v_scales, const int64_t *numels, int dtype, int grad_dtype,
                       int state_bits, const AdamArgs<1> &common, cudaStream_t st) {
  AdamArgs<CAP> a;
  a.tensors = count;
  a.lr = common.lr, a.beta1 = common.beta1, a.beta2 = common.beta2, a.eps = common.eps, a.decay = common.decay;
  a.rest1 = common.rest1, a.rest2 = common.rest2, a.grad_scale = common.grad_scale, a.log_beta1 = common.log_beta1, a.log_beta2 = common.log_beta2;
  a.step_size = common.step_size, a.root = common.root, a.lr_at = common.lr_at, a.step_at = common.step_at;
  int64_t blocks = 0;
  for (int i = 0; i < count; i++) blocks += (numels[from + i] + kAdamBlock - 1) / kAdamBlock;
  // A warp finds its tensor once for up to 32 blocks (4 of 32-bit moments, which are as fast one by one and faster side by side:
  // 174M float32 weights 719 us in fours, 743 in 32s), as long as every SM's 64 warps have two such tasks.
  a.chunk = (int)std::min<int64_t>(state_bits == 8 ? 32 : 4, std::max<int64_t>(1, blocks / (148 * 64 * 2)));
  int64_t tasks = 0;
  for (int i = 0; i < count; i++) {
    const int k = from + i;
    a.tensor[i] = AdamTensor{params[k], grads[k], masters ? masters[k] : nullptr, m[k], v[k], m_scales ? m_scales[k] : nullptr,
                             v_scales ? v_scales[k] : nullptr, numels[k]};
    a.aligned[i] = wide_aligned(a.tensor[i], (int)element_size(dtype), (int)element_size(grad_dtype), state_bits / 8);
    a.first[i] = (int)tasks;
    tasks += (numels[k] + kAdamBlock * a.chunk - 1) / (kAdamBlock * a.chunk);
  }
  a.first[count] = (int)tasks;
  if (tasks == 0) return 0;
  adamw_dispatch<CAP>(a, dtype, grad_dtype, state_bits == 8, masters != nullptr, st);
  return 1;
}

extern "C" int sph_adamw_step(int64_t tensors, void *const *params, const void *const *grads, float *const *masters, void *const *m,
                              void *const *v, float *const *m_scales, float *const *v_scales, const int64_t *numels, int dtype,
                              int grad_dtype, int state_bits, double lr, double beta1, double beta2, double eps, double weight_decay,
                              double grad_scale, double step, const float *lr_at, const float *step_at, void *stream) {
  SPH_RANGE("sph_adamw_step");
  if (!element_dtype(dtype) || !element_dtype(grad_dtype) || (grad_dtype != SPH_F32 && grad_dtype != dtype) ||
      (state_bits != 8 && state_bits != 32) || (masters && dtype == SPH_F32))
    return SPH_ERR_UNSUPPORTED;
  if (tensors < 0 || (tensors > 0 && (!params || !grads || !m || !v || !numels)) || !(beta1 >= 0 && beta1 < 1) ||
      !(beta2 >= 0 && beta2 < 1) || !(eps >= 0) || (!step_at && !(step >= 1)) || (lr_at && !step_at) ||
      (state_bits == 8 && tensors > 0 && (!m_scales || !v_scales)))
    return SPH_ERR_INVALID_ARGUMENT;
  for (int64_t i = 0; i < tensors; i++) {
    if (numels[i] < 0 || (numels[i] > 0 && (!params[i] || !grads[i] || !m[i] || !v[i] || (masters && !masters[i]) ||
                                            (state_bits == 8 && (!m_scales[i] || !v_scales[i])))))
      return SPH_ERR_INVALID_ARGUMENT;
    if (numels[i] > ((int64_t)1 << 38)) return SPH_ERR_TOO_LARGE;
  }
  AdamArgs<1> c{};
  c.lr = (float)lr, c.beta1 = (float)beta1, c.beta2 = (float)beta2, c.eps = (float)eps, c.decay = (float)weight_decay;
  c.rest1 = (float)(1.0 - beta1), c.rest2 = (float)(1.0 - beta2), c.grad_scale = (float)grad_scale;
  c.log_beta1 = log(beta1), c.log_beta2 = log(beta2);
  c.lr_at = lr_at, c.step_at = step_at;
  if (!step_at) {
    c.step_size = (float)(lr / (1.0 - pow(beta1, step)));
    c.root = (float)(1.0 / sqrt(1.0 - pow(beta2, step)));
  }
  cudaStream_t st = (cudaStream_t)stream;
  int launches = 0;
  for (int64_t from = 0; from < tensors;) {
    // as many tensors as the parameters hold and 2^31 blocks number
    int count = 0;
    int64_t blocks = 0;
    while (from + count < tensors && count < kMaxTensors) {
      blocks += (numels[from + count] + kAdamBlock - 1) / kAdamBlock;
      if (blocks > 0x7fffff00ll && count > 0) break;
      count++;
    }
    if (count <= kFewTensors)
      launches += adamw_group<kFewTensors>((int)from, count, params, grads, masters, m, v, m_scales, v_scales, numels, dtype, grad_dtype,
                                           state_bits, c, st);
    else
      launches += adamw_group<kMaxTensors>((int)from, count, params, grads, masters, m, v, m_scales, v_scales, numels, dtype, grad_dtype,
                                           state_bits, c, st);
    from += count;
  }
  return launches ? launch_status(launches) : SPH_OK;
}

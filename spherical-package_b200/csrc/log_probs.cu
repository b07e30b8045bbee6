// Log probabilities of given classes, entropies and the most probable classes, over rows (rows, C) or planes (outer, C, inner):
//
//     m = max x, S = sum e^(x - m), T = sum e^(x - m) (x - m);   lse = m + ln S;   H = ln S - T / S;   log p_j = x_j - lse
//
// and the gradient, with p_j = e^(x_j - lse), g the gradient of the target's log probability, h that of H and t_i those of the
// most probable classes c_i:
//
//     dx_j = -p_j (g + sum t + h (log p_j + H)) + [j = target] g + sum_i [j = c_i] t_i
//
// A class with the logit -inf has p = 0 and adds nothing to H.  A distribution whose every logit is -inf is empty: log
// probabilities -inf, H = 0, no gradient.  +inf and NaN make the distribution NaN.  Targets equal to ignore_index have log
// probability 0 and no gradient; other targets outside [0, C) NaN.  Equal logits are ordered by their index, NaN before numbers.
#include "element.cuh"

namespace sph {

struct LogProbArgs {
  const void *x;
  const int64_t *target;
  float *log_probs, *entropy, *lse, *top;  // top (outer, k, inner)
  int64_t *top_index;
  int64_t outer, inner, x_stride, ignore_index;
  int C, k;
};

// Order of the candidates as one number: larger is better; value first (NaN above all), then the lower index.
__device__ __forceinline__ unsigned long long candidate(float v, int index) {
  unsigned u = __float_as_uint(v + 0.f);  // (-0 and 0 are equal)
  u = v != v ? 0xffffffffu : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)u << 32) | (0xffffffffu - (unsigned)index);
}
__device__ __forceinline__ int candidate_index(unsigned long long c) { return (int)(0xffffffffu - (unsigned)c); }

// Running softmax statistics of a part of a distribution.
struct Stats {
  float m = -INFINITY, s = 0.f, t = 0.f;
  __device__ __forceinline__ void add(float x) {
    const float n = fmaxf(m, x), base = n == -INFINITY ? 0.f : n;
    rescale(base);
    m = n;
    const float d = x - base, e = expf(d);
    s += e;
    t += e * fmaxf(d, -1e4f);
  }
  // The sums for the maximum `base` instead of m: e^(x-b) = e^(x-m) e^(m-b), and t's terms move by m - b.
  __device__ __forceinline__ void rescale(float base) {
    const float d = m - base;
    if (d == 0.f || m == -INFINITY) return;  // (nothing but -inf so far: the sums are 0, or NaN)
    const float f = expf(d);
    t = (t + s * fmaxf(d, -1e4f)) * f;
    s *= f;
  }
  __device__ __forceinline__ void join(Stats o) {
    const float n = fmaxf(m, o.m), base = n == -INFINITY ? 0.f : n;
    rescale(base);
    o.rescale(base);
    m = n;
    s += o.s;
    t += o.t;
  }
  __device__ __forceinline__ float lse() const { return s == 0.f ? -INFINITY : (m == -INFINITY ? 0.f : m) + logf(s); }
  __device__ __forceinline__ float entropy() const {
    const float h = s == 0.f ? 0.f : logf(s) - t / s;
    return h < 0.f ? 0.f : h;
  }
};

__device__ __forceinline__ float target_log_prob(const LogProbArgs &a, int64_t t, float lse, float x_t) {
  if (t == a.ignore_index) return 0.f;
  if (t < 0 || t >= a.C) return NAN;
  return lse == -INFINITY ? -INFINITY : x_t - lse;
}

template <typename T> __global__ void __launch_bounds__(256) log_probs_rows_kernel(LogProbArgs a) {
  __shared__ Stats stats[8];
  __shared__ unsigned long long best[8];
  const int64_t row = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T *x = (const T *)a.x + row * a.x_stride;
  Stats st;
  for (int c = threadIdx.x; c < a.C; c += 256) st.add(to_float(x[c]));
  for (int d = 16; d > 0; d >>= 1) {
    Stats o;
    o.m = __shfl_xor_sync(0xffffffffu, st.m, d);
    o.s = __shfl_xor_sync(0xffffffffu, st.s, d);
    o.t = __shfl_xor_sync(0xffffffffu, st.t, d);
    st.join(o);
  }
  if (lane == 0) stats[warp] = st;
  __syncthreads();
  st = stats[0];
  for (int i = 1; i < 8; i++) st.join(stats[i]);
  const float lse = st.lse();
  if (threadIdx.x == 0) {
    const int64_t t = a.target[row];
    a.log_probs[row] = target_log_prob(a, t, lse, t >= 0 && t < a.C ? to_float(x[t]) : 0.f);
    a.entropy[row] = st.entropy();
    if (a.lse) a.lse[row] = lse;
  }
  unsigned long long last = ~0ull;
  for (int i = 0; i < a.k; i++) {  // the best that comes after the last one
    unsigned long long mine = 0;
    for (int c = threadIdx.x; c < a.C; c += 256) {
      const unsigned long long q = candidate(to_float(x[c]), c);
      if (q < last && q > mine) mine = q;
    }
    for (int d = 16; d > 0; d >>= 1) {
      const unsigned long long o = __shfl_xor_sync(0xffffffffu, mine, d);
      if (o > mine) mine = o;
    }
    if (lane == 0) best[warp] = mine;
    __syncthreads();
    last = best[0];
    for (int w = 1; w < 8; w++)
      if (best[w] > last) last = best[w];
    __syncthreads();
    if (threadIdx.x == 0) {
      const int c = candidate_index(last);
      a.top_index[row * a.k + i] = c;
      a.top[row * a.k + i] = lse == -INFINITY ? -INFINITY : to_float(x[c]) - lse;
    }
  }
}

template <typename T> __global__ void __launch_bounds__(256) log_probs_planes_kernel(LogProbArgs a) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= a.outer * a.inner) return;
  const int64_t o = at / a.inner, i = at % a.inner;
  const T *x = (const T *)a.x + o * a.C * a.inner + i;
  Stats st;
  for (int c = 0; c < a.C; c++) st.add(to_float(x[c * a.inner]));
  const float lse = st.lse();
  const int64_t t = a.target[at];
  a.log_probs[at] = target_log_prob(a, t, lse, t >= 0 && t < a.C ? to_float(x[t * a.inner]) : 0.f);
  a.entropy[at] = st.entropy();
  if (a.lse) a.lse[at] = lse;
  unsigned long long last = ~0ull;
  for (int j = 0; j < a.k; j++) {
    unsigned long long mine = 0;
    for (int c = 0; c < a.C; c++) {
      const unsigned long long q = candidate(to_float(x[c * a.inner]), c);
      if (q < last && q > mine) mine = q;
    }
    last = mine;
    const int c = candidate_index(mine);
    const int64_t to = (o * a.k + j) * a.inner + i;
    a.top_index[to] = c;
    a.top[to] = lse == -INFINITY ? -INFINITY : to_float(x[(int64_t)c * a.inner]) - lse;
  }
}

struct LogProbGradArgs {
  const void *x;
  const int64_t *target, *top_index;
  const float *lse, *entropy, *g, *h, *t;
  void *gx;
  int64_t outer, inner, x_stride, ignore_index, g_stride, h_stride;  // g_stride, h_stride: 1, or 0 for one value for all
  int C, k;
};

// What the elements of one distribution share.
struct RowGrad {
  float lse, entropy, g, h, all;  // all = g + sum t
  int64_t target;
  __device__ __forceinline__ float of(float x) const {
    const float d = x - lse, p = lse == -INFINITY ? 0.f : expf(d);
    return -p * (all + h * (fmaxf(d, -1e4f) + entropy));
  }
};
// `at`: the distribution's number, `o`, `i`: its parts.
__device__ __forceinline__ RowGrad row_grad(const LogProbGradArgs &a, int64_t at, int64_t o, int64_t i) {
  RowGrad r;
  r.lse = a.lse[at];
  r.entropy = a.entropy[at];
  r.target = a.target[at];
  const bool none = r.target == a.ignore_index || !a.g || r.lse == -INFINITY;
  r.g = none ? 0.f : r.target < 0 || r.target >= a.C ? NAN : a.g[at * a.g_stride];
  r.h = a.h ? a.h[at * a.h_stride] : 0.f;
  r.all = r.g;
  if (a.t && r.lse != -INFINITY)
    for (int j = 0; j < a.k; j++) r.all += a.t[(o * a.k + j) * a.inner + i];
  return r;
}
// The class c's own gradients: the target's, and those of the most probable classes.
__device__ __forceinline__ float own_grad(const LogProbGradArgs &a, const RowGrad &r, int64_t o, int64_t i, int c) {
  float v = c == r.target ? r.g : 0.f;
  if (a.t && r.lse != -INFINITY)
    for (int j = 0; j < a.k; j++) {
      const int64_t at = (o * a.k + j) * a.inner + i;
      if (a.top_index[at] == c) v += a.t[at];
    }
  return v;
}

template <typename T> __global__ void __launch_bounds__(256) log_probs_rows_grad_kernel(LogProbGradArgs a) {
  const int64_t row = blockIdx.x;
  const T *x = (const T *)a.x + row * a.x_stride;
  T *gx = (T *)a.gx + row * a.C;
  const RowGrad r = row_grad(a, row, row, 0);
  for (int c = threadIdx.x; c < a.C; c += 256) gx[c] = from_float<T>(r.of(to_float(x[c])) + own_grad(a, r, row, 0, c));
}

template <typename T> __global__ void __launch_bounds__(256) log_probs_planes_grad_kernel(LogProbGradArgs a) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= a.outer * a.inner) return;
  const int64_t o = at / a.inner, i = at % a.inner, base = o * a.C * a.inner + i;
  const RowGrad r = row_grad(a, at, o, i);
  for (int c = 0; c < a.C; c++)
    ((T *)a.gx)[base + c * a.inner] = from_float<T>(r.of(to_float(((const T *)a.x)[base + c * a.inner])) + own_grad(a, r, o, i, c));
}

inline int log_probs_sizes(int64_t outer, int64_t C, int64_t inner, int64_t k) {
  if (outer < 0 || C < 1 || inner < 1 || k < 0 || k > C) return SPH_ERR_INVALID_ARGUMENT;
  if (C >= ((int64_t)1 << 30) || outer >= ((int64_t)1 << 31) || inner >= ((int64_t)1 << 31)) return SPH_ERR_TOO_LARGE;
  if (outer > 0 && inner > (((int64_t)1 << 38) / outer)) return SPH_ERR_TOO_LARGE;
  return SPH_OK;
}

}  // namespace sph

using namespace sph;

extern "C" int sph_token_log_probs_forward(const void *x, const int64_t *target, float *log_probs, float *entropy, float *lse,
                                           float *top, int64_t *top_index, int64_t outer, int64_t C, int64_t inner, int64_t x_stride,
                                           int64_t k, int64_t ignore_index, int dtype, void *stream) {
  SPH_RANGE("sph_token_log_probs_forward");
  if (!element_dtype(dtype)) return SPH_ERR_UNSUPPORTED;
  if (const int rc = log_probs_sizes(outer, C, inner, k)) return rc;
  if (outer == 0) return SPH_OK;
  if (!x || !target || !log_probs || !entropy || (k > 0 && (!top || !top_index)) || (inner == 1 && outer > 1 && x_stride < C))
    return SPH_ERR_INVALID_ARGUMENT;
  const LogProbArgs a{x, target, log_probs, entropy, lse, top, top_index, outer, inner, x_stride, ignore_index, (int)C, (int)k};
  cudaStream_t st = (cudaStream_t)stream;
  SPH_DISPATCH_ELEMENT(dtype, {
    if (inner == 1)
      log_probs_rows_kernel<T><<<(unsigned)outer, 256, 0, st>>>(a);
    else
      log_probs_planes_kernel<T><<<(unsigned)((outer * inner + 255) / 256), 256, 0, st>>>(a);
  });
  return launch_status();
}

extern "C" int sph_token_log_probs_backward(const void *x, const int64_t *target, const float *lse, const float *entropy,
                                            const int64_t *top_index, const float *g, int64_t g_stride, const float *h,
                                            int64_t h_stride, const float *t, void *gx, int64_t outer, int64_t C, int64_t inner,
                                            int64_t x_stride, int64_t k, int64_t ignore_index, int dtype, void *stream) {
  SPH_RANGE("sph_token_log_probs_backward");
  if (!element_dtype(dtype)) return SPH_ERR_UNSUPPORTED;
  if (const int rc = log_probs_sizes(outer, C, inner, k)) return rc;
  if (outer == 0) return SPH_OK;
  if (!x || !target || !lse || !entropy || !gx || (t && (k == 0 || !top_index)) || (inner == 1 && outer > 1 && x_stride < C) ||
      g_stride < 0 || g_stride > 1 || h_stride < 0 || h_stride > 1)
    return SPH_ERR_INVALID_ARGUMENT;
  const LogProbGradArgs a{x, target, top_index, lse, entropy, g, h, t, gx, outer, inner, x_stride, ignore_index, g_stride, h_stride,
                          (int)C, (int)k};
  cudaStream_t st = (cudaStream_t)stream;
  SPH_DISPATCH_ELEMENT(dtype, {
    if (inner == 1)
      log_probs_rows_grad_kernel<T><<<(unsigned)outer, 256, 0, st>>>(a);
    else
      log_probs_planes_grad_kernel<T><<<(unsigned)((outer * inner + 255) / 256), 256, 0, st>>>(a);
  });
  return launch_status();
}

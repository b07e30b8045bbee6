// Root-mean-square norm over the channels of rows (rows, C) or planes (outer, C, inner), with the residual's addition:
//
//     s = residual + x, rounded to the type it is stored in;  rstd = (mean_c s^2 + eps)^(-1/2);  y = s rstd w
//
// y in the data's type, or in e4m3 with one float32 scale per norm.  Backward, with g = dy w and u = s rstd:
//
//     dx = dresidual = rstd (g - u mean_c(g u)) + ds;   dw_c = sum over the norms of dy u
//
// Sums, means and rstd are float32; the only rounding on the way is that of s, which is an output itself, so that the
// gradient is that of the function computed.
#include "element.cuh"

namespace sph {

struct NormArgs {
  const void *x, *residual, *weight;
  void *sum, *out;
  float *scale, *rstd;
  int64_t outer, inner, x_stride, r_stride;  // strides of rows, in elements (planes are dense)
  int C;
  float eps, inv_c;
  bool weight_f32;
};

// One block per row (inner == 1).
template <typename T, bool E4M3> __global__ void __launch_bounds__(256) norm_rows_kernel(NormArgs a) {
  __shared__ float shared[8];
  const int64_t row = blockIdx.x;
  const T *x = (const T *)a.x + row * a.x_stride;
  const T *r = a.residual ? (const T *)a.residual + row * a.r_stride : nullptr;
  T *sum = (T *)a.sum + row * a.C;
  float sq = 0.f;
  for (int c = threadIdx.x; c < a.C; c += 256) {
    float v = to_float(x[c]);
    if (r) {
      const T s = from_float<T>(v + to_float(r[c]));
      sum[c] = s;
      v = to_float(s);
    }
    sq += v * v;
  }
  sq = block_join(sq, shared, [](float p, float q) { return p + q; });
  const float rstd = 1.f / sqrtf(sq * a.inv_c + a.eps);
  if (threadIdx.x == 0 && a.rstd) a.rstd[row] = rstd;
  const T *s = r ? sum : x;
  Scale sc{1.f, 1.f};
  if (E4M3) {
    float amax = 0.f;
    for (int c = threadIdx.x; c < a.C; c += 256)
      amax = max_nan(amax, fabsf(to_float(s[c]) * rstd * (a.weight ? load_weight<T>(a.weight, c, a.weight_f32) : 1.f)));
    amax = block_join(amax, shared, [](float p, float q) { return max_nan(p, q); });
    sc = Scale::of(amax);
    if (threadIdx.x == 0) a.scale[row] = sc.scale;
  }
  for (int c = threadIdx.x; c < a.C; c += 256) {
    const float y = to_float(s[c]) * rstd * (a.weight ? load_weight<T>(a.weight, c, a.weight_f32) : 1.f);
    if (E4M3)
      ((__nv_fp8_storage_t *)a.out)[row * a.C + c] = to_e4m3(y * sc.inverse);
    else
      ((T *)a.out)[row * a.C + c] = from_float<T>(y);
  }
}

// One thread per pixel.
template <typename T, bool E4M3> __global__ void __launch_bounds__(256) norm_planes_kernel(NormArgs a) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= a.outer * a.inner) return;
  const int64_t base = at / a.inner * a.C * a.inner + at % a.inner;
  const T *x = (const T *)a.x + base, *r = a.residual ? (const T *)a.residual + base : nullptr;
  T *sum = (T *)a.sum + base;
  float sq = 0.f;
  for (int c = 0; c < a.C; c++) {
    float v = to_float(x[c * a.inner]);
    if (r) {
      const T s = from_float<T>(v + to_float(r[c * a.inner]));
      sum[c * a.inner] = s;
      v = to_float(s);
    }
    sq += v * v;
  }
  const float rstd = 1.f / sqrtf(sq * a.inv_c + a.eps);
  if (a.rstd) a.rstd[at] = rstd;
  const T *s = r ? sum : x;
  Scale sc{1.f, 1.f};
  if (E4M3) {
    float amax = 0.f;
    for (int c = 0; c < a.C; c++)
      amax = max_nan(amax, fabsf(to_float(s[c * a.inner]) * rstd * (a.weight ? load_weight<T>(a.weight, c, a.weight_f32) : 1.f)));
    sc = Scale::of(amax);
    a.scale[at] = sc.scale;
  }
  for (int c = 0; c < a.C; c++) {
    const float y = to_float(s[c * a.inner]) * rstd * (a.weight ? load_weight<T>(a.weight, c, a.weight_f32) : 1.f);
    if (E4M3)
      ((__nv_fp8_storage_t *)a.out)[base + c * a.inner] = to_e4m3(y * sc.inverse);
    else
      ((T *)a.out)[base + c * a.inner] = from_float<T>(y);
  }
}

struct NormGradArgs {
  const void *gout, *gsum, *s, *weight;
  const float *rstd;
  void *gx, *gw;
  float *partial;  // (splits, C)
  int64_t outer, inner, s_stride;
  int C, splits;
  float inv_c;
  bool weight_f32;
};

template <typename T> __global__ void __launch_bounds__(256) norm_rows_grad_kernel(NormGradArgs a) {
  __shared__ float shared[8];
  const int64_t row = blockIdx.x;
  const T *s = (const T *)a.s + row * a.s_stride, *gy = (const T *)a.gout + row * a.C;
  const float rstd = a.rstd[row];
  float dot = 0.f;
  for (int c = threadIdx.x; c < a.C; c += 256)
    dot += to_float(gy[c]) * (a.weight ? load_weight<T>(a.weight, c, a.weight_f32) : 1.f) * (to_float(s[c]) * rstd);
  dot = block_join(dot, shared, [](float p, float q) { return p + q; }) * a.inv_c;
  for (int c = threadIdx.x; c < a.C; c += 256) {
    const float g = to_float(gy[c]) * (a.weight ? load_weight<T>(a.weight, c, a.weight_f32) : 1.f);
    float v = rstd * (g - to_float(s[c]) * rstd * dot);
    if (a.gsum) v += to_float(((const T *)a.gsum)[row * a.C + c]);
    ((T *)a.gx)[row * a.C + c] = from_float<T>(v);
  }
}

template <typename T> __global__ void __launch_bounds__(256) norm_planes_grad_kernel(NormGradArgs a) {
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= a.outer * a.inner) return;
  const int64_t base = at / a.inner * a.C * a.inner + at % a.inner;
  const T *s = (const T *)a.s + base, *gy = (const T *)a.gout + base;
  const float rstd = a.rstd[at];
  float dot = 0.f;
  for (int c = 0; c < a.C; c++)
    dot += to_float(gy[c * a.inner]) * (a.weight ? load_weight<T>(a.weight, c, a.weight_f32) : 1.f) * (to_float(s[c * a.inner]) * rstd);
  dot *= a.inv_c;
  for (int c = 0; c < a.C; c++) {
    const float g = to_float(gy[c * a.inner]) * (a.weight ? load_weight<T>(a.weight, c, a.weight_f32) : 1.f);
    float v = rstd * (g - to_float(s[c * a.inner]) * rstd * dot);
    if (a.gsum) v += to_float(((const T *)a.gsum)[base + c * a.inner]);
    ((T *)a.gx)[base + c * a.inner] = from_float<T>(v);
  }
}

// Weight gradient: a block of 32 x 8 sums a slice of the norms for 32 channels (rows) or one channel (planes).
template <typename T> __global__ void __launch_bounds__(256) norm_rows_weight_kernel(NormGradArgs a) {
  __shared__ float shared[8][32];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), part = threadIdx.x >> 5;
  float v = 0.f;
  if (c < a.C)
    for (int64_t row = (int64_t)blockIdx.y * 8 + part; row < a.outer; row += (int64_t)a.splits * 8)
      v += to_float(((const T *)a.gout)[row * a.C + c]) * (to_float(((const T *)a.s)[row * a.s_stride + c]) * a.rstd[row]);
  shared[part][threadIdx.x & 31] = v;
  __syncthreads();
  if (part == 0 && c < a.C) {
    for (int i = 1; i < 8; i++) v += shared[i][threadIdx.x];
    a.partial[(int64_t)blockIdx.y * a.C + c] = v;
  }
}

template <typename T> __global__ void __launch_bounds__(256) norm_planes_weight_kernel(NormGradArgs a) {
  __shared__ float shared[8];
  const int c = blockIdx.x;
  float v = 0.f;
  for (int64_t at = (int64_t)blockIdx.y * 256 + threadIdx.x; at < a.outer * a.inner; at += (int64_t)a.splits * 256) {
    const int64_t i = (at / a.inner * a.C + c) * a.inner + at % a.inner;
    v += to_float(((const T *)a.gout)[i]) * (to_float(((const T *)a.s)[i]) * a.rstd[at]);
  }
  v = block_join(v, shared, [](float p, float q) { return p + q; });
  if (threadIdx.x == 0) a.partial[(int64_t)blockIdx.y * a.C + c] = v;
}

template <typename T> __global__ void __launch_bounds__(256) norm_weight_reduce_kernel(NormGradArgs a) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.C) return;
  float v = 0.f;
  for (int i = 0; i < a.splits; i++) v += a.partial[(int64_t)i * a.C + c];
  store_weight<T>(a.gw, c, v, a.weight_f32);
}

// Slices of the norms that the weight gradient is summed in: enough blocks for the GPU, at least 64 norms each.
inline int norm_splits(int64_t outer, int64_t C, int64_t inner) {
  const int64_t blocks = inner == 1 ? (C + 31) / 32 : C, norms = outer * inner;
  const int64_t want = (148 * 8 + blocks - 1) / blocks, most = (norms + 63) / 64;
  return (int)(want < most ? (want < 1 ? 1 : want) : (most < 1 ? 1 : most));
}

inline int norm_sizes(int64_t outer, int64_t C, int64_t inner) {
  if (outer < 0 || C < 1 || inner < 1) return SPH_ERR_INVALID_ARGUMENT;
  if (C >= ((int64_t)1 << 30) || outer >= ((int64_t)1 << 31) || inner >= ((int64_t)1 << 31)) return SPH_ERR_TOO_LARGE;
  if (outer > 0 && inner > (((int64_t)1 << 38) / outer)) return SPH_ERR_TOO_LARGE;
  return SPH_OK;
}

}  // namespace sph

using namespace sph;

extern "C" int sph_rms_norm_forward(const void *x, const void *residual, const void *weight, void *sum, void *out, float *scale,
                                    float *rstd, int64_t outer, int64_t C, int64_t inner, int64_t x_stride, int64_t r_stride,
                                    double eps, int dtype, int weight_dtype, void *stream) {
  SPH_RANGE("sph_rms_norm_forward");
  if (!element_dtype(dtype) || (weight && weight_dtype != SPH_F32 && weight_dtype != dtype)) return SPH_ERR_UNSUPPORTED;
  if (const int rc = norm_sizes(outer, C, inner)) return rc;
  if (outer == 0) return SPH_OK;
  if (!x || !out || (residual != nullptr) != (sum != nullptr) || !(eps >= 0)) return SPH_ERR_INVALID_ARGUMENT;
  if (inner == 1 && (x_stride < (outer > 1 ? C : 0) || (residual && r_stride < (outer > 1 ? C : 0)))) return SPH_ERR_INVALID_ARGUMENT;
  const NormArgs a{x, residual, weight, sum, out, scale, rstd, outer, inner, x_stride, r_stride, (int)C, (float)eps, 1.f / (float)C,
                   weight_dtype == SPH_F32};
  cudaStream_t st = (cudaStream_t)stream;
  SPH_DISPATCH_ELEMENT(dtype, {
    if (inner == 1 && scale)
      norm_rows_kernel<T, true><<<(unsigned)outer, 256, 0, st>>>(a);
    else if (inner == 1)
      norm_rows_kernel<T, false><<<(unsigned)outer, 256, 0, st>>>(a);
    else if (scale)
      norm_planes_kernel<T, true><<<(unsigned)((outer * inner + 255) / 256), 256, 0, st>>>(a);
    else
      norm_planes_kernel<T, false><<<(unsigned)((outer * inner + 255) / 256), 256, 0, st>>>(a);
  });
  return launch_status();
}

extern "C" size_t sph_rms_norm_workspace_bytes(int64_t outer, int64_t C, int64_t inner) {
  if (norm_sizes(outer, C, inner) != SPH_OK) return 0;
  return sizeof(float) * (size_t)norm_splits(outer, C, inner) * (size_t)C;
}

extern "C" int sph_rms_norm_backward(const void *gout, const void *gsum, const void *s, const void *weight, const float *rstd,
                                     void *gx, void *gw, int64_t outer, int64_t C, int64_t inner, int64_t s_stride, int dtype,
                                     int weight_dtype, void *ws, size_t ws_bytes, void *stream) {
  SPH_RANGE("sph_rms_norm_backward");
  if (!element_dtype(dtype) || (weight && weight_dtype != SPH_F32 && weight_dtype != dtype)) return SPH_ERR_UNSUPPORTED;
  if (const int rc = norm_sizes(outer, C, inner)) return rc;
  if ((!gx && !gw) || (gw && !weight)) return SPH_ERR_INVALID_ARGUMENT;
  if (outer > 0 && (!gout || !s || !rstd || (inner == 1 && s_stride < (outer > 1 ? C : 0)))) return SPH_ERR_INVALID_ARGUMENT;
  if (gw && (!ws || ws_bytes < sph_rms_norm_workspace_bytes(outer, C, inner))) return SPH_ERR_WORKSPACE_TOO_SMALL;
  const NormGradArgs a{gout, gsum, s, weight, rstd, gx, gw, (float *)ws, outer, inner, s_stride, (int)C, norm_splits(outer, C, inner),
                       1.f / (float)C, weight_dtype == SPH_F32};
  cudaStream_t st = (cudaStream_t)stream;
  int launches = 0;
  SPH_DISPATCH_ELEMENT(dtype, {
    if (gx && outer > 0) {
      if (inner == 1)
        norm_rows_grad_kernel<T><<<(unsigned)outer, 256, 0, st>>>(a);
      else
        norm_planes_grad_kernel<T><<<(unsigned)((outer * inner + 255) / 256), 256, 0, st>>>(a);
      launches++;
    }
    if (gw) {
      if (inner == 1)
        norm_rows_weight_kernel<T><<<dim3((unsigned)cdiv(C, 32), a.splits), 256, 0, st>>>(a);
      else
        norm_planes_weight_kernel<T><<<dim3((unsigned)C, a.splits), 256, 0, st>>>(a);
      norm_weight_reduce_kernel<T><<<(unsigned)cdiv(C, 256), 256, 0, st>>>(a);
      launches += 2;
    }
  });
  return launch_status(launches);
}

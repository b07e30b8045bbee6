// Norms over the channels of planes, forward; see norm.cuh for the formulas, planes.cuh for how the planes are read.
#include "norm.cuh"
#include "planes.cuh"

namespace sph {

// HBM bounds it where planes are aligned: 16 x 256 x 128 x 256 float32 with a residual take 347 us (6.2 TB/s).  Odd planes are read
// and written one pixel at a time behind the copies and are bound by issue: 3 x 96 x 181 x 333 bf16 to 8 bits 23 us (2.3 TB/s).
template <typename T, bool E4M3, bool ADD, int MODE, int LOG, int U> __global__ void __launch_bounds__(kPlaneThreads, 4) norm_planes_kernel(NormArgs a, PlaneTile tile) {
  using L = Lane<T, MODE, LOG, U>;
  using G = Geometry<T, MODE, LOG, U>;
  constexpr int N = L::N;
  __shared__ float shared[2][kPlaneThreads * N];
  __shared__ float weight[kMostPlanes];
  constexpr int ACROSS = G::ACROSS;
  const int first = (threadIdx.x >> 5) & (ACROSS - 1);
  const Run<MODE, G::PIXELS> run(tile, blockIdx.x, a.outer, a.C, a.inner);
  T *s = (T *)plane_memory, *add = s + a.C * G::PITCH;
  copy_run<T, MODE, LOG, U>(s, (const T *)a.x, run);
  if (ADD) copy_run<T, MODE, LOG, U>(add, (const T *)a.residual, run);
  copies_end();
  keep_weights<T>(weight, a.weight, a.weight_f32, a.C);
  const L px(run, first);
  const int64_t step = ACROSS * a.inner, zero = MODE == kShifted ? run.offset(0) : 0;
  const Rows<T, MODE, LOG, U> mine(s, (const T *)a.x, zero, first, px.col, a.inner);
  const Rows<T, MODE, LOG, U> other(add, (const T *)(ADD ? a.residual : a.x), zero, first, px.col, a.inner);
  const int count = (a.C - first + ACROSS - 1) >> LOG;  // channels of this warp
  const float *w = weight + first;
  copies_wait<0>();
  __syncthreads();
  float v[N], most[N];  // sums of squares; largest |s w|
#pragma unroll
  for (int i = 0; i < N; i++) v[i] = most[i] = 0.f;
  int64_t plane = 0;
#pragma unroll 8
  for (int k = 0; k < count; k++, plane += step) {
    typename L::P q = L::load(mine(k));
    if (ADD) {
      const typename L::P o = L::load(other(k));
#pragma unroll
      for (int i = 0; i < N; i++) q.t[i] = from_float<T>(to_float(q.t[i]) + to_float(o.t[i]));
      L::keep(mine(k), q);
      px.store((T *)a.sum, plane, q);
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
      const float f = to_float(q.t[i]);
      v[i] = fmaf(f, f, v[i]);
      if (E4M3) most[i] = max_nan(most[i], fabsf(f * w[k * ACROSS]));
    }
  }
  plane_join<LOG>(v, shared[0], [](float p, float q) { return p + q; });
  if (E4M3) plane_join<LOG>(most, shared[1], [](float p, float q) { return max_nan(p, q); });
  float rstd[N], inverse[N];
#pragma unroll
  for (int i = 0; i < N; i++) {
    rstd[i] = 1.f / sqrtf(v[i] * a.inv_c + a.eps);
    if (first == 0 && px.in[i] && a.rstd) a.rstd[px.norm[i]] = rstd[i];
    if (E4M3) {
      const Scale sc = Scale::of(most[i], rstd[i]);
      if (first == 0 && px.in[i]) a.scale[px.norm[i]] = sc.scale;
      inverse[i] = sc.inverse;
    }
  }
  plane = 0;
#pragma unroll 8
  for (int k = 0; k < count; k++, plane += step) {
    typename L::P q = L::load(mine(k));
    float y[N];
#pragma unroll
    for (int i = 0; i < N; i++) y[i] = E4M3 ? to_float(q.t[i]) * w[k * ACROSS] * inverse[i] : to_float(q.t[i]) * rstd[i] * w[k * ACROSS];
    if (E4M3) {
      px.store_e4m3((__nv_fp8_storage_t *)a.out, plane, y);
    } else {
#pragma unroll
      for (int i = 0; i < N; i++) q.t[i] = from_float<T>(y[i]);
      px.store((T *)a.out, plane, q);
    }
  }
}

template <typename T, bool E4M3> void norm_planes_launch(const NormArgs &a, cudaStream_t st) {
  const Mode mode = plane_mode<T>(a.C, a.inner, planes_aligned<T>(a.inner, {a.x, a.residual, a.sum, a.out}));
  SPH_DISPATCH_PLANES(mode, a.C, {
    const PlaneTile tile = PlaneTile::of<G, MODE>(a.outer, a.inner);
    if (a.residual)
      plane_launch<G, T>(norm_planes_kernel<T, E4M3, true, MODE, LOG, U>, a, tile, 2, (unsigned)tile.runs, st);
    else
      plane_launch<G, T>(norm_planes_kernel<T, E4M3, false, MODE, LOG, U>, a, tile, 1, (unsigned)tile.runs, st);
  })
}

void norm_planes_forward(const NormArgs &a, int dtype, cudaStream_t st) {
  SPH_DISPATCH_ELEMENT(dtype, {
    if (a.scale)
      norm_planes_launch<T, true>(a, st);
    else
      norm_planes_launch<T, false>(a, st);
  });
}

}  // namespace sph

// Norms over the channels of planes, backward; see norm.cuh for the formulas, planes.cuh for how the planes are read.
#include "norm.cuh"
#include "planes.cuh"

namespace sph {

// Backward: the blocks walk over the runs of pixels; a warp's channels, up to K, stay the same, and its lanes keep their parts of
// the weight gradients in registers.  16 x 256 x 128 x 256 float32 with both output gradients take 345 us (6.2 TB/s), HBM's rate;
// with addresses and weights from memory in the loops, 81 instructions a value instead of about 30, 457.
template <typename T, int K, bool ADD, int MODE, int LOG, int U>
__global__ void __launch_bounds__(kPlaneThreads, K <= 32 ? 3 : 2) norm_planes_grad_kernel(NormGradArgs a, PlaneTile tile) {
  using L = Lane<T, MODE, LOG, U>;
  using G = Geometry<T, MODE, LOG, U>;
  constexpr int N = L::N, ACROSS = G::ACROSS;
  __shared__ float shared[2][kPlaneThreads * N];
  __shared__ float weight[kMostPlanes];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, first = warp & (ACROSS - 1);
  const int mine = (a.C - first + ACROSS - 1) >> LOG;  // channels of this warp
  T *s = (T *)plane_memory, *g = s + a.C * G::PITCH, *add = g + a.C * G::PITCH;
  float gw[K];
#pragma unroll
  for (int k = 0; k < K; k++) gw[k] = 0.f;
  keep_weights<T>(weight, a.weight, a.weight_f32, a.C);
  const int64_t step = ACROSS * a.inner;
  int turn = 0;
  for (int64_t index = blockIdx.x; index < tile.runs; index += gridDim.x, turn ^= 1) {
    const Run<MODE, G::PIXELS> run(tile, index, a.outer, a.C, a.inner);
    copy_run<T, MODE, LOG, U>(s, (const T *)a.s, run);
    copy_run<T, MODE, LOG, U>(g, (const T *)a.gout, run);
    copies_end();
    if (ADD && a.gx) copy_run<T, MODE, LOG, U>(add, (const T *)a.gsum, run);
    copies_end();
    const L px(run, first);
    float rstd[N], dot[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
      rstd[i] = px.in[i] ? a.rstd[px.norm[i]] : 0.f;
      dot[i] = 0.f;
    }
    const int64_t zero = MODE == kShifted ? run.offset(0) : 0;
    using R = Rows<T, MODE, LOG, U>;
    const R sp(s, (const T *)a.s, zero, first, px.col, a.inner), gp(g, (const T *)a.gout, zero, first, px.col, a.inner),
        ap(add, (const T *)(ADD ? a.gsum : a.gout), zero, first, px.col, a.inner);
    const auto take = [&](int k) {
      const typename L::P p = L::load(sp(k)), q = L::load(gp(k));
      const float w = weight[first + k * ACROSS];
#pragma unroll
      for (int i = 0; i < N; i++) {
        const float gu = to_float(q.t[i]) * (to_float(p.t[i]) * rstd[i]);
        gw[k] += px.in[i] ? gu : 0.f;
        dot[i] = fmaf(gu, w, dot[i]);
      }
    };
    copies_wait<1>();
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; k += 8) {
      if (k + 8 <= mine) {
#pragma unroll
        for (int j = 0; j < 8; j++) take(k + j);
      } else if (k < mine) {
#pragma unroll
        for (int j = 0; j < 7; j++)
          if (k + j < mine) take(k + j);
      }
    }
    if (a.gx) {
      plane_join<LOG>(dot, shared[turn], [](float p, float q) { return p + q; });
#pragma unroll
      for (int i = 0; i < N; i++) dot[i] *= -rstd[i] * rstd[i] * a.inv_c;
      copies_wait<0>();
      if (ADD) __syncthreads();
      const float *wp = weight + first;
      int64_t plane = 0;
      const auto give = [&](int k) {
        typename L::P p = L::load(sp(k)), q = L::load(gp(k)), r;
        if (ADD) r = L::load(ap(k));
        const float w = wp[k * ACROSS];
#pragma unroll
        for (int i = 0; i < N; i++) {
          const float v = fmaf(to_float(q.t[i]) * w, rstd[i], to_float(p.t[i]) * dot[i]);
          p.t[i] = from_float<T>(ADD ? v + to_float(r.t[i]) : v);
        }
        px.store((T *)a.gx, plane, p);
        plane += step;
      };
      int k = 0;
      for (; k + 8 <= mine; k += 8) {
#pragma unroll
        for (int j = 0; j < 8; j++) give(k + j);
      }
#pragma unroll
      for (int j = 0; j < 7; j++)
        if (k + j < mine) give(k + j);
    }
    __syncthreads();  // everybody is done with the run
  }
  if (!a.gw) return;
  float *sums = &shared[0][0];  // (warp, k): 8 K floats
#pragma unroll
  for (int k = 0; k < K; k++) {
    const float v = warp_sum(gw[k]);
    if (lane == 0) sums[warp * K + k] = v;
  }
  __syncthreads();
  for (int c = threadIdx.x; c < a.C; c += kPlaneThreads) {
    float v = 0.f;
#pragma unroll
    for (int w = c & (ACROSS - 1); w < kPlaneWarps; w += ACROSS) v += sums[w * K + (c >> LOG)];
    a.partial[(int64_t)blockIdx.x * a.C + c] = v;
  }
}

template <typename T, int K, int MODE, int LOG, int U> void norm_planes_grad_launch(NormGradArgs &a, cudaStream_t st) {
  using G = Geometry<T, MODE, LOG, U>;
  const PlaneTile tile = PlaneTile::of<G, MODE>(a.outer, a.inner);
  // as many blocks as are on the SMs at once: three by their registers, or what shared memory leaves room for
  const int fit = 225 * 1024 / ((int)sizeof(T) * a.C * G::PITCH * (a.gsum ? 3 : 2) + 6 * 1024 + 1024);
  a.splits = (int)std::min<int64_t>(a.splits, std::min<int64_t>(tile.runs, 148 * (fit >= 3 && K <= 32 ? 3 : fit >= 2 ? 2 : 1)));
  if (a.gsum)
    plane_launch<G, T>(norm_planes_grad_kernel<T, K, true, MODE, LOG, U>, a, tile, 3, a.splits, st);
  else
    plane_launch<G, T>(norm_planes_grad_kernel<T, K, false, MODE, LOG, U>, a, tile, 2, a.splits, st);
}

void norm_planes_backward(NormGradArgs &a, int dtype, cudaStream_t st) {
  SPH_DISPATCH_ELEMENT(dtype, {
    const Mode mode = plane_mode<T>(a.C, a.inner, planes_aligned<T>(a.inner, {a.s, a.gout, a.gsum, a.gx}));
    SPH_DISPATCH_PLANES(mode, a.C, {
      if constexpr (U == 2)
        norm_planes_grad_launch<T, kTwice / 8, MODE, LOG, U>(a, st);
      else if constexpr (LOG == 0)
        norm_planes_grad_launch<T, kAlone, MODE, LOG, U>(a, st);
      else if (a.C <= 256)
        norm_planes_grad_launch<T, 32, MODE, LOG, U>(a, st);
      else
        norm_planes_grad_launch<T, 64, MODE, LOG, U>(a, st);
    })
  });
}

}  // namespace sph

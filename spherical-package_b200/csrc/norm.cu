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

#include <initializer_list>

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
template <typename T, bool E4M3> __global__ void __launch_bounds__(256) norm_long_rows_kernel(NormArgs a) {
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
template <typename T, bool E4M3> __global__ void __launch_bounds__(256) norm_deep_planes_kernel(NormArgs a) {
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

template <typename T> __global__ void __launch_bounds__(256) norm_long_rows_grad_kernel(NormGradArgs a) {
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

template <typename T> __global__ void __launch_bounds__(256) norm_deep_planes_grad_kernel(NormGradArgs a) {
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
template <typename T> __global__ void __launch_bounds__(256) norm_long_rows_weight_kernel(NormGradArgs a) {
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

template <typename T> __global__ void __launch_bounds__(256) norm_deep_planes_weight_kernel(NormGradArgs a) {
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

// Sums of the partial weight gradients: 32 channels a block, eight threads over the splits of each.
template <typename T> __global__ void __launch_bounds__(256) norm_weight_reduce_kernel(NormGradArgs a) {
  __shared__ float shared[8][32];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (c < a.C)
    for (int i = part; i < a.splits; i += 8) v += a.partial[(int64_t)i * a.C + c];
  shared[part][lane] = v;
  __syncthreads();
  if (part == 0 && c < a.C) {
    for (int i = 1; i < 8; i++) v += shared[i][lane];
    store_weight<T>(a.gw, c, v, a.weight_f32);
  }
}

// ---- rows in registers -----------------------------------------------------------------------------------------------
// N neighbouring elements: 16 bytes of a row where every row of every tensor starts on a 16-byte boundary, else one.
template <typename T, int N> struct Piece {
  T t[N];
  __device__ __forceinline__ void load(const T *p) {
    if constexpr (N == 1) {
      t[0] = *p;
    } else {
      union { uint4 u; T t[N]; } q;
      q.u = *(const uint4 *)p;
#pragma unroll
      for (int i = 0; i < N; i++) t[i] = q.t[i];
    }
  }
  __device__ __forceinline__ void store(T *p) const {
    if constexpr (N == 1) {
      *p = t[0];
    } else {
      union { uint4 u; T t[N]; } q;
#pragma unroll
      for (int i = 0; i < N; i++) q.t[i] = t[i];
      *(uint4 *)p = q.u;
    }
  }
};
template <int N> __device__ __forceinline__ void store_e4m3(__nv_fp8_storage_t *p, const float (&v)[N]) {
  if constexpr (N == 1) {
    *p = to_e4m3(v[0]);
  } else {
    unsigned q[N / 4];
#pragma unroll
    for (int i = 0; i < N / 4; i++)
      q[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i], v[4 * i + 1]), __NV_SATFINITE, __NV_E4M3) |
             (unsigned)__nv_cvt_float2_to_fp8x2(make_float2(v[4 * i + 2], v[4 * i + 3]), __NV_SATFINITE, __NV_E4M3) << 16;
    if constexpr (N == 8) *(uint2 *)p = make_uint2(q[0], q[1]);
    else *(unsigned *)p = q[0];
  }
}
// The N weights from channel c on, as floats.
template <typename T, int N> __device__ __forceinline__ void load_weights(const void *w, int c, bool f32, float (&v)[N]) {
  if (!w) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = 1.f;
  } else if (f32) {
    if constexpr (N == 1) {
      v[0] = __ldg((const float *)w + c);
    } else {
#pragma unroll
      for (int i = 0; i < N / 4; i++) {
        const float4 q = __ldg((const float4 *)((const float *)w + c) + i);
        v[4 * i] = q.x, v[4 * i + 1] = q.y, v[4 * i + 2] = q.z, v[4 * i + 3] = q.w;
      }
    }
  } else {
    Piece<T, N> p;
    p.load((const T *)w + c);
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = to_float(p.t[i]);
  }
}

// Joins over the threads of a row: a warp, or the whole block (`shared`: 32 floats, not those of the join before).
template <bool WARP, class F> __device__ __forceinline__ float row_join(float v, float *shared, F f, float none) {
  v = warp_join(v, f);
  if (WARP) return v;
  const int lane = threadIdx.x & 31;
  if (lane == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_join(lane < (int)(blockDim.x >> 5) ? shared[lane] : none, f);
}
template <bool WARP> __device__ __forceinline__ float row_sum(float v, float *shared) {
  return row_join<WARP>(v, shared, [](float p, float q) { return p + q; }, 0.f);
}

// A row is held by a warp (WARP) or by a block, E elements a thread in pieces of N: every tensor is read and written once.
template <typename T, bool E4M3, int N, int E, bool WARP> __global__ void __launch_bounds__(WARP ? 256 : 512) norm_rows_kernel(NormArgs a) {
  constexpr int V = E / N;
  __shared__ float shared[2][32];
  const int threads = WARP ? 32 : (int)blockDim.x, thread = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int64_t row = WARP ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
  if (WARP && row >= a.outer) return;
  const T *x = (const T *)a.x + row * a.x_stride, *r = a.residual ? (const T *)a.residual + row * a.r_stride : nullptr;
  Piece<T, N> s[V], add[V];
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int c = (thread + i * threads) * N;
    if (c < a.C) {
      s[i].load(x + c);
      if (r) add[i].load(r + c);
    }
  }
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int c = (thread + i * threads) * N;
    if (c < a.C) {
      if (r) {
#pragma unroll
        for (int j = 0; j < N; j++) s[i].t[j] = from_float<T>(to_float(s[i].t[j]) + to_float(add[i].t[j]));
        s[i].store((T *)a.sum + row * a.C + c);
      }
#pragma unroll
      for (int j = 0; j < N; j++) sq = fmaf(to_float(s[i].t[j]), to_float(s[i].t[j]), sq);
    }
  }
  const float rstd = 1.f / sqrtf(row_sum<WARP>(sq, shared[0]) * a.inv_c + a.eps);
  if (thread == 0 && a.rstd) a.rstd[row] = rstd;
  Scale sc{1.f, 1.f};
  if (E4M3) {
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < V; i++) {
      const int c = (thread + i * threads) * N;
      if (c < a.C) {
        float w[N];
        load_weights<T, N>(a.weight, c, a.weight_f32, w);
#pragma unroll
        for (int j = 0; j < N; j++) amax = max_nan(amax, fabsf(to_float(s[i].t[j]) * rstd * w[j]));
      }
    }
    sc = Scale::of(row_join<WARP>(amax, shared[1], [](float p, float q) { return max_nan(p, q); }, 0.f));
    if (thread == 0) a.scale[row] = sc.scale;
  }
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int c = (thread + i * threads) * N;
    if (c < a.C) {
      float y[N];
      load_weights<T, N>(a.weight, c, a.weight_f32, y);
#pragma unroll
      for (int j = 0; j < N; j++) y[j] = to_float(s[i].t[j]) * rstd * y[j];
      if (E4M3) {
#pragma unroll
        for (int j = 0; j < N; j++) y[j] *= sc.inverse;
        store_e4m3<N>((__nv_fp8_storage_t *)a.out + row * a.C + c, y);
      } else {
#pragma unroll
        for (int j = 0; j < N; j++) s[i].t[j] = from_float<T>(y[j]);
        s[i].store((T *)a.out + row * a.C + c);
      }
    }
  }
}

// Backward: the blocks walk over the rows; a thread's channels stay the same, and their weight gradients in its registers.
template <typename T, int N, int E, bool WARP> __global__ void __launch_bounds__(WARP ? 256 : 512) norm_rows_grad_kernel(NormGradArgs a) {
  constexpr int V = E / N;
  __shared__ float shared[2][32];
  __shared__ float sums[WARP ? 1024 : 1];
  const int threads = WARP ? 32 : (int)blockDim.x, thread = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int64_t first = WARP ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x, step = WARP ? (int64_t)gridDim.x * 8 : gridDim.x;
  float gw[V][N];
#pragma unroll
  for (int i = 0; i < V; i++)
#pragma unroll
    for (int j = 0; j < N; j++) gw[i][j] = 0.f;
  int turn = 0;
  for (int64_t row = first; row < a.outer; row += step, turn ^= 1) {
    const T *s_at = (const T *)a.s + row * a.s_stride, *g_at = (const T *)a.gout + row * a.C, *p_at = (const T *)a.gsum + row * a.C;
    Piece<T, N> s[V], g[V], p[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
      const int c = (thread + i * threads) * N;
      if (c < a.C) {
        s[i].load(s_at + c);
        g[i].load(g_at + c);
        if (a.gsum && a.gx) p[i].load(p_at + c);
      }
    }
    const float rstd = a.rstd[row];
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < V; i++) {
      const int c = (thread + i * threads) * N;
      if (c < a.C) {
        float w[N];
        load_weights<T, N>(a.weight, c, a.weight_f32, w);
#pragma unroll
        for (int j = 0; j < N; j++) {
          const float gu = to_float(g[i].t[j]) * (to_float(s[i].t[j]) * rstd);
          gw[i][j] += gu;
          dot = fmaf(gu, w[j], dot);
        }
      }
    }
    if (!a.gx) continue;
    dot = row_sum<WARP>(dot, shared[turn]) * a.inv_c;
#pragma unroll
    for (int i = 0; i < V; i++) {
      const int c = (thread + i * threads) * N;
      if (c < a.C) {
        float w[N];
        load_weights<T, N>(a.weight, c, a.weight_f32, w);
#pragma unroll
        for (int j = 0; j < N; j++) {
          float v = rstd * (to_float(g[i].t[j]) * w[j] - to_float(s[i].t[j]) * rstd * dot);
          if (a.gsum) v += to_float(p[i].t[j]);
          s[i].t[j] = from_float<T>(v);
        }
        s[i].store((T *)a.gx + row * a.C + c);
      }
    }
  }
  if (!a.gw) return;
  if (WARP) {  // the eight warps' sums, one after the other
    for (int c = threadIdx.x; c < a.C; c += 256) sums[c] = 0.f;
    for (int w = 0; w < 8; w++) {
      __syncthreads();
      if ((int)(threadIdx.x >> 5) == w)
#pragma unroll
        for (int i = 0; i < V; i++)
#pragma unroll
          for (int j = 0; j < N; j++) {
            const int c = (thread + i * 32) * N + j;
            if (c < a.C) sums[c] += gw[i][j];
          }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.C; c += 256) a.partial[(int64_t)blockIdx.x * a.C + c] = sums[c];
  } else {
#pragma unroll
    for (int i = 0; i < V; i++)
#pragma unroll
      for (int j = 0; j < N; j++) {
        const int c = (thread + i * threads) * N + j;
        if (c < a.C) a.partial[(int64_t)blockIdx.x * a.C + c] = gw[i][j];
      }
  }
}

// ---- planes through shared memory ------------------------------------------------------------------------------------
// A block of 8 warps takes a run of pixels with all their channels into shared memory by asynchronous copies, so that every
// tensor is read and written once; two or three blocks a SM copy and compute in turn.  `across` warps share the channels of a
// unit of 128 bytes a channel (32 float32 or 64 16-bit pixels), the others have further units; what a norm needs of all its
// channels is joined through shared memory.
template <typename T> struct Pixels {  // a lane's: 4 bytes of a channel
  static constexpr int N = 4 / (int)sizeof(T);
  union {
    unsigned w;
    T t[N];
  };
};
constexpr int kPlaneWarps = 8, kPlaneThreads = 32 * kPlaneWarps;
struct PlaneTile {
  int across_log;  // log2 of the warps that share a unit's channels
  FastDiv plane;   // pixels of a plane, where all pixels are fewer than 2^31
  bool small, wide;  // wide: 16 bytes may be copied at once
  // K: channels a warp may have.
  static PlaneTile of(int64_t outer, int64_t C, int64_t inner, int K) {
    PlaneTile t;
    t.across_log = 0;
    while (t.across_log < 3 && ((int64_t)K << t.across_log) < C) t.across_log++;
    t.small = outer * inner < ((int64_t)1 << 31);
    t.plane = FastDiv::make(t.small ? (unsigned)inner : 1u);
    t.wide = false;
    return t;
  }
  __host__ __device__ __forceinline__ int units() const { return kPlaneWarps >> across_log; }
  __host__ __device__ __forceinline__ int pixels(int n) const { return units() * 32 * n; }
  // Offset of channel 0 of a pixel.
  __device__ __forceinline__ int64_t offset(int64_t at, int64_t C, int64_t inner) const {
    const int64_t o = small ? (int64_t)plane.div((unsigned)at) : at / inner;
    return o * C * inner + (at - o * inner);
  }
};

__device__ __forceinline__ void copy_16(void *to, const void *from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_4(void *to, const void *from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }

// Copies the run of pixels from `start` on, all C channels, to [channel][pixels of the tile].
template <typename T> __device__ __forceinline__ void copy_tile(T *to, const T *from, int64_t start, int64_t total, int C, int64_t inner, const PlaneTile &tile) {
  const int pixels = tile.pixels(Pixels<T>::N);
  constexpr int N = 16 / (int)sizeof(T);
  if (tile.wide) {
    const int cols = pixels / N, col = (threadIdx.x & (cols - 1)) * N, rows = kPlaneThreads / cols;
    if (start + col >= total) return;
    const T *p = from + tile.offset(start + col, C, inner);
    for (int c = threadIdx.x / cols; c < C; c += rows) copy_16(to + c * pixels + col, p + c * inner);
  } else {  // a thread a pixel: of 32, 64, ... 512
    for (int col = threadIdx.x & (pixels - 1); col < pixels; col += kPlaneThreads) {
      if (start + col >= total) return;
      const T *p = from + tile.offset(start + col, C, inner);
      const int rows = pixels < kPlaneThreads ? kPlaneThreads / pixels : 1;
      if constexpr (sizeof(T) == 4) {
        for (int c = threadIdx.x / pixels; c < C; c += rows) copy_4(to + c * pixels + col, p + c * inner);
      } else {
#pragma unroll 8
        for (int c = threadIdx.x / pixels; c < C; c += rows) to[c * pixels + col] = p[c * inner];
      }
    }
  }
}

// A lane's pixels in the tile, and where they are in the tensors.
template <typename T> struct LanePixels {
  static constexpr int N = Pixels<T>::N;
  int64_t at, off[N];
  int col;
  bool in[N], pair;  // pair: both (or the one) in bounds, neighbours, and 4 bytes may be written at once
  __device__ __forceinline__ LanePixels(int64_t start, int64_t total, int C, int64_t inner, const PlaneTile &tile) {
    col = ((threadIdx.x >> 5 >> tile.across_log) * 32 + (threadIdx.x & 31)) * N;
    at = start + col;
#pragma unroll
    for (int i = 0; i < N; i++) {
      in[i] = at + i < total;
      off[i] = in[i] ? tile.offset(at + i, C, inner) : 0;
    }
    pair = in[0] && (N == 1 || tile.wide);
  }
  __device__ __forceinline__ void store(T *to, int64_t plane, const Pixels<T> &v) const {
    if (pair) {
      *(unsigned *)(to + off[0] + plane) = v.w;
    } else {
#pragma unroll
      for (int i = 0; i < N; i++)
        if (in[i]) to[off[i] + plane] = v.t[i];
    }
  }
};

// Joins a value of each of the lane's pixels over the warps that share them.  `shared`: 8 x 32 x N floats.
template <int N, class F> __device__ __forceinline__ void plane_join(float (&v)[N], float *shared, int across_log, F f) {
  if (across_log == 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = 1 << across_log, mates = warp & ~(n - 1);
#pragma unroll
  for (int i = 0; i < N; i++) shared[(warp * N + i) * 32 + lane] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; i++) v[i] = shared[(mates * N + i) * 32 + lane];
  for (int w = 1; w < n; w++)
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = f(v[i], shared[((mates + w) * N + i) * 32 + lane]);
}

extern __shared__ __align__(16) unsigned char plane_memory[];

template <typename T, bool E4M3, bool ADD> __global__ void __launch_bounds__(kPlaneThreads, 3) norm_planes_kernel(NormArgs a, PlaneTile tile) {
  constexpr int N = Pixels<T>::N;
  __shared__ float shared[2][kPlaneThreads * N];
  const int pixels = tile.pixels(N), across = 1 << tile.across_log, first = (threadIdx.x >> 5) & (across - 1);
  const int64_t total = a.outer * a.inner, start = (int64_t)blockIdx.x * pixels;
  T *s = (T *)plane_memory, *add = s + (int64_t)a.C * pixels;
  copy_tile(s, (const T *)a.x, start, total, a.C, a.inner, tile);
  if (ADD) copy_tile(add, (const T *)a.residual, start, total, a.C, a.inner, tile);
  copies_end();
  const LanePixels<T> px(start, total, a.C, a.inner, tile);
  copies_wait<0>();
  __syncthreads();
  float v[N];
#pragma unroll
  for (int i = 0; i < N; i++) v[i] = 0.f;
#pragma unroll 4
  for (int c = first; c < a.C; c += across) {
    Pixels<T> p;
    p.w = *(const unsigned *)(s + c * pixels + px.col);
    if (ADD) {
      Pixels<T> q;
      q.w = *(const unsigned *)(add + c * pixels + px.col);
#pragma unroll
      for (int i = 0; i < N; i++) p.t[i] = from_float<T>(to_float(p.t[i]) + to_float(q.t[i]));
      *(unsigned *)(s + c * pixels + px.col) = p.w;
      px.store((T *)a.sum, c * a.inner, p);
    }
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = fmaf(to_float(p.t[i]), to_float(p.t[i]), v[i]);
  }
  plane_join<N>(v, shared[0], tile.across_log, [](float p, float q) { return p + q; });
  float rstd[N], scale[N];
#pragma unroll
  for (int i = 0; i < N; i++) {
    rstd[i] = 1.f / sqrtf(v[i] * a.inv_c + a.eps);
    if (first == 0 && px.in[i] && a.rstd) a.rstd[px.at + i] = rstd[i];
  }
  if (E4M3) {
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = 0.f;
#pragma unroll 4
    for (int c = first; c < a.C; c += across) {
      const float w = a.weight ? load_weight<T>(a.weight, c, a.weight_f32) : 1.f;
      Pixels<T> p;
      p.w = *(const unsigned *)(s + c * pixels + px.col);
#pragma unroll
      for (int i = 0; i < N; i++) v[i] = max_nan(v[i], fabsf(to_float(p.t[i]) * rstd[i] * w));
    }
    plane_join<N>(v, shared[1], tile.across_log, [](float p, float q) { return max_nan(p, q); });
#pragma unroll
    for (int i = 0; i < N; i++) {
      const Scale sc = Scale::of(v[i]);
      scale[i] = sc.inverse;
      if (first == 0 && px.in[i]) a.scale[px.at + i] = sc.scale;
    }
  }
#pragma unroll 4
  for (int c = first; c < a.C; c += across) {
    const float w = a.weight ? load_weight<T>(a.weight, c, a.weight_f32) : 1.f;
    const int64_t plane = c * a.inner;
    Pixels<T> p;
    p.w = *(const unsigned *)(s + c * pixels + px.col);
    float y[N];
#pragma unroll
    for (int i = 0; i < N; i++) y[i] = to_float(p.t[i]) * rstd[i] * w;
    if (E4M3) {
      __nv_fp8_storage_t *out = (__nv_fp8_storage_t *)a.out;
#pragma unroll
      for (int i = 0; i < N; i++) y[i] *= scale[i];
      if (N == 2 && px.pair) {
        *(__nv_fp8x2_storage_t *)(out + px.off[0] + plane) = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[N - 1]), __NV_SATFINITE, __NV_E4M3);
      } else {
#pragma unroll
        for (int i = 0; i < N; i++)
          if (px.in[i]) out[px.off[i] + plane] = to_e4m3(y[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; i++) p.t[i] = from_float<T>(y[i]);
      px.store((T *)a.out, plane, p);
    }
  }
}

// Backward: the blocks walk over the runs of pixels; a warp's channels, up to K, stay the same, and its lanes keep their parts of
// the weight gradients in registers.
template <typename T, int K, bool ADD>
__global__ void __launch_bounds__(kPlaneThreads, K <= 32 ? 3 : 2) norm_planes_grad_kernel(NormGradArgs a, PlaneTile tile) {
  constexpr int N = Pixels<T>::N;
  __shared__ float shared[2][kPlaneThreads * N];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pixels = tile.pixels(N), across = 1 << tile.across_log, first = warp & (across - 1);
  const int64_t total = a.outer * a.inner;
  T *s = (T *)plane_memory, *g = s + (int64_t)a.C * pixels, *add = g + (int64_t)a.C * pixels;
  float gw[K];
#pragma unroll
  for (int k = 0; k < K; k++) gw[k] = 0.f;
  int turn = 0;
  for (int64_t start = (int64_t)blockIdx.x * pixels; start < total; start += (int64_t)gridDim.x * pixels, turn ^= 1) {
    copy_tile(s, (const T *)a.s, start, total, a.C, a.inner, tile);
    copy_tile(g, (const T *)a.gout, start, total, a.C, a.inner, tile);
    copies_end();
    if (ADD && a.gx) copy_tile(add, (const T *)a.gsum, start, total, a.C, a.inner, tile);
    copies_end();
    const LanePixels<T> px(start, total, a.C, a.inner, tile);
    float rstd[N], dot[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
      rstd[i] = px.in[i] ? a.rstd[px.at + i] : 0.f;
      dot[i] = 0.f;
    }
    copies_wait<1>();
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; k++) {
      const int c = first + (k << tile.across_log);
      if (c < a.C) {
        const float w = a.weight ? load_weight<T>(a.weight, c, a.weight_f32) : 1.f;
        Pixels<T> p, q;
        p.w = *(const unsigned *)(s + c * pixels + px.col);
        q.w = *(const unsigned *)(g + c * pixels + px.col);
#pragma unroll
        for (int i = 0; i < N; i++) {
          const float gu = px.in[i] ? to_float(q.t[i]) * (to_float(p.t[i]) * rstd[i]) : 0.f;
          gw[k] += gu;
          dot[i] = fmaf(gu, w, dot[i]);
        }
      }
    }
    if (a.gx) {
      plane_join<N>(dot, shared[turn], tile.across_log, [](float p, float q) { return p + q; });
#pragma unroll
      for (int i = 0; i < N; i++) dot[i] *= rstd[i] * a.inv_c;
      copies_wait<0>();
      if (ADD) __syncthreads();
#pragma unroll 4
      for (int c = first; c < a.C; c += across) {
        const float w = a.weight ? load_weight<T>(a.weight, c, a.weight_f32) : 1.f;
        Pixels<T> p, q, r;
        p.w = *(const unsigned *)(s + c * pixels + px.col);
        q.w = *(const unsigned *)(g + c * pixels + px.col);
        if (ADD) r.w = *(const unsigned *)(add + c * pixels + px.col);
#pragma unroll
        for (int i = 0; i < N; i++) {
          float v = rstd[i] * (to_float(q.t[i]) * w - to_float(p.t[i]) * dot[i]);
          if (ADD) v += to_float(r.t[i]);
          p.t[i] = from_float<T>(v);
        }
        px.store((T *)a.gx, c * a.inner, p);
      }
    }
    __syncthreads();  // everybody is done with the tile
  }
  if (!a.gw) return;
  float *sums = &shared[0][0];  // (warp, k): 8 K floats
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; k++) {
    const float v = warp_sum(gw[k]);
    if (lane == 0) sums[warp * K + k] = v;
  }
  __syncthreads();
  for (int c = threadIdx.x; c < a.C; c += kPlaneThreads) {
    const int k = c >> tile.across_log;
    float v = 0.f;
    for (int w = c & (across - 1); w < kPlaneWarps; w += across) v += sums[w * K + k];
    a.partial[(int64_t)blockIdx.x * a.C + c] = v;
  }
}

// Which kernel takes a call, and in how many blocks its weight gradient is summed.
enum NormPath { kLongRows, kWarpRows, kBlockRows, kPlanes, kDeepPlanes };
inline NormPath norm_path(int64_t C, int64_t inner) {
  return inner > 1 ? (C <= 512 ? kPlanes : kDeepPlanes) : C <= 1024 ? kWarpRows : C <= 16384 ? kBlockRows : kLongRows;
}
inline int norm_splits(int64_t outer, int64_t C, int64_t inner) {
  const int64_t norms = outer * inner;
  int64_t want, most;
  switch (norm_path(C, inner)) {
    case kWarpRows: want = 148 * 4, most = (norms + 7) / 8; break;
    case kBlockRows: want = 148 * 3, most = norms; break;
    case kPlanes: want = 148 * 2, most = (norms + 31) / 32; break;
    default: {
      const int64_t blocks = inner == 1 ? (C + 31) / 32 : C;  // enough blocks for the GPU, at least 64 norms each
      want = (148 * 8 + blocks - 1) / blocks, most = (norms + 63) / 64;
    }
  }
  const int64_t n = want < most ? want : most;
  return (int)(n < 1 ? 1 : n);
}

// Whether every row of a tensor starts on a 16-byte boundary.
inline bool rows_aligned(const void *p, int64_t stride, size_t size) {
  return (uintptr_t)p % 16 == 0 && stride * (int64_t)size % 16 == 0;
}

template <typename T, bool E4M3, int N, int E> void norm_rows_launch(const NormArgs &a, cudaStream_t st) {
  if (norm_path(a.C, 1) == kWarpRows)
    norm_rows_kernel<T, E4M3, N, E, true><<<(unsigned)((a.outer + 7) / 8), 256, 0, st>>>(a);
  else
    norm_rows_kernel<T, E4M3, N, E, false><<<(unsigned)a.outer, 32 * cdiv(a.C, 32 * E), 0, st>>>(a);
}
// Elements a thread holds: 32 a lane for up to 1024 in a warp; in blocks 8 where 512 threads are enough, 16, or 32.
template <typename T, bool E4M3, int N> void norm_rows_pick(const NormArgs &a, cudaStream_t st) {
  const int64_t per = norm_path(a.C, 1) == kWarpRows ? (a.C + 31) / 32 : (a.C + 511) / 512;
  if (per <= 8)
    norm_rows_launch<T, E4M3, N, 8>(a, st);
  else if (per <= 16)
    norm_rows_launch<T, E4M3, N, 16>(a, st);
  else
    norm_rows_launch<T, E4M3, N, 32>(a, st);
}

// Whether 16 bytes of a plane may be copied at once.
template <typename T> bool planes_aligned(int64_t inner, std::initializer_list<const void *> ps) {
  uintptr_t bits = (uintptr_t)inner * sizeof(T);
  for (const void *p : ps) bits |= (uintptr_t)p;
  return bits % 16 == 0;
}
// Launches a kernel over tiles of `tensors` tensors in shared memory.
template <typename T, class A> void plane_launch(void (*kernel)(A, PlaneTile), const A &a, const PlaneTile &tile, int tensors, unsigned blocks, cudaStream_t st) {
  const int bytes = (int)sizeof(T) * a.C * tile.pixels(Pixels<T>::N) * tensors;
  if (bytes > 32768) cudaFuncSetAttribute((const void *)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  kernel<<<blocks, kPlaneThreads, bytes, st>>>(a, tile);
}
template <typename T, bool E4M3> void norm_planes_launch(const NormArgs &a, cudaStream_t st) {
  PlaneTile tile = PlaneTile::of(a.outer, a.C, a.inner, 16);
  tile.wide = planes_aligned<T>(a.inner, {a.x, a.residual, a.sum, a.out});
  const int64_t pixels = tile.pixels(Pixels<T>::N);
  const unsigned blocks = (unsigned)((a.outer * a.inner + pixels - 1) / pixels);
  if (a.residual)
    plane_launch<T>(norm_planes_kernel<T, E4M3, true>, a, tile, 2, blocks, st);
  else
    plane_launch<T>(norm_planes_kernel<T, E4M3, false>, a, tile, 1, blocks, st);
}

template <typename T, bool E4M3> void norm_launch(const NormArgs &a, cudaStream_t st) {
  constexpr int N = 16 / (int)sizeof(T);
  switch (norm_path(a.C, a.inner)) {
    case kWarpRows:
    case kBlockRows:
      if (rows_aligned(a.x, a.x_stride, sizeof(T)) && a.C % N == 0 && rows_aligned(a.residual, a.r_stride, sizeof(T)) &&
          ((uintptr_t)a.sum % 16 | (uintptr_t)a.out % 16 | (uintptr_t)a.weight % 16) == 0)
        norm_rows_pick<T, E4M3, N>(a, st);
      else
        norm_rows_pick<T, E4M3, 1>(a, st);
      break;
    case kPlanes:
      norm_planes_launch<T, E4M3>(a, st);
      break;
    case kLongRows: norm_long_rows_kernel<T, E4M3><<<(unsigned)a.outer, 256, 0, st>>>(a); break;
    default: norm_deep_planes_kernel<T, E4M3><<<(unsigned)((a.outer * a.inner + 255) / 256), 256, 0, st>>>(a);
  }
}

template <typename T, int N, int E> void norm_rows_grad_launch(const NormGradArgs &a, cudaStream_t st) {
  if (norm_path(a.C, 1) == kWarpRows)
    norm_rows_grad_kernel<T, N, E, true><<<a.splits, 256, 0, st>>>(a);
  else
    norm_rows_grad_kernel<T, N, E, false><<<a.splits, 32 * cdiv(a.C, 32 * E), 0, st>>>(a);
}
template <typename T, int N> void norm_rows_grad_pick(const NormGradArgs &a, cudaStream_t st) {
  const int64_t per = norm_path(a.C, 1) == kWarpRows ? (a.C + 31) / 32 : (a.C + 511) / 512;
  if (per <= 8)
    norm_rows_grad_launch<T, N, 8>(a, st);
  else if (per <= 16)
    norm_rows_grad_launch<T, N, 16>(a, st);
  else
    norm_rows_grad_launch<T, N, 32>(a, st);
}
template <typename T, int K> void norm_planes_grad_launch(const NormGradArgs &a, cudaStream_t st) {
  PlaneTile tile = PlaneTile::of(a.outer, a.C, a.inner, 16);
  tile.wide = planes_aligned<T>(a.inner, {a.s, a.gout, a.gsum, a.gx});
  if (a.gsum)
    plane_launch<T>(norm_planes_grad_kernel<T, K, true>, a, tile, 3, a.splits, st);
  else
    plane_launch<T>(norm_planes_grad_kernel<T, K, false>, a, tile, 2, a.splits, st);
}

// Kernels launched.
template <typename T> int norm_grad_launch(const NormGradArgs &a, cudaStream_t st) {
  constexpr int N = 16 / (int)sizeof(T);
  int launches = 0;
  if (a.outer > 0) {
    launches = 1;
    switch (norm_path(a.C, a.inner)) {
      case kWarpRows:
      case kBlockRows:
        if (rows_aligned(a.s, a.s_stride, sizeof(T)) && a.C % N == 0 &&
            ((uintptr_t)a.gout % 16 | (uintptr_t)a.gsum % 16 | (uintptr_t)a.gx % 16 | (uintptr_t)a.weight % 16) == 0)
          norm_rows_grad_pick<T, N>(a, st);
        else
          norm_rows_grad_pick<T, 1>(a, st);
        break;
      case kPlanes:
        if (a.C <= 128)
          norm_planes_grad_launch<T, 16>(a, st);
        else if (a.C <= 256)
          norm_planes_grad_launch<T, 32>(a, st);
        else
          norm_planes_grad_launch<T, 64>(a, st);
        break;
      case kLongRows:
        if (a.gx) norm_long_rows_grad_kernel<T><<<(unsigned)a.outer, 256, 0, st>>>(a);
        if (a.gw) norm_long_rows_weight_kernel<T><<<dim3((unsigned)cdiv(a.C, 32), a.splits), 256, 0, st>>>(a);
        launches = (a.gx ? 1 : 0) + (a.gw ? 1 : 0);
        break;
      default:
        if (a.gx) norm_deep_planes_grad_kernel<T><<<(unsigned)((a.outer * a.inner + 255) / 256), 256, 0, st>>>(a);
        if (a.gw) norm_deep_planes_weight_kernel<T><<<dim3((unsigned)a.C, a.splits), 256, 0, st>>>(a);
        launches = (a.gx ? 1 : 0) + (a.gw ? 1 : 0);
    }
  }
  if (a.gw) {
    norm_weight_reduce_kernel<T><<<(unsigned)cdiv(a.C, 32), 256, 0, st>>>(a);
    launches++;
  }
  return launches;
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
    if (scale)
      norm_launch<T, true>(a, st);
    else
      norm_launch<T, false>(a, st);
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
  const NormGradArgs a{gout, gsum, s, weight, rstd, gx, gw, (float *)ws, outer, inner, s_stride, (int)C, outer > 0 ? norm_splits(outer, C, inner) : 0,
                       1.f / (float)C, weight_dtype == SPH_F32};
  cudaStream_t st = (cudaStream_t)stream;
  int launches = 0;
  SPH_DISPATCH_ELEMENT(dtype, launches = norm_grad_launch<T>(a, st));
  return launch_status(launches);
}

// Norms over rows and over planes of many channels; see norm.cuh for the formulas.
#include "norm.cuh"

namespace sph {

// One block per row (inner == 1), of any number of channels, one element a thread at a time: read twice, to 8 bits three times, all but
// the first time from L2.  Issue and few bytes on their way bound it: 1024 x 32768 bf16 with a residual take 162 us (1.7 TB/s), 64 rows
// of 32768 with gradients 190 us of latency.
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
    float most = 0.f;
    for (int c = threadIdx.x; c < a.C; c += 256)
      most = max_nan(most, fabsf(to_float(s[c]) * (a.weight ? load_weight<T>(a.weight, c, a.weight_f32) : 1.f)));
    most = block_join(most, shared, [](float p, float q) { return max_nan(p, q); });
    sc = Scale::of(most, rstd);
    if (threadIdx.x == 0) a.scale[row] = sc.scale;
  }
  for (int c = threadIdx.x; c < a.C; c += 256) {
    const float v = to_float(s[c]), w = a.weight ? load_weight<T>(a.weight, c, a.weight_f32) : 1.f;
    if (E4M3)
      ((__nv_fp8_storage_t *)a.out)[row * a.C + c] = to_e4m3(v * w * sc.inverse);
    else
      ((T *)a.out)[row * a.C + c] = from_float<T>(v * rstd * w);
  }
}

// One thread per pixel, for more than kMostPlanes channels: with three tensors in the backward pass those fill a block's shared memory
// (float32, 32 pixels: 221 KB).  Read as the long rows are.  Few pixels are few threads, whose chain of loads is all that counts:
// 8 x 1024 x 16 x 32 bf16 with a residual take 777 us forward and 560 backward, 16 blocks on 148 SMs.
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
    float most = 0.f;
    for (int c = 0; c < a.C; c++)
      most = max_nan(most, fabsf(to_float(s[c * a.inner]) * (a.weight ? load_weight<T>(a.weight, c, a.weight_f32) : 1.f)));
    sc = Scale::of(most, rstd);
    a.scale[at] = sc.scale;
  }
  for (int c = 0; c < a.C; c++) {
    const float v = to_float(s[c * a.inner]), w = a.weight ? load_weight<T>(a.weight, c, a.weight_f32) : 1.f;
    if (E4M3)
      ((__nv_fp8_storage_t *)a.out)[base + c * a.inner] = to_e4m3(v * w * sc.inverse);
    else
      ((T *)a.out)[base + c * a.inner] = from_float<T>(v * rstd * w);
  }
}

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

// Weight gradient of long rows and deep planes, which reads both tensors again: a block of 32 x 8 sums a slice of the norms for 32
// channels (rows) or one channel (planes).  8 x 1024 x 16 x 32 bf16: 22 us.
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

// Sums of the partial weight gradients: 32 channels a block, 32 threads over the splits of each.
template <typename T> __global__ void __launch_bounds__(1024) norm_weight_reduce_kernel(NormGradArgs a) {
  __shared__ float shared[32][33];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (c < a.C)
    for (int i = part; i < a.splits; i += 32) v += a.partial[(int64_t)i * a.C + c];
  shared[part][lane] = v;
  __syncthreads();
  v = warp_sum(shared[lane][part]);  // (a warp a channel)
  const int mine = blockIdx.x * 32 + part;
  if (lane == 0 && mine < a.C) store_weight<T>(a.gw, mine, v, a.weight_f32);
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

// Joins over the threads of a row: `lanes` of a warp (a power of two), or the whole block (`shared`: 32 floats, not those of the
// join before).
template <bool WARP, class F> __device__ __forceinline__ float row_join(float v, float *shared, F f, float none, int lanes) {
  if (WARP) return lanes_join(v, lanes, f);
  v = warp_join(v, f);
  const int lane = threadIdx.x & 31;
  if (lane == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_join(lane < (int)(blockDim.x >> 5) ? shared[lane] : none, f);
}
template <bool WARP> __device__ __forceinline__ float row_sum(float v, float *shared, int lanes) {
  return row_join<WARP>(v, shared, [](float p, float q) { return p + q; }, 0.f, lanes);
}

// A row is held by a warp (WARP) or by a block, E elements a thread in pieces of N: every tensor is read and written once.
// AHEAD: the blocks walk over the rows, and the next ones are on their way into shared memory, where every thread reads what it
// has copied itself.  HBM bounds it: 8192 x 4096 bf16 with a residual take 45 us (5.9 TB/s; 50 without copying ahead), one row of 5120
// to 8 bits 3 us, a launch and two barriers.  More than one row ahead gains nothing (backward of the same: 50 us with two stages, 51 and
// 53 with three and four; rows of 16384 133 us a pass and 174, whose third stage leaves no room for a second block).
constexpr int kRowStages = 2;
template <typename T, bool E4M3, int N, int E, bool WARP, bool AHEAD>
__global__ void __launch_bounds__(WARP ? 256 : 512, AHEAD && E == 8 ? (WARP ? 4 : 2) : 1) norm_rows_kernel(NormArgs a) {
  constexpr int V = E / N;
  extern __shared__ __align__(16) unsigned char row_memory[];
  __shared__ float shared[2][2][32];
  const int threads = WARP ? a.lanes : (int)blockDim.x, thread = WARP ? threadIdx.x & (threads - 1) : threadIdx.x, lane = threadIdx.x & 31;
  const int each = WARP ? 256 / threads : 1;  // rows of a block at once
  const int64_t first = WARP ? (int64_t)blockIdx.x * each + threadIdx.x / threads : blockIdx.x, step = (int64_t)gridDim.x * each;
  const int tensors = a.residual ? 2 : 1;
  const auto slot = [&](int stage, int tensor, int i) {
    return (uint4 *)row_memory + threadIdx.x + ((stage * tensors + tensor) * V + i) * (int)blockDim.x;
  };
  const auto copy = [&](int64_t row, int stage) {
    if (row < a.outer) {
#pragma unroll
      for (int i = 0; i < V; i++) {
        const int c = (thread + i * threads) * N;
        if (c < a.C) {
          copy_16(slot(stage, 0, i), (const T *)a.x + row * a.x_stride + c);
          if (a.residual) copy_16(slot(stage, 1, i), (const T *)a.residual + row * a.r_stride + c);
        }
      }
    }
    copies_end();
  };
  if (AHEAD)
    for (int d = 0; d < kRowStages - 1; d++) copy(first + d * step, d);
  int turn = 0, stage = 0;
  // (the lanes of a warp stay together: those past the last row work on nothing)
  for (int64_t row = first; row - (WARP ? lane / threads : 0) < a.outer; row += step, turn ^= 1) {
    const int C = !WARP || row < a.outer ? a.C : 0;
    Piece<T, N> s[V], add[V];
    if (AHEAD) {
      copy(row + (kRowStages - 1) * step, stage == 0 ? kRowStages - 1 : stage - 1);
      copies_wait<kRowStages - 1>();
    }
#pragma unroll
    for (int i = 0; i < V; i++) {
      const int c = (thread + i * threads) * N;
      if (c < C) {
        s[i].load(AHEAD ? (const T *)slot(stage, 0, i) : (const T *)a.x + row * a.x_stride + c);
        if (a.residual) add[i].load(AHEAD ? (const T *)slot(stage, 1, i) : (const T *)a.residual + row * a.r_stride + c);
      }
    }
    float sq = 0.f, most = 0.f;  // sum of squares; largest |s w|
#pragma unroll
    for (int i = 0; i < V; i++) {
      const int c = (thread + i * threads) * N;
      if (c < C) {
        if (a.residual) {
#pragma unroll
          for (int j = 0; j < N; j++) s[i].t[j] = from_float<T>(to_float(s[i].t[j]) + to_float(add[i].t[j]));
          s[i].store((T *)a.sum + row * a.C + c);
        }
        float w[N];
        if (E4M3) load_weights<T, N>(a.weight, c, a.weight_f32, w);
#pragma unroll
        for (int j = 0; j < N; j++) {
          const float f = to_float(s[i].t[j]);
          sq = fmaf(f, f, sq);
          if (E4M3) most = max_nan(most, fabsf(f * w[j]));
        }
      }
    }
    if (E4M3) {  // both joins behind one barrier
      most = lanes_join(most, WARP ? threads : 32, [](float p, float q) { return max_nan(p, q); });
      if (!WARP && lane == 0) shared[turn][1][threadIdx.x >> 5] = most;
    }
    const float rstd = 1.f / sqrtf(row_sum<WARP>(sq, shared[turn][0], threads) * a.inv_c + a.eps);
    if (thread == 0 && a.rstd && C) a.rstd[row] = rstd;
    float inverse = 0.f;  // (E4M3)
    if (E4M3) {
      if (!WARP)
        most = warp_join(lane < (int)(blockDim.x >> 5) ? shared[turn][1][lane] : 0.f, [](float p, float q) { return max_nan(p, q); });
      const Scale sc = Scale::of(most, rstd);
      if (thread == 0 && C) a.scale[row] = sc.scale;
      inverse = sc.inverse;
    }
#pragma unroll
    for (int i = 0; i < V; i++) {
      const int c = (thread + i * threads) * N;
      if (c < C) {
        float y[N];
        load_weights<T, N>(a.weight, c, a.weight_f32, y);
#pragma unroll
        for (int j = 0; j < N; j++) y[j] = E4M3 ? to_float(s[i].t[j]) * y[j] * inverse : to_float(s[i].t[j]) * rstd * y[j];
        if (E4M3) {
          store_e4m3<N>((__nv_fp8_storage_t *)a.out + row * a.C + c, y);
        } else {
#pragma unroll
          for (int j = 0; j < N; j++) s[i].t[j] = from_float<T>(y[j]);
          s[i].store((T *)a.out + row * a.C + c);
        }
      }
    }
    stage = stage == kRowStages - 1 ? 0 : stage + 1;
  }
}

// Backward: the blocks walk over the rows; a thread's channels stay the same, and their weights and weight gradients in its
// registers, so that the weight gradient costs no second pass over both tensors.  8192 x 4096 bf16 with both output gradients: 50 us
// (5.4 TB/s; 83 without copying ahead, between whose rows nothing was on its way).
template <typename T, int N, int E, bool WARP, bool ADD, bool AHEAD>
__global__ void __launch_bounds__(WARP ? 256 : 512, E == 8 ? (WARP ? 4 : 2) : 1) norm_rows_grad_kernel(NormGradArgs a) {
  constexpr int V = E / N, TENSORS = ADD ? 3 : 2;
  extern __shared__ __align__(16) unsigned char row_memory[];
  __shared__ float shared[2][32];
  __shared__ float sums[WARP ? 1024 : 1];
  const int threads = WARP ? a.lanes : (int)blockDim.x, thread = WARP ? threadIdx.x & (threads - 1) : threadIdx.x, lane = threadIdx.x & 31;
  const int each = WARP ? 256 / threads : 1;  // rows of a block at once
  const int64_t first = WARP ? (int64_t)blockIdx.x * each + threadIdx.x / threads : blockIdx.x, step = (int64_t)gridDim.x * each;
  uint4 *slots = (uint4 *)row_memory + threadIdx.x;  // (stage, tensor, piece) x threads of the block
  const auto slot = [&](int stage, int tensor, int i) { return slots + ((stage * TENSORS + tensor) * V + i) * (int)blockDim.x; };
  const auto copy = [&](int64_t row, int stage) {
    if (row < a.outer) {
#pragma unroll
      for (int i = 0; i < V; i++) {
        const int c = (thread + i * threads) * N;
        if (c < a.C) {
          copy_16(slot(stage, 0, i), (const T *)a.s + row * a.s_stride + c);
          copy_16(slot(stage, 1, i), (const T *)a.gout + row * a.C + c);
          if (ADD) copy_16(slot(stage, 2, i), (const T *)a.gsum + row * a.C + c);
        }
      }
    }
    copies_end();
  };
  float w[V][N], gw[V][N];
#pragma unroll
  for (int i = 0; i < V; i++) {
    const int c = (thread + i * threads) * N;
    if (c < a.C) load_weights<T, N>(a.weight, c, a.weight_f32, w[i]);
#pragma unroll
    for (int j = 0; j < N; j++) gw[i][j] = 0.f;
  }
  if (AHEAD)
    for (int d = 0; d < kRowStages - 1; d++) copy(first + d * step, d);
  int turn = 0, stage = 0;
  float rstd_next = first < a.outer ? a.rstd[first] : 0.f;
  for (int64_t row = first; row - (WARP ? lane / threads : 0) < a.outer; row += step, turn ^= 1) {
    const int C = !WARP || row < a.outer ? a.C : 0;
    const float rstd = rstd_next;
    if (row + step < a.outer) rstd_next = a.rstd[row + step];
    Piece<T, N> s[V], g[V], p[V];
    if (AHEAD) {
      copy(row + (kRowStages - 1) * step, stage == 0 ? kRowStages - 1 : stage - 1);
      copies_wait<kRowStages - 1>();
    }
#pragma unroll
    for (int i = 0; i < V; i++) {
      const int c = (thread + i * threads) * N;
      if (c < C) {
        if (AHEAD) {
          s[i].load((const T *)slot(stage, 0, i));
          g[i].load((const T *)slot(stage, 1, i));
        } else {
          s[i].load((const T *)a.s + row * a.s_stride + c);
          g[i].load((const T *)a.gout + row * a.C + c);
          if (ADD) p[i].load((const T *)a.gsum + row * a.C + c);
        }
      }
    }
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < V; i++) {
      const int c = (thread + i * threads) * N;
      if (c < C) {
#pragma unroll
        for (int j = 0; j < N; j++) {
          const float gu = to_float(g[i].t[j]) * (to_float(s[i].t[j]) * rstd);
          gw[i][j] += gu;
          dot = fmaf(gu, w[i][j], dot);
        }
      }
    }
    if (a.gx) {
      dot = row_sum<WARP>(dot, shared[turn], threads) * (-rstd * rstd * a.inv_c);
#pragma unroll
      for (int i = 0; i < V; i++) {
        const int c = (thread + i * threads) * N;
        if (c < C) {
          if (AHEAD && ADD) p[i].load((const T *)slot(stage, 2, i));
#pragma unroll
          for (int j = 0; j < N; j++) {
            const float v = fmaf(to_float(g[i].t[j]) * w[i][j], rstd, to_float(s[i].t[j]) * dot);
            s[i].t[j] = from_float<T>(ADD ? v + to_float(p[i].t[j]) : v);
          }
          s[i].store((T *)a.gx + row * a.C + c);
        }
      }
    }
    stage = stage == kRowStages - 1 ? 0 : stage + 1;
  }
  if (!a.gw) return;
  if (WARP) {  // the rows' sums in each warp, and the eight warps' sums, one after the other
#pragma unroll
    for (int i = 0; i < V; i++)
#pragma unroll
      for (int j = 0; j < N; j++)
        for (int d = threads; d < 32; d <<= 1) gw[i][j] += __shfl_xor_sync(0xffffffffu, gw[i][j], d);
    for (int c = threadIdx.x; c < a.C; c += 256) sums[c] = 0.f;
    for (int k = 0; k < 8; k++) {
      __syncthreads();
      if ((int)(threadIdx.x >> 5) == k && lane < threads)
#pragma unroll
        for (int i = 0; i < V; i++)
#pragma unroll
          for (int j = 0; j < N; j++) {
            const int c = (thread + i * threads) * N + j;
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

// Whether every row of a tensor starts on a 16-byte boundary.
inline bool rows_aligned(const void *p, int64_t stride, size_t size) {
  return (uintptr_t)p % 16 == 0 && stride * (int64_t)size % 16 == 0;
}

template <typename T, bool E4M3, int N, int E, bool WARP> void norm_rows_launch(const NormArgs &a, cudaStream_t st) {
  const int threads = WARP ? 256 : norm_row_threads(a.C), each = WARP ? 256 / a.lanes : 1;
  const int bytes = kRowStages * (a.residual ? 2 : 1) * E * (int)sizeof(T) * threads;
  const int64_t blocks = (a.outer + each - 1) / each;
  if constexpr (N > 1 && !WARP) {
    // Copying ahead pays from four rows a block on; the blocks are as many as there is room for on the SMs.
    const int fit = std::min((E == 8 ? 1024 : 512) / threads, 220 * 1024 / (bytes + 2048));
    if (fit >= 1 && blocks >= 4 * 148 * fit) {
      if (bytes > 32768)
        cudaFuncSetAttribute((const void *)norm_rows_kernel<T, E4M3, N, E, WARP, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
      norm_rows_kernel<T, E4M3, N, E, WARP, true><<<148 * fit, threads, bytes, st>>>(a);
      return;
    }
  }
  norm_rows_kernel<T, E4M3, N, E, WARP, false><<<(unsigned)blocks, threads, 0, st>>>(a);
}
template <typename T, bool E4M3, int N> void norm_rows_pick(NormArgs a, cudaStream_t st) {
  const bool warp = norm_path(a.C, 1) == kWarpRows;
  a.lanes = norm_row_lanes(a.C);
  switch (norm_row_elements(a.C)) {
    case 8: return warp ? norm_rows_launch<T, E4M3, N, 8, true>(a, st) : norm_rows_launch<T, E4M3, N, 8, false>(a, st);
    case 16: return warp ? norm_rows_launch<T, E4M3, N, 16, true>(a, st) : norm_rows_launch<T, E4M3, N, 16, false>(a, st);
    default: return warp ? norm_rows_launch<T, E4M3, N, 32, true>(a, st) : norm_rows_launch<T, E4M3, N, 32, false>(a, st);
  }
}

template <typename T, bool E4M3> void norm_launch(const NormArgs &a, int dtype, cudaStream_t st) {
  constexpr int N = 16 / (int)sizeof(T);
  switch (norm_path(a.C, a.inner)) {
    case kWarpRows:
    case kBlockRows:
      if (rows_aligned(a.x, a.x_stride, sizeof(T)) && a.C % N == 0 && rows_aligned(a.residual, a.r_stride, sizeof(T)) &&
          ((uintptr_t)a.sum % 16 | (uintptr_t)a.out % 16 | (uintptr_t)a.weight % 16) == 0)
        norm_rows_pick<T, E4M3, N>(a, st);
      else if (!norm_flat_forward(a, dtype, st))
        norm_rows_pick<T, E4M3, 1>(a, st);
      break;
    case kPlanes:
      norm_planes_forward(a, dtype, st);
      break;
    case kLongRows: norm_long_rows_kernel<T, E4M3><<<(unsigned)a.outer, 256, 0, st>>>(a); break;
    default: norm_deep_planes_kernel<T, E4M3><<<(unsigned)((a.outer * a.inner + 255) / 256), 256, 0, st>>>(a);
  }
}

template <typename T, int N, int E, bool WARP> void norm_rows_grad_launch(NormGradArgs &a, cudaStream_t st) {
  a.splits = std::min(a.splits, 148 * (WARP ? (E == 8 ? 4 : E == 16 ? 2 : 1) : std::max(1, (E == 8 ? 1024 : 512) / norm_row_threads(a.C))));
  const int threads = WARP ? 256 : norm_row_threads(a.C), tensors = a.gsum ? 3 : 2;
  const int bytes = kRowStages * tensors * E * (int)sizeof(T) * threads;
  if constexpr (N > 1) {
    if (bytes <= kMostRowStages) {
      void (*kernel)(NormGradArgs) = a.gsum ? norm_rows_grad_kernel<T, N, E, WARP, true, true> : norm_rows_grad_kernel<T, N, E, WARP, false, true>;
      if (bytes > 32768) cudaFuncSetAttribute((const void *)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
      kernel<<<a.splits, threads, bytes, st>>>(a);
      return;
    }
  }
  (a.gsum ? norm_rows_grad_kernel<T, N, E, WARP, true, false> : norm_rows_grad_kernel<T, N, E, WARP, false, false>)<<<a.splits, threads, 0, st>>>(a);
}
template <typename T, int N> void norm_rows_grad_pick(NormGradArgs &a, cudaStream_t st) {
  const bool warp = norm_path(a.C, 1) == kWarpRows;
  a.lanes = norm_row_lanes(a.C);
  switch (norm_row_elements(a.C)) {
    case 8: return warp ? norm_rows_grad_launch<T, N, 8, true>(a, st) : norm_rows_grad_launch<T, N, 8, false>(a, st);
    case 16: return warp ? norm_rows_grad_launch<T, N, 16, true>(a, st) : norm_rows_grad_launch<T, N, 16, false>(a, st);
    default: return warp ? norm_rows_grad_launch<T, N, 32, true>(a, st) : norm_rows_grad_launch<T, N, 32, false>(a, st);
  }
}

// Kernels launched.
template <typename T> int norm_grad_launch(NormGradArgs &a, int dtype, cudaStream_t st) {
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
        else if (!norm_flat_backward(a, dtype, st))
          norm_rows_grad_pick<T, 1>(a, st);
        break;
      case kPlanes:
        norm_planes_backward(a, dtype, st);
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
    norm_weight_reduce_kernel<T><<<(unsigned)cdiv(a.C, 32), 1024, 0, st>>>(a);
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
      norm_launch<T, true>(a, dtype, st);
    else
      norm_launch<T, false>(a, dtype, st);
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
  NormGradArgs a{gout, gsum, s, weight, rstd, gx, gw, (float *)ws, outer, inner, s_stride, (int)C, outer > 0 ? norm_splits(outer, C, inner) : 0,
                       1.f / (float)C, weight_dtype == SPH_F32};
  cudaStream_t st = (cudaStream_t)stream;
  int launches = 0;
  SPH_DISPATCH_ELEMENT(dtype, launches = norm_grad_launch<T>(a, dtype, st));
  return launch_status(launches);
}

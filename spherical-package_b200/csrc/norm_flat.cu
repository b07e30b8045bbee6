// Norms over rows that do not start on 16-byte boundaries (channels of an odd number), from dense tensors; see norm.cuh for the
// formulas.  A block takes some whole rows, which lie one behind the other, as one run of elements into shared memory, by
// asynchronous copies of 16 bytes from the boundary before the run on, works on them one element at a time there, and writes the run
// back the same way: only its ends are read and written in single elements.  Issue bounds it (some 20 instructions a value):
// 33.5M bf16 in rows of 4099 with a residual take 102 us forward (2.6 TB/s) and 144 backward; element by element from global memory
// 570 and 321.
#include "norm.cuh"

namespace sph {

// The run of `count` elements from g on; `shift` is how far g is behind a boundary, and the run in shared memory too.
template <typename T> __device__ __forceinline__ int run_shift(const T *g) { return (int)((uintptr_t)g % 16 / sizeof(T)); }
template <typename T> __device__ __forceinline__ void run_in(T *to, const T *g, int shift, int count) {
  constexpr int V = 16 / (int)sizeof(T);
  for (int j = threadIdx.x; j * V < shift + count; j += blockDim.x) {
    const int at = j * V - shift;
    if (at >= 0 && at + V <= count) {
      copy_16(to + j * V, g + at);
    } else {
      for (int e = 0; e < V; e++)
        if (at + e >= 0 && at + e < count) to[j * V + e] = g[at + e];
    }
  }
}
template <typename T> __device__ __forceinline__ void run_out(T *g, const T *from, int shift, int count) {
  constexpr int V = 16 / (int)sizeof(T);
  for (int j = threadIdx.x; j * V < shift + count; j += blockDim.x) {
    const int at = j * V - shift;
    if (at >= 0 && at + V <= count) {
      *(uint4 *)(g + at) = *(const uint4 *)(from + j * V);
    } else {
      for (int e = 0; e < V; e++)
        if (at + e >= 0 && at + e < count) g[at + e] = from[j * V + e];
    }
  }
}

// A thread's weights: in registers, or, in blocks that have but a row or two, read where they are used (4099 channels of bf16,
// with gradients: 522 us with them in registers, 256 us without; 333 channels: 239 and 322).
template <typename T, int E, bool BLOCK> struct RowWeights {
  float kept[BLOCK ? 1 : E];
  const void *from;
  int thread, threads;
  bool f32;
  __device__ __forceinline__ RowWeights(const void *w, bool f32, int C, int thread, int threads) : from(w), thread(thread), threads(threads), f32(f32) {
    if (!BLOCK) {
#pragma unroll
      for (int j = 0; j < E; j++) kept[BLOCK ? 0 : j] = w && thread + j * threads < C ? load_weight<T>(w, thread + j * threads, f32) : 1.f;
    }
  }
  __device__ __forceinline__ float operator()(int j) const {
    return !BLOCK ? kept[BLOCK ? 0 : j] : from ? load_weight<T>(from, thread + j * threads, f32) : 1.f;
  }
};

extern __shared__ __align__(16) unsigned char flat_memory[];

struct FlatTile {
  int rows, lanes_log;  // rows of a tile; log2 of the lanes of a row (rows of a block each: 5)
  int room;             // bytes in shared memory for a run of a tensor
};

template <typename T, bool E4M3, bool ADD, int E, bool BLOCK> __global__ void __launch_bounds__(BLOCK ? 512 : 256, BLOCK ? 2 : 3) norm_flat_kernel(NormArgs a, FlatTile tile) {
  __shared__ float shared[2][2][16];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int threads = BLOCK ? (int)blockDim.x : 1 << tile.lanes_log, thread = BLOCK ? (int)threadIdx.x : lane & (threads - 1);
  const int64_t row0 = (int64_t)blockIdx.x * tile.rows, e0 = row0 * a.C;
  const int rows = (int)min((int64_t)tile.rows, a.outer - row0), count = rows * a.C, shift = run_shift((const T *)a.x + e0);
  T *x = (T *)flat_memory, *r = (T *)(flat_memory + tile.room);
  unsigned char *q = flat_memory + (ADD ? 2 : 1) * tile.room;  // (E4M3)
  const int q_shift = run_shift((const unsigned char *)a.out + e0);
  run_in(x, (const T *)a.x + e0, shift, count);
  if (ADD) run_in(r, (const T *)a.residual + e0, shift, count);
  copies_end();
  const RowWeights<T, E, BLOCK> w(a.weight, a.weight_f32, a.C, thread, threads);
  copies_wait<0>();
  __syncthreads();
  const int step = BLOCK ? 1 : (int)blockDim.x >> tile.lanes_log, sub = BLOCK ? 0 : lane >> tile.lanes_log;
  int turn = 0;
  for (int i0 = BLOCK ? 0 : warp * (32 >> tile.lanes_log); i0 < rows; i0 += step, turn ^= 1) {
    const int i = i0 + sub;
    const bool on = i < rows;
    T *at = x + shift + (on ? i : 0) * a.C + thread;
    const T *rt = r + (at - x);
    float v[E], sq = 0.f, most = 0.f;
#pragma unroll
    for (int j = 0; j < E; j++) {
      v[j] = 0.f;
      if (thread + j * threads < a.C && on) {
        v[j] = to_float(at[j * threads]);
        if (ADD) {
          const T s = from_float<T>(v[j] + to_float(rt[j * threads]));
          at[j * threads] = s;
          v[j] = to_float(s);
        }
      }
      sq = fmaf(v[j], v[j], sq);
      if (E4M3 && thread + j * threads < a.C) most = max_nan(most, fabsf(v[j] * w(j)));
    }
    const auto add = [](float p, float q) { return p + q; };
    const auto larger = [](float p, float q) { return max_nan(p, q); };
    sq = lanes_join(sq, BLOCK ? 32 : threads, add);
    if (E4M3) most = lanes_join(most, BLOCK ? 32 : threads, larger);
    if (BLOCK) {
      if (lane == 0) {
        shared[turn][0][warp] = sq;
        if (E4M3) shared[turn][1][warp] = most;
      }
      __syncthreads();
      const bool has = lane < (int)(blockDim.x >> 5);
      sq = warp_join(has ? shared[turn][0][lane] : 0.f, add);
      if (E4M3) most = warp_join(has ? shared[turn][1][lane] : 0.f, larger);
    }
    const float rstd = 1.f / sqrtf(sq * a.inv_c + a.eps);
    float inverse = 0.f;  // (E4M3)
    if (on && thread == 0 && a.rstd) a.rstd[row0 + i] = rstd;
    if (E4M3) {
      const Scale sc = Scale::of(most, rstd);
      if (on && thread == 0) a.scale[row0 + i] = sc.scale;
      inverse = sc.inverse;
    }
    T *out = ADD ? r + (at - x) : at;
#pragma unroll
    for (int j = 0; j < E; j++)
      if (thread + j * threads < a.C && on) {
        const float y = E4M3 ? v[j] * w(j) * inverse : v[j] * rstd * w(j);
        if (E4M3)
          q[q_shift + i * a.C + thread + j * threads] = to_e4m3(y);
        else
          out[j * threads] = from_float<T>(y);
      }
  }
  __syncthreads();
  if (ADD) run_out((T *)a.sum + e0, x, shift, count);
  if (E4M3)
    run_out((unsigned char *)a.out + e0, q, q_shift, count);
  else
    run_out((T *)a.out + e0, ADD ? r : x, shift, count);
}

// Backward: the blocks walk over the tiles; a thread's channels stay the same, and their weight gradients in its registers.
template <typename T, bool ADD, int E, bool BLOCK> __global__ void __launch_bounds__(BLOCK ? 512 : 256, BLOCK ? (E <= 16 ? 2 : 1) : 3) norm_flat_grad_kernel(NormGradArgs a, FlatTile tile, int tiles) {
  __shared__ float shared[2][16];
  __shared__ float sums[BLOCK ? 1 : 1024];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int threads = BLOCK ? (int)blockDim.x : 1 << tile.lanes_log, thread = BLOCK ? (int)threadIdx.x : lane & (threads - 1);
  T *s = (T *)flat_memory, *g = (T *)(flat_memory + tile.room), *p = (T *)(flat_memory + 2 * tile.room);
  const RowWeights<T, E, BLOCK> w(a.weight, a.weight_f32, a.C, thread, threads);
  float gw[E];
#pragma unroll
  for (int j = 0; j < E; j++) gw[j] = 0.f;
  const int step = BLOCK ? 1 : (int)blockDim.x >> tile.lanes_log, sub = BLOCK ? 0 : lane >> tile.lanes_log;
  int turn = 0;
  for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int64_t row0 = (int64_t)t * tile.rows, e0 = row0 * a.C;
    const int rows = (int)min((int64_t)tile.rows, a.outer - row0), count = rows * a.C, shift = run_shift((const T *)a.s + e0);
    run_in(s, (const T *)a.s + e0, shift, count);
    run_in(g, (const T *)a.gout + e0, shift, count);
    if (ADD && a.gx) run_in(p, (const T *)a.gsum + e0, shift, count);
    copies_end();
    copies_wait<0>();
    __syncthreads();
    for (int i0 = BLOCK ? 0 : warp * (32 >> tile.lanes_log); i0 < rows; i0 += step, turn ^= 1) {
      const int i = i0 + sub;
      const bool on = i < rows;
      const int at = shift + (on ? i : 0) * a.C + thread;
      const float rstd = on ? a.rstd[row0 + i] : 0.f;
      float dot = 0.f;
#pragma unroll
      for (int j = 0; j < E; j++)
        if (thread + j * threads < a.C && on) {
          const float gu = to_float(g[at + j * threads]) * (to_float(s[at + j * threads]) * rstd);
          gw[j] += gu;
          dot = fmaf(gu, w(j), dot);
        }
      if (!a.gx) continue;
      const auto add = [](float p, float q) { return p + q; };
      dot = lanes_join(dot, BLOCK ? 32 : threads, add);
      if (BLOCK) {
        if (lane == 0) shared[turn][warp] = dot;
        __syncthreads();
        dot = warp_join(lane < (int)(blockDim.x >> 5) ? shared[turn][lane] : 0.f, add);
      }
      dot *= -rstd * rstd * a.inv_c;
#pragma unroll
      for (int j = 0; j < E; j++)
        if (thread + j * threads < a.C && on) {
          const int k = at + j * threads;
          float v = fmaf(to_float(g[k]) * w(j), rstd, to_float(s[k]) * dot);
          if (ADD) v += to_float(p[k]);
          s[k] = from_float<T>(v);
        }
    }
    __syncthreads();
    if (a.gx) {
      run_out((T *)a.gx + e0, s, shift, count);
      __syncthreads();
    }
  }
  if (!a.gw) return;
  if constexpr (BLOCK) {
#pragma unroll
    for (int j = 0; j < E; j++)
      if (thread + j * threads < a.C) a.partial[(int64_t)blockIdx.x * a.C + thread + j * threads] = gw[j];
  } else {
#pragma unroll
    for (int j = 0; j < E; j++)
      for (int d = threads; d < 32; d <<= 1) gw[j] += __shfl_xor_sync(0xffffffffu, gw[j], d);
    for (int c = threadIdx.x; c < a.C; c += 256) sums[c] = 0.f;
    for (int k = 0; k < 8; k++) {  // the warps' sums, one after the other
      __syncthreads();
      if (warp == k && lane < threads)
#pragma unroll
        for (int j = 0; j < E; j++)
          if (thread + j * threads < a.C) sums[thread + j * threads] += gw[j];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < a.C; c += 256) a.partial[(int64_t)blockIdx.x * a.C + c] = sums[c];
  }
}

// A tile: rows of about 12 KB a tensor, fewer where there would be fewer than two tiles a SM, and the lanes that share a row,
// eight channels each where it has up to 256.
static FlatTile flat_tile(int64_t outer, int64_t C, int size) {
  FlatTile t;
  t.lanes_log = 0;
  while (t.lanes_log < 5 && (int64_t)8 << t.lanes_log < C) t.lanes_log++;
  const int64_t most = std::max<int64_t>(1, 12288 / (C * size)), even = std::max<int64_t>(1, outer / (2 * 148));
  t.rows = (int)std::min(most, even);
  t.room = (int)((t.rows * C * size + 32 + 15) / 16 * 16);
  return t;
}

// Rows of up to 512 channels have lanes of a warp, others a block, of up to 512 threads.
static int flat_threads(int64_t C, int E) { return 32 * cdiv(C, 32 * E); }
template <typename T, bool E4M3, bool ADD, int E, bool BLOCK> static void flat_launch(const NormArgs &a, cudaStream_t st) {
  const FlatTile tile = flat_tile(a.outer, a.C, sizeof(T));
  constexpr bool block = BLOCK;
  const int bytes = tile.room * (ADD ? 2 : 1) + (E4M3 ? (tile.rows * a.C + 47) / 16 * 16 : 0);
  void (*kernel)(NormArgs, FlatTile) = norm_flat_kernel<T, E4M3, ADD, E, BLOCK>;
  if (bytes > 32768) cudaFuncSetAttribute((const void *)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  kernel<<<(unsigned)((a.outer + tile.rows - 1) / tile.rows), block ? flat_threads(a.C, E) : 256, bytes, st>>>(a, tile);
}
template <typename T, bool ADD, int E, bool BLOCK> static void flat_grad_launch(NormGradArgs &a, cudaStream_t st) {
  const FlatTile tile = flat_tile(a.outer, a.C, sizeof(T));
  constexpr bool block = BLOCK;
  const int bytes = tile.room * (ADD ? 3 : 2), threads = block ? flat_threads(a.C, E) : 256;
  const int64_t tiles = (a.outer + tile.rows - 1) / tile.rows;
  void (*kernel)(NormGradArgs, FlatTile, int) = norm_flat_grad_kernel<T, ADD, E, BLOCK>;
  if (bytes > 32768) cudaFuncSetAttribute((const void *)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  // as many blocks as are on the SMs at once, by registers and by shared memory
  const int fit = std::min(block ? std::max(1, (E <= 16 ? 1024 : 512) / threads) : 3, 220 * 1024 / (bytes + 6144));
  a.splits = (int)std::min<int64_t>(a.splits, std::min<int64_t>(tiles, 148 * fit));
  kernel<<<a.splits, threads, bytes, st>>>(a, tile, (int)tiles);
}

#define SPH_FLAT(e, b, ...) { constexpr int E = e; constexpr bool BLOCK = b; __VA_ARGS__; }
#define SPH_DISPATCH_FLAT(C, ...)                                      \
  if (C <= 256) SPH_FLAT(8, false, __VA_ARGS__)                        \
  else if (C <= 512) SPH_FLAT(16, false, __VA_ARGS__)                  \
  else if (C <= 4096) SPH_FLAT(8, true, __VA_ARGS__)                   \
  else if (C <= 8192) SPH_FLAT(16, true, __VA_ARGS__)                  \
  else SPH_FLAT(32, true, __VA_ARGS__)

bool norm_flat_forward(const NormArgs &a, int dtype, cudaStream_t st) {
  const uintptr_t x = (uintptr_t)a.x;
  if ((a.outer > 1 && (a.x_stride != a.C || (a.residual && a.r_stride != a.C))) || (a.residual && ((x ^ (uintptr_t)a.residual) % 16 || (x ^ (uintptr_t)a.sum) % 16)) ||
      (!a.scale && (x ^ (uintptr_t)a.out) % 16))
    return false;
  SPH_DISPATCH_ELEMENT(dtype, SPH_DISPATCH_FLAT(a.C, {
    if (a.scale)
      a.residual ? flat_launch<T, true, true, E, BLOCK>(a, st) : flat_launch<T, true, false, E, BLOCK>(a, st);
    else
      a.residual ? flat_launch<T, false, true, E, BLOCK>(a, st) : flat_launch<T, false, false, E, BLOCK>(a, st);
  }));
  return true;
}

bool norm_flat_backward(NormGradArgs &a, int dtype, cudaStream_t st) {
  const uintptr_t s = (uintptr_t)a.s;
  if ((a.outer > 1 && a.s_stride != a.C) || (s ^ (uintptr_t)a.gout) % 16 || (a.gsum && (s ^ (uintptr_t)a.gsum) % 16) ||
      (a.gx && (s ^ (uintptr_t)a.gx) % 16))
    return false;
  SPH_DISPATCH_ELEMENT(dtype, SPH_DISPATCH_FLAT(a.C, { a.gsum ? flat_grad_launch<T, true, E, BLOCK>(a, st) : flat_grad_launch<T, false, E, BLOCK>(a, st); }));
  return true;
}

}  // namespace sph

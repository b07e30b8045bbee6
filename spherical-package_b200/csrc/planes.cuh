// Runs of pixels with all their channels in shared memory.
#pragma once

#include <algorithm>
#include <initializer_list>

#include "element.cuh"

namespace sph {

// ---- planes through shared memory ------------------------------------------------------------------------------------
// A block of 8 warps takes a run of pixels with all their channels into shared memory by asynchronous copies, so that every
// tensor is read and written once; two or more blocks a SM copy and compute in turn.  `across` warps share the channels of a
// unit of 32 float32 or 64 16-bit pixels, the others have further units; what a norm needs of all its channels is joined
// through shared memory.  Rows of a channel are copied
//   kWide    16 bytes at a time, where planes start on 16-byte boundaries; a lane has 4 bytes, neighbouring pixels;
//   kShifted 16 bytes at a time too, from the boundary before the run on, so that a row lies in shared memory as far off a
//            boundary as in its tensor; a lane has every 32nd pixel, and a run stays in its image;
//   kSingle  pixel by pixel (small images, few channels).
enum Mode { kWide, kShifted, kSingle };
template <typename T, int U> union Pixels {  // a lane's, of a channel: 4 or 8 bytes
  static constexpr int N = 4 * U / (int)sizeof(T);
  unsigned w[U];
  T t[N];
  __device__ __forceinline__ Pixels() {}
};
constexpr int kPlaneWarps = 8, kPlaneThreads = 32 * kPlaneWarps, kMostPlanes = 512;
// LOG: log2 of the warps that share a unit's channels, 0 (one warp has them all) or 3.  U: 4-byte parts of a lane.
template <typename T, int MODE, int LOG, int U> struct Geometry {
  static constexpr int N = Pixels<T, U>::N, V = 16 / (int)sizeof(T);
  static constexpr int ACROSS = 1 << LOG, PIXELS = 256 * N >> LOG;  // of a run
  static constexpr int PITCH = PIXELS + (MODE == kShifted ? V : 0);  // elements from a channel's row to the next
  static constexpr int ROW = ACROSS * PITCH;                         // to a warp's next channel
};
struct PlaneTile {
  FastDiv by;    // by the pixels of a plane, or, shifted, by a plane's runs
  bool small;    // fewer than 2^31 pixels in all
  int64_t runs;  // in all
  template <class G, int MODE> static PlaneTile of(int64_t outer, int64_t inner) {
    PlaneTile t;
    const int64_t total = outer * inner, each = (inner + G::PIXELS - 1) / G::PIXELS;
    t.runs = MODE == kShifted ? outer * each : (total + G::PIXELS - 1) / G::PIXELS;
    t.small = total < ((int64_t)1 << 31);
    t.by = FastDiv::make(!t.small ? 1u : (unsigned)(MODE == kShifted ? each : inner));
    return t;
  }
};
// Channels one warp may have alone; with more, eight share them; and up to which a lane has eight bytes of each, so that what
// a run costs whatever its channels spreads over more pixels (8-bit norms of 3 x 96 x 181 x 333 bf16 28.7 us with four, 24.9 with
// eight).
constexpr int kAlone = 32, kTwice = 128;
// Runs that end with their image are to be an eighth more at most, counted in runs of one part of 4 bytes a lane; lanes of two parts
// have runs twice as long, which may be half more, and are still faster than single elements (256 x 96 x 11 x 17 bf16 with gradients and
// a residual: 43 us, 70 in single elements; 128 x 128 x 17 x 11: 31 and 57; 256 x 128 x 5 x 19 float32: 37 and 43).
template <typename T> Mode plane_mode(int64_t C, int64_t inner, bool aligned) {
  const int64_t pixels = C > kAlone ? Geometry<T, kShifted, 3, 1>::PIXELS : Geometry<T, kShifted, 0, 1>::PIXELS;
  return aligned ? kWide : 8 * ((inner + pixels - 1) / pixels * pixels) <= 9 * inner ? kShifted : kSingle;
}

// A run of pixels: offset of channel 0 of its pixel i, and the norms' numbers.
template <int MODE, int PIXELS> struct Run {
  int64_t start, image, inner, total;  // kShifted: start and image are this run's, else pixels are numbered through
  int C;
  const PlaneTile &tile;
  __device__ __forceinline__ Run(const PlaneTile &tile, int64_t index, int64_t outer, int C, int64_t inner)
      : inner(inner), total(outer * inner), C(C), tile(tile) {
    if (MODE == kShifted) {
      const int64_t each = (inner + PIXELS - 1) / PIXELS;
      image = tile.small ? (int64_t)tile.by.div((unsigned)index) : index / each;
      start = (index - image * each) * PIXELS;
    } else {
      start = index * PIXELS;
    }
  }
  __device__ __forceinline__ bool has(int i) const { return MODE == kShifted ? start + i < inner : start + i < total; }
  __device__ __forceinline__ int64_t norm(int i) const { return MODE == kShifted ? image * inner + start + i : start + i; }
  __device__ __forceinline__ int64_t offset(int i) const {
    if (MODE == kShifted) return image * C * inner + start + i;
    const int64_t at = start + i, o = tile.small ? (int64_t)tile.by.div((unsigned)at) : at / inner;
    return o * C * inner + (at - o * inner);
  }
};

// Elements between the 16-byte boundary before a channel's run and the run (kShifted), the same for a warp's channels.
template <typename T> __device__ __forceinline__ int shift_of(const T *from, int64_t offset, int c, int64_t inner) {
  return (int)(((uintptr_t)(from + offset) / sizeof(T) + (uintptr_t)c * (uintptr_t)inner) & (16 / sizeof(T) - 1));
}

// Where a lane finds its pixels of a warp's k-th channel in shared memory.  A row's shift is the same for all channels of one of
// eight warps (every eighth, and shifts repeat every V at the latest), and another for each of a warp's alone.
template <typename T, int MODE, int LOG, int U> struct Rows {
  using G = Geometry<T, MODE, LOG, U>;
  T *base;
  int shift, step;
  __device__ __forceinline__ Rows(T *tile, const T *from, int64_t offset, int first, int col, int64_t inner) : base(tile + first * G::PITCH + col) {
    shift = MODE == kShifted ? shift_of(from, offset, first, inner) : 0;
    step = (int)(inner & (G::V - 1));
    if (LOG == 3) base += shift;
  }
  __device__ __forceinline__ T *operator()(int k) const {
    return base + k * G::ROW + (MODE == kShifted && LOG == 0 ? (shift + k * step) & (G::V - 1) : 0);
  }
};

// Copies a run, all channels.
template <typename T, int MODE, int LOG, int U, class R> __device__ __forceinline__ void copy_run(T *to, const T *from, const R &run) {
  using G = Geometry<T, MODE, LOG, U>;
  constexpr int V = G::V;
  if constexpr (MODE == kWide) {
    constexpr int COLS = G::PIXELS / V, ROWS = kPlaneThreads / COLS;
    const int col = (threadIdx.x % COLS) * V, first = threadIdx.x / COLS;
    if (!run.has(col)) return;
    const T *p = from + run.offset(col) + first * run.inner;
    const int64_t step = ROWS * run.inner;
    T *q = to + first * G::PITCH + col;
#pragma unroll 4
    for (int c = first; c < run.C; c += ROWS, p += step, q += ROWS * G::PITCH) copy_16(q, p);
  } else if constexpr (MODE == kShifted) {
    constexpr int PIECES = G::PIXELS / V + 1;  // a row's, from the boundary before it
    const T *base = from + run.offset(0), *last = from + run.total * run.C;
    const int count = (int)min((int64_t)G::PIXELS, run.inner - run.start);
    if constexpr (LOG == 3) {  // a warp its own channels, whose shift is one
      const int first = threadIdx.x >> 5, piece = threadIdx.x & 31, at = piece * V - shift_of(base, 0, first, run.inner);
      // (all but the tensor's first and last pixels have something before and behind them)
      const bool whole = base - V >= from && base + (run.C - 1) * run.inner + G::PIXELS + V <= last;
      if (piece >= PIECES || at >= count) return;
      const T *p = base + first * run.inner + at;
      T *q = to + first * G::PITCH + piece * V;
      const int64_t step = G::ACROSS * run.inner;
      if (whole) {
#pragma unroll 4
        for (int c = first; c < run.C; c += G::ACROSS, p += step, q += G::ROW) copy_16(q, p);
      } else {
        for (int c = first; c < run.C; c += G::ACROSS, p += step, q += G::ROW) {
          if (p >= from && p + V <= last) {
            copy_16(q, p);
          } else {
            for (int e = 0; e < V; e++)
              if (at + e >= 0 && at + e < count) q[e] = p[e];
          }
        }
      }
      return;
    }
#pragma unroll 4
    for (int i = threadIdx.x; i < run.C * PIECES; i += kPlaneThreads) {
      const int c = i / PIECES, j = i % PIECES, at = j * V - shift_of(base, 0, c, run.inner);
      if (at >= count) continue;
      const T *p = base + c * run.inner + at;
      T *q = to + c * G::PITCH + j * V;
      if (p >= from && p + V <= last) {
        copy_16(q, p);
      } else {  // the tensor's first and last pixels
        for (int e = 0; e < V; e++)
          if (at + e >= 0 && at + e < count) q[e] = p[e];
      }
    }
  } else {
    constexpr int COLS = G::PIXELS < kPlaneThreads ? G::PIXELS : kPlaneThreads, ROWS = kPlaneThreads / COLS;
#pragma unroll
    for (int col = threadIdx.x % COLS; col < G::PIXELS; col += COLS) {
      if (!run.has(col)) return;
      const int first = threadIdx.x / COLS;
      const T *p = from + run.offset(col) + first * run.inner;
      const int64_t step = ROWS * run.inner;
      T *q = to + first * G::PITCH + col;
      if constexpr (sizeof(T) == 4) {
#pragma unroll 4
        for (int c = first; c < run.C; c += ROWS, p += step, q += ROWS * G::PITCH) copy_4(q, p);
      } else {
        for (int c = first; c < run.C; c += ROWS * 16) {
          T v[16];
#pragma unroll
          for (int e = 0; e < 16; e++)
            if (c + e * ROWS < run.C) v[e] = p[e * step];
#pragma unroll
          for (int e = 0; e < 16; e++)
            if (c + e * ROWS < run.C) q[e * ROWS * G::PITCH] = v[e];
          p += 16 * step, q += 16 * ROWS * G::PITCH;
        }
      }
    }
  }
}

// A lane's pixels of a run: col, col + 1 (kWide) or col, col + 32.
template <typename T, int MODE, int LOG, int U> struct Lane {
  using P = Pixels<T, U>;
  static constexpr int N = P::N, STEP = MODE == kWide ? 1 : 32;
  int col;
  bool in[N];
  int64_t norm[N], off[N];  // of the warp's first channel
  template <class R> __device__ __forceinline__ Lane(const R &run, int first) {
    const int lane = threadIdx.x & 31;
    col = (threadIdx.x >> 5 >> LOG) * 32 * N + (MODE == kWide ? lane * N : lane);
#pragma unroll
    for (int i = 0; i < N; i++) {
      in[i] = run.has(col + i * STEP);
      norm[i] = run.norm(col + i * STEP);
      off[i] = in[i] && (MODE == kSingle || i == 0) ? run.offset(col + i * STEP) + first * run.inner : 0;
    }
  }
  // (The pixels of a shifted run are in one image.)
  __device__ __forceinline__ int64_t at(int i) const { return MODE == kShifted ? off[0] + i * STEP : off[i]; }
  static __device__ __forceinline__ void words(const T *p, P &v) {
    if constexpr (U == 1) {
      v.w[0] = *(const unsigned *)p;
    } else {
      const uint2 q = *(const uint2 *)p;
      v.w[0] = q.x, v.w[1] = q.y;
    }
  }
  static __device__ __forceinline__ void put_words(T *p, const P &v) {
    if constexpr (U == 1) *(unsigned *)p = v.w[0];
    else *(uint2 *)p = make_uint2(v.w[0], v.w[1]);
  }
  static __device__ __forceinline__ P load(const T *p) {
    P v;
    if constexpr (MODE == kWide) {
      words(p, v);
    } else {
#pragma unroll
      for (int i = 0; i < N; i++) v.t[i] = p[i * STEP];
    }
    return v;
  }
  static __device__ __forceinline__ void keep(T *p, const P &v) {
    if constexpr (MODE == kWide) {
      put_words(p, v);
    } else {
#pragma unroll
      for (int i = 0; i < N; i++) p[i * STEP] = v.t[i];
    }
  }
  // `plane`: elements from the warp's first channel.
  __device__ __forceinline__ void store(T *to, int64_t plane, const P &v) const {
    if constexpr (MODE == kWide) {
      if (in[0]) put_words(to + off[0] + plane, v);
    } else {
#pragma unroll
      for (int i = 0; i < N; i++)
        if (in[i]) to[at(i) + plane] = v.t[i];
    }
  }
  __device__ __forceinline__ void store_e4m3(__nv_fp8_storage_t *to, int64_t plane, const float (&y)[N]) const {
    if constexpr (MODE == kWide && N == 1) {
      if (in[0]) to[off[0] + plane] = to_e4m3(y[0]);
    } else if constexpr (MODE == kWide) {
      if (in[0]) {
        const unsigned a = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3);
        if constexpr (N == 2) {
          *(__nv_fp8x2_storage_t *)(to + off[0] + plane) = (__nv_fp8x2_storage_t)a;
        } else {
          const unsigned b = __nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3);
          *(unsigned *)(to + off[0] + plane) = a | b << 16;
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; i++)
        if (in[i]) to[at(i) + plane] = to_e4m3(y[i]);
    }
  }
};

// Joins a value of each of the lane's pixels over the warps that share them.  `shared`: 8 x 32 x N floats.
template <int LOG, int N, class F> __device__ __forceinline__ void plane_join(float (&v)[N], float *shared, F f) {
  if (LOG == 0) return;
  constexpr int n = 1 << LOG;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, mates = warp & ~(n - 1);
#pragma unroll
  for (int i = 0; i < N; i++) shared[(warp * N + i) * 32 + lane] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; i++) v[i] = shared[(mates * N + i) * 32 + lane];
#pragma unroll
  for (int w = 1; w < n; w++)
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = f(v[i], shared[((mates + w) * N + i) * 32 + lane]);
}

// The weights as floats, ones without.
template <typename T> __device__ __forceinline__ void keep_weights(float *to, const void *w, bool f32, int C) {
  for (int c = threadIdx.x; c < C; c += kPlaneThreads) to[c] = w ? load_weight<T>(w, c, f32) : 1.f;
}

extern __shared__ __align__(16) unsigned char plane_memory[];

// Whether 16 bytes of a plane may be copied at once.
template <typename T> bool planes_aligned(int64_t inner, std::initializer_list<const void *> ps) {
  uintptr_t bits = (uintptr_t)inner * sizeof(T);
  for (const void *p : ps) bits |= (uintptr_t)p;
  return bits % 16 == 0;
}
// Launches a kernel over runs of `tensors` tensors in shared memory.
template <class G, typename T, class A>
void plane_launch(void (*kernel)(A, PlaneTile), const A &a, const PlaneTile &tile, int tensors, unsigned blocks, cudaStream_t st) {
  const int bytes = (int)sizeof(T) * a.C * G::PITCH * tensors;
  if (bytes > 32768) cudaFuncSetAttribute((const void *)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  kernel<<<blocks, kPlaneThreads, bytes, st>>>(a, tile);
}
// Run a statement with MODE, LOG, U and the geometry G.
#define SPH_PLANES(M, L, P, ...) { constexpr int MODE = M, LOG = L, U = P; using G = Geometry<T, MODE, LOG, U>; __VA_ARGS__; }
#define SPH_PLANES_OF(M, C, ...)                                       \
  if (C <= kTwice) SPH_PLANES(M, 3, 2, __VA_ARGS__)                    \
  else SPH_PLANES(M, 3, 1, __VA_ARGS__)
#define SPH_DISPATCH_PLANES(mode, C, ...)                              \
  if (C <= kAlone) {                                                   \
    if (mode == kWide) SPH_PLANES(kWide, 0, 1, __VA_ARGS__)            \
    else if (mode == kShifted) SPH_PLANES(kShifted, 0, 1, __VA_ARGS__) \
    else SPH_PLANES(kSingle, 0, 1, __VA_ARGS__)                        \
  } else {                                                             \
    if (mode == kWide) { SPH_PLANES_OF(kWide, C, __VA_ARGS__) }        \
    else if (mode == kShifted) { SPH_PLANES_OF(kShifted, C, __VA_ARGS__) } \
    else { SPH_PLANES_OF(kSingle, C, __VA_ARGS__) }                    \
  }

}  // namespace sph

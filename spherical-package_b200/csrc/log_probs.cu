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

#include <cooperative_groups.h>

#include <algorithm>

namespace sph {

namespace cg = cooperative_groups;

struct LogProbArgs {
  const void *x;
  const int64_t *target;
  float *log_probs, *entropy, *top;  // top (outer, k, inner)
  float2 *stats;                     // (m, S) of each distribution, for the backward pass
  int64_t *top_index;
  int64_t outer, inner, x_stride, ignore_index;
  int C, k;
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// 2^d for d <= 0 (or NaN), 0 far below.
__device__ __forceinline__ float exp2_fast(float d) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  return r;
}
// log2 e times a logit's distance from the maximum; what is infinitely far below stops at a finite distance whose exponential
// is 0, so that 0 times it is 0.
constexpr float kFar = -1000.f;
__device__ __forceinline__ float distance(float x, float base) { return max_nan((x - base) * kLog2e, kFar); }

// Order of the candidates as one number: larger is better; value first (NaN above all), then the lower index.
__device__ __forceinline__ unsigned order_of(float v) {
  const unsigned u = __float_as_uint(v + 0.f);  // (-0 and 0 are equal)
  return v != v ? 0xffffffffu : (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned order) {
  return order == 0xffffffffu ? NAN : __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
using Candidate = unsigned long long;
__device__ __forceinline__ Candidate candidate(unsigned order, int index) {
  return ((Candidate)order << 32) | (0xffffffffu - (unsigned)index);
}
__device__ __forceinline__ int candidate_index(Candidate c) { return (int)(0xffffffffu - (unsigned)c); }

// Softmax statistics of a part of a distribution: its maximum, and with d = (x - m) log2 e the sums of 2^d and of 2^d d.
struct Stats {
  float m = -INFINITY, s = 0.f, t = 0.f;
  __device__ __forceinline__ float4 packed() const { return make_float4(m, s, t, 0.f); }
  static __device__ __forceinline__ Stats of(float4 v) {
    Stats r;
    r.m = v.x, r.s = v.y, r.t = v.z;
    return r;
  }
  // The maximum that distances are measured from: a finite one while there is nothing but -inf.
  static __device__ __forceinline__ float base(float m) { return m == -INFINITY ? 0.f : m; }
  // The sums for another, not smaller maximum: 2^d' = 2^d 2^c and 2^d' d' = (2^d d + 2^d c) 2^c with c = (m - n) log2 e.
  __device__ __forceinline__ void move_to(float n) {
    if (m == n) return;
    const float c = distance(m, base(n)), f = exp2_fast(c);
    t = fmaf(s, c, t) * f;
    s *= f;
    m = n;
  }
  __device__ __forceinline__ void add(float x) {
    move_to(max_nan(m, x));
    const float d = distance(x, base(m)), e = exp2_fast(d);
    s += e;
    t = fmaf(e, d, t);
  }
  __device__ __forceinline__ void join(Stats o) {
    const float n = max_nan(m, o.m);
    move_to(n);
    o.move_to(n);
    s += o.s;
    t += o.t;
  }
  // Over groups of `lanes` neighbouring lanes of the warp, the same in each.
  __device__ __forceinline__ void join_lanes(int lanes) {
    move_to(lanes_join(m, lanes, [](float a, float b) { return max_nan(a, b); }));
    const auto add = [](float a, float b) { return a + b; };
    s = lanes_join(s, lanes, add);
    t = lanes_join(t, lanes, add);
  }
  __device__ __forceinline__ void join_warp() { join_lanes(32); }
  __device__ __forceinline__ float entropy() const {
    const float h = s == 0.f ? 0.f : logf(s) - kLn2 * (t / s);
    return h < 0.f ? 0.f : h;
  }
  __device__ __forceinline__ float log_prob(float x) const { return s == 0.f ? -INFINITY : (x - m) - logf(s); }
};

__device__ __forceinline__ void write_stats(const LogProbArgs &a, int64_t at, const Stats &st, int64_t t, float x_t) {
  a.log_probs[at] = t == a.ignore_index ? 0.f : t < 0 || t >= a.C ? NAN : st.log_prob(x_t);
  a.entropy[at] = st.entropy();
  if (a.stats) a.stats[at] = make_float2(Stats::base(st.m), st.s);
}

// ---- rows ------------------------------------------------------------------------------------------------------------
// A thread's part of a tile: V vectors of logits in registers.
template <typename T, int V> struct Tile {
  static constexpr int N = RowVector<T>::N;
  RowVector<T> v[V];
  // The vectors at, at + step, ... below `end`; the others are -inf.
  __device__ __forceinline__ void load(const T *row, int at, int step, int end, int shift, int C) {
    const T *p = row + ((int64_t)at * N - shift);
    if (at * N >= shift && at + (V - 1) * step < end && (at + (V - 1) * step) * N - shift + N <= C) {
#pragma unroll
      for (int i = 0; i < V; i++) v[i].u = *(const uint4 *)(p + i * step * N);
    } else {
      const T none = from_float<T>(-INFINITY);
#pragma unroll
      for (int i = 0; i < V; i++) v[i].load(row, at + i * step < end ? (at + i * step) * N - shift : C, C, none);
    }
  }
  __device__ __forceinline__ float largest() const {
    if constexpr (sizeof(T) == 4) {
      float m = v[0].at(0);
#pragma unroll
      for (int i = 0; i < V; i++)
#pragma unroll
        for (int j = 0; j < N; j++) m = max_nan(m, v[i].at(j));
      return m;
    } else {  // two at once
      auto m = word_as_two<T>(v[0].u.x);
#pragma unroll
      for (int i = 0; i < V; i++) {
        m = __hmax2_nan(m, word_as_two<T>(v[i].u.x));
        m = __hmax2_nan(m, word_as_two<T>(v[i].u.y));
        m = __hmax2_nan(m, word_as_two<T>(v[i].u.z));
        m = __hmax2_nan(m, word_as_two<T>(v[i].u.w));
      }
      return max_nan(to_float(m.x), to_float(m.y));
    }
  }
  __device__ __forceinline__ void add_to(Stats &st, float largest) const {
    st.move_to(max_nan(st.m, largest));
    const float base = Stats::base(st.m);
    const float2 off = make_float2(-base, -base), scale = make_float2(kLog2e, kLog2e);
    float2 s = make_float2(0.f, 0.f), t = s;
#pragma unroll
    for (int i = 0; i < V; i++)
#pragma unroll
      for (int j = 0; j < N / 2; j++) {
        float2 d = mul_pair(add_pair(v[i].pair(j), off), scale);
        d.x = max_nan(d.x, kFar), d.y = max_nan(d.y, kFar);
        const float2 e = make_float2(exp2_fast(d.x), exp2_fast(d.y));
        s = add_pair(s, e);
        t = fma_pair(e, d, t);
      }
    st.s += s.x + s.y;
    st.t += t.x + t.y;
  }
  // f(order, index) for each logit of order `least` or better.
  template <class F> __device__ __forceinline__ void each(unsigned least, int at, int step, int end, int shift, int C, F f) const {
    const float bound = value_of(least);
#pragma unroll
    for (int i = 0; i < V; i++)
#pragma unroll
      for (int j = 0; j < N; j++) {
        const float value = v[i].at(j);
        if (value < bound) continue;  // (a bound that is NaN lets all pass)
        const unsigned o = order_of(value);
        const int index = (at + i * step) * N - shift + j;
        if (o >= least && at + i * step < end && index >= 0 && index < C) f(o, index);
      }
  }
};

// The k best of n candidates in shared memory, by counting for each how many are better (they are all different).
__device__ __forceinline__ void rank_candidates(const Candidate *from, int n, int k, Candidate *best) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const Candidate mine = from[i];
    int rank = 0;
    for (int j = 0; j < n; j++) rank += from[j] > mine;
    if (rank < k) best[rank] = mine;
  }
}

// The k-th largest of the lanes' values (k <= 32).
__device__ __forceinline__ unsigned kth_largest(unsigned v, int k) {
  unsigned most = 0;
  for (int i = 0; i < k; i++) {
    most = __reduce_max_sync(0xffffffffu, v);
    const unsigned who = __ballot_sync(0xffffffffu, v == most);
    if ((threadIdx.x & 31) == __ffs(who) - 1) v = 0;
  }
  return most;
}

constexpr int kRowThreads = 256, kMostTop = 32, kMostCandidates = 1024, kMostCluster = 16;

// A row belongs to a cluster of blocks (gridDim.x of them, one where there are rows enough); a block walks its run of vectors in
// tiles held in registers, each read once, the next one while it works on one.  With TOP (k > 0) it finds the best of each tile
// without looking at most of it: the k-th largest of the maxima of 32 groups of threads is a bound that k logits reach and few
// others do.  The blocks of a cluster put what they found into the first one's shared memory.  A few rows are latency: 8 x 131072
// float32 with the best eight take 7.7 us in clusters of 16 (4.2 without best; 15 where the first block fetched the others' lists one by
// one, 287 by one block a row in nine passes); 1000 x 32000 49 us (2.6 TB/s), by the barriers and scans of each row's first tile.
template <typename T, bool TOP> struct RowKernel {
  static constexpr int V = TOP ? 32 / RowVector<T>::N : 4, TILE = kRowThreads * V * RowVector<T>::N;  // logits of a tile
};
template <typename T, bool TOP> __global__ void __launch_bounds__(kRowThreads, TOP ? 3 : 4) log_probs_rows_kernel(LogProbArgs a) {
  constexpr int V = RowKernel<T, TOP>::V;
  __shared__ float4 stats[8], parts[kMostCluster], whole;
  __shared__ unsigned group_best[32];
  __shared__ Candidate best[2][kMostTop];
  __shared__ Candidate pool[TOP ? kMostCandidates : 1], gathered[TOP ? kMostCluster * kMostTop : 1];
  __shared__ int pooled;
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = (int)gridDim.x, part = (int)blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
  if (row >= a.outer) return;  // (the whole cluster)
  if (blocks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // I have started
  const T *x = (const T *)a.x + row * a.x_stride;
  const int shift = RowVector<T>::shift_of(x), vectors = (int)(((int64_t)a.C + shift + RowVector<T>::N - 1) / RowVector<T>::N);
  const int per = (vectors + blocks - 1) / blocks, from = min(part * per, vectors), end = min(from + per, vectors);
  Stats st;
  int have = 0, now = 0;  // candidates kept so far, in best[now]
  Tile<T, V> tile;
  tile.load(x, from + threadIdx.x, kRowThreads, end, shift, a.C);
  // (two loads behind one another that would otherwise wait at the end)
  const int64_t target = threadIdx.x == 0 && part == 0 ? a.target[row] : -1;
  const float x_t = target >= 0 && target < a.C ? to_float(x[target]) : 0.f;
  constexpr int STEP = kRowThreads * V;
  if (!TOP) {
    for (int v0 = from; v0 < end; v0 += 2 * STEP) {
      Tile<T, V> next;
      next.load(x, v0 + STEP + threadIdx.x, kRowThreads, end, shift, a.C);
      tile.add_to(st, tile.largest());
      tile.load(x, v0 + 2 * STEP + threadIdx.x, kRowThreads, end, shift, a.C);
      next.add_to(st, next.largest());
    }
  }
  for (int v0 = from; TOP && v0 < end; v0 += STEP) {
    const int at = v0 + threadIdx.x;
    const float largest = tile.largest();
    // Once there are k, only what is better than the worst of them counts, and most tiles have nothing of that.
    const unsigned mine = order_of(largest);
    const bool full = have == a.k;
    const Candidate worst = full ? best[now][a.k - 1] : 0;
    if (!full || __syncthreads_or(mine >= (unsigned)(worst >> 32))) {
      if (!full) {
        unsigned o = mine;
#pragma unroll
        for (int d = 4; d > 0; d >>= 1) o = max(o, __shfl_xor_sync(0xffffffffu, o, d));
        if ((lane & 7) == 0) group_best[threadIdx.x >> 3] = o;
      }
      if (threadIdx.x < have) pool[threadIdx.x] = best[now][threadIdx.x];
      if (threadIdx.x == 0) pooled = have;
      __syncthreads();
      const unsigned least = full ? (unsigned)(worst >> 32) : kth_largest(group_best[lane], a.k);
      if (mine >= least)
        tile.each(least, at, kRowThreads, end, shift, a.C, [&](unsigned order, int index) {
          const Candidate c = candidate(order, index);
          if (c > worst) {
            const int to = atomicAdd(&pooled, 1);
            if (to < kMostCandidates) pool[to] = c;
          }
        });
      __syncthreads();
      const int n = pooled;
      if (n <= kMostCandidates) {
        rank_candidates(pool, n, a.k, best[now ^ 1]);
        have = min(n, a.k);
      } else {  // very many alike: one after the other, each the best below the last
        Candidate last = ~0ull;
        for (int i = 0; i < a.k; i++) {
          Candidate c = 0;
          if (threadIdx.x < have && best[now][threadIdx.x] < last) c = best[now][threadIdx.x];
          tile.each(0, at, kRowThreads, end, shift, a.C, [&](unsigned order, int index) {
            const Candidate q = candidate(order, index);
            if (q < last && q > c) c = q;
          });
#pragma unroll
          for (int d = 16; d > 0; d >>= 1) {
            const Candidate o2 = __shfl_xor_sync(0xffffffffu, c, d);
            c = o2 > c ? o2 : c;
          }
          __syncthreads();
          if (lane == 0) pool[warp] = c;
          __syncthreads();
          c = pool[0];
          for (int w = 1; w < 8; w++) c = pool[w] > c ? pool[w] : c;
          last = c;
          if (threadIdx.x == 0) best[now ^ 1][i] = c;
        }
        have = a.k;
      }
      now ^= 1;
      __syncthreads();
    }
    tile.add_to(st, largest);
    if (v0 + STEP < end) tile.load(x, at + STEP, kRowThreads, end, shift, a.C);
  }
  st.join_warp();
  if (lane == 0) stats[warp] = st.packed();
  __syncthreads();
  if (blocks > 1) {
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // every block has started, so its shared memory may be written
    if (warp == 0) {
      st = Stats::of(stats[lane & 7]);
      st.join_lanes(8);
      if (lane == 0) cluster.map_shared_rank(&parts[0], 0)[part] = st.packed();
    }
    if (TOP && threadIdx.x < a.k)
      cluster.map_shared_rank(&gathered[0], 0)[part * a.k + threadIdx.x] = threadIdx.x < have ? best[now][threadIdx.x] : 0;
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (part != 0) return;
    if (TOP) {
      rank_candidates(gathered, blocks * a.k, a.k, best[now ^ 1]);
      now ^= 1;
    }
  }
  if (warp == 0) {
    const int n = blocks > 1 ? blocks : 8;
    st = lane < n ? Stats::of(blocks > 1 ? parts[lane] : stats[lane]) : Stats();
    st.join_lanes(kMostCluster);
    if (lane == 0) {
      whole = st.packed();
      write_stats(a, row, st, target, x_t);
    }
  }
  if (!TOP) return;
  __syncthreads();
  if (threadIdx.x < a.k) {
    const Candidate c = best[now][threadIdx.x];
    a.top_index[row * a.k + threadIdx.x] = candidate_index(c);
    a.top[row * a.k + threadIdx.x] = Stats::of(whole).log_prob(value_of((unsigned)(c >> 32)));
  }
}

// Many rows without best classes: the blocks walk over the rows, and their next tiles, of the next rows too, are on their way into
// shared memory, where every thread reads what it has copied itself.  4096 x 32000 bf16 take 59 us (4.4 TB/s): 45 us of loads; of the
// exponentials (131M at 16 a cycle of an SM are 29 us) and of issue not all hides behind them; with a block a row 66 us.
constexpr int kRowStages = 3, kStreamThreads = 128, kStreamBlocks = 8;
template <typename T> __global__ void __launch_bounds__(kStreamThreads, kStreamBlocks) log_probs_stream_kernel(LogProbArgs a) {
  constexpr int V = 4, N = RowVector<T>::N, STEP = kStreamThreads * V;
  extern __shared__ __align__(16) unsigned char row_memory[];
  __shared__ float4 stats[2][kStreamThreads / 32];
  RowVector<T> *slots = (RowVector<T> *)row_memory + threadIdx.x;  // (stage, vector) x threads
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T none = from_float<T>(-INFINITY);
  struct Place {  // a tile
    int64_t row;
    int v0, shift, vectors;
    const T *x;
    __device__ __forceinline__ void open(const LogProbArgs &a, int64_t r) {
      row = r, v0 = 0;
      x = (const T *)a.x + r * a.x_stride;
      shift = RowVector<T>::shift_of(x);
      vectors = (int)(((int64_t)a.C + shift + N - 1) / N);
    }
    __device__ __forceinline__ void next(const LogProbArgs &a) {
      v0 += STEP;
      if (v0 >= vectors) open(a, row + gridDim.x);
    }
  };
  Place ahead, here;
  ahead.open(a, blockIdx.x);
  here = ahead;
  const auto copy = [&](int stage) {
    if (ahead.row < a.outer) {
#pragma unroll
      for (int i = 0; i < V; i++) {
        const int at = ahead.v0 + i * kStreamThreads + threadIdx.x, first = at * N - ahead.shift;
        RowVector<T> *to = slots + (stage * V + i) * kStreamThreads;
        if (first >= 0 && first + N <= a.C)
          copy_16(to, ahead.x + first);
        else if (at < ahead.vectors)
          for (int j = 0; j < N; j++) to->t[j] = first + j >= 0 && first + j < a.C ? ahead.x[first + j] : none;
      }
      ahead.next(a);
    }
    copies_end();
  };
  for (int d = 0; d < kRowStages - 1; d++) copy(d);
  Stats st;
  int stage = 0, turn = 0;
  // the row's target and its logit, the first fetched a row ahead
  int64_t target = -1, target_next = threadIdx.x == 0 && here.row < a.outer ? a.target[here.row] : -1;
  float x_t = 0.f;
  while (here.row < a.outer) {
    if (threadIdx.x == 0 && here.v0 == 0) {
      target = target_next;
      x_t = target >= 0 && target < a.C ? to_float(here.x[target]) : 0.f;
      if (here.row + gridDim.x < a.outer) target_next = a.target[here.row + gridDim.x];
    }
    copy(stage == 0 ? kRowStages - 1 : stage - 1);
    copies_wait<kRowStages - 1>();
    Tile<T, V> tile;
#pragma unroll
    for (int i = 0; i < V; i++) {
      if (here.v0 + i * kStreamThreads + (int)threadIdx.x < here.vectors) {
        tile.v[i].u = slots[(stage * V + i) * kStreamThreads].u;
      } else {
#pragma unroll
        for (int j = 0; j < N; j++) tile.v[i].t[j] = none;
      }
    }
    tile.add_to(st, tile.largest());
    stage = stage == kRowStages - 1 ? 0 : stage + 1;
    const int64_t row = here.row;
    here.next(a);
    if (here.row == row) continue;
    st.join_warp();
    if (lane == 0) stats[turn][warp] = st.packed();
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int i = 1; i < kStreamThreads / 32; i++) st.join(Stats::of(stats[turn][i]));
      write_stats(a, row, st, target, x_t);
    }
    st = Stats();
    turn ^= 1;
  }
}

// Rows of up to 1024 classes: a warp each (or `lanes` of one, a power of two, where no best are asked for), their logits in
// registers; the best by the same bound, of the maxima of the lanes.
template <typename T, bool TOP, int E> __global__ void __launch_bounds__(256, TOP ? 2 : 4) log_probs_warp_kernel(LogProbArgs a, int lanes) {
  constexpr int V = E / RowVector<T>::N, POOL = 96;
  __shared__ Candidate pools[TOP ? 8 : 1][POOL];
  __shared__ int counts[8];
  if (TOP) lanes = 32;
  const int lane = threadIdx.x & (lanes - 1), warp = threadIdx.x >> 5;
  const int64_t row = (int64_t)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
  const bool on = row < a.outer;
  if (TOP && !on) return;
  const T *x = (const T *)a.x + (on ? row : 0) * a.x_stride;
  const int shift = RowVector<T>::shift_of(x), vectors = on ? (a.C + shift + RowVector<T>::N - 1) / RowVector<T>::N : 0;
  Tile<T, V> tile;
  tile.load(x, lane, lanes, vectors, shift, a.C);
  const int64_t t = on ? a.target[row] : -1;
  const float x_t = t >= 0 && t < a.C ? to_float(x[t]) : 0.f, largest = tile.largest();
  Stats st;
  tile.add_to(st, largest);
  st.join_lanes(lanes);
  if (lane == 0 && on) write_stats(a, row, st, t, x_t);
  if (!TOP) return;
  const auto put = [&](int i, Candidate c) {
    a.top_index[row * a.k + i] = candidate_index(c);
    a.top[row * a.k + i] = st.log_prob(value_of((unsigned)(c >> 32)));
  };
  Candidate *pool = pools[TOP ? warp : 0];
  int n = POOL + 1;
  if (a.k <= 32) {
    const unsigned mine = order_of(largest), least = kth_largest(mine, a.k);
    if (lane == 0) counts[warp] = 0;
    __syncwarp();
    if (mine >= least)
      tile.each(least, lane, 32, vectors, shift, a.C, [&](unsigned order, int index) {
        const int to = atomicAdd(&counts[warp], 1);
        if (to < POOL) pool[to] = candidate(order, index);
      });
    __syncwarp();
    n = counts[warp];
  }
  if (n <= POOL) {
    for (int i = lane; i < n; i += 32) {
      const Candidate c = pool[i];
      int rank = 0;
      for (int j = 0; j < n; j++) rank += pool[j] > c;
      if (rank < a.k) put(rank, c);
    }
    return;
  }
  Candidate last = ~0ull;  // very many alike, or wanted: each the best below the last
  for (int i = 0; i < a.k; i++) {
    Candidate c = 0;
    tile.each(0, lane, 32, vectors, shift, a.C, [&](unsigned order, int index) {
      const Candidate q = candidate(order, index);
      if (q < last && q > c) c = q;
    });
    const unsigned order = __reduce_max_sync(0xffffffffu, (unsigned)(c >> 32));
    const unsigned index = __reduce_max_sync(0xffffffffu, (unsigned)(c >> 32) == order ? (unsigned)c : 0u);
    last = (Candidate)order << 32 | index;
    if (lane == 0) put(i, last);
  }
}

// More of the best than the kernels above keep: a block a row, and after the statistics a pass over the row for each of them, which
// finds the best below the last.  Reads from L2 by one SM bound it: 8 x 131072 float32 with the best 50 take 1.9 ms, 39 us each.
template <typename T> __global__ void __launch_bounds__(256) log_probs_many_kernel(LogProbArgs a) {
  __shared__ Candidate best[8];
  __shared__ float4 stats[8];
  const int64_t row = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T *x = (const T *)a.x + row * a.x_stride;
  Stats st;
  for (int c = threadIdx.x; c < a.C; c += 256) st.add(to_float(x[c]));
  st.join_warp();
  if (lane == 0) stats[warp] = st.packed();
  __syncthreads();
  st = Stats::of(stats[0]);
  for (int i = 1; i < 8; i++) st.join(Stats::of(stats[i]));
  if (threadIdx.x == 0) {
    const int64_t t = a.target[row];
    write_stats(a, row, st, t, t >= 0 && t < a.C ? to_float(x[t]) : 0.f);
  }
  Candidate last = ~0ull;
  for (int i = 0; i < a.k; i++) {
    Candidate mine = 0;
    for (int c = threadIdx.x; c < a.C; c += 256) {
      const Candidate q = candidate(order_of(to_float(x[c])), c);
      if (q < last && q > mine) mine = q;
    }
    for (int d = 16; d > 0; d >>= 1) {
      const Candidate o = __shfl_xor_sync(0xffffffffu, mine, d);
      if (o > mine) mine = o;
    }
    if (lane == 0) best[warp] = mine;
    __syncthreads();
    last = best[0];
    for (int w = 1; w < 8; w++)
      if (best[w] > last) last = best[w];
    __syncthreads();
    if (threadIdx.x == 0) {
      a.top_index[row * a.k + i] = candidate_index(last);
      a.top[row * a.k + i] = st.log_prob(value_of((unsigned)(last >> 32)));
    }
  }
}

// ---- planes ----------------------------------------------------------------------------------------------------------
// P neighbouring pixels of a channel: four where planes are aligned for that, else one.
template <typename T, int P> union PixelVector {
  T t[P];
  uint4 q;
  uint2 d;
  __device__ __forceinline__ PixelVector() {}
  __device__ __forceinline__ void load(const T *p) {
    if constexpr (P == 1) t[0] = *p;
    else if constexpr (sizeof(T) == 4) q = *(const uint4 *)p;
    else d = *(const uint2 *)p;
  }
  __device__ __forceinline__ void store(T *p) const {
    if constexpr (P == 1) *p = t[0];
    else if constexpr (sizeof(T) == 4) *(uint4 *)p = q;
    else *(uint2 *)p = d;
  }
};
// Numbers of pixels into their image and the rest.
struct PlaneIndex {
  FastDiv by;
  int64_t inner;
  bool small;
  static PlaneIndex of(int64_t outer, int64_t inner) {
    const bool small = outer * inner < ((int64_t)1 << 31);
    return PlaneIndex{FastDiv::make(small ? (unsigned)inner : 1u), inner, small};
  }
  __device__ __forceinline__ int64_t image(int64_t at) const { return small ? (int64_t)by.div((unsigned)at) : at / inner; }
};

// The K best logits of a pixel so far, the best first; of equal ones the first that came.
template <int K> struct Best {
  unsigned order[K];
  int index[K];
  __device__ __forceinline__ Best() {
#pragma unroll
    for (int i = 0; i < K; i++) order[i] = 0, index[i] = -1;
  }
  __device__ __forceinline__ void take(float v, int c) {
    const unsigned o = order_of(v);
    if (o <= order[K - 1]) return;  // (every order is above 0)
#pragma unroll
    for (int i = K - 1; i >= 0; i--) {
      const bool here = o > order[i], above = i > 0 && o > order[i > 0 ? i - 1 : 0];
      order[i] = above ? order[i > 0 ? i - 1 : 0] : here ? o : order[i];
      index[i] = above ? index[i > 0 ? i - 1 : 0] : here ? c : index[i];
    }
  }
  __device__ __forceinline__ int class_at(int j) const { return index[j]; }
  __device__ __forceinline__ float value_at(int j) const { return value_of(order[j]); }
};
// The same of 16-bit logits of up to 65536 classes, in one word each: the order of the logit's 16 bits above, the class counted from
// the last below.  (40 classes of 2.1M bf16 pixels, the best eight: 292 us in two words, 252 in one.)
template <typename T, int K> struct BestPacked {
  unsigned key[K];
  __device__ __forceinline__ BestPacked() {
#pragma unroll
    for (int i = 0; i < K; i++) key[i] = 0;
  }
  __device__ __forceinline__ void take(T v, int c) {
    const float f = to_float(v);
    const unsigned bits = f == 0.f ? 0u : (unsigned)*reinterpret_cast<const unsigned short *>(&v);
    unsigned x = (f != f ? 0xffff0000u : (bits & 0x8000u ? ~bits & 0xffffu : bits | 0x8000u) << 16) | (0xffffu - (unsigned)c);
    if (x <= key[K - 1]) return;
#pragma unroll
    for (int i = 0; i < K; i++) {
      const unsigned most = max(key[i], x);
      x = min(key[i], x);
      key[i] = most;
    }
  }
  __device__ __forceinline__ int class_at(int j) const { return (int)(0xffffu - (key[j] & 0xffffu)); }
  __device__ __forceinline__ float value_at(int j) const {
    const unsigned o = key[j] >> 16;
    const unsigned short bits = (unsigned short)(o & 0x8000u ? o & 0x7fffu : ~o);
    return o == 0xffffu ? NAN : to_float(*reinterpret_cast<const T *>(&bits));
  }
};

// Channels read at once; by a thread of one pixel that keeps the best, which has fewer bytes on their way for its work, twice as
// many (20503 bf16 pixels of 41 classes, the best three: 8.0 us by eight, 6.4 by sixteen; without best 71 us by eight, 81 by sixteen
// for 2.1M pixels of 40).
constexpr int kPlaneChannels = 8;

// A thread has P pixels and walks over their channels, some at a time; with K > 0 it keeps the K best of them on
// the way.  8 x 13 x 512 x 1024 float32 take 68 us (4.7 TB/s with targets and results) and 91 backward (6.1 TB/s).
template <typename T, int P, int K, bool PACKED> __global__ void __launch_bounds__(128) log_probs_planes_kernel(LogProbArgs a, PlaneIndex index) {
  constexpr int CHANNELS = P == 1 && K > 0 ? 2 * kPlaneChannels : kPlaneChannels;
  const int64_t at = ((int64_t)blockIdx.x * 128 + threadIdx.x) * P;
  if (at >= a.outer * a.inner) return;
  const int64_t o = index.image(at), i = at - o * a.inner;
  const T *x = (const T *)a.x + o * a.C * a.inner + i;
  Stats st[P];
  typename std::conditional<PACKED, BestPacked<T, K ? K : 1>, Best<K ? K : 1>>::type best[P];
  int64_t target[P];
  float x_t[P];  // the target's logit, found on the way
#pragma unroll
  for (int p = 0; p < P; p++) target[p] = a.target[at + p], x_t[p] = 0.f;
  for (int c0 = 0; c0 < a.C; c0 += CHANNELS) {
    PixelVector<T, P> v[CHANNELS];
#pragma unroll
    for (int c = 0; c < CHANNELS; c++) {
      if (c0 + c < a.C) {
        v[c].load(x + (c0 + c) * a.inner);
      } else {
#pragma unroll
        for (int p = 0; p < P; p++) v[c].t[p] = from_float<T>(-INFINITY);
      }
    }
#pragma unroll
    for (int p = 0; p < P; p++) {
      float most = to_float(v[0].t[p]);
#pragma unroll
      for (int c = 1; c < CHANNELS; c++) most = max_nan(most, to_float(v[c].t[p]));
      st[p].move_to(max_nan(st[p].m, most));
      const float base = Stats::base(st[p].m);
#pragma unroll
      for (int c = 0; c < CHANNELS; c++) {
        const float d = distance(to_float(v[c].t[p]), base), e = exp2_fast(d);
        st[p].s += e;
        st[p].t = fmaf(e, d, st[p].t);
        if (c0 + c == (int)target[p]) x_t[p] = to_float(v[c].t[p]);  // (a target beyond 32 bits is none of the classes, and its logit not looked at)
        if (K > 0 && c0 + c < a.C) {  // (asking first whether the largest of the eight is better costs more than it saves)
          if constexpr (PACKED) best[p].take(v[c].t[p], c0 + c);
          else best[p].take(to_float(v[c].t[p]), c0 + c);
        }
      }
    }
  }
#pragma unroll
  for (int p = 0; p < P; p++) {
    write_stats(a, at + p, st[p], target[p], x_t[p]);
#pragma unroll
    for (int j = 0; j < K; j++)
      if (j < a.k) {
        const int64_t to = (o * a.k + j) * a.inner + i + p;
        a.top_index[to] = best[p].class_at(j);
        a.top[to] = st[p].log_prob(best[p].value_at(j));
      }
  }
}

// The best beyond the first eight, eight more in each pass over the channels: those that come after the last.
template <typename T> __global__ void __launch_bounds__(128) log_probs_planes_more_kernel(LogProbArgs a, PlaneIndex index) {
  const int64_t at = (int64_t)blockIdx.x * 128 + threadIdx.x;
  if (at >= a.outer * a.inner) return;
  const int64_t o = index.image(at), i = at - o * a.inner;
  const T *x = (const T *)a.x + o * a.C * a.inner + i;
  Stats st;
  for (int c = 0; c < a.C; c++) st.add(to_float(x[c * a.inner]));
  int64_t to = (o * a.k + 7) * a.inner + i;
  int last = (int)a.top_index[to];
  for (int done = 8; done < a.k; done += 8) {
    const unsigned least = order_of(to_float(x[last * a.inner]));
    Best<8> best;
    for (int c = 0; c < a.C; c++) {
      const unsigned order = order_of(to_float(x[c * a.inner]));
      if (order < least || (order == least && c > last)) best.take(to_float(x[c * a.inner]), c);
    }
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (done + j < a.k) {
        to += a.inner;
        last = best.class_at(j);
        a.top_index[to] = last;
        a.top[to] = st.log_prob(best.value_at(j));
      }
  }
}

template <typename T, int P, bool PACKED> void launch_planes(const LogProbArgs &a, cudaStream_t st) {
  const PlaneIndex index = PlaneIndex::of(a.outer, a.inner);
  const int64_t threads = a.outer * a.inner / P;
  const unsigned blocks = (unsigned)((threads + 127) / 128);
  if (a.k == 0)
    log_probs_planes_kernel<T, P, 0, false><<<blocks, 128, 0, st>>>(a, index);
  else if (a.k == 1)
    log_probs_planes_kernel<T, P, 1, PACKED><<<blocks, 128, 0, st>>>(a, index);
  else if constexpr (P == 1 || PACKED) {  // (lists of four pixels in two words each would not fit the registers)
    if (a.k <= 4)
      log_probs_planes_kernel<T, P, 4, PACKED><<<blocks, 128, 0, st>>>(a, index);
    else
      log_probs_planes_kernel<T, P, 8, PACKED><<<blocks, 128, 0, st>>>(a, index);
  }
}
template <typename T> bool planes_of_four(int64_t inner, const void *x, const void *gx = nullptr) {
  return inner % 4 == 0 && ((uintptr_t)x | (uintptr_t)gx) % (4 * sizeof(T)) == 0;
}
// Kernels launched.
template <typename T> int launch_planes(const LogProbArgs &a, cudaStream_t st) {
  const bool four = planes_of_four<T>(a.inner, a.x);
  if constexpr (sizeof(T) == 2) {
    if (a.C <= 65536)
      four ? launch_planes<T, 4, true>(a, st) : launch_planes<T, 1, true>(a, st);
    else
      launch_planes<T, 1, false>(a, st);
  } else {
    four && a.k <= 1 ? launch_planes<T, 4, false>(a, st) : launch_planes<T, 1, false>(a, st);
  }
  if (a.k <= 8) return 1;
  log_probs_planes_more_kernel<T><<<(unsigned)((a.outer * a.inner + 127) / 128), 128, 0, st>>>(a, PlaneIndex::of(a.outer, a.inner));
  return 2;
}

// ---- gradient --------------------------------------------------------------------------------------------------------
struct LogProbGradArgs {
  const void *x;
  const int64_t *target, *top_index;
  const float2 *stats;
  const float *entropy, *g, *h, *t;
  void *gx;
  int64_t outer, inner, x_stride, ignore_index, g_stride, h_stride;  // g_stride, h_stride: 1, or 0 for one value for all
  int C, k;
};

// What the elements of one distribution share.  With e = 2^d, d = (x - m) log2 e, p = e / S and log p = ln2 d - ln S:
//     -p (g + sum t + h (log p + H)) = e (flat + slope d)
struct RowGrad {
  float m, flat, slope, g;
  int64_t target;
  bool tops;
  __device__ __forceinline__ float of(float x) const {
    const float d = distance(x, m);
    return exp2_fast(d) * fmaf(slope, d, flat);
  }
  __device__ __forceinline__ float2 of(float2 x) const {
    float2 d = mul_pair(add_pair(x, make_float2(-m, -m)), make_float2(kLog2e, kLog2e));
    d.x = max_nan(d.x, kFar), d.y = max_nan(d.y, kFar);
    return mul_pair(make_float2(exp2_fast(d.x), exp2_fast(d.y)), fma_pair(make_float2(slope, slope), d, make_float2(flat, flat)));
  }
};
// `at`: the distribution's number, `o`, `i`: its parts.
__device__ __forceinline__ RowGrad row_grad(const LogProbGradArgs &a, int64_t at, int64_t o, int64_t i) {
  RowGrad r;
  const float2 st = a.stats[at];
  const bool empty = st.y == 0.f;
  r.m = st.x;
  r.target = a.target[at];
  r.tops = a.t != nullptr && !empty;
  r.g = !a.g || empty || r.target == a.ignore_index ? 0.f : r.target < 0 || r.target >= a.C ? NAN : a.g[at * a.g_stride];
  const float h = a.h && !empty ? a.h[at * a.h_stride] : 0.f;
  float all = r.g;
  if (r.tops)
    for (int j = 0; j < a.k; j++) all += a.t[(o * a.k + j) * a.inner + i];
  const float inverse = empty ? 0.f : 1.f / st.y;
  r.slope = -h * kLn2 * inverse;
  r.flat = empty ? 0.f : -(all + h * (a.entropy[at] - logf(st.y))) * inverse;
  return r;
}
// The class c's own gradients: the target's, and those of the most probable classes.
__device__ __forceinline__ float own_grad(const LogProbGradArgs &a, const RowGrad &r, int64_t o, int64_t i, int c) {
  float v = c == r.target ? r.g : 0.f;
  if (r.tops)
    for (int j = 0; j < a.k; j++) {
      const int64_t at = (o * a.k + j) * a.inner + i;
      if (a.top_index[at] == c) v += a.t[at];
    }
  return v;
}

// A block takes a run of a row's vectors; the most probable classes are put right behind it.  HBM bounds it: 4096 x 32000 bf16 take
// 79 us (6.7 TB/s).
template <typename T> __global__ void __launch_bounds__(256) log_probs_rows_grad_kernel(LogProbGradArgs a) {
  constexpr int N = RowVector<T>::N;
  const int64_t row = blockIdx.y + (int64_t)blockIdx.z * gridDim.y;
  if (row >= a.outer) return;
  const T *x = (const T *)a.x + row * a.x_stride;
  T *gx = (T *)a.gx + row * a.C;
  const RowGrad r = row_grad(a, row, row, 0);
  const int shift = RowVector<T>::shift_of(gx), vectors = (int)(((int64_t)a.C + shift + N - 1) / N);
  const bool alike = RowVector<T>::shift_of(x) == shift;
  const int per = (vectors + (int)gridDim.x - 1) / (int)gridDim.x, from = min((int)blockIdx.x * per, vectors), end = min(from + per, vectors);
  const T none = from_float<T>(-INFINITY);
  const int target = r.target >= 0 && r.target < a.C ? (int)r.target : -1;
  for (int v0 = from; v0 < end; v0 += 256 * 4) {
    RowVector<T> v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int at = v0 + i * 256 + threadIdx.x, first = at < end ? at * N - shift : a.C;
      if (alike) {
        v[i].load(x, first, a.C, none);
      } else {
#pragma unroll
        for (int j = 0; j < N; j++) v[i].t[j] = first + j >= 0 && first + j < a.C ? x[first + j] : none;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int at = v0 + i * 256 + threadIdx.x, first = at < end ? at * N - shift : a.C;
      const bool here = target >= first && target < first + N;
      const float g_t = here ? r.of(v[i].at_any(target - first)) + r.g : 0.f;
#pragma unroll
      for (int j = 0; j < N / 2; j++) v[i].set_pair(j, r.of(v[i].pair(j)));
      if (here) v[i].set_any(target - first, g_t);
      v[i].store(gx, first, a.C);
    }
  }
  if (!r.tops) return;
  __syncthreads();
  for (int j = threadIdx.x; j < a.k; j += 256) {
    const int64_t c = a.top_index[row * a.k + j];
    if (c < 0 || c >= a.C) continue;
    const int v = (int)((c + shift) / N);
    if (v >= from && v < end) gx[c] = from_float<T>(r.of(to_float(x[c])) + own_grad(a, r, row, 0, (int)c));
  }
}

// A thread has P pixels, as in the forward pass.
template <typename T, int P> __global__ void __launch_bounds__(128) log_probs_planes_grad_kernel(LogProbGradArgs a, PlaneIndex index) {
  constexpr int CHANNELS = kPlaneChannels;
  const int64_t at = ((int64_t)blockIdx.x * 128 + threadIdx.x) * P;
  if (at >= a.outer * a.inner) return;
  const int64_t o = index.image(at), i = at - o * a.inner, base = o * a.C * a.inner + i;
  const T *x = (const T *)a.x + base;
  T *gx = (T *)a.gx + base;
  PixelVector<T, P> v[CHANNELS];
  const auto read = [&](int c0) {
#pragma unroll
    for (int c = 0; c < CHANNELS; c++)
      if (c0 + c < a.C) v[c].load(x + (c0 + c) * a.inner);
  };
  read(0);  // (on their way while what the pixels share is read)
  RowGrad r[P];
  int target[P];
#pragma unroll
  for (int p = 0; p < P; p++) {
    r[p] = row_grad(a, at + p, o, i + p);
    target[p] = r[p].target >= 0 && r[p].target < a.C ? (int)r[p].target : -1;
  }
  for (int c0 = 0; c0 < a.C; c0 += CHANNELS) {
    if (c0 > 0) read(c0);
#pragma unroll
    for (int c = 0; c < CHANNELS; c++)
      if (c0 + c < a.C) {
#pragma unroll
        for (int p = 0; p < P; p++) {
          const float d = r[p].of(to_float(v[c].t[p]));
          v[c].t[p] = from_float<T>(c0 + c == target[p] ? d + r[p].g : d);
        }
        v[c].store(gx + (c0 + c) * a.inner);
      }
  }
#pragma unroll
  for (int p = 0; p < P; p++)  // the most probable classes right behind
    if (r[p].tops)
      for (int j = 0; j < a.k; j++) {
        const int64_t c = a.top_index[(o * a.k + j) * a.inner + i + p];
        if (c >= 0 && c < a.C)
          gx[c * a.inner + p] = from_float<T>(r[p].of(to_float(x[c * a.inner + p])) + own_grad(a, r[p], o, i + p, (int)c));
      }
}
template <typename T> void launch_planes_grad(const LogProbGradArgs &a, cudaStream_t st) {
  const PlaneIndex index = PlaneIndex::of(a.outer, a.inner);
  const int64_t pixels = a.outer * a.inner;
  if (planes_of_four<T>(a.inner, a.x, a.gx))
    log_probs_planes_grad_kernel<T, 4><<<(unsigned)((pixels / 4 + 127) / 128), 128, 0, st>>>(a, index);
  else
    log_probs_planes_grad_kernel<T, 1><<<(unsigned)((pixels + 127) / 128), 128, 0, st>>>(a, index);
}

// Rows of up to 1024 classes: `lanes` of a warp each.
template <typename T> __global__ void __launch_bounds__(256) log_probs_warp_grad_kernel(LogProbGradArgs a, int lanes) {
  constexpr int N = RowVector<T>::N;
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t row = (int64_t)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
  const bool on = row < a.outer;
  const T *x = (const T *)a.x + (on ? row : 0) * a.x_stride;
  T *gx = (T *)a.gx + (on ? row : 0) * a.C;
  const RowGrad r = row_grad(a, on ? row : 0, on ? row : 0, 0);
  const int shift = RowVector<T>::shift_of(gx), vectors = on ? (a.C + shift + N - 1) / N : 0;
  const bool alike = RowVector<T>::shift_of(x) == shift;
  const T none = from_float<T>(-INFINITY);
  const int target = r.target >= 0 && r.target < a.C ? (int)r.target : -1;
  for (int at = lane; at < vectors; at += lanes) {
    const int first = at * N - shift;
    RowVector<T> v;
    if (alike) {
      v.load(x, first, a.C, none);
    } else {
#pragma unroll
      for (int j = 0; j < N; j++) v.t[j] = first + j >= 0 && first + j < a.C ? x[first + j] : none;
    }
    const bool here = target >= first && target < first + N;
    const float g_t = here ? r.of(v.at_any(target - first)) + r.g : 0.f;
#pragma unroll
    for (int j = 0; j < N / 2; j++) v.set_pair(j, r.of(v.pair(j)));
    if (here) v.set_any(target - first, g_t);
    v.store(gx, first, a.C);
  }
  if (!a.t) return;
  __syncwarp();
  for (int j = lane; j < a.k && on && r.tops; j += lanes) {
    const int64_t c = a.top_index[row * a.k + j];
    if (c >= 0 && c < a.C) gx[c] = from_float<T>(r.of(to_float(x[c])) + own_grad(a, r, row, 0, (int)c));
  }
}
// Lanes for a row: eight classes each, and what a row's start may take of a vector.
template <typename T> int row_lanes(int64_t C) {
  int n = 1;
  while (n < 32 && 8 * n < C + RowVector<T>::N - 1) n *= 2;
  return n;
}

// Blocks for a row: enough for two on each SM, no more than the row has tiles.
inline int blocks_per_row(int64_t rows, int64_t C, int64_t tile, int most) {
  const int64_t tiles = (C + tile - 1) / tile;
  int n = 1;
  while (n < most && n < tiles && n * rows < 2 * 148) n *= 2;
  return n;
}
// Rows as a grid's second and third dimension.
inline dim3 row_grid(int n, int64_t rows) {
  const unsigned y = rows < 65535 ? (unsigned)rows : 65535u;
  return dim3((unsigned)n, y, (unsigned)((rows + y - 1) / y));
}

template <typename T> cudaError_t launch_rows(const LogProbArgs &a, cudaStream_t st) {
  const int n = blocks_per_row(a.outer, a.C, a.k > 0 ? RowKernel<T, true>::TILE : RowKernel<T, false>::TILE, kMostCluster);
  if (a.k == 0 && n == 1) {
    constexpr int bytes = kRowStages * 4 * kStreamThreads * 16;
    static_assert(bytes <= 32768, "more needs an attribute of the kernel");
    log_probs_stream_kernel<T><<<(unsigned)std::min<int64_t>(a.outer, 148 * kStreamBlocks), kStreamThreads, bytes, st>>>(a);
    return cudaGetLastError();
  }
  void (*kernel)(LogProbArgs) = a.k > 0 ? log_probs_rows_kernel<T, true> : log_probs_rows_kernel<T, false>;
  cudaLaunchConfig_t config = {};
  config.gridDim = row_grid(n, a.outer);
  config.blockDim = dim3(kRowThreads);
  config.stream = st;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = (unsigned)n;
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  if (n > 8) {
    const cudaError_t e = cudaFuncSetAttribute((const void *)kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
  }
  return cudaLaunchKernelEx(&config, kernel, a);
}

inline int log_probs_sizes(int64_t outer, int64_t C, int64_t inner, int64_t k) {
  if (outer < 0 || C < 1 || inner < 1 || k < 0 || k > C) return SPH_ERR_INVALID_ARGUMENT;
  if (C >= ((int64_t)1 << 30) || outer >= ((int64_t)1 << 31) || inner >= ((int64_t)1 << 31)) return SPH_ERR_TOO_LARGE;
  if (outer > 0 && inner > (((int64_t)1 << 38) / outer)) return SPH_ERR_TOO_LARGE;
  return SPH_OK;
}

}  // namespace sph

using namespace sph;

extern "C" int sph_token_log_probs_forward(const void *x, const int64_t *target, float *log_probs, float *entropy, float *stats,
                                           float *top, int64_t *top_index, int64_t outer, int64_t C, int64_t inner, int64_t x_stride,
                                           int64_t k, int64_t ignore_index, int dtype, void *stream) {
  SPH_RANGE("sph_token_log_probs_forward");
  if (!element_dtype(dtype)) return SPH_ERR_UNSUPPORTED;
  if (const int rc = log_probs_sizes(outer, C, inner, k)) return rc;
  if (outer == 0) return SPH_OK;
  if (!x || !target || !log_probs || !entropy || (k > 0 && (!top || !top_index)) || (inner == 1 && outer > 1 && x_stride < C))
    return SPH_ERR_INVALID_ARGUMENT;
  const LogProbArgs a{x, target, log_probs, entropy, top, (float2 *)stats, top_index, outer, inner, x_stride, ignore_index, (int)C, (int)k};
  cudaStream_t st = (cudaStream_t)stream;
  int launches = 1;
  SPH_DISPATCH_ELEMENT(dtype, {
    if (inner == 1 && C <= 1024 - RowVector<T>::N) {  // (a row's start may take a part of a vector)
      const int lanes = k > 0 ? 32 : row_lanes<T>(C), rows = 256 / lanes;
      // (a lane has 16 logits where those are enough, else 32)
      (k > 0 ? log_probs_warp_kernel<T, true, 32> : C <= 512 - RowVector<T>::N ? log_probs_warp_kernel<T, false, 16> : log_probs_warp_kernel<T, false, 32>)<<<(unsigned)((outer + rows - 1) / rows), 256, 0, st>>>(a, lanes);
    } else if (inner == 1 && k > kMostTop)
      log_probs_many_kernel<T><<<(unsigned)outer, 256, 0, st>>>(a);
    else if (inner == 1) {
      if (launch_rows<T>(a, st) != cudaSuccess) {
        cudaGetLastError();
        return SPH_ERR_CUDA;
      }
    } else
      launches = launch_planes<T>(a, st);
  });
  return launch_status(launches);
}

extern "C" int sph_token_log_probs_backward(const void *x, const int64_t *target, const float *stats, const float *entropy,
                                            const int64_t *top_index, const float *g, int64_t g_stride, const float *h,
                                            int64_t h_stride, const float *t, void *gx, int64_t outer, int64_t C, int64_t inner,
                                            int64_t x_stride, int64_t k, int64_t ignore_index, int dtype, void *stream) {
  SPH_RANGE("sph_token_log_probs_backward");
  if (!element_dtype(dtype)) return SPH_ERR_UNSUPPORTED;
  if (const int rc = log_probs_sizes(outer, C, inner, k)) return rc;
  if (outer == 0) return SPH_OK;
  if (!x || !target || !stats || !entropy || !gx || (t && (k == 0 || !top_index)) || (inner == 1 && outer > 1 && x_stride < C) ||
      g_stride < 0 || g_stride > 1 || h_stride < 0 || h_stride > 1)
    return SPH_ERR_INVALID_ARGUMENT;
  const LogProbGradArgs a{x, target, top_index, (const float2 *)stats, entropy, g, h, t, gx, outer, inner, x_stride, ignore_index, g_stride, h_stride,
                          (int)C, (int)k};
  cudaStream_t st = (cudaStream_t)stream;
  SPH_DISPATCH_ELEMENT(dtype, {
    if (inner == 1 && C <= 1024 - RowVector<T>::N) {
      const int lanes = row_lanes<T>(C), rows = 256 / lanes;
      log_probs_warp_grad_kernel<T><<<(unsigned)((outer + rows - 1) / rows), 256, 0, st>>>(a, lanes);
    } else if (inner == 1)
      log_probs_rows_grad_kernel<T><<<row_grid(blocks_per_row(outer, C, 256 * RowVector<T>::N, 64), outer), 256, 0, st>>>(a);
    else
      launch_planes_grad<T>(a, st);
  });
  return launch_status();
}

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
#pragma once

#include <algorithm>

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
  int lanes;  // of a row that has a part of a warp
};

struct NormGradArgs {
  const void *gout, *gsum, *s, *weight;
  const float *rstd;
  void *gx, *gw;
  float *partial;  // (splits, C)
  int64_t outer, inner, s_stride;
  int C, splits;
  float inv_c;
  bool weight_f32;
  int lanes;  // of a row that has a part of a warp
};

// Which kernel takes a call, and in how many blocks its weight gradient is summed.
enum NormPath { kLongRows, kWarpRows, kBlockRows, kPlanes, kDeepPlanes };
inline NormPath norm_path(int64_t C, int64_t inner) {
  return inner > 1 ? (C <= 512 ? kPlanes : kDeepPlanes) : C <= 1024 ? kWarpRows : C <= 16384 ? kBlockRows : kLongRows;
}
// Rows in registers: elements a thread holds (32 a lane are the 1024 of a warp, blocks have up to 512 threads), and the threads
// of a block that has a row.
inline int norm_row_elements(int64_t C) {
  const int64_t per = C <= 1024 ? (C + 31) / 32 : (C + 511) / 512;
  return per <= 8 ? 8 : per <= 16 ? 16 : 32;
}
// Lanes of a warp that share a row, with up to eight elements each where the row has no more than 256.
inline int norm_row_lanes(int64_t C) {
  int n = 1;
  while (n < 32 && (int64_t)8 * n < C) n *= 2;
  return n;
}
inline int norm_row_threads(int64_t C) { return 32 * cdiv(C, 32 * norm_row_elements(C)); }
// Shared memory that a block may have for the rows ahead.
constexpr int kMostRowStages = 216 * 1024;
inline int norm_splits(int64_t outer, int64_t C, int64_t inner) {
  const int64_t norms = outer * inner;
  int64_t want, most;
  switch (norm_path(C, inner)) {
    // as many blocks as may be on the SMs at once; the launches take as many as are
    case kWarpRows: want = 148 * 4, most = (norms + 7) / 8; break;
    case kBlockRows: want = 148 * std::max(1, (norm_row_elements(C) <= 16 ? 1024 : 512) / norm_row_threads(C)), most = norms; break;
    case kPlanes: want = 148 * 3, most = (norms + 31) / 32; break;
    default: {
      const int64_t blocks = inner == 1 ? (C + 31) / 32 : C;  // enough blocks for the GPU, at least 64 norms each
      want = (148 * 8 + blocks - 1) / blocks, most = (norms + 63) / 64;
    }
  }
  const int64_t n = want < most ? want : most;
  return (int)(n < 1 ? 1 : n);
}

// norm_planes.cu: a plane's channels through shared memory, dtype one of SPH_F32, SPH_BF16, SPH_F16.
void norm_planes_forward(const NormArgs &a, int dtype, cudaStream_t st);
// (backward: may take fewer splits)
void norm_planes_backward(NormGradArgs &a, int dtype, cudaStream_t st);

// norm_flat.cu: rows of dense tensors that do not start on 16-byte boundaries; false where the tensors do not lie alike.
bool norm_flat_forward(const NormArgs &a, int dtype, cudaStream_t st);
bool norm_flat_backward(NormGradArgs &a, int dtype, cudaStream_t st);

}  // namespace sph

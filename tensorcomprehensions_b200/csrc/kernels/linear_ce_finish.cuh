// The last kernel of the cross entropy's gradient.
#pragma once

#include "linear_ce.cuh"
#include "pair_gemm.cuh"

namespace tcb200 {
namespace lce {

// dX: the splits' sums added in order, scaled, rounded once and put back in the rows' places; zero where a row has no target.
// Where a wait gave up no number is better than a wrong one: all of dX and dW (dw_elems values) become NaN.
template <typename T>
__global__ void __launch_bounds__(256) finish_kernel(Rows r, const float* sums, int64_t ld,
                                                     int64_t n, int64_t d, float scale, T* dx, T* dw,
                                                     int64_t dw_elems, int* dev_status) {
  pdl_sync();
  if (dev_status && r.head->status && blockIdx.x == 0 && threadIdx.x == 0) atomicCAS(dev_status, 0, r.head->status);
  const float nan = __int_as_float(0x7fffffff);
  const bool bad = r.head->status != 0;
  if (bad && dw)
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < dw_elems; i += (int64_t)gridDim.x * blockDim.x) dw[i] = from_float<T>(nan);
  if (!dx) return;
  const float gscale = r.head->gscale;
  const int splits = r.head->splits;
  const int64_t plane = ((int64_t)r.head->live + pg::kTile - 1) / pg::kTile * pg::kTile * ld;
  const int64_t per_row = ld / 8;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n * per_row; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / per_row, c = (i % per_row) * 8;
    const int at = r.place[row];
    const float k = (at >= 0 && r.factor_x ? r.factor_x[at] : gscale) * scale;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (at >= 0) {
#pragma unroll 4
      for (int s = 0; s < splits; ++s) {
        const float4* p = reinterpret_cast<const float4*>(sums + s * plane + at * ld + c);
        const float4 a = p[0], b = p[1];
        v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
        v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
      }
    }
    T* dst = dx + row * d + c;
    alignas(16) T w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = from_float<T>(bad ? nan : (at >= 0 ? v[j] * k : 0.f));
    if (c + 8 <= d && ((uintptr_t)dst & 15) == 0) {
#pragma unroll
      for (int q = 0; q < (int)sizeof(T) / 2; ++q) reinterpret_cast<uint4*>(dst)[q] = reinterpret_cast<uint4*>(w)[q];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < d) dst[j] = w[j];
    }
  }
}

}  // namespace lce
}  // namespace tcb200

// What the kernels of the linear layer's cross entropy share.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"

namespace tcb200 {
namespace lce {

// What the kernels share besides the operands, at the head of the workspace.
struct Head {
  int live;      // rows with a target
  int status;    // a bounded wait that gave up
  float gscale;  // largest |g| of the live rows
  int splits;    // partial sums of dX
  int spread;    // live rows where some row of dX has a scale of its own, else 0 (float16)
};

struct Rows {
  Head* head;
  int* place;     // [n] row -> live row, -1 without a target
  int* target;    // [n_pad] of a live row; -1: outside [0, V)
  float* share;   // [n_pad] g of a live row / gscale (backward)
  float* share_x; // [n_pad] null, or g / factor_x: what dZ is formed with for dX (float16)
  float* factor_x;// [n_pad] null, or gscale, or the power of two that is a row's own scale
  float* lse;     // [n_pad] of a live row (backward)
};

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float(float v) { return v; }
template <> __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

template <> __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float(float v) { return v; }
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }

constexpr float kLog2e = 1.4426950408889634f;

// exp(x), x <= 0: the base-2 exponential of the hardware (results below the smallest normal number become 0); the product
// rounds x log2(e) to 2^-24 of itself
__device__ __forceinline__ float exp_neg(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * kLog2e));
  return y;
}
// two exp(x - shift): the packed fp32 instructions do the same arithmetic in half the issue slots
__device__ __forceinline__ float2 exp_neg2(float2 x, float2 neg_shift) {
  const float2 d = __fmul2_rn(__fadd2_rn(x, neg_shift), make_float2(kLog2e, kLog2e));
  float2 y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y.x) : "f"(d.x));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y.y) : "f"(d.y));
  return y;
}

// Running maximum and sum of exp(z - maximum).  An empty pair is (-inf, 0).
struct Running {
  float top = -INFINITY, sum = 0.f;
  __device__ __forceinline__ void join(float2 x) {
    // fmaxf drops a NaN maximum; its sum is NaN then too and survives
    const float m = fmaxf(top, x.x), shift = m == -INFINITY ? 0.f : m;
    sum = sum * exp_neg(top - shift) + x.y * exp_neg(x.x - shift);
    top = m;
  }
};
// Few rows (linear_ce_few.cu): whether its kernels take a problem, the pairs of a row (or the planes of dX) that they leave, and the
// launches.  `place` and `target` of the rows, the head and the pairs are written as the other path's kernels write them.
constexpr int kFewRows = 16;
bool few_forward_ok(const tcb200_linear_ce_t& p);
bool few_backward_ok(const tcb200_linear_ce_t& p);
int64_t few_blocks(const tcb200_linear_ce_t& p, int sms, bool backward);
int few_forward(const tcb200_linear_ce_t& p, const void* X, const void* W, const void* target, const Rows& r, float2* part,
                float* hit, int64_t n_pad, int device, int sms, cudaStream_t s);
int few_backward(const tcb200_linear_ce_t& p, const void* X, const void* W, const void* target, const float* lse,
                 const float* g, int64_t g_stride, const Rows& r, float* sums, int64_t plane, int64_t ld, void* dX, void* dW,
                 int device, int sms, cudaStream_t s);

}  // namespace lce
}  // namespace tcb200

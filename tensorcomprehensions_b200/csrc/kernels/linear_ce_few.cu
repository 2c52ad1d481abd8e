// Cross entropy of a linear layer for few rows (one token to eight): bound by the pass over W.
//
// A tensor-core tile would be almost empty, so the products run on the fp32 units, in one pass: a warp takes four entries of
// the vocabulary at a time, its lanes go along D with wide loads, and the rows of X sit in shared memory as fp32, read once
// for the four entries.  Forward leaves a pair (maximum, sum) per row and block.  Backward needs no second pass over W in
// memory: a block takes 32 entries, gets their logits as the forward does, turns them into dZ in shared memory, and goes over
// the same 32 entries (now in the L2) once more with a thread per column group for dW = dZ^T X and its share of
// dX = dZ W.  dX is summed per block in shared memory and over the blocks by a second kernel, in fixed order.
// dZ stays fp32, and no operand is packed, whatever W's type and alignment.
#include "linear_ce.cuh"

namespace tcb200 {
namespace lce {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kPerWarp = 4;                    // vocabulary entries a warp takes at a time
constexpr int kPerBlock = kWarps * kPerWarp;
constexpr int kForwardSmem = 100 << 10;        // two blocks an SM
constexpr int kBackwardSmem = 200 << 10;       // X and dX

struct Few {
  const void* target;
  int index_bytes;
  int64_t ignore, n, d, v, ldx, ldw;
  __device__ int64_t index(int i) const {
    return index_bytes == 8 ? static_cast<const int64_t*>(target)[i] : (int64_t)static_cast<const int32_t*>(target)[i];
  }
};

// Elements a lane takes at a time: 16 bytes where all rows start on 16-byte boundaries, else one.
template <typename T, bool VEC> struct Step { static constexpr int n = VEC ? 16 / (int)sizeof(T) : 1; };

// Where column c of a row of X stands in shared memory: lanes read 128 bits each, free of conflicts.
template <int W>
__host__ __device__ __forceinline__ int slot(int c) {
  return W == 8 ? (c / 256) * 256 + ((c % 8) / 4) * 128 + ((c % 256) / 8) * 4 + c % 4 : c;
}
__host__ __device__ inline int64_t padded(int64_t d) { return (d + 255) / 256 * 256; }

template <int W, typename T>
__device__ __forceinline__ void load_w(const T* p, int64_t left, float* w) {
  if (W == 1) {
    w[0] = left > 0 ? to_float(p[0]) : 0.f;
  } else if (left >= W) {
    alignas(16) T v[W];
    *reinterpret_cast<uint4*>(v) = __ldg(reinterpret_cast<const uint4*>(p));
#pragma unroll
    for (int j = 0; j < W; ++j) w[j] = to_float(v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) w[j] = j < left ? to_float(p[j]) : 0.f;
  }
}
template <int W>
__device__ __forceinline__ void load_x(const float* row, int c, float* x) {
  if (W == 1) {
    x[0] = row[c];
  } else {
#pragma unroll
    for (int j = 0; j < W; j += 4) {
      const float4 q = *reinterpret_cast<const float4*>(row + slot<W>(c + j));
      x[j] = q.x; x[j + 1] = q.y; x[j + 2] = q.z; x[j + 3] = q.w;
    }
  }
}

// The rows of X as fp32; rows without a target, and what lies behind column d, are zero.
template <int NR, int W, typename T>
__device__ __forceinline__ void stage_x(const Few& f, const T* x, float* sx) {
  const int dp = (int)padded(f.d);
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const bool live = r < f.n && f.index(r) != f.ignore;
#pragma unroll 4
    for (int c = threadIdx.x; c < dp; c += kThreads)
      sx[r * dp + slot<W>(c)] = live && c < f.d ? to_float(x[r * f.ldx + c]) : 0.f;
  }
}

// The logits of entries v0 .. v0 + 3 for all rows.  Lane l gets value l / (32 / (4 NR)) of the list [row][entry].
template <int NR, int W, typename T>
__device__ __forceinline__ float logits_of(const Few& f, const T* w, int64_t v0, const float* sx) {
  const int lane = threadIdx.x & 31, dp = (int)padded(f.d);
  float acc[NR * kPerWarp];
#pragma unroll
  for (int i = 0; i < NR * kPerWarp; ++i) acc[i] = 0.f;
  const T* row[kPerWarp];
#pragma unroll
  for (int e = 0; e < kPerWarp; ++e) row[e] = w + min(v0 + e, f.v - 1) * f.ldw;
#pragma unroll 2
  for (int c = lane * W; c < (int)f.d; c += 32 * W) {
    float wv[kPerWarp][W];
#pragma unroll
    for (int e = 0; e < kPerWarp; ++e) load_w<W>(row[e] + c, f.d - c, wv[e]);
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      float xv[W];
      load_x<W>(sx + r * dp, c, xv);
#pragma unroll
      for (int e = 0; e < kPerWarp; ++e)
#pragma unroll
        for (int j = 0; j < W; ++j) acc[r * kPerWarp + e] = fmaf(xv[j], wv[e][j], acc[r * kPerWarp + e]);
    }
  }
  // halves of the list change sides until a lane holds one value, then the rest of the lanes are added
  int n = NR * kPerWarp;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    if (n > 1) {
      n /= 2;
      const bool up = lane & o;
#pragma unroll
      for (int i = 0; i < NR * kPerWarp / 2; ++i)
        if (i < n) {
          const float keep = up ? acc[i + n] : acc[i], send = up ? acc[i] : acc[i + n];
          acc[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
    } else {
      acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], o);
    }
  }
  return acc[0];
}

template <int NR, bool VEC, typename T>
__global__ void __launch_bounds__(kThreads) few_forward_kernel(Few f, const T* x, const T* w, Rows rows, float2* part,
                                                               float* hit, int64_t n_pad) {
  constexpr int W = Step<T, VEC>::n, SHARE = 32 / (NR * kPerWarp);
  extern __shared__ float sx[];
  __shared__ float2 pairs[kWarps][32];
  pdl_sync();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  stage_x<NR, W>(f, x, sx);
  if (blockIdx.x == 0 && threadIdx.x < f.n) {
    const int64_t t = f.index(threadIdx.x);
    rows.place[threadIdx.x] = t != f.ignore ? (int)threadIdx.x : -1;
    rows.target[threadIdx.x] = t >= 0 && t < f.v ? (int)t : -1;
    if (threadIdx.x == 0) *rows.head = Head{(int)f.n, 0, 1.f};
  }
  const int value = lane / SHARE, r = value / kPerWarp, e = value % kPerWarp;
  const int64_t t = r < f.n ? f.index(r) : -1;
  __syncthreads();
  Running run;
  for (int64_t v0 = ((int64_t)blockIdx.x * kWarps + warp) * kPerWarp; v0 < f.v; v0 += (int64_t)gridDim.x * kPerBlock) {
    const float z = logits_of<NR, W>(f, w, v0, sx);
    if (lane % SHARE == 0 && r < f.n && v0 + e < f.v) {
      run.join(make_float2(z, 1.f));
      if (v0 + e == t) hit[r] = z;
    }
  }
  pairs[warp][lane] = make_float2(run.top, run.sum);
  __syncthreads();
  if (threadIdx.x < f.n) {
    Running all;
    for (int k = 0; k < kWarps; ++k)
      for (int i = 0; i < kPerWarp; ++i) all.join(pairs[k][(threadIdx.x * kPerWarp + i) * SHARE]);
    part[blockIdx.x * n_pad + threadIdx.x] = make_float2(all.top, all.sum);
  }
}

template <int NR, bool VEC, typename T>
__global__ void __launch_bounds__(kThreads) few_backward_kernel(Few f, const T* x, const T* w, const float* lse,
                                                                const float* g, int64_t g_stride, Rows rows, float* sums,
                                                                int64_t plane, int64_t ld, T* dw, int need_x) {
  constexpr int W = Step<T, VEC>::n, SHARE = 32 / (NR * kPerWarp);
  extern __shared__ float sx[];
  __shared__ float dz[kPerBlock][NR];
  pdl_sync();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, dp = (int)padded(f.d);
  float* sdx = sx + NR * dp;
  stage_x<NR, W>(f, x, sx);
  for (int i = threadIdx.x; i < NR * dp; i += kThreads) sdx[i] = 0.f;
  if (blockIdx.x == 0 && threadIdx.x < f.n) {
    rows.place[threadIdx.x] = f.index(threadIdx.x) != f.ignore ? (int)threadIdx.x : -1;
    if (threadIdx.x == 0) *rows.head = Head{(int)f.n, 0, 1.f};
  }
  const int value = lane / SHARE, r = value / kPerWarp, e = value % kPerWarp;
  const int64_t t = r < f.n ? f.index(r) : f.ignore;
  const bool live = r < f.n && t != f.ignore;
  const float l = live ? lse[r] : 0.f;
  const float up = !live ? 0.f : t >= 0 && t < f.v ? g[r * g_stride] : __int_as_float(0x7fffffff);
  __syncthreads();
  for (int64_t b0 = (int64_t)blockIdx.x * kPerBlock; b0 < f.v; b0 += (int64_t)gridDim.x * kPerBlock) {
    const int64_t v0 = b0 + warp * kPerWarp;
    const float z = logits_of<NR, W>(f, w, v0, sx);
    if (lane % SHARE == 0) {
      const float p = expf(z - l);
      dz[warp * kPerWarp + e][r] = live && v0 + e < f.v ? up * (v0 + e == t ? p - 1.f : p) : 0.f;
    }
    __syncthreads();
    const int have = (int)min((int64_t)kPerBlock, f.v - b0);
    for (int c = threadIdx.x * W; c < (int)f.d; c += kThreads * W) {
      float xv[NR][W], a[NR][W];
#pragma unroll
      for (int i = 0; i < NR; ++i) {
        load_x<W>(sx + i * dp, c, xv[i]);
#pragma unroll
        for (int j = 0; j < W; ++j) a[i][j] = 0.f;
      }
#pragma unroll 4
      for (int k = 0; k < have; ++k) {
        float wv[W], out[W];
        load_w<W>(w + (b0 + k) * f.ldw + c, f.d - c, wv);
#pragma unroll
        for (int j = 0; j < W; ++j) out[j] = 0.f;
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          const float s = dz[k][i];
#pragma unroll
          for (int j = 0; j < W; ++j) {
            out[j] = fmaf(s, xv[i][j], out[j]);
            a[i][j] = fmaf(s, wv[j], a[i][j]);
          }
        }
        if (dw) {
          T* dst = dw + (b0 + k) * f.d + c;
          if (W == 1) {
            dst[0] = from_float<T>(out[0]);
          } else {  // the rows' length is a multiple of W here
            alignas(16) T q[W];
#pragma unroll
            for (int j = 0; j < W; ++j) q[j] = from_float<T>(out[j]);
            *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<uint4*>(q);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) sdx[i * dp + slot<W>(c + j)] += a[i][j];  // this thread's columns
    }
    __syncthreads();  // dz is written again
  }
  if (need_x)
    for (int i = threadIdx.x; i < (int)f.n * (int)ld; i += kThreads) {
      const int row = i / (int)ld, c = i % (int)ld;
      sums[blockIdx.x * plane + row * ld + c] = sdx[row * dp + slot<W>(c)];
    }
}

// dX: the blocks' sums, 32 columns x 32 lanes of blocks at a time, joined in a fixed order.
template <typename T>
__global__ void __launch_bounds__(1024) few_finish_kernel(Rows rows, const float* sums, int planes, int64_t plane, int64_t ld,
                                                          int64_t d, T* dx) {
  __shared__ float share[32][33];
  pdl_sync();
  const int64_t row = blockIdx.y, c = blockIdx.x * 32ll + threadIdx.x;
  float v = 0.f;
  if (c < ld)
#pragma unroll 4
    for (int s = threadIdx.y; s < planes; s += 32) v += sums[s * plane + row * ld + c];
  share[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  v = share[threadIdx.x][threadIdx.y];
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int64_t out = blockIdx.x * 32ll + threadIdx.y;
  if (threadIdx.x == 0 && out < d) dx[row * d + out] = from_float<T>(rows.place[row] < 0 ? 0.f : v);
}

int padded_rows(int64_t n) { return n <= 1 ? 1 : n <= 2 ? 2 : n <= 4 ? 4 : 8; }
int64_t forward_smem(const tcb200_linear_ce_t& p) { return padded_rows(p.N) * padded(p.D) * 4; }

Few few_of(const tcb200_linear_ce_t& p, const void* target) {
  return {target, p.index_bytes, p.ignore_index, p.N, p.D, p.V, p.ldx, p.ldw};
}

template <int NR, bool VEC, typename T>
int forward_launch(const tcb200_linear_ce_t& p, const void* X, const void* W, const void* target, const Rows& r, float2* part,
                   float* hit, int64_t n_pad, int device, int sms, cudaStream_t s) {
  static std::atomic<uint64_t> configured{0};
  TCB200_CUDA_TRY(ensure_dynamic_smem(few_forward_kernel<NR, VEC, T>, kForwardSmem, device, configured));
  TCB200_CUDA_TRY(launch_pdl(few_forward_kernel<NR, VEC, T>, dim3((unsigned)few_blocks(p, sms)), dim3(kThreads),
                             (size_t)forward_smem(p), s, few_of(p, target), static_cast<const T*>(X), static_cast<const T*>(W), r,
                             part, hit, n_pad));
  return TCB200_OK;
}
template <int NR, bool VEC, typename T>
int backward_launch(const tcb200_linear_ce_t& p, const void* X, const void* W, const void* target, const float* lse,
                    const float* g, int64_t g_stride, const Rows& r, float* sums, int64_t plane, int64_t ld, void* dX,
                    void* dW, int device, int sms, cudaStream_t s) {
  static std::atomic<uint64_t> configured{0};
  TCB200_CUDA_TRY(ensure_dynamic_smem(few_backward_kernel<NR, VEC, T>, kBackwardSmem, device, configured));
  TCB200_CUDA_TRY(launch_pdl(few_backward_kernel<NR, VEC, T>, dim3((unsigned)few_blocks(p, sms)), dim3(kThreads),
                             (size_t)(2 * forward_smem(p)), s, few_of(p, target), static_cast<const T*>(X),
                             static_cast<const T*>(W), lse, g, g_stride, r, sums, plane, ld, static_cast<T*>(dW), (int)(dX != nullptr)));
  if (dX)
    TCB200_CUDA_TRY(launch_pdl(few_finish_kernel<T>, dim3((unsigned)ceil_div(p.D, 32), (unsigned)p.N), dim3(32, 32), 0, s, r,
                               static_cast<const float*>(sums), (int)few_blocks(p, sms), plane, ld, p.D, static_cast<T*>(dX)));
  return TCB200_OK;
}

bool aligned_rows(const void* base, int64_t ld, size_t bytes) { return ((uintptr_t)base & 15) == 0 && ld * bytes % 16 == 0; }

#define TCB200_FEW_CASE(NR, CALL)                                      \
  case NR:                                                              \
    if (p.dtype == TCB200_F32) return vec ? CALL<NR, true, float> ARGS : CALL<NR, false, float> ARGS;       \
    if (p.dtype == TCB200_F16) return vec ? CALL<NR, true, __half> ARGS : CALL<NR, false, __half> ARGS;     \
    return vec ? CALL<NR, true, __nv_bfloat16> ARGS : CALL<NR, false, __nv_bfloat16> ARGS;

}  // namespace

bool few_forward_ok(const tcb200_linear_ce_t& p) { return p.N <= kFewRows && forward_smem(p) <= kForwardSmem; }
bool few_backward_ok(const tcb200_linear_ce_t& p) { return p.N <= kFewRows && 2 * forward_smem(p) <= kBackwardSmem; }
int64_t few_blocks(const tcb200_linear_ce_t& p, int sms) { return std::min<int64_t>(ceil_div(p.V, kPerBlock), 2ll * sms); }

int few_forward(const tcb200_linear_ce_t& p, const void* X, const void* W, const void* target, const Rows& r, float2* part,
                float* hit, int64_t n_pad, int device, int sms, cudaStream_t s) {
  const bool vec = aligned_rows(W, p.ldw, p.dtype == TCB200_F32 ? 4 : 2);
#define ARGS (p, X, W, target, r, part, hit, n_pad, device, sms, s)
  switch (padded_rows(p.N)) {
    TCB200_FEW_CASE(1, forward_launch)
    TCB200_FEW_CASE(2, forward_launch)
    TCB200_FEW_CASE(4, forward_launch)
    TCB200_FEW_CASE(8, forward_launch)
  }
#undef ARGS
  return TCB200_ERR_UNSUPPORTED;
}

int few_backward(const tcb200_linear_ce_t& p, const void* X, const void* W, const void* target, const float* lse,
                 const float* g, int64_t g_stride, const Rows& r, float* sums, int64_t plane, int64_t ld, void* dX, void* dW,
                 int device, int sms, cudaStream_t s) {
  const size_t bytes = p.dtype == TCB200_F32 ? 4 : 2;
  // whole vectors along D in W and in dW
  const bool vec = aligned_rows(W, p.ldw, bytes) && aligned_rows(dW, p.D, bytes);
#define ARGS (p, X, W, target, lse, g, g_stride, r, sums, plane, ld, dX, dW, device, sms, s)
  switch (padded_rows(p.N)) {
    TCB200_FEW_CASE(1, backward_launch)
    TCB200_FEW_CASE(2, backward_launch)
    TCB200_FEW_CASE(4, backward_launch)
    TCB200_FEW_CASE(8, backward_launch)
  }
#undef ARGS
  return TCB200_ERR_UNSUPPORTED;
}

}  // namespace lce
}  // namespace tcb200

// Softmax cross entropy of a linear layer over a large vocabulary, without keeping its logits.
//
//   z = X W^T,  lse_n = log sum_v exp z_nv,  loss_n = lse_n - z_{n, t_n}
//   dZ_nv = g_n (exp(z_nv - lse_n) - [v = t_n]),  dX = dZ W,  dW = dZ^T X
//
// Forward: one pass of the pair product (pair_gemm.cuh) over the vocabulary.  A thread of its epilogue owns 128 logits of
// a row and leaves their maximum and the sum of exp(z - maximum); a second kernel joins these per row.  The logits never reach
// memory.  Backward, per piece of the vocabulary: the product again, with an epilogue that writes dZ of the piece; then
// dX += dZ W and dW = dZ^T X from it.  The work is 2 N D V operations forward and 6 N D V backward on the tensor cores,
// which bound it from a few hundred rows up; below that one pass over W does.
//
// Rows are compacted first: rows without a target (target == ignore_index) cost nothing, and what their X holds, infinities
// and NaN included, is never read.  The number of rows that remain stays on the device (pg::Args::live).
#include <string.h>

#include <mutex>

#include "linear_ce.cuh"
#include "linear_ce_finish.cuh"
#include "pair_gemm.cuh"

namespace tcb200 {
namespace pg {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiledFn encode_fn() {
  static std::mutex mu;
  static EncodeTiledFn fn = nullptr;
  std::lock_guard<std::mutex> lock(mu);
  if (!fn) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
    else
      (void)cudaGetLastError();
  }
  return fn;
}

// k-major: box of 64 columns (k) x `rows`.  mn-major: box of 64 columns (m or n) x 64 rows (k).  Zeros out of bounds.
int make_map(CUtensorMap* tm, const Operand& o, bool bf16, bool mn_major, int rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return TCB200_ERR_CUDA;
  cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)o.planes};
  const int64_t plane = o.planes > 1 ? o.plane_stride : o.rows * o.ld;
  cuuint64_t strides[2] = {(cuuint64_t)o.ld * 2, (cuuint64_t)plane * 2};
  cuuint32_t box[3] = {kBK, (cuuint32_t)(mn_major ? kBK : rows), 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(tm, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                  const_cast<void*>(o.base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? TCB200_OK : TCB200_ERR_CUDA;
}

int make_out_map(CUtensorMap* tm, const Operand& o, int bytes) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return TCB200_ERR_CUDA;
  cuuint64_t dims[3] = {(cuuint64_t)o.cols, (cuuint64_t)o.rows, (cuuint64_t)o.planes};
  const int64_t plane = o.planes > 1 ? o.plane_stride : o.rows * o.ld;
  cuuint64_t strides[2] = {(cuuint64_t)(o.ld * bytes), (cuuint64_t)(plane * bytes)};
  cuuint32_t box[3] = {(cuuint32_t)(128 / bytes), 32, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  // 16-bit words move as they are
  CUresult r = fn(tm, bytes == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                  const_cast<void*>(o.base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? TCB200_OK : TCB200_ERR_CUDA;
}

int make_plain_map(CUtensorMap* tm, const void* base, int dtype, int64_t cols, int64_t rows, int64_t ld, int box_cols, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return TCB200_ERR_CUDA;
  const int64_t bytes = dtype == TCB200_F32 ? 4 : 2;
  cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, 1};
  cuuint64_t strides[2] = {(cuuint64_t)(ld * bytes), (cuuint64_t)(rows * ld * bytes)};
  cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(tm, bytes == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims,
                  strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? TCB200_OK : TCB200_ERR_CUDA;
}

}  // namespace pg

using namespace lce;

namespace {

using pg::kTile;

// ---- operands -------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint16_t bits(__nv_bfloat16 v) { return __bfloat16_as_ushort(v); }
__device__ __forceinline__ uint16_t bits(__half v) { return __half_as_ushort(v); }

// float32 operands.  The logits take two f16 planes of the row scaled by a power of two, v 2^e = h0 + 2^-11 h1: the row's largest
// value lies in [2^14, 2^15), values down to 2^-29 of it keep 22 significand bits and smaller ones 2^-50 of it (with h1 unscaled:
// 2^-17 and 2^-40, and a row with a value 2^24 times the others had its logits off by 2^-16).  Three products, 2^-11 (h1 h0 + h0 h1)
// + h0 h0, then give z to fp32's accuracy, half of what bf16 planes need, and 2^-e is taken off in the epilogue.  The gradient's products sum over the rows that such scales belong to, so they take three bf16 planes without
// any, v = p0 + p1 + p2 with 24 significand bits, and the six products with i + j <= 2.  A value that is not finite is carried
// by the first plane alone.
constexpr float kLargest = 3.402823466e38f;
__device__ __forceinline__ void split2(float v, uint16_t* h) {
  const __half a = __float2half_rn(v);
  float r = v - __half2float(a);
  if (!(fabsf(r) <= kLargest)) r = 0.f;
  h[0] = bits(a);
  h[1] = bits(__float2half_rn(r * (float)(1 << pg::kLowShift)));
}
__device__ __forceinline__ void split3(float v, uint16_t* p) {
  const __nv_bfloat16 a = __float2bfloat16_rn(v);
  float r = v - __bfloat162float(a);
  if (!(fabsf(r) <= kLargest)) r = 0.f;
  const __nv_bfloat16 b = __float2bfloat16_rn(r);
  r -= __bfloat162float(b);
  p[0] = bits(a);
  p[1] = bits(b);
  p[2] = bits(__float2bfloat16_rn(r));
}

// Eight columns of a row; zero behind the last.
template <typename T>
__device__ __forceinline__ void load8(const T* src, int64_t left, T* v) {
  if (left >= 8 && ((uintptr_t)src & 15) == 0) {
#pragma unroll
    for (int q = 0; q < (int)sizeof(T) / 2; ++q) reinterpret_cast<uint4*>(v)[q] = __ldg(reinterpret_cast<const uint4*>(src) + q);
  } else {
    memset(v, 0, 8 * sizeof(T));
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) v[j] = src[j];
  }
}

// Where a row's planes go: `scaled` two f16 planes and the row's factor 2^-e, `plain` three bf16 planes (float32), or
// `plain` alone, the row as it is (16-bit types).  Null: not wanted.
struct Planes {
  uint16_t *plain, *scaled;
  float* factor;
  int64_t stride;  // elements from one plane to the next
};

// L lanes (a warp, or half or a quarter of one where rows are short) pack a row of float32; source null: a row of zeros;
// `write` false: nothing (the lanes take part in the shuffles all the same).  Rows of up to 16 L columns stay in registers
// between finding their largest value and writing; longer ones are read again.
template <int L>
__device__ __forceinline__ void pack_row(const float* src, bool write, int64_t d, int64_t dp, const Planes& o, int64_t row) {
  constexpr int SPAN = L * 8, HOLD = 2;
  const int lane = threadIdx.x & (L - 1);
  auto load = [&](int64_t c0, float* v) {
    if (src && c0 + lane * 8 < d) load8(src + c0 + lane * 8, d - c0 - lane * 8, v);
    else memset(v, 0, 32);
  };
  float top = 0.f;
  auto look = [&](const float* v) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float a = fabsf(v[j]);
      if (a <= kLargest) top = fmaxf(top, a);
    }
  };
  alignas(16) float held[HOLD][8];
#pragma unroll
  for (int h = 0; h < HOLD; ++h)
    if (h * SPAN < dp) load(h * SPAN, held[h]);
#pragma unroll
  for (int h = 0; h < HOLD; ++h)
    if (h * SPAN < dp) look(held[h]);
  for (int64_t c0 = HOLD * SPAN; c0 < d; c0 += SPAN) {
    alignas(16) float v[8];
    load(c0, v);
    look(v);
  }
#pragma unroll
  for (int q = L / 2; q; q >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, q));
  int e = 0;
  if (top > 0.f) {
    frexpf(top, &e);
    e = 15 - e;
  }
  e = min(e, 126);  // (the smallest e is -113; both 2^e and 2^-e are normal numbers)
  const float scale = ldexpf(1.f, e);
  if (lane == 0 && write) o.factor[row] = ldexpf(1.f, -e);
  auto emit = [&](int64_t c, const float* v) {
    if (!write || c >= dp) return;
    alignas(16) uint16_t h[2][8], p[3][8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint16_t q[3];
      split2(v[j] * scale, q);
      h[0][j] = q[0]; h[1][j] = q[1];
      split3(v[j], q);
      p[0][j] = q[0]; p[1][j] = q[1]; p[2][j] = q[2];
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) *reinterpret_cast<uint4*>(o.scaled + k * o.stride + row * dp + c) = *reinterpret_cast<uint4*>(h[k]);
    if (o.plain)
#pragma unroll
      for (int k = 0; k < 3; ++k) *reinterpret_cast<uint4*>(o.plain + k * o.stride + row * dp + c) = *reinterpret_cast<uint4*>(p[k]);
  };
#pragma unroll
  for (int h = 0; h < HOLD; ++h)
    if (h * SPAN < dp) emit(h * SPAN + lane * 8, held[h]);
  for (int64_t c0 = HOLD * SPAN; c0 < dp; c0 += SPAN) {
    alignas(16) float v[8];
    load(c0, v);
    emit(c0 + lane * 8, v);
  }
}
// Rows first, first + stride, ... below `rows` of a warp; source(r) is their address or null.
template <int L, typename Source>
__device__ __forceinline__ void pack_rows_of(int64_t first, int64_t stride, int64_t rows, int64_t d, int64_t dp, const Planes& o, int64_t row0,
                                             Source source) {
  constexpr int PER = 32 / L;
  const int mine = (threadIdx.x & 31) / L;
  for (int64_t r = first * PER; r < rows; r += stride * PER) {
    const bool there = r + mine < rows;
    pack_row<L>(there ? source(r + mine) : nullptr, there, d, dp, o, row0 + r + mine);
  }
}
template <typename Source>
__device__ __forceinline__ void pack_rows(int64_t first, int64_t stride, int64_t rows, int64_t d, int64_t dp, const Planes& o, int64_t row0,
                                          Source source) {
  if (dp <= 64) pack_rows_of<8>(first, stride, rows, d, dp, o, row0, source);
  else if (dp <= 128) pack_rows_of<16>(first, stride, rows, d, dp, o, row0, source);
  else pack_rows_of<32>(first, stride, rows, d, dp, o, row0, source);
}

// Entries of W as operand planes of [rows][dp], dp = d rounded up to 8.
__global__ void __launch_bounds__(256) pack_rows_kernel(const float* in, int64_t ld, int64_t rows, int64_t d, int64_t dp, Planes o) {
  pdl_sync();
  const int warp = threadIdx.x >> 5;
  pack_rows(blockIdx.x * 8 + warp, gridDim.x * 8, rows, d, dp, o, 0, [&](int64_t r) { return in + r * ld; });
}
__global__ void __launch_bounds__(256) pack_kernel(const __half* in, int64_t ld, int64_t rows, int64_t d, int64_t dp, Planes o) {
  pdl_sync();
  // a piece has fewer than 2^31 groups of eight (it is 256 MiB, or 4096 entries of at most 2^20 columns)
  const uint32_t per_row = (uint32_t)(dp / 8), total = (uint32_t)rows * per_row;
  for (uint32_t i = blockIdx.x * blockDim.x + threadIdx.x; i < total; i += gridDim.x * blockDim.x) {
    const int64_t r = i / per_row, c = (i % per_row) * 8;
    alignas(16) __half v[8];
    load8(in + r * ld + c, d - c, v);
    *reinterpret_cast<uint4*>(o.plain + r * dp + c) = *reinterpret_cast<uint4*>(v);
  }
}

// The rows with a target, and X of them as operand planes [planes][n_pad][dp]; rows behind the last live one, up to a whole
// tile, are zero.  Every block reads all targets (and all g, for the largest of them) and knows from them where its own
// rows go: one launch instead of two that wait for one another, and the order of the live rows, and with it every later
// sum, does not depend on timing.
// It also settles how often the sum of dX is split: by the live rows, which the host does not know.
struct Splits {
  int64_t tiles;        // rows, in tiles, that the stack of partial sums has room for
  int64_t tiles_n;      // tiles of a row of dX
  int kb, products, pairs;
};
constexpr int kRowThreads = 512;
// float16 keeps dZ / max|g| with 2^14 (GradEpi): a row's small probabilities leave its range as |g| / max|g| falls, which costs dX of
// the row 1e-3 of itself at 2^-24, 3e-2 at 2^-32 and all from 2^-39 on.  From this share down (where nothing is lost yet) a row's
// dZ has a power of two of its own for dX.  dW, a sum over rows, takes the common scale: what it loses, 2^-39 max|g|, is below
// float16's steps unless max|g| passes 2^15.
constexpr float kSmallShare = 1.f / 65536;
template <typename T, typename Index>
__global__ void __launch_bounds__(kRowThreads, 2) rows_kernel(const Index* target, int64_t n, int64_t v, int64_t ignore,
                                                           const float* g, int64_t g_stride, const float* lse, Rows r,
                                                           const T* x, int64_t ld, int64_t d, int64_t dp, Planes o, Splits sp) {
  __shared__ int before_of[kRowThreads / 32], all_of[kRowThreads / 32];
  __shared__ float top_of[kRowThreads / 32], least_of[kRowThreads / 32];
  __shared__ int list[kRowThreads];
  pdl_sync();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t per_block = (n + gridDim.x - 1) / gridDim.x;
  const int64_t r0 = min(n, blockIdx.x * per_block), r1 = min(n, r0 + per_block);
  int before = 0, all = 0;
  float top = 0.f, least = INFINITY;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < n; i += kRowThreads) {
    const bool live = (int64_t)target[i] != ignore;
    all += live;
    before += live && i < r0;
    if (g && live) {
      const float ax = fabsf(g[i * g_stride]);
      if (ax <= 3.402823466e38f) top = fmaxf(top, ax);  // the largest finite one: not NaN, not infinite
      if (ax > 0.f) least = fminf(least, ax);
    }
  }
  for (int o = 16; o; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    all += __shfl_xor_sync(0xffffffffu, all, o);
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
  }
  if (lane == 0) {
    before_of[warp] = before;
    all_of[warp] = all;
    top_of[warp] = top;
    least_of[warp] = least;
  }
  __syncthreads();
  before = all = 0;
  for (int w = 0; w < kRowThreads / 32; ++w) {
    before += before_of[w];
    all += all_of[w];
    top = fmaxf(top, top_of[w]);
    least = fminf(least, least_of[w]);
  }
  const float small = top * kSmallShare;  // rows of a smaller |g| have a scale of their own in dX
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    r.head->live = all;
    r.head->status = 0;
    r.head->gscale = top > 0.f ? top : 1.f;
    r.head->spread = r.share_x && least < small ? all : 0;
    const int64_t tiles_m = (all + (int64_t)kTile - 1) / kTile, tiles = tiles_m * sp.tiles_n;
    r.head->splits = tiles == 0 || tiles > 1 << 20
                         ? 1
                         : pg::choose_splits((int)tiles, sp.kb, sp.products, sp.pairs, (int)min(sp.tiles / tiles_m, (int64_t)pg::kMaxSplits));
  }
  const uint32_t per_row = (uint32_t)(dp / 8);
  // 512 rows at a time: their places, then their X
  for (int64_t base = r0; base < r1; base += kRowThreads) {
    const int64_t i = base + threadIdx.x;
    const int64_t t = i < r1 ? (int64_t)target[i] : ignore;
    const bool live = t != ignore;
    const unsigned votes = __ballot_sync(0xffffffffu, live);
    __syncthreads();  // the counts and the list of the round before have been read
    if (lane == 0) before_of[warp] = __popc(votes);
    __syncthreads();
    int at = __popc(votes & ((1u << lane) - 1)), count = 0;
    for (int w = 0; w < kRowThreads / 32; ++w) {
      if (w < warp) at += before_of[w];
      count += before_of[w];
    }
    if (i < r1) r.place[i] = live ? before + at : -1;
    if (live) {
      const bool inside = t >= 0 && t < v;
      list[at] = (int)(i - base);
      r.target[before + at] = inside ? (int)t : -1;
      if (g) {
        // dZ is kept with g / max|g|: where all rows share one g, as under a mean, that is exactly 1 and the rounding
        // of dZ to 16 bits does not meet g's significand
        const float x = g[i * g_stride];
        const float share = !inside ? __int_as_float(0x7fffffff) : top > 0.f ? x / top : x;
        r.share[before + at] = share;
        if (r.share_x) {
          const bool own = inside && x != 0.f && fabsf(x) < small;
          int e = 0;
          const float part = own ? frexpf(x, &e) : share;
          r.share_x[before + at] = part;
          r.factor_x[before + at] = own ? ldexpf(1.f, e) : top > 0.f ? top : 1.f;
        }
        r.lse[before + at] = lse[i];
      }
    }
    __syncthreads();
    if constexpr (sizeof(T) == 4) {
      pack_rows(warp, kRowThreads / 32, count, d, dp, o, before, [&](int64_t j) { return x + (base + list[j]) * ld; });
    } else {
      const uint32_t items = (uint32_t)count * per_row;
      constexpr int U = 4;  // loads in flight a thread
      for (uint32_t k0 = threadIdx.x; k0 < items; k0 += U * kRowThreads) {
        alignas(16) T v[U][8];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint32_t k = k0 + u * kRowThreads, j = k / per_row;
          const int64_t c = (k % per_row) * 8;
          if (k < items) load8(x + (base + list[j]) * ld + c, d - c, v[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint32_t k = k0 + u * kRowThreads, j = k / per_row;
          const int64_t c = (k % per_row) * 8;
          if (k < items) *reinterpret_cast<uint4*>(o.plain + (before + j) * dp + c) = *reinterpret_cast<uint4*>(v[u]);
        }
      }
    }
    before += count;
  }
  const int64_t end = (all + (int64_t)kTile - 1) / kTile * kTile;
  if constexpr (sizeof(T) == 4) {
    pack_rows(blockIdx.x * (kRowThreads / 32) + warp, gridDim.x * (kRowThreads / 32), end - all, d, dp, o, all,
              [](int64_t) { return (const float*)nullptr; });
  } else {
    for (int64_t k = blockIdx.x * (int64_t)kRowThreads + threadIdx.x; k < (end - all) * per_row; k += (int64_t)gridDim.x * kRowThreads)
      *reinterpret_cast<uint4*>(o.plain + all * dp + k * 8) = make_uint4(0, 0, 0, 0);
  }
}

// ---- epilogues ------------------------------------------------------------------------------------------------------
// float32 operands are scaled by row (pack_row): the logits of a thread's row and columns, unscaled.
template <int C>
__device__ __forceinline__ void unscale(float (&acc)[C], const float* row_factor, const float* col_factor, int row, int col0) {
  const float f = row_factor[row];
#pragma unroll
  for (int j = 0; j < C; j += 4) {
    const float4 q = *reinterpret_cast<const float4*>(col_factor + col0 + j);
    acc[j] *= f * q.x; acc[j + 1] *= f * q.y; acc[j + 2] *= f * q.z; acc[j + 3] *= f * q.w;
  }
}

// Forward: maximum and sum of exp(z - maximum) over this thread's columns, and the target's logit.
template <bool F32>
struct ForwardEpi {
  static constexpr int kColumns = 128;
  static constexpr bool kDirect = false;
  static constexpr bool kShifted = F32;
  const Head* head;
  const int* target;
  float2* part;      // [parts][n_pad]
  float* hit;        // [n_pad] the target's logit
  int64_t n_pad, v0, v, part0;  // first vocabulary entry of this launch, entries of it; number of its first part
  const float *row_factor, *col_factor;
  template <int C>
  __device__ void operator()(float (&acc)[C], int row, int col0, int, const CUtensorMap*, const pg::Out&) const {
    const bool live = row < head->live;
    if (col0 >= v || !__any_sync(0xffffffffu, live)) return;
    if (F32 && live) unscale(acc, row_factor, col_factor, row, col0);
    const int have = (int)min(v - col0, (int64_t)C);
    const int64_t at = live ? (int64_t)target[row] - v0 - col0 : -1;
    const int t = at >= 0 && at < have ? (int)at : -1;
    if (have < C) {  // the same for all lanes
#pragma unroll
      for (int j = 0; j < C; ++j)
        if (j >= have) acc[j] = -INFINITY;
    }
    if (__any_sync(0xffffffffu, t >= 0)) {  // rare: a warp's rows have their target in 32 x C of the logits
      float z = 0.f;
#pragma unroll
      for (int j = 0; j < C; ++j)
        if (j == t) z = acc[j];
      if (t >= 0) hit[row] = z;
    }
    float top = acc[0];
#pragma unroll
    for (int j = 1; j < C; ++j) top = fmaxf(top, acc[j]);
    // all -inf: the sum is empty, and -inf - -inf would make NaN of it; all NaN: the sum says so
    const float shift = top == -INFINITY || top != top ? 0.f : top;
    const float2 neg = make_float2(-shift, -shift);
    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
    for (int j = 0; j < C; j += 2) sum[(j >> 1) & 1] = __fadd2_rn(sum[(j >> 1) & 1], exp_neg2(make_float2(acc[j], acc[j + 1]), neg));
    if (live) part[(part0 + col0 / C) * n_pad + row] = make_float2(top != top ? -INFINITY : top, (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y));
  }
};

// Joins the parts of a row: lse, and the loss lse - z_target.  32 rows x 32 lanes of parts a block, four loads in flight a
// thread; a row's parts are joined in a fixed order.
__global__ void __launch_bounds__(1024) join_kernel(Rows r, const float2* part, const float* hit, int64_t parts,
                                                    int64_t n_pad, int64_t n, float* loss, float* lse, int* dev_status) {
  __shared__ float2 share[32][33];
  pdl_sync();
  if (dev_status && r.head->status && blockIdx.x == 0 && threadIdx.x + threadIdx.y == 0)
    atomicCAS(dev_status, 0, r.head->status);
  const int64_t i = blockIdx.x * 32 + threadIdx.x;
  const int64_t at = i < n ? r.place[i] : -1;
  const float2 none = make_float2(-INFINITY, 0.f);
  Running run;
  if (at >= 0) {
    for (int64_t p = threadIdx.y; p < parts; p += 128) {
      float2 x[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = p + 32 * k < parts ? part[(p + 32 * k) * n_pad + at] : none;
#pragma unroll
      for (int k = 0; k < 4; ++k) run.join(x[k]);
    }
  }
  share[threadIdx.y][threadIdx.x] = make_float2(run.top, run.sum);
  __syncthreads();
  // row threadIdx.y of the block, its 32 lanes joined by a warp
  const float2 mine = share[threadIdx.x][threadIdx.y];
  run.top = mine.x;
  run.sum = mine.y;
  for (int o = 16; o; o >>= 1)
    run.join(make_float2(__shfl_xor_sync(0xffffffffu, run.top, o), __shfl_xor_sync(0xffffffffu, run.sum, o)));
  const int64_t row = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x != 0 || row >= n) return;
  const int place = r.place[row];
  const float nan = __int_as_float(0x7fffffff);
  float l = run.top + logf(run.sum), e = 0.f;
  if (place < 0) l = 0.f;
  else if (r.target[place] < 0) e = nan;  // a target outside the vocabulary
  else e = (run.top - hit[place]) + logf(run.sum);
  if (r.head->status) l = e = nan;        // a wait gave up: no number is better than a wrong one
  loss[row] = e;
  lse[row] = l;
}

// dZ of a piece, as operand planes [planes][n_pad][ld].  f16 values carry 2^14: probabilities from 2^-28 up then keep all
// of their 11 bits (1 / 2^-14 is f16's smallest normal number), and |dZ| <= 2^14 stays in range.
constexpr float kHalfScale = 16384.f;
enum { kF32 = 0, kF16 = 1, kBF16 = 2 };

template <int TYPE>
struct GradEpi {
  // three planes of a float32 value are five times the work of one rounding: sixteen warps of 64 columns
  // (1024 x 1024 x 16384: 120 -> 102 us), where 16-bit types lose by them (4096 x 2048 x 32000: 348 -> 361 us)
  static constexpr int kColumns = TYPE == kF32 ? 64 : 128;
  static constexpr bool kDirect = TYPE != kF32;  // (float32 dZ above: 164k cycles without, 173k with)
  static constexpr bool kShifted = TYPE == kF32;
  const Head* head;
  const int* target;
  const float* share;
  const float* lse;
  int64_t ld, v0, v;
  const float *row_factor, *col_factor;
  template <int C>
  __device__ void operator()(float (&acc)[C], int row, int col0, int, const CUtensorMap* tm, const pg::Out& out) const {
    if (col0 >= ld) return;
    const bool live = row < head->live;
    if (TYPE == kF32 && live) unscale(acc, row_factor, col_factor, row, col0);
    const float g = live ? share[row] : 0.f, l = live ? lse[row] : 0.f;
    const int64_t at = live ? (int64_t)target[row] - v0 - col0 : -1;
    const int t = at >= 0 && at < C ? (int)at : -1;
    const float2 neg = make_float2(-l, -l), g2 = make_float2(g, g);
#pragma unroll
    for (int c = 0; c < C; c += 2) {
      float2 p;
      if (TYPE == kF32) p = make_float2(expf(acc[c] - l), expf(acc[c + 1] - l));
      else p = exp_neg2(make_float2(acc[c], acc[c + 1]), neg);
      acc[c] = p.x;
      acc[c + 1] = p.y;
    }
    if (__any_sync(0xffffffffu, t >= 0)) {  // rare, as in the forward pass
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (c == t) acc[c] -= 1.f;
    }
#pragma unroll
    for (int c = 0; c < C; c += 2) {
      const float2 x = __fmul2_rn(make_float2(acc[c], acc[c + 1]), g2);
      acc[c] = x.x;
      acc[c + 1] = x.y;
    }
    // rows behind the last live one, and what lies behind the vocabulary, are summed over by the products that follow: zero
    const int have = live ? (int)min(v - col0, (int64_t)C) : 0;
    if (__any_sync(0xffffffffu, have < C)) {
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (c >= have) acc[c] = 0.f;
    }
#pragma unroll
    for (int p = 0; p < (TYPE == kF32 ? 3 : 1); ++p) {
#pragma unroll
      for (int h = 0; h < C; h += 64) {  // a box: 64 columns
        out.begin();
#pragma unroll
        for (int c = 0; c < 64; c += 8) {
          alignas(16) uint16_t w[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            float& x = acc[h + c + j];
            if (TYPE == kF16) {
              w[j] = bits(__float2half_rn(x * kHalfScale));
            } else {
              const __nv_bfloat16 b = __float2bfloat16_rn(x);
              w[j] = bits(b);
              // what is left for the next plane; a value that is not finite is carried by the first plane alone
              if (TYPE == kF32) x = fabsf(x) <= 3.0e38f ? x - __bfloat162float(b) : 0.f;
            }
          }
          out.put(c / 8, *reinterpret_cast<uint4*>(w));
        }
        out.send(tm, col0 + h, row - out.lane, p);
      }
    }
  }
};

// dX of a piece: fp32 sums, a stack of partial ones where the vocabulary is split, added to over the pieces.
struct SumEpi {
  static constexpr int kColumns = 128;
  static constexpr bool kDirect = false;
  static constexpr bool kShifted = false;
  const Head* head;
  int64_t ld;  // columns of the sums
  int add;
  template <int C>
  __device__ void operator()(float (&acc)[C], int row, int col0, int split, const CUtensorMap* tm, const pg::Out& out) const {
    const int at = row - out.lane + split * ((head->live + kTile - 1) / kTile * kTile);
#pragma unroll
    for (int h = 0; h < C; h += 32) {
      if (col0 + h >= ld) return;
      out.begin();
#pragma unroll
      for (int c = 0; c < 32; c += 4)
        out.put(c / 4, make_uint4(__float_as_uint(acc[h + c]), __float_as_uint(acc[h + c + 1]), __float_as_uint(acc[h + c + 2]),
                                  __float_as_uint(acc[h + c + 3])));
      if (add) out.send_add(tm, col0 + h, at, 0);
      else out.send(tm, col0 + h, at, 0);
    }
  }
};

// dW of a piece: whole sums, scaled and rounded once.
template <typename T>
struct WeightEpi {
  static constexpr int kColumns = 128;
  static constexpr bool kDirect = false;
  static constexpr bool kShifted = false;
  const Head* head;
  T* dst;
  int64_t rows, d;
  float scale;
  int tma;  // rows start on 16-byte boundaries
  template <int C>
  __device__ void operator()(float (&acc)[C], int row, int col0, int, const CUtensorMap* tm, const pg::Out& out) const {
    const int row0 = row - out.lane;
    if (row0 >= rows) return;
    const float k = head->gscale * scale;
    constexpr int W = 16 / sizeof(T), COLS = 128 / sizeof(T);
#pragma unroll
    for (int h = 0; h < C; h += COLS) {
      if (col0 + h >= d) return;
      out.begin();
#pragma unroll
      for (int c = 0; c < COLS; c += W) {
        alignas(16) T w[W];
#pragma unroll
        for (int j = 0; j < W; ++j) w[j] = from_float<T>(acc[h + c + j] * k);
        out.put(c / W, *reinterpret_cast<uint4*>(w));
      }
      if (tma) {
        out.send(tm, col0 + h, row0, 0);
      } else {  // lane by lane along a row
        __syncwarp();
        const int have = (int)min(rows - row0, (int64_t)32);
        for (int r = 0; r < have; ++r)
#pragma unroll
          for (int c = 0; c < COLS; c += 32)
            if (col0 + h + c + out.lane < d)
              dst[(row0 + r) * d + col0 + h + c + out.lane] = *static_cast<const T*>(out.at(r, c + out.lane, sizeof(T)));
        __syncwarp();
      }
    }
  }
};

// ---- host -----------------------------------------------------------------------------------------------------------
constexpr int64_t kPieceBytes = 256ll << 20;  // dZ of a piece, and a packed piece of W

struct Layout {
  int64_t n_pad, dp, planes, sum_rows;
  int64_t fwd_piece, bwd_piece;  // vocabulary entries per piece
  int64_t parts;                 // of a row's logits, one per drain warp's columns
  int fwd_bn, bwd_bn, dw_bn;     // columns of a tile: logits forward, logits backward, dW
  int splits, split_for;         // partial sums of dX that there is room for; k-blocks that their number is chosen for
  bool few_fwd, few_bwd;         // the kernels for few rows: nothing is packed, no dZ is kept
  int64_t fwd_bytes, bwd_bytes;
  // byte offsets
  int64_t place, target, share, lse, share_x, factor_x, hit, part, x, x_scaled, x_factor, w_fwd, w_fwd_factor, w_bwd, w_bwd_scaled, w_bwd_factor, dz,
      sums;
};

bool pack_w(const tcb200_linear_ce_t& p) { return p.dtype == TCB200_F32 || p.pack_w; }

int layout_of(const tcb200_linear_ce_t* q, int sms, Layout* l) {
  if (!q) return TCB200_ERR_INVALID_ARGUMENT;
  const tcb200_linear_ce_t& p = *q;
  if (p.N < 0 || p.D < 1 || p.V < 1 || p.ldx < p.D || p.ldw < p.D) return TCB200_ERR_INVALID_ARGUMENT;
  if (p.dtype != TCB200_F32 && p.dtype != TCB200_F16 && p.dtype != TCB200_BF16) return TCB200_ERR_INVALID_ARGUMENT;
  if (p.index_bytes != 4 && p.index_bytes != 8) return TCB200_ERR_INVALID_ARGUMENT;
  const int64_t limit = (1ll << 31) - 1024;
  if (p.N > limit || p.V > limit || p.D > (1ll << 20) || p.ldw > (1ll << 38) || p.ldx > (1ll << 38)) return TCB200_ERR_TOO_LARGE;
  if (!pack_w(p) && p.ldw % 8 != 0) return TCB200_ERR_ALIGNMENT;
  l->n_pad = round_up(std::max<int64_t>(p.N, 1), kTile);
  l->dp = round_up(p.D, 64);  // packed rows start on 128-byte lines
  l->planes = p.dtype == TCB200_F32 ? 3 : 1;
  const int64_t v_pad = round_up(p.V, kTile);
  // A packed piece of W, and dZ of a piece, take at most 256 MiB where that leaves 4096 entries a piece; pieces are even.
  auto piece = [&](int64_t bytes_per_entry) {
    const int64_t most = std::max<int64_t>(kPieceBytes / bytes_per_entry / kTile * kTile, 16 * kTile);
    const int64_t pieces = ceil_div(v_pad, most);
    return round_up(ceil_div(v_pad, pieces), kTile);
  };
  l->fwd_piece = pack_w(p) ? piece(l->dp * 2 * std::min<int64_t>(l->planes, 2)) : v_pad;
  l->bwd_piece = piece(2 * l->planes * (pack_w(p) ? std::max(l->dp, l->n_pad) : l->n_pad));
  const bool f32 = p.dtype == TCB200_F32;
  const int products = f32 ? 6 : 1, z_products = f32 ? 3 : 1;
  l->fwd_bn = pg::tile_columns(l->n_pad, l->fwd_piece, p.D, z_products, sms);
  l->bwd_bn = pg::tile_columns(l->n_pad, l->bwd_piece, p.D, z_products, sms);
  l->dw_bn = pg::tile_columns(l->bwd_piece, p.D, p.N, products, sms);
  l->few_fwd = few_forward_ok(p);
  l->few_bwd = few_backward_ok(p);
  l->parts = l->few_fwd ? few_blocks(p, sms, false) : ceil_div(p.V, l->fwd_bn / 2);
  // dX has few tiles and a long sum, which is split (pg::choose_splits) by the live rows; there is room for the partial sums of
  // all rows, 256 MiB of them at most.
  const int64_t tiles = (l->n_pad / kTile) * ceil_div(p.D, kTile);
  l->split_for = (int)ceil_div(l->bwd_piece, pg::kBK);
  l->splits = tiles > 1 << 20 ? 1 : pg::choose_splits((int)tiles, l->split_for, products, std::max(1, sms / 2),
                                                      (int)std::max<int64_t>(1, std::min<int64_t>(pg::kMaxSplits, kPieceBytes / (l->n_pad * l->dp * 4))));
  if (l->few_bwd) l->splits = (int)few_blocks(p, sms, true);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t here = at;
    at += round_up(std::max<int64_t>(bytes, 16), 1024);
    return here;
  };
  take(sizeof(Head));
  l->place = take(p.N * 4);
  l->target = take(l->n_pad * 4);
  l->share = take(l->n_pad * 4);
  l->lse = take(l->n_pad * 4);
  l->share_x = take(p.dtype == TCB200_F16 ? l->n_pad * 4 : 0);
  l->factor_x = take(p.dtype == TCB200_F16 ? l->n_pad * 4 : 0);
  // X: the plain planes, unless float32 goes forward, and the scaled ones of float32
  const int64_t x_plane = l->few_fwd && l->few_bwd ? 0 : l->n_pad * l->dp * 2;
  l->x_factor = take(f32 ? l->n_pad * 4 : 0);
  l->x_scaled = take(f32 ? 2 * x_plane : 0);
  if (!f32) l->x = take(x_plane);
  const int64_t common = at;
  l->hit = take(l->n_pad * 4);
  l->part = take(l->parts * l->n_pad * 8);
  // W: one packed piece
  const int64_t fwd_plane = pack_w(p) && !l->few_fwd ? l->fwd_piece * l->dp * 2 : 0;
  l->w_fwd = take(f32 ? 2 * fwd_plane : fwd_plane);
  l->w_fwd_factor = take(f32 ? l->fwd_piece * 4 : 0);
  l->fwd_bytes = at;
  at = common;
  if (f32) l->x = take(3 * x_plane);  // (backward only)
  const int64_t bwd_plane = pack_w(p) && !l->few_bwd ? l->bwd_piece * l->dp * 2 : 0;
  l->w_bwd = take(l->planes * bwd_plane);
  l->w_bwd_scaled = take(f32 ? 2 * bwd_plane : 0);
  l->w_bwd_factor = take(f32 ? l->bwd_piece * 4 : 0);
  l->dz = take(l->few_bwd ? 0 : l->planes * l->n_pad * l->bwd_piece * 2);
  l->sum_rows = l->few_bwd ? kFewRows : l->n_pad;
  l->sums = take((int64_t)l->splits * l->sum_rows * l->dp * 4);
  l->bwd_bytes = at;
  return TCB200_OK;
}

Rows rows_of(char* ws, const Layout& l) {
  Rows r;
  r.head = reinterpret_cast<Head*>(ws);
  r.place = reinterpret_cast<int*>(ws + l.place);
  r.target = reinterpret_cast<int*>(ws + l.target);
  r.share = reinterpret_cast<float*>(ws + l.share);
  r.lse = reinterpret_cast<float*>(ws + l.lse);
  r.share_x = r.factor_x = nullptr;
  return r;
}

template <typename T, typename Index>
int launch_rows_typed(const tcb200_linear_ce_t& p, const Layout& l, const void* X, const void* target, const float* g,
                      int64_t g_stride, const float* lse, const Rows& r, const Planes& o, int sms, cudaStream_t s) {
  // blocks enough for the rows' copies, zero rows of the last tile among them
  const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(l.n_pad * (l.dp / 8), kRowThreads), 2ll * sms);
  TCB200_CUDA_TRY(launch_pdl(rows_kernel<T, Index>, dim3(blocks), dim3(kRowThreads), 0, s, static_cast<const Index*>(target),
                             p.N, p.V, p.ignore_index, g, g_stride, lse, r, static_cast<const T*>(X), p.ldx, p.D, l.dp, o,
                             Splits{l.splits * (l.n_pad / kTile), ceil_div(p.D, kTile), l.split_for,
                                    l.planes == 3 ? 6 : 1, std::max(1, sms / 2)}));
  return TCB200_OK;
}
// f16 and bf16 are copied as they are
int launch_rows(const tcb200_linear_ce_t& p, const Layout& l, const void* X, const void* target, const float* g,
                int64_t g_stride, const float* lse, const Rows& r, char* ws, int sms, cudaStream_t s) {
  Planes o{p.dtype == TCB200_F32 && !g ? nullptr : reinterpret_cast<uint16_t*>(ws + l.x), reinterpret_cast<uint16_t*>(ws + l.x_scaled),
           reinterpret_cast<float*>(ws + l.x_factor), l.n_pad * l.dp};
  const bool f32 = p.dtype == TCB200_F32, wide = p.index_bytes == 8;
  auto fn = f32 ? (wide ? launch_rows_typed<float, int64_t> : launch_rows_typed<float, int32_t>)
                : (wide ? launch_rows_typed<__half, int64_t> : launch_rows_typed<__half, int32_t>);
  return fn(p, l, X, target, g, g_stride, lse, r, o, sms, s);
}

int launch_pack(const tcb200_linear_ce_t& p, const Layout& l, const void* in, int64_t rows, const Planes& o, int sms, cudaStream_t s) {
  if (p.dtype == TCB200_F32) {
    const dim3 grid((unsigned)std::max<int64_t>(1, std::min<int64_t>(ceil_div(rows, 8), 8ll * sms)));
    TCB200_CUDA_TRY(launch_pdl(pack_rows_kernel, grid, dim3(256), 0, s, static_cast<const float*>(in), p.ldw, rows, p.D, l.dp, o));
  } else {
    const dim3 grid((unsigned)std::max<int64_t>(1, std::min<int64_t>(ceil_div(rows * (l.dp / 8), 256), 8ll * sms)));
    TCB200_CUDA_TRY(launch_pdl(pack_kernel, grid, dim3(256), 0, s, static_cast<const __half*>(in), p.ldw, rows, p.D, l.dp, o));
  }
  return TCB200_OK;
}

size_t elem_bytes(const tcb200_linear_ce_t& p) { return p.dtype == TCB200_F32 ? 4 : 2; }

// `products`: plane products per k-block.  `forward`: the loss keeps fp32 accuracy whatever the inputs' type.
pg::Args gemm_args(int64_t M, int64_t N, int64_t K, const int* live, int live_is_k, int* status, int products, bool forward) {
  pg::Args a = {};
  a.M = M;
  a.N = N;
  a.K = K;
  a.live = live;
  a.live_is_k = live_is_k;
  a.products = products;
  // A drain every 512 k (32 MMAs), 256 k of float32 operands (16 MMAs of the largest planes after those of smaller ones): the
  // truncation of the tensor core's sums then stays near 2^-20 of a term's size.  Gradients that are rounded to 16 bits
  // in the end take 1024 k: half as many drains, which leaves the epilogues twice the time before they hold up the MMAs
  // (dZ of 4096 x 2048 x 32000: 414 -> 350 us).
  a.chunk_kb = products > 1 ? 4 : forward ? 8 : 16;
  a.dev_status = status;
  return a;
}

// The operands of entries [v0, v0 + v) of W: in place, or packed into `o` (rows of dp).  `z` is the logits' operand, `plain` the
// gradient's.
int w_operands(const tcb200_linear_ce_t& p, const Layout& l, const void* W, int64_t v0, int64_t v, const Planes& o, int sms,
               cudaStream_t s, pg::Operand* z, pg::Operand* plain) {
  const char* base = static_cast<const char*>(W) + (size_t)v0 * p.ldw * elem_bytes(p);
  if (!pack_w(p)) {
    *z = *plain = {base, p.D, v, p.ldw, 1, 0};
    return TCB200_OK;
  }
  *plain = {o.plain, l.dp, v, l.dp, l.planes, o.stride};
  *z = p.dtype == TCB200_F32 ? pg::Operand{o.scaled, l.dp, v, l.dp, 2, o.stride} : *plain;
  return launch_pack(p, l, base, v, o, sms, s);
}

int current_device(int* device) {
  TCB200_CUDA_TRY(cudaGetDevice(device));
  return TCB200_OK;
}

template <typename T, int TYPE>
int backward_typed(const tcb200_linear_ce_t& p, const Layout& l, const void* W, const Rows& r, char* ws, T* dX, T* dW,
                   int device, int sms, cudaStream_t s, int* status, int* dev_status) {
  const bool bf16 = TYPE != kF16, f32 = TYPE == kF32;
  const float scale = TYPE == kF16 ? 1.f / kHalfScale : 1.f;
  const int products = f32 ? 6 : 1;
  const pg::Operand x{ws + l.x, l.dp, l.n_pad, l.dp, l.planes, l.n_pad * l.dp};
  const pg::Operand zx = f32 ? pg::Operand{ws + l.x_scaled, l.dp, l.n_pad, l.dp, 2, l.n_pad * l.dp} : x;
  const Planes packed{reinterpret_cast<uint16_t*>(ws + l.w_bwd), reinterpret_cast<uint16_t*>(ws + l.w_bwd_scaled),
                      reinterpret_cast<float*>(ws + l.w_bwd_factor), l.bwd_piece * l.dp};
  float* sums = reinterpret_cast<float*>(ws + l.sums);
  const int* live = &r.head->live;
  const float* share = dX && r.share_x ? r.share_x : r.share;
  int st;
  for (int64_t v0 = 0; v0 < p.V; v0 += l.bwd_piece) {
    const int64_t v = std::min(l.bwd_piece, p.V - v0), ld = l.bwd_piece;
    pg::Operand zw, w;
    if ((st = w_operands(p, l, W, v0, v, packed, sms, s, &zw, &w)) != TCB200_OK) return st;
    uint16_t* dz = reinterpret_cast<uint16_t*>(ws + l.dz);
    GradEpi<TYPE> ge{r.head, r.target, share, r.lse, ld, v0, v, reinterpret_cast<const float*>(ws + l.x_factor), packed.factor};
    CUtensorMap tc;
    if ((st = pg::make_out_map(&tc, {dz, ld, l.n_pad, ld, l.planes, l.n_pad * ld}, 2)) != TCB200_OK) return st;
    st = pg::launch_columns<false, false>(l.bwd_bn, zx, zw, TYPE == kBF16, gemm_args(p.N, v, p.D, live, 0, status, f32 ? 3 : 1, false), tc,
                                          ge, device, sms, s);
    if (st != TCB200_OK) return st;
    const pg::Operand z{dz, v, l.n_pad, ld, l.planes, l.n_pad * ld};
    if (dX) {
      const SumEpi se{r.head, l.dp, v0 > 0};
      st = pg::make_out_map(&tc, {sums, l.dp, l.splits * l.n_pad, l.dp, 1, 0}, 4);
      if (st != TCB200_OK) return st;
      pg::Args a = gemm_args(p.N, p.D, v, live, 0, status, products, false);
      a.splits = &r.head->splits;
      if ((st = pg::launch<256, false, true>(z, w, bf16, a, tc, se, device, sms, s)) != TCB200_OK) return st;
    }
    if (dW && share != r.share) {  // dZ once more with the common scale, where some row had another: no tile otherwise
      ge.share = r.share;
      if ((st = pg::make_out_map(&tc, {dz, ld, l.n_pad, ld, l.planes, l.n_pad * ld}, 2)) != TCB200_OK) return st;
      st = pg::launch_columns<false, false>(l.bwd_bn, zx, zw, false, gemm_args(p.N, v, p.D, &r.head->spread, 0, status, 1, false), tc, ge,
                                            device, sms, s);
      if (st != TCB200_OK) return st;
    }
    if (dW) {
      T* out = dW + v0 * p.D;
      const int tma = (p.D * sizeof(T)) % 16 == 0 && ((uintptr_t)out & 15) == 0;
      if (tma && (st = pg::make_out_map(&tc, {out, p.D, v, p.D, 1, 0}, sizeof(T))) != TCB200_OK) return st;
      const WeightEpi<T> we{r.head, out, v, p.D, scale, tma};
      st = pg::launch_columns<true, true>(l.dw_bn, z, x, bf16, gemm_args(v, p.D, p.N, live, 1, status, products, false), tc, we, device,
                                          sms, s);
      if (st != TCB200_OK) return st;
    }
  }
  const dim3 grid((unsigned)std::max<int64_t>(1, std::min<int64_t>(ceil_div(p.N * (l.dp / 8), 256), 8ll * sms)));
  TCB200_CUDA_TRY(launch_pdl(finish_kernel<T>, grid, dim3(256), 0, s, r, static_cast<const float*>(sums), l.dp, p.N, p.D, scale, dX, dW, p.V * p.D,
                             dev_status));
  return TCB200_OK;
}

}  // namespace
}  // namespace tcb200

using namespace tcb200;

extern "C" {

int tcb200_linear_ce_workspace(const tcb200_linear_ce_t* problem, int64_t* forward_bytes, int64_t* backward_bytes) {
  Layout l;
  const int st = layout_of(problem, sm_count(-1), &l);
  if (st != TCB200_OK) return st;
  if (forward_bytes) *forward_bytes = l.fwd_bytes;
  if (backward_bytes) *backward_bytes = l.bwd_bytes;
  return TCB200_OK;
}

int tcb200_linear_ce_forward(const tcb200_linear_ce_t* problem, const void* X, const void* W, const void* target,
                             float* loss, float* lse, void* workspace, int64_t workspace_bytes, tcb200_stream_t stream,
                             int* dev_status) {
  Layout l;
  int device, st = layout_of(problem, sm_count(-1), &l);
  if (st != TCB200_OK) return st;
  const tcb200_linear_ce_t& p = *problem;
  if (p.N == 0) return TCB200_OK;
  if (!X || !W || !target || !loss || !lse || !workspace) return TCB200_ERR_INVALID_ARGUMENT;
  if (workspace_bytes < l.fwd_bytes) return TCB200_ERR_INVALID_ARGUMENT;
  if (((uintptr_t)workspace & 127) || (!pack_w(p) && ((uintptr_t)W & 15))) return TCB200_ERR_ALIGNMENT;
  if ((st = current_device(&device)) != TCB200_OK) return st;
  const int sms = sm_count(device);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  const Rows r = rows_of(ws, l);
  int* status = &r.head->status;
  float2* part = reinterpret_cast<float2*>(ws + l.part);
  float* hit = reinterpret_cast<float*>(ws + l.hit);
  st = l.few_fwd ? few_forward(p, X, W, target, r, part, hit, l.n_pad, device, sms, s)
                 : launch_rows(p, l, X, target, nullptr, 0, nullptr, r, ws, sms, s);
  if (st != TCB200_OK) return st;
  const bool f32 = p.dtype == TCB200_F32;
  const pg::Operand x = f32 ? pg::Operand{ws + l.x_scaled, l.dp, l.n_pad, l.dp, 2, l.n_pad * l.dp}
                            : pg::Operand{ws + l.x, l.dp, l.n_pad, l.dp, 1, 0};
  uint16_t* packed = reinterpret_cast<uint16_t*>(ws + l.w_fwd);
  const Planes o{f32 ? nullptr : packed, f32 ? packed : nullptr, reinterpret_cast<float*>(ws + l.w_fwd_factor), l.fwd_piece * l.dp};
  for (int64_t v0 = l.few_fwd ? p.V : 0; v0 < p.V; v0 += l.fwd_piece) {
    const int64_t v = std::min(l.fwd_piece, p.V - v0), part0 = v0 / (l.fwd_bn / 2);
    pg::Operand w, unused;
    if ((st = w_operands(p, l, W, v0, v, o, sms, s, &w, &unused)) != TCB200_OK) return st;
    const pg::Args args = gemm_args(p.N, v, p.D, &r.head->live, 0, status, f32 ? 3 : 1, true);
    if (f32) {
      const ForwardEpi<true> e{r.head, r.target, part, hit, l.n_pad, v0, v, part0, reinterpret_cast<const float*>(ws + l.x_factor), o.factor};
      st = pg::launch_columns<false, false>(l.fwd_bn, x, w, false, args, CUtensorMap{}, e, device, sms, s);
    } else {
      const ForwardEpi<false> e{r.head, r.target, part, hit, l.n_pad, v0, v, part0, nullptr, nullptr};
      st = pg::launch_columns<false, false>(l.fwd_bn, x, w, p.dtype == TCB200_BF16, args, CUtensorMap{}, e, device, sms, s);
    }
    if (st != TCB200_OK) return st;
  }
  TCB200_CUDA_TRY(launch_pdl(join_kernel, dim3((unsigned)ceil_div(p.N, 32)), dim3(32, 32), 0, s, r,
                             static_cast<const float2*>(part), static_cast<const float*>(hit), l.parts, l.n_pad, p.N, loss, lse, dev_status));
  return TCB200_OK;
}

int tcb200_linear_ce_backward(const tcb200_linear_ce_t* problem, const void* X, const void* W, const void* target,
                              const float* lse, const float* grad_loss, int64_t grad_stride, void* dX, void* dW,
                              void* workspace, int64_t workspace_bytes, tcb200_stream_t stream, int* dev_status) {
  Layout l;
  int device, st = layout_of(problem, sm_count(-1), &l);
  if (st != TCB200_OK) return st;
  const tcb200_linear_ce_t& p = *problem;
  if (!dX && !dW) return TCB200_OK;
  if (grad_stride < 0) return TCB200_ERR_INVALID_ARGUMENT;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (p.N == 0) {  // no rows: dX is empty, dW the empty sum
    if (dW) TCB200_CUDA_TRY(cudaMemsetAsync(dW, 0, (size_t)p.V * p.D * elem_bytes(p), s));
    return TCB200_OK;
  }
  if (!X || !W || !target || !lse || !grad_loss || !workspace) return TCB200_ERR_INVALID_ARGUMENT;
  if (workspace_bytes < l.bwd_bytes) return TCB200_ERR_INVALID_ARGUMENT;
  if (((uintptr_t)workspace & 127) || (!pack_w(p) && ((uintptr_t)W & 15))) return TCB200_ERR_ALIGNMENT;
  if ((st = current_device(&device)) != TCB200_OK) return st;
  const int sms = sm_count(device);
  char* ws = static_cast<char*>(workspace);
  Rows r = rows_of(ws, l);
  int* status = &r.head->status;
  if (p.dtype == TCB200_F16 && dX && !l.few_bwd) {
    r.share_x = reinterpret_cast<float*>(ws + l.share_x);
    r.factor_x = reinterpret_cast<float*>(ws + l.factor_x);
  }
  if (l.few_bwd)
    return few_backward(p, X, W, target, lse, grad_loss, grad_stride, r, reinterpret_cast<float*>(ws + l.sums),
                        l.sum_rows * l.dp, l.dp, dX, dW, device, sms, s);
  st = launch_rows(p, l, X, target, grad_loss, grad_stride, lse, r, ws, sms, s);
  if (st != TCB200_OK) return st;
  switch (p.dtype) {
    case TCB200_F32:
      return backward_typed<float, kF32>(p, l, W, r, ws, static_cast<float*>(dX), static_cast<float*>(dW), device, sms, s, status, dev_status);
    case TCB200_F16:
      return backward_typed<__half, kF16>(p, l, W, r, ws, static_cast<__half*>(dX), static_cast<__half*>(dW), device, sms, s, status, dev_status);
    default:
      return backward_typed<__nv_bfloat16, kBF16>(p, l, W, r, ws, static_cast<__nv_bfloat16*>(dX), static_cast<__nv_bfloat16*>(dW),
                                                  device, sms, s, status, dev_status);
  }
}

}  // extern "C"

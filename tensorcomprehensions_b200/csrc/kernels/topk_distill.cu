// Distillation from a teacher's K largest logits, forward and backward.
//
//   q = softmax(teacher / T) over a row's K entries,  p = softmax(logits / T) over V
//   loss = T^2 sum_k q_k (ln q_k - ln p_{i_k}),  dlogits_v = T g (p_v - sum_{k: i_k = v} q_k)
//
// Both directions are one pass over [N, V] and bound by HBM: forward reads it, backward reads it and writes as much
// (4096 x 131072 bf16: 160 us, 6.7 TB/s, and 344 us, 6.3 TB/s).
//
// Forward: a cluster of CTAs takes a row (one CTA where the rows alone fill the device, up to eight where there are few), each
// thread keeps the running maximum and sum of its elements, the CTAs' pairs meet in the first CTA's shared memory.  The
// K entries are fetched before the pass over the row, so their latency hides behind it.
// Backward: the row's maximum and sum are known, so a CTA takes any stretch of a row: it writes T g p for all of it, then, behind
// a block barrier, writes the entries' places again with q taken off.  Equal indices are found by marking places in a bitmap;
// only they are compared with all entries (100 x 32000 f16, K = 4000, both directions: 4.1 ms with every entry compared, 69 us
// marked).  p - q is formed in fp32 and rounded once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "async.cuh"
#include "common.cuh"

namespace tcb200 {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

template <typename T> __device__ __forceinline__ float load1(const T* p);
template <> __device__ __forceinline__ float load1(const float* p) { return __ldg(p); }
template <> __device__ __forceinline__ float load1(const __half* p) { return __half2float(__ldg(p)); }
template <> __device__ __forceinline__ float load1(const __nv_bfloat16* p) { return __bfloat162float(__ldg(p)); }

template <typename T> __device__ __forceinline__ T make1(float v);
template <> __device__ __forceinline__ float make1(float v) { return v; }
template <> __device__ __forceinline__ __half make1(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 make1(float v) { return __float2bfloat16_rn(v); }

// 16 bytes of read-once data as floats
__device__ __forceinline__ uint4 load_raw(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ void store_raw(void* p, const uint4& v) {
  asm volatile("st.global.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// base-2 exponential; results below the smallest normal number become 0
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Eight 16-bit or four 32-bit elements of 16 bytes.
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int n = 4;
  static __device__ __forceinline__ float maximum(const uint4& r) {
    return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
  }
  static __device__ __forceinline__ void unpack(const uint4& r, float* v) {
    v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* v) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
};
template <> struct Vec<__half> {
  static constexpr int n = 8;
  static __device__ __forceinline__ float maximum(const uint4& r) {
    const __half2* h = reinterpret_cast<const __half2*>(&r);
    const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ void unpack(const uint4& r, float* v) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x; v[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int n = 8;
  static __device__ __forceinline__ float maximum(const uint4& r) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
  static __device__ __forceinline__ void unpack(const uint4& r, float* v) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

struct Entries {
  const void* indices;
  const void* teacher;
  int64_t ld_indices, ld_teacher;
  int k, index_bytes, teacher_dtype;
  __device__ int64_t index(int64_t row, int j) const {
    const int64_t at = row * ld_indices + j;
    return index_bytes == 8 ? __ldg(static_cast<const long long*>(indices) + at)
                            : (int64_t)__ldg(static_cast<const int*>(indices) + at);
  }
  __device__ float logit(int64_t row, int j) const {
    const int64_t at = row * ld_teacher + j;
    if (teacher_dtype == TCB200_F32) return load1(static_cast<const float*>(teacher) + at);
    if (teacher_dtype == TCB200_F16) return load1(static_cast<const __half*>(teacher) + at);
    return load1(static_cast<const __nv_bfloat16*>(teacher) + at);
  }
};

// exp((x - top) * T^-1).  The difference is taken first: it is exact where exp is not small, and rows of a type's lowest value
// neither overflow nor lose their sum, as x * scale - top * scale in one multiply-add would.
__device__ __forceinline__ float exp_from(float x, float top, float scale) { return exp2_fast((x - top) * scale); }

// Two exp((x - top) / T), x <= top, to about two units in the last place of float32 (below 2^-126: 0).  The exponent d log2(e) / T
// takes two floats, hi + lo on either side of the product, since rounded to one it is off by 2^-24 of itself and exp by that
// times the distance d (2^-18 at 60): 2^(t + r) = 2^t (1 + r ln 2) with t the rounded product and r what it leaves, d lo included.
// 512 x 50021 float32, K = 100, both directions: 69.8 us; with expf 74.8 us, with 2^t alone 68.8 us.
struct Exponent {
  float hi, lo;
};
__device__ __forceinline__ float2 exp_exact2(float2 x, float top, const Exponent& s) {
  const float floor = -160.f / s.hi;
  float2 d = __fadd2_rn(x, make_float2(-top, -top));
  d = make_float2(fmaxf(d.x, floor), fmaxf(d.y, floor));  // -inf too; a row with NaN is NaN by its sum
  const float2 neg = __fmul2_rn(d, make_float2(-s.hi, -s.hi));
  float2 r = __ffma2_rn(d, make_float2(s.hi, s.hi), neg);
  r = __ffma2_rn(d, make_float2(s.lo, s.lo), r);
  r = __fmul2_rn(r, make_float2(kLn2, kLn2));
  const float2 y = make_float2(exp2_fast(-neg.x), exp2_fast(-neg.y));
  return __ffma2_rn(y, r, y);
}

// Running maximum and sum of exp((x - maximum) * scale).  An empty pair is (-inf, 0).  A maximum drops NaN; the sum keeps it.
struct Running {
  float top = -INFINITY, sum = 0.f;
  __device__ __forceinline__ void join(float t, float s, float scale) {
    const float m = fmaxf(top, t), shift = m == -INFINITY ? 0.f : m;
    sum = sum * exp2_fast((top - shift) * scale) + s * exp2_fast((t - shift) * scale);
    top = m;
  }
  // moves the maximum up to m before elements of at most m are added
  __device__ __forceinline__ void raise(float m, float scale) {
    if (m > top) {
      sum *= exp2_fast((top - m) * scale);  // 0 while top is -inf
      top = m;
    }
  }
  __device__ __forceinline__ void one(float x, float scale) {
    raise(x, scale);
    sum += exp_from(x, top == -INFINITY ? 0.f : top, scale);
  }
  template <typename T, int U>
  __device__ __forceinline__ void vectors(const uint4 (&raw)[U], float scale) {
    float m = Vec<T>::maximum(raw[0]);
#pragma unroll
    for (int u = 1; u < U; ++u) m = fmaxf(m, Vec<T>::maximum(raw[u]));
    raise(m, scale);
    const float shift = top == -INFINITY ? 0.f : top;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[Vec<T>::n];
      Vec<T>::unpack(raw[u], x);
#pragma unroll
      for (int j = 0; j < Vec<T>::n; ++j) s[j & 3] += exp_from(x[j], shift, scale);
    }
    sum += (s[0] + s[1]) + (s[2] + s[3]);
  }
};

// The pair of a whole warp: the maximum first, then the sums moved to it, so that the shuffles carry one exponential.
__device__ __forceinline__ Running warp_join(Running r, float scale) {
  float m = r.top;
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  r.raise(m, scale);
  for (int o = 16; o; o >>= 1) r.sum += __shfl_xor_sync(0xffffffffu, r.sum, o);
  return r;
}
// All threads get the block's pairs (two at once); `share` holds two pairs a warp.  Pairs are joined in a fixed order.
template <int kThreads>
__device__ __forceinline__ void block_join(Running& a, Running& b, float scale, float4* share) {
  a = warp_join(a, scale);
  b = warp_join(b, scale);
  if ((threadIdx.x & 31) == 0) share[threadIdx.x >> 5] = make_float4(a.top, a.sum, b.top, b.sum);
  __syncthreads();
  // every warp joins the warps' pairs, a lane each
  const int lane = threadIdx.x & 31;
  const float4 x = lane < kThreads / 32 ? share[lane] : make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
  a.top = x.x; a.sum = x.y;
  b.top = x.z; b.sum = x.w;
  a = warp_join(a, scale);
  b = warp_join(b, scale);
}

// [first, last) of a row for part `i` of `n`: whole 64-element steps, so that the parts' inner bounds keep the alignment of the row
__device__ __forceinline__ void stretch(int64_t v, int i, int n, int64_t* first, int64_t* last) {
  const int64_t step = ((v + n - 1) / n + 63) / 64 * 64;
  *first = min(v, i * step);
  *last = min(v, *first + step);
}

constexpr int kMaxCluster = 8;

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads) distill_forward_kernel(const T* logits, int64_t ld, int64_t v, Entries e,
                                                                   float temperature, float* loss, float* stats, int parts) {
  __shared__ float4 share[kThreads / 32];
  __shared__ float sums[kThreads / 32];
  __shared__ float2 gathered[kMaxCluster];
  // A CTA's shared memory may be touched by its peers only once it runs: all say so here, and wait behind their stretch.
  if (parts > 1) cluster_arrive();
  pdl_sync();
  const int rank = (int)(blockIdx.x % parts);
  const int64_t row = blockIdx.x / parts;
  const T* z = logits + row * ld;
  const float inv = 1.f / temperature, scale = kLog2e * inv;
  // The first entry of a thread (all of them where K is at most the block) is fetched here and used behind the row.
  const bool mine = rank == 0 && threadIdx.x < e.k;
  const int64_t place = mine ? e.index(row, threadIdx.x) : -1;
  const float teacher = mine ? e.logit(row, threadIdx.x) : 0.f;
  int64_t first, last;
  stretch(v, rank, parts, &first, &last);
  Running r;
  constexpr int W = Vec<T>::n;
  // elements up to the first 16-byte boundary, whole vectors, the rest
  const int64_t head = min(last, first + (int64_t)((16 - ((uintptr_t)(z + first) & 15)) & 15) / (int64_t)sizeof(T));
  const int vecs = (int)((last - head) / W);
  const T* body = z + head;
  int i = threadIdx.x;
  constexpr int U = 4;  // loads in flight a thread
  for (; i + (U - 1) * kThreads < vecs; i += U * kThreads) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = load_raw(body + (int64_t)(i + u * kThreads) * W);
    r.vectors<T, U>(raw, scale);
  }
  for (; i < vecs; i += kThreads) {
    const uint4 raw[1] = {load_raw(body + (int64_t)i * W)};
    r.vectors<T, 1>(raw, scale);
  }
  if (first + threadIdx.x < head) r.one(load1(z + first + threadIdx.x), scale);
  const int64_t rest = head + (int64_t)vecs * W + threadIdx.x;
  if (rest < last) r.one(load1(z + rest), scale);
  // the entries' maximum and sum go along with the row's
  const float student = place >= 0 && place < v ? load1(z + place) : 0.f;
  bool bad = place >= v;
  Running t;
  if (place >= 0) t.one(teacher, scale);
  if (rank == 0)
    for (int j = threadIdx.x + kThreads; j < e.k; j += kThreads) {
      const int64_t at = e.index(row, j);
      bad |= at >= v;
      if (at >= 0) t.one(e.logit(row, j), scale);
    }
  block_join<kThreads>(r, t, scale, share);
  if (parts > 1) {
    __syncwarp();
    cluster_wait();
    if (threadIdx.x == 0) {
      uint32_t at;
      asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(smem_u32(&gathered[rank])));
      asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(at), "f"(r.top), "f"(r.sum) : "memory");
    }
    __syncwarp();
    cluster_sync_all();
    if (rank != 0) return;
    r = Running();
    for (int c = 0; c < parts; ++c) r.join(gathered[c].x, gathered[c].y, scale);
  }
  // the sum of q (ln q - ln p); both logs are taken against their maxima, where they are exact to fp32
  const float log_sum = logf(r.sum), log_weight = logf(t.sum);
  auto term = [&](float x, float y) {
    if (x == -INFINITY) return 0.f;
    const float lq = (x - t.top) * inv - log_weight, q = expf(lq);
    return q <= 0.f ? 0.f : q * (lq - ((y - r.top) * inv - log_sum));  // (NaN goes through)
  };
  float sum = place >= 0 ? term(teacher, student) : 0.f;
  for (int j = threadIdx.x + kThreads; j < e.k; j += kThreads) {
    const int64_t at = e.index(row, j);
    if (at >= 0 && at < v) sum += term(e.logit(row, j), load1(z + at));
  }
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = sum;
  const bool any_bad = __syncthreads_or(bad);
  if (threadIdx.x == 0) {
    sum = 0.f;
    for (int w = 0; w < kThreads / 32; ++w) sum += sums[w];
    const float nan = __int_as_float(0x7fffffff);
    const bool none = t.top == -INFINITY && t.sum == 0.f;
    loss[row] = any_bad ? nan : none ? 0.f : temperature * temperature * sum;
    stats[3 * row] = r.top;
    stats[3 * row + 1] = r.sum;
    stats[3 * row + 2] = any_bad ? nan : none ? -INFINITY : log_weight;
  }
}

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads) distill_backward_kernel(const T* logits, int64_t ld, int64_t v, Entries e,
                                                                    float temperature, Exponent exponent, const float* stats, const float* g,
                                                                    int64_t g_stride, T* dlogits, int parts) {
  // Teacher logits, then q, of the entries of this stretch, their places in it (-1: none), two bits a place: taken by an entry,
  // by more than one.  q comes from the difference to the largest teacher logit, as in the forward pass: exact where exp is not
  // small, whatever the logits' size.  The maximum is found again here, among entries that are read anyway.
  extern __shared__ float entry_mem[];
  __shared__ float tops[kThreads / 32];
  pdl_sync();
  const int64_t row = blockIdx.x / parts;
  int64_t first, last;
  stretch(v, (int)(blockIdx.x % parts), parts, &first, &last);
  const T* z = logits + row * ld;
  T* out = dlogits + row * v;
  float* eq = entry_mem;
  int* ei = reinterpret_cast<int*>(entry_mem + e.k);
  uint32_t* taken = reinterpret_cast<uint32_t*>(ei + e.k);
  const int words = (int)((last - first + 31) / 32);
  for (int j = threadIdx.x; j < 2 * words; j += kThreads) taken[j] = 0;  // (used behind the first barrier)
  const float inv = 1.f / temperature;
  const float top = stats[3 * row], sum = stats[3 * row + 1], log_weight = stats[3 * row + 2];
  const bool none = log_weight == -INFINITY;
  float up = temperature * g[row * g_stride];
  if (log_weight != log_weight) up = log_weight;  // an index outside the vocabulary: the row is NaN
  float best = -INFINITY;
  for (int j = threadIdx.x; j < e.k; j += kThreads) {
    const int64_t i = e.index(row, j);
    const float x = i >= 0 ? e.logit(row, j) : -INFINITY;
    best = fmaxf(best, x);
    ei[j] = i >= first && i < last && !none ? (int)(i - first) : -1;
    eq[j] = x;
  }
  for (int o = 16; o; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = best;
  constexpr int W = Vec<T>::n;
  const float weight = up / sum;
  // float32 results show the rounding of the exponent, 16-bit ones do not
  auto exp_two = [&](float2 x) {
    if (sizeof(T) == 4) return exp_exact2(x, top, exponent);
    return make_float2(exp_from(x.x, top, exponent.hi), exp_from(x.y, top, exponent.hi));
  };
  auto grad_two = [&](float2 x) {
    const float2 p = exp_two(x);
    return none ? make_float2(0.f, 0.f) : make_float2(weight * p.x, weight * p.y);
  };
  auto grad = [&](float x) { return grad_two(make_float2(x, x)).x; };
  const bool same = (((uintptr_t)(z + first) ^ (uintptr_t)(out + first)) & 15) == 0;
  // where the two rows sit differently on their 16-byte lines, every element goes by itself
  const int64_t head = same ? min(last, first + (int64_t)((16 - ((uintptr_t)(z + first) & 15)) & 15) / (int64_t)sizeof(T)) : last;
  const int vecs = (int)((last - head) / W);
  for (int64_t i = first + threadIdx.x; i < head; i += kThreads) out[i] = make1<T>(grad(load1(z + i)));
  int i = threadIdx.x;
  constexpr int U = 4;
  for (; i + (U - 1) * kThreads < vecs; i += U * kThreads) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = load_raw(z + head + (int64_t)(i + u * kThreads) * W);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      alignas(8) float x[W];
      Vec<T>::unpack(raw[u], x);
#pragma unroll
      for (int j = 0; j < W; j += 2) *reinterpret_cast<float2*>(x + j) = grad_two(make_float2(x[j], x[j + 1]));
      store_raw(out + head + (int64_t)(i + u * kThreads) * W, Vec<T>::pack(x));
    }
  }
  for (; i < vecs; i += kThreads) {
    alignas(8) float x[W];
    Vec<T>::unpack(load_raw(z + head + (int64_t)i * W), x);
#pragma unroll
    for (int j = 0; j < W; j += 2) *reinterpret_cast<float2*>(x + j) = grad_two(make_float2(x[j], x[j + 1]));
    store_raw(out + head + (int64_t)i * W, Vec<T>::pack(x));
  }
  const int64_t at = head + (int64_t)vecs * W + threadIdx.x;
  if (at < last) {
    out[at] = make1<T>(grad(load1(z + at)));
  }
  __syncthreads();  // the entries' places are written again behind this
  for (int w = 0; w < kThreads / 32; ++w) best = fmaxf(best, tops[w]);
  for (int j = threadIdx.x; j < e.k; j += kThreads) {
    if (ei[j] < 0) continue;
    eq[j] = expf((eq[j] - best) * inv - log_weight);
    const uint32_t bit = 1u << (ei[j] & 31);
    if (atomicOr(&taken[ei[j] >> 5], bit) & bit) atomicOr(&taken[words + (ei[j] >> 5)], bit);
  }
  __syncthreads();
  for (int j = threadIdx.x; j < e.k; j += kThreads) {
    if (ei[j] < 0) continue;
    float q = eq[j];
    if (taken[words + (ei[j] >> 5)] >> (ei[j] & 31) & 1) {
      q = 0.f;  // all entries of this place, in order: equal indices write equal values
      for (int m = 0; m < e.k; ++m) q += ei[m] == ei[j] ? eq[m] : 0.f;
    }
    const float x = load1(z + first + ei[j]), p = exp_two(make_float2(x, x)).x / sum;
    out[first + ei[j]] = make1<T>(up * (p - q));
  }
}

// The loss carries T^2 and the exponents log2(e) / T: T^2 has to be a normal number, or the loss is infinite, NaN or lost (then 1 / T
// is one too: T lies between 2^-63 and 2^64).
bool temperature_ok(float t) {
  const float square = t * t;
  return t > 0.f && square >= 1.17549435e-38f && square <= 3.402823466e38f;
}

int check(const tcb200_topk_distill_t* p) {
  if (!p) return TCB200_ERR_INVALID_ARGUMENT;
  auto type_ok = [](int t) { return t == TCB200_F32 || t == TCB200_F16 || t == TCB200_BF16; };
  if (p->N < 0 || p->V < 1 || p->K < 1 || p->ld_logits < p->V || p->ld_indices < p->K || p->ld_teacher < p->K ||
      !type_ok(p->logits_dtype) || !type_ok(p->teacher_dtype) || (p->index_bytes != 4 && p->index_bytes != 8) ||
      !temperature_ok(p->temperature))
    return TCB200_ERR_INVALID_ARGUMENT;
  if (p->K > TCB200_TOPK_MAX || p->V >= (1ll << 31) || p->N >= (1ll << 27)) return TCB200_ERR_TOO_LARGE;
  return TCB200_OK;
}

Entries entries_of(const tcb200_topk_distill_t& p, const void* indices, const void* teacher) {
  return {indices, teacher, p.ld_indices, p.ld_teacher, (int)p.K, p.index_bytes, p.teacher_dtype};
}

// Threads of a CTA.  A short row is bound by its chain of loads and joins, not by its bytes: where the rows alone fill the device,
// two warps a row keep four times as many rows in flight as eight do (8192 x 600 f16, K = 20: 32 -> 13 us forward, 23 -> 13 us
// backward; 4096 x 8000 bf16, K = 50: 28 -> 20 and 28 -> 24).  Rows of 32 KB are better off with eight (4096 x 8000 f32 backward:
// 58 -> 53 us), and so are many entries (8192 x 600 f16, K = 250 forward: 59 -> 47 us).
int threads_for(const tcb200_topk_distill_t& p, int sms) {
  const int64_t row = p.V * (p.logits_dtype == TCB200_F32 ? 4 : 2);
  return p.N >= 8ll * sms && row <= 16384 && p.K <= 128 ? 64 : 256;
}

template <typename T>
int forward_typed(const tcb200_topk_distill_t& p, const void* logits, const Entries& e, float* loss, float* stats,
                  cudaStream_t s) {
  const int sms = sm_count(-1);
  // clusters while the rows make fewer than eight CTAs an SM and a CTA keeps 2048 elements
  int parts = 1;
  while (parts < kMaxCluster && p.N * parts < 8ll * sms && p.V / (parts * 2) >= 2048) parts *= 2;
  cudaLaunchConfig_t cfg = {};
  const int threads = threads_for(p, sms);
  cfg.gridDim = dim3((unsigned)(p.N * parts));
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = parts;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = parts > 1 ? 2 : 1;  // (a cluster of one is scheduled as slowly as any: 13 -> 22 us for 8192 x 600 f16)
  const auto kernel = threads == 64 ? distill_forward_kernel<T, 64> : distill_forward_kernel<T, 256>;
  TCB200_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, static_cast<const T*>(logits), p.ld_logits, p.V, e,
                                     p.temperature, loss, stats, parts));
  return TCB200_OK;
}

template <typename T>
int backward_typed(const tcb200_topk_distill_t& p, const void* logits, const Entries& e, const float* stats, const float* g,
                   int64_t g_stride, void* dlogits, cudaStream_t s) {
  const int sms = sm_count(-1);
  // stretches of at most 32768 elements, and of 2048 and more while the rows make fewer than eight CTAs an SM
  // (4096 x 131072 bf16, stretches of 8192 / 32768 / 65536 / 131072: 407 / 340 / 356 / 361 us)
  const int64_t fill = std::min<int64_t>(8ll * sms / p.N, p.V / 2048);
  const int parts = (int)std::max<int64_t>({1, fill, ceil_div(p.V, 32768)});
  // at most 32 KB of entries and 8 KB of bits
  const size_t smem = (size_t)p.K * 8 + (size_t)ceil_div(ceil_div(p.V, (int64_t)parts), (int64_t)64) * 16;
  const int threads = threads_for(p, sms);
  const double exact = 1.4426950408889634 / (double)p.temperature;
  const Exponent exponent{(float)exact, (float)(exact - (double)(float)exact)};
  const auto kernel = threads == 64 ? distill_backward_kernel<T, 64> : distill_backward_kernel<T, 256>;
  TCB200_CUDA_TRY(launch_pdl(kernel, dim3((unsigned)(p.N * parts)), dim3(threads), smem, s,
                             static_cast<const T*>(logits), p.ld_logits, p.V, e, p.temperature, exponent, stats, g, g_stride,
                             static_cast<T*>(dlogits), parts));
  return TCB200_OK;
}

}  // namespace
}  // namespace tcb200

using namespace tcb200;

extern "C" {

int tcb200_topk_distill_forward(const tcb200_topk_distill_t* problem, const void* logits, const void* indices,
                                const void* teacher, float* loss, float* stats, tcb200_stream_t stream) {
  const int st = check(problem);
  if (st != TCB200_OK) return st;
  const tcb200_topk_distill_t& p = *problem;
  if (p.N == 0) return TCB200_OK;
  if (!logits || !indices || !teacher || !loss || !stats) return TCB200_ERR_INVALID_ARGUMENT;
  const Entries e = entries_of(p, indices, teacher);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (p.logits_dtype) {
    case TCB200_F32: return forward_typed<float>(p, logits, e, loss, stats, s);
    case TCB200_F16: return forward_typed<__half>(p, logits, e, loss, stats, s);
    default: return forward_typed<__nv_bfloat16>(p, logits, e, loss, stats, s);
  }
}

int tcb200_topk_distill_backward(const tcb200_topk_distill_t* problem, const void* logits, const void* indices,
                                 const void* teacher, const float* stats, const float* grad_loss, int64_t grad_stride,
                                 void* dlogits, tcb200_stream_t stream) {
  const int st = check(problem);
  if (st != TCB200_OK) return st;
  const tcb200_topk_distill_t& p = *problem;
  if (p.N == 0) return TCB200_OK;
  if (!logits || !indices || !teacher || !stats || !grad_loss || !dlogits || grad_stride < 0) return TCB200_ERR_INVALID_ARGUMENT;
  const Entries e = entries_of(p, indices, teacher);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  switch (p.logits_dtype) {
    case TCB200_F32: return backward_typed<float>(p, logits, e, stats, grad_loss, grad_stride, dlogits, s);
    case TCB200_F16: return backward_typed<__half>(p, logits, e, stats, grad_loss, grad_stride, dlogits, s);
    default: return backward_typed<__nv_bfloat16>(p, logits, e, stats, grad_loss, grad_stride, dlogits, s);
  }
}

}  // extern "C"

// Distillation from a teacher's K largest logits, forward and backward.
//
//   q = softmax(teacher / T) over a row's K entries,  p = softmax(logits / T) over V
//   loss = T^2 sum_k q_k (ln q_k - ln p_{i_k}),  dlogits_v = T g (p_v - sum_{k: i_k = v} q_k)
//
// Both directions are one pass over [N, V] and bound by HBM: forward reads it, backward reads it and writes as much.
//
// Forward: a cluster of CTAs takes a row (one CTA where the rows alone fill the device, up to eight where there are few), each
// thread keeps the running maximum and sum of its elements, the CTAs' pairs meet in the first CTA's shared memory.  The
// K entries and the student's logits at their places are fetched before the pass over the row, so their latency hides
// behind it.
// Backward: the row's maximum and sum are known, so a CTA takes any stretch of a row: it writes T g p for all of it, then, behind a block barrier,
// writes the entries' places again with q taken off.  p - q is formed in fp32 and rounded once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "async.cuh"
#include "common.cuh"

namespace tcb200 {
namespace {

constexpr int kThreads = 512;
constexpr float kLog2e = 1.4426950408889634f;

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
  asm volatile("st.global.cs.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int n = 4;
  static __device__ __forceinline__ void unpack(const uint4& r, float* v) {
    v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* v) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
};
template <> struct Vec<__half> {
  static constexpr int n = 8;
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

// Running maximum and sum of exp((x - maximum) * scale).  An empty pair is (-inf, 0).
struct Running {
  float top = -INFINITY, sum = 0.f;
  __device__ __forceinline__ void join(float t, float s, float scale) {
    const float m = fmaxf(top, t), shift = m == -INFINITY ? 0.f : m;
    sum = sum * exp2f((top - shift) * scale) + s * exp2f((t - shift) * scale);
    top = m;
  }
  template <int N>
  __device__ __forceinline__ void add(const float* v, float scale) {
    float m = v[0];
#pragma unroll
    for (int j = 1; j < N; ++j) m = fmaxf(m, v[j]);
    m = fmaxf(m, top);
    const float shift = m == -INFINITY ? 0.f : m;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < N; ++j) s += exp2f((v[j] - shift) * scale);
    sum = (m > top ? sum * exp2f((top - shift) * scale) : sum) + s;  // sum is 0 while top is -inf
    top = m;
  }
};

// All threads get the block's pair; `share` holds one pair a warp.  Pairs are joined in a fixed order.
__device__ __forceinline__ Running block_join(Running r, float scale, float2* share) {
  for (int o = 16; o; o >>= 1)
    r.join(__shfl_xor_sync(0xffffffffu, r.top, o), __shfl_xor_sync(0xffffffffu, r.sum, o), scale);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) share[threadIdx.x >> 5] = make_float2(r.top, r.sum);
  __syncthreads();
  Running all;
  for (int w = 0; w < kThreads / 32; ++w) all.join(share[w].x, share[w].y, scale);
  return all;
}
__device__ __forceinline__ float block_sum(float v, float2* share) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) share[threadIdx.x >> 5].x = v;
  __syncthreads();
  float all = 0.f;
  for (int w = 0; w < kThreads / 32; ++w) all += share[w].x;
  return all;
}

// [first, last) of a row for part `i` of `n`: whole 64-element steps, so that the parts' inner bounds keep the alignment of the row
__device__ __forceinline__ void stretch(int64_t v, int i, int n, int64_t* first, int64_t* last) {
  const int64_t step = ((v + n - 1) / n + 63) / 64 * 64;
  *first = min(v, i * step);
  *last = min(v, *first + step);
}

constexpr int kMaxCluster = 8;

template <typename T>
__global__ void __launch_bounds__(kThreads) distill_forward_kernel(const T* logits, int64_t ld, int64_t v, Entries e,
                                                                   float temperature, float* loss, float* stats, int parts) {
  extern __shared__ float entry_mem[];       // teacher / T, then the student's logit of each entry
  __shared__ float2 share[kThreads / 32];
  __shared__ float2 gathered[kMaxCluster];
  __shared__ int bad;
  pdl_sync();
  const int rank = (int)(blockIdx.x % parts);
  const int64_t row = blockIdx.x / parts;
  const T* z = logits + row * ld;
  float* et = entry_mem;
  float* ez = entry_mem + e.k;
  const float inv = 1.f / temperature, scale = kLog2e * inv;
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  if (rank == 0) {
    for (int j = threadIdx.x; j < e.k; j += kThreads) {
      const int64_t i = e.index(row, j);
      float t = e.logit(row, j), s = 0.f;
      if (i >= v) bad = 1;
      if (i < 0) t = -INFINITY;
      if (i >= 0 && i < v) s = load1(z + i);
      et[j] = t;
      ez[j] = s;
    }
  }
  int64_t first, last;
  stretch(v, rank, parts, &first, &last);
  Running r;
  constexpr int W = Vec<T>::n;
  // elements up to the first 16-byte boundary, whole vectors, the rest
  const int64_t head = min(last, first + (int64_t)((16 - ((uintptr_t)(z + first) & 15)) & 15) / (int64_t)sizeof(T));
  const int64_t vecs = (last - head) / W;
  if (first + threadIdx.x < head) {
    const float x = load1(z + first + threadIdx.x);
    r.add<1>(&x, scale);
  }
  const T* body = z + head;
  int64_t i = threadIdx.x;
  constexpr int U = 4;  // loads in flight a thread
  for (; i + (U - 1) * kThreads < vecs; i += U * kThreads) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = load_raw(body + (i + u * kThreads) * W);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[W];
      Vec<T>::unpack(raw[u], x);
      r.add<W>(x, scale);
    }
  }
  for (; i < vecs; i += kThreads) {
    float x[W];
    Vec<T>::unpack(load_raw(body + i * W), x);
    r.add<W>(x, scale);
  }
  if (head + vecs * W + threadIdx.x < last) {
    const float x = load1(z + head + vecs * W + threadIdx.x);
    r.add<1>(&x, scale);
  }
  r = block_join(r, scale, share);
  if (parts > 1) {
    if (threadIdx.x == 0) {
      uint32_t at;
      asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(smem_u32(&gathered[rank])));
      asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(at), "f"(r.top), "f"(r.sum) : "memory");
    }
    cluster_sync_all();
    if (rank != 0) return;
    r = Running();
    for (int c = 0; c < parts; ++c) r.join(gathered[c].x, gathered[c].y, scale);
  }
  const float log_sum = logf(r.sum);
  // the entries: softmax of the teacher's logits, then the sum of q (ln q - ln p)
  Running t;
  for (int j = threadIdx.x; j < e.k; j += kThreads) t.add<1>(&et[j], scale);
  t = block_join(t, scale, share);
  const float log_weight = logf(t.sum);
  float sum = 0.f;
  for (int j = threadIdx.x; j < e.k; j += kThreads) {
    if (et[j] == -INFINITY) continue;
    const float lq = (et[j] - t.top) * inv - log_weight, q = exp2f(lq * kLog2e);
    // both logs are taken against their maxima, where they are exact to fp32
    if (!(q <= 0.f)) sum += q * (lq - ((ez[j] - r.top) * inv - log_sum));
  }
  sum = block_sum(sum, share);
  if (threadIdx.x == 0) {
    const float nan = __int_as_float(0x7fffffff);
    const bool none = t.top == -INFINITY && !(t.sum != t.sum);
    loss[row] = bad ? nan : none ? 0.f : temperature * temperature * sum;
    stats[3 * row] = r.top;
    stats[3 * row + 1] = r.sum;
    stats[3 * row + 2] = bad ? nan : none ? -INFINITY : t.top * inv + log_weight;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) distill_backward_kernel(const T* logits, int64_t ld, int64_t v, Entries e,
                                                                    float temperature, const float* stats, const float* g,
                                                                    int64_t g_stride, T* dlogits, int parts) {
  extern __shared__ float entry_mem[];  // q of the entries of this stretch, then their places in it (-1: none)
  pdl_sync();
  const int64_t row = blockIdx.x / parts;
  int64_t first, last;
  stretch(v, (int)(blockIdx.x % parts), parts, &first, &last);
  const T* z = logits + row * ld;
  T* out = dlogits + row * v;
  float* eq = entry_mem;
  int* ei = reinterpret_cast<int*>(entry_mem + e.k);
  const float inv = 1.f / temperature, scale = kLog2e * inv;
  const float top = stats[3 * row], sum = stats[3 * row + 1], log_weight = stats[3 * row + 2];
  const bool none = log_weight == -INFINITY;
  float up = temperature * g[row * g_stride];
  if (log_weight != log_weight) up = log_weight;  // an index outside the vocabulary: the row is NaN
  for (int j = threadIdx.x; j < e.k; j += kThreads) {
    const int64_t i = e.index(row, j);
    const bool mine = i >= first && i < last && !none;
    ei[j] = mine ? (int)(i - first) : -1;
    eq[j] = mine ? exp2f((e.logit(row, j) * inv - log_weight) * kLog2e) : 0.f;
  }
  constexpr int W = Vec<T>::n;
  // x - top is taken first: it is exact where p is not small, and a product rounded before it would not be
  const float weight = up / sum;
  auto grad = [&](float x) { return none ? 0.f : weight * exp2f((x - top) * scale); };
  const bool same = (((uintptr_t)(z + first) ^ (uintptr_t)(out + first)) & 15) == 0;
  // where the two rows sit differently on their 16-byte lines, every element goes by itself
  const int64_t head = same ? min(last, first + (int64_t)((16 - ((uintptr_t)(z + first) & 15)) & 15) / (int64_t)sizeof(T)) : last;
  const int64_t vecs = (last - head) / W;
  for (int64_t i = first + threadIdx.x; i < head; i += kThreads) out[i] = make1<T>(grad(load1(z + i)));
  int64_t i = threadIdx.x;
  constexpr int U = 4;
  for (; i + (U - 1) * kThreads < vecs; i += U * kThreads) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = load_raw(z + head + (i + u * kThreads) * W);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[W];
      Vec<T>::unpack(raw[u], x);
#pragma unroll
      for (int j = 0; j < W; ++j) x[j] = grad(x[j]);
      store_raw(out + head + (i + u * kThreads) * W, Vec<T>::pack(x));
    }
  }
  for (; i < vecs; i += kThreads) {
    float x[W];
    Vec<T>::unpack(load_raw(z + head + i * W), x);
#pragma unroll
    for (int j = 0; j < W; ++j) x[j] = grad(x[j]);
    store_raw(out + head + i * W, Vec<T>::pack(x));
  }
  if (head + vecs * W + threadIdx.x < last) {
    const int64_t at = head + vecs * W + threadIdx.x;
    out[at] = make1<T>(grad(load1(z + at)));
  }
  __syncthreads();  // the entries' places are written again behind this
  for (int j = threadIdx.x; j < e.k; j += kThreads) {
    if (ei[j] < 0) continue;
    float q = 0.f;  // all entries of this place, in order: equal indices write equal values
    for (int m = 0; m < e.k; ++m) q += ei[m] == ei[j] ? eq[m] : 0.f;
    const float p = exp2f((load1(z + first + ei[j]) - top) * scale) / sum;
    out[first + ei[j]] = make1<T>(up * (p - q));
  }
}

int check(const tcb200_topk_distill_t* p) {
  if (!p) return TCB200_ERR_INVALID_ARGUMENT;
  auto type_ok = [](int t) { return t == TCB200_F32 || t == TCB200_F16 || t == TCB200_BF16; };
  if (p->N < 0 || p->V < 1 || p->K < 1 || p->ld_logits < p->V || p->ld_indices < p->K || p->ld_teacher < p->K ||
      !type_ok(p->logits_dtype) || !type_ok(p->teacher_dtype) || (p->index_bytes != 4 && p->index_bytes != 8) ||
      !(p->temperature > 0.f) || !(p->temperature <= 3.402823466e38f))
    return TCB200_ERR_INVALID_ARGUMENT;
  if (p->K > TCB200_TOPK_MAX || p->V >= (1ll << 31) || p->N >= (1ll << 27)) return TCB200_ERR_TOO_LARGE;
  return TCB200_OK;
}

Entries entries_of(const tcb200_topk_distill_t& p, const void* indices, const void* teacher) {
  return {indices, teacher, p.ld_indices, p.ld_teacher, (int)p.K, p.index_bytes, p.teacher_dtype};
}

template <typename T>
int forward_typed(const tcb200_topk_distill_t& p, const void* logits, const Entries& e, float* loss, float* stats,
                  cudaStream_t s) {
  const int sms = sm_count(-1);
  // clusters while the rows leave the device (two CTAs an SM) idle and a CTA keeps 2048 elements
  int parts = 1;
  while (parts < kMaxCluster && p.N * parts * 2 <= 2 * sms && p.V / (parts * 2) >= 2048) parts *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.N * parts));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = (size_t)p.K * 8;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = parts;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  TCB200_CUDA_TRY(cudaLaunchKernelEx(&cfg, distill_forward_kernel<T>, static_cast<const T*>(logits), p.ld_logits, p.V, e,
                                     p.temperature, loss, stats, parts));
  return TCB200_OK;
}

template <typename T>
int backward_typed(const tcb200_topk_distill_t& p, const void* logits, const Entries& e, const float* stats, const float* g,
                   int64_t g_stride, void* dlogits, cudaStream_t s) {
  const int sms = sm_count(-1);
  // stretches of 2048 elements and more while the rows leave the device (four CTAs an SM) idle
  const int parts = (int)std::max<int64_t>(1, std::min<int64_t>(4ll * sms / p.N, p.V / 2048));
  TCB200_CUDA_TRY(launch_pdl(distill_backward_kernel<T>, dim3((unsigned)(p.N * parts)), dim3(kThreads), (size_t)p.K * 8, s,
                             static_cast<const T*>(logits), p.ld_logits, p.V, e, p.temperature, stats, g, g_stride,
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

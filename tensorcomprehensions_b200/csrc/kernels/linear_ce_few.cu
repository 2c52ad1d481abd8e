// Cross entropy of a linear layer for few rows: one token to sixteen where W would have to be packed for the tensor cores (float32, or
// 16-bit rows that start anywhere), and the forward pass of up to four rows of 16-bit types in place.  Bound by the pass over W.
//
// The products run on the fp32 units, in one pass: a warp takes four entries of the vocabulary at a time, its lanes go along D
// with wide loads, one chunk ahead, and the rows of X sit in shared memory as fp32, read once for the four entries.  Forward
// leaves a pair (maximum, sum) per row and block.  Backward needs no second pass over W in memory: a block gets the logits of
// its 32 entries as the forward does, turns them into dZ in shared memory, and goes over the same entries (now in the L2) once
// more with a thread per column group for dW = dZ^T X and its share of dX = dZ W.  dX is summed per block in shared memory and
// over the blocks by a second kernel, in fixed order.  dZ stays fp32, and nothing is packed.
#include "linear_ce.cuh"
#include "pair_gemm.cuh"

namespace tcb200 {
namespace lce {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kForwardSmem = 92 << 10;         // X: two blocks an SM at least, or one and the ring
constexpr int kBackwardSmem = 200 << 10;       // X and dX

// vocabulary entries a warp takes at a time: its sums are at most 32, one a lane in the end
__host__ __device__ constexpr int entries(int nr) { return nr <= 8 ? 4 : 32 / nr; }

struct Few {
  const void* target;
  int index_bytes;
  int64_t ignore, n, d, v, ldx, ldw;
  __device__ int64_t index(int i) const {
    return index_bytes == 8 ? static_cast<const int64_t*>(target)[i] : (int64_t)static_cast<const int32_t*>(target)[i];
  }
};

// A lane takes 16 bytes of a row at a time: E consecutive elements where all rows start on 16-byte boundaries (VEC), else
// every 32nd one.  32 lanes cover a chunk of 32 E columns.
template <typename T> struct Step {
  static constexpr int E = 16 / (int)sizeof(T), CHUNK = 32 * E;
};
template <typename T, bool VEC>
__device__ __forceinline__ int column(int lane, int j) { return VEC ? lane * Step<T>::E + j : j * 32 + lane; }

__host__ __device__ inline int64_t padded(int64_t d) { return (d + 255) / 256 * 256; }

template <typename T>
struct alignas(16) Raw {
  T v[Step<T>::E];
};
// A lane's elements of the chunk that starts at column c; zero behind column d.
template <typename T, bool VEC>
__device__ __forceinline__ Raw<T> load_chunk(const T* row, int c, int d, int lane) {
  constexpr int E = Step<T>::E;
  Raw<T> r;
  if (VEC && c + lane * E + E <= d) {
    *reinterpret_cast<uint4*>(&r) = __ldg(reinterpret_cast<const uint4*>(row + c + lane * E));
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int at = c + column<T, VEC>(lane, j);
      r.v[j] = at < d ? row[at] : from_float<T>(0.f);
    }
  }
  return r;
}
template <typename T, bool VEC>
__device__ __forceinline__ void load_x(const float* row, int c, int lane, float* x) {
  constexpr int E = Step<T>::E;
  if (VEC) {
#pragma unroll
    for (int j = 0; j < E; j += 4) {
      const float4 q = *reinterpret_cast<const float4*>(row + c + lane * E + j);
      x[j] = q.x; x[j + 1] = q.y; x[j + 2] = q.z; x[j + 3] = q.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j) x[j] = row[c + j * 32 + lane];
  }
}

// The rows of X as fp32; rows without a target, and what lies behind column d, are zero.
template <int NR, typename T>
__device__ __forceinline__ void stage_x(const Few& f, const T* x, float* sx) {
  const int dp = (int)padded(f.d);
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const bool live = r < f.n && f.index(r) != f.ignore;
#pragma unroll 4
    for (int c = threadIdx.x; c < dp; c += kThreads)
      sx[r * dp + c] = live && c < f.d ? to_float(x[r * f.ldx + c]) : 0.f;
  }
}

// The list acc, one per lane, summed over the warp: lane l gets value l / (32 / N).  Halves of the list change sides until a
// lane holds one value, then the rest of the lanes are added.
template <int N>
__device__ __forceinline__ float spread(float (&acc)[N], int lane) {
  int n = N;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    if (n > 1) {
      n /= 2;
      const bool up = lane & o;
#pragma unroll
      for (int i = 0; i < N / 2; ++i)
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

// A warp's entries of W as a stream of chunks, always one chunk ahead: the loads of a chunk are under way while the one before
// is multiplied, from one group of entries to the next too.
template <typename T, bool VEC, int PER>
struct Stream {
  const T* w;
  int64_t v, ldw;
  int d, lane;
  Raw<T> next[PER];
  __device__ __forceinline__ void fetch(int64_t v0, int c) {
#pragma unroll
    for (int e = 0; e < PER; ++e) next[e] = load_chunk<T, VEC>(w + min(v0 + e, v - 1) * ldw, c, d, lane);
  }
};

// The logits of the warp's entries from v0 for all rows, whose first chunk has been fetched; fetches that of those from v1 too.
// Lane l gets value l / (32 / (NR PER)) of the list [row][entry].
template <int NR, bool VEC, typename T>
__device__ __forceinline__ float logits_of(Stream<T, VEC, entries(NR)>& st, int64_t v0, int64_t v1, const float* sx, int dp) {
  constexpr int PER = entries(NR), E = Step<T>::E, CHUNK = Step<T>::CHUNK;
  float acc[NR * PER];
#pragma unroll
  for (int i = 0; i < NR * PER; ++i) acc[i] = 0.f;
  for (int c = 0; c < st.d; c += CHUNK) {
    Raw<T> now[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) now[e] = st.next[e];
    if (c + CHUNK < st.d) st.fetch(v0, c + CHUNK);
    else if (v1 < st.v) st.fetch(v1, 0);
    float wv[PER][E];
#pragma unroll
    for (int e = 0; e < PER; ++e)
#pragma unroll
      for (int j = 0; j < E; ++j) wv[e][j] = to_float(now[e].v[j]);
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      float xv[E];
      load_x<T, VEC>(sx + r * dp, c, st.lane, xv);
#pragma unroll
      for (int e = 0; e < PER; ++e)
#pragma unroll
        for (int j = 0; j < E; ++j) acc[r * PER + e] = fmaf(xv[j], wv[e][j], acc[r * PER + e]);
    }
  }
  return spread<NR * PER>(acc, st.lane);
}

// blocks of an SM: registers for the chunk ahead and the sums
__host__ __device__ constexpr int blocks_per_sm(int nr) { return nr <= 2 ? 3 : nr <= 8 ? 2 : 1; }

template <int NR, bool VEC, typename T>
__global__ void __launch_bounds__(kThreads, blocks_per_sm(NR)) few_forward_kernel(Few f, const T* x, const T* w, Rows rows, float2* part,
                                                               float* hit, int64_t n_pad) {
  constexpr int PER = entries(NR), SHARE = 32 / (NR * PER);
  extern __shared__ __align__(16) float sx[];
  __shared__ float2 pairs[kWarps][32];
  pdl_sync();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  stage_x<NR>(f, x, sx);
  if (blockIdx.x == 0 && threadIdx.x < f.n) {
    const int64_t t = f.index(threadIdx.x);
    rows.place[threadIdx.x] = t != f.ignore ? (int)threadIdx.x : -1;
    rows.target[threadIdx.x] = t >= 0 && t < f.v ? (int)t : -1;
    if (threadIdx.x == 0) *rows.head = Head{(int)f.n, 0, 1.f, 1};
  }
  const int value = lane / SHARE, r = value / PER, e = value % PER;
  const int64_t t = r < f.n ? f.index(r) : -1;
  __syncthreads();  // X is staged
  Running run;
  const int64_t step = (int64_t)gridDim.x * kWarps * PER;
  int64_t v0 = ((int64_t)blockIdx.x * kWarps + warp) * PER;
  Stream<T, VEC, PER> st{w, f.v, f.ldw, (int)f.d, lane};
  if (v0 < f.v) st.fetch(v0, 0);
  for (; v0 < f.v; v0 += step) {
    const float z = logits_of<NR, VEC>(st, v0, v0 + step, sx, (int)padded(f.d));
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
      for (int i = 0; i < PER; ++i) all.join(pairs[k][(threadIdx.x * PER + i) * SHARE]);
    part[blockIdx.x * n_pad + threadIdx.x] = make_float2(all.top, all.sum);
  }
}

// Forward where the rows of W start on 16-byte boundaries: a producer warp keeps a ring of boxes (32 entries x 512 bytes) full
// with TMA loads, 128 KB of them under way, and eight warps multiply, four entries each.  The plain loads above keep a
// quarter of that in flight (1 x 4096 x 128000 bf16: 560 us; this kernel 162 us, 6.5 TB/s).
constexpr int kRing = 8, kBoxRows = 32, kBoxBytes = kBoxRows * 512;
__host__ __device__ constexpr int ring_bytes() { return kRing * kBoxBytes + 128; }
constexpr int kRingSmem = ring_bytes() + kForwardSmem;
static_assert(kRingSmem <= 224 * 1024, "the ring and X exceed shared memory");
template <int NR, typename T>
__global__ void __launch_bounds__(kThreads + 32, 1) few_ring_kernel(const __grid_constant__ CUtensorMap tm, Few f, const T* x, Rows rows,
                                                                    float2* part, float* hit, int64_t n_pad) {
  constexpr int E = Step<T>::E, CHUNK = Step<T>::CHUNK, PER = 4, SHARE = 32 / (NR * PER);
  static_assert(CHUNK * sizeof(T) == 512 && kWarps * PER == kBoxRows, "a box is a chunk of the block's entries");
  extern __shared__ __align__(128) uint8_t ring[];
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + kRing * kBoxBytes);
  uint64_t* empty = full + kRing;
  float* sx = reinterpret_cast<float*>(ring + ring_bytes());
  __shared__ float2 pairs[kWarps][32];
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, dp = (int)padded(f.d);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kRing; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], kWarps);
    }
    abort_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  pdl_sync();
  if (blockIdx.x == 0 && threadIdx.x < f.n) {
    const int64_t t = f.index(threadIdx.x);
    rows.place[threadIdx.x] = t != f.ignore ? (int)threadIdx.x : -1;
    rows.target[threadIdx.x] = t >= 0 && t < f.v ? (int)t : -1;
    if (threadIdx.x == 0) *rows.head = Head{(int)f.n, 0, 1.f, 1};
  }
  int* status = &rows.head->status;
  const int groups = (int)((f.v + kBoxRows - 1) / kBoxRows), chunks = (int)((f.d + CHUNK - 1) / CHUNK);
  if (warp == kWarps) {
    if (lane == 0) {
      int s = 0;
      uint32_t phase = 1;
      bool ok = true;
      for (int g = blockIdx.x; g < groups && ok; g += gridDim.x)
        for (int c = 0; c < chunks; ++c) {
          ok = mbar_wait(&empty[s], phase, 31, status, abort_flag);
          if (!ok) break;
          mbar_expect_tx(&full[s], kBoxBytes);
          tma_load_3d(ring + s * kBoxBytes, &tm, c * CHUNK, g * kBoxRows, 0, &full[s]);
          if (++s == kRing) {
            s = 0;
            phase ^= 1;
          }
        }
    }
  } else {
    stage_x<NR>(f, x, sx);
    asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");  // the multiplying warps
    const int value = lane / SHARE, r = value / PER, e = value % PER;
    const int64_t t = r < f.n ? f.index(r) : -1;
    Running run;
    int s = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int g = blockIdx.x; g < groups && ok; g += gridDim.x) {
      float acc[NR * PER];
#pragma unroll
      for (int i = 0; i < NR * PER; ++i) acc[i] = 0.f;
      for (int c = 0; c < chunks; ++c) {
        ok = mbar_wait(&full[s], phase, 32, status, abort_flag);
        if (!ok) break;
        const T* box = reinterpret_cast<const T*>(ring + s * kBoxBytes) + warp * PER * CHUNK + lane * E;
        Raw<T> now[PER];
#pragma unroll
        for (int k = 0; k < PER; ++k) *reinterpret_cast<uint4*>(&now[k]) = *reinterpret_cast<const uint4*>(box + k * CHUNK);
        float wv[PER][E];
#pragma unroll
        for (int k = 0; k < PER; ++k)
#pragma unroll
          for (int j = 0; j < E; ++j) wv[k][j] = to_float(now[k].v[j]);
        mbar_arrive_warp(&empty[s]);  // the box is in registers
        if (++s == kRing) {
          s = 0;
          phase ^= 1;
        }
#pragma unroll
        for (int i = 0; i < NR; ++i) {
          float xv[E];
          load_x<T, true>(sx + i * dp, c * CHUNK, lane, xv);
#pragma unroll
          for (int k = 0; k < PER; ++k)
#pragma unroll
            for (int j = 0; j < E; ++j) acc[i * PER + k] = fmaf(xv[j], wv[k][j], acc[i * PER + k]);
        }
      }
      if (!ok) break;
      const float z = spread<NR * PER>(acc, lane);
      const int64_t v = (int64_t)g * kBoxRows + warp * PER + e;
      if (lane % SHARE == 0 && r < f.n && v < f.v) {
        run.join(make_float2(z, 1.f));
        if (v == t) hit[r] = z;
      }
    }
    pairs[warp][lane] = make_float2(run.top, run.sum);
    asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
    if (threadIdx.x < f.n) {
      Running all;
      for (int k = 0; k < kWarps; ++k)
        for (int i = 0; i < PER; ++i) all.join(pairs[k][(threadIdx.x * PER + i) * SHARE]);
      part[blockIdx.x * n_pad + threadIdx.x] = make_float2(all.top, all.sum);
    }
  }
}

// 8 bytes, or one element, of a row
template <typename T, int COLS>
struct alignas(COLS * sizeof(T)) Cols {
  T v[COLS];
  __device__ __forceinline__ void load(const T* p) {
    if (COLS == 1) v[0] = p[0];
    else *reinterpret_cast<uint2*>(v) = __ldg(reinterpret_cast<const uint2*>(p));
  }
  __device__ __forceinline__ void store(T* p) const {
    if (COLS == 1) p[0] = v[0];
    else *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(v);
  }
};

template <int NR, bool VEC, typename T>
__global__ void __launch_bounds__(kThreads, NR <= 2 ? 2 : 1) few_backward_kernel(Few f, const T* x, const T* w, const float* lse,
                                                                const float* g, int64_t g_stride, Rows rows, float* sums,
                                                                int64_t plane, int64_t ld, T* dw, int need_x) {
  constexpr int PER = entries(NR), PER_BLOCK = kWarps * PER, SHARE = 32 / (NR * PER), COLS = VEC ? 8 / (int)sizeof(T) : 1, AHEAD = 8;
  extern __shared__ __align__(16) float sx[];
  __shared__ __align__(16) float dz[PER_BLOCK][NR];
  pdl_sync();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, dp = (int)padded(f.d);
  float* sdx = sx + NR * dp;
  stage_x<NR>(f, x, sx);
  for (int i = threadIdx.x; i < NR * dp; i += kThreads) sdx[i] = 0.f;
  if (blockIdx.x == 0 && threadIdx.x < f.n) {
    rows.place[threadIdx.x] = f.index(threadIdx.x) != f.ignore ? (int)threadIdx.x : -1;
    if (threadIdx.x == 0) *rows.head = Head{(int)f.n, 0, 1.f, 1};
  }
  const int value = lane / SHARE, r = value / PER, e = value % PER;
  const int64_t t = r < f.n ? f.index(r) : f.ignore;
  const bool live = r < f.n && t != f.ignore;
  const float l = live ? lse[r] : 0.f;
  const float up = !live ? 0.f : t >= 0 && t < f.v ? g[r * g_stride] : __int_as_float(0x7fffffff);
  __syncthreads();
  const int64_t step = (int64_t)gridDim.x * PER_BLOCK;
  Stream<T, VEC, PER> st{w, f.v, f.ldw, (int)f.d, lane};
  st.fetch((int64_t)blockIdx.x * PER_BLOCK + warp * PER, 0);
  for (int64_t b0 = (int64_t)blockIdx.x * PER_BLOCK; b0 < f.v; b0 += step) {
    const int64_t v0 = b0 + warp * PER;
    const float z = logits_of<NR, VEC>(st, v0, v0 + step, sx, dp);
    if (lane % SHARE == 0) {
      const float p = expf(z - l);
      dz[warp * PER + e][r] = live && v0 + e < f.v ? up * (v0 + e == t ? p - 1.f : p) : 0.f;
    }
    __syncthreads();
    // The same entries, now in the L2, with a thread per group of COLS columns: dW goes out, the share of dX is added up.
    const int have = (int)min((int64_t)PER_BLOCK, f.v - b0);
    for (int c = threadIdx.x * COLS; c < (int)f.d; c += kThreads * COLS) {
      float xv[NR][COLS], a[NR][COLS];
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int j = 0; j < COLS; ++j) {
          xv[i][j] = sx[i * dp + c + j];
          a[i][j] = 0.f;
        }
      for (int k0 = 0; k0 < have; k0 += AHEAD) {
        Cols<T, COLS> raw[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) raw[u].load(w + (b0 + min(k0 + u, have - 1)) * f.ldw + c);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          if (k0 + u >= have) break;
          float out[COLS];
#pragma unroll
          for (int j = 0; j < COLS; ++j) out[j] = 0.f;
#pragma unroll
          for (int i = 0; i < NR; ++i) {
            const float s = dz[k0 + u][i];
#pragma unroll
            for (int j = 0; j < COLS; ++j) {
              out[j] = fmaf(s, xv[i][j], out[j]);
              a[i][j] = fmaf(s, to_float(raw[u].v[j]), a[i][j]);
            }
          }
          if (dw) {
            Cols<T, COLS> q;
#pragma unroll
            for (int j = 0; j < COLS; ++j) q.v[j] = from_float<T>(out[j]);
            q.store(dw + (b0 + k0 + u) * f.d + c);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < NR; ++i)
#pragma unroll
        for (int j = 0; j < COLS; ++j) sdx[i * dp + c + j] += a[i][j];  // this thread's columns
    }
    __syncthreads();  // dz is written again
  }
  if (need_x)
    for (int i = threadIdx.x; i < (int)f.n * (int)ld; i += kThreads) {
      const int row = i / (int)ld, c = i % (int)ld;
      sums[blockIdx.x * plane + row * ld + c] = sdx[row * dp + c];
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

__host__ __device__ constexpr int padded_rows(int64_t n) { return n <= 1 ? 1 : n <= 2 ? 2 : n <= 4 ? 4 : n <= 8 ? 8 : 16; }
int64_t forward_smem(const tcb200_linear_ce_t& p) { return padded_rows(p.N) * padded(p.D) * 4; }

Few few_of(const tcb200_linear_ce_t& p, const void* target) {
  return {target, p.index_bytes, p.ignore_index, p.N, p.D, p.V, p.ldx, p.ldw};
}

bool aligned_rows(const void* base, int64_t ld, size_t bytes) { return ((uintptr_t)base & 15) == 0 && ld * bytes % 16 == 0; }

template <int NR, typename T>
int ring_launch(const tcb200_linear_ce_t& p, const void* X, const void* W, const void* target, const Rows& r, float2* part,
                float* hit, int64_t n_pad, int device, int sms, cudaStream_t s) {
  CUtensorMap tm;
  const int st = pg::make_plain_map(&tm, W, p.dtype, p.D, p.V, p.ldw, Step<T>::CHUNK, kBoxRows);
  if (st != TCB200_OK) return st;
  static std::atomic<uint64_t> configured{0};
  TCB200_CUDA_TRY(ensure_dynamic_smem(few_ring_kernel<NR, T>, kRingSmem, device, configured));
  TCB200_CUDA_TRY(launch_pdl(few_ring_kernel<NR, T>, dim3((unsigned)few_blocks(p, sms, false)), dim3(kThreads + 32),
                             (size_t)(ring_bytes() + forward_smem(p)), s, tm, few_of(p, target), static_cast<const T*>(X), r, part, hit,
                             n_pad));
  return TCB200_OK;
}

template <int NR, bool VEC, typename T>
int forward_launch(const tcb200_linear_ce_t& p, const void* X, const void* W, const void* target, const Rows& r, float2* part,
                   float* hit, int64_t n_pad, int device, int sms, cudaStream_t s) {
  static std::atomic<uint64_t> configured{0};
  TCB200_CUDA_TRY(ensure_dynamic_smem(few_forward_kernel<NR, VEC, T>, kForwardSmem, device, configured));
  TCB200_CUDA_TRY(launch_pdl(few_forward_kernel<NR, VEC, T>, dim3((unsigned)few_blocks(p, sms, false)), dim3(kThreads),
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
  TCB200_CUDA_TRY(launch_pdl(few_backward_kernel<NR, VEC, T>, dim3((unsigned)few_blocks(p, sms, true)), dim3(kThreads),
                             (size_t)(2 * forward_smem(p)), s, few_of(p, target), static_cast<const T*>(X),
                             static_cast<const T*>(W), lse, g, g_stride, r, sums, plane, ld, static_cast<T*>(dW), (int)(dX != nullptr)));
  if (dX)
    TCB200_CUDA_TRY(launch_pdl(few_finish_kernel<T>, dim3((unsigned)ceil_div(p.D, 32), (unsigned)p.N), dim3(32, 32), 0, s, r,
                               static_cast<const float*>(sums), (int)few_blocks(p, sms, true), plane, ld, p.D, static_cast<T*>(dX)));
  return TCB200_OK;
}

// 16-bit types come here with rows that start anywhere; float32 rows of that kind too, or (F32VEC) any
#define TCB200_FEW_CASE(NR, CALL, F32VEC)                                                                       \
  case NR:                                                                                                       \
    if (p.dtype == TCB200_F32) return F32VEC && vec ? CALL<NR, F32VEC, float> ARGS : CALL<NR, false, float> ARGS; \
    if (p.dtype == TCB200_F16) return CALL<NR, false, __half> ARGS;                                             \
    return CALL<NR, false, __nv_bfloat16> ARGS;

}  // namespace

// 4 x 2048 x 50000 float32, forward and gradient: 355 us here, 1155 us on the tensor cores; 6 x 92 x 38224 f16 with rows to be
// packed 91 and 136 us; 8 x 2048 x 50000 bf16 with aligned rows 546 and 224 us.
// The ring needs rows on 16-byte boundaries.  16-bit rows of W need no packing for the tensor cores either, which win from five
// rows up (8 x 2048 x 50000 bf16, forward: 56 us, here 83 us; one row of 4096 x 128000: 203 and 162 us).
bool ring_ok(const tcb200_linear_ce_t& p) {
  return p.N <= (p.dtype == TCB200_F32 ? 8 : 4) && !p.pack_w && p.ldw * (p.dtype == TCB200_F32 ? 4 : 2) % 16 == 0;
}
bool few_rows(const tcb200_linear_ce_t& p) { return p.dtype == TCB200_F32 ? p.N <= kFewRows : p.pack_w && p.N <= kFewRows / 2; }
bool few_forward_ok(const tcb200_linear_ce_t& p) { return (few_rows(p) || ring_ok(p)) && forward_smem(p) <= kForwardSmem; }
bool few_backward_ok(const tcb200_linear_ce_t& p) { return few_rows(p) && 2 * forward_smem(p) <= kBackwardSmem; }
int64_t few_blocks(const tcb200_linear_ce_t& p, int sms, bool backward) {
  const int nr = padded_rows(p.N);
  const int64_t per_sm = backward ? 2 : ring_ok(p) ? 1 : blocks_per_sm(nr);
  return std::min<int64_t>(ceil_div(p.V, kWarps * entries(nr)), sms * per_sm);
}

int few_forward(const tcb200_linear_ce_t& p, const void* X, const void* W, const void* target, const Rows& r, float2* part,
                float* hit, int64_t n_pad, int device, int sms, cudaStream_t s) {
  const bool vec = aligned_rows(W, p.ldw, p.dtype == TCB200_F32 ? 4 : 2);
#define ARGS (p, X, W, target, r, part, hit, n_pad, device, sms, s)
  if (vec && ring_ok(p)) {
#define TCB200_RING_CASE(NR)                                      \
  case NR:                                                        \
    if (p.dtype == TCB200_F32) return ring_launch<NR, float> ARGS; \
    if (p.dtype == TCB200_F16) return ring_launch<NR, __half> ARGS; \
    return ring_launch<NR, __nv_bfloat16> ARGS;
    switch (padded_rows(p.N)) {
      TCB200_RING_CASE(1)
      TCB200_RING_CASE(2)
      TCB200_RING_CASE(4)
      TCB200_RING_CASE(8)
    }
  }
  switch (padded_rows(p.N)) {
    TCB200_FEW_CASE(1, forward_launch, false)
    TCB200_FEW_CASE(2, forward_launch, false)
    TCB200_FEW_CASE(4, forward_launch, false)
    TCB200_FEW_CASE(8, forward_launch, false)
    case 16: return vec ? forward_launch<16, true, float> ARGS : forward_launch<16, false, float> ARGS;
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
    TCB200_FEW_CASE(1, backward_launch, true)
    TCB200_FEW_CASE(2, backward_launch, true)
    TCB200_FEW_CASE(4, backward_launch, true)
    TCB200_FEW_CASE(8, backward_launch, true)
    case 16: return vec ? backward_launch<16, true, float> ARGS : backward_launch<16, false, float> ARGS;
  }
#undef ARGS
  return TCB200_ERR_UNSUPPORTED;
}

}  // namespace lce
}  // namespace tcb200

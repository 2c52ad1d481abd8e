// 16-bit matrix products on CTA pairs with fp32 accuracy of the sum, shared by the kernels of the large-vocabulary
// losses (sm_100a).  One pair computes a tile C(m, n) = sum_k A(m, k) B(n, k) of 256 rows and BN = 256 or 128 columns; the
// epilogue is a functor that gets a row and C consecutive columns of it in registers.
//
// Operands are f16 or bf16 (both the same), each either k-major (rows of k) or mn-major (rows of m or n): the three
// products of a linear layer's training step (X W^T, dZ W, dZ^T X) then read the same arrays without a transposed copy.
// float32 operands arrive as two f16 planes (11 + 11 significand bits, scaled, the low plane by another 2^11) or three bf16 planes
// (8 + 8 + 8); of the plane products those with i + j <= 1, or <= 2, are summed, smallest first: the largest dropped one is
// 2^-22, or 2^-24, of the product at most.  The 2^11 is taken off the accumulator by the MMA that begins the product of the high
// planes.
//
// Roles of a CTA: 4 BN / C warps drain the accumulator and run the epilogue, one issues the TMA loads of this CTA's 128 rows
// of A and BN / 2 of the tile's BN rows of B, and the leader's last one issues the MMAs (M = 256, N = BN, K = 16) of both CTAs.  In both issuing warps all lanes run the loop and one elected lane issues, so that descriptors and addresses stay in
// uniform registers.  With loops that only lane 0 ran, a k-block's loads took 400 cycles to issue and its four MMAs 300, and a
// k-block 740 cycles where its MMAs take 512 (4096 x 2048 x 32000, forward: 393 us; now 332 us, 1.62 PFLOP/s).  Of the rest
// two issuers with half of the columns each, shorter or longer rings (4 to 6 stages) and higher boxes gained nothing.
// The tensor core adds into its accumulator with truncation, so a sum of hundreds of MMAs drifts
// (about half an ulp each, all the same way); the accumulator is therefore drained every `chunk_kb` k-blocks into registers
// and the chunks are added there with rounding to nearest.  Two accumulators of 256 columns alternate, so the drain of one
// runs under the MMAs of the other.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "tcgen05.cuh"

namespace tcb200 {
namespace pg {

constexpr int kTile = 256;      // tile rows of a pair, and its columns at most
constexpr int kHalf = 128;      // rows of A, and of B at most, that one CTA loads
constexpr int kBK = 64;         // k of a stage: one 128-byte swizzle row of 16-bit values
constexpr int kOperandBytes = kHalf * kBK * 2;
constexpr int kStageBytes = 2 * kOperandBytes;
// BN: columns of a tile; C: columns of a drain warp (there are four lane quarters of tensor memory).
__host__ __device__ constexpr int drain_warps(int bn, int c) { return 4 * (bn / c); }
__host__ __device__ constexpr int block_threads(int bn, int c) { return (drain_warps(bn, c) + 2) * 32; }
__host__ __device__ constexpr int stages(int bn, int c) { return drain_warps(bn, c) > 8 ? 5 : 6; }
constexpr int kBarrierBytes = 256;
constexpr int kOutBytes = 4096;  // staging of a drain warp: 32 rows of 128 bytes
__host__ __device__ constexpr int out_offset(int bn, int c) { return stages(bn, c) * kStageBytes; }
__host__ __device__ constexpr int barrier_offset(int bn, int c) { return out_offset(bn, c) + drain_warps(bn, c) * kOutBytes; }
__host__ __device__ constexpr int smem_bytes(int bn, int c) { return barrier_offset(bn, c) + kBarrierBytes + 1024; }
static_assert(smem_bytes(256, 128) <= 227 * 1024 && smem_bytes(256, 64) <= 227 * 1024, "the stages exceed shared memory");
constexpr int kMaxProducts = 6;

struct Args {
  int64_t M, N, K;          // extents; one of them may be replaced by *live
  const int* live;          // null, or a device count that replaces M (live_is_k = 0) or K (live_is_k = 1)
  int live_is_k;
  int products;             // plane products per k-block: 1, or 3 or 6 for float32
  int pa[kMaxProducts], pb[kMaxProducts];
  int chunk_kb;             // k-blocks per drain
  const int* splits;        // null, or a device count of units that the reduction of a tile is split over
  uint32_t idesc;           // instruction descriptor
  int* dev_status;
};

// Loads whose completion is counted on a barrier of either CTA of the pair: the peer's loads arrive on the leader's.
__device__ __forceinline__ void tma_load_3d_pair(void* dst, const CUtensorMap* tm, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
      "%3, %4}], [%5];" ::"r"(smem_u32(dst)),
      "l"(tm), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ uint32_t map_to_rank(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void umma_f16_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                              uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// D = A B + D 2^-kLowShift
constexpr int kLowShift = 11;
__device__ __forceinline__ void umma_f16_pair_shifted(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.eq.u32 p, 0, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p, %4;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "n"(kLowShift)
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// Shared-memory descriptors, 128-byte swizzle.  k-major: rows of 64 k, 8-row groups 1024 bytes apart.  mn-major: groups of 64
// m (or n) of 64 k-rows of 128 bytes each; 8-row groups of k 1024 bytes apart, groups of 64 m kBK * 128 bytes apart.
template <bool MN>
__device__ __forceinline__ uint64_t operand_desc(uint32_t saddr) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr & 0x3FFFF) >> 4);
  d |= (uint64_t)(MN ? (kBK * 128) >> 4 : 1) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;  // descriptor version of sm_100
  d |= (uint64_t)2 << 61;  // 128-byte swizzle
  return d;
}
// bytes from one MMA's k (16) to the next within a stage
template <bool MN>
__host__ __device__ constexpr uint32_t k_step_bytes() { return MN ? 16 * 128 : 32; }

// kind::f16: D = f32, A = B = f16 (bf16 = 0) or bf16, each k-major or mn-major.
__host__ inline uint32_t make_idesc(bool bf16, bool a_mn, bool b_mn, int bn) {
  const uint32_t t = bf16 ? 1 : 0;
  return (1u << 4) | (t << 7) | (t << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(bn >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}

// One operand stage of this CTA: ROWS (128 or 64) rows of m (or n) from mn0, 64 k from k0.
template <bool MN, int ROWS>
__device__ __forceinline__ void load_operand(uint8_t* dst, const CUtensorMap* tm, int mn0, int k0, int plane, uint32_t bar) {
  if (MN) {
    tma_load_3d_pair(dst, tm, mn0, k0, plane, bar);
    if (ROWS > 64) tma_load_3d_pair(dst + kBK * 128, tm, mn0 + 64, k0, plane, bar);
  } else {
    tma_load_3d_pair(dst, tm, k0, mn0, plane, bar);
  }
}

// Splits of a reduction over `kb` k-blocks of `products` plane products whose result has `tiles` tiles, at most `most`: the number
// that ends first on `pairs` pairs.  In k-blocks of a pair: rounds x (a unit's k-blocks + 8 for its start and epilogue) + what
// adding the partial sums costs (writing and reading a tile of one takes about 9).  Candidates are one, and what fills whole
// rounds with units of eight k-blocks and more.
__host__ __device__ inline int choose_splits(int tiles, int kb, int products, int pairs, int most) {
  const int steps = kb * products, shortest = steps / 8 < kb ? steps / 8 : kb;
  if (most > shortest) most = shortest;
  int best = 1;
  int64_t least = INT64_MAX;
  for (int rounds = 0; rounds <= 7; ++rounds) {
    int s = rounds ? (int)((int64_t)rounds * pairs / tiles) : 1;
    if (s > most) s = most;
    if (s < 1) continue;
    const int64_t cost = (int64_t)((tiles * s + pairs - 1) / pairs) * ((steps + s - 1) / s + 8) + (int64_t)s * (9 * tiles / pairs + 1);
    if (cost < least) {
      least = cost;
      best = s;
    }
  }
  return best;
}
constexpr int kMaxSplits = 64;

// A unit is (tile, split).  Tiles are taken in groups of 8 tile rows, rows fastest inside a group: the pairs that run at the
// same time then share rows of B (8 pairs each) and of A, which the L2 serves.
struct Units {
  int64_t tiles_m, tiles_n, units;
  int kb, splits, split_kb;
  __device__ Units(const Args& a, int bn) {
    int64_t M = a.M, K = a.K;
    if (a.live) (a.live_is_k ? K : M) = *a.live;
    tiles_m = (M + kTile - 1) / kTile;
    tiles_n = (a.N + bn - 1) / bn;
    kb = (int)((K + kBK - 1) / kBK);
    splits = a.splits ? *a.splits : 1;
    split_kb = (kb + splits - 1) / splits;
    units = tiles_m * tiles_n * splits;
  }
  __device__ void locate(int64_t u, int64_t* tm, int64_t* tn, int* split, int* kb0, int* nkb) const {
    const int64_t tiles = tiles_m * tiles_n;
    *split = (int)(u / tiles);
    int64_t t = u % tiles;
    const int64_t per_group = 8 * tiles_n, g = t / per_group;
    const int64_t rows = tiles_m - g * 8 < 8 ? tiles_m - g * 8 : 8;
    t -= g * per_group;
    *tm = g * 8 + t % rows;
    *tn = t / rows;
    *kb0 = *split * split_kb;
    const int left = kb - *kb0;
    *nkb = left < 0 ? 0 : (left < split_kb ? left : split_kb);
  }
};

// How an epilogue writes: a thread owns a row, so stores straight from its registers touch 32 rows an instruction.  Instead a
// warp puts 32 rows x 128 bytes into its staging buffer (16-byte chunks permuted as the 128-byte swizzle does: free of
// bank conflicts) and one lane sends the box with a TMA store, which clips at the tensor's edge.
struct Out {
  uint8_t* buf;
  int lane;
  // the previous box has left the buffer
  __device__ __forceinline__ void begin() const {
    if (lane == 0) tma_store_wait_read();
    __syncwarp();
  }
  __device__ __forceinline__ void put(int chunk, const uint4& v) const {
    *reinterpret_cast<uint4*>(buf + lane * 128 + ((chunk ^ (lane & 7)) << 4)) = v;
  }
  __device__ __forceinline__ void send(const CUtensorMap* tm, int x, int y, int z) const {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) {
      tma_store_3d(tm, buf, x, y, z);
      tma_store_commit();
    }
  }
  // the same, added to what memory holds (fp32)
  __device__ __forceinline__ void send_add(const CUtensorMap* tm, int x, int y, int z) const {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) {
      asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(tm),
                   "r"(x), "r"(y), "r"(z), "r"(smem_u32(buf))
                   : "memory");
      tma_store_commit();
    }
  }
  // element `col` (of `bytes` bytes) of row `row`, for rows that no TMA store can address
  __device__ __forceinline__ const void* at(int row, int col, int bytes) const {
    const int b = col * bytes;
    return buf + row * 128 + (((b >> 4) ^ (row & 7)) << 4) + (b & 15);
  }
};

// Epi: struct with  template <int C> __device__ void operator()(float (&acc)[C], int row, int col0, int split,
// const CUtensorMap* tm, const Out& out), where row and col0 are the thread's row and first of its C columns (both may lie outside
// the result), and the constants kColumns and kDirect (below) and kShifted (operands are two scaled planes: three products).
template <int BN, int C, bool A_MN, bool B_MN, class Epi>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(block_threads(BN, C), 1)
pair_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                 const __grid_constant__ CUtensorMap tmC, const __grid_constant__ Args a, const __grid_constant__ Epi epi) {
  static_assert(BN == 256 || BN == 128, "an operand's mn-major rows are whole 64-element groups in each CTA");
  constexpr int B_ROWS = BN / 2;  // rows of B that this CTA loads
  constexpr int DRAIN = drain_warps(BN, C), kStages = stages(BN, C);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + barrier_offset(BN, C));  // used in the leader: both CTAs' loads
  uint64_t* empty = full + kStages;
  uint64_t* acc_full = empty + kStages;   // [2]
  uint64_t* acc_empty = acc_full + 2;     // [2], used in the leader: the drain warps of both CTAs
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  static_assert((2 * kStages + 4) * 8 + 8 <= kBarrierBytes, "barrier area");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int64_t pair = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * DRAIN);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == DRAIN + 1) tmem_alloc_pair(tmem_slot, 512);
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  pdl_sync();
  const uint32_t tmem_base = *tmem_slot;

  const Units units(a, BN);

  if (warp == DRAIN) {
    // ------------------------------------------------ TMA producer
    const bool issuer = elect_one();
    const uint32_t full0 = map_to_rank(&full[0], 0);
    int s = 0;
    uint32_t phase = 1;
    bool ok = true;
    for (int64_t u = pair; u < units.units && ok; u += num_pairs) {
      int64_t tm, tn;
      int split, kb0, nkb;
      units.locate(u, &tm, &tn, &split, &kb0, &nkb);
      const int m0 = (int)(tm * kTile) + (int)rank * kHalf, n0 = (int)(tn * BN) + (int)rank * B_ROWS;
      for (int c0 = 0; c0 < nkb && ok; c0 += a.chunk_kb) {
        const int c1 = c0 + a.chunk_kb < nkb ? c0 + a.chunk_kb : nkb;
        for (int p = 0; p < a.products && ok; ++p)
          for (int kb = c0; kb < c1; ++kb) {
            ok = mbar_wait(&empty[s], phase, 21, a.dev_status, abort_flag);
            if (!ok) break;
            if (issuer) {
              if (rank == 0) mbar_expect_tx(&full[s], 2 * (kOperandBytes + B_ROWS * kBK * 2));
              uint8_t* dst = smem + s * kStageBytes;
              load_operand<A_MN, kHalf>(dst, &tmA, m0, (kb0 + kb) * kBK, a.pa[p], full0 + s * 8);
              load_operand<B_MN, B_ROWS>(dst + kOperandBytes, &tmB, n0, (kb0 + kb) * kBK, a.pb[p], full0 + s * 8);
            }
            __syncwarp();
            if (++s == kStages) {
              s = 0;
              phase ^= 1;
            }
          }
      }
    }
  } else if (warp == DRAIN + 1) {
    // ------------------------------------------------ MMA issuer
    if (rank == 0) {
      const bool issuer = elect_one();
      const uint32_t smem0 = __shfl_sync(0xffffffffu, smem_u32(smem), 0);
      const uint32_t tmem0 = __shfl_sync(0xffffffffu, tmem_base, 0);
      int s = 0;
      uint32_t phase = 0, chunk = 0;
      bool ok = true;
      for (int64_t u = pair; u < units.units && ok; u += num_pairs) {
        int64_t tm, tn;
        int split, kb0, nkb;
        units.locate(u, &tm, &tn, &split, &kb0, &nkb);
        for (int c0 = 0; c0 < nkb && ok; c0 += a.chunk_kb, ++chunk) {
          const int c1 = c0 + a.chunk_kb < nkb ? c0 + a.chunk_kb : nkb;
          const int steps = (c1 - c0) * a.products;
          const int b = chunk & 1;
          ok = mbar_wait(&acc_empty[b], ((chunk >> 1) & 1) ^ 1, 22, a.dev_status, abort_flag);
          if (!ok) break;
          tc_fence_after();
          // (a loop of its own around the shift: with a choice in one loop the descriptors leave the uniform registers)
          auto step = [&](int i, auto shift) {
            ok = mbar_wait(&full[s], phase, 23, a.dev_status, abort_flag);
            if (!ok) return;
            tc_fence_after();
            const uint32_t sa = smem0 + s * kStageBytes, sb = sa + kOperandBytes;
            const uint64_t da = operand_desc<A_MN>(sa), db = operand_desc<B_MN>(sb);
            if (issuer) {
              if constexpr (decltype(shift)::value) umma_f16_pair_shifted(tmem0 + b * kTile, da, db, a.idesc);
#pragma unroll
              for (int k = decltype(shift)::value; k < kBK / 16; ++k)
                umma_f16_pair(tmem0 + b * kTile, da + (uint64_t)(k * k_step_bytes<A_MN>() >> 4),
                              db + (uint64_t)(k * k_step_bytes<B_MN>() >> 4), a.idesc, k > 0 || i > 0);
              umma_commit_pair(&empty[s]);
              if (i == steps - 1) umma_commit_pair(&acc_full[b]);
            }
            __syncwarp();
            if (++s == kStages) {
              s = 0;
              phase ^= 1;
            }
          };
          int i = 0;
          if constexpr (Epi::kShifted) {  // the high planes' product begins at the last third of the steps
            for (; i < steps - (c1 - c0) && ok; ++i) step(i, std::false_type{});
            if (ok) step(i++, std::true_type{});
          }
          for (; i < steps && ok; ++i) step(i, std::false_type{});
        }
      }
    }
  } else {
    // ------------------------------------------------ drain + epilogue
    const int q = warp & 3, part = warp >> 2;  // tensor-memory lane quarter; which columns
    const uint32_t lane_base = (uint32_t)(q * 32) << 16;
    const Out out{smem + out_offset(BN, C) + warp * kOutBytes, lane};
    uint32_t chunk = 0;
    bool ok = true;
    for (int64_t u = pair; u < units.units && ok; u += num_pairs) {
      int64_t tm, tn;
      int split, kb0, nkb;
      units.locate(u, &tm, &tn, &split, &kb0, &nkb);
      float acc[C];
      if (!Epi::kDirect || nkb == 0) {
#pragma unroll
        for (int j = 0; j < C; ++j) acc[j] = 0.f;
      }
      for (int c0 = 0; c0 < nkb; c0 += a.chunk_kb, ++chunk) {
        const int b = chunk & 1;
        ok = mbar_wait(&acc_full[b], (chunk >> 1) & 1, 24, a.dev_status, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const uint32_t src = tmem_base + b * kTile + lane_base + part * C;
        if (Epi::kDirect && c0 == 0) {  // the first chunk lands in the sums themselves: one round trip for all of it
#pragma unroll
          for (int g = 0; g < C / 16; ++g) tmem_ld16_nowait(src + g * 16, acc + g * 16);
          tmem_wait_ld();
          tc_fence_before();
          mbar_arrive_warp_remote(&acc_empty[b], 0);
#pragma unroll
          for (int j = 0; j < C; ++j) asm volatile("" : "+f"(acc[j]));  // no use moves in front of the wait
          continue;
        }
#pragma unroll
        for (int g = 0; g < C / 16; ++g) {
          float v[16];
          tmem_ld16_nowait(src + g * 16, v);
          tmem_wait_ld();
          if (g == C / 16 - 1) {
            tc_fence_before();
            mbar_arrive_warp_remote(&acc_empty[b], 0);
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            asm volatile("" : "+f"(v[j]));
            acc[g * 16 + j] += v[j];
          }
        }
      }
      if (!ok) break;
      epi(acc, (int)(tm * kTile) + (int)rank * kHalf + q * 32 + lane, (int)(tn * BN) + part * C, split, &tmC, out);
    }
    if (lane == 0) tma_store_wait_all();
  }

  tc_fence_before();
  __syncwarp();
  cluster_sync_all();  // no CTA leaves (or frees tensor memory) while its peer may still use it
  if (warp == DRAIN + 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// ---- host -----------------------------------------------------------------------------------------------------------
// One operand: [planes][rows][cols] 16-bit values, rows `ld` apart (ld * 2 and the base multiples of 16).
struct Operand {
  const void* base;
  int64_t cols, rows, ld, planes, plane_stride;
};
int make_map(CUtensorMap* tm, const Operand& o, bool bf16, bool mn_major, int rows);
// An output [planes][rows][cols] of 2- or 4-byte elements, written in boxes of 32 rows x 128 bytes.
int make_out_map(CUtensorMap* tm, const Operand& o, int bytes);
// A matrix of `dtype` elements read in boxes without a swizzle (zeros out of bounds); base and row stride multiples of 16 bytes.
int make_plain_map(CUtensorMap* tm, const void* base, int dtype, int64_t cols, int64_t rows, int64_t ld, int box_cols, int box_rows);

// Columns of a tile: 128 where that finishes earlier, which is where tiles of 256 leave pairs without work.  A k-block takes a
// pair about 530 cycles with 256 columns and 400 with 128 (the loads, not the MMAs, bound it then); a unit's start, drain
// and epilogue about 6000 and 4000.
inline int tile_columns(int64_t M, int64_t N, int64_t K, int products, int sms) {
  const int64_t pairs = std::max(1, sms / 2), tiles_m = ceil_div(M, kTile), steps = ceil_div(K, kBK) * products;
  const int64_t wide = ceil_div(tiles_m * ceil_div(N, 256), pairs) * (530 * steps + 6000);
  const int64_t narrow = ceil_div(tiles_m * ceil_div(N, 128), pairs) * (400 * steps + 4000);
  return narrow < wide ? 128 : 256;
}

// kDirect: whether a tile's first chunk is loaded into the sums instead of added to zeros.  It saves 128 additions and seven round
// trips to tensor memory, and costs registers while the tile before is still being written: cycles of a launch without and
// with it: dZ of 2010 x 1000 x 25088 bf16 157k and 137k, but its logits 217k and 247k, and dW of 777 x 1001 x 30011 97k and 120k.
// Columns of a drain warp: 128 of a wide tile (eight warps), unless the epilogue asks for fewer (Epi::kColumns).
template <int BN, bool A_MN, bool B_MN, class Epi>
int launch(const Operand& A, const Operand& B, bool bf16, Args args, const CUtensorMap& tc, const Epi& epi, int device, int sms,
           cudaStream_t s) {
  constexpr int C = Epi::kColumns < BN / 2 ? Epi::kColumns : BN / 2, BYTES = smem_bytes(BN, C);
  CUtensorMap ta, tb;
  int st = make_map(&ta, A, bf16, A_MN, kHalf);
  if (st == TCB200_OK) st = make_map(&tb, B, bf16, B_MN, BN / 2);
  if (st != TCB200_OK) return st;
  args.idesc = make_idesc(bf16, A_MN, B_MN, BN);
  // the planes of each product, smallest products first: of one plane, of two (i + j <= 1) or of three (i + j <= 2)
  static const int pa[6] = {2, 1, 0, 1, 0, 0}, pb[6] = {0, 1, 2, 0, 1, 0};
  for (int i = 0; i < args.products; ++i) {
    args.pa[i] = pa[6 - args.products + i];
    args.pb[i] = pb[6 - args.products + i];
  }
  const int64_t tiles = ceil_div(args.M, kTile) * ceil_div(args.N, BN);
  if (tiles == 0) return TCB200_OK;
  // (a split result takes all pairs: how many units there are only the kernel knows)
  const unsigned pairs = (unsigned)std::min<int64_t>(args.splits ? INT64_MAX : tiles, std::max(1, sms / 2));
  static std::atomic<uint64_t> configured{0};
  TCB200_CUDA_TRY(ensure_dynamic_smem(pair_gemm_kernel<BN, C, A_MN, B_MN, Epi>, BYTES, device, configured));
  TCB200_CUDA_TRY(launch_pdl(pair_gemm_kernel<BN, C, A_MN, B_MN, Epi>, dim3(2 * pairs), dim3(block_threads(BN, C)), BYTES, s, ta, tb, tc, args, epi));
  return TCB200_OK;
}
template <bool A_MN, bool B_MN, class Epi>
int launch_columns(int bn, const Operand& A, const Operand& B, bool bf16, const Args& args, const CUtensorMap& tc, const Epi& epi,
                   int device, int sms, cudaStream_t s) {
  return bn == 128 ? launch<128, A_MN, B_MN, Epi>(A, B, bf16, args, tc, epi, device, sms, s)
                   : launch<256, A_MN, B_MN, Epi>(A, B, bf16, args, tc, epi, device, sms, s);
}

}  // namespace pg
}  // namespace tcb200

// The gated feed-forward layer on the tensor cores (tcgen05), bf16 and fp32.
//
// One persistent kernel serves the four products of the layer:
//   kForward  h = act(x Wg) * (x Wu)         a tile is 256 rows x 128 columns of both projections:
//                                            one MMA of N = 256 over [Wg tile | Wu tile]
//   kGrads    dG, dU from the same tiles and dh (the projections are formed again at every K, not kept: no memory
//             between the passes, at the price of their 4 K flops: 144 us at 16384 x 1024 -> 2816 bf16, where two
//             fp32 values an element, written and read back, would move 740 MB, an estimated 110 us)
//   kInput    dx = dG Wg^T + dU Wu^T         the two products in one accumulator
//   kWeights  dWg = x^T dG, dWu = x^T dU     both from one load of x, split over the rows
// A tile belongs to a cluster of two CTAs on neighbouring SMs (cta_group::2): each holds 128 of its 256 rows
// and one half of the columns of B (of the projections: one of them each), the leader issues one MMA of M =
// 256 over both, and each has its own rows of the accumulator. So a CTA loads 32 KB for 512 cycles of MMA;
// alone it would load 48 KB, and 148 SMs doing that draw 12 TB/s from L2 (measured: 178 us forward, 1.06
// PFLOP/s). Pairs walk the tiles (of half the width where that fills more SMs). Warp 0 loads 64-deep blocks
// by TMA into a ring of six stages, signalling the leader; the leader's warp 1 issues the MMAs into one of
// two 256-column accumulators in tensor memory, and eight epilogue warps drain the other: activation and
// product in registers, the result through 4 KB of shared memory per warp to TMA stores.
//
// fp32 operands are three bf16 planes each, x = x0 + x1 + x2 (24 bits), and a product is the six
// plane products whose size reaches 2^-24 of it: (2,0) (0,2) (1,1) (0,1) (1,0) (0,0), added in that
// order, smallest first, from one load of each plane. The accumulator truncates, so for fp32 it is handed to
// fp32 registers after every 64-deep block (24 MMAs); a sixth of the bf16 rate remains, which is
// four times what the CUDA cores' fp32 FMA does.
//
// A bf16 layer's accumulator is not handed over: each 16-deep step truncates it by 2^-22 of its value at most, so a
// sum over a depth d is off by d 2^-26 of its terms' absolute sum at most (2^-12 at 16384).
//
// Bound by the tensor cores: 16384 x 1024 -> 2816 bf16 takes 126 us forward (1.50 PFLOP/s, pipe 88 % active),
// 144 us for dG and dU (76 %), 130 us for dx (93 %; 256 tiles on 74 pairs, 3.5 waves in 4), 136 + 16 us for dW.
// With the descriptors formed by the issuing lane instead of kept in uniform registers the issue of an MMA
// cost about as much as its 128 cycles: 158, 172, 163 and 163 us.
#include <type_traits>

#include "gemm_sm100.cuh"
#include "glu.cuh"
#include "launch.cuh"

namespace bt {

int operator_error_word(int** word);

namespace glu {
namespace {

using namespace umma;

enum Mode { kForward, kGrads, kInput, kWeights };

constexpr int kAB = BM * BK * 2;
constexpr int kPairs = kNumSMs / 2;
// N columns of the MMA: 256, or 128 where that many would leave SMs without a tile.
template <int N>
struct Ring {
  static constexpr int kStages = 6;
  static constexpr int kStageBytes = kAB + N / 2 * BK * 2;  // of one CTA of the pair
  static constexpr int kSmem = kStages * kStageBytes + kEpiWarps * kEpiWarpBytes + 1024 + 256;
  static_assert(kSmem <= kMaxSmem, "stage ring");
};

struct Params {
  CUtensorMap map[12];
  CUtensorMap out[6], in;
  int M, N, K;        // of the product: rows and columns of the output, depth
  int act;
  int splits, depth;  // kWeights: 64-deep blocks of a split
  void *o0, *o1;      // outputs where their rows do not suit TMA stores (ldo), else null
  const void* dh;     // the same for dh
  int64_t ldo;
  int plane_rows;     // kWeights with splits: rows of one partial plane
  int* err;
};

// ---- the two CTAs of a pair ----
__device__ __forceinline__ uint32_t pair_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void pair_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A load into this CTA's shared memory that reports to the leader's barrier.
__device__ __forceinline__ void pair_load_2d(void* dst, const CUtensorMap* map, int c0, int c1, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(smem_u32(bar) & 0xFEFFFFFFu)
      : "memory");
}
__device__ __forceinline__ void pair_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrives at the barrier of both CTAs when the MMAs issued so far are done.
__device__ __forceinline__ void pair_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
__device__ __forceinline__ void leader_arrive(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .b32 a;\n\t"
      "mapa.shared::cluster.u32 a, %0, 0;\n\t"
      "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [a];\n\t}" ::"r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void pair_tmem_alloc(uint32_t* slot, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(ncols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void pair_tmem_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}

template <class T>
__device__ __forceinline__ T from_f32(float x) {
  if constexpr (sizeof(T) == 2) return __float2bfloat16_rn(x);
  return x;
}

__device__ __forceinline__ void tma_store(const CUtensorMap* map, const void* src, int c, int r, int lane) {
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    tma_store_2d(map, src, c, r);
    bulk_commit();
  }
}

__device__ __forceinline__ void staging_free(int lane) {
  if (lane == 0) bulk_wait_read_all();
  __syncwarp();
}

// A 32 x 32 tile whose rows do not suit TMA: staged as fp32, written with lanes along the columns.
template <class T>
__device__ __forceinline__ void store_plain(T* out, int64_t ld, int row0, int col0, int rows, int cols,
                                            uint8_t* buf, int lane, const float (&v)[32]) {
  stage_row_f32(buf, lane, v);
  __syncwarp();
  const int n = min(32, rows - row0);
  if (col0 + lane < cols)
    for (int r = 0; r < n; ++r)
      out[(row0 + r) * ld + col0 + lane] = from_f32<T>(
          *reinterpret_cast<const float*>(buf + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4));
  __syncwarp();
}

template <class T>
__device__ __forceinline__ void load_plain(const T* in, int64_t ld, int row0, int col0, int rows, int cols,
                                           uint8_t* buf, int lane) {
  for (int r = 0; r < 32; ++r) {
    float v = 0.f;
    if (row0 + r < rows && col0 + lane < cols) {
      const T x = in[(row0 + r) * ld + col0 + lane];
      if constexpr (sizeof(T) == 2) v = __bfloat162float(x); else v = x;
    }
    *reinterpret_cast<float*>(buf + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4) = v;
  }
  __syncwarp();
}

__device__ __forceinline__ void row_f32(const uint8_t* buf, int lane, float (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float4 p = load_row_f32(buf, lane, j);
    v[4 * j] = p.x, v[4 * j + 1] = p.y, v[4 * j + 2] = p.z, v[4 * j + 3] = p.w;
  }
}
__device__ __forceinline__ void row_bf16(const uint8_t* buf, int lane, float (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint4 w = *reinterpret_cast<const uint4*>(buf + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4));
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = *reinterpret_cast<const __nv_bfloat162*>(&ws[i]);
      v[8 * j + 2 * i] = __low2float(h);
      v[8 * j + 2 * i + 1] = __high2float(h);
    }
  }
}

// An output tile in T: through a TMA store (map) or plainly (p.o).
template <class T>
__device__ __forceinline__ void put(const CUtensorMap* map, void* plain, const Params& p, int row0, int col0,
                                    uint8_t* buf, int lane, const float (&v)[32]) {
  staging_free(lane);
  if (plain) {
    store_plain(static_cast<T*>(plain), p.ldo, row0, col0, p.M, p.N, buf, lane, v);
    return;
  }
  if constexpr (sizeof(T) == 2) stage_row_bf16(buf, nullptr, lane, v);
  else stage_row_f32(buf, lane, v);
  tma_store(map, buf, col0, row0, lane);
}

// What the first plane of v is rounded from: a finite v beyond bf16's largest value would round to infinity. (An
// infinite one leaves an infinite remainder and stays what it is.)
__device__ __forceinline__ float within_bf16(float v) {
  constexpr float kMost = 0x1.fep127f;
  return fminf(fmaxf(v, -kMost), kMost);
}

// v as three bf16 planes, v = v0 + v1 + v2 to 24 bits.
__device__ __forceinline__ void put_planes(const CUtensorMap* maps, int row0, int col0, uint8_t* buf, int lane,
                                           float (&v)[32]) {
  staging_free(lane);
  {
    float first[32];
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      first[j] = within_bf16(v[j]);
      v[j] -= __bfloat162float(__float2bfloat16_rn(first[j]));
    }
    stage_row_bf16(buf, nullptr, lane, first);
  }
  stage_row_bf16(buf + 2048, nullptr, lane, v);
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    tma_store_2d(&maps[0], buf, col0, row0);
    tma_store_2d(&maps[1], buf + 2048, col0, row0);
    bulk_commit();
  }
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] -= __bfloat162float(__float2bfloat16_rn(v[j]));
  staging_free(lane);
  stage_row_bf16(buf, nullptr, lane, v);
  tma_store(&maps[2], buf, col0, row0, lane);
}

// T: the layer's type. An fp32 layer's operands are planes and its accumulator is handed over after
// every 64-deep block.
template <class T, Mode kMode, int kN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) glu_kernel(const __grid_constant__ Params p) {
  constexpr int kStages = Ring<kN>::kStages, kStageBytes = Ring<kN>::kStageBytes;
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr bool kDual = kMode != kInput;
  constexpr bool A_MN = kMode == kWeights, B_MN = kMode != kInput;
  constexpr int kP = kF32 ? 3 : 1, kSums = kDual ? 1 : 2;  // planes of an operand, products in a sum
  constexpr int kTileN = kDual ? kN / 2 : kN;
  constexpr int kGroups = kN / 64;  // groups of 32 accumulator columns of an epilogue warp
  // 64-deep blocks between two hand-overs of the accumulator: bf16 results keep 2^-8, which the truncation of a
  // whole product reaches at no depth below 2^18
  constexpr int kHand = kF32 ? 1 : 1 << 30;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi_smem = smem + kStages * kStageBytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(epi_smem + kEpiWarps * kEpiWarpBytes);
  uint64_t* empty = full + kStages;
  uint64_t* acc_full = empty + kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* epi_in = acc_empty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(epi_in + kEpiWarps);
  __shared__ int s_fail;
  const int warp = __shfl_sync(~0u, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  pdl_trigger();
  if (threadIdx.x == 0) {
    s_fail = 0;
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], 2 * kEpiWarps);  // (the leader's) both CTAs' epilogue warps
    }
    for (int w = 0; w < kEpiWarps; ++w) mbar_init(&epi_in[w], 1);
    fence_mbar_init();
  }
  if (warp == 1) pair_tmem_alloc(tmem_slot, 2 * kN);
  fence_before_sync();
  __syncwarp();
  pair_sync();
  fence_after_sync();
  const int rank = (int)pair_rank();
  const uint32_t tmem = *tmem_slot;
  auto failed = [&]() { return *(volatile int*)&s_fail != 0; };
  pdl_wait();
  const int ntn = ceil_div(p.N, kTileN), ntm = ceil_div(p.M, 2 * BM);
  const int nk = ceil_div(p.K, BK);
  const int tiles = ntm * ntn * p.splits;
  // the splits of one tile lie far apart, the column tiles of one row block together
  auto where = [&](int t, int& m0, int& n0, int& k0, int& k1, int& split) {
    split = t / (ntm * ntn);
    const int u = t % (ntm * ntn);
    m0 = u / ntn * (2 * BM) + rank * BM;
    n0 = u % ntn * kTileN;
    k0 = split * p.depth;
    k1 = min(nk, k0 + p.depth);
  };

  if (warp == 0) {
    if (lane == 0) {
      int g = 0;
      for (int t = blockIdx.x >> 1; t < tiles && !failed(); t += gridDim.x >> 1) {
        int m0, n0, k0, k1, split;
        where(t, m0, n0, k0, k1, split);
        for (int kb = k0; kb < k1 && !failed(); ++kb) {
          const int k = kb * BK;
          for (int e = 0; e < kSums * kP; ++e, ++g) {
            const int s = g % kStages;
            if (g >= kStages && !mbar_wait_bounded(&empty[s], ((g / kStages) - 1) & 1)) {
              atomicExch(&s_fail, kErrTimeoutEmpty);
              break;
            }
            uint8_t* sa = smem + s * kStageBytes;
            uint8_t* sb = sa + kAB;
            // both CTAs' bytes
            if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * kStageBytes);
            const int q = e / kP, z = kP - 1 - e % kP;  // the smallest plane first
            const CUtensorMap* ma = &p.map[kDual ? z : q * kP + z];
            const CUtensorMap* mb = &p.map[kDual ? (1 + rank) * kP + z : (2 + q) * kP + z];
            if (A_MN) {
              pair_load_2d(sa, ma, m0, k, &full[s]);
              pair_load_2d(sa + 8192, ma, m0 + 64, k, &full[s]);
            } else {
              pair_load_2d(sa, ma, k, m0, &full[s]);
            }
            if (kDual) {
#pragma unroll
              for (int j = 0; j < kN / 128; ++j) pair_load_2d(sb + j * 8192, mb, n0 + 64 * j, k, &full[s]);
            } else {
              pair_load_2d(sb, mb, k, n0 + rank * (kN / 2), &full[s]);
            }
          }
        }
      }
      // every stage is consumed (and so loaded) before the pair may leave
      for (int i = max(0, g - kStages); i < g; ++i)
        if (!mbar_wait_bounded(&empty[i % kStages], (i / kStages) & 1)) atomicExch(&s_fail, kErrTimeoutEmpty);
    }
  } else if (warp == 1) {
    if (rank == 0) {
      // M = 256 over the pair. The whole warp walks along and one lane issues, so that descriptors stay in
      // uniform registers; a stage's and a step's are the first ones plus a constant (16-byte units).
      constexpr uint32_t idesc = instr_desc<kN, A_MN, B_MN>() + ((uint32_t)(BM >> 4) << 24);
      const uint64_t desc_a = operand_desc<A_MN>(smem_u32(smem), 0), desc_b = operand_desc<B_MN>(smem_u32(smem) + kAB, 0);
      constexpr uint64_t kStepA = (A_MN ? 2048 : 32) >> 4, kStepB = (B_MN ? 2048 : 32) >> 4;
      const bool leader = elect_one();
      int s = 0, c = 0;  // the ring's stage and (its parity) round, the accumulator
      uint32_t round = 0;
      bool ok = true;
      for (int t = blockIdx.x >> 1; t < tiles && ok && !failed(); t += gridDim.x >> 1) {
        int m0, n0, k0, k1, split;
        where(t, m0, n0, k0, k1, split);
        for (int kb = k0; kb < k1 && ok; ++kb) {
          bool keep = (kb - k0) % kHand != 0;
          if (!keep && c >= 2) {
            if (!mbar_wait_bounded(&acc_empty[c & 1], ((c >> 1) - 1) & 1)) {
              if (lane == 0) atomicExch(&s_fail, kErrTimeoutAcc);
              ok = false;
              break;
            }
            fence_after_sync();
          }
          const uint32_t acc = tmem + (uint32_t)((c & 1) * kN);
          for (int q = 0; q < kSums && ok; ++q) {
            int at[kP];  // the planes' stages, by plane
#pragma unroll
            for (int e = 0; e < kP; ++e) {
              if (!mbar_wait_bounded(&full[s], round)) {
                if (lane == 0) atomicExch(&s_fail, kErrTimeoutFull);
                ok = false;
              }
              at[kP - 1 - e] = s;
              if (++s == kStages) s = 0, round ^= 1;
            }
            if (!ok) break;
            fence_after_sync();
            if (leader) {
              auto product = [&](int x, int y) {
                const uint64_t a = desc_a + (uint64_t)(at[x] * (kStageBytes >> 4));
                const uint64_t b = desc_b + (uint64_t)(at[y] * (kStageBytes >> 4));
#pragma unroll
                for (int k = 0; k < BK / 16; ++k) {
                  pair_mma(acc, a + k * kStepA, b + k * kStepB, idesc, keep ? 1u : 0u);
                  keep = true;
                }
              };
              if constexpr (kP == 3) {
                product(2, 0);
                product(0, 2);
                pair_commit(&empty[at[2]]);
                product(1, 1);
                product(0, 1);
                product(1, 0);
                pair_commit(&empty[at[1]]);
              }
              product(0, 0);
              pair_commit(&empty[at[0]]);
            }
            keep = true;
            __syncwarp();
          }
          if (ok && ((kb - k0) % kHand == kHand - 1 || kb == k1 - 1)) {
            if (leader) pair_commit(&acc_full[c & 1]);
            __syncwarp();
            ++c;
          }
        }
      }
    }
  } else {
    // Epilogue: rows 32 q .. of the tile, thread = row; half of the columns (of each projection).
    const int q = warp & 3, half = (warp - 2) >> 2;
    uint8_t* buf = epi_smem + (warp - 2) * kEpiWarpBytes;
    uint64_t* ibar = &epi_in[warp - 2];
    const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16);
    // TMEM column of this warp's group j: half of the groups of each projection, or all of the one product
    constexpr int kEach = kDual ? kGroups / 2 : kGroups;
    auto column = [&](int j) { return j / kEach * (kN / 2) + half * (kEach * 32) + j % kEach * 32; };
    float run[kF32 ? kGroups : 1][32];
    int c = 0, loads = 0;
    bool ok = true;
    for (int t = blockIdx.x >> 1; t < tiles && ok && !failed(); t += gridDim.x >> 1) {
      int m0, n0, k0, k1, split;
      where(t, m0, n0, k0, k1, split);
      const int row0 = m0 + q * 32;
      if constexpr (kF32) {
#pragma unroll
        for (int j = 0; j < kGroups; ++j)
#pragma unroll
          for (int i = 0; i < 32; ++i) run[j][i] = 0.f;
        for (int kb = k0; kb < k1; ++kb, ++c) {
          ok = mbar_wait_bounded(&acc_full[c & 1], (c >> 1) & 1);
          if (!ok) break;
          fence_after_sync();
#pragma unroll
          for (int j = 0; j < kGroups; ++j) {
            float v[32];
            tmem_ld32(lanes + (uint32_t)((c & 1) * kN + column(j)), v);
#pragma unroll
            for (int i = 0; i < 32; ++i) run[j][i] += v[i];
          }
          fence_before_sync();
          __syncwarp();
          if (lane == 0) leader_arrive(&acc_empty[c & 1]);
        }
      } else {
        ok = mbar_wait_bounded(&acc_full[c & 1], (c >> 1) & 1);
        fence_after_sync();
      }
      if (!ok) {
        if (lane == 0) atomicExch(&s_fail, kErrTimeoutAcc);
        break;
      }
      const uint32_t acc = lanes + (uint32_t)((c & 1) * kN);
      auto group = [&](int j, float (&v)[32]) {
        if constexpr (kF32) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = run[j][i];
        } else {
          tmem_ld32(acc + (uint32_t)column(j), v);
        }
      };
      auto release = [&]() {
        if constexpr (!kF32) {
          fence_before_sync();
          __syncwarp();
          if (lane == 0) leader_arrive(&acc_empty[c & 1]);
          ++c;
        }
      };
      if constexpr (kMode == kForward || kMode == kGrads) {
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
          const int col0 = n0 + half * (kEach * 32) + 32 * j;
          const bool in = col0 < p.N && row0 < p.M;
          if (kMode == kGrads && in) {
            staging_free(lane);
            if (p.dh) {
              load_plain(static_cast<const T*>(p.dh), (int64_t)p.N, row0, col0, p.M, p.N, buf, lane);
            } else if (lane == 0) {
              mbar_arrive_expect_tx(ibar, 32 * 32 * sizeof(T));
              tma_load_2d(buf, &p.in, col0, row0, ibar);
            }
          }
          float g[32], u[32];
          group(j, g);
          group(kEach + j, u);
          if (j == kEach - 1) release();
          if constexpr (kMode == kForward) {
            if (!in) continue;
            with_act(p.act, [&](auto tag) {
#pragma unroll
              for (int i = 0; i < 32; ++i) g[i] = gate_act<decltype(tag)::value>(g[i]) * u[i];
            });
            put<T>(&p.out[0], p.o0, p, row0, col0, buf, lane, g);
          } else {
            if (!in) continue;
            float d[32];
            if (p.dh) {
              row_f32(buf, lane, d);
            } else {
              if (!mbar_wait_bounded(ibar, loads & 1)) {
                if (lane == 0) atomicExch(&s_fail, kErrTimeoutEpiIn);
                ok = false;
              }
              ++loads;
              if constexpr (kF32) row_f32(buf, lane, d);
              else row_bf16(buf, lane, d);
            }
            __syncwarp();
            with_act(p.act, [&](auto tag) {
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                float dg, du;
                gate_grads<decltype(tag)::value>(g[i], u[i], d[i], dg, du);
                g[i] = dg;
                u[i] = du;
              }
            });
            if constexpr (kF32) {
              put_planes(&p.out[0], row0, col0, buf, lane, g);
              put_planes(&p.out[3], row0, col0, buf, lane, u);
            } else {
              stage_row_bf16(buf, nullptr, lane, g);
              stage_row_bf16(buf + 2048, nullptr, lane, u);
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) {
                tma_store_2d(&p.out[0], buf, col0, row0);
                tma_store_2d(&p.out[1], buf + 2048, col0, row0);
                bulk_commit();
              }
            }
          }
        }
      } else if constexpr (kMode == kInput) {
#pragma unroll
        for (int j = 0; j < kGroups; ++j) {
          const int col0 = n0 + half * (kN / 2) + 32 * j;
          float v[32];
          group(j, v);
          if (j == kGroups - 1) release();
          if (col0 < p.N && row0 < p.M) put<T>(&p.out[0], p.o0, p, row0, col0, buf, lane, v);
        }
      } else {
#pragma unroll
        for (int j = 0; j < kGroups; ++j) {
          const int which = j / kEach, col0 = n0 + half * (kEach * 32) + 32 * (j % kEach);
          float v[32];
          group(j, v);
          if (j == kGroups - 1) release();
          if (col0 >= p.N || row0 >= p.M) continue;
          if (p.splits > 1) {  // one partial plane for each split and weight
            put<float>(&p.out[0], nullptr, p, (2 * split + which) * p.plane_rows + row0, col0, buf, lane, v);
          } else {
            put<T>(&p.out[which], which ? p.o1 : p.o0, p, row0, col0, buf, lane, v);
          }
        }
      }
    }
    if (lane == 0) bulk_wait_all();
    __syncwarp();
  }
  fence_before_sync();
  __syncwarp();
  pair_sync();
  if (warp == 1) {
    fence_after_sync();
    pair_tmem_dealloc(tmem, 2 * kN);
  }
  if (threadIdx.x == 0 && s_fail) atomicExch(p.err, s_fail);
}

// The operands that are not read in place, as the kernel reads them: rows of ld (a multiple of 8) bf16,
// kPlanes planes of them. blockIdx.y: which one; thread: eight columns of a row.
struct Copies {
  struct {
    const void* src;
    __nv_bfloat16* dst;
    int64_t rows;
    int cols, ld;
  } of[3];
};
template <class T, int kPlanes>
__global__ void __launch_bounds__(256) planes_kernel(const __grid_constant__ Copies copies) {
  const auto& o = copies.of[blockIdx.y];
  const int per = o.ld / 8;
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= o.rows * per) return;
  const int64_t r = e / per;
  const int c = (int)(e % per) * 8;
  const T* s = static_cast<const T*>(o.src) + r * o.cols + c;
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = 0.f;
    if (c + i < o.cols) {
      if constexpr (sizeof(T) == 2) v[i] = __bfloat162float(s[i]); else v[i] = s[i];
    }
  }
#pragma unroll
  for (int k = 0; k < kPlanes; ++k) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = kPlanes > 1 && k == 0 ? pack_bf16(within_bf16(v[2 * i]), within_bf16(v[2 * i + 1]))
                                   : pack_bf16(v[2 * i], v[2 * i + 1]);
      const __nv_bfloat162 h = *reinterpret_cast<const __nv_bfloat162*>(&w[i]);
      v[2 * i] -= __low2float(h);
      v[2 * i + 1] -= __high2float(h);
    }
    *reinterpret_cast<uint4*>(o.dst + (k * o.rows + r) * o.ld + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// dWg and dWu: the splits' partial planes [splits][2][plane_rows][ld] added in their order.
template <class T>
__global__ void __launch_bounds__(256) join_kernel(const float* part, int splits, int rows, int cols, int plane_rows,
                                                   int ld, T* dwg, T* dwu) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int per = ld / 4;
  if (e >= (int64_t)rows * per) return;
  const int r = (int)(e / per), c = (int)(e % per) * 4;
  const float* s = part + ((int64_t)blockIdx.y * plane_rows + r) * ld + c;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = 0; k < splits; ++k) {
    const float4 b = *reinterpret_cast<const float4*>(s + (int64_t)2 * k * plane_rows * ld);
    a.x += b.x, a.y += b.y, a.z += b.z, a.w += b.w;
  }
  T* o = (blockIdx.y ? dwu : dwg) + (int64_t)r * cols + c;
  const float v[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (c + i < cols) o[i] = from_f32<T>(v[i]);
}

int round_up(int x, int m) { return (x + m - 1) / m * m; }
int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

// Splits of the rows for the weight gradients: whole waves of tiles against the partial planes' way
// through memory (written and read once at about 5 TB/s); a 64-deep block of a tile takes 0.3 us
// (fp32: six times that).
int choose_splits(int M, int K, int N, int planes) {
  const int tiles = ceil_div(K, 2 * BM) * ceil_div(N, 128), nk = ceil_div(M, BK);
  const double block = planes == 3 ? 1.8 : 0.3;
  int best = 1;
  double least = 1e30;
  for (int s = 1; s <= 32 && s <= nk; ++s) {
    const double us = ceil_div(tiles * s, kPairs) * ceil_div(nk, s) * block +
                      (s > 1 ? 2.0 + s * 2.0 * K * N * 8 / 5e6 : 0.0);
    if (us < least) least = us, best = s;
  }
  return ceil_div(nk, ceil_div(nk, best));
}

// The layer's operands in the workspace: planes of x and of the weights (bf16 layers whose rows suit
// TMA are read where they are), of dG and dU, and the weight gradients' partial planes.
struct Plan {
  int planes, ldk, ldn, splits, plane_rows, ldp;
  int64_t x, wg, wu, dg, du, part, bytes;  // offsets; x, wg, wu: -1 read in place
};

Plan plan_of(const Layer& l, bool f32, bool backward) {
  Plan w{};
  w.planes = f32 ? 3 : 1;
  w.ldk = round_up(l.K, 8);
  w.ldn = round_up(l.N, 8);
  int64_t at = 0;
  auto take = [&](int64_t elems, int64_t size) {
    const int64_t o = at;
    at += align256(elems * size);
    return o;
  };
  const bool copy_x = f32 || l.K % 8, copy_w = f32 || l.N % 8;
  w.x = copy_x ? take((int64_t)w.planes * l.M * w.ldk, 2) : -1;
  w.wg = copy_w ? take((int64_t)w.planes * l.K * w.ldn, 2) : -1;
  w.wu = copy_w ? take((int64_t)w.planes * l.K * w.ldn, 2) : -1;
  w.splits = 1;
  if (backward) {
    w.dg = take((int64_t)w.planes * l.M * w.ldn, 2);
    w.du = take((int64_t)w.planes * l.M * w.ldn, 2);
    w.splits = choose_splits(l.M, l.K, l.N, w.planes);
    w.plane_rows = round_up(l.K, 2 * BM);
    w.ldp = round_up(l.N, 4);
    if (w.splits > 1) w.part = take((int64_t)2 * w.splits * w.plane_rows * w.ldp, 4);
  }
  w.bytes = at;
  return w;
}

template <class T>
struct Run {
  static constexpr bool kF32 = sizeof(T) == 4;
  static constexpr int kP = kF32 ? 3 : 1;
  const Layer& l;
  Plan w;
  char* ws;
  cudaStream_t s;
  const __nv_bfloat16 *x, *wg, *wu;
  int ldx, ldw;

  int operands() {
    ldx = w.x < 0 ? l.K : w.ldk;
    ldw = w.wg < 0 ? l.N : w.ldn;
    Copies c{};
    int n = 0;
    int64_t most = 0;
    auto operand = [&](const void* src, int64_t rows, int cols, int ld, int64_t at) -> const __nv_bfloat16* {
      if (at < 0) return static_cast<const __nv_bfloat16*>(src);
      __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(ws + at);
      c.of[n++] = {src, dst, rows, cols, ld};
      most = max(most, rows * (ld / 8));
      return dst;
    };
    x = operand(l.x, l.M, l.K, w.ldk, w.x);
    wg = operand(l.wg, l.K, l.N, w.ldn, w.wg);
    wu = operand(l.wu, l.K, l.N, w.ldn, w.wu);
    if (n > 0) {
      planes_kernel<T, kP><<<dim3((unsigned)ceil_div64(most, 256), n), 256, 0, s>>>(c);
      BT_LAUNCH_CHECK("gated layer operand planes");
    }
    return BT_OK;
  }
  // Maps of an operand's planes, `box` rows of 64 columns at a time.
  int maps(CUtensorMap* m, const __nv_bfloat16* base, int64_t rows, int cols, int ld, int box) {
    for (int k = 0; k < kP; ++k)
      BT_TRY(encode_map(&m[k], base + k * rows * ld, cols, rows, (uint64_t)ld * 2, 64, box));
    return BT_OK;
  }
  // Whether tiles of half the width finish sooner: they take six tenths of the time each.
  static bool narrow(int M, int N, int splits, bool dual) {
    const int rows = ceil_div(M, 2 * BM) * splits, w = dual ? 128 : 256;
    return 0.6 * ceil_div(rows * ceil_div(N, w / 2), kPairs) < ceil_div(rows * ceil_div(N, w), kPairs);
  }
  template <Mode kMode, int kN>
  int launch_n(Params& p) {
    auto kernel = glu_kernel<T, kMode, kN>;
    static std::atomic<uint64_t> allowed{0};
    BT_TRY(allow_smem(kernel, Ring<kN>::kSmem, allowed));
    BT_TRY(operator_error_word(&p.err));
    const int tiles = ceil_div(p.M, 2 * BM) * ceil_div(p.N, kMode == kInput ? kN : kN / 2) * p.splits;
    BT_CUDA(launch_pdl(kernel, dim3(2 * min(tiles, kPairs)), dim3(kThreads), Ring<kN>::kSmem, s, p));
    return BT_OK;
  }
  template <Mode kMode>
  int launch(Params& p) {
    return narrow(p.M, p.N, p.splits, kMode != kInput) ? launch_n<kMode, 128>(p) : launch_n<kMode, 256>(p);
  }
  // A row-major T output (or dh) of `cols` columns: by TMA where its rows suit it.
  static bool suits(int cols) { return cols % (16 / (int)sizeof(T)) == 0; }
  int tile_map(CUtensorMap* m, const void* base, int64_t rows, int cols) {
    return encode_tile_map(m, base, kF32, cols, rows, (uint64_t)cols * sizeof(T), kF32 ? 128 : 64);
  }

  // G and U of every tile: h, or dG and dU into the workspace.
  template <Mode kMode>
  int project(void* h) {
    Params p{};
    p.M = l.M, p.N = l.N, p.K = l.K, p.act = l.act, p.splits = 1, p.depth = ceil_div(l.K, BK);
    BT_TRY(maps(&p.map[0], x, l.M, l.K, ldx, BM));
    BT_TRY(maps(&p.map[kP], wg, l.K, l.N, ldw, 64));
    BT_TRY(maps(&p.map[2 * kP], wu, l.K, l.N, ldw, 64));
    p.ldo = l.N;
    if constexpr (kMode == kForward) {
      if (suits(l.N)) BT_TRY(tile_map(&p.out[0], h, l.M, l.N));
      else p.o0 = h;
    } else {
      for (int k = 0; k < 2 * kP; ++k) {
        const char* base = ws + (k < kP ? w.dg : w.du) + (int64_t)(k % kP) * l.M * w.ldn * 2;
        BT_TRY(encode_tile_map(&p.out[k], base, false, l.N, l.M, (uint64_t)w.ldn * 2, 64));
      }
      if (suits(l.N)) BT_TRY(tile_map(&p.in, l.dh, l.M, l.N));
      else p.dh = l.dh;
    }
    return launch<kMode>(p);
  }
  int input(void* dx) {
    Params p{};
    p.M = l.M, p.N = l.K, p.K = l.N, p.splits = 1, p.depth = ceil_div(l.N, BK);
    BT_TRY(maps(&p.map[0], reinterpret_cast<const __nv_bfloat16*>(ws + w.dg), l.M, l.N, w.ldn, BM));
    BT_TRY(maps(&p.map[kP], reinterpret_cast<const __nv_bfloat16*>(ws + w.du), l.M, l.N, w.ldn, BM));
    const int box = narrow(p.M, p.N, 1, false) ? 64 : 128;  // one CTA's half
    BT_TRY(maps(&p.map[2 * kP], wg, l.K, l.N, ldw, box));
    BT_TRY(maps(&p.map[3 * kP], wu, l.K, l.N, ldw, box));
    p.ldo = l.K;
    if (suits(l.K)) BT_TRY(tile_map(&p.out[0], dx, l.M, l.K));
    else p.o0 = dx;
    return launch<kInput>(p);
  }
  int weights(void* dwg, void* dwu) {
    Params p{};
    p.M = l.K, p.N = l.N, p.K = l.M;
    p.splits = w.splits;
    p.depth = ceil_div(ceil_div(l.M, BK), w.splits);
    BT_TRY(maps(&p.map[0], x, l.M, l.K, ldx, 64));
    BT_TRY(maps(&p.map[kP], reinterpret_cast<const __nv_bfloat16*>(ws + w.dg), l.M, l.N, w.ldn, 64));
    BT_TRY(maps(&p.map[2 * kP], reinterpret_cast<const __nv_bfloat16*>(ws + w.du), l.M, l.N, w.ldn, 64));
    p.ldo = l.N;
    p.plane_rows = w.plane_rows;
    float* part = reinterpret_cast<float*>(ws + w.part);
    if (w.splits > 1) {
      BT_TRY(encode_tile_map(&p.out[0], part, true, l.N, (uint64_t)2 * w.splits * w.plane_rows, (uint64_t)w.ldp * 4, 128));
    } else if (suits(l.N)) {
      BT_TRY(tile_map(&p.out[0], dwg, l.K, l.N));
      BT_TRY(tile_map(&p.out[1], dwu, l.K, l.N));
    } else {
      p.o0 = dwg;
      p.o1 = dwu;
    }
    BT_TRY(launch<kWeights>(p));
    if (w.splits > 1) {
      const dim3 grid((unsigned)ceil_div64((int64_t)l.K * (w.ldp / 4), 256), 2);
      join_kernel<T><<<grid, 256, 0, s>>>(part, w.splits, l.K, l.N, w.plane_rows, w.ldp, static_cast<T*>(dwg),
                                          static_cast<T*>(dwu));
      BT_LAUNCH_CHECK("gated layer weight gradients");
    }
    return BT_OK;
  }
};

}  // namespace

int64_t workspace_of(const Layer& l, bool f32, bool backward) { return plan_of(l, f32, backward).bytes; }

template <class T>
static int forward_t(const Layer& l, void* h, char* ws, cudaStream_t s) {
  Run<T> r{l, plan_of(l, sizeof(T) == 4, false), ws, s};
  BT_TRY(r.operands());
  return r.template project<kForward>(h);
}

template <class T>
static int backward_t(const Layer& l, void* dx, void* dwg, void* dwu, char* ws, cudaStream_t s) {
  Run<T> r{l, plan_of(l, sizeof(T) == 4, true), ws, s};
  BT_TRY(r.operands());
  BT_TRY(r.template project<kGrads>(nullptr));
  if (dx) BT_TRY(r.input(dx));
  if (dwg) BT_TRY(r.weights(dwg, dwu));
  return BT_OK;
}

int forward(const Layer& l, bool f32, void* h, char* ws, cudaStream_t s) {
  return f32 ? forward_t<float>(l, h, ws, s) : forward_t<__nv_bfloat16>(l, h, ws, s);
}

int backward(const Layer& l, bool f32, void* dx, void* dwg, void* dwu, char* ws, cudaStream_t s) {
  return f32 ? backward_t<float>(l, dx, dwg, dwu, ws, s) : backward_t<__nv_bfloat16>(l, dx, dwg, dwu, ws, s);
}

}  // namespace glu
}  // namespace bt

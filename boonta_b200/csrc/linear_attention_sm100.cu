// Linear attention with a decay per head on the tensor cores (tcgen05), bf16 inputs (the operation:
// linear_attention.cuh).
//
// A block takes one (batch row, head) and 64 columns of c and of the state after the other, and walks its
// positions 128 at a time. In a chunk, with p the position of a row, w_j = in_scale e^{(n - 1 - p_j) g}, and everything
// accumulated in fp32:
//   P0 = a b^T                                     [128 x 128]  tensor memory
//   O  = a S                                       [128 x 64]   S: bf16 copy of the state in shared memory
//   L  = b^T (w c)                                 [Da x 64]    w c as three bf16 planes (24 bits)
//   S  = e^{(n - 1 + e0) g} S + L
// and for a head with |g| <= 0.23 (its weights across a chunk stay above e^-30), where S is copied with
// its decay over the chunk to come:
//   P  = P0, 0 above the diagonal and across a cut, to bf16 in place of P0
//   O += P (w c), the first two planes;   out = out_scale e^{(p - n + 1) g} O
// so that no weight meets the 128 x 128 scores. For a head that decays faster those factors would leave
// the range of fp32, and the weights go where they are at most 1:
//   P  = in_scale P0 e^{(p_i - p_j) g}, 0 above the diagonal and across a cut
//   O  = e^{(p + e0) g} O + P c;   out = out_scale O
// The state itself stays in fp32 registers for the whole walk. Only two factors are rounded to bf16, P
// and the copy of S that O reads, and both go only into outputs that are rounded to bf16 themselves
// (each adds 2^-9 root mean square at most); the state, which is handed on in fp32, comes from exact
// products: b is bf16 already, and w c keeps its 24 bits (down to 2^-133; with weights above e^-30 the 16 bits
// that outputs take are whole for values above 2^-73).
//
// Backwards the tiles stay in the order of time and the positions run against it: p = 127 - r.
//
// Warp 8 loads the tiles and issues the MMAs; warps 0 to 7 do everything in registers, two threads
// to a row. A chunk is a chain of dependent steps, so the chain is cut where it can be (w c is formed
// while a b^T runs, L runs while P is formed, the outputs are written while the next tiles come), and two
// blocks share an SM: 256 of the 512 columns of tensor memory each, and at most 113 KB of shared memory
// (planes of w c in place of a, which P0 and O are done with). Nothing that can be formed again is kept in
// registers across a chunk: what spills goes through an L1 that shared memory leaves next to nothing of.
//
// Measured: 16 x 2000 x 8 heads x 64/128 forward 77 us (2.7 TB/s of its 205 MB, tensor pipe 39 %); 512 x 128
// x 4 x 64 with resets forward 65 us, its three gradients 170 us (a forward pass without resets: 53); 2 x 8191 x 16 x
// 128 forward 97 us after 62 us for the splits' sums and their join, gradients 335 us. Bound by the chain: 0.4
// instructions a cycle and scheduler, a quarter of a warp's time in waits for tensor memory, barriers and tiles.
//
// A cut hides what lies before it, whatever it holds: masked scores and states are dropped, not multiplied. Values
// of c are operands of a whole chunk's products, so in a chunk with a cut those that are not finite are taken out of
// the tile first (a look at every value and one barrier a chunk: 512 x 128 x 4 x 64 training pass 217 -> 223 us).
#include <type_traits>

#include "f32x2.cuh"
#include "gemm_sm100.cuh"
#include "launch.cuh"
#include "linear_attention.cuh"

namespace bt {

int operator_error_word(int** word);

namespace la {
namespace {

using umma::fence_after_sync;
using umma::fence_before_sync;
using umma::mma_bf16;
using umma::mma_commit;
using umma::pack_bf16;
using umma::smem_desc;
using umma::tmem_ld32;

constexpr int kC = 128, kDS = 64;
constexpr int kWorkers = 256, kThreads = kWorkers + 32;
constexpr int kBlock = kC * 128;  // 128 rows of 64 bf16, 128-byte swizzle
constexpr uint32_t kCols = 256;   // tensor memory: P0 (P in the first quarter of each half), L, O
constexpr uint32_t kLCol = 128, kOCol = 192;
constexpr int kErrAlignment = 15;
constexpr float kWeakDecay = -0.23f;

template <int DA>
struct Cfg {
  static constexpr int kNA = DA / 64;  // 64-wide blocks of a and b
  static constexpr int kA = 0, kB = kNA * kBlock, kCc = 2 * kNA * kBlock, kS = kCc + kBlock;
  static constexpr int kP2 = kS + DA * 128;  // planes that do not fit into a's buffer
  static constexpr int kPlanes = kP2 + (3 - kNA) * kBlock;
  static constexpr int kBar = kPlanes;
  static constexpr int kOp = kBar + 80 + 4 * (kC + 4) + 16 + 32;
  static constexpr int kBytes = kOp + (sizeof(Op) + 15) / 16 * 16;
  __device__ static int plane(int k) { return k < kNA ? kA + k * kBlock : kP2 + (k - kNA) * kBlock; }
};
static_assert(2 * (Cfg<128>::kBytes + 1024) <= 228 * 1024, "two blocks on an SM");

struct Maps {
  CUtensorMap a[3], b[3], c[3], out[3];
};

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int t, int h, int b,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(t), "r"(h), "r"(b), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void tma_prefetch_4d(const CUtensorMap* map, int x, int t, int h, int b) {
  asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %3, %4}];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(t), "r"(h), "r"(b)
               : "memory");
}
__device__ __forceinline__ void tma_store_4d(const CUtensorMap* map, const void* src, int x, int t, int h, int b) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(t), "r"(h), "r"(b), "r"(smem_u32(src))
               : "memory");
}

// D (tensor memory) += A (tensor memory, two K elements a column) B (shared memory).
__device__ __forceinline__ void mma_bf16_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld16(uint32_t addr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}

// The bits lo .. hi of a word (positions outside 0 .. 31 allowed).
__device__ __forceinline__ unsigned bits(int lo, int hi) {
  const unsigned from = lo <= 0 ? ~0u : lo > 31 ? 0u : ~0u << lo;
  const unsigned to = hi < 0 ? 0u : hi >= 31 ? ~0u : ~0u >> (31 - hi);
  return from & to;
}

template <bool A_MN, bool B_MN, int N>
__device__ __forceinline__ constexpr uint32_t idesc() {
  return umma::instr_desc<N, A_MN, B_MN>();
}

// The eight worker warps (named barrier 1), and the two of them that share 32 rows (2 to 5).
__device__ __forceinline__ void sync_workers() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ void sync_pair(int quarter) { asm volatile("bar.sync %0, 64;" ::"r"(2 + quarter) : "memory"); }

// sync_workers, and whether any of them says yes.
__device__ __forceinline__ bool any_worker(bool yes) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred q, 1, 256, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"((uint32_t)yes)
      : "memory");
  return any != 0;
}

// Whether any of eight bf16 is not finite: one more in its last place carries such an exponent into the sign.
__device__ __forceinline__ bool any_odd(const uint4& v) {
  auto carry = [](uint32_t w) { return (w & 0x7f807f80u) + 0x00800080u; };
  return ((carry(v.x) | carry(v.y) | carry(v.z) | carry(v.w)) & 0x80008000u) != 0;
}
// Which of two (bit 0: the lower one), and of eight.
__device__ __forceinline__ uint32_t odd_of(uint32_t w) {
  return ((w & 0x7f80u) == 0x7f80u ? 1u : 0u) | ((w & 0x7f800000u) == 0x7f800000u ? 2u : 0u);
}
__device__ __forceinline__ uint32_t odd_of(const uint4& v) {
  return odd_of(v.x) | odd_of(v.y) << 2 | odd_of(v.z) << 4 | odd_of(v.w) << 6;
}

// A value whose descendants the compiler does not take out of a loop.
__device__ __forceinline__ int opaque(int x) {
  asm volatile("" : "+r"(x));
  return x;
}

// Four lanes' rows of 16 values, four at a time, turned about: lane l's piece j becomes lane j's piece l.
// A row's 64 bytes are then read or written by four neighbouring lanes at once.
__device__ __forceinline__ void turn_quads(float* s, int lane) {
#pragma unroll
  for (int bit = 1; bit <= 2; bit <<= 1) {
    const bool up = lane & bit;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j & bit) continue;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        float &a = s[4 * j + u], &b = s[4 * (j + bit) + u];
        const float y = __shfl_xor_sync(~0u, up ? a : b, bit);
        if (up) a = y; else b = y;
      }
    }
  }
}

// A sequence of the launch: one (batch row, head) and 64 columns of c (one or two slices of them). A block
// takes every gridDim.x-th; the heads and slices of a batch row follow one another.
struct Seq {
  int batch, at;  // at: head * slices + slice
  int per, slices, by_batch, by_at;
  __device__ Seq(const Op& o, int w, int stride) {
    slices = o.Dc > kDS ? 2 : 1;
    per = o.heads * slices;
    batch = w / per;
    at = w - batch * per;
    by_batch = stride / per;
    by_at = stride - by_batch * per;
  }
  __device__ __forceinline__ void advance() {
    batch += by_batch;
    at += by_at;
    if (at >= per) {
      at -= per;
      ++batch;
    }
  }
  __device__ __forceinline__ int head() const { return slices == 2 ? at >> 1 : at; }
  __device__ __forceinline__ int d0() const { return slices == 2 ? (at & 1) * kDS : 0; }
};

// kOut: outputs, from the state that enters the split; else the split's own sum. kCuts: there are resets.
template <int DA, bool kOut, bool kCuts>
__global__ void __launch_bounds__(kThreads, 2)
    chunk_tc_kernel(const __grid_constant__ Ops ops, const __grid_constant__ Maps maps, int* err) {
  using F = Cfg<DA>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + F::kBar);
  // full: tiles loaded; done_a: P0 and a S computed; done_l, done_o: L, O computed; has_w, has_p,
  // has_s: the workers' planes, P and state (and tensor memory read) are in place
  uint64_t *full = bars, *done_a = bars + 1, *done_l = bars + 2, *done_o = bars + 3, *has_w = bars + 4,
           *has_p = bars + 5, *has_s = bars + 6;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 7);
  volatile int* s_fail = reinterpret_cast<int*>(bars + 8);
  float* pw = reinterpret_cast<float*>(smem + F::kBar + 80);  // e^{i g}
  float* pl = pw + kC + 4;  // what the rounding left of e^{i g}, i = 127, 128, n and n - 1 of the last chunk
  unsigned* s_cut = reinterpret_cast<unsigned*>(pl + 4);  // [2][4] the cuts of a chunk, a bit a position

  // a copy in shared memory, so that what is rarely needed holds no registers
  Op& o = *reinterpret_cast<Op*>(smem + F::kOp);
  if (threadIdx.x < sizeof(Op) / 4)
    reinterpret_cast<uint32_t*>(&o)[threadIdx.x] = reinterpret_cast<const uint32_t*>(&ops.op[blockIdx.z])[threadIdx.x];
  __syncthreads();
  if ((int)blockIdx.x >= o.batch * o.heads * ceil_div(o.Dc, kDS)) return;
  if (smem_u32(smem) & 1023) {  // the swizzled tiles count on it
    if (threadIdx.x == 0) atomicExch(err, kErrAlignment);
    return;
  }
  const int split = blockIdx.y;
  const int begin = split * o.split_len, end = min(o.steps, begin + o.split_len);
  const int tid = threadIdx.x, warp = __shfl_sync(~0u, tid >> 5, 0), lane = tid & 31;
  const int na = min(F::kNA, ceil_div(o.Da, 64));
  const uint32_t base = smem_u32(smem);
  const bool reverse = o.reverse;

  auto time_of = [&](int i0) { return reverse ? o.steps - i0 - kC : i0; };
  auto load = [&](const Seq& q, int i0) {
    const int t0 = time_of(i0);
    mbar_arrive_expect_tx(full, ((kOut ? 2 : 1) * na + 1) * kBlock);
    tma_load_4d(smem + F::kCc, &maps.c[blockIdx.z], q.d0(), t0, q.head(), q.batch, full);
    for (int x = 0; x < na; ++x) {
      if (kOut) tma_load_4d(smem + F::kA + x * kBlock, &maps.a[blockIdx.z], 64 * x, t0, q.head(), q.batch, full);
      tma_load_4d(smem + F::kB + x * kBlock, &maps.b[blockIdx.z], 64 * x, t0, q.head(), q.batch, full);
    }
  };
  // towards L2, a chunk ahead of its load
  auto prefetch = [&](const Seq& q, int i0) {
    const int t0 = time_of(i0);
    tma_prefetch_4d(&maps.c[blockIdx.z], q.d0(), t0, q.head(), q.batch);
    for (int x = 0; x < na; ++x) {
      if (kOut) tma_prefetch_4d(&maps.a[blockIdx.z], 64 * x, t0, q.head(), q.batch);
      tma_prefetch_4d(&maps.b[blockIdx.z], 64 * x, t0, q.head(), q.batch);
    }
  };
  // the chunk after (q, i0) in this block's walk
  auto advance = [&](Seq& q, int& i0) {
    i0 += kC;
    if (i0 >= end) {
      i0 = begin;
      q.advance();
    }
    return q.batch < o.batch;
  };
  if (warp == 8) {
    if (lane == 0) {
      *s_fail = 0;
      for (int i = 0; i < 4; ++i) mbar_init(bars + i, 1);
      for (int i = 4; i < 7; ++i) mbar_init(bars + i, kWorkers / 32);
      fence_mbar_init();
      Seq q(o, blockIdx.x, gridDim.x);
      int i0 = begin;
      load(q, i0);
      if (advance(q, i0)) prefetch(q, i0);
    }
    __syncwarp();
    umma::tmem_alloc(tmem_slot, kCols);
  }
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  // A wait that gives up is recorded, and no wait after it is taken: the block runs to its end.
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (*s_fail) return;
    if (!mbar_wait_bounded(bar, parity)) *s_fail = 1;
    fence_after_sync();
  };
  auto decay_of = [&](int head) { return clamped_decay(o.log_decay[head]); };

  if (warp == 8) {
    // Descriptors of the tiles; a step along the contraction adds to the address field (16-byte units).
    const uint64_t da = smem_desc(base + F::kA, 16, 1024), db = smem_desc(base + F::kB, 16, 1024);
    const uint64_t ds = smem_desc(base + F::kS, 8192, 1024), dc = smem_desc(base + F::kCc, 8192, 1024);
    // b by columns: the second 64 rows of a 64-wide b are its first ones again
    const uint64_t dbt = smem_desc(base + F::kB, na == 2 ? kBlock : 0, 1024);
    const uint64_t dp[3] = {smem_desc(base + F::plane(0), 8192, 1024), smem_desc(base + F::plane(1), 8192, 1024),
                            smem_desc(base + F::plane(2), 8192, 1024)};
    const bool leader = elect_one();
    uint32_t parity = 0;
    Seq q(o, blockIdx.x, gridDim.x);
    int i0 = begin, head = q.head();
    bool weak = decay_of(head) >= kWeakDecay;
    for (bool more = true; more; parity ^= 1) {
      wait(full, parity);
      if (kOut) {
        wait(has_s, parity);
        if (*s_fail) break;
        if (leader) {
#pragma unroll
          for (int x = 0; x < DA / 16; ++x)
            if (x < 4 || na == 2) {
              const uint64_t off = ((x >> 2) * kBlock + (x & 3) * 32) >> 4;
              mma_bf16(tmem, da + off, db + off, idesc<false, false, 128>(), x > 0);
            }
#pragma unroll
          for (int x = 0; x < DA / 16; ++x)
            if (x < 4 || na == 2) {
              const uint64_t off = ((x >> 2) * kBlock + (x & 3) * 32) >> 4;
              mma_bf16(tmem + kOCol, da + off, ds + (x * 2048 >> 4), idesc<false, true, 64>(), x > 0);
            }
          mma_commit(done_a);
        }
        __syncwarp();
      }
      wait(has_w, parity);
      if (*s_fail) break;
      if (leader) {
#pragma unroll
        for (int q = 2; q >= 0; --q)  // smallest first
#pragma unroll
          for (int x = 0; x < kC / 16; ++x)
            mma_bf16(tmem + kLCol, dbt + (x * 2048 >> 4), dp[q] + (x * 2048 >> 4), idesc<true, true, 64>(), q < 2 || x > 0);
        mma_commit(done_l);
      }
      __syncwarp();
      if (kOut) {
        wait(has_p, parity);
        if (*s_fail) break;
        if (leader) {
          if (weak) {
#pragma unroll
            for (int q = 1; q >= 0; --q)
#pragma unroll
              for (int x = 0; x < kC / 16; ++x)
                mma_bf16_ts(tmem + kOCol, tmem + (x >> 2) * 64 + (x & 3) * 8, dp[q] + (x * 2048 >> 4),
                            idesc<false, true, 64>(), 1);
          } else {
#pragma unroll
            for (int x = 0; x < kC / 16; ++x)
              mma_bf16_ts(tmem + kOCol, tmem + (x >> 2) * 64 + (x & 3) * 8, dc + (x * 2048 >> 4),
                          idesc<false, true, 64>(), 1);
          }
          mma_commit(done_o);
        }
        __syncwarp();
        wait(done_o, parity);
      }
      wait(done_l, parity);
      if (*s_fail) break;
      more = advance(q, i0);
      if (!more) break;
      if (leader) {
        load(q, i0);
        Seq q2 = q;
        int i2 = i0;
        if (advance(q2, i2)) prefetch(q2, i2);
      }
      __syncwarp();
      if (q.head() != head) {
        head = q.head();
        weak = decay_of(head) >= kWeakDecay;
      }
    }
    if (*s_fail) {
      // let copies and MMAs in flight end before the block's memory goes
      mbar_wait_bounded(full, parity);
      mbar_wait_bounded(done_a, parity);
      mbar_wait_bounded(done_l, parity);
      mbar_wait_bounded(done_o, parity);
    }
  } else {
    const int row0 = (warp & 3) * 32 + lane, half0 = warp >> 2, lane0 = lane;  // tensor memory lane, column half
    uint8_t* const smem0 = smem;
    // A worker's piece of the state: row k, columns y0 .. (the rows of L repeat where Da <= 64, and the
    // second copy takes the other half of the columns).
    constexpr int kSC = DA == 128 ? 32 : 16;
    auto row_of_state = [&]() { return DA == 128 ? opaque(row0) : opaque(row0) & 63; };
    auto column_of_state = [&]() { return DA == 128 ? opaque(half0) * 32 : (opaque(row0) >> 6) * 32 + half0 * 16; };
    float s[kSC];
    auto put_state = [&]() {
      const int k = row_of_state(), y0 = column_of_state();
#pragma unroll
      for (int i = 0; i < kSC; i += 8) {
        uint32_t w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) w[u] = pack_bf16(s[i + 2 * u], s[i + 2 * u + 1]);
        *reinterpret_cast<uint4*>(smem + F::kS + k * 128 + ((((y0 + i) >> 3) ^ (k & 7)) << 4)) =
            make_uint4(w[0], w[1], w[2], w[3]);
      }
    };
    // where a sequence's entering state lies (null: zeros), and by which strides
    const bool local = kOut && split > 0;
    auto state_in = [&](const Seq& q, int k, int y0, int& sx, int& sy) -> const float* {
      const float* all = !kOut ? nullptr : local ? o.local + (size_t)(split - 1) * o.batch * o.heads * (o.Da * o.Dc) : o.init;
      if (!all) return nullptr;
      sx = local ? o.Dc : o.sx;
      sy = local ? 1 : o.sy;
      return all + (size_t)(q.batch * o.heads + q.head()) * (o.Da * o.Dc) + k * sx + (q.d0() + y0) * sy;
    };
    // (a state's rows start on 16-byte boundaries where its columns lie together and Dc is a multiple of 4)
    const bool whole_in = (local || o.sy == 1) && o.Dc % 4 == 0 && ((uintptr_t)(local ? o.local : o.init) & 15) == 0;
    auto load_state = [&](const Seq& q) {
      int sx = 0, sy = 0;
      const int k = row_of_state(), y0 = column_of_state();
      const float* from = state_in(q, k, y0, sx, sy);
      const int left = from ? o.Dc - q.d0() - y0 : 0;  // columns of this piece that there are
      if (whole_in) {
        const int l = lane & 3;
#pragma unroll
        for (int i = 0; i < kSC; i += 4) {
          const int r = (i >> 2 & 3) - l, c = (i & ~15) + 4 * l;  // the row's neighbour, and its columns
          const float4 f = k + r < o.Da && c < left ? *reinterpret_cast<const float4*>(from + r * sx + c)
                                                    : make_float4(0.f, 0.f, 0.f, 0.f);
          s[i] = f.x, s[i + 1] = f.y, s[i + 2] = f.z, s[i + 3] = f.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < kSC; ++i) s[i] = k < o.Da && i < left ? from[i * sy] : 0.f;
      }
    };
    // after load_state, before the state is used
    auto settle_state = [&]() {
      if (whole_in)
#pragma unroll
        for (int i = 0; i < kSC; i += 16) turn_quads(s + i, lane);
    };
    // what the walk leaves of s: the final state, or the split's own sum
    auto store_state = [&](const Seq& q) {
      float* const all = !kOut ? o.local + (size_t)split * o.batch * o.heads * (o.Da * o.Dc)
                               : split == o.nsplit - 1 ? o.fin : nullptr;
      if (!all) return;
      const int k = row_of_state(), y0 = column_of_state();
      const int tx = kOut ? o.sx : o.Dc, ty = kOut ? o.sy : 1;
      const bool whole_out = ty == 1 && o.Dc % 4 == 0 && ((uintptr_t)all & 15) == 0;
      // backwards the way out of the last position passes reset[0] and one decay more
      const bool out = kOut && reverse;
      const bool dropped = out && o.reset && o.reset[q.batch * o.reset_batch];
      const float f = out ? pw[1] : 1.f;
      float* to = all + (size_t)(q.batch * o.heads + q.head()) * (o.Da * o.Dc) + k * tx + (q.d0() + y0) * ty;
      const int left = o.Dc - q.d0() - y0;
      // s is not read again
#pragma unroll
      for (int i = 0; i < kSC; ++i) s[i] = dropped ? 0.f : f * s[i];
      if (whole_out) {
        const int l = lane & 3;
#pragma unroll
        for (int i = 0; i < kSC; i += 16) turn_quads(s + i, lane);
#pragma unroll
        for (int i = 0; i < kSC; i += 4) {
          const int r = (i >> 2 & 3) - l, c = (i & ~15) + 4 * l;
          if (k + r < o.Da && c < left)
            *reinterpret_cast<float4*>(to + r * tx + c) = make_float4(s[i], s[i + 1], s[i + 2], s[i + 3]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kSC; ++i)
          if (k < o.Da && i < left) to[i * ty] = s[i];
      }
    };
    uint32_t parity = 0;
    int head = -1;
    bool weak = true;
    Seq q(o, blockIdx.x, gridDim.x);
    auto cut_at = [&](int batch, int i0) { return tid < kC && i0 + tid < end && op_cut(o, batch, i0 + tid); };
    bool cut = kCuts && cut_at(q.batch, begin);
    load_state(q);
    auto arrive = [&](uint64_t* bar) {
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };

    for (bool more = true; more;) {
      if (q.head() != head) {
        head = q.head();
        const float g = decay_of(head);
        weak = g >= kWeakDecay;
        sync_workers();  // nobody reads the last head's powers any more
        if (tid <= kC) {
          pw[tid] = (float)exp((double)tid * (double)g);
        } else if (tid >= kWorkers - 4) {
          const int last = end - begin - (end - begin - 1) / kC * kC;
          const int x = tid - (kWorkers - 4);
          const double e = exp((double)(x == 0 ? kC - 1 : x == 1 ? kC : x == 2 ? last : last - 1) * (double)g);
          pl[x] = (float)(e - (double)(float)e);
        }
        sync_workers();
      }
      Seq next = q;
      next.advance();
      more = next.batch < o.batch;
      settle_state();
      bool any_cut = false;
      int e0 = (reverse && split == 0) ? 0 : 1;
      // s takes its decay over the n positions to come, and its copy goes where O's product reads it. The
      // factor in two parts: its rounding, met once a chunk, would add up over a long memory.
      auto hand_state = [&](int n) {
        if (kOut && !weak) put_state();
        const float keep = pw[n - 1 + e0], keep_lo = pl[n == kC ? e0 : 3 - e0];
#pragma unroll
        for (int i = 0; i < kSC; ++i) s[i] = fmaf(keep, s[i], keep_lo * s[i]);
        if (kOut && weak) put_state();
        fence_proxy_async_smem();
      };
      hand_state(min(kC, end - begin));
      if (kOut) arrive(has_s);

      for (int i0 = begin; i0 < end; i0 += kC, parity ^= 1) {
        const int n = min(kC, end - i0);
        const bool ends = i0 + kC >= end;
        // what follows from a thread's place is formed anew in every chunk: kept, it would crowd the registers out
        // into local memory, for which shared memory leaves next to no L1
        const int row = opaque(row0), half = opaque(half0), lane = opaque(lane0);
        const int p = reverse ? kC - 1 - row : row;
        uint8_t* const smem = smem0 + opaque(0);
        uint8_t* const stage = smem + F::kP2 + (row >> 5) * 4096 + half * 2048;  // in plane rows of this warp pair
        const uint32_t lanes = tmem + ((uint32_t)(row & 96) << 16);
        const int y0 = DA == 128 ? half * 32 : (row >> 6) * 32 + half * 16;
        // the last cut of the chunk, and the last one at or before p (-1: none)
        int last = -1, lo = -1;
        bool odd = false;
        unsigned* cuts = s_cut + 4 * parity;
        if (kCuts && tid < kC) {
          const unsigned m = __ballot_sync(~0u, cut);
          if (lane == 0) cuts[warp] = m;
          cut = (!ends || more) && cut_at(ends ? next.batch : q.batch, ends ? begin : i0 + kC);
        }
        wait(full, parity);
        if (kCuts) {
          if constexpr (kOut) {
#pragma unroll
            for (int u = 0; u < 4; ++u)
              odd |= any_odd(*reinterpret_cast<const uint4*>(smem + F::kCc + row * 128 + (((half * 4 + u) ^ (row & 7)) << 4)));
            odd = any_worker(odd);
          } else {
            sync_workers();
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const unsigned m = cuts[x], own = m & bits(0, p - 32 * x);
            if (m) last = 32 * x + 31 - __clz(m);
            if (own) lo = 32 * x + 31 - __clz(own);
          }
          any_cut |= last >= 0;
        }
        // Values of c that are not finite, in a chunk with a cut: the products would carry them across it as 0 times
        // themselves. They are taken out of the tile, and what they reach (their column of the later outputs of
        // their own stretch, and of the state where no cut follows) is set to NaN at the end. A bit a column.
        uint32_t odd_out = 0, odd_state = 0;
        if (kOut && kCuts && odd && last >= 0) {
          auto columns = [&](int from, int to, int c0, int count) {
            uint32_t m = 0;
            for (int at = from; at <= to; ++at) {
              const int r = reverse ? kC - 1 - at : at;
              for (int u = 0; u < count; u += 8)
                m |= odd_of(*reinterpret_cast<const uint4*>(smem + F::kCc + r * 128 + ((((c0 + u) >> 3) ^ (r & 7)) << 4))) << u;
            }
            return m;
          };
          odd_out = columns(max(lo, 0), min(p, n - 1), 32 * half, 32);
          odd_state = columns(last, n - 1, y0, kSC);
          sync_workers();
          for (int u = 0; u < 4; ++u) {
            uint4* const at = reinterpret_cast<uint4*>(smem + F::kCc + row * 128 + (((half * 4 + u) ^ (row & 7)) << 4));
            uint32_t w[4] = {at->x, at->y, at->z, at->w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t m = odd_of(w[i]);
              w[i] &= ~((m & 1 ? 0xffffu : 0u) | (m & 2 ? 0xffff0000u : 0u));
            }
            *at = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        if (kOut) {
          // the pair's last outputs have left their staging rows
          if (lane == 0) umma::bulk_wait_read_all();
          sync_pair(row >> 5);
        }
        {  // w c: this thread's row, half of the columns
          const float wf = p < n ? o.in_scale * pw[n - 1 - p] : 0.f;
          const uint64_t wp = pair(wf, wf);
          // 24 bits cut into 8 + 8 + 8: each plane takes the leading bits, the rest is exact
          auto cut_up = [&](int off, uint4 (&y)[3]) {
            uint4 x = *reinterpret_cast<const uint4*>(smem + F::kCc + off);
            if (!kOut && last > p) x = make_uint4(0, 0, 0, 0);  // hidden by a cut, whatever it holds
            const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
            uint32_t t[3][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint64_t v = mul2(wp, pair_of_bf16(xs[i]));
#pragma unroll
              for (int z = 0; z < 3; ++z) {
                t[z][i] = __byte_perm((uint32_t)v, (uint32_t)(v >> 32), 0x7632);
                if (z < 2) v = sub2(v, v & 0xffff0000ffff0000ull);
              }
            }
#pragma unroll
            for (int z = 0; z < 3; ++z) y[z] = make_uint4(t[z][0], t[z][1], t[z][2], t[z][3]);
          };
          auto place = [&](int u) { return row * 128 + (((half * 4 + u) ^ (row & 7)) << 4); };
          // Planes 0 (and 1) take a's place and wait for O's product. One plane is held until then; two would not
          // fit in the registers, and forming them twice cost more than waiting first (2 x 8191 x 16 x 128
          // training pass: 503 us, 485 so).
          uint4 held[4], y[3];
          if (F::kNA == 2 && kOut) wait(done_a, parity);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            cut_up(place(u), y);
            if (F::kNA == 1) held[u] = y[0];
#pragma unroll
            for (int z = F::kNA == 1 ? 1 : 0; z < 3; ++z) *reinterpret_cast<uint4*>(smem + F::plane(z) + place(u)) = y[z];
          }
          if (F::kNA == 1) {
            if (kOut) wait(done_a, parity);
#pragma unroll
            for (int u = 0; u < 4; ++u) *reinterpret_cast<uint4*>(smem + F::plane(0) + place(u)) = held[u];
          }
          if (last > p) {  // what a cut hides has no part in L; P0 is done with its row of b
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
              for (int x = 0; x < F::kNA; ++x)
                *reinterpret_cast<uint4*>(smem + F::kB + x * kBlock + row * 128 + (half * 4 + u) * 16) =
                    make_uint4(0, 0, 0, 0);
          }
        }
        fence_proxy_async_smem();
        arrive(has_w);
        if (kOut) {
          if (!weak || last >= 0) {
            // the rows of a S by the decay since the state; a cut drops it whatever it holds
            const float reach = lo >= 0 || p >= n ? 0.f : weak ? 1.f : pw[p + e0];
#pragma unroll 1
            for (int j = 0; j < 2; ++j) {
              float v[16];
              uint32_t x[16];
              tmem_ld16(lanes + kOCol + 32 * half + 16 * j, v);
#pragma unroll
              for (int i = 0; i < 16; ++i) x[i] = reach != 0.f ? __float_as_uint(reach * v[i]) : 0u;
              tmem_st16(lanes + kOCol + 32 * half + 16 * j, x);
            }
          }
          // P: this warp's 32 rows against the columns 64 half .. 64 half + 63, 16 at a time. It takes the place
          // of the first half of them: what it replaces is read by then.
          const int first = max(lo, 0);  // columns of positions first .. p count
#pragma unroll 1
          for (int u = 0; u < 4; ++u) {
            const int c0 = 64 * half + 16 * u;
            const unsigned m = (reverse ? bits(kC - 1 - c0 - p, kC - 1 - c0 - first) : bits(first - c0, p - c0)) & 0xffffu;
            uint32_t pk[8];
            if (__all_sync(~0u, m == 0)) {
#pragma unroll
              for (int i = 0; i < 8; ++i) pk[i] = 0;
            } else {
              float v[16];
              tmem_ld16(lanes + c0, v);
              if (!weak) {
                // e^{(p_i - p_j) g}: only where the column comes no later than the row
                const int gap0 = reverse ? c0 - row : row - c0, dir = reverse ? 1 : -1;
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] *= o.in_scale * pw[max(0, gap0 + dir * i)];
              }
              if (!__all_sync(~0u, m == 0xffffu)) {
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = m >> i & 1 ? v[i] : 0.f;
              }
#pragma unroll
              for (int i = 0; i < 8; ++i) pk[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
            }
            tmem_st8(lanes + 64 * half + 8 * u, pk);
          }
          tmem_wait_st();
          arrive(has_p);
        }
        wait(done_l, parity);
        {
          float l[kSC];
          if constexpr (kSC == 32) tmem_ld32(lanes + kLCol + y0, l);
          else tmem_ld16(lanes + kLCol + y0, l);
#pragma unroll
          for (int i = 0; i < kSC; ++i) s[i] = (last < 0 ? s[i] : 0.f) + l[i];
          if (kOut && kCuts && odd_state)
#pragma unroll
            for (int i = 0; i < kSC; ++i) s[i] = odd_state >> i & 1 ? __int_as_float(0x7fffffff) : s[i];
        }
        e0 = 1;
        if (!ends) {
          hand_state(min(kC, end - i0 - kC));
        } else {
          store_state(q);
          if (!kOut && tid == 0 && q.at == 0) o.cut[split * o.batch + q.batch] = any_cut;
          if (more) load_state(next);  // comes in while the outputs go out
        }
        if (kOut) {
          wait(done_o, parity);
          const float f = weak && p < n ? o.out_scale / pw[n - 1 - p] : o.out_scale;
          const int t0 = time_of(i0), x0 = q.d0() + 32 * half;
#pragma unroll 1
          for (int j = 0; j < 2; ++j) {
            float v[16];
            tmem_ld16(lanes + kOCol + 32 * half + 16 * j, v);
            if (j == 1 && !ends) arrive(has_s);
            if (kCuts && odd_out)
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] = odd_out >> (16 * j + i) & 1 ? __int_as_float(0x7fffffff) : v[i];
            uint4 y[2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
              y[i] = make_uint4(pack_bf16(f * v[8 * i], f * v[8 * i + 1]), pack_bf16(f * v[8 * i + 2], f * v[8 * i + 3]),
                                pack_bf16(f * v[8 * i + 4], f * v[8 * i + 5]), pack_bf16(f * v[8 * i + 6], f * v[8 * i + 7]));
            if (t0 >= 0) {  // (the 64-byte swizzle of a row of 32)
#pragma unroll
              for (int i = 0; i < 2; ++i)
                *reinterpret_cast<uint4*>(stage + lane * 64 + (((2 * j + i) ^ (lane >> 1 & 3)) << 4)) = y[i];
            } else if (p < n) {  // a first chunk in time that begins before step 0
              __nv_bfloat16* out = static_cast<__nv_bfloat16*>(o.out) + q.batch * o.out_batch +
                                   (int64_t)(t0 + row) * o.out_step + q.head() * o.out_head + x0 + 16 * j;
#pragma unroll
              for (int i = 0; i < 2; ++i)  // Dc is a multiple of 8 (suits_tensor_cores)
                if (x0 + 16 * j + 8 * i < o.Dc) *reinterpret_cast<uint4*>(out + 8 * i) = y[i];
            }
          }
          if (t0 >= 0) {
            // rows behind the last step and columns behind Dc fall away in the store
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && x0 < o.Dc) {
              tma_store_4d(&maps.out[blockIdx.z], stage, x0, t0 + 32 * (warp & 3), q.head(), q.batch);
              umma::bulk_commit();
            }
          }
        }
      }
      q = next;
    }
    if (lane == 0) umma::bulk_wait_all();
    __syncwarp();
  }
  fence_before_sync();
  __syncthreads();
  if (warp == 8) {
    fence_after_sync();
    umma::tmem_dealloc(tmem, kCols);
    if (lane == 0 && *s_fail) atomicExch(err, umma::kErrTimeoutFull);
  }
}

int map_rows(CUtensorMap* m, const Op& o, const Rows& r, int d) {
  const uint64_t dims[4] = {(uint64_t)d, (uint64_t)o.steps, (uint64_t)o.heads, (uint64_t)o.batch};
  const uint64_t strides[3] = {(uint64_t)r.step * 2, (uint64_t)r.head * 2, (uint64_t)r.batch * 2};
  const uint32_t box[4] = {64, kC, 1, 1};
  return umma::encode_map_4d(m, r.p, dims, strides, box, 128);
}

int map_out(CUtensorMap* m, const Op& o) {
  const uint64_t dims[4] = {(uint64_t)o.Dc, (uint64_t)o.steps, (uint64_t)o.heads, (uint64_t)o.batch};
  const uint64_t strides[3] = {(uint64_t)o.out_step * 2, (uint64_t)o.out_head * 2, (uint64_t)o.out_batch * 2};
  const uint32_t box[4] = {32, 32, 1, 1};
  return umma::encode_map_4d(m, o.out, dims, strides, box, 64);
}

}  // namespace

bool suits_tensor_cores(const Op& o) {
  auto rows = [&](const Rows& r) {
    auto ok = [](int64_t s, int n) { return n <= 1 || (s > 0 && s % 8 == 0 && s < ((int64_t)1 << 38)); };
    return ((uintptr_t)r.p & 15) == 0 && ok(r.step, o.steps) && ok(r.head, o.heads) && ok(r.batch, o.batch);
  };
  // A TMA store writes whole 16-byte pieces: behind a row that ends inside one it would overwrite what lies there.
  return o.Dc % 8 == 0 && rows(o.a) && rows(o.b) && rows(o.c) && ((uintptr_t)o.out & 15) == 0 && o.out_step % 8 == 0 &&
         o.out_head % 8 == 0 && o.out_batch % 8 == 0;
}

int run_tensor_cores(Ops& ops, cudaStream_t stream) {
  Maps maps;
  int da = 0, blocks = 0, per = 1;
  for (int i = 0; i < ops.n; ++i) {
    const Op& o = ops.op[i];
    const int slices = ceil_div(o.Dc, kDS);
    da = max(da, o.Da);
    blocks = max(blocks, o.batch * o.heads * slices);
    per = max(per, o.heads * slices);
    BT_TRY(map_rows(&maps.a[i], o, o.a, o.Da));
    BT_TRY(map_rows(&maps.b[i], o, o.b, o.Da));
    BT_TRY(map_rows(&maps.c[i], o, o.c, o.Dc));
    BT_TRY(map_out(&maps.out[i], o));
  }
  int* err = nullptr;
  BT_TRY(operator_error_word(&err));
  const Op& o = ops.op[0];
  auto go = [&](auto size, auto cuts) -> int {
    constexpr int DA = decltype(size)::value;
    constexpr bool kCuts = decltype(cuts)::value;
    auto sums = chunk_tc_kernel<DA, false, kCuts>;
    auto outs = chunk_tc_kernel<DA, true, kCuts>;
    constexpr int kSmem = Cfg<DA>::kBytes;
    static std::atomic<uint64_t> allowed[2];
    BT_TRY(allow_smem(outs, kSmem, allowed[0]));
    // Two blocks an SM in all, each with every so many-th sequence: the same head again and again where the
    // heads allow it (its powers are kept).
    auto wide = [&](int splits) {
      const int room = max(1, 2 * kNumSMs / (splits * ops.n));
      return min(blocks, room > per ? room / per * per : room);
    };
    if (o.nsplit > 1) {
      BT_TRY(allow_smem(sums, kSmem, allowed[1]));
      sums<<<dim3(wide(o.nsplit - 1), o.nsplit - 1, ops.n), kThreads, kSmem, stream>>>(ops, maps, err);
      BT_LAUNCH_CHECK("linear attention split sums");
      BT_TRY(launch_join(ops, stream));
    }
    outs<<<dim3(wide(o.nsplit), o.nsplit, ops.n), kThreads, kSmem, stream>>>(ops, maps, err);
    BT_LAUNCH_CHECK("linear attention");
    return BT_OK;
  };
  // Unrolls without resets take none of the cuts' work (16 x 2000 x 8 x 64/128 forward: 82 us so, 86 with it).
  using Narrow = std::integral_constant<int, 64>;
  using Wide = std::integral_constant<int, 128>;
  if (o.reset) return da <= 64 ? go(Narrow{}, std::true_type{}) : go(Wide{}, std::true_type{});
  return da <= 64 ? go(Narrow{}, std::false_type{}) : go(Wide{}, std::false_type{});
}

}  // namespace la
}  // namespace bt

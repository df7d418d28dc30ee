// Linear attention with a decay per head on the tensor cores (tcgen05), bf16 inputs (the operation:
// linear_attention.cuh).
//
// A block owns one (batch row, head), 64 columns of c and of the state, and walks its positions 128 at
// a time. In a chunk, with p the position of a row and everything accumulated in fp32:
//   P0 = a b^T                                     [128 x 128]  tensor memory
//   O2 = a S                                       [128 x 64]   S: bf16 copy of the state in shared memory
//   P  = P0 * e^{(p_i - p_j) g}, 0 above the diagonal and across a cut, to bf16 in tensor memory
//   O1 = P c                                       [128 x 64]   P is the A operand from tensor memory
//   L  = b^T (w c), w_j = e^{(n - 1 - p_j) g}      [Da x 64]    w c as three bf16 planes (24 bits)
//   out = in_scale O1 + e^{(p + e0) g} O2, times out_scale;   S = e^{(n - 1 + e0) g} S + in_scale L
// The state itself stays in fp32 registers for the whole walk. Only two factors are rounded to bf16, P
// and the copy of S that O2 reads, and both go only into outputs that are rounded to bf16 themselves
// (each adds 2^-9 root mean square at most); the state, which is handed on in fp32, comes from exact
// products: b is bf16 already, and w c keeps 24 bits.
//
// Backwards the tiles stay in the order of time and the positions run against it: p = 127 - r.
//
// Bound by HBM (4 elements of traffic per element of out); a chunk is a chain of dependent steps
// (load, MMA, registers, MMA, ...), so two blocks share an SM and fill each other's waits: 256 of the
// 512 columns of tensor memory each (P in place of P0, L in the half of P0 that P leaves), and at most
// 113 KB of shared memory (two planes of w c in place of a, which O2 is done with).
#include <type_traits>

#include "gemm_sm100.cuh"
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

constexpr int kC = 128, kDS = 64, kThreads = 256;
constexpr int kBlock = kC * 128;  // 128 rows of 64 bf16, 128-byte swizzle
constexpr uint32_t kCols = 256;   // tensor memory: P0 / P | L, O1, O2
constexpr int kErrAlignment = 15;
constexpr uint32_t kLCol = 64, kO1Col = 128, kO2Col = 192;

template <int DA>
struct Cfg {
  static constexpr int kNA = DA / 64;  // 64-wide blocks of a and b
  static constexpr int kA = 0, kB = kNA * kBlock, kCc = 2 * kNA * kBlock, kS = kCc + kBlock;
  static constexpr int kP2 = kS + DA * 128;  // planes that do not fit into a's buffer
  static constexpr int kPlanes = kP2 + (3 - kNA) * kBlock;
  static constexpr int kBar = kPlanes;
  static constexpr int kBytes = kBar + 64 + 4 * (kC + 4) + 16 + kC + 16;
  __device__ static int plane(int k) { return k < kNA ? kA + k * kBlock : kP2 + (k - kNA) * kBlock; }
};
static_assert(2 * (Cfg<128>::kBytes + 1024) <= 228 * 1024, "two blocks on an SM");

struct Maps {
  CUtensorMap a[3], b[3], c[3];
};

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int t, int h, int b,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(t), "r"(h), "r"(b), "r"(smem_u32(bar))
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

template <bool A_MN, bool B_MN, int N>
__device__ __forceinline__ constexpr uint32_t idesc() {
  return umma::instr_desc<N, A_MN, B_MN>();
}

// kOut: outputs, from the state that enters the split; else the split's own sum.
template <int DA, bool kOut>
__global__ void __launch_bounds__(kThreads, 2)
    chunk_tc_kernel(const __grid_constant__ Ops ops, const __grid_constant__ Maps maps, int* err) {
  using F = Cfg<DA>;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + F::kBar);
  uint64_t *full = bars, *bar_p = bars + 1, *bar_a = bars + 2, *bar_o = bars + 3, *bar_l = bars + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 5);
  float* pw = reinterpret_cast<float*>(smem + F::kBar + 64);  // e^{i g}
  float* pl = pw + kC + 4;  // what the rounding left of e^{i g}, i = 127, 128, n and n - 1 of the last chunk
  uint8_t* seg = reinterpret_cast<uint8_t*>(pl + 4);  // cuts up to and with a position
  unsigned* s_cut = reinterpret_cast<unsigned*>(seg + kC);

  const Op& o = ops.op[blockIdx.z];
  const CUtensorMap *ma = &maps.a[blockIdx.z], *mb = &maps.b[blockIdx.z], *mc = &maps.c[blockIdx.z];
  const int slices = ceil_div(o.Dc, kDS);
  if ((int)blockIdx.x >= o.batch * o.heads * slices) return;
  if (smem_u32(smem) & 1023) {  // the swizzled tiles count on it
    if (threadIdx.x == 0) atomicExch(err, kErrAlignment);
    return;
  }
  const int bh = blockIdx.x / slices, d0 = blockIdx.x % slices * kDS;
  const int batch = bh / o.heads, head = bh % o.heads;
  const int split = blockIdx.y;
  const int begin = split * o.split_len, end = min(o.steps, begin + o.split_len);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = (warp & 3) * 32 + lane, half = warp >> 2;  // tensor memory lane, column half
  const float g = fmaxf(o.log_decay[head], kMinLogDecay);
  const size_t elems = (size_t)o.Da * o.Dc;
  const int na = min(F::kNA, ceil_div(o.Da, 64));

  if (tid == 0) {
    mbar_init(full, 1);
    mbar_init(bar_p, 1);
    mbar_init(bar_a, 1);
    mbar_init(bar_o, 1);
    mbar_init(bar_l, 1);
    fence_mbar_init();
  }
  if (warp == 0) umma::tmem_alloc(tmem_slot, kCols);
  if (tid <= kC) pw[tid] = (float)exp((double)tid * (double)g);
  if (tid >= 252) {
    const int last = max(1, end - begin) - (max(1, end - begin) - 1) / kC * kC;
    const int i = tid == 252 ? kC - 1 : tid == 253 ? kC : tid == 254 ? last : last - 1;
    const double e = exp((double)i * (double)g);
    pl[tid - 252] = (float)(e - (double)(float)e);
  }
  // This thread's piece of the state: row k, columns y0 .. (the rows of L repeat where Da <= 64, and
  // the second copy takes the other half of the columns).
  constexpr int kSC = DA == 128 ? 32 : 16;
  const int k = DA == 128 ? row : row & 63;
  const int y0 = DA == 128 ? half * 32 : (row >> 6) * 32 + half * 16;
  float s[kSC];
  {
    const float* from = nullptr;
    int64_t sx = o.sx, sy = o.sy;
    if (kOut) {
      if (split > 0) {
        from = o.local + ((size_t)(split - 1) * o.batch * o.heads + bh) * elems;
        sx = o.Dc;
        sy = 1;
      } else if (o.init) {
        from = o.init + bh * elems;
      }
    }
#pragma unroll
    for (int i = 0; i < kSC; ++i)
      s[i] = from && k < o.Da && d0 + y0 + i < o.Dc ? from[k * sx + (d0 + y0 + i) * sy] : 0.f;
  }
  auto put_state = [&]() {
#pragma unroll
    for (int i = 0; i < kSC; i += 8) {
      uint32_t w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) w[u] = pack_bf16(s[i + 2 * u], s[i + 2 * u + 1]);
      *reinterpret_cast<uint4*>(smem + F::kS + k * 128 + ((((y0 + i) >> 3) ^ (k & 7)) << 4)) =
          make_uint4(w[0], w[1], w[2], w[3]);
    }
  };
  if (kOut) put_state();
  fence_proxy_async_smem();
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
  const uint32_t base = smem_u32(smem);

  auto load = [&](int i0) {
    const int t0 = o.reverse ? o.steps - i0 - kC : i0;
    mbar_arrive_expect_tx(full, ((kOut ? 2 : 1) * na + 1) * kBlock);
    for (int x = 0; x < na; ++x) {
      if (kOut) tma_load_4d(smem + F::kA + x * kBlock, ma, 64 * x, t0, head, batch, full);
      tma_load_4d(smem + F::kB + x * kBlock, mb, 64 * x, t0, head, batch, full);
    }
    tma_load_4d(smem + F::kCc, mc, d0, t0, head, batch, full);
  };
  bool ok = true;
  bool loading = false;
  if (tid == 0 && begin < end) {
    load(begin);
    loading = true;
  }
  bool any_cut = false;
  int e0 = (o.reverse && split == 0) ? 0 : 1;
  uint32_t parity = 0;
  const int p = o.reverse ? kC - 1 - row : row;  // the position of this thread's row

  for (int i0 = begin; i0 < end; i0 += kC, parity ^= 1) {
    const int n = min(kC, end - i0);
    // the cuts of the chunk's positions
    if (o.reset) {
      if (tid < kC) {
        const unsigned m = __ballot_sync(~0u, tid < n && op_cut(o, batch, i0 + tid));
        if (lane == 0) s_cut[warp] = m;
      }
      __syncthreads();
      if (tid < kC) {
        int c = __popc(s_cut[warp] & (~0u >> (31 - lane)));
        for (int w = 0; w < warp; ++w) c += __popc(s_cut[w]);
        seg[tid] = (uint8_t)c;
      }
      __syncthreads();
    }
    const int seg_end = o.reset ? seg[kC - 1] : 0;
    const int seg_p = o.reset ? seg[p] : 0;
    any_cut |= seg_end > 0;

    ok &= mbar_wait_bounded(full, parity);
    if (tid == 0) loading = false;
    if (kOut) {
      if (tid == 0) {
        fence_after_sync();
#pragma unroll
        for (int x = 0; x < DA / 16; ++x) {
          if (x >= na * 4) break;
          const uint32_t off = (x >> 2) * kBlock + (x & 3) * 32;
          mma_bf16(tmem, smem_desc(base + F::kA + off, 16, 1024), smem_desc(base + F::kB + off, 16, 1024),
                   idesc<false, false, 128>(), x > 0);
        }
        mma_commit(bar_p);
#pragma unroll
        for (int x = 0; x < DA / 16; ++x) {
          if (x >= na * 4) break;
          const uint32_t off = (x >> 2) * kBlock + (x & 3) * 32;
          mma_bf16(tmem + kO2Col, smem_desc(base + F::kA + off, 16, 1024),
                   smem_desc(base + F::kS + x * 2048, 8192, 1024), idesc<false, true, 64>(), x > 0);
        }
        mma_commit(bar_a);
      }
      ok &= mbar_wait_bounded(bar_p, parity);
      fence_after_sync();
      // P: this warp's 32 rows against the column blocks 2 half and 2 half + 1
      uint32_t pk[2][16];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int blk = 2 * half + u, wr = warp & 3;
        const bool past = o.reverse ? blk < wr : blk > wr;  // every position of it comes later
        if (past) {
#pragma unroll
          for (int i = 0; i < 16; ++i) pk[u][i] = 0;
          continue;
        }
        float v[32];
        tmem_ld32(lanes + 32 * blk, v);
        const int gap0 = o.reverse ? 32 * blk - row : row - 32 * blk;  // p_i - p_j of column 0
        const int dir = o.reverse ? 1 : -1;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const int gap = gap0 + dir * i;
          v[i] = gap >= 0 ? v[i] * pw[gap >= 0 ? gap : 0] : 0.f;
        }
        if (seg_end > 0) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const int c = 32 * blk + i;
            if (seg[o.reverse ? kC - 1 - c : c] != seg_p) v[i] = 0.f;
          }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) pk[u][i] = pack_bf16(v[2 * i], v[2 * i + 1]);
      }
      fence_before_sync();
      __syncthreads();  // P0 is read everywhere before P replaces it
      fence_after_sync();
      tmem_st16(lanes + 32 * half, pk[0]);
      tmem_st16(lanes + 32 * half + 16, pk[1]);
      tmem_wait_st();
      fence_before_sync();
      __syncthreads();
      if (tid == 0) {
        fence_after_sync();
#pragma unroll
        for (int x = 0; x < kC / 16; ++x)
          mma_bf16_ts(tmem + kO1Col, tmem + x * 8, smem_desc(base + F::kCc + x * 2048, 8192, 1024),
                      idesc<false, true, 64>(), x > 0);
        mma_commit(bar_o);
      }
      ok &= mbar_wait_bounded(bar_a, parity);  // O2 has read a: its buffer takes planes
    }
    {  // w c: this thread's row, half of the columns
      const bool in = p < n && seg_p == seg_end;
      const float w = in ? pw[n - 1 - p] : 0.f;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int off = row * 128 + (((half * 4 + u) ^ (row & 7)) << 4);
        const uint4 x = *reinterpret_cast<const uint4*>(smem + F::kCc + off);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const __nv_bfloat162 h = *reinterpret_cast<const __nv_bfloat162*>(&xs[i]);
          v[2 * i] = in ? w * __low2float(h) : 0.f;
          v[2 * i + 1] = in ? w * __high2float(h) : 0.f;
        }
#pragma unroll
        for (int q = 0; q < 3; ++q) {
          uint32_t y[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            y[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
            const __nv_bfloat162 h = *reinterpret_cast<const __nv_bfloat162*>(&y[i]);
            v[2 * i] -= __low2float(h);
            v[2 * i + 1] -= __high2float(h);
          }
          *reinterpret_cast<uint4*>(smem + F::plane(q) + off) = make_uint4(y[0], y[1], y[2], y[3]);
        }
      }
    }
    fence_proxy_async_smem();
    __syncthreads();
    if (tid == 0) {
      fence_after_sync();
      bool acc = false;
#pragma unroll
      for (int q = 2; q >= 0; --q)  // smallest first
#pragma unroll
        for (int x = 0; x < kC / 16; ++x) {
          // the second 64 rows of a 64-wide b are its first ones again
          mma_bf16(tmem + kLCol, smem_desc(base + F::kB + x * 2048, na == 2 ? kBlock : 0, 1024),
                   smem_desc(base + F::plane(q) + x * 2048, 8192, 1024), idesc<true, true, 64>(), acc);
          acc = true;
        }
      mma_commit(bar_l);
    }
    if (kOut) {
      ok &= mbar_wait_bounded(bar_o, parity);
      fence_after_sync();
      float o1[32], o2[32];
      tmem_ld32(lanes + kO1Col + 32 * half, o1);
      tmem_ld32(lanes + kO2Col + 32 * half, o2);
      if (p < n) {
        const float reach = seg_p == 0 ? pw[p + e0] * o.out_scale : 0.f;
        const float own = o.in_scale * o.out_scale;
        const int t = o.reverse ? o.steps - 1 - i0 - p : i0 + p;
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(o.out) + batch * o.out_batch +
                             (int64_t)t * o.out_step + head * o.out_head + d0 + 32 * half;
        // a cut drops the state whatever it holds, not 0 times it
#pragma unroll
        for (int i = 0; i < 32; ++i) o1[i] = reach != 0.f ? own * o1[i] + reach * o2[i] : own * o1[i];
        const int left = o.Dc - d0 - 32 * half;
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
          if (i + 8 <= left) {
            *reinterpret_cast<uint4*>(out + i) =
                make_uint4(pack_bf16(o1[i], o1[i + 1]), pack_bf16(o1[i + 2], o1[i + 3]),
                           pack_bf16(o1[i + 4], o1[i + 5]), pack_bf16(o1[i + 6], o1[i + 7]));
          } else {
#pragma unroll
            for (int u = 0; u < 8; ++u)
              if (i + u < left) out[i + u] = __float2bfloat16_rn(o1[i + u]);
          }
        }
      }
    }
    ok &= mbar_wait_bounded(bar_l, parity);
    fence_after_sync();
    if (tid == 0 && ok && i0 + kC < end) {
      load(i0 + kC);
      loading = true;
    }
    {
      // the factor in two parts: its rounding, met once a chunk, would add up over a long memory
      const float keep = pw[n - 1 + e0], keep_lo = pl[n == kC ? e0 : 3 - e0];
      float l[kSC];
      if constexpr (kSC == 32) tmem_ld32(lanes + kLCol + y0, l);
      else tmem_ld16(lanes + kLCol + y0, l);
#pragma unroll
      for (int i = 0; i < kSC; ++i) {
        const float old = seg_end == 0 ? fmaf(keep, s[i], keep_lo * s[i]) : 0.f;
        s[i] = old + o.in_scale * l[i];
      }
    }
    if (kOut) put_state();
    e0 = 1;
    fence_proxy_async_smem();
    fence_before_sync();
    if (__syncthreads_or(!ok)) {
      ok = false;
      break;
    }
    fence_after_sync();
  }
  if (!ok && tid == 0) {
    // let the copies and MMAs in flight end before the block's memory goes
    if (loading) mbar_wait_bounded(full, parity ^ 1);
    mbar_wait_bounded(bar_l, parity);
    atomicExch(err, umma::kErrTimeoutFull);
  }
  {
    float* to = nullptr;
    int64_t sx = o.sx, sy = o.sy;
    float last = 1.f;
    if (kOut) {
      if (o.fin && split == o.nsplit - 1) {
        to = o.fin + bh * elems;
        if (o.reverse && o.steps > 0) {
          last = pw[1];
          if (o.reset && o.reset[batch * o.reset_batch]) last = 0.f;
        }
      }
    } else {
      to = o.local + ((size_t)split * o.batch * o.heads + bh) * elems;
      sx = o.Dc;
      sy = 1;
      if (tid == 0 && d0 == 0 && head == 0) o.cut[split * o.batch + batch] = any_cut;
    }
    if (to && k < o.Da) {
#pragma unroll
      for (int i = 0; i < kSC; ++i)
        if (d0 + y0 + i < o.Dc) to[k * sx + (d0 + y0 + i) * sy] = last == 0.f ? 0.f : last * s[i];
    }
  }
  fence_before_sync();
  __syncthreads();
  if (warp == 0) {
    fence_after_sync();
    umma::tmem_dealloc(tmem, kCols);
  }
}

int map_rows(CUtensorMap* m, const Op& o, const Rows& r, int d) {
  const uint64_t dims[4] = {(uint64_t)d, (uint64_t)o.steps, (uint64_t)o.heads, (uint64_t)o.batch};
  const uint64_t strides[3] = {(uint64_t)r.step * 2, (uint64_t)r.head * 2, (uint64_t)r.batch * 2};
  const uint32_t box[4] = {64, kC, 1, 1};
  return umma::encode_map_4d(m, r.p, dims, strides, box);
}

}  // namespace

bool suits_tensor_cores(const Op& o) {
  auto rows = [&](const Rows& r) {
    auto ok = [](int64_t s, int n) { return n <= 1 || (s > 0 && s % 8 == 0 && s < ((int64_t)1 << 38)); };
    return ((uintptr_t)r.p & 15) == 0 && ok(r.step, o.steps) && ok(r.head, o.heads) && ok(r.batch, o.batch);
  };
  return rows(o.a) && rows(o.b) && rows(o.c) && ((uintptr_t)o.out & 15) == 0 && o.out_step % 8 == 0 &&
         o.out_head % 8 == 0 && o.out_batch % 8 == 0;
}

int run_tensor_cores(Ops& ops, cudaStream_t stream) {
  Maps maps;
  int da = 0, blocks = 0;
  for (int i = 0; i < ops.n; ++i) {
    const Op& o = ops.op[i];
    da = max(da, o.Da);
    blocks = max(blocks, o.batch * o.heads * ceil_div(o.Dc, kDS));
    BT_TRY(map_rows(&maps.a[i], o, o.a, o.Da));
    BT_TRY(map_rows(&maps.b[i], o, o.b, o.Da));
    BT_TRY(map_rows(&maps.c[i], o, o.c, o.Dc));
  }
  int* err = nullptr;
  BT_TRY(operator_error_word(&err));
  const Op& o = ops.op[0];
  auto go = [&](auto size) -> int {
    constexpr int DA = decltype(size)::value;
    auto sums = chunk_tc_kernel<DA, false>;
    auto outs = chunk_tc_kernel<DA, true>;
    constexpr int kSmem = Cfg<DA>::kBytes;
    BT_CUDA(cudaFuncSetAttribute(outs, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    if (o.nsplit > 1) {
      BT_CUDA(cudaFuncSetAttribute(sums, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
      sums<<<dim3(blocks, o.nsplit - 1, ops.n), kThreads, kSmem, stream>>>(ops, maps, err);
      BT_LAUNCH_CHECK("linear attention split sums");
      BT_TRY(launch_join(ops, stream));
    }
    outs<<<dim3(blocks, o.nsplit, ops.n), kThreads, kSmem, stream>>>(ops, maps, err);
    BT_LAUNCH_CHECK("linear attention");
    return BT_OK;
  };
  if (da <= 64) return go(std::integral_constant<int, 64>{});
  return go(std::integral_constant<int, 128>{});
}

}  // namespace la
}  // namespace bt

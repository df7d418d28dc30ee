// Root-mean-square norms of the queries and keys of every head with the position rotation in the
// same pass, forward and backward.
//
//   n = x * r * w,  r = 1 / sqrt(mean(x^2) + eps)                       (per row of one head)
//   y = n with its pairs (n_a, n_b)_i turned by pos * f_i:  y_a = n_a cos - n_b sin,
//                                                           y_b = n_b cos + n_a sin
// backward, with xh = x r:  g = dy turned back, dw = sum over rows of g xh,
//   u = g w,  dx = r (u - xh mean(u xh)); r is formed again from x, which is read anyway.
//
// Bound by HBM: forward 2, backward 3 elements per element of x. A block takes a few tokens: it
// forms their cosines and sines once in shared memory (angle in 64 bits, reduced to one turn
// before the 32-bit sine, so far positions keep their phase), then a group of lanes takes one row
// (a token's query or key head) with 16-byte loads; the partner of an element, half a rotation
// away, comes through the group's row in shared memory. The weight gradients are summed per thread
// over the block's rows, over the block's groups in shared memory, and over the blocks by a second
// launch, each in a fixed order.
#include <type_traits>

#include "common.cuh"

namespace bt {
namespace rot {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 8;  // tokens of a block's pass
constexpr int kMaxDim = 256;

struct Rows {
  void* p;
  int64_t batch, step, head;
};

struct Args {
  Rows q, k, yq, yk;    // x and y, or x and dx
  Rows gq, gk;          // dy (backward)
  const void *wq, *wk;  // nullable: ones
  const int64_t* pos;
  int64_t pos_batch, pos_step;
  const double* freq;
  int64_t tokens;
  int steps, hq, hk, D, half;
  bool interleaved;
  float eps;
  int per;         // tokens of a pass
  float* partial;  // [blocks][2][D] (backward)
};

template <class T>
__device__ __forceinline__ float to_float(T x) {
  if constexpr (sizeof(T) == 2) return __bfloat162float(x);
  return x;
}
template <class T>
__device__ __forceinline__ T from_float(float x) {
  if constexpr (sizeof(T) == 2) return __float2bfloat16_rn(x);
  return x;
}

template <class T, int V>
__device__ __forceinline__ void load(const T* p, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = to_float(*p);
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = to_float(t[i]);
  }
}
template <class T, int V>
__device__ __forceinline__ void store(T* p, const float (&v)[V]) {
  if constexpr (V == 1) {
    *p = from_float<T>(v[0]);
  } else {
    uint4 u;
    T* t = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < V; ++i) t[i] = from_float<T>(v[i]);
    *reinterpret_cast<uint4*>(p) = u;
  }
}

// x[c][i] holds feature (c * G + lane) * V + i of the row. Turns it by the token's angles (sign 1),
// or back (-1); `row` is the group's staging row.
template <int V, int NC>
__device__ __forceinline__ void turn(const Args& a, float (&x)[NC][V], float* row, const float* cs,
                                     float sign, int lane, int G, bool on) {
  const int rd = 2 * a.half;
  if (V > 1 && a.interleaved && (rd % V) == 0) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int d = (c * G + lane) * V;
      if (!on || d >= rd) continue;
#pragma unroll
      for (int i = 0; i + 1 < V; i += 2) {
        const float co = cs[(d + i) >> 1], si = sign * cs[a.half + ((d + i) >> 1)];
        const float p = x[c][i], q = x[c][i + 1];
        x[c][i] = p * co - q * si;
        x[c][i + 1] = q * co + p * si;
      }
    }
    return;
  }
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int d = (c * G + lane) * V + i;
      if (d < rd) row[d] = x[c][i];
    }
  __syncwarp();
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int d = (c * G + lane) * V + i;
      if (d >= rd) continue;
      const int pair = a.interleaved ? d >> 1 : d % a.half;
      const bool second = a.interleaved ? d & 1 : d >= a.half;
      const float other = row[a.interleaved ? d ^ 1 : (second ? d - a.half : d + a.half)];
      const float co = cs[pair], si = sign * cs[a.half + pair];
      x[c][i] = second ? x[c][i] * co + other * si : x[c][i] * co - other * si;
    }
  __syncwarp();
}

template <class T, class W, int V, int NC, bool kBack>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const __grid_constant__ Args a, int G) {
  extern __shared__ float sm[];
  float* cs = sm;                                 // [per][2 half]
  float* rows = sm + a.per * 2 * a.half;          // [groups][D] staging rows
  const int lane = threadIdx.x % G, group = threadIdx.x / G, groups = kThreads / G;
  float* row = rows + group * a.D;
  const unsigned mask = G == 32 ? ~0u : ((1u << G) - 1u) << ((threadIdx.x & 31) / G * G);
  float w[2][NC][V], dw[kBack ? 2 : 1][NC][V];
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int d = (c * G + lane) * V + i;
      const bool in = d < a.D;
      w[0][c][i] = in && a.wq ? to_float(static_cast<const W*>(a.wq)[d]) : 1.f;
      w[1][c][i] = in && a.wk ? to_float(static_cast<const W*>(a.wk)[d]) : 1.f;
      if (kBack) dw[0][c][i] = dw[kBack ? 1 : 0][c][i] = 0.f;
    }
  const int H = a.hq + a.hk;
  const float inv = 1.f / (float)a.D;
  for (int64_t t0 = (int64_t)blockIdx.x * a.per; t0 < a.tokens; t0 += (int64_t)gridDim.x * a.per) {
    const int n = (int)min((int64_t)a.per, a.tokens - t0);
    __syncthreads();
    for (int e = threadIdx.x; e < n * a.half; e += kThreads) {
      const int64_t t = t0 + e / a.half;
      const double ang = (double)a.pos[t / a.steps * a.pos_batch + t % a.steps * a.pos_step] *
                         a.freq[e % a.half];
      // one turn: 2 pi as the sum of two doubles
      const double k = rint(ang * 0.15915494309189535);
      const double red = fma(-k, 2.4492935982947064e-16, fma(-k, 6.283185307179586, ang));
      float s, c;
      sincosf((float)red, &s, &c);
      cs[e / a.half * 2 * a.half + e % a.half] = c;
      cs[e / a.half * 2 * a.half + a.half + e % a.half] = s;
    }
    __syncthreads();
    // every group walks the same number of rows, so that its warp's shuffles meet
    for (int r0 = 0; r0 < n * H; r0 += groups) {
      const int r = r0 + group;
      const bool on = r < n * H;
      const int tok = on ? r / H : 0, h = on ? r % H : 0;
      const int64_t t = t0 + tok, b = t / a.steps, st = t % a.steps;
      const bool key = h >= a.hq;
      const int hh = key ? h - a.hq : h;
      const Rows& src = key ? a.k : a.q;
      const T* xp = static_cast<const T*>(src.p) + b * src.batch + st * src.step + hh * src.head;
      float x[NC][V], g[kBack ? NC : 1][V];
      float ss = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int d = (c * G + lane) * V;
        if (on && d < a.D) {
          load<T, V>(xp + d, x[c]);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) x[c][i] = 0.f;
        }
      }
      if constexpr (kBack) {
        const Rows& gs = key ? a.gk : a.gq;
        const T* gp = static_cast<const T*>(gs.p) + b * gs.batch + st * gs.step + hh * gs.head;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int d = (c * G + lane) * V;
          if (on && d < a.D) {
            load<T, V>(gp + d, g[c]);
          } else {
#pragma unroll
            for (int i = 0; i < V; ++i) g[c][i] = 0.f;
          }
        }
      }
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i) ss += x[c][i] * x[c][i];
      for (int o = G >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
      const float rs = rsqrtf(ss * inv + a.eps);
      const float* ct = cs + tok * 2 * a.half;
      if constexpr (!kBack) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int i = 0; i < V; ++i) x[c][i] *= rs * (key ? w[1][c][i] : w[0][c][i]);
        turn<V, NC>(a, x, row, ct, 1.f, lane, G, on);
      } else {
        turn<V, NC>(a, g, row, ct, -1.f, lane, G, on);
        float m = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            x[c][i] *= rs;
            const float p = on ? g[c][i] * x[c][i] : 0.f;
            if (key) dw[kBack ? 1 : 0][c][i] += p; else dw[0][c][i] += p;
            g[c][i] *= key ? w[1][c][i] : w[0][c][i];
            m += g[c][i] * x[c][i];
          }
        for (int o = G >> 1; o > 0; o >>= 1) m += __shfl_xor_sync(mask, m, o);
        m *= inv;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int i = 0; i < V; ++i) x[c][i] = rs * (g[c][i] - x[c][i] * m);
      }
      const Rows& dst = key ? a.yk : a.yq;
      T* yp = static_cast<T*>(dst.p) + b * dst.batch + st * dst.step + hh * dst.head;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int d = (c * G + lane) * V;
        if (on && d < a.D) store<T, V>(yp + d, x[c]);
      }
    }
  }
  if constexpr (kBack) {
    // the groups' sums, one after the other
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int d = (c * G + lane) * V + i;
          if (d < a.D) row[d] = which ? dw[kBack ? 1 : 0][c][i] : dw[0][c][i];
        }
      __syncthreads();
      for (int d = threadIdx.x; d < a.D; d += kThreads) {
        float s = 0.f;
        for (int u = 0; u < groups; ++u) s += rows[u * a.D + d];
        a.partial[((size_t)blockIdx.x * 2 + which) * a.D + d] = s;
      }
    }
  }
}

// dw[which][d] = sum over the blocks: one block per (which, 32 features), a warp's lanes on
// neighbouring features, its eight warps on every eighth partial.
template <class W>
__global__ void __launch_bounds__(256) weight_kernel(const float* partial, int blocks, int D, W* dwq, W* dwk) {
  __shared__ double part[8][33];
  const int which = blockIdx.y, d = blockIdx.x * 32 + (threadIdx.x & 31), warp = threadIdx.x >> 5;
  double s = 0.0;
  if (d < D)
    for (int b = warp; b < blocks; b += 8) s += (double)partial[((size_t)b * 2 + which) * D + d];
  part[warp][threadIdx.x & 31] = s;
  __syncthreads();
  W* to = which ? dwk : dwq;
  if (warp == 0 && d < D && to) {
    double t = 0.0;
    for (int u = 0; u < 8; ++u) t += part[u][threadIdx.x];
    to[d] = from_float<W>((float)t);
  }
}

// Blocks of the backward: its partial sums have one row for each.
int backward_blocks(int64_t tokens, int per) {
  const int64_t n = ceil_div64(tokens, per);
  return (int)(n < 4 * kNumSMs ? n : 4 * kNumSMs);
}

int tokens_per_pass(int64_t tokens, int rows) {
  // enough rows for every group of a block, but a block for every SM first
  int per = 1;
  while (per < kMaxTokens && per * rows < 64 && ceil_div64(tokens, per * 2) >= 2 * kNumSMs) per *= 2;
  return per;
}

struct Call {
  Args a;
  int dtype, wdtype;
  bool vec;
};

template <class T, class W, bool kBack>
int launch(const Call& c, int blocks, cudaStream_t s) {
  const Args& a = c.a;
  const int V = c.vec ? 16 / (int)sizeof(T) : 1;
  const int chunks = ceil_div(a.D, V);
  int G = 1;
  while (G < 32 && G < chunks) G *= 2;
  const int nc = ceil_div(chunks, G);
  const size_t smem = ((size_t)a.per * 2 * a.half + (size_t)(kThreads / G) * a.D) * 4;
  auto go = [&](auto vv, auto cc) -> int {
    constexpr int VV = decltype(vv)::value, CC = decltype(cc)::value;
    auto kernel = rotary_kernel<T, W, VV, CC, kBack>;
    if (smem > 48 * 1024)
      BT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    kernel<<<blocks, kThreads, smem, s>>>(a, G);
    BT_LAUNCH_CHECK("query/key norms with rotation");
    return BT_OK;
  };
  if (c.vec) {
    constexpr int VT = 16 / (int)sizeof(T);
    if (nc == 1) return go(std::integral_constant<int, VT>{}, std::integral_constant<int, 1>{});
    return go(std::integral_constant<int, VT>{}, std::integral_constant<int, 2>{});
  }
  return go(std::integral_constant<int, 1>{}, std::integral_constant<int, kMaxDim / 32>{});
}

template <bool kBack>
int dispatch(const Call& c, int blocks, cudaStream_t s) {
  if (c.dtype == BT_DTYPE_BF16)
    return c.wdtype == BT_DTYPE_BF16 ? launch<__nv_bfloat16, __nv_bfloat16, kBack>(c, blocks, s)
                                     : launch<__nv_bfloat16, float, kBack>(c, blocks, s);
  return c.wdtype == BT_DTYPE_BF16 ? launch<float, __nv_bfloat16, kBack>(c, blocks, s)
                                   : launch<float, float, kBack>(c, blocks, s);
}

int check(const bt_qk_norm_rotary_shape* s, const char* who) {
  BT_CHECK_ARG(s, "%s: null shape", who);
  BT_CHECK_ARG(s->batch >= 0 && s->steps >= 0 && s->q_heads >= 0 && s->k_heads >= 0, "%s: negative size", who);
  BT_CHECK_ARG(s->dim >= 1 && s->dim <= kMaxDim, "%s: heads of %d features (1 to %d are supported)", who,
               s->dim, kMaxDim);
  BT_CHECK_ARG(s->half >= 0 && 2 * s->half <= s->dim, "%s: %d frequencies for heads of %d features", who,
               s->half, s->dim);
  BT_CHECK_ARG((s->dtype == BT_DTYPE_F32 || s->dtype == BT_DTYPE_BF16) &&
                   (s->weight_dtype == BT_DTYPE_F32 || s->weight_dtype == BT_DTYPE_BF16),
               "%s: dtype %d, weight dtype %d", who, s->dtype, s->weight_dtype);
  BT_CHECK_ARG(s->q_heads + (int64_t)s->k_heads <= 65536, "%s: %d + %d heads", who, s->q_heads, s->k_heads);
  const bool some = (int64_t)s->batch * s->steps > 0;
  BT_CHECK_ARG(!some || ((s->positions || !s->half) && (s->frequencies || !s->half)), "%s: null positions or frequencies", who);
  return BT_OK;
}

Rows rows_of(const bt_heads* h) { return Rows{h->data, h->batch_stride, h->step_stride, h->head_stride}; }

bool aligned(const bt_heads* h, int heads, int esize) {
  if (heads == 0) return true;
  const int64_t m = 16 / esize;
  return ((uintptr_t)h->data & 15) == 0 && h->batch_stride % m == 0 && h->step_stride % m == 0 &&
         h->head_stride % m == 0;
}

Call call_of(const bt_qk_norm_rotary_shape* s, const bt_heads* q, const bt_heads* k, const void* wq,
             const void* wk, const bt_heads* yq, const bt_heads* yk) {
  Call c{};
  Args& a = c.a;
  a.q = rows_of(q);
  a.k = rows_of(k);
  a.yq = rows_of(yq);
  a.yk = rows_of(yk);
  a.wq = wq;
  a.wk = wk;
  a.pos = s->positions;
  a.pos_batch = s->positions_batch_stride;
  a.pos_step = s->positions_step_stride;
  a.freq = s->frequencies;
  a.tokens = (int64_t)s->batch * s->steps;
  a.steps = s->steps;
  a.hq = s->q_heads;
  a.hk = s->k_heads;
  a.D = s->dim;
  a.half = s->half;
  a.interleaved = s->interleaved != 0;
  a.eps = s->eps;
  a.per = tokens_per_pass(a.tokens, max(1, a.hq + a.hk));
  c.dtype = s->dtype;
  c.wdtype = s->weight_dtype;
  const int e = s->dtype == BT_DTYPE_BF16 ? 2 : 4;
  c.vec = (s->dim * e) % 16 == 0 && aligned(q, a.hq, e) && aligned(k, a.hk, e) && aligned(yq, a.hq, e) &&
          aligned(yk, a.hk, e);
  return c;
}

bool rows_ok(const bt_qk_norm_rotary_shape* s, const bt_heads* h, int heads) {
  return h && (h->data || (int64_t)s->batch * s->steps * heads == 0);
}

}  // namespace
}  // namespace rot
}  // namespace bt

using namespace bt;

extern "C" int bt_qk_norm_rotary(const bt_qk_norm_rotary_shape* s, const bt_heads* q, const bt_heads* k,
                                 const void* q_weight, const void* k_weight, const bt_heads* q_out,
                                 const bt_heads* k_out, void* stream) {
  BT_TRY(rot::check(s, "bt_qk_norm_rotary"));
  BT_CHECK_ARG(rot::rows_ok(s, q, s->q_heads) && rot::rows_ok(s, k, s->k_heads) &&
                   rot::rows_ok(s, q_out, s->q_heads) && rot::rows_ok(s, k_out, s->k_heads),
               "bt_qk_norm_rotary: null pointer");
  const rot::Call c = rot::call_of(s, q, k, q_weight, k_weight, q_out, k_out);
  if (c.a.tokens == 0 || c.a.hq + c.a.hk == 0) return BT_OK;
  const int64_t n = ceil_div64(c.a.tokens, c.a.per);
  return rot::dispatch<false>(c, (int)(n < 65535 * 16 ? n : 65535 * 16), (cudaStream_t)stream);
}

extern "C" int64_t bt_qk_norm_rotary_workspace(const bt_qk_norm_rotary_shape* s) {
  if (rot::check(s, "bt_qk_norm_rotary_workspace") != BT_OK) return -1;
  const int64_t tokens = (int64_t)s->batch * s->steps;
  const int per = rot::tokens_per_pass(tokens, max(1, s->q_heads + s->k_heads));
  return (int64_t)rot::backward_blocks(tokens, per) * 2 * s->dim * 4;
}

extern "C" int bt_qk_norm_rotary_backward(const bt_qk_norm_rotary_shape* s, const bt_heads* q,
                                          const bt_heads* k, const void* q_weight,
                                          const void* k_weight, const bt_heads* dq_out,
                                          const bt_heads* dk_out, const bt_heads* dq,
                                          const bt_heads* dk, void* dq_weight, void* dk_weight,
                                          void* workspace, int64_t workspace_bytes, void* stream) {
  BT_TRY(rot::check(s, "bt_qk_norm_rotary_backward"));
  BT_CHECK_ARG(rot::rows_ok(s, q, s->q_heads) && rot::rows_ok(s, k, s->k_heads) &&
                   rot::rows_ok(s, dq_out, s->q_heads) && rot::rows_ok(s, dk_out, s->k_heads) &&
                   rot::rows_ok(s, dq, s->q_heads) && rot::rows_ok(s, dk, s->k_heads),
               "bt_qk_norm_rotary_backward: null pointer");
  rot::Call c = rot::call_of(s, q, k, q_weight, k_weight, dq, dk);
  const int e = s->dtype == BT_DTYPE_BF16 ? 2 : 4;
  c.a.gq = rot::rows_of(dq_out);
  c.a.gk = rot::rows_of(dk_out);
  c.vec = c.vec && rot::aligned(dq_out, c.a.hq, e) && rot::aligned(dk_out, c.a.hk, e);
  const int blocks = rot::backward_blocks(c.a.tokens, c.a.per);
  const int64_t need = (int64_t)blocks * 2 * s->dim * 4;
  BT_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need),
               "bt_qk_norm_rotary_backward: workspace of %lld bytes, %lld needed",
               (long long)workspace_bytes, (long long)need);
  c.a.partial = static_cast<float*>(workspace);
  if (blocks > 0) BT_TRY(rot::dispatch<true>(c, blocks, (cudaStream_t)stream));
  if (dq_weight || dk_weight) {
    const dim3 grid(ceil_div(s->dim, 32), 2);
    if (s->weight_dtype == BT_DTYPE_BF16)
      rot::weight_kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(
          c.a.partial, blocks, s->dim, static_cast<__nv_bfloat16*>(dq_weight), static_cast<__nv_bfloat16*>(dk_weight));
    else
      rot::weight_kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(
          c.a.partial, blocks, s->dim, static_cast<float*>(dq_weight), static_cast<float*>(dk_weight));
    BT_LAUNCH_CHECK("query/key norm weight gradients");
  }
  return BT_OK;
}

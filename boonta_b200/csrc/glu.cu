// The gated feed-forward layer on CUDA cores, and the C entry points.
//
//   forward   h = act(G) * U,                      G = x Wg, U = x Wu
//   backward  G, U formed again tile by tile;  dG = dh U act'(G), dU = dh act(G);
//             dx = dG Wg^T + dU Wu^T,  dWg = x^T dG,  dWu = x^T dU
//
// Tiles of 64 x 64 outputs, 16 deep, 256 threads with 4 x 4 outputs each (of both projections),
// everything in fp32.
#include <type_traits>

#include "glu.cuh"

namespace bt {
namespace glu {
namespace {

constexpr int kTile = 64, kDepth = 16, kThreads = 256;

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

// A tile [kDepth][kTile] of an operand (index i along the output, k along the contraction).
template <class T>
__device__ __forceinline__ void load_tile(const T* p, int64_t si, int64_t sk, int i0, int k0, int I,
                                          int K, float (&to)[kDepth][kTile + 4]) {
  for (int e = threadIdx.x; e < kDepth * kTile; e += kThreads) {
    const int i = si == 1 ? e % kTile : e / kDepth, k = si == 1 ? e / kTile : e % kDepth;
    to[k][i] = i0 + i < I && k0 + k < K ? to_float(p[(i0 + i) * si + (k0 + k) * sk]) : 0.f;
  }
}

__device__ __forceinline__ void add_product(const float (&a)[kDepth][kTile + 4],
                                            const float (&b)[kDepth][kTile + 4], float (&acc)[4][4]) {
  const int r = (threadIdx.x >> 4) * 4, c = (threadIdx.x & 15) * 4;
#pragma unroll
  for (int k = 0; k < kDepth; ++k) {
    const float4 x = *reinterpret_cast<const float4*>(&a[k][r]);
    const float4 y = *reinterpret_cast<const float4*>(&b[k][c]);
    const float xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] += xs[i] * ys[j];
  }
}

enum Mode { kForward, kGrads, kInput, kWeights };

struct Args {
  Layer l;
  void *o1, *o2;  // h; dG, dU; dx; dWg, dWu
  const void *dg, *du;
};

// kForward / kGrads: [M, N] from x with both weights. kInput: dx [M, K] from dG, Wg and dU, Wu.
// kWeights: dWg, dWu [K, N] from x with dG and dU.
template <class T, Mode kMode>
__global__ void __launch_bounds__(kThreads) simt_kernel(const Args a) {
  __shared__ __align__(16) float sa[kDepth][kTile + 4], sb[2][kDepth][kTile + 4];
  const Layer& l = a.l;
  const int I = kMode == kWeights ? l.K : l.M, J = kMode == kInput ? l.K : l.N;
  const int C = kMode == kWeights ? l.M : kMode == kInput ? l.N : l.K;
  const int jt = ceil_div(J, kTile);
  const int i0 = (int)(blockIdx.x / jt) * kTile, j0 = (int)(blockIdx.x % jt) * kTile;
  const T *x = static_cast<const T*>(l.x), *wg = static_cast<const T*>(l.wg), *wu = static_cast<const T*>(l.wu);
  const T *dg = static_cast<const T*>(a.dg), *du = static_cast<const T*>(a.du);
  float acc[2][4][4] = {};
  for (int k0 = 0; k0 < C; k0 += kDepth) {
    if constexpr (kMode == kInput) {
      for (int p = 0; p < 2; ++p) {
        __syncthreads();
        load_tile(p ? du : dg, (int64_t)l.N, (int64_t)1, i0, k0, I, C, sa);
        load_tile(p ? wu : wg, l.ldw, (int64_t)1, j0, k0, J, C, sb[0]);
        __syncthreads();
        add_product(sa, sb[0], acc[0]);
      }
    } else {
      __syncthreads();
      if constexpr (kMode == kWeights) {
        load_tile(x, (int64_t)1, l.ldx, i0, k0, I, C, sa);
        load_tile(dg, (int64_t)1, (int64_t)l.N, j0, k0, J, C, sb[0]);
        load_tile(du, (int64_t)1, (int64_t)l.N, j0, k0, J, C, sb[1]);
      } else {
        load_tile(x, l.ldx, (int64_t)1, i0, k0, I, C, sa);
        load_tile(wg, (int64_t)1, l.ldw, j0, k0, J, C, sb[0]);
        load_tile(wu, (int64_t)1, l.ldw, j0, k0, J, C, sb[1]);
      }
      __syncthreads();
      add_product(sa, sb[0], acc[0]);
      add_product(sa, sb[1], acc[1]);
    }
  }
  T *o1 = static_cast<T*>(a.o1), *o2 = static_cast<T*>(a.o2);
  const int r = i0 + (threadIdx.x >> 4) * 4, c = j0 + (threadIdx.x & 15) * 4;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (r + i >= I || c + j >= J) continue;
      const size_t at = (size_t)(r + i) * J + c + j;
      const float g = acc[0][i][j], u = acc[1][i][j];
      if constexpr (kMode == kForward) {
        o1[at] = from_float<T>(act_forward(g, l.act) * u);
      } else if constexpr (kMode == kGrads) {
        const float dh = to_float(static_cast<const T*>(l.dh)[(r + i) * l.lddh + c + j]);
        o1[at] = from_float<T>(dh * u * act_grad(g, act_forward(g, l.act), l.act));
        o2[at] = from_float<T>(dh * act_forward(g, l.act));
      } else {
        o1[at] = from_float<T>(g);
        if constexpr (kMode == kWeights) o2[at] = from_float<T>(u);
      }
    }
}

template <class T, Mode kMode>
int run(const Args& a, cudaStream_t s) {
  const int I = kMode == kWeights ? a.l.K : a.l.M, J = kMode == kInput ? a.l.K : a.l.N;
  if (I == 0 || J == 0) return BT_OK;
  const int64_t tiles = (int64_t)ceil_div(I, kTile) * ceil_div(J, kTile);
  simt_kernel<T, kMode><<<(unsigned)tiles, kThreads, 0, s>>>(a);
  BT_LAUNCH_CHECK("gated layer");
  return BT_OK;
}

template <class T>
int backward(const Layer& l, void* dg, void* du, void* dx, void* dwg, void* dwu, cudaStream_t s) {
  Args a{l, dg, du, dg, du};
  BT_TRY((run<T, kGrads>(a, s)));
  if (dx) {
    a.o1 = dx;
    BT_TRY((run<T, kInput>(a, s)));
  }
  if (dwg) {
    a.o1 = dwg;
    a.o2 = dwu;
    BT_TRY((run<T, kWeights>(a, s)));
  }
  return BT_OK;
}

int check(const bt_glu_shape* s, const char* who) {
  BT_CHECK_ARG(s, "%s: null shape", who);
  BT_CHECK_ARG(s->rows >= 0 && s->in_features >= 1 && s->out_features >= 1, "%s: %d rows, %d to %d features",
               who, s->rows, s->in_features, s->out_features);
  BT_CHECK_ARG(s->dtype == BT_DTYPE_F32 || s->dtype == BT_DTYPE_BF16, "%s: dtype %d", who, s->dtype);
  BT_CHECK_ARG(s->activation >= BT_ACT_NONE && s->activation <= BT_ACT_SILU, "%s: activation %d", who,
               s->activation);
  BT_CHECK_ARG((int64_t)ceil_div(s->rows, kTile) * ceil_div(max(s->in_features, s->out_features), kTile) < (1ll << 31),
               "%s: too many tiles", who);
  return BT_OK;
}

}  // namespace
}  // namespace glu
}  // namespace bt

using namespace bt;

extern "C" int64_t bt_glu_workspace(const bt_glu_shape* s, int32_t backward) {
  if (glu::check(s, "bt_glu_workspace") != BT_OK) return -1;
  const int64_t e = s->dtype == BT_DTYPE_BF16 ? 2 : 4;
  return backward ? 2 * (((int64_t)s->rows * s->out_features * e + 255) / 256 * 256) : 0;
}

extern "C" int bt_glu(const bt_glu_shape* s, const void* x, const void* w_gate, const void* w_up,
                      void* out, void* workspace, int64_t workspace_bytes, void* stream) {
  BT_TRY(glu::check(s, "bt_glu"));
  (void)workspace;
  (void)workspace_bytes;
  if (s->rows == 0) return BT_OK;
  BT_CHECK_ARG(x && w_gate && w_up && out, "bt_glu: null pointer");
  const glu::Layer l{s->rows, s->out_features, s->in_features, s->activation, x, w_gate, w_up, nullptr,
                     s->in_features, s->out_features, s->out_features};
  const glu::Args a{l, out, nullptr, nullptr, nullptr};
  return s->dtype == BT_DTYPE_BF16 ? glu::run<__nv_bfloat16, glu::kForward>(a, (cudaStream_t)stream)
                                   : glu::run<float, glu::kForward>(a, (cudaStream_t)stream);
}

extern "C" int bt_glu_backward(const bt_glu_shape* s, const void* x, const void* w_gate,
                               const void* w_up, const void* dout, void* dx, void* dw_gate,
                               void* dw_up, void* workspace, int64_t workspace_bytes, void* stream) {
  BT_TRY(glu::check(s, "bt_glu_backward"));
  BT_CHECK_ARG((dw_gate == nullptr) == (dw_up == nullptr), "bt_glu_backward: one of dw_gate and dw_up is null");
  BT_CHECK_ARG(s->rows == 0 || (x && w_gate && w_up && dout), "bt_glu_backward: null pointer");
  const int64_t need = bt_glu_workspace(s, 1);
  BT_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need),
               "bt_glu_backward: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
               (long long)need);
  const glu::Layer l{s->rows, s->out_features, s->in_features, s->activation, x, w_gate, w_up, dout,
                     s->in_features, s->out_features, s->out_features};
  char* w = static_cast<char*>(workspace);
  void *dg = w, *du = w + need / 2;
  return s->dtype == BT_DTYPE_BF16
             ? glu::backward<__nv_bfloat16>(l, dg, du, dx, dw_gate, dw_up, (cudaStream_t)stream)
             : glu::backward<float>(l, dg, du, dx, dw_gate, dw_up, (cudaStream_t)stream);
}

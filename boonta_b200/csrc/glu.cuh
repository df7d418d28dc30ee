// The gated feed-forward layer h = act(x Wg) * (x Wu): what its files share.
#pragma once

#include "common.cuh"

namespace bt {
namespace glu {

// One gated layer: x [M, K], Wg and Wu [K, N], dh [M, N], row-major without gaps.
struct Layer {
  int M, N, K, act;
  const void *x, *wg, *wu, *dh;
};

// The activation of a gate and its slope. relu as the other ones: a gate that is not a number is not closed by it.
template <int A>
__device__ __forceinline__ float gate_act(float g) {
  if constexpr (A == BT_ACT_RELU) return g <= 0.f ? 0.f : g;
  return act_fwd<A>(g);
}
template <int A>
__device__ __forceinline__ float gate_slope(float g) {
  if constexpr (A == BT_ACT_RELU) return g <= 0.f ? 0.f : g == g ? 1.f : g;
  return act_dz<A>(g);
}

// The gradients of gate and up projection from their values: dg = dh u act'(g), du = dh act(g).
template <int A>
__device__ __forceinline__ void gate_grads(float g, float u, float dh, float& dg, float& du) {
  dg = dh * u * gate_slope<A>(g);
  du = dh * gate_act<A>(g);
}

// Tensor cores (glu_sm100.cu). ws: workspace_of bytes.
int64_t workspace_of(const Layer& l, bool f32, bool backward);
int forward(const Layer& l, bool f32, void* h, char* ws, cudaStream_t s);
int backward(const Layer& l, bool f32, void* dx, void* dwg, void* dwu, char* ws, cudaStream_t s);

}  // namespace glu
}  // namespace bt

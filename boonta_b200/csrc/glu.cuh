// The gated feed-forward layer h = act(x Wg) * (x Wu): what its kernels share.
#pragma once

#include "common.cuh"

namespace bt {
namespace glu {

// One gated layer: x [M, K], Wg and Wu [K, N], h and dh [M, N], row-major.
struct Layer {
  int M, N, K, act;
  const void *x, *wg, *wu, *dh;
  int64_t ldx, ldw, lddh;
};

// The gradients of gate and up projection from their values: dg = dh u act'(g), du = dh act(g).
template <int A>
__device__ __forceinline__ void gate_grads(float g, float u, float dh, float& dg, float& du) {
  dg = dh * u * act_dz<A>(g);
  du = dh * act_fwd<A>(g);
}

}  // namespace glu
}  // namespace bt

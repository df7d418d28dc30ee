// Linear attention with a decay per head: the operation its forward and backward passes share.
//
//   S_t = [not cut_t] e^{g_h} S_{t-1} + in_scale b_t c_t^T,    out_t = out_scale S_t^T a_t
//
// over the steps of one (batch row, head), taken first to last or last to first. With
// (a, b, c) = (q, k, v) forwards this is the attention itself. Its gradients are the same
// operation: dq takes (dout, v, k) forwards with the state transposed; dv takes (k, q, dout) and
// dk takes (v, dout, q) backwards, both on the reversed state R_t = scale q_t dout_t^T +
// [not reset_{t+1}] e^g R_{t+1} (dk on its transpose), which starts from the gradient of the
// final state and ends as the gradient of the initial one.
//
// Position i counts steps in the order taken. cut(i) is reset[t] forwards and reset[t + 1]
// backwards (there is none before the last step), and the state given at the start decays once
// before position 0 forwards, not at all backwards; backwards the final state decays once more
// (and is cut by reset[0]) on its way out.
#pragma once

#include "common.cuh"

namespace bt {
namespace la {

struct Rows {  // [batch, steps, heads, features], features contiguous; strides in elements
  const void* p;
  int64_t batch, step, head;
};

struct Op {
  Rows a, b, c;
  void* out;
  int64_t out_batch, out_step, out_head;
  const float* init;  // [batch * heads][Da * Dc], element (x, y) at x * sx + y * sy; null: zeros
  float* fin;         // the same layout; null: not wanted
  int sx, sy;
  const float* log_decay;  // [heads]
  const uint8_t* reset;    // nullable
  int64_t reset_batch, reset_step;
  int batch, steps, heads, Da, Dc;
  float in_scale, out_scale;
  bool reverse;
  // splits of the steps: `local` [nsplit - 1][batch * heads][Da * Dc] holds the own sum of each split but the
  // last, then the state that enters the split after it; `cut` [nsplit - 1][batch] whether a split has a cut
  int nsplit, split_len;
  float* local;
  int* cut;
};

struct Ops {  // one launch's operations, of the same sequences
  Op op[3];
  int n;
};

// bf16 on the tensor cores (linear_attention_sm100.cu): where every row starts on a 16-byte boundary and the
// output's rows end on one.
bool suits_tensor_cores(const Op& o);
int run_tensor_cores(Ops& ops, cudaStream_t stream);
// Turns the splits' own sums into the states that enter the splits (linear_attention.cu).
int launch_join(const Ops& ops, cudaStream_t stream);

// A log decay below this has e^{n g} = 0 for n >= 1 and keeps e^{0 g} = 1 (an infinite one
// would give 0 * inf).
constexpr float kMinLogDecay = -1e4f;

__device__ __forceinline__ float clamped_decay(float g) { return g < kMinLogDecay ? kMinLogDecay : g; }

__device__ __forceinline__ int op_time(const Op& o, int i) { return o.reverse ? o.steps - 1 - i : i; }

// Whether the state is cleared before position i.
__device__ __forceinline__ bool op_cut(const Op& o, int b, int i) {
  if (o.reset == nullptr || i >= o.steps) return false;
  const int t = o.reverse ? o.steps - i : i;
  if (t >= o.steps) return false;
  return o.reset[b * o.reset_batch + t * o.reset_step] != 0;
}

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

}  // namespace la
}  // namespace bt

// C entry points of the gated feed-forward layer (the kernels: glu_sm100.cu).
#include "glu.cuh"

namespace bt {
namespace glu {
namespace {

int check(const bt_glu_shape* s, const char* who) {
  BT_CHECK_ARG(s, "%s: null shape", who);
  BT_CHECK_ARG(s->rows >= 0 && s->in_features >= 1 && s->out_features >= 1, "%s: %d rows, %d to %d features",
               who, s->rows, s->in_features, s->out_features);
  BT_CHECK_ARG(s->in_features <= (1 << 20) && s->out_features <= (1 << 20) && s->rows <= (1 << 28),
               "%s: %d rows, %d to %d features: too many", who, s->rows, s->in_features, s->out_features);
  BT_CHECK_ARG(s->dtype == BT_DTYPE_F32 || s->dtype == BT_DTYPE_BF16, "%s: dtype %d", who, s->dtype);
  BT_CHECK_ARG(s->activation >= BT_ACT_NONE && s->activation <= BT_ACT_SILU, "%s: activation %d", who,
               s->activation);
  return BT_OK;
}

bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

Layer layer_of(const bt_glu_shape* s, const void* x, const void* wg, const void* wu, const void* dh) {
  return Layer{s->rows, s->out_features, s->in_features, s->activation, x, wg, wu, dh};
}

}  // namespace
}  // namespace glu
}  // namespace bt

using namespace bt;

extern "C" int64_t bt_glu_workspace(const bt_glu_shape* s, int32_t backward) {
  if (glu::check(s, "bt_glu_workspace") != BT_OK) return -1;
  if (s->rows == 0) return 0;
  return glu::workspace_of(glu::layer_of(s, nullptr, nullptr, nullptr, nullptr), s->dtype == BT_DTYPE_F32,
                           backward != 0);
}

extern "C" int bt_glu(const bt_glu_shape* s, const void* x, const void* w_gate, const void* w_up,
                      void* out, void* workspace, int64_t workspace_bytes, void* stream) {
  BT_TRY(glu::check(s, "bt_glu"));
  if (s->rows == 0) return BT_OK;
  BT_CHECK_ARG(x && w_gate && w_up && out, "bt_glu: null pointer");
  BT_CHECK_ARG(glu::aligned(x) && glu::aligned(w_gate) && glu::aligned(w_up) && glu::aligned(out) &&
                   glu::aligned(workspace),
               "bt_glu: a pointer is not 16-byte aligned");
  const int64_t need = bt_glu_workspace(s, 0);
  BT_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need), "bt_glu: workspace of %lld bytes, %lld needed",
               (long long)workspace_bytes, (long long)need);
  return glu::forward(glu::layer_of(s, x, w_gate, w_up, nullptr), s->dtype == BT_DTYPE_F32, out,
                      static_cast<char*>(workspace), (cudaStream_t)stream);
}

extern "C" int bt_glu_backward(const bt_glu_shape* s, const void* x, const void* w_gate,
                               const void* w_up, const void* dout, void* dx, void* dw_gate,
                               void* dw_up, void* workspace, int64_t workspace_bytes, void* stream) {
  BT_TRY(glu::check(s, "bt_glu_backward"));
  BT_CHECK_ARG((dw_gate == nullptr) == (dw_up == nullptr), "bt_glu_backward: one of dw_gate and dw_up is null");
  if (s->rows == 0) {
    const size_t bytes = (size_t)s->in_features * s->out_features * (s->dtype == BT_DTYPE_F32 ? 4 : 2);
    if (dw_gate) {
      BT_CUDA(cudaMemsetAsync(dw_gate, 0, bytes, (cudaStream_t)stream));
      BT_CUDA(cudaMemsetAsync(dw_up, 0, bytes, (cudaStream_t)stream));
    }
    return BT_OK;
  }
  BT_CHECK_ARG(x && w_gate && w_up && dout, "bt_glu_backward: null pointer");
  BT_CHECK_ARG(glu::aligned(x) && glu::aligned(w_gate) && glu::aligned(w_up) && glu::aligned(dout) &&
                   glu::aligned(dx) && glu::aligned(dw_gate) && glu::aligned(dw_up) && glu::aligned(workspace),
               "bt_glu_backward: a pointer is not 16-byte aligned");
  const int64_t need = bt_glu_workspace(s, 1);
  BT_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need),
               "bt_glu_backward: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
               (long long)need);
  return glu::backward(glu::layer_of(s, x, w_gate, w_up, dout), s->dtype == BT_DTYPE_F32, dx, dw_gate, dw_up,
                       static_cast<char*>(workspace), (cudaStream_t)stream);
}

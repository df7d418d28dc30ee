// Linear attention with a decay per head on CUDA cores, its splits along the steps, the
// single-step form, and the C entry points (the operation: linear_attention.cuh).
//
// Chunked form, 32 positions at a time, everything in fp32:
//   P = (a b^T) * e^{(i - j) g} on and below the diagonal, 0 across a cut
//   out = out_scale (in_scale P c + e^{(i + e0) g} a S)      rows before the chunk's first cut
//   S = e^{(n - 1 + e0) g} S + in_scale sum_j e^{(n - 1 - j) g} b_j c_j^T
// A block owns one (batch row, head) and DS columns of c; the state stays in shared memory for the
// block's whole walk. It serves float32, and bf16 whose rows do not start (outputs: and end) on 16-byte boundaries. A row
// takes only the columns from its last cut to itself, so what a cut or the future hides is not read, whatever
// it holds. Bound by the latency of the walk where sequences are few: blocks of 16 columns then, four times
// as many, each a third as long (48 x 100 x 3 x 48 float32, forward: 83 us with 64 columns, 47 with 16). Where they
// are many it is bound by its products: 512 x 128 x 4 x 64 float32 forward 502 us, training pass 1978 (8.6 and 6.5 TFLOP/s);
// bf16 with 60 features 743 and 2652, where 64 take 53 and 174 on the tensor cores.
// Sequences too few to fill the GPU are split along the steps: a first
// launch sums each split from an empty state, a second joins the sums into the states that enter
// the splits (S_{s+1} = e^{len g} S_s + local_s), a third runs the splits from those.
#include <type_traits>

#include "launch.cuh"
#include "linear_attention.cuh"

namespace bt {
namespace la {
namespace {

constexpr int kC = 32;       // positions of a chunk
constexpr int kThreads = 256;
constexpr int kWide = 64, kNarrow = 16;  // columns of c (and of the state) of a block

template <int DA, int DS>
struct Smem {
  float a[kC][DA + 4], b[kC][DA + 4], c[kC][DS + 4], s[DA][DS + 4], p[kC][kC + 1];
  float pw[kC + 2], pl[kC + 2];  // e^{i g} and what its rounding left
  int first[kC];                 // of a row: the first position of its own stretch between cuts
};

template <class T, int W>
__device__ __forceinline__ void load_rows(const Op& o, const Rows& r, int batch, int head, int i0, int n, int d0, int d,
                                          float* dst, int ld, bool vec) {
  const T* p = static_cast<const T*>(r.p) + batch * r.batch + head * r.head + d0;
  if (sizeof(T) == 4 && vec) {  // rows on 16-byte boundaries, a multiple of 4 columns
#pragma unroll
    for (int e = threadIdx.x; e < kC * W / 4; e += kThreads) {
      const int i = e / (W / 4), x = e % (W / 4) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < n && d0 + x < d) v = *reinterpret_cast<const float4*>(p + (int64_t)op_time(o, i0 + i) * r.step + x);
      *reinterpret_cast<float4*>(dst + i * ld + x) = v;
    }
    return;
  }
#pragma unroll 8
  for (int e = threadIdx.x; e < kC * W; e += kThreads) {
    const int i = e / W, x = e % W;
    float v = 0.f;
    if (i < n && d0 + x < d) v = to_float(p[(int64_t)op_time(o, i0 + i) * r.step + x]);
    dst[i * ld + x] = v;
  }
}

// kOut: outputs and (split s) from the state that enters the split; else the split's own sum.
template <class T, int DA, int DS, bool kOut>
__global__ void __launch_bounds__(kThreads) chunk_kernel(const __grid_constant__ Ops ops, bool vec) {
  const Op& o = ops.op[blockIdx.z];
  extern __shared__ __align__(16) uint8_t raw[];
  Smem<DA, DS>& sm = *reinterpret_cast<Smem<DA, DS>*>(raw);
  const int slices = ceil_div(o.Dc, DS);
  if ((int)blockIdx.x >= o.batch * o.heads * slices) return;
  const int bh = blockIdx.x / slices, d0 = blockIdx.x % slices * DS;
  const int batch = bh / o.heads, head = bh % o.heads;
  const int split = blockIdx.y;
  const int begin = split * o.split_len, end = min(o.steps, begin + o.split_len);
  const int tid = threadIdx.x;
  const float g = clamped_decay(o.log_decay[head]);
  const int DcV = min(DS, o.Dc - d0);
  const size_t elems = (size_t)o.Da * o.Dc;

  const float* from = nullptr;
  int sx = o.sx, sy = o.sy;
  if (kOut) {
    if (split > 0) {
      from = o.local + ((size_t)(split - 1) * o.batch * o.heads + bh) * elems;
      sx = o.Dc;
      sy = 1;
    } else if (o.init) {
      from = o.init + bh * elems;
    }
  }
#pragma unroll 4
  for (int e = tid; e < DA * DS; e += kThreads) {
    // neighbouring threads along the state's own rows
    const int x = sy == 1 ? e / DS : e % DA, y = sy == 1 ? e % DS : e / DA;
    sm.s[x][y] = from && x < o.Da && y < DcV ? from[(size_t)x * sx + (size_t)(d0 + y) * sy] : 0.f;
  }
  if (tid < kC + 2) {
    const double e = exp((double)tid * (double)g);
    sm.pw[tid] = (float)e;
    sm.pl[tid] = (float)(e - (double)(float)e);
  }
  bool any_cut = false;
  // decays that the entering state meets before position `begin`
  int e0 = (o.reverse && split == 0) ? 0 : 1;

  for (int i0 = begin; i0 < end; i0 += kC) {
    const int n = min(kC, end - i0);
    __syncthreads();
    if (kOut) load_rows<T, DA>(o, o.a, batch, head, i0, n, 0, o.Da, &sm.a[0][0], DA + 4, vec);
    load_rows<T, DA>(o, o.b, batch, head, i0, n, 0, o.Da, &sm.b[0][0], DA + 4, vec);
    load_rows<T, DS>(o, o.c, batch, head, i0, n, d0, o.Dc, &sm.c[0][0], DS + 4, vec);
    if (tid < kC) {
      const unsigned m = __ballot_sync(~0u, tid < n && op_cut(o, batch, i0 + tid));
      const unsigned own = m & (~0u >> (31 - tid));
      sm.first[tid] = own ? 31 - __clz(own) : -1;
    }
    __syncthreads();
    const int last = sm.first[kC - 1];  // the chunk's last cut; what comes before it leaves nothing
    any_cut |= last >= 0;

    if (kOut) {
      {  // P: row i = tid / 8, columns tid % 8 + 8 m
        const int i = tid >> 3, j0 = tid & 7;
        float acc[4] = {};
#pragma unroll 4
        for (int k = 0; k < DA; k += 4) {
          const float4 x = *reinterpret_cast<const float4*>(&sm.a[i][k]);
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const float4 y = *reinterpret_cast<const float4*>(&sm.b[j0 + 8 * m][k]);
            acc[m] += x.x * y.x + x.y * y.y + x.z * y.z + x.w * y.w;
          }
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          const int j = j0 + 8 * m;
          sm.p[i][j] = j <= i && j >= sm.first[i] ? acc[m] * sm.pw[i - j] * o.in_scale : 0.f;
        }
      }
      __syncthreads();
      // out: row i = tid / 8, columns DS / 8 of them
      constexpr int kW = DS / 8;
      const int i = tid >> 3, y = (tid & 7) * kW;
      float acc[kW] = {}, st[kW] = {};
      const int first = sm.first[i];
      for (int j = max(first, 0); j <= i; ++j) {
        const float p = sm.p[i][j];
#pragma unroll
        for (int w = 0; w < kW; ++w) acc[w] += p * sm.c[j][y + w];
      }
      if (first < 0) {
#pragma unroll 4
        for (int k = 0; k < DA; k += 4) {
          const float4 x = *reinterpret_cast<const float4*>(&sm.a[i][k]);
          const float xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int v = 0; v < 4; ++v)
#pragma unroll
            for (int w = 0; w < kW; ++w) st[w] += xs[v] * sm.s[k + v][y + w];
        }
        const float reach = sm.pw[i + e0];
#pragma unroll
        for (int w = 0; w < kW; ++w) acc[w] += reach != 0.f ? reach * st[w] : 0.f;
      }
      if (i < n) {
        T* out = static_cast<T*>(o.out) + batch * o.out_batch + (int64_t)op_time(o, i0 + i) * o.out_step +
                 head * o.out_head + d0 + y;
#pragma unroll
        for (int w = 0; w < kW; ++w)
          if (y + w < DcV) out[w] = from_float<T>(acc[w] * o.out_scale);
      }
      __syncthreads();
    }
    {  // state: kR rows, four columns
      constexpr int kCols = DS / 4, kR = DA * kCols / kThreads;
      const int x0 = tid / kCols * kR, y = tid % kCols * 4;
      // the same factor meets the state once a chunk, so its rounding would add up over a long
      // memory: two parts leave only the roundings of the sums, which do not lean one way
      const float keep = sm.pw[n - 1 + e0], keep_lo = sm.pl[n - 1 + e0];
      float acc[kR][4];
#pragma unroll
      for (int u = 0; u < kR; ++u)
#pragma unroll
        for (int w = 0; w < 4; ++w)
          acc[u][w] = last < 0 ? fmaf(keep, sm.s[x0 + u][y + w], keep_lo * sm.s[x0 + u][y + w]) : 0.f;
#pragma unroll 4
      for (int j = max(last, 0); j < n; ++j) {
        const float wj = sm.pw[n - 1 - j] * o.in_scale;
        const float4 c = *reinterpret_cast<const float4*>(&sm.c[j][y]);
        const float4 wc = make_float4(c.x * wj, c.y * wj, c.z * wj, c.w * wj);
#pragma unroll
        for (int u = 0; u < kR; ++u) {
          const float b = sm.b[j][x0 + u];
          acc[u][0] += b * wc.x;
          acc[u][1] += b * wc.y;
          acc[u][2] += b * wc.z;
          acc[u][3] += b * wc.w;
        }
      }
#pragma unroll
      for (int u = 0; u < kR; ++u)
        *reinterpret_cast<float4*>(&sm.s[x0 + u][y]) =
            make_float4(acc[u][0], acc[u][1], acc[u][2], acc[u][3]);
    }
    e0 = 1;
  }
  __syncthreads();
  float* to = nullptr;
  float way_out = 1.f;
  if (kOut) {
    if (o.fin && split == o.nsplit - 1) {
      to = o.fin + bh * elems;
      sx = o.sx;
      sy = o.sy;
      // backwards: the way out of position steps - 1 passes reset[0] and one decay
      if (o.reverse && o.steps > 0) {
        way_out = sm.pw[1];
        if (o.reset && o.reset[batch * o.reset_batch]) way_out = 0.f;
      }
    }
  } else {
    to = o.local + ((size_t)split * o.batch * o.heads + bh) * elems;
    sx = o.Dc;
    sy = 1;
    if (tid == 0 && d0 == 0 && head == 0) o.cut[split * o.batch + batch] = any_cut;
  }
  if (to) {
#pragma unroll 4
    for (int e = tid; e < DA * DS; e += kThreads) {
      const int x = sy == 1 ? e / DS : e % DA, y = sy == 1 ? e % DS : e / DA;
      if (x < o.Da && y < DcV)
        to[(size_t)x * sx + (size_t)(d0 + y) * sy] = way_out == 0.f ? 0.f : way_out * sm.s[x][y];
    }
  }
}

// local[s], the own sum of split s < nsplit - 1, becomes the state that enters split s + 1.
__global__ void join_kernel(const __grid_constant__ Ops ops) {
  const Op& o = ops.op[blockIdx.y];
  const int64_t elems = (int64_t)o.Da * o.Dc, total = elems * o.batch * o.heads;
  const int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (e >= total) return;
  const int64_t bh = e / elems;
  const int batch = (int)(bh / o.heads), x = (int)(e % elems / o.Dc), y = (int)(e % o.Dc);
  const float g = clamped_decay(o.log_decay[bh % o.heads]);
  float s = o.init ? o.init[bh * elems + (int64_t)x * o.sx + (int64_t)y * o.sy] : 0.f;
  const double full = exp((double)o.split_len * (double)g);
  const double first = o.reverse ? exp((double)(o.split_len - 1) * (double)g) : full;
  // the sums come eight at a time: only the states follow from one another
  for (int k0 = 0; k0 + 1 < o.nsplit; k0 += 8) {
    float own[8];
    bool cut[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const bool in = k0 + u + 1 < o.nsplit;
      own[u] = in ? o.local[(int64_t)(k0 + u) * total + e] : 0.f;
      cut[u] = in && o.cut[(k0 + u) * o.batch + batch];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (k0 + u + 1 >= o.nsplit) break;
      s = cut[u] ? own[u] : (float)((k0 + u == 0 ? first : full) * (double)s + (double)own[u]);
      o.local[(int64_t)(k0 + u) * total + e] = s;
    }
  }
}

// One position of every (batch row, head): S' = [not reset] e^g S + k v^T, out = scale S'^T q.
// A block takes one (batch row, head); thread (r, y) holds the columns V y .. V y + V - 1 of the
// rows r, r + R, ...; the partial sums of out meet in shared memory in a fixed order. `next` may be
// `state` itself: every element is read and written by one thread. Bound by HBM: the state once in and
// once out, eight rows of a thread on their way at a time (4096 x 8 x 64 x 64: 182 us, 5.9 TB/s).
template <class T, int V>
__global__ void __launch_bounds__(kThreads)
    step_kernel(const Rows q, const Rows k, const Rows v, const float* log_decay,
                const uint8_t* reset, int64_t reset_batch, const float* state, float* next, T* out,
                int heads, int Dk, int Dv, float scale) {
  extern __shared__ float part[];  // [R][Dv padded to V], then q, k [Dk] each
  const int bh = blockIdx.x, batch = bh / heads, head = bh % heads;
  const int cols = ceil_div(Dv, V), R = blockDim.x / cols;
  float* sq = part + R * cols * V;
  float* sk = sq + Dk;
  const T* qp = static_cast<const T*>(q.p) + batch * q.batch + head * q.head;
  const T* kp = static_cast<const T*>(k.p) + batch * k.batch + head * k.head;
  const T* vp = static_cast<const T*>(v.p) + batch * v.batch + head * v.head;
  for (int i = threadIdx.x; i < Dk; i += blockDim.x) {
    sq[i] = to_float(qp[i]);
    sk[i] = to_float(kp[i]);
  }
  const bool cut = reset && reset[batch * reset_batch];
  const float decay = expf(clamped_decay(log_decay[head]));
  const int r = threadIdx.x / cols, y = threadIdx.x % cols * V;
  const bool on = r < R;
  float val[V], acc[V];
#pragma unroll
  for (int w = 0; w < V; ++w) {
    val[w] = on && y + w < Dv ? to_float(vp[y + w]) : 0.f;
    acc[w] = 0.f;
  }
  __syncthreads();
  const int64_t base = (int64_t)bh * Dk * Dv;
  if (on) {
#pragma unroll 8
    for (int x = r; x < Dk; x += R) {
      float s[V];
      if (cut) {
#pragma unroll
        for (int w = 0; w < V; ++w) s[w] = 0.f;
      } else if constexpr (V == 4) {
        const float4 f = __ldcs(reinterpret_cast<const float4*>(state + base + (int64_t)x * Dv + y));
        s[0] = f.x, s[1] = f.y, s[2] = f.z, s[3] = f.w;
      } else {
        s[0] = state[base + (int64_t)x * Dv + y];
      }
#pragma unroll
      for (int w = 0; w < V; ++w) {
        s[w] = decay * s[w] + sk[x] * val[w];
        acc[w] += sq[x] * s[w];
      }
      if constexpr (V == 4)
        __stcs(reinterpret_cast<float4*>(next + base + (int64_t)x * Dv + y), make_float4(s[0], s[1], s[2], s[3]));
      else
        next[base + (int64_t)x * Dv + y] = s[0];
    }
#pragma unroll
    for (int w = 0; w < V; ++w) part[r * cols * V + y + w] = acc[w];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < Dv; c += blockDim.x) {
    float s = 0.f;
    for (int u = 0; u < R; ++u) s += part[u * cols * V + c];
    out[(int64_t)bh * Dv + c] = from_float<T>(s * scale);
  }
}

template <class T, int DA, int DS>
int run_chunks(const Ops& ops, bool vec, cudaStream_t stream) {
  const Op& o = ops.op[0];
  constexpr int kSmem = sizeof(Smem<DA, DS>);
  static std::atomic<uint64_t> allowed[2];
  int blocks = 0;
  for (int i = 0; i < ops.n; ++i) blocks = max(blocks, o.batch * o.heads * ceil_div(ops.op[i].Dc, DS));
  if (o.nsplit > 1) {
    BT_TRY(allow_smem(chunk_kernel<T, DA, DS, false>, kSmem, allowed[1]));
    chunk_kernel<T, DA, DS, false><<<dim3(blocks, o.nsplit - 1, ops.n), kThreads, kSmem, stream>>>(ops, vec);
    BT_LAUNCH_CHECK("linear attention split sums");
    BT_TRY(launch_join(ops, stream));
  }
  BT_TRY(allow_smem(chunk_kernel<T, DA, DS, true>, kSmem, allowed[0]));
  chunk_kernel<T, DA, DS, true><<<dim3(blocks, o.nsplit, ops.n), kThreads, kSmem, stream>>>(ops, vec);
  BT_LAUNCH_CHECK("linear attention");
  return BT_OK;
}

template <class T>
int run_ops(const Ops& ops, cudaStream_t stream) {
  int da = 0, dc = 0;
  bool vec = sizeof(T) == 4;
  for (int i = 0; i < ops.n; ++i) {
    const Op& o = ops.op[i];
    da = max(da, o.Da);
    dc = max(dc, o.Dc);
    auto rows = [&](const Rows& r) {
      auto ok = [](int64_t s, int n) { return n <= 1 || s % 4 == 0; };
      return ((uintptr_t)r.p & 15) == 0 && ok(r.step, o.steps) && ok(r.head, o.heads) && ok(r.batch, o.batch);
    };
    vec = vec && o.Da % 4 == 0 && o.Dc % 4 == 0 && rows(o.a) && rows(o.b) && rows(o.c);
  }
  // narrow blocks while wide ones would not fill the SMs twice (three operations of the case above:
  // 103 us wide, 125 narrow)
  const Op& o = ops.op[0];
  const bool narrow = (int64_t)o.batch * o.heads * ceil_div(dc, kWide) * o.nsplit * ops.n < 2 * kNumSMs;
  if (da <= 64)
    return narrow ? run_chunks<T, 64, kNarrow>(ops, vec, stream) : run_chunks<T, 64, kWide>(ops, vec, stream);
  return narrow ? run_chunks<T, 128, kNarrow>(ops, vec, stream) : run_chunks<T, 128, kWide>(ops, vec, stream);
}

// Splits of the steps: the number whose launches are the shortest, in units of the walk over 128 steps. Two
// blocks share an SM (one alone is faster by about a third); a sequence costs a unit to begin and end, the
// sums of the splits half of a full walk, and the two more launches about two units.
void choose_splits(const bt_linear_attention_shape* s, int ops, int* nsplit, int* len) {
  const int64_t blocks = (int64_t)s->batch * s->heads * ceil_div(max(s->key_dim, s->value_dim), kWide) * ops;
  const int chunks = max(1, ceil_div(s->steps, 128));
  int best = chunks;
  double least = 1e300;
  for (int n = 1; n <= 64 && n <= chunks; ++n) {
    const int each = ceil_div(chunks, n), have = ceil_div(chunks, each);
    auto walk = [&](int64_t items, double unit) {
      const double shared = items <= kNumSMs ? 0.65 : 1.0;
      return (double)ceil_div64(items, 2 * kNumSMs) * (each * unit + 1.0) * shared;
    };
    const double t = walk(blocks * have, 1.0) + (have > 1 ? walk(blocks * (have - 1), 0.5) + 2.0 : 0.0);
    if (t < least) least = t, best = each;
  }
  *len = best * 128;
  *nsplit = max(1, ceil_div(s->steps, *len));
}

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

int check_shape(const bt_linear_attention_shape* s, const char* who) {
  BT_CHECK_ARG(s, "%s: null shape", who);
  BT_CHECK_ARG(s->batch >= 0 && s->steps >= 0 && s->heads >= 0, "%s: negative size", who);
  BT_CHECK_ARG(s->steps <= INT32_MAX - 256, "%s: %d steps are too many", who, s->steps);  // a chunk's end is an int
  BT_CHECK_ARG(s->key_dim >= 1 && s->key_dim <= 128 && s->value_dim >= 1 && s->value_dim <= 128,
               "%s: heads of %d and %d features (1 to 128 are supported)", who, s->key_dim,
               s->value_dim);
  BT_CHECK_ARG((int64_t)s->batch * s->heads <= (1 << 29), "%s: %d x %d sequences are too many", who,
               s->batch, s->heads);
  BT_CHECK_ARG(s->dtype == BT_DTYPE_F32 || s->dtype == BT_DTYPE_BF16, "%s: dtype %d", who, s->dtype);
  BT_CHECK_ARG(s->log_decay || s->batch * s->heads == 0, "%s: null log_decay", who);
  return BT_OK;
}

int64_t workspace_bytes(const bt_linear_attention_shape* s, int ops) {
  int nsplit, len;
  choose_splits(s, ops, &nsplit, &len);
  if (nsplit == 1) return 0;
  const int64_t state = (int64_t)s->batch * s->heads * s->key_dim * s->value_dim * 4;
  return ops * (align256((nsplit - 1) * state) + align256((int64_t)(nsplit - 1) * s->batch * 4));
}

Rows rows_of(const bt_heads& h) { return Rows{h.data, h.batch_stride, h.step_stride, h.head_stride}; }

Op op_of(const bt_linear_attention_shape* s, const bt_heads& a, const bt_heads& b, const bt_heads& c,
         const bt_heads& out, bool transposed, bool reverse) {
  Op o{};
  o.a = rows_of(a);
  o.b = rows_of(b);
  o.c = rows_of(c);
  o.out = out.data;
  o.out_batch = out.batch_stride;
  o.out_step = out.step_stride;
  o.out_head = out.head_stride;
  o.sx = transposed ? 1 : s->value_dim;
  o.sy = transposed ? s->value_dim : 1;
  o.Da = transposed ? s->value_dim : s->key_dim;
  o.Dc = transposed ? s->key_dim : s->value_dim;
  o.log_decay = s->log_decay;
  o.reset = s->reset;
  o.reset_batch = s->reset_batch_stride;
  o.reset_step = s->reset_step_stride;
  o.batch = s->batch;
  o.steps = s->steps;
  o.heads = s->heads;
  o.in_scale = reverse ? s->scale : 1.f;
  o.out_scale = reverse ? 1.f : s->scale;
  o.reverse = reverse;
  return o;
}

int launch(const bt_linear_attention_shape* s, Ops& ops, void* workspace, int64_t bytes,
           cudaStream_t stream, const char* who) {
  int nsplit, len;
  choose_splits(s, ops.n, &nsplit, &len);
  const int64_t need = workspace_bytes(s, ops.n);
  BT_CHECK_ARG(need == 0 || (workspace && bytes >= need), "%s: workspace of %lld bytes, %lld needed",
               who, (long long)bytes, (long long)need);
  BT_CHECK_ARG(((uintptr_t)workspace & 15) == 0, "%s: workspace not 16-byte aligned", who);
  char* w = static_cast<char*>(workspace);
  for (int i = 0; i < ops.n; ++i) {
    Op& o = ops.op[i];
    o.nsplit = nsplit;
    o.split_len = len;
    if (nsplit > 1) {
      const int64_t state = (int64_t)s->batch * s->heads * s->key_dim * s->value_dim * 4;
      o.local = reinterpret_cast<float*>(w);
      w += align256((nsplit - 1) * state);
      o.cut = reinterpret_cast<int*>(w);
      w += align256((int64_t)(nsplit - 1) * s->batch * 4);
    }
  }
  if (s->batch == 0 || s->heads == 0) return BT_OK;
  if (s->dtype == BT_DTYPE_F32) return run_ops<float>(ops, stream);
  bool suits = s->steps > 0;
  for (int i = 0; i < ops.n; ++i) suits = suits && suits_tensor_cores(ops.op[i]);
  return suits ? run_tensor_cores(ops, stream) : run_ops<__nv_bfloat16>(ops, stream);
}

}  // namespace

int launch_join(const Ops& ops, cudaStream_t stream) {
  int64_t total = 0;
  for (int i = 0; i < ops.n; ++i)
    total = max(total, (int64_t)ops.op[i].batch * ops.op[i].heads * ops.op[i].Da * ops.op[i].Dc);
  join_kernel<<<dim3((unsigned)ceil_div64(total, 256), ops.n), 256, 0, stream>>>(ops);
  BT_LAUNCH_CHECK("linear attention join");
  return BT_OK;
}

namespace {

bool rows_ok(const bt_linear_attention_shape* s, const bt_heads* h) {
  return h && (h->data || (int64_t)s->batch * s->steps * s->heads == 0);
}

}  // namespace
}  // namespace la
}  // namespace bt

using namespace bt;

extern "C" int64_t bt_linear_attention_workspace(const bt_linear_attention_shape* s, int32_t backward) {
  if (la::check_shape(s, "bt_linear_attention_workspace") != BT_OK) return -1;
  return la::workspace_bytes(s, backward ? 3 : 1);
}

extern "C" int bt_linear_attention(const bt_linear_attention_shape* s, const bt_heads* q,
                                   const bt_heads* k, const bt_heads* v, const float* state,
                                   const bt_heads* out, float* final_state, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  BT_TRY(la::check_shape(s, "bt_linear_attention"));
  BT_CHECK_ARG(la::rows_ok(s, q) && la::rows_ok(s, k) && la::rows_ok(s, v) && la::rows_ok(s, out) &&
                   (final_state || s->batch * s->heads == 0),
               "bt_linear_attention: null pointer");
  la::Ops ops{};
  ops.n = 1;
  ops.op[0] = la::op_of(s, *q, *k, *v, *out, false, false);
  ops.op[0].init = state;
  ops.op[0].fin = final_state;
  return la::launch(s, ops, workspace, workspace_bytes, (cudaStream_t)stream, "bt_linear_attention");
}

extern "C" int bt_linear_attention_backward(const bt_linear_attention_shape* s, const bt_heads* q,
                                            const bt_heads* k, const bt_heads* v,
                                            const float* state, const bt_heads* dout,
                                            const float* dfinal_state, const bt_heads* dq,
                                            const bt_heads* dk, const bt_heads* dv, float* dstate,
                                            void* workspace, int64_t workspace_bytes, void* stream) {
  BT_TRY(la::check_shape(s, "bt_linear_attention_backward"));
  BT_CHECK_ARG(la::rows_ok(s, q) && la::rows_ok(s, k) && la::rows_ok(s, v) && la::rows_ok(s, dout) &&
                   la::rows_ok(s, dq) && la::rows_ok(s, dk) && la::rows_ok(s, dv) &&
                   (dstate || s->batch * s->heads == 0),
               "bt_linear_attention_backward: null pointer");
  la::Ops ops{};
  ops.n = 3;
  ops.op[0] = la::op_of(s, *dout, *v, *k, *dq, true, false);
  ops.op[0].init = state;
  ops.op[1] = la::op_of(s, *k, *q, *dout, *dv, false, true);
  ops.op[1].init = dfinal_state;
  ops.op[1].fin = dstate;
  ops.op[2] = la::op_of(s, *v, *dout, *q, *dk, true, true);
  ops.op[2].init = dfinal_state;
  return la::launch(s, ops, workspace, workspace_bytes, (cudaStream_t)stream,
                    "bt_linear_attention_backward");
}

extern "C" int bt_linear_attention_step(const bt_linear_attention_shape* s, const bt_heads* q,
                                        const bt_heads* k, const bt_heads* v, const float* state,
                                        void* out, float* new_state, void* stream) {
  BT_TRY(la::check_shape(s, "bt_linear_attention_step"));
  BT_CHECK_ARG(s->steps == 1, "bt_linear_attention_step: %d steps", s->steps);
  const int64_t n = (int64_t)s->batch * s->heads;
  if (n == 0) return BT_OK;
  BT_CHECK_ARG(la::rows_ok(s, q) && la::rows_ok(s, k) && la::rows_ok(s, v) && state && out && new_state,
               "bt_linear_attention_step: null pointer");
  const bool vec = s->value_dim % 4 == 0 && (((uintptr_t)state | (uintptr_t)new_state) & 15) == 0;
  auto go = [&](auto tag, auto width) -> int {
    using T = decltype(tag);
    constexpr int V = decltype(width)::value;
    const int cols = ceil_div(s->value_dim, V), threads = 128, R = threads / cols;
    const size_t smem = (size_t)(R * cols * V + 2 * s->key_dim) * 4;
    la::step_kernel<T, V><<<(unsigned)n, threads, smem, (cudaStream_t)stream>>>(
        la::rows_of(*q), la::rows_of(*k), la::rows_of(*v), s->log_decay, s->reset,
        s->reset_batch_stride, state, new_state, static_cast<T*>(out), s->heads, s->key_dim,
        s->value_dim, s->scale);
    BT_LAUNCH_CHECK("linear attention step");
    return BT_OK;
  };
  if (s->dtype == BT_DTYPE_BF16)
    return vec ? go(__nv_bfloat16{}, std::integral_constant<int, 4>{})
               : go(__nv_bfloat16{}, std::integral_constant<int, 1>{});
  return vec ? go(float{}, std::integral_constant<int, 4>{}) : go(float{}, std::integral_constant<int, 1>{});
}

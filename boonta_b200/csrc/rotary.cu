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
// forms their cosines and sines once in shared memory (a frequency is a 64-bit fraction of a turn, so
// that a position's product with it drops whole turns exactly and far positions keep their phase, to
// |position| 2^-64 + 2^-32 of a turn). A
// group of lanes then walks rows (query or key heads) of one token with 16-byte loads, several rows on
// their way at a time, its cosines and sines in registers; the partner of an element, half a rotation
// away, comes from another lane. Where the rotated half does not fall on whole lanes, partners go through the group's row
// in shared memory. The weight gradients are summed per thread over its rows, over the block's groups
// in shared memory, and over the blocks by a second launch, each in a fixed order.
//
// Measured: 4 x 4096 tokens x (16 + 4) heads x 128 bf16, forward 55 us (3.1 TB/s), backward 95 us (2.7 TB/s)
// and 6 us for the weights: four (backward two) rows of 16 bytes a lane in flight and three blocks an SM leave
// it at the latency of shuffles and loads, 0.5 instructions a cycle and scheduler.
#include <type_traits>

#include "common.cuh"
#include "f32x2.cuh"

namespace bt {
namespace rot {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 16;  // tokens of a block's pass
constexpr int kMaxDim = 256;

// Shared memory of a launch: the angles of kMaxTokens tokens and a row for each group. Groups of G lanes hold rows of
// at most 2 G vectors of at most 8 values (or 8 G single ones), so kThreads / G of them hold 16 kThreads values.
constexpr size_t kMaxSmem = (size_t)(kMaxTokens * kMaxDim + 16 * kThreads) * 4;
static_assert(kMaxSmem <= 48 * 1024, "no attribute needed");

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

// V neighbouring elements as they lie in memory; as values, and (V even) as pairs.
template <class T, int V>
struct Raw {
  uint32_t w[4];
  __device__ __forceinline__ void load(const T* p) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
  }
  __device__ __forceinline__ void zero() { w[0] = w[1] = w[2] = w[3] = 0; }
  __device__ __forceinline__ Raw from_lane(unsigned mask, int lane, int G) const {
    Raw r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = __shfl_sync(mask, w[i], lane, G);
    return r;
  }
  __device__ __forceinline__ void get(uint64_t (&v)[V / 2]) const {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      if constexpr (sizeof(T) == 2) v[i] = pair_of_bf16(w[i]);
      else v[i] = (uint64_t)w[2 * i + 1] << 32 | w[2 * i];
    }
  }
  __device__ __forceinline__ void get(float (&v)[V]) const {
    uint64_t p[V / 2];
    get(p);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) v[2 * i] = low(p[i]), v[2 * i + 1] = high(p[i]);
  }
};
template <class T>
struct Raw<T, 1> {
  T t;
  __device__ __forceinline__ void load(const T* p) { t = *p; }
  __device__ __forceinline__ void zero() { t = from_float<T>(0.f); }
  __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = to_float(t); }
};

template <class T, int N>
__device__ __forceinline__ void store(T* p, const uint64_t (&v)[N]) {
  if constexpr (sizeof(T) == 2)
    *reinterpret_cast<uint4*>(p) = make_uint4(bf16_of_pair(v[0]), bf16_of_pair(v[1]), bf16_of_pair(v[2]), bf16_of_pair(v[3]));
  else
    *reinterpret_cast<float4*>(p) = make_float4(low(v[0]), high(v[0]), low(v[1]), high(v[1]));
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

// The fraction of a turn that `freq` radians are, in 2^-64 (whole turns fall away). 1 / (2 pi) in two doubles and the
// product's remainder: off by 2^-64 of a turn, where one double alone would be off by 2^-54 of the angle, which a
// far position multiplies.
__device__ __forceinline__ uint64_t turns_of(double freq) {
  constexpr double kInv = 0x1.45f306dc9c883p-3, kInvLow = -0x1.6b01ec5417056p-57;
  const double t = freq * kInv, rest = fma(freq, kInv, -t) + freq * kInvLow;
  auto fixed = [](double x) { return (uint64_t)__double2ll_rn((x - rint(x)) * 0x1p64); };
  return fixed(t) + fixed(rest);
}

// Where a lane's elements find their angles and partners. x[c][i] holds feature (c * G + lane) * V + i.
enum Pairing {
  kLanes,     // (i, i + half), half a multiple of V, one chunk per lane: the partner is another lane's
  kNeighbours,  // (2 i, 2 i + 1) and V even: the partner is the lane's own
  kStaged     // anything else, through shared memory
};

// A lane's pairs of the rotation x -> x c + partner(x) s (the sign of the sine in s), kept for a token's
// rows. In kLanes the partner is the same element of another lane, in kNeighbours the other one of the pair.
template <int N>
struct Turn {
  uint64_t c[N], s[N];
};

template <Pairing kP, int N>
__device__ __forceinline__ void load_turn(const Args& a, const float* cs, int lane, Turn<N>& t) {
  const int d = lane * 2 * N;
#pragma unroll
  for (int i = 0; i < N; ++i) t.c[i] = pair(1.f, 1.f), t.s[i] = 0;
  if (d >= 2 * a.half) return;
  const float* sn = cs + a.half;
  if constexpr (kP == kLanes) {
    const bool second = d >= a.half;
    const int k = second ? d - a.half : d;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      t.c[i] = pair(cs[k + 2 * i], cs[k + 2 * i + 1]);
      t.s[i] = second ? pair(sn[k + 2 * i], sn[k + 2 * i + 1]) : pair(-sn[k + 2 * i], -sn[k + 2 * i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (d / 2 + i < a.half) {
        t.c[i] = pair(cs[d / 2 + i], cs[d / 2 + i]);
        t.s[i] = pair(-sn[d / 2 + i], sn[d / 2 + i]);
      }
  }
}

__device__ __forceinline__ uint64_t swapped(uint64_t a) { return a << 32 | a >> 32; }

// Turns x by the token's angles (sign 1), or back (-1), through the group's row in shared memory.
template <int V, int NC>
__device__ __forceinline__ void turn(const Args& a, float (&x)[NC][V], float* row, const float* cs, float sign,
                                     int lane, int G) {
  const int rd = 2 * a.half;
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
      const bool second = a.interleaved ? d & 1 : d >= a.half;
      const int k = a.interleaved ? d >> 1 : second ? d - a.half : d;
      const float other = row[a.interleaved ? d ^ 1 : (second ? d - a.half : d + a.half)];
      const float co = cs[k], si = sign * cs[a.half + k];
      x[c][i] = second ? x[c][i] * co + other * si : x[c][i] * co - other * si;
    }
  __syncwarp();
}

// G lanes to a row (kG where the launch knows them); a token's rows go round `share` groups, kRows of them on their way at a time, and a
// block's pass takes a.per tokens.
template <class T, class W, int V, int NC, Pairing kP, int kG, bool kBack>
__global__ void __launch_bounds__(kThreads, NC == 1 ? 3 : 1)
    rotary_kernel(const __grid_constant__ Args a, int lanes, int share) {
  const int G = kG ? kG : lanes;
  constexpr int kRows = NC > 2 ? 1 : kBack ? 2 : 4;
  extern __shared__ __align__(16) float sm[];
  float* cs = sm;                                 // [per][2 half]
  float* rows = sm + a.per * 2 * a.half;          // [groups][D] staging rows
  __shared__ int64_t s_off[kMaxTokens][6];        // element offsets of a token in q, k, yq, yk, gq, gk
  __shared__ int64_t s_pos[kMaxTokens];
  __shared__ uint64_t s_freq[kMaxDim / 2];        // turns a position, in 2^-64
  const int lane = threadIdx.x % G, group = threadIdx.x / G, groups = kThreads / G;
  float* row = rows + group * a.D;
  const unsigned mask = G == 32 ? ~0u : ((1u << G) - 1u) << ((threadIdx.x & 31) / G * G);
  const int tok = group / share, first = group % share;
  float dw[kBack ? 2 : 1][NC][V];
#pragma unroll
  for (int c = 0; c < NC; ++c)
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (kBack) dw[0][c][i] = dw[kBack ? 1 : 0][c][i] = 0.f;
  for (int i = threadIdx.x; i < a.half; i += kThreads) s_freq[i] = turns_of(a.freq[i]);
  const float inv = 1.f / (float)a.D;
  for (int64_t t0 = (int64_t)blockIdx.x * a.per; t0 < a.tokens; t0 += (int64_t)gridDim.x * a.per) {
    const int n = (int)min((int64_t)a.per, a.tokens - t0);
    __syncthreads();
    if (threadIdx.x < n) {
      const int64_t t = t0 + threadIdx.x;
      const int64_t b = a.tokens >> 31 ? t / a.steps : (int64_t)((unsigned)t / (unsigned)a.steps), st = t - b * a.steps;
      s_pos[threadIdx.x] = a.half ? a.pos[b * a.pos_batch + st * a.pos_step] : 0;
      int64_t* f = s_off[threadIdx.x];
      f[0] = b * a.q.batch + st * a.q.step;
      f[1] = b * a.k.batch + st * a.k.step;
      f[2] = b * a.yq.batch + st * a.yq.step;
      f[3] = b * a.yk.batch + st * a.yk.step;
      f[4] = b * a.gq.batch + st * a.gq.step;
      f[5] = b * a.gk.batch + st * a.gk.step;
    }
    __syncthreads();
    // groups without a token walk along: a warp's lanes stay together
    const bool mine = tok < n;
    const int64_t* f = s_off[mine ? tok : 0];
    Raw<T, V> nx[kRows][NC], ng[kBack ? kRows : 1][NC];
    // the rows h, h + share, .. of queries (0) or keys (1)
    auto fetch = [&](int which, int h) {
      const T* xp = static_cast<const T*>(which ? a.k.p : a.q.p) + f[which];
      const T* gp = static_cast<const T*>(which ? a.gk.p : a.gq.p) + f[4 + which];
      const int64_t xh = which ? a.k.head : a.q.head, gh = which ? a.gk.head : a.gq.head;
#pragma unroll
      for (int r = 0; r < kRows; ++r, h += share)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const int d = (c * G + lane) * V;
          nx[r][c].zero();
          if (kBack) ng[kBack ? r : 0][c].zero();
          if (mine && h < (which ? a.hk : a.hq) && d < a.D) {
            nx[r][c].load(xp + h * xh + d);
            if (kBack) ng[kBack ? r : 0][c].load(gp + h * gh + d);
          }
        }
    };
    fetch(0, first);  // on their way while the angles are formed
    for (int e = threadIdx.x; e < n * a.half; e += kThreads) {
      const int u = (unsigned)e / (unsigned)a.half, i = e - u * a.half;
      // the product's whole turns leave a 64-bit word by themselves; what stays, in half turns
      const int32_t turn = (int32_t)((uint64_t)s_pos[u] * s_freq[i] >> 32);
      float s, c;
      sincospif((float)turn * 0x1p-31f, &s, &c);
      cs[u * 2 * a.half + i] = c;
      cs[u * 2 * a.half + a.half + i] = s;
    }
    __syncthreads();
    const float* ct = cs + (mine ? tok : 0) * 2 * a.half;
    constexpr int N = kP == kStaged ? 1 : V / 2;
    Turn<N> tn;
    if constexpr (kP != kStaged) load_turn<kP, N>(a, ct, lane, tn);
    const int half_lanes = a.half / V;  // kLanes
    const int partner = lane < half_lanes ? lane + half_lanes : lane < 2 * half_lanes ? lane - half_lanes : lane;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const int H = which ? a.hk : a.hq;
      float w[NC][V];
      const void* wp = which ? a.wk : a.wq;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int d = (c * G + lane) * V + i;
          w[c][i] = d < a.D && wp ? to_float(static_cast<const W*>(wp)[d]) : 1.f;
        }
      float wo[V];  // the partner lane's weights
      if constexpr (kP == kLanes && !kBack)
#pragma unroll
        for (int i = 0; i < V; ++i) wo[i] = __shfl_sync(mask, w[0][i], partner, G);
      T* yp = static_cast<T*>(which ? a.yk.p : a.yq.p) + f[2 + which];
      const int64_t yh = which ? a.yk.head : a.yq.head;
      if (which) fetch(1, first);
      for (int h0 = 0; h0 < H; h0 += kRows * share) {
        if (h0) fetch(which, h0 + first);
        float rss[kRows];
        if constexpr (kP != kStaged) {
          // the rows' sums side by side: their shuffles do not wait for one another
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            uint64_t x[N], sq = 0;
            nx[r][0].get(x);
#pragma unroll
            for (int i = 0; i < N; ++i) sq = fma2(x[i], x[i], sq);
            rss[r] = low(sq) + high(sq);
          }
#pragma unroll
          for (int o = G >> 1; o > 0; o >>= 1)
#pragma unroll
            for (int r = 0; r < kRows; ++r) rss[r] += __shfl_xor_sync(mask, rss[r], o);
#pragma unroll
          for (int r = 0; r < kRows; ++r) rss[r] = rsqrtf(rss[r] * inv + a.eps);
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const int h = h0 + r * share + first;
          const bool on = mine && h < H;
          if constexpr (kP != kStaged) {
            const int d = lane * V;
            uint64_t x[N];
            nx[r][0].get(x);
            const float rs = rss[r];
            const uint64_t rr = pair(rs, rs);
            if constexpr (!kBack) {
              // the weights before the exchange: the partner's own
              uint64_t y[N], z[N];
#pragma unroll
              for (int i = 0; i < N; ++i) y[i] = mul2(x[i], pair(w[0][2 * i], w[0][2 * i + 1]));
              if constexpr (kP == kLanes) {
                nx[r][0].from_lane(mask, partner, G).get(z);
#pragma unroll
                for (int i = 0; i < N; ++i) z[i] = mul2(z[i], pair(wo[2 * i], wo[2 * i + 1]));
              } else {
#pragma unroll
                for (int i = 0; i < N; ++i) z[i] = swapped(y[i]);
              }
#pragma unroll
              for (int i = 0; i < N; ++i) x[i] = mul2(rr, fma2(y[i], tn.c[i], mul2(z[i], tn.s[i])));
            } else {
              uint64_t g[N], z[N], m2 = 0;
              ng[r][0].get(g);
              if constexpr (kP == kLanes) {
                ng[r][0].from_lane(mask, partner, G).get(z);
              } else {
#pragma unroll
                for (int i = 0; i < N; ++i) z[i] = swapped(g[i]);
              }
              // back: the sines change their sign
#pragma unroll
              for (int i = 0; i < N; ++i) {
                g[i] = sub2(mul2(g[i], tn.c[i]), mul2(z[i], tn.s[i]));
                const uint64_t gx = mul2(g[i], x[i]);
                const uint64_t ww = pair(w[0][2 * i], w[0][2 * i + 1]);
                const uint64_t was = pair(dw[kBack ? which : 0][0][2 * i], dw[kBack ? which : 0][0][2 * i + 1]);
                const uint64_t sum = fma2(gx, rr, was);
                dw[kBack ? which : 0][0][2 * i] = on ? low(sum) : low(was);
                dw[kBack ? which : 0][0][2 * i + 1] = on ? high(sum) : high(was);
                m2 = fma2(gx, ww, m2);
                g[i] = mul2(g[i], ww);
              }
              float m = low(m2) + high(m2);
#pragma unroll
              for (int o = G >> 1; o > 0; o >>= 1) m += __shfl_xor_sync(mask, m, o);
              // dx = r (u - x r^2 mean(u x))
              m *= inv * rs * rs;
              const uint64_t mm = pair(-m, -m);
#pragma unroll
              for (int i = 0; i < N; ++i) x[i] = mul2(rr, fma2(x[i], mm, g[i]));
            }
            if (on && d < a.D) store<T, N>(yp + h * yh + d, x);
          } else {
            float x[NC][V], g[kBack ? NC : 1][V];
#pragma unroll
            for (int c = 0; c < NC; ++c) {
              nx[r][c].get(x[c]);
              if constexpr (kBack) ng[r][c].get(g[c]);
            }
            float ss = 0.f;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
              for (int i = 0; i < V; ++i) ss += x[c][i] * x[c][i];
            for (int o = G >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
            const float rs = rsqrtf(ss * inv + a.eps);
            if constexpr (!kBack) {
#pragma unroll
              for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < V; ++i) x[c][i] *= rs * w[c][i];
              turn<V, NC>(a, x, row, ct, 1.f, lane, G);
            } else {
              turn<V, NC>(a, g, row, ct, -1.f, lane, G);
              float m = 0.f;
#pragma unroll
              for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                  x[c][i] *= rs;
                  dw[kBack ? which : 0][c][i] += on ? g[c][i] * x[c][i] : 0.f;
                  g[c][i] *= w[c][i];
                  m += g[c][i] * x[c][i];
                }
              for (int o = G >> 1; o > 0; o >>= 1) m += __shfl_xor_sync(mask, m, o);
              m *= inv;
#pragma unroll
              for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < V; ++i) x[c][i] = rs * (g[c][i] - x[c][i] * m);
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) {
              const int d = (c * G + lane) * V;
              if (on && d < a.D) store<T, V>(yp + h * yh + d, x[c]);
            }
          }
        }
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
// neighbouring features, its 32 warps on every 32nd partial.
template <class W>
__global__ void __launch_bounds__(1024) weight_kernel(const float* partial, int blocks, int D, W* dwq, W* dwk) {
  __shared__ double part[32][33];
  const int which = blockIdx.y, d = blockIdx.x * 32 + (threadIdx.x & 31), warp = threadIdx.x >> 5;
  double s = 0.0;
  if (d < D)
#pragma unroll 4
    for (int b = warp; b < blocks; b += 32) s += (double)partial[((size_t)b * 2 + which) * D + d];
  part[warp][threadIdx.x & 31] = s;
  __syncthreads();
  W* to = which ? dwk : dwq;
  if (warp == 0 && d < D && to) {
    double t = 0.0;
#pragma unroll
    for (int u = 0; u < 32; ++u) t += part[u][threadIdx.x];
    to[d] = from_float<W>((float)t);
  }
}

// Blocks of the backward: its partial sums have one row for each. At most three an SM, which fit.
constexpr int kMaxBlocks = 3 * kNumSMs;
int backward_blocks(int64_t tokens, int per) {
  const int64_t n = ceil_div64(tokens, per);
  return (int)(n < kMaxBlocks ? n : kMaxBlocks);
}

// Lanes of a row, and the groups that share a token's rows: at most one for each row, fewer where
// there are tokens enough to fill the GPU twice over with the rest.
void shape_of(int64_t tokens, int rows, int chunks, int* G, int* share) {
  *G = 1;
  while (*G < 32 && *G < chunks) *G *= 2;
  const int groups = kThreads / *G;
  int s = max(1, groups / kMaxTokens);
  while (s < groups && (s * 2 <= rows || s < 2) && ceil_div64(tokens * s, groups) < 2 * kNumSMs) s *= 2;
  *share = min(s, groups);
}

struct Call {
  Args a;
  int dtype, wdtype, G, share;
  bool vec;
};

template <class T, class W, bool kBack>
int launch(const Call& c, int blocks, cudaStream_t s) {
  const Args& a = c.a;
  const int V = c.vec ? 16 / (int)sizeof(T) : 1;
  const int nc = ceil_div(ceil_div(a.D, V), c.G);
  auto go = [&](auto vv, auto cc, auto pp, auto gg) -> int {
    constexpr int VV = decltype(vv)::value, CC = decltype(cc)::value;
    constexpr Pairing kP = decltype(pp)::value;
    auto kernel = rotary_kernel<T, W, VV, CC, kP, decltype(gg)::value, kBack>;
    const bool staged = kP == kStaged || kBack;
    const size_t smem = ((size_t)a.per * 2 * a.half + (staged ? (size_t)(kThreads / c.G) * a.D : 0)) * 4;
    BT_CHECK_ARG(smem <= kMaxSmem, "query/key norms: %zu bytes of shared memory", smem);
    kernel<<<blocks, kThreads, smem, s>>>(a, c.G, c.share);
    BT_LAUNCH_CHECK("query/key norms with rotation");
    return BT_OK;
  };
  constexpr int VT = 16 / (int)sizeof(T);
  using Lanes = std::integral_constant<Pairing, kLanes>;
  using Neighbours = std::integral_constant<Pairing, kNeighbours>;
  using Staged = std::integral_constant<Pairing, kStaged>;
  using Vec = std::integral_constant<int, VT>;
  using One = std::integral_constant<int, 1>;
  using Any = std::integral_constant<int, 0>;
  if (c.vec && nc == 1 && c.G >= 8 && (a.interleaved || a.half % VT == 0)) {
    // Rows of 8, 16 or 32 lanes (bf16: 64, 128, 256 features), partners on whole lanes: forward and backward of 2^25
    // elements 47 and 72 us in bf16 (128 features), 53 and 68 in float32.
    auto wide = [&](auto pp) -> int {
      if (c.G == 8) return go(Vec{}, One{}, pp, std::integral_constant<int, 8>{});
      if (c.G == 16) return go(Vec{}, One{}, pp, std::integral_constant<int, 16>{});
      return go(Vec{}, One{}, pp, std::integral_constant<int, 32>{});
    };
    return a.interleaved ? wide(Neighbours{}) : wide(Lanes{});
  }
  // The others, partners through shared memory, for lack of lanes or because the rotated half ends inside one: bf16 128
  // features with half 60 232 and 297 us, 32 features 336 and 317, float32 256 features (two vectors a lane) 162
  // and 199. Features that do not fill vectors go one by one: 33 features 1215 and 1617 us.
  if (c.vec) return go(Vec{}, std::integral_constant<int, 2>{}, Staged{}, Any{});
  return go(One{}, std::integral_constant<int, kMaxDim / 32>{}, Staged{}, Any{});
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

// The launch's shape, once it is known whether rows are read in vectors.
void shape_call(Call& c) {
  const int V = c.vec ? (c.dtype == BT_DTYPE_BF16 ? 8 : 4) : 1;
  shape_of(c.a.tokens, max(1, c.a.hq + c.a.hk), ceil_div(c.a.D, V), &c.G, &c.share);
  c.a.per = kThreads / c.G / c.share;
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
  c.dtype = s->dtype;
  c.wdtype = s->weight_dtype;
  const int e = s->dtype == BT_DTYPE_BF16 ? 2 : 4;
  c.vec = (s->dim * e) % 16 == 0 && aligned(q, a.hq, e) && aligned(k, a.hk, e) && aligned(yq, a.hq, e) &&
          aligned(yk, a.hk, e);
  shape_call(c);
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
  // one row of sums for each block, of which there are at most so many whatever the launch's shape
  const int64_t tokens = (int64_t)s->batch * s->steps;
  return (int64_t)rot::backward_blocks(tokens, 1) * 2 * s->dim * 4;
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
  rot::shape_call(c);
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
      rot::weight_kernel<<<grid, 1024, 0, (cudaStream_t)stream>>>(
          c.a.partial, blocks, s->dim, static_cast<__nv_bfloat16*>(dq_weight), static_cast<__nv_bfloat16*>(dk_weight));
    else
      rot::weight_kernel<<<grid, 1024, 0, (cudaStream_t)stream>>>(
          c.a.partial, blocks, s->dim, static_cast<float*>(dq_weight), static_cast<float*>(dk_weight));
    BT_LAUNCH_CHECK("query/key norm weight gradients");
  }
  return BT_OK;
}

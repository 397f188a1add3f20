// Activations kept in 8 bits for the backward pass, and the passes that make and use them (sm_100a):
//
//   checkpoint8            x -> (q, scale), groups of 128 values with a scale of their own
//   checkpoint8_restore    (q, scale) -> x'
//   rmsnorm_checkpoint8    RMSNorm and the 8-bit copy of its input from one read of x
//   rmsnorm_backward8      the backward of RMSNorm with x' in the place of x:
//                            n = x' r;  dx = r (dy g - n mean(dy g n));  dg = sum_rows dy n
//                          no power of r is formed, which would leave the normal numbers where x does not:
//                          n comes from the levels in one product, level (scale r)
//   silu_mul               h = silu(gate) * up, with the 8-bit copies of both factors on request
//   silu_mul_backward      dgate = dh up s (1 + gate (1 - s)), dup = dh gate s, s = sigmoid(gate)
//
// All are bound by memory: every operand is touched once.  The lanes that hold one group are
// neighbours, so a group's largest magnitude is a few shuffles and nothing goes through shared memory.
// [16384,8192] bf16, calls by themselves: silu_mul with both copies and its backward from them 346 us = 6.3
// TB/s over the two, silu_mul alone 129 us, its backward from tensors 201, copy and restore 133 us = 6.1 TB/s;
// [32768,4096] bf16: RMSNorm with the copy and its backward 283 us = 4.8 TB/s (0.73 of the measured copy
// bandwidth: 64 registers, some spilled in the backward, two thirds of the issue slots busy).
#include <algorithm>

#include "quant8.cuh"
#include "row_tile.cuh"

namespace vb {
namespace {

// How a group of up to 128 neighbouring values lies in the lanes of a warp: L lanes with W vectors of
// V values each.  VEC: 16-byte vectors (needs rows of whole vectors, 16-byte aligned); else single
// values.  What a lane works out per group (its place, the scale) is shared by its W vectors.
template <class T, bool VEC, int WV> struct Lanes {
  static constexpr int V = VEC ? 16 / sizeof(T) : 1;
  static constexpr int W = VEC ? WV : 4;
  static constexpr int L = kQ8Group / (V * W);
  static constexpr int N = V * W;  // values per lane
  struct Raw { Vec<T, V> v[W]; };
  struct Q { typename Q8Raw<V>::type v[W]; };
  static __device__ __forceinline__ int off(int lane, int w) { return (w * L + lane) * V; }

  static __device__ __forceinline__ Raw load(const T* group, int lane, int len) {
    Raw r;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (off(lane, w) < len) r.v[w] = *reinterpret_cast<const Vec<T, V>*>(group + off(lane, w));
      else r.v[w] = Vec<T, V>{};
    }
    return r;
  }
  static __device__ __forceinline__ void widen(const Raw& r, float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = to_f(r.v[i / V].v[i % V]);
  }
  static __device__ __forceinline__ void store(T* group, int lane, int len, const float (&v)[N]) {
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (off(lane, w) >= len) continue;
      Vec<T, V> r;
#pragma unroll
      for (int e = 0; e < V; ++e) r.v[e] = from_f<T>(v[w * V + e]);
      *reinterpret_cast<Vec<T, V>*>(group + off(lane, w)) = r;
    }
  }
  static __device__ __forceinline__ Q load_q(const uint8_t* group, int lane, int len) {
    Q q{};
#pragma unroll
    for (int w = 0; w < W; ++w)
      if (off(lane, w) < len) q.v[w] = *reinterpret_cast<const typename Q8Raw<V>::type*>(group + off(lane, w));
    return q;
  }
  template <int F> static __device__ __forceinline__ void widen_q(const Q& q, float scale, float (&v)[N]) {
#pragma unroll
    for (int w = 0; w < W; ++w) q8_widen<F, V>(q.v[w], scale, *reinterpret_cast<float(*)[V]>(&v[w * V]));
  }
  // quantises the group: returns its stored scale
  template <int F>
  static __device__ __forceinline__ float store_q(uint8_t* group, int lane, int len, const Raw& raw, const float (&v)[N]) {
    const Q8Scale s = q8_scale<F>(group_mag<T, V, W, L>(raw.v));
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (off(lane, w) >= len) continue;
      if constexpr (VEC) q8_store<F, V>(group + off(lane, w), *reinterpret_cast<const float(*)[V]>(&v[w * V]), s.up);
      else group[off(lane, w)] = q8_pack1<F>(v[w], s.up);
    }
    return s.down;
  }
};

// the groups of [rows, cols] in order: group i is group `g` of row `row`
struct Groups {
  int64_t total, per_row, cols;
  FastDiv div;
  int small;
  int flat;  // dense rows of whole groups: the groups lie one behind the other
  // dense: every operand's row stride is the row length
  void fill(int64_t rows, int64_t c, bool dense) {
    cols = c;
    per_row = (c + kQ8Group - 1) / kQ8Group;
    total = rows * per_row;
    small = total < (int64_t{1} << 31);
    flat = dense && c % kQ8Group == 0;
    if (small) div = FastDiv(static_cast<uint32_t>(per_row));
  }
  __device__ __forceinline__ void find(int64_t i, int64_t& row, int64_t& col, int& len) const {
    if (flat) {
      row = 0;
      col = i * kQ8Group;
      len = kQ8Group;
      return;
    }
    int64_t g;
    if (small) {
      uint32_t q, r;
      div.divmod(static_cast<uint32_t>(i), q, r);
      row = q; g = r;
    } else {
      row = i / per_row; g = i - row * per_row;
    }
    col = g * kQ8Group;
    len = static_cast<int>(min(int64_t{kQ8Group}, cols - col));
  }
};

struct CkParams {
  const void* x;
  void* out;
  uint8_t* q;
  float* scale;
  int64_t x_stride;
  Groups g;
};

// Short blocks, one group per thread and several vectors of it per lane: what a lane works out per group
// (18 instructions per value with one vector per lane) is shared.  [16384,8192] bf16, copy and
// restore: one vector 172 us, two 141, four 133; gated activation, both passes: 379, 340, 361.  Four groups
// of one vector in flight per thread instead took 222 and 409 us.
constexpr int kCkThreads = 128;
constexpr int kCopyVecs = 4;
constexpr int kGluVecs = 2;

template <class T, bool VEC, int F, int WV, int U>
__global__ void __launch_bounds__(kCkThreads) checkpoint8_kernel(const __grid_constant__ CkParams p) {
  using A = Lanes<T, VEC, WV>;
  constexpr int S = kCkThreads / A::L;
  const int lane = threadIdx.x % A::L;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (S * U) + threadIdx.x / A::L;
  typename A::Raw x[U];
  int64_t row[U], col[U];
  int len[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = first + u * S;
    len[u] = 0; row[u] = col[u] = 0;
    if (i < p.g.total) p.g.find(i, row[u], col[u], len[u]);
    x[u] = A::load(static_cast<const T*>(p.x) + row[u] * p.x_stride + col[u], lane, len[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float v[A::N];
    A::widen(x[u], v);
    const float s = A::template store_q<F>(p.q + row[u] * p.g.cols + col[u], lane, len[u], x[u], v);
    if (lane == 0 && len[u]) p.scale[first + u * S] = s;
  }
}

template <class T, bool VEC, int F, int WV, int U>
__global__ void __launch_bounds__(kCkThreads) restore8_kernel(const __grid_constant__ CkParams p) {
  using A = Lanes<T, VEC, WV>;
  constexpr int S = kCkThreads / A::L;
  const int lane = threadIdx.x % A::L;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (S * U) + threadIdx.x / A::L;
  typename A::Q q[U];
  float s[U];
  int64_t row[U], col[U];
  int len[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = first + u * S;
    len[u] = 0; row[u] = col[u] = 0; s[u] = 0.f;
    if (i < p.g.total) {
      p.g.find(i, row[u], col[u], len[u]);
      s[u] = __ldg(p.scale + i);
    }
    q[u] = A::load_q(p.q + row[u] * p.g.cols + col[u], lane, len[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float v[A::N];
    A::template widen_q<F>(q[u], s[u], v);
    A::store(static_cast<T*>(p.out) + row[u] * p.g.cols + col[u], lane, len[u], v);
  }
}

// ---------------------------------------------------------------------------------------
// gated activation
// ---------------------------------------------------------------------------------------
// 1 / (1 + exp(-x)).  For 16-bit storage exp(-x) is 2^(-x log2 e) on the special-function unit: the
// rounded product is off by at most |x| 2^-23 in the exponent, 2^-18 of the value where that is
// smallest (|x| < 40; further out the sigmoid itself is below 2^-57 or rounds to one).
// Below x = -87.3 the result is no normal number, and times x and another factor it may be one again in
// fp32 and bf16.  fp32 takes the reciprocal that keeps it; bf16, where that costs 3 to 8 % ([16384,8192],
// both passes), divides 1/16 + exp(-x) / 16 instead, the sixteenth taken off in the exponent.
template <class T> __device__ __forceinline__ float sigmoid(float x) {
  float e, r;
  if constexpr (sizeof(T) == 4) {
    asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.f + expf(-x)));
    return r;
  }
  constexpr bool WIDE = std::is_same_v<T, __nv_bfloat16>;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(x, -1.4426950408889634f, WIDE ? -4.f : 0.f)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"((WIDE ? 0.0625f : 1.f) + e));
  return WIDE ? 0.0625f * r : r;
}

struct GluParams {
  const void* dout;    // backward
  const void* gate;    // storage type, or levels
  const void* up;
  const float* gate_scale;
  const float* up_scale;
  void* out;           // forward
  void* dgate;
  void* dup;
  uint8_t* q_gate;
  uint8_t* q_up;
  float* s_gate;
  float* s_up;
  int64_t dout_stride, gate_stride, up_stride;
  Groups g;
};

// KEEP: also writes the 8-bit copies
template <class T, bool VEC, int F, bool KEEP, int WV, int U>
__global__ void __launch_bounds__(kCkThreads) silu_mul_kernel(const __grid_constant__ GluParams p) {
  using A = Lanes<T, VEC, WV>;
  constexpr int S = kCkThreads / A::L;
  const int lane = threadIdx.x % A::L;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (S * U) + threadIdx.x / A::L;
  typename A::Raw ga[U], up[U];
  int64_t row[U], col[U];
  int len[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = first + u * S;
    len[u] = 0; row[u] = col[u] = 0;
    if (i < p.g.total) p.g.find(i, row[u], col[u], len[u]);
    ga[u] = A::load(static_cast<const T*>(p.gate) + row[u] * p.gate_stride + col[u], lane, len[u]);
    up[u] = A::load(static_cast<const T*>(p.up) + row[u] * p.up_stride + col[u], lane, len[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float a[A::N], b[A::N], h[A::N];
    A::widen(ga[u], a);
    A::widen(up[u], b);
#pragma unroll
    for (int e = 0; e < A::N; ++e) h[e] = a[e] * sigmoid<T>(a[e]) * b[e];
    const int64_t at = row[u] * p.g.cols + col[u];
    A::store(static_cast<T*>(p.out) + at, lane, len[u], h);
    if constexpr (KEEP) {
      const float sa = A::template store_q<F>(p.q_gate + at, lane, len[u], ga[u], a);
      const float sb = A::template store_q<F>(p.q_up + at, lane, len[u], up[u], b);
      if (lane == 0 && len[u]) {
        p.s_gate[first + u * S] = sa;
        p.s_up[first + u * S] = sb;
      }
    }
  }
}

// KEPT: gate and up come from their 8-bit copies
template <class T, bool VEC, int F, bool KEPT, int WV, int U>
__global__ void __launch_bounds__(kCkThreads) silu_mul_bwd_kernel(const __grid_constant__ GluParams p) {
  using A = Lanes<T, VEC, WV>;
  constexpr int S = kCkThreads / A::L;
  const int lane = threadIdx.x % A::L;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (S * U) + threadIdx.x / A::L;
  typename A::Raw d[U], ga[U], up[U];
  typename A::Q qa[U], qb[U];
  float sa[U], sb[U];
  int64_t row[U], col[U];
  int len[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i = first + u * S;
    len[u] = 0; row[u] = col[u] = 0; sa[u] = sb[u] = 0.f;
    if (i < p.g.total) p.g.find(i, row[u], col[u], len[u]);
    d[u] = A::load(static_cast<const T*>(p.dout) + row[u] * p.dout_stride + col[u], lane, len[u]);
    if constexpr (KEPT) {
      const int64_t at = row[u] * p.g.cols + col[u];
      qa[u] = A::load_q(static_cast<const uint8_t*>(p.gate) + at, lane, len[u]);
      qb[u] = A::load_q(static_cast<const uint8_t*>(p.up) + at, lane, len[u]);
      if (len[u]) {
        sa[u] = __ldg(p.gate_scale + i);
        sb[u] = __ldg(p.up_scale + i);
      }
    } else {
      ga[u] = A::load(static_cast<const T*>(p.gate) + row[u] * p.gate_stride + col[u], lane, len[u]);
      up[u] = A::load(static_cast<const T*>(p.up) + row[u] * p.up_stride + col[u], lane, len[u]);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float a[A::N], b[A::N], da[A::N], db[A::N], dv[A::N];
    if constexpr (KEPT) {
      A::template widen_q<F>(qa[u], sa[u], a);
      A::template widen_q<F>(qb[u], sb[u], b);
    } else {
      A::widen(ga[u], a);
      A::widen(up[u], b);
    }
    A::widen(d[u], dv);
#pragma unroll
    for (int e = 0; e < A::N; ++e) {
      const float s = sigmoid<T>(a[e]);
      da[e] = dv[e] * b[e] * s * (1.f + a[e] * (1.f - s));
      db[e] = dv[e] * a[e] * s;
    }
    const int64_t at = row[u] * p.g.cols + col[u];
    A::store(static_cast<T*>(p.dgate) + at, lane, len[u], da);
    A::store(static_cast<T*>(p.dup) + at, lane, len[u], db);
  }
}

// ---------------------------------------------------------------------------------------
// RMSNorm with the 8-bit copy of its input, and its backward from that copy
// ---------------------------------------------------------------------------------------
struct Norm8Params {
  const void* x;       // forward
  const void* dy;      // backward
  const float* gamma;
  void* out;           // forward: the norm; backward: dx
  uint8_t* q;
  float* scale;
  float* inv;
  float* ws;           // backward: [workers][cols] partial sums of dgamma, or null
  int64_t rows, cols, groups;
  int64_t chunk;       // rows of a worker
  int64_t stride;      // of x or dy
  float eps;
};

// Rows staged in shared memory as in residual_norm: a worker (a warp when TPR lanes of it share a row,
// else the block) walks neighbouring rows, a thread reads back only what it copied itself.
constexpr int kNormElts = 16;
// group of 128 values that chunk c of this thread belongs to, counted from the row's start
template <class A> __device__ __forceinline__ int chunk_group(int j0, int c) { return (j0 + A::off(c, 0)) / kQ8Group; }

template <class T, int V, int TPR, int F>
__global__ void __launch_bounds__(TPR ? 256 : 1024, TPR ? 4 : 1) rmsnorm8_kernel(const __grid_constant__ Norm8Params p) {
  using A = RowChunks<T, V, TPR, kNormElts>;
  constexpr int C = A::C;
  constexpr int RW = TPR ? 32 / TPR : 1;
  // chunks (of this thread) and lanes that hold one group together
  constexpr int GC = V > 1 ? 1 : 2, GL = V > 1 ? kQ8Group / V : 32;
  static_assert(A::STEP % GL == 0, "a group's lanes are neighbours");
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float4 red[2][TPR ? 1 : 32];
  const int rl = TPR ? static_cast<int>(threadIdx.x & 31) / A::STEP : 0;
  const int j0 = A::base(), left = static_cast<int>(p.cols) - j0;
  const float inv_cols = 1.f / static_cast<float>(p.cols);
  unsigned char* gbuf = smem + static_cast<size_t>(threadIdx.x >> 5) * (A::WARP_FACTORS + A::WARP_ARRAY);
  unsigned char* xbuf = gbuf + A::WARP_FACTORS;
  A::zero_rest(xbuf, true, left);
  A::sync();
  const int seg = A::segment(), seg_left = static_cast<int>(p.cols) - seg;
  const int64_t worker = TPR ? static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32 : blockIdx.x;
  const int64_t begin = min(worker * p.chunk, p.rows);
  const int todo = static_cast<int>(min(p.chunk, p.rows - begin));
  const T* x_at = static_cast<const T*>(p.x) + (begin + rl) * p.stride + seg;
  if (rl < todo) A::copy(xbuf, x_at, seg_left, p.x);
  copy_commit();
  A::fill_factors(gbuf, left, [&](int o) { return p.gamma ? p.gamma[j0 + o] : 1.f; });
  T* out = static_cast<T*>(p.out) + (begin + rl) * p.cols + j0;
  uint8_t* q = p.q + (begin + rl) * p.cols + j0;
  float* scale = p.scale + (begin + rl) * p.groups;
  int phase = 0;
  for (int r0 = 0; r0 < todo; r0 += RW) {
    const bool live = RW == 1 || r0 + rl < todo;
    copy_wait<0>();
    A::sync();
    float x[kNormElts];
    float s[1] = {0.f};
#pragma unroll
    for (int c0 = 0; c0 < A::N; c0 += GC) {
      Vec<T, C> raw[GC];
#pragma unroll
      for (int k = 0; k < GC; ++k) {
        A::read_raw(xbuf, A::shift(p.x, p.stride, begin + r0 + rl), c0 + k, raw[k]);
#pragma unroll
        for (int e = 0; e < C; ++e) {
          x[(c0 + k) * C + e] = to_f(raw[k].v[e]);
          s[0] = fmaf(x[(c0 + k) * C + e], x[(c0 + k) * C + e], s[0]);
        }
      }
      // the 8-bit copy needs nothing of the row's sum
      const Q8Scale sc = q8_scale<F>(group_mag<T, C, GC, GL>(raw));
      if (live && A::off(c0, 0) < left) {
        if constexpr (V > 1) {
          q8_store<F, V>(q + A::off(c0, 0), *reinterpret_cast<const float(*)[V]>(&x[c0 * C]), sc.up);
        } else {
#pragma unroll
          for (int i = 0; i < GC * C; ++i)
            if (A::off(c0 + i / C, i % C) < left) q[A::off(c0 + i / C, i % C)] = q8_pack1<F>(x[c0 * C + i], sc.up);
        }
        if ((threadIdx.x & 31) % GL == 0) scale[chunk_group<A>(j0, c0)] = sc.down;
      }
    }
    x_at += RW * p.stride;
    A::sync();
    if (r0 + RW + rl < todo) A::copy(xbuf, x_at, seg_left, p.x);
    copy_commit();
    if (!live) s[0] = 0.f;
    sum_row<TPR, 1>(s, &red[0][0], phase);
    const float inv = rsqrtf(s[0] * inv_cols + p.eps);
    if (live) {
#pragma unroll
      for (int c = 0; c < A::N; ++c) {
        float g[C];
        A::read_factors(gbuf, c, g);
#pragma unroll
        for (int e = 0; e < C; ++e) g[e] *= x[c * C + e] * inv;
        A::write(out, c, left, g);
      }
      if (j0 == 0 && p.inv) p.inv[begin + r0 + rl] = inv;
    }
    out += RW * p.cols;
    q += RW * p.cols;
    scale += RW * p.groups;
  }
  copy_wait<0>();
}

// any length and alignment: a block per row, a warp per group
template <class T, int F>
__global__ void __launch_bounds__(256) rmsnorm8_stream_kernel(const __grid_constant__ Norm8Params p) {
  using A = Lanes<T, false, 4>;
  __shared__ float red[2][1][8];
  RowFold<256, 1, 256> fold{red};
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.stride;
    float s[1] = {0.f};
    for (int64_t g = w; g < p.groups; g += 8) {
      const int len = static_cast<int>(min(int64_t{kQ8Group}, p.cols - g * kQ8Group));
      const typename A::Raw raw = A::load(x + g * kQ8Group, lane, len);
      float v[A::N];
      A::widen(raw, v);
#pragma unroll
      for (int e = 0; e < A::N; ++e) s[0] = fmaf(v[e], v[e], s[0]);
      const float sc = A::template store_q<F>(p.q + row * p.cols + g * kQ8Group, lane, len, raw, v);
      if (lane == 0) p.scale[row * p.groups + g] = sc;
    }
    fold(s);
    const float inv = rsqrtf(s[0] / static_cast<float>(p.cols) + p.eps);
    for (int64_t j = threadIdx.x; j < p.cols; j += 256)
      static_cast<T*>(p.out)[row * p.cols + j] = from_f<T>(to_f(x[j]) * inv * (p.gamma ? p.gamma[j] : 1.f));
    if (threadIdx.x == 0 && p.inv) p.inv[row] = inv;
  }
}

template <class T, int V, int TPR, int F>
__global__ void __launch_bounds__(TPR ? 256 : 1024, TPR ? 2 : 1) rmsnorm_bwd8_kernel(const __grid_constant__ Norm8Params p) {
  using A = RowChunks<T, V, TPR, kNormElts>;
  using Q = RowChunks<uint8_t, V, TPR, kNormElts>;
  constexpr int C = A::C, E = kNormElts;
  constexpr int RW = TPR ? 32 / TPR : 1;
  constexpr int GC = V > 1 ? 1 : 2;    // chunks of this thread in one group
  constexpr int NS = A::N / GC;        // scales of this thread
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float4 red[2][TPR ? 1 : 32];
  const int rl = TPR ? static_cast<int>(threadIdx.x & 31) / A::STEP : 0;
  const int j0 = A::base(), left = static_cast<int>(p.cols) - j0;
  const float inv_cols = 1.f / static_cast<float>(p.cols);
  unsigned char* gbuf = smem + static_cast<size_t>(threadIdx.x >> 5) * (A::WARP_FACTORS + A::WARP_ARRAY + Q::WARP_ARRAY);
  unsigned char* dbuf = gbuf + A::WARP_FACTORS;
  unsigned char* qbuf = dbuf + A::WARP_ARRAY;
  A::zero_rest(dbuf, true, left);
  Q::zero_rest(qbuf, true, left);
  A::sync();
  const int seg = A::segment(), seg_left = static_cast<int>(p.cols) - seg;
  const int64_t worker = TPR ? static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32 : blockIdx.x;
  const int64_t begin = min(worker * p.chunk, p.rows);
  const int todo = static_cast<int>(min(p.chunk, p.rows - begin));
  const T* dy_at = static_cast<const T*>(p.dy) + (begin + rl) * p.stride + seg;
  const uint8_t* q_at = p.q + (begin + rl) * p.cols + seg;
  const float* scale_at = p.scale + (begin + rl) * p.groups;
  const float* inv_at = p.inv + begin + rl;
  int ahead = rl;
  float sc_next[NS], inv_next;
  auto fetch = [&] {
    inv_next = 0.f;
#pragma unroll
    for (int i = 0; i < NS; ++i) sc_next[i] = 0.f;
    if (ahead < todo) {
      A::copy(dbuf, dy_at, seg_left, p.dy);
      Q::copy(qbuf, q_at, seg_left, p.q);
      inv_next = *inv_at;
#pragma unroll
      for (int i = 0; i < NS; ++i)
        if (A::off(i * GC, 0) < left) sc_next[i] = __ldg(scale_at + chunk_group<A>(j0, i * GC));
    }
    ahead += RW;
    dy_at += RW * p.stride;
    q_at += RW * p.cols;
    scale_at += RW * p.groups;
    inv_at += RW;
    copy_commit();
  };
  fetch();
  A::fill_factors(gbuf, left, [&](int o) { return p.gamma ? p.gamma[j0 + o] : 1.f; });
  T* dx = static_cast<T*>(p.out) + (begin + rl) * p.cols + j0;
  float sum[E];
#pragma unroll
  for (int i = 0; i < E; ++i) sum[i] = 0.f;
  int phase = 0;
  for (int r0 = 0; r0 < todo; r0 += RW) {
    const bool live = RW == 1 || r0 + rl < todo;
    copy_wait<0>();
    A::sync();
    const int64_t row = begin + r0 + rl;
    const float inv = inv_next;
    float x[E];  // normed
    Vec<T, C> dy[A::N];
    float s[1] = {0.f};
    if (live) {
#pragma unroll
      for (int c = 0; c < A::N; ++c) {
        float g[C];
        A::read_raw(dbuf, A::shift(p.dy, p.stride, row), c, dy[c]);
        A::read_factors(gbuf, c, g);
        Vec<uint8_t, C> lv;
        Q::read_raw(qbuf, Q::shift(p.q, p.cols, row), c, lv);
        const float sc = sc_next[c / GC] * inv;
        if constexpr (V > 1) {
          q8_widen<F, V>(*reinterpret_cast<const typename Q8Raw<V>::type*>(&lv), sc, *reinterpret_cast<float(*)[V]>(&x[c * C]));
        } else {
#pragma unroll
          for (int e = 0; e < C; ++e) x[c * C + e] = __fmul_rn(q8_level1<F>(lv.v[e]), sc);
        }
#pragma unroll
        for (int e = 0; e < C; ++e) {
          const int i = c * C + e;
          const float t = to_f(dy[c].v[e]) * x[i];
          sum[i] += t;
          s[0] = fmaf(t, g[e], s[0]);
        }
      }
    }
    // 16-bit rows stay in registers, and the next row's copies run through the reduction and the stores
    // ([32768,4096] bf16, both passes: 302 -> 278 us; 32-bit rows are too many registers, 222 -> 230 us)
    constexpr bool kEarly = sizeof(T) == 2;
    if constexpr (kEarly) {
      A::sync();
      fetch();
    }
    sum_row<TPR, 1>(s, &red[0][0], phase);
    const float k = inv * inv_cols * s[0];
    if (live) {
#pragma unroll
      for (int c = 0; c < A::N; ++c) {
        float d[C], g[C];
        if constexpr (!kEarly) A::read_raw(dbuf, A::shift(p.dy, p.stride, row), c, dy[c]);
        A::read_factors(gbuf, c, g);
#pragma unroll
        for (int e = 0; e < C; ++e) d[e] = fmaf(inv * to_f(dy[c].v[e]), g[e], -k * x[c * C + e]);
        A::write(dx, c, left, d);
      }
    }
    dx += RW * p.cols;
    if constexpr (!kEarly) {
      A::sync();
      fetch();
    }
  }
  copy_wait<0>();
  if (p.ws == nullptr) return;
  if constexpr (RW > 1) {  // the worker's rows at a time
#pragma unroll
    for (int i = 0; i < E; ++i)
#pragma unroll
      for (int d = TPR; d < 32; d <<= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], d);
  }
  if (rl == 0) {
    float* w = p.ws + worker * p.cols + j0;
#pragma unroll
    for (int c = 0; c < A::N; ++c)
#pragma unroll
      for (int e = 0; e < C; ++e)
        if (A::off(c, e) < left) w[A::off(c, e)] = sum[c * C + e];
  }
}

template <class T, int F>
__global__ void __launch_bounds__(256) rmsnorm_bwd8_stream_kernel(const __grid_constant__ Norm8Params p) {
  __shared__ float red[2][1][8];
  RowFold<256, 1, 256> fold{red};
  const int t = threadIdx.x;
  float* w = p.ws ? p.ws + static_cast<int64_t>(blockIdx.x) * p.cols : nullptr;
  if (w)
    for (int64_t j = t; j < p.cols; j += 256) w[j] = 0.f;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* dy = static_cast<const T*>(p.dy) + row * p.stride;
    const uint8_t* q = p.q + row * p.cols;
    const float* sc = p.scale + row * p.groups;
    const float inv = p.inv[row];
    float s[1] = {0.f};
    for (int64_t j = t; j < p.cols; j += 256) {
      const float d = to_f(dy[j]) * __fmul_rn(q8_level1<F>(q[j]), sc[j / kQ8Group]);
      if (w) w[j] = fmaf(d, inv, w[j]);
      s[0] = fmaf(d, p.gamma ? p.gamma[j] : 1.f, s[0]);
    }
    fold(s);
    const float c = s[0] * inv / static_cast<float>(p.cols) * inv;  // dx = r (dy g - c x')
    for (int64_t j = t; j < p.cols; j += 256) {
      const float x = __fmul_rn(q8_level1<F>(q[j]), sc[j / kQ8Group]);
      static_cast<T*>(p.out)[row * p.cols + j] =
          from_f<T>(inv * fmaf(to_f(dy[j]), p.gamma ? p.gamma[j] : 1.f, -c * x));
    }
  }
}

__global__ void __launch_bounds__(kStripThreads) rmsnorm_bwd8_fold_kernel(float* dgamma, const float* ws, int64_t parts, int64_t cols) {
  __shared__ float sm[kStripThreads / 32][8];
  const float s = strip_sum(ws, parts, cols, sm);
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 8 + threadIdx.x;
  if (threadIdx.x < 8 && c < cols) dgamma[c] = s;
}

// ---------------------------------------------------------------------------------------
inline unsigned flat_grid(int64_t groups, int lanes, int u) {
  const int64_t per = int64_t{kCkThreads} / lanes * u;
  return static_cast<unsigned>((groups + per - 1) / per);
}
inline bool rows_fit(int64_t groups) { return groups < (int64_t{1} << 32); }  // at least four groups per block

// calls fn(format constant)
#define VB_FORMAT(format, F, ...)                                                     \
  do {                                                                                \
    if ((format) == VBT_B200_Q8_INT8) { constexpr int F = VBT_B200_Q8_INT8; __VA_ARGS__; } \
    else { constexpr int F = VBT_B200_Q8_E4M3; __VA_ARGS__; }                         \
  } while (0)

template <class T>
void launch_checkpoint(const CkParams& p, int format, bool restore, cudaStream_t s) {
  constexpr int VW = 16 / sizeof(T);
  const bool vec = p.g.cols % VW == 0 && p.x_stride % VW == 0 && a16(p.x) && a16(p.out) &&
                   reinterpret_cast<uintptr_t>(p.q) % VW == 0;
  constexpr int WV = kCopyVecs, U = 1;
  unsigned grid = 0;
#define VB_CK(VEC)                                                                   \
  do {                                                                               \
    grid = flat_grid(p.g.total, Lanes<T, VEC, WV>::L, U);                            \
    if (restore) VB_FORMAT(format, F, (restore8_kernel<T, VEC, F, WV, U><<<grid, kCkThreads, 0, s>>>(p)));    \
    else VB_FORMAT(format, F, (checkpoint8_kernel<T, VEC, F, WV, U><<<grid, kCkThreads, 0, s>>>(p)));         \
  } while (0)
  if (vec) VB_CK(true);
  else VB_CK(false);
#undef VB_CK
  note_launch(VBT_B200_FAMILY_ROWOP, VBT_B200_WK_CHECKPOINT8, dim3(grid), dim3(kCkThreads), vec ? VW : 1, 1, 0, 1,
              p.g.total / p.g.per_row * p.g.cols, p.g.cols, 0, s);
}

template <class T>
void launch_glu(const GluParams& p, int format, bool backward, bool kept, cudaStream_t s) {
  constexpr int VW = 16 / sizeof(T);
  auto q_ok = [&](const void* q) { return reinterpret_cast<uintptr_t>(q) % VW == 0; };
  bool vec = p.g.cols % VW == 0 && a16(p.out) && a16(p.dout) && a16(p.dgate) && a16(p.dup) &&
             p.dout_stride % VW == 0 && q_ok(p.q_gate) && q_ok(p.q_up);
  if (backward && kept) vec = vec && q_ok(p.gate) && q_ok(p.up);
  else vec = vec && a16(p.gate) && a16(p.up) && p.gate_stride % VW == 0 && p.up_stride % VW == 0;
  constexpr int WV = kGluVecs, U = 1;
  unsigned grid = 0;
#define VB_GLU(VEC)                                                                                             \
  do {                                                                                                          \
    grid = flat_grid(p.g.total, Lanes<T, VEC, WV>::L, U);                                                       \
    if (!backward && !kept) silu_mul_kernel<T, VEC, 0, false, WV, U><<<grid, kCkThreads, 0, s>>>(p);                \
    else if (!backward) VB_FORMAT(format, F, (silu_mul_kernel<T, VEC, F, true, WV, U><<<grid, kCkThreads, 0, s>>>(p)));   \
    else if (!kept) silu_mul_bwd_kernel<T, VEC, 0, false, WV, U><<<grid, kCkThreads, 0, s>>>(p);                    \
    else VB_FORMAT(format, F, (silu_mul_bwd_kernel<T, VEC, F, true, WV, U><<<grid, kCkThreads, 0, s>>>(p)));              \
  } while (0)
  if (vec) VB_GLU(true);
  else VB_GLU(false);
#undef VB_GLU
  note_launch(VBT_B200_FAMILY_ROWOP, VBT_B200_WK_SILU_MUL, dim3(grid), dim3(kCkThreads), vec ? VW : 1, 1, 0, 1,
              p.g.total / p.g.per_row * p.g.cols, p.g.cols, 0, s);
}

// How a row kernel of this file runs: TPR lanes of a warp share a row (0: the block does), `workers`
// of them with a run of `chunk` rows each; threads == 0: the stream kernel.
struct NormShape {
  int tpr, threads, smem;
  int64_t chunk, workers;
  unsigned grid;
};
template <class Bytes>
inline NormShape norm_shape(int64_t rows, int64_t cols, int elt, bool vec, Bytes bytes, int sms) {
  NormShape h{};
  const int64_t lanes = (cols + kNormElts - 1) / kNormElts;
  if (lanes > 1024) return h;
  // a group of 128 values lies in 16 lanes of 16-bit vectors, else in 32
  h.tpr = lanes <= 16 && elt == 2 && vec ? 16 : lanes <= 32 ? 32 : 0;
  h.threads = h.tpr ? 256 : static_cast<int>((lanes + 31) / 32 * 32);
  h.smem = h.threads * bytes(elt, vec, h.tpr);
  if (h.smem > kSmemPerBlock - 1024) return NormShape{};
  const int per_block = h.tpr ? h.threads / 32 : 1;
  const int per_sm = std::max(1, std::min(1024 / h.threads, kSmemPerSm / (h.smem + (h.tpr ? 1024 : 2048))));
  const int64_t most = int64_t{sms} * per_sm * per_block;
  h.chunk = (rows + most - 1) / most;
  h.grid = static_cast<unsigned>(((rows + h.chunk - 1) / h.chunk + per_block - 1) / per_block);
  h.workers = int64_t{h.grid} * per_block;
  return h;
}
// shared memory per thread: gamma and a row of x, or of dy and the levels
constexpr int norm8_bytes(int elt, bool vec, int tpr) { return kNormElts * 4 + row_bytes_per_thread(kNormElts, elt, vec, tpr); }
constexpr int bwd8_bytes(int elt, bool vec, int tpr) {
  return kNormElts * 4 + row_bytes_per_thread(kNormElts, elt, vec, tpr) + row_bytes_per_thread(kNormElts, 1, vec, tpr);
}

#define VB_ROW8(KERNEL, V, TPR)                                                       \
  VB_FORMAT(format, F, do {                                                           \
    static std::atomic<uint64_t> done{0};                                             \
    VB_CUDA(allow_shared(KERNEL<T, V, TPR, F>, device, done, kSmemPerBlock - 1024));                       \
    KERNEL<T, V, TPR, F><<<h.grid, h.threads, h.smem, s>>>(p);                        \
  } while (0))
// single values of 16 bits may share a row between 32 lanes only (a group lies in 32 of them)
#define VB_ROW8_ALL(KERNEL)                                                           \
  do {                                                                                \
    if (vec) {                                                                        \
      if constexpr (VW == 8) {                                                        \
        if (h.tpr == 16) { VB_ROW8(KERNEL, VW, 16); break; }                          \
      }                                                                               \
      if (h.tpr == 32) VB_ROW8(KERNEL, VW, 32);                                       \
      else VB_ROW8(KERNEL, VW, 0);                                                    \
    } else if (h.tpr == 32) VB_ROW8(KERNEL, 1, 32);                                   \
    else VB_ROW8(KERNEL, 1, 0);                                                       \
  } while (0)

template <class T>
vbt_b200_status launch_norm8(Norm8Params p, int format, cudaStream_t s, int device) {
  constexpr int VW = 16 / sizeof(T);
  const int sms = sm_count(device);
  const bool vec = p.cols % VW == 0 && p.stride % VW == 0 && a16(p.x) && a16(p.out) &&
                   reinterpret_cast<uintptr_t>(p.q) % VW == 0;
  const NormShape h = norm_shape(p.rows, p.cols, sizeof(T), vec, norm8_bytes, sms);
  unsigned g = h.grid;
  p.chunk = h.chunk;
  if (h.threads == 0) {
    g = static_cast<unsigned>(std::min<int64_t>(p.rows, int64_t{sms} * 8));
    VB_FORMAT(format, F, (rmsnorm8_stream_kernel<T, F><<<g, 256, 0, s>>>(p)));
  } else {
    VB_ROW8_ALL(rmsnorm8_kernel);
  }
  VB_LAUNCH_CHECK();
  note_launch(VBT_B200_FAMILY_ROWOP, VBT_B200_WK_CHECKPOINT8, dim3(g), dim3(h.threads ? h.threads : 256), vec ? VW : 1, 1,
              0, 1, p.rows * p.cols, p.cols, 0, s);
  return VBT_B200_OK;
}

inline int64_t bwd8_stream_blocks(int64_t rows, int sms) { return std::min<int64_t>(rows, int64_t{sms} * 6); }

template <class T>
vbt_b200_status launch_norm_bwd8(Norm8Params p, float* dgamma, int format, cudaStream_t s, int device) {
  constexpr int VW = 16 / sizeof(T);
  const int sms = sm_count(device);
  const bool vec = p.cols % VW == 0 && p.stride % VW == 0 && a16(p.dy) && a16(p.out) &&
                   reinterpret_cast<uintptr_t>(p.q) % VW == 0;
  const NormShape h = norm_shape(p.rows, p.cols, sizeof(T), vec, bwd8_bytes, sms);
  int64_t parts = h.workers;
  unsigned g = h.grid;
  p.chunk = h.chunk;
  if (h.threads == 0) {
    parts = bwd8_stream_blocks(p.rows, sms);
    g = static_cast<unsigned>(parts);
    VB_FORMAT(format, F, (rmsnorm_bwd8_stream_kernel<T, F><<<g, 256, 0, s>>>(p)));
  } else {
    VB_ROW8_ALL(rmsnorm_bwd8_kernel);
  }
  VB_LAUNCH_CHECK();
  if (p.ws) rmsnorm_bwd8_fold_kernel<<<static_cast<unsigned>((p.cols + 7) / 8), kStripThreads, 0, s>>>(dgamma, p.ws, parts, p.cols);
  VB_LAUNCH_CHECK();
  note_launch(VBT_B200_FAMILY_ROWOP, VBT_B200_WK_RMSNORM_BACKWARD8, dim3(g), dim3(h.threads ? h.threads : 256), vec ? VW : 1,
              1, 0, p.ws ? 2 : 1, p.rows * p.cols, p.cols, p.ws ? static_cast<size_t>(parts) * p.cols * 4 : 0, s);
  return VBT_B200_OK;
}
#undef VB_ROW8_ALL
#undef VB_ROW8

vbt_b200_status check_common(const char* name, int32_t dtype, int32_t format, int64_t rows, int64_t cols) {
  VB_ARG(rows >= 0 && cols >= 0, std::string(name) + ": negative size");
  VB_ARG(rows < (int64_t{1} << 36), std::string(name) + ": too many rows");
  VB_ARG(is_float_dtype(dtype), std::string(name) + ": expected a floating dtype");
  VB_ARG(format == VBT_B200_Q8_INT8 || format == VBT_B200_Q8_E4M3, std::string(name) + ": unknown 8-bit format");
  VB_ARG(cols == 0 || rows_fit(rows * ((cols + kQ8Group - 1) / kQ8Group)), std::string(name) + ": too many groups");
  return VBT_B200_OK;
}

#define VB_BY_DTYPE(dtype, T, ...)                                            \
  switch (dtype) {                                                            \
    case VBT_B200_F32: { using T = float; __VA_ARGS__; break; }               \
    case VBT_B200_F16: { using T = __half; __VA_ARGS__; break; }              \
    default: { using T = __nv_bfloat16; __VA_ARGS__; break; }                 \
  }

}  // namespace
}  // namespace vb

extern "C" {

vbt_b200_status vbt_b200_checkpoint8(void* q, float* scale, const void* x, int32_t dtype, int32_t format, int64_t rows,
                                     int64_t cols, int64_t x_row_stride, void* stream) {
  using namespace vb;
  VB_TRY(check_common("checkpoint8", dtype, format, rows, cols));
  if (rows == 0 || cols == 0) return VBT_B200_OK;
  VB_ARG(q && scale && x, "checkpoint8: null pointer");
  VB_ARG(x_row_stride >= 0, "checkpoint8: negative row stride");
  DeviceScope scope(q);
  CkParams p{};
  p.x = x; p.q = static_cast<uint8_t*>(q); p.scale = scale; p.x_stride = x_row_stride;
  p.g.fill(rows, cols, x_row_stride == cols);
  VB_BY_DTYPE(dtype, T, launch_checkpoint<T>(p, format, false, static_cast<cudaStream_t>(stream)));
  VB_LAUNCH_CHECK();
  return VBT_B200_OK;
}

vbt_b200_status vbt_b200_checkpoint8_restore(void* out, const void* q, const float* scale, int32_t dtype, int32_t format,
                                             int64_t rows, int64_t cols, void* stream) {
  using namespace vb;
  VB_TRY(check_common("checkpoint8_restore", dtype, format, rows, cols));
  if (rows == 0 || cols == 0) return VBT_B200_OK;
  VB_ARG(out && q && scale, "checkpoint8_restore: null pointer");
  DeviceScope scope(out);
  CkParams p{};
  p.out = out; p.q = static_cast<uint8_t*>(const_cast<void*>(q)); p.scale = const_cast<float*>(scale);
  p.g.fill(rows, cols, true);
  VB_BY_DTYPE(dtype, T, launch_checkpoint<T>(p, format, true, static_cast<cudaStream_t>(stream)));
  VB_LAUNCH_CHECK();
  return VBT_B200_OK;
}

vbt_b200_status vbt_b200_rmsnorm_checkpoint8(void* out, float* inv_rms, void* q, float* scale, const void* x,
                                             const float* gamma, int32_t dtype, int32_t format, int64_t rows,
                                             int64_t cols, int64_t x_row_stride, float eps, void* stream) {
  using namespace vb;
  VB_TRY(check_common("rmsnorm_checkpoint8", dtype, format, rows, cols));
  if (rows == 0 || cols == 0) return VBT_B200_OK;
  VB_ARG(out && q && scale && x, "rmsnorm_checkpoint8: null pointer");
  VB_ARG(x_row_stride >= 0, "rmsnorm_checkpoint8: negative row stride");
  DeviceScope scope(out);
  Norm8Params p{};
  p.x = x; p.gamma = gamma; p.out = out; p.q = static_cast<uint8_t*>(q); p.scale = scale; p.inv = inv_rms;
  p.rows = rows; p.cols = cols; p.groups = (cols + kQ8Group - 1) / kQ8Group; p.stride = x_row_stride; p.eps = eps;
  VB_BY_DTYPE(dtype, T, VB_TRY(launch_norm8<T>(p, format, static_cast<cudaStream_t>(stream), scope.device())));
  VB_LAUNCH_CHECK();
  return VBT_B200_OK;
}

vbt_b200_status vbt_b200_rmsnorm_backward8_workspace_bytes(int64_t rows, int64_t cols, int32_t dtype, int32_t device,
                                                           size_t* bytes) {
  using namespace vb;
  VB_ARG(bytes != nullptr, "rmsnorm_backward8: null output");
  VB_TRY(check_common("rmsnorm_backward8", dtype, VBT_B200_Q8_INT8, rows, cols));
  // whichever form the pointers' alignment takes
  const int sms = sm_count(device), elt = itemsize(dtype);
  int64_t parts = bwd8_stream_blocks(rows, sms);
  for (bool vec : {false, true})
    if (rows > 0 && cols > 0) parts = std::max(parts, norm_shape(rows, cols, elt, vec, bwd8_bytes, sms).workers);
  *bytes = static_cast<size_t>(parts) * static_cast<size_t>(cols) * 4;
  return VBT_B200_OK;
}

vbt_b200_status vbt_b200_rmsnorm_backward8(void* dx, float* dgamma, const void* dy, const void* q, const float* scale,
                                           const float* inv_rms, const float* gamma, int32_t dtype, int32_t format,
                                           int64_t rows, int64_t cols, int64_t dy_row_stride, void* workspace,
                                           size_t workspace_bytes, void* stream) {
  using namespace vb;
  VB_TRY(check_common("rmsnorm_backward8", dtype, format, rows, cols));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (cols == 0) return VBT_B200_OK;
  if (rows == 0) {
    if (dgamma) {
      DeviceScope scope(dgamma);
      VB_CUDA(cudaMemsetAsync(dgamma, 0, static_cast<size_t>(cols) * 4, s));
    }
    return VBT_B200_OK;
  }
  VB_ARG(dx && dy && q && scale && inv_rms, "rmsnorm_backward8: null pointer");
  VB_ARG(dy_row_stride >= 0, "rmsnorm_backward8: negative row stride");
  DeviceScope scope(dx);
  Norm8Params p{};
  p.dy = dy; p.gamma = gamma; p.out = dx; p.q = static_cast<uint8_t*>(const_cast<void*>(q));
  p.scale = const_cast<float*>(scale); p.inv = const_cast<float*>(inv_rms);
  p.rows = rows; p.cols = cols; p.groups = (cols + kQ8Group - 1) / kQ8Group; p.stride = dy_row_stride;
  if (dgamma) {
    size_t need = 0;
    VB_TRY(vbt_b200_rmsnorm_backward8_workspace_bytes(rows, cols, dtype, scope.device(), &need));
    VB_ARG(workspace != nullptr && workspace_bytes >= need,
           "rmsnorm_backward8: workspace too small (see vbt_b200_rmsnorm_backward8_workspace_bytes)");
    p.ws = static_cast<float*>(workspace);
  }
  VB_BY_DTYPE(dtype, T, VB_TRY(launch_norm_bwd8<T>(p, dgamma, format, s, scope.device())));
  VB_LAUNCH_CHECK();
  return VBT_B200_OK;
}

vbt_b200_status vbt_b200_silu_mul(void* out, void* q_gate, float* scale_gate, void* q_up, float* scale_up,
                                  const void* gate, const void* up, int32_t dtype, int32_t format, int64_t rows,
                                  int64_t cols, int64_t gate_row_stride, int64_t up_row_stride, void* stream) {
  using namespace vb;
  VB_TRY(check_common("silu_mul", dtype, format, rows, cols));
  if (rows == 0 || cols == 0) return VBT_B200_OK;
  VB_ARG(out && gate && up, "silu_mul: null pointer");
  VB_ARG(q_gate == nullptr || (scale_gate && q_up && scale_up), "silu_mul: the 8-bit copies need all four outputs");
  VB_ARG(gate_row_stride >= 0 && up_row_stride >= 0, "silu_mul: negative row stride");
  DeviceScope scope(out);
  GluParams p{};
  p.gate = gate; p.up = up; p.out = out; p.gate_stride = gate_row_stride; p.up_stride = up_row_stride;
  p.q_gate = static_cast<uint8_t*>(q_gate); p.s_gate = scale_gate;
  p.q_up = static_cast<uint8_t*>(q_up); p.s_up = scale_up;
  p.g.fill(rows, cols, gate_row_stride == cols && up_row_stride == cols);
  VB_BY_DTYPE(dtype, T, launch_glu<T>(p, format, false, q_gate != nullptr, static_cast<cudaStream_t>(stream)));
  VB_LAUNCH_CHECK();
  return VBT_B200_OK;
}

vbt_b200_status vbt_b200_silu_mul_backward(void* dgate, void* dup, const void* dout, const void* gate,
                                           const float* scale_gate, const void* up, const float* scale_up,
                                           int32_t dtype, int32_t format, int64_t rows, int64_t cols,
                                           int64_t dout_row_stride, int64_t gate_row_stride, int64_t up_row_stride,
                                           void* stream) {
  using namespace vb;
  VB_TRY(check_common("silu_mul_backward", dtype, format, rows, cols));
  if (rows == 0 || cols == 0) return VBT_B200_OK;
  VB_ARG(dgate && dup && dout && gate && up, "silu_mul_backward: null pointer");
  VB_ARG((scale_gate == nullptr) == (scale_up == nullptr), "silu_mul_backward: both factors or neither in 8 bits");
  VB_ARG(dout_row_stride >= 0 && gate_row_stride >= 0 && up_row_stride >= 0, "silu_mul_backward: negative row stride");
  DeviceScope scope(dgate);
  GluParams p{};
  p.dout = dout; p.gate = gate; p.up = up; p.gate_scale = scale_gate; p.up_scale = scale_up;
  p.dgate = dgate; p.dup = dup;
  p.dout_stride = dout_row_stride; p.gate_stride = gate_row_stride; p.up_stride = up_row_stride;
  p.g.fill(rows, cols, dout_row_stride == cols && (scale_gate || (gate_row_stride == cols && up_row_stride == cols)));
  VB_BY_DTYPE(dtype, T, launch_glu<T>(p, format, true, scale_gate != nullptr, static_cast<cudaStream_t>(stream)));
  VB_LAUNCH_CHECK();
  return VBT_B200_OK;
}

}  // extern "C"

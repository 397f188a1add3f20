// The join of a transformer branch with the residual stream between two RMS norms, forward and
// backward (sm_100a).
//
//   v = y * i1 * g1,  i1 = rsqrt(mean(y^2) + eps)          (the norm behind the branch; v = y without)
//   r = a * x + b * gate * v
//   n = r * i2 * g2,  i2 = rsqrt(mean(r^2) + eps)          (the norm in front of the next block)
//
// Backward, with G the gradient that arrives at r:
//   G   = dr + i2 * (dn * g2) - r * i2^3 * mean(dn * g2 * r)
//   dx  = a * G                         dg2   = sum_rows dn * r * i2
//   dv  = b * G * gate                  dgate = sum_(rows of the gate row) b * G * y * i1 * g1
//   dy  = i1 * dv * g1 - y * i1^3 * mean(dv * g1 * y)       dg1 = sum_rows dv * y * i1
//
// The second mean of the backward needs G, which needs the first.  It splits into sums that do not:
//   sum(dv g1 y) = sum(w y (dr + i2 dn g2)) - c sum(w y r),  w = b gate g1, c = i2^3 mean(dn g2 r),
// so a row costs one reduction of three sums.  The forward's two sums stay apart: sum(r^2) expanded
// in x and v would cancel where the branch nearly undoes the stream.
#include <algorithm>

#include "row_tile.cuh"

namespace vb {
namespace {

struct JoinParams {
  const void* x;
  const void* y;
  const float* g1;
  const void* gate;
  const float* g2;
  void* r;
  void* n;
  float* inv1;
  float* inv2;
  int64_t rows, cols;
  int64_t x_stride, y_stride, gate_stride;  // elements
  int64_t per;                              // rows that share a gate row
  FastDiv per_div;                          // the same when rows < 2^31
  int small_rows;
  float a, b, eps;
  int post, pre;
};

__device__ __forceinline__ int64_t gate_row(const JoinParams& p, int64_t row) {
  return p.small_rows ? static_cast<int64_t>(p.per_div.div(static_cast<uint32_t>(row))) : row / p.per;
}

// TPR threads per row, VPL vectors of V elements per thread, rows in registers: x and y are read
// once, r and n written once.
template <class T, int V, int VPL, int TPR>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) residual_norm_kernel(const __grid_constant__ JoinParams p) {
  constexpr int THREADS = TPR < 256 ? 256 : TPR;
  constexpr int R = THREADS / TPR;
  __shared__ float red[2][1][THREADS / 32];
  RowFold<TPR, 1, THREADS> fold{red};
  const int rl = threadIdx.x / TPR, tl = threadIdx.x % TPR;
  const int nvec = static_cast<int>(p.cols / V);
  // every thread of a block makes the same number of rounds (barriers inside)
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * R; r0 < p.rows; r0 += static_cast<int64_t>(gridDim.x) * R) {
    const bool live = r0 + rl < p.rows;
    const int64_t row = live ? r0 + rl : 0;
    const int nv = live ? nvec : 0;
    Vec<T, V> x[VPL], y[VPL], gt[VPL];
    load_vecs<T, V, VPL>(static_cast<const T*>(p.y) + row * p.y_stride, tl, TPR, nv, y);
    load_vecs<T, V, VPL>(static_cast<const T*>(p.x) + row * p.x_stride, tl, TPR, nv, x);
    if (p.gate != nullptr)
      load_vecs<T, V, VPL>(static_cast<const T*>(p.gate) + gate_row(p, row) * p.gate_stride, tl, TPR, nv, gt);
    float s[1];
    float i1 = 1.f;
    if (p.post) {
      s[0] = 0.f;
#pragma unroll
      for (int k = 0; k < VPL; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) s[0] = fmaf(to_f(y[k].v[e]), to_f(y[k].v[e]), s[0]);
      fold(s);
      i1 = rsqrtf(s[0] / static_cast<float>(p.cols) + p.eps);
    }
    const float bi = p.b * i1;
    float r[VPL][V];
    s[0] = 0.f;
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
      float g[V];
      load_floats<V>(p.post ? p.g1 : nullptr, tl + k * TPR, nv, g, 1.f);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float c = bi * g[e];
        if (p.gate != nullptr) c *= to_f(gt[k].v[e]);
        r[k][e] = fmaf(p.a, to_f(x[k].v[e]), c * to_f(y[k].v[e]));
        s[0] = fmaf(r[k][e], r[k][e], s[0]);
      }
    }
    float i2 = 0.f;
    if (p.pre) {
      fold(s);
      i2 = rsqrtf(s[0] / static_cast<float>(p.cols) + p.eps);
    }
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
      const int j = tl + k * TPR;
      if (j >= nv) continue;
      Vec<T, V> o;
#pragma unroll
      for (int e = 0; e < V; ++e) o.v[e] = from_f<T>(r[k][e]);
      *reinterpret_cast<Vec<T, V>*>(static_cast<T*>(p.r) + row * p.cols + static_cast<int64_t>(j) * V) = o;
      if (p.pre) {
        float g[V];
        load_floats<V>(p.g2, j, nv, g, 1.f);
#pragma unroll
        for (int e = 0; e < V; ++e) o.v[e] = from_f<T>(r[k][e] * i2 * g[e]);
        *reinterpret_cast<Vec<T, V>*>(static_cast<T*>(p.n) + row * p.cols + static_cast<int64_t>(j) * V) = o;
      }
    }
    if (live && tl == 0) {
      if (p.post && p.inv1) p.inv1[row] = i1;
      if (p.pre && p.inv2) p.inv2[row] = i2;
    }
  }
}

// rows of any length and alignment: a block per row, scalar accesses, the row read once per sum
// (again from L2)
template <class T>
__global__ void __launch_bounds__(512) residual_norm_stream_kernel(const __grid_constant__ JoinParams p) {
  constexpr int THREADS = 512;
  __shared__ float red[2][1][THREADS / 32];
  RowFold<THREADS, 1, THREADS> fold{red};
  const int t = threadIdx.x;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    const T* y = static_cast<const T*>(p.y) + row * p.y_stride;
    const T* gate = p.gate ? static_cast<const T*>(p.gate) + gate_row(p, row) * p.gate_stride : nullptr;
    float s[1];
    float i1 = 1.f, i2 = 0.f;
    if (p.post) {
      s[0] = 0.f;
      for (int64_t j = t; j < p.cols; j += THREADS) s[0] = fmaf(to_f(y[j]), to_f(y[j]), s[0]);
      fold(s);
      i1 = rsqrtf(s[0] / static_cast<float>(p.cols) + p.eps);
    }
    const float bi = p.b * i1;
    auto value = [&](int64_t j) {
      float c = bi;
      if (p.post && p.g1) c *= p.g1[j];
      if (gate) c *= to_f(gate[j]);
      return fmaf(p.a, to_f(x[j]), c * to_f(y[j]));
    };
    if (p.pre) {
      s[0] = 0.f;
      for (int64_t j = t; j < p.cols; j += THREADS) {
        const float r = value(j);
        s[0] = fmaf(r, r, s[0]);
      }
      fold(s);
      i2 = rsqrtf(s[0] / static_cast<float>(p.cols) + p.eps);
    }
    for (int64_t j = t; j < p.cols; j += THREADS) {
      const float r = value(j);
      static_cast<T*>(p.r)[row * p.cols + j] = from_f<T>(r);
      if (p.pre) static_cast<T*>(p.n)[row * p.cols + j] = from_f<T>(r * i2 * (p.g2 ? p.g2[j] : 1.f));
    }
    if (t == 0) {
      if (p.post && p.inv1) p.inv1[row] = i1;
      if (p.pre && p.inv2) p.inv2[row] = i2;
    }
  }
}

template <class T>
vbt_b200_status launch_join(const JoinParams& p, cudaStream_t s, int device) {
  constexpr int VW = 16 / sizeof(T);
  constexpr int E = 16;  // values of a row per thread and operand
  const int sms = sm_count(device);
  const bool vec = p.cols % VW == 0 && p.x_stride % VW == 0 && p.y_stride % VW == 0 && p.gate_stride % VW == 0 &&
                   a16(p.x) && a16(p.y) && a16(p.gate) && a16(p.r) && a16(p.n) && a16(p.g1) && a16(p.g2);
  auto grid = [&](int rows_per_block, int per_sm) {
    const int64_t units = (p.rows + rows_per_block - 1) / rows_per_block;
    return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(units, int64_t{sms} * per_sm)));
  };
  unsigned g = 0;
  int threads = 256;
#define VB_JOIN(V, TPR)                                                         \
  do {                                                                          \
    threads = TPR < 256 ? 256 : TPR;                                            \
    g = grid(threads / TPR, 2048 / threads);                                    \
    residual_norm_kernel<T, V, E / V, TPR><<<g, threads, 0, s>>>(p);            \
  } while (0)
#define VB_JOIN_LADDER(V)                   \
  if (p.cols <= 8 * E) VB_JOIN(V, 8);       \
  else if (p.cols <= 32 * E) VB_JOIN(V, 32);     \
  else if (p.cols <= 128 * E) VB_JOIN(V, 128);   \
  else if (p.cols <= 256 * E) VB_JOIN(V, 256);   \
  else if (p.cols <= 512 * E) VB_JOIN(V, 512);   \
  else VB_JOIN(V, 1024)
  if (p.cols > 1024 * E) {
    threads = 512;
    g = grid(1, 4);
    residual_norm_stream_kernel<T><<<g, threads, 0, s>>>(p);
  } else if (vec) {
    VB_JOIN_LADDER(VW);
  } else {
    VB_JOIN_LADDER(1);
  }
#undef VB_JOIN_LADDER
#undef VB_JOIN
  VB_LAUNCH_CHECK();
  note_launch(VBT_B200_FAMILY_ROWOP, VBT_B200_WK_RESIDUAL_NORM, dim3(g), dim3(threads), vec ? VW : 1, 1, 0, 1,
              p.rows * p.cols, p.cols, 0, s);
  return VBT_B200_OK;
}

// ---------------------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------------------
enum { GATE_NONE = 0, GATE_SHARED = 1, GATE_ROW = 2 };

struct JoinBwdParams {
  const void* dr;    // may be null
  const void* dn;    // with pre
  const void* y;     // with post, or for dgate
  const void* r;     // with pre
  const float* inv1;
  const float* inv2;
  const float* g1;
  const void* gate;
  const float* g2;
  void* dx;
  void* dy;
  void* dgate;       // storage dtype; null to skip
  float* ws_g1;      // [gridDim.x][cols] partial sums of dgamma_post, or null
  float* ws_g2;      // the same of dgamma_pre
  float* ws_gate;    // [units][cols] when a gate row's rows are cut into several units; the stream
                     // kernel sums whole ones in [gridDim.x][cols]
  int64_t rows, cols;
  int64_t dr_stride, dn_stride, y_stride, r_stride, gate_stride;
  int64_t per;       // rows of one gate row (GATE_SHARED), else all rows
  int64_t chunk;     // rows of one unit
  int64_t cuts;      // units per gate row
  int64_t units;
  float a, b;
  int post, pre;
};

// A block walks units of neighbouring rows that share one gate row.  P = G * y * i1 is summed over
// a unit in registers; at the unit's end it gives the gate's gradient (b * g1 * P) and its part of
// dgamma_post (b * gate * P).  A gate row of its own per row (GATE_ROW) is a factor of the sum.
template <class T, int V, int VPL, int TPR, int MODE>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) residual_norm_bwd_kernel(const __grid_constant__ JoinBwdParams p) {
  constexpr int THREADS = TPR < 128 ? 128 : TPR;
  constexpr int R = THREADS / TPR;
  constexpr int E = V * VPL;
  __shared__ float red[2][3][THREADS / 32];
  __shared__ float slots[R > 1 ? E * (THREADS + TPR) : 1];
  RowFold<TPR, 3, THREADS> fold{red};
  const int rl = threadIdx.x / TPR, tl = threadIdx.x % TPR;
  const int nvec = static_cast<int>(p.cols / V);
  const float inv_cols = 1.f / static_cast<float>(p.cols);
  float sum1[E], sum2[E], tot1[MODE == GATE_SHARED ? E : 1];
#pragma unroll
  for (int e = 0; e < E; ++e) sum1[e] = sum2[e] = 0.f;
  if constexpr (MODE == GATE_SHARED)
#pragma unroll
    for (int e = 0; e < E; ++e) tot1[e] = 0.f;
  // adds the R row slots' values in slot order; every slot gets the result
  auto over_slots = [&](float (&v)[E]) {
    if constexpr (R > 1) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e) slots[e * (THREADS + TPR) + threadIdx.x] = v[e];
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < R; ++k) t += slots[e * (THREADS + TPR) + k * TPR + tl];
        v[e] = t;
      }
    }
  };
  for (int64_t u = blockIdx.x; u < p.units; u += gridDim.x) {
    const int64_t group = u / p.cuts;
    const int64_t begin = group * p.per + (u - group * p.cuts) * p.chunk;
    const int64_t end = min(begin + p.chunk, (group + 1) * p.per);
    const T* gate = MODE == GATE_SHARED ? static_cast<const T*>(p.gate) + group * p.gate_stride : nullptr;
    for (int64_t r0 = begin; r0 < end; r0 += R) {
      const bool live = r0 + rl < end;
      const int64_t row = live ? r0 + rl : begin;
      const int nv = live ? nvec : 0;
      Vec<T, V> dr[VPL], dn[VPL], y[VPL], rr[VPL], gt[VPL];
      load_vecs<T, V, VPL>(static_cast<const T*>(p.dr) + row * p.dr_stride, tl, TPR, p.dr ? nv : 0, dr);
      load_vecs<T, V, VPL>(static_cast<const T*>(p.dn) + row * p.dn_stride, tl, TPR, p.pre ? nv : 0, dn);
      load_vecs<T, V, VPL>(static_cast<const T*>(p.r) + row * p.r_stride, tl, TPR, p.pre ? nv : 0, rr);
      load_vecs<T, V, VPL>(static_cast<const T*>(p.y) + row * p.y_stride, tl, TPR, p.y ? nv : 0, y);
      if constexpr (MODE == GATE_ROW)
        load_vecs<T, V, VPL>(static_cast<const T*>(p.gate) + row * p.gate_stride, tl, TPR, nv, gt);
      if constexpr (MODE == GATE_SHARED) load_vecs<T, V, VPL>(gate, tl, TPR, nv, gt);
      const float i1 = p.post ? p.inv1[row] : 1.f;
      const float i2 = p.pre ? p.inv2[row] : 0.f;
      float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < VPL; ++k) {
        float g1[V], g2[V];
        load_floats<V>(p.post ? p.g1 : nullptr, tl + k * TPR, nv, g1, 1.f);
        load_floats<V>(p.pre ? p.g2 : nullptr, tl + k * TPR, nv, g2, 1.f);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float d = to_f(dn[k].v[e]), rv = to_f(rr[k].v[e]), yv = to_f(y[k].v[e]);
          float w = p.b * g1[e];
          if constexpr (MODE != GATE_NONE) w *= to_f(gt[k].v[e]);
          const float dg = d * g2[e], wy = w * yv;
          s[0] = fmaf(dg, rv, s[0]);
          s[1] = fmaf(wy, fmaf(i2, dg, to_f(dr[k].v[e])), s[1]);
          s[2] = fmaf(wy, rv, s[2]);
          sum2[k * V + e] = fmaf(d * i2, rv, sum2[k * V + e]);
        }
      }
      fold(s);
      const float c2 = i2 * i2 * i2 * s[0] * inv_cols;
      const float c1 = p.post ? i1 * i1 * i1 * (s[1] - c2 * s[2]) * inv_cols : 0.f;
#pragma unroll
      for (int k = 0; k < VPL; ++k) {
        const int j = tl + k * TPR;
        if (j >= nv) continue;
        float g1[V], g2[V];
        load_floats<V>(p.post ? p.g1 : nullptr, j, nv, g1, 1.f);
        load_floats<V>(p.pre ? p.g2 : nullptr, j, nv, g2, 1.f);
        Vec<T, V> ox, oy, og;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float rv = to_f(rr[k].v[e]), yv = to_f(y[k].v[e]);
          const float G = fmaf(-c2, rv, fmaf(i2 * to_f(dn[k].v[e]), g2[e], to_f(dr[k].v[e])));
          float bg = p.b * G;
          const float hat = yv * i1;
          const float full = bg * hat;
          ox.v[e] = from_f<T>(p.a * G);
          if constexpr (MODE == GATE_ROW) og.v[e] = from_f<T>(full * g1[e]);
          if constexpr (MODE != GATE_NONE) bg *= to_f(gt[k].v[e]);
          sum1[k * V + e] += MODE == GATE_ROW ? bg * hat : full;
          // without the norm dy does not depend on y, not even on a NaN in it
          oy.v[e] = from_f<T>(p.post ? fmaf(i1 * bg, g1[e], -c1 * yv) : bg);
        }
        const int64_t at = row * p.cols + static_cast<int64_t>(j) * V;
        *reinterpret_cast<Vec<T, V>*>(static_cast<T*>(p.dx) + at) = ox;
        *reinterpret_cast<Vec<T, V>*>(static_cast<T*>(p.dy) + at) = oy;
        if (MODE == GATE_ROW && p.dgate) *reinterpret_cast<Vec<T, V>*>(static_cast<T*>(p.dgate) + at) = og;
      }
    }
    if constexpr (MODE == GATE_SHARED) {
      over_slots(sum1);
#pragma unroll
      for (int k = 0; k < VPL; ++k) {
        const int j = tl + k * TPR;
        if (j >= nvec) continue;
        float g1[V];
        load_floats<V>(p.post ? p.g1 : nullptr, j, nvec, g1, 1.f);
        const Vec<T, V> gv = *reinterpret_cast<const Vec<T, V>*>(gate + static_cast<int64_t>(j) * V);
        Vec<T, V> og;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float P = sum1[k * V + e];
          og.v[e] = from_f<T>(P * g1[e]);
          tot1[k * V + e] = fmaf(P, to_f(gv.v[e]), tot1[k * V + e]);
          if (p.ws_gate && rl == 0) p.ws_gate[u * p.cols + static_cast<int64_t>(j) * V + e] = P * g1[e];
          sum1[k * V + e] = 0.f;
        }
        if (p.dgate && p.ws_gate == nullptr && rl == 0)
          *reinterpret_cast<Vec<T, V>*>(static_cast<T*>(p.dgate) + group * p.cols + static_cast<int64_t>(j) * V) = og;
      }
    }
  }
  if constexpr (MODE != GATE_SHARED) over_slots(sum1);
  over_slots(sum2);
  if (rl == 0) {
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
      const int j = tl + k * TPR;
      if (j >= nvec) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int64_t at = static_cast<int64_t>(blockIdx.x) * p.cols + static_cast<int64_t>(j) * V + e;
        if (p.ws_g1) p.ws_g1[at] = MODE == GATE_SHARED ? tot1[k * V + e] : sum1[k * V + e];
        if (p.ws_g2) p.ws_g2[at] = sum2[k * V + e];
      }
    }
  }
}

// any length and alignment: a block per unit, scalar accesses, each row read twice (again from L2);
// the column sums live in the block's own workspace rows (a column is always the same thread's)
template <class T, int MODE>
__global__ void __launch_bounds__(512) residual_norm_bwd_stream_kernel(const __grid_constant__ JoinBwdParams p) {
  constexpr int THREADS = 512;
  __shared__ float red[2][3][THREADS / 32];
  RowFold<THREADS, 3, THREADS> fold{red};
  const int t = threadIdx.x;
  const float inv_cols = 1.f / static_cast<float>(p.cols);
  float* s1 = p.ws_g1 ? p.ws_g1 + static_cast<int64_t>(blockIdx.x) * p.cols : nullptr;
  float* s2 = p.ws_g2 ? p.ws_g2 + static_cast<int64_t>(blockIdx.x) * p.cols : nullptr;
  for (int64_t j = t; j < p.cols; j += THREADS) {
    if (s1) s1[j] = 0.f;
    if (s2) s2[j] = 0.f;
  }
  for (int64_t u = blockIdx.x; u < p.units; u += gridDim.x) {
    const int64_t group = u / p.cuts;
    const int64_t begin = group * p.per + (u - group * p.cuts) * p.chunk;
    const int64_t end = min(begin + p.chunk, (group + 1) * p.per);
    float* sg = MODE == GATE_SHARED && p.ws_gate ? p.ws_gate + (p.cuts > 1 ? u : blockIdx.x) * p.cols : nullptr;
    if (sg)
      for (int64_t j = t; j < p.cols; j += THREADS) sg[j] = 0.f;
    for (int64_t row = begin; row < end; ++row) {
      const T* dr = p.dr ? static_cast<const T*>(p.dr) + row * p.dr_stride : nullptr;
      const T* dn = p.pre ? static_cast<const T*>(p.dn) + row * p.dn_stride : nullptr;
      const T* rr = p.pre ? static_cast<const T*>(p.r) + row * p.r_stride : nullptr;
      const T* y = p.y ? static_cast<const T*>(p.y) + row * p.y_stride : nullptr;
      const T* gt = MODE == GATE_NONE ? nullptr
                                      : static_cast<const T*>(p.gate) + (MODE == GATE_ROW ? row : group) * p.gate_stride;
      const float i1 = p.post ? p.inv1[row] : 1.f;
      const float i2 = p.pre ? p.inv2[row] : 0.f;
      float s[3] = {0.f, 0.f, 0.f};
      for (int64_t j = t; j < p.cols; j += THREADS) {
        const float d = dn ? to_f(dn[j]) : 0.f, rv = rr ? to_f(rr[j]) : 0.f, yv = y ? to_f(y[j]) : 0.f;
        float w = p.b * (p.post && p.g1 ? p.g1[j] : 1.f);
        if (gt) w *= to_f(gt[j]);
        const float dg = d * (p.pre && p.g2 ? p.g2[j] : 1.f), wy = w * yv;
        s[0] = fmaf(dg, rv, s[0]);
        s[1] = fmaf(wy, fmaf(i2, dg, dr ? to_f(dr[j]) : 0.f), s[1]);
        s[2] = fmaf(wy, rv, s[2]);
        if (s2) s2[j] = fmaf(d * i2, rv, s2[j]);
      }
      fold(s);
      const float c2 = i2 * i2 * i2 * s[0] * inv_cols;
      const float c1 = p.post ? i1 * i1 * i1 * (s[1] - c2 * s[2]) * inv_cols : 0.f;
      for (int64_t j = t; j < p.cols; j += THREADS) {
        const float d = dn ? to_f(dn[j]) : 0.f, rv = rr ? to_f(rr[j]) : 0.f, yv = y ? to_f(y[j]) : 0.f;
        const float g1 = p.post && p.g1 ? p.g1[j] : 1.f;
        const float G = fmaf(-c2, rv, fmaf(i2 * d, p.pre && p.g2 ? p.g2[j] : 1.f, dr ? to_f(dr[j]) : 0.f));
        float bg = p.b * G;
        const float hat = yv * i1, full = bg * hat;
        const int64_t at = row * p.cols + j;
        static_cast<T*>(p.dx)[at] = from_f<T>(p.a * G);
        if (MODE == GATE_ROW && p.dgate) static_cast<T*>(p.dgate)[at] = from_f<T>(full * g1);
        if (gt) bg *= to_f(gt[j]);
        if (sg) sg[j] = fmaf(full, g1, sg[j]);
        if (s1) s1[j] = fmaf(bg, hat, s1[j]);
        static_cast<T*>(p.dy)[at] = from_f<T>(p.post ? fmaf(i1 * bg, g1, -c1 * yv) : bg);
      }
    }
    if (sg && p.cuts == 1)
      for (int64_t j = t; j < p.cols; j += THREADS) static_cast<T*>(p.dgate)[group * p.cols + j] = from_f<T>(sg[j]);
  }
}

// Column sums of partial rows in a fixed order: blockIdx.y 0 and 1 fold dgamma_post and
// dgamma_pre over the blocks' rows, the others a gate row each over its units.  A block owns a strip of 8
// columns (one 32-byte sector per partial row); its 256 threads take 32 rows per step.
struct JoinFoldParams {
  float* out1;
  float* out2;
  void* dgate;
  const float* ws1;
  const float* ws2;
  const float* ws_gate;
  int64_t cols, parts, cuts, gates;
  int first;  // what blockIdx.y == 0 stands for
};
template <class T>
__global__ void __launch_bounds__(256) residual_norm_fold_kernel(const __grid_constant__ JoinFoldParams p) {
  __shared__ float sm[8][8];
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x & 7);
  for (int64_t what = blockIdx.y + p.first; what < p.gates + 2; what += gridDim.y) {
    if ((what == 0 && !p.out1) || (what == 1 && !p.out2)) continue;
    const float* src = what == 0 ? p.ws1 : what == 1 ? p.ws2 : p.ws_gate + (what - 2) * p.cuts * p.cols;
    const int64_t n = what < 2 ? p.parts : p.cuts;
    const float s = strip_sum(src, n, p.cols, sm);
    if (threadIdx.x < 8 && c < p.cols) {
      if (what == 0) p.out1[c] = s;
      else if (what == 1) p.out2[c] = s;
      else static_cast<T*>(p.dgate)[(what - 2) * p.cols + c] = from_f<T>(s);
    }
    __syncthreads();
  }
}

constexpr int kBwdEltsPerThread(int elt) { return elt == 2 ? 16 : 8; }
// threads per row of the backward for rows of `cols` values; 0: the stream kernel
inline int join_bwd_tpr(int64_t cols, int elt) {
  const int e = kBwdEltsPerThread(elt);
  for (int tpr : {8, 32, 128, 256, 512})
    if (cols <= int64_t{tpr} * e) return tpr;
  return 0;
}
// how the rows are cut: units of `chunk` rows, `cuts` of them per gate row, on `blocks` blocks.
// As many units as the card has block slots, unless that leaves a block less than two rows.
struct JoinCut {
  int64_t chunk, cuts, units, blocks;
};
inline JoinCut join_cut(int64_t rows, int64_t per, int sms) {
  const int64_t groups = rows / per, target = int64_t{sms} * 4;
  JoinCut c;
  c.cuts = std::max<int64_t>(1, std::min<int64_t>((per + 1) / 2, (target + groups - 1) / groups));
  c.chunk = (per + c.cuts - 1) / c.cuts;
  c.cuts = (per + c.chunk - 1) / c.chunk;
  c.units = groups * c.cuts;
  c.blocks = std::min<int64_t>(c.units, target);
  return c;
}

template <class T>
vbt_b200_status launch_join_bwd(JoinBwdParams p, int mode, float* dg1, float* dg2, float* ws, cudaStream_t s, int device) {
  constexpr int VW = 16 / sizeof(T);
  constexpr int E = kBwdEltsPerThread(sizeof(T));
  const JoinCut cut = join_cut(p.rows, p.per, sm_count(device));
  p.chunk = cut.chunk; p.cuts = cut.cuts; p.units = cut.units;
  const unsigned g = static_cast<unsigned>(cut.blocks);
  float* at = ws;
  if (dg1) { p.ws_g1 = at; at += cut.blocks * p.cols; }
  if (dg2) { p.ws_g2 = at; at += cut.blocks * p.cols; }
  const bool split_gate = mode == GATE_SHARED && p.dgate != nullptr && cut.cuts > 1;
  const int tpr = join_bwd_tpr(p.cols, sizeof(T));
  // the stream kernel sums a gate row in memory even where it has all its rows
  if (split_gate || (mode == GATE_SHARED && p.dgate != nullptr && tpr == 0)) p.ws_gate = at;
  const bool vec = p.cols % VW == 0 && p.dr_stride % VW == 0 && p.dn_stride % VW == 0 && p.y_stride % VW == 0 &&
                   p.r_stride % VW == 0 && p.gate_stride % VW == 0 && a16(p.dr) && a16(p.dn) && a16(p.y) && a16(p.r) &&
                   a16(p.gate) && a16(p.dx) && a16(p.dy) && a16(p.dgate) && a16(p.g1) && a16(p.g2);
  int threads = 512;
#define VB_JB(V, TPR, MODE)                                                                    \
  do {                                                                                         \
    threads = TPR < 128 ? 128 : TPR;                                                           \
    residual_norm_bwd_kernel<T, V, E / V, TPR, MODE><<<g, threads, 0, s>>>(p);                 \
  } while (0)
#define VB_JB_LADDER(V, MODE)                 \
  switch (tpr) {                              \
    case 8: VB_JB(V, 8, MODE); break;         \
    case 32: VB_JB(V, 32, MODE); break;       \
    case 128: VB_JB(V, 128, MODE); break;     \
    case 256: VB_JB(V, 256, MODE); break;     \
    case 512: VB_JB(V, 512, MODE); break;     \
    default: residual_norm_bwd_stream_kernel<T, MODE><<<g, threads, 0, s>>>(p); \
  }
#define VB_JB_MODE(MODE)                  \
  if (vec) { VB_JB_LADDER(VW, MODE); }    \
  else { VB_JB_LADDER(1, MODE); }
  if (mode == GATE_NONE) { VB_JB_MODE(GATE_NONE); }
  else if (mode == GATE_SHARED) { VB_JB_MODE(GATE_SHARED); }
  else { VB_JB_MODE(GATE_ROW); }
#undef VB_JB_MODE
#undef VB_JB_LADDER
#undef VB_JB
  VB_LAUNCH_CHECK();
  int launches = 1;
  if (dg1 || dg2 || split_gate) {
    JoinFoldParams f{};
    f.out1 = dg1; f.out2 = dg2; f.dgate = p.dgate;
    f.ws1 = p.ws_g1; f.ws2 = p.ws_g2; f.ws_gate = p.ws_gate;
    f.cols = p.cols; f.parts = cut.blocks; f.cuts = cut.cuts; f.gates = split_gate ? p.rows / p.per : 0;
    f.first = dg1 ? 0 : dg2 ? 1 : 2;
    const int64_t ny = f.gates + 2 - f.first;
    dim3 fg(static_cast<unsigned>((p.cols + 7) / 8), static_cast<unsigned>(std::min<int64_t>(ny, 65535)));
    residual_norm_fold_kernel<T><<<fg, 256, 0, s>>>(f);
    VB_LAUNCH_CHECK();
    ++launches;
  }
  note_launch(VBT_B200_FAMILY_ROWOP, VBT_B200_WK_RESIDUAL_NORM_BACKWARD, dim3(g), dim3(threads), vec ? VW : 1,
              static_cast<int>(cut.cuts), 0, launches, p.rows * p.cols, p.cols, 0, s);
  return VBT_B200_OK;
}

}  // namespace
}  // namespace vb

extern "C" {

vbt_b200_status vbt_b200_residual_norm(void* r, void* n, float* inv_post, float* inv_pre, const void* x, const void* y,
                                       const float* gamma_post, const void* gate, const float* gamma_pre,
                                       int32_t dtype, int64_t rows, int64_t cols, int64_t x_row_stride,
                                       int64_t y_row_stride, int64_t gate_row_stride, int64_t rows_per_gate,
                                       float residual_scale, float branch_scale, float eps, int32_t flags,
                                       void* stream) {
  using namespace vb;
  const char* name = "residual_norm";
  VB_ARG(rows >= 0 && cols >= 0, std::string(name) + ": negative size");
  VB_ARG(is_float_dtype(dtype), std::string(name) + ": expected a floating dtype");
  if (rows == 0 || cols == 0) return VBT_B200_OK;
  const bool pre = flags & VBT_B200_RESNORM_PRE, post = flags & VBT_B200_RESNORM_POST;
  VB_ARG(x && y && r && (n || !pre), std::string(name) + ": null pointer");
  VB_ARG(x_row_stride >= 0 && y_row_stride >= 0 && gate_row_stride >= 0, std::string(name) + ": negative row stride");
  VB_ARG(gate == nullptr || (rows_per_gate > 0 && rows % rows_per_gate == 0),
         std::string(name) + ": rows_per_gate does not divide rows");
  DeviceScope scope(r);
  JoinParams p{};
  p.x = x; p.y = y; p.g1 = gamma_post; p.gate = gate; p.g2 = gamma_pre;
  p.r = r; p.n = pre ? n : nullptr; p.inv1 = inv_post; p.inv2 = inv_pre;
  p.rows = rows; p.cols = cols; p.x_stride = x_row_stride; p.y_stride = y_row_stride;
  p.gate_stride = gate ? gate_row_stride : 0;
  p.per = gate ? rows_per_gate : rows;
  p.small_rows = rows < (int64_t{1} << 31);
  if (p.small_rows) p.per_div = FastDiv(static_cast<uint32_t>(p.per));
  p.a = residual_scale; p.b = branch_scale; p.eps = eps; p.post = post; p.pre = pre;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case VBT_B200_F32: return launch_join<float>(p, s, scope.device());
    case VBT_B200_F16: return launch_join<__half>(p, s, scope.device());
    default: return launch_join<__nv_bfloat16>(p, s, scope.device());
  }
}

vbt_b200_status vbt_b200_residual_norm_backward_workspace_bytes(int64_t rows, int64_t cols, int32_t dtype,
                                                                int64_t rows_per_gate, int32_t device,
                                                                size_t* bytes) {
  using namespace vb;
  const char* name = "residual_norm_backward";
  VB_ARG(bytes != nullptr, std::string(name) + ": null output");
  VB_ARG(rows >= 0 && cols >= 0, std::string(name) + ": negative size");
  VB_ARG(is_float_dtype(dtype), std::string(name) + ": expected a floating dtype");
  VB_ARG(rows == 0 || (rows_per_gate > 0 && rows % rows_per_gate == 0),
         std::string(name) + ": rows_per_gate does not divide rows");
  *bytes = 0;
  if (rows == 0) return VBT_B200_OK;
  // a gate row of its own per row is no sum over rows: the rows are cut as if one gate row served all
  const JoinCut c = join_cut(rows, rows_per_gate == 1 ? rows : rows_per_gate, sm_count(device));
  *bytes = static_cast<size_t>(2 * c.blocks + (c.cuts > 1 ? c.units : c.blocks)) * static_cast<size_t>(cols) * 4;
  return VBT_B200_OK;
}

vbt_b200_status vbt_b200_residual_norm_backward(
    void* dx, void* dy, float* dgamma_post, void* dgate, float* dgamma_pre, const void* dr, const void* dn,
    const void* y, const void* r, const float* inv_post, const float* inv_pre, const float* gamma_post,
    const void* gate, const float* gamma_pre, int32_t dtype, int64_t rows, int64_t cols, int64_t dr_row_stride,
    int64_t dn_row_stride, int64_t y_row_stride, int64_t r_row_stride, int64_t gate_row_stride,
    int64_t rows_per_gate, float residual_scale, float branch_scale, int32_t flags, void* workspace,
    size_t workspace_bytes, void* stream) {
  using namespace vb;
  const char* name = "residual_norm_backward";
  VB_ARG(rows >= 0 && cols >= 0, std::string(name) + ": negative size");
  VB_ARG(is_float_dtype(dtype), std::string(name) + ": expected a floating dtype");
  const bool pre = flags & VBT_B200_RESNORM_PRE, post = flags & VBT_B200_RESNORM_POST;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (cols == 0) return VBT_B200_OK;
  VB_ARG(dgate == nullptr || gate != nullptr, std::string(name) + ": dgate without a gate");
  VB_ARG(dgamma_post == nullptr || post, std::string(name) + ": dgamma_post without the norm behind the branch");
  VB_ARG(dgamma_pre == nullptr || pre, std::string(name) + ": dgamma_pre without the norm in front of the next block");
  VB_ARG(gate == nullptr || (rows_per_gate > 0 && rows % rows_per_gate == 0),
         std::string(name) + ": rows_per_gate does not divide rows");
  if (rows == 0) {  // sums over no rows; a gate shared by no rows has no gradient rows either
    for (float* o : {dgamma_post, dgamma_pre})
      if (o) {
        DeviceScope scope(o);
        VB_CUDA(cudaMemsetAsync(o, 0, static_cast<size_t>(cols) * 4, s));
      }
    return VBT_B200_OK;
  }
  VB_ARG(dx && dy && (dn || dr), std::string(name) + ": null pointer");
  VB_ARG(!pre || (dn && r && inv_pre), std::string(name) + ": the norm in front of the next block needs dn, r and inv_pre");
  VB_ARG(!post || (y && inv_post), std::string(name) + ": the norm behind the branch needs y and inv_post");
  VB_ARG(dgate == nullptr || y != nullptr, std::string(name) + ": dgate needs y");
  VB_ARG(dr_row_stride >= 0 && dn_row_stride >= 0 && y_row_stride >= 0 && r_row_stride >= 0 && gate_row_stride >= 0,
         std::string(name) + ": negative row stride");
  DeviceScope scope(dx);
  const int mode = gate == nullptr ? GATE_NONE : rows_per_gate == 1 && rows > 1 ? GATE_ROW : GATE_SHARED;
  size_t need = 0;
  VB_TRY(vbt_b200_residual_norm_backward_workspace_bytes(rows, cols, dtype, gate ? rows_per_gate : rows, scope.device(), &need));
  VB_ARG((dgamma_post == nullptr && dgamma_pre == nullptr && dgate == nullptr) ||
             (workspace != nullptr && workspace_bytes >= need),
         std::string(name) + ": workspace too small (see vbt_b200_residual_norm_backward_workspace_bytes)");
  JoinBwdParams p{};
  p.dr = dr; p.dn = pre ? dn : nullptr; p.y = y; p.r = pre ? r : nullptr;
  p.inv1 = inv_post; p.inv2 = inv_pre; p.g1 = gamma_post; p.gate = gate; p.g2 = gamma_pre;
  p.dx = dx; p.dy = dy; p.dgate = dgate;
  p.rows = rows; p.cols = cols;
  p.dr_stride = dr ? dr_row_stride : 0; p.dn_stride = pre ? dn_row_stride : 0; p.y_stride = y ? y_row_stride : 0;
  p.r_stride = pre ? r_row_stride : 0; p.gate_stride = gate ? gate_row_stride : 0;
  p.per = mode == GATE_SHARED ? rows_per_gate : rows;
  p.a = residual_scale; p.b = branch_scale; p.post = post; p.pre = pre;
  float* ws = static_cast<float*>(workspace);
  switch (dtype) {
    case VBT_B200_F32: return launch_join_bwd<float>(p, mode, dgamma_post, dgamma_pre, ws, s, scope.device());
    case VBT_B200_F16: return launch_join_bwd<__half>(p, mode, dgamma_post, dgamma_pre, ws, s, scope.device());
    default: return launch_join_bwd<__nv_bfloat16>(p, mode, dgamma_post, dgamma_pre, ws, s, scope.device());
  }
}

}  // extern "C"

// Backward of residual_norm (sm_100a):
//
//   G   = dr + i2 * (dn * g2) - r * i2^3 * mean(dn * g2 * r)
//   dx  = a * G                         dg2   = sum_rows dn * r * i2
//   dv  = b * G * gate                  dgate = sum_(rows of the gate row) b * G * y * i1 * g1
//   dy  = i1 * dv * g1 - y * i1^3 * mean(dv * g1 * y)       dg1 = sum_rows dv * y * i1
//
// The second mean needs G, which needs the first.  It splits into sums that do not:
//   sum(dv g1 y) = sum(w y (dr + i2 dn g2)) - c i2 sum(w y r),  w = b gate g1, c = i2^2 mean(dn g2 r),
// so a row costs one reduction of three sums.
// A product of several i leaves the normal numbers for rows far from one (i^3 does for an rms above 5e12
// or below 2e-13).  Such rows, told by their i, are brought near one in place by i's power of two, which
// rounds nothing: r i = (r 2^k) (i 2^-k).  A factor per value instead, i (r i), took 4 to 8 % longer.
//
// Bound by memory and, close behind, by instructions: four rows read, two written, 14 fp32 operations
// and six conversions per value.  [32768,4096] bf16 with a gate row per 4096 rows takes 295 us = 5.5
// TB/s, 0.83 of the measured copy bandwidth (16 warps per SM at 128 registers, half of the issue slots
// busy).  What it came through: rows in registers 678 us; staged by asynchronous copies 370; one base per
// warp and compile-time offsets instead of an address per access (744 instructions per warp and row
// against 964) 314; units of neighbouring rows rather than every n-th one 306 (379).  Arithmetic on
// float pairs was slower here (335: moves to pair the registers), and so were one block per SM with
// four rows in flight (759), eight values per thread (424), and one row in flight (333).
#include <algorithm>

#include "row_tile.cuh"

namespace vb {
namespace {

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
  float* ws_g1;      // [workers][cols] partial sums of dgamma_post, or null
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
  int ranks;         // blocks that share a row
};

// A worker (a warp when TPR lanes of it share a row, else the block) walks a range of neighbouring
// units, each a run of rows that share one gate row.  Rows arrive in shared memory by asynchronous
// copies, `stages` rows ahead; a thread reads back only what it copied itself, once for the three
// sums and once for the outputs, so a row needs no barrier but the one of its reduction, and no
// registers between the two passes.  w = b * gate * g1 and g2 lie beside them.
// The sum over a unit of G * y * i1 gives the gate's gradient (times b * g1) and the unit's part of
// dgamma_post (times b * gate).  A gate row of its own per row (GATE_ROW) is a factor of the sum.
// Values of a row per thread: two sums per column and the gradient at r stay in registers for each.  Single
// values: 16-bit ones fare better with sixteen ([16384,4095] bf16, a gate row per 2048: 251 us, 364 with eight),
// 32-bit ones with eight where blocks are small ([6151,1365], a gate row for all: 69 us, 75 with sixteen; not
// [8192,4095] without a gate, 194 and 179).
constexpr int kVecElts = 16;
template <class T> constexpr int kSingleElts = sizeof(T) == 2 ? 16 : 8;
constexpr int kBwdMaxThreads = 512;   // of a block that shares a row

// A row is far from one if its i is.  16-bit floats of five exponent bits never are.
template <class T> __device__ __forceinline__ bool far_row(float i) {
  if constexpr (std::is_same_v<T, __half>) return false;
  return (i > 0x1p25f && i < __int_as_float(0x7f800000)) || (i < 0x1p-25f && i >= 0x1p-126f);
}
__device__ __forceinline__ float power_of_two(float i) { return __int_as_float(__float_as_int(i) & 0x7f800000); }

template <class T, int V, int TPR, int MODE, int STAGES>
__global__ void __launch_bounds__(TPR ? 256 : kBwdMaxThreads, TPR ? 2 : 1) residual_norm_bwd_kernel(const __grid_constant__ JoinBwdParams p) {
  constexpr int E = V > 1 ? kVecElts : kSingleElts<T>;
  using A = RowChunks<T, V, TPR, E>;
  constexpr int C = A::C;
  constexpr int RW = TPR ? 32 / TPR : 1;                 // rows a worker takes at once
  constexpr int ARRAYS = MODE == GATE_ROW ? 5 : 4;       // dr, dn, r, y, gate
  extern __shared__ __align__(16) unsigned char smem[];
  const int ranks = TPR ? 1 : p.ranks;
  const int warp0 = ranks > 1 ? cluster_rank() * static_cast<int>(blockDim.x >> 5) : 0;
  if (ranks > 1) cluster_sync();  // the other blocks' shared memory is there
  const int rl = TPR ? static_cast<int>(threadIdx.x & 31) / A::STEP : 0;
  const int j0 = A::base(warp0), left = static_cast<int>(p.cols) - j0;
  const float inv_cols = 1.f / static_cast<float>(p.cols);
  // a warp's part of the shared memory: w, g2, then STAGES times the arrays
  unsigned char* wbuf = smem + static_cast<size_t>(threadIdx.x >> 5) * (2 * A::WARP_FACTORS + STAGES * ARRAYS * A::WARP_ARRAY);
  float4* red = reinterpret_cast<float4*>(smem + static_cast<size_t>(blockDim.x >> 5) *
                                                     (2 * A::WARP_FACTORS + STAGES * ARRAYS * A::WARP_ARRAY));
  unsigned char* gbuf = wbuf + A::WARP_FACTORS;
  unsigned char* ring = gbuf + A::WARP_FACTORS;
  auto buf = [&](int stage, int array) { return ring + stage * (ARRAYS * A::WARP_ARRAY) + array * A::WARP_ARRAY; };
  for (int st = 0; st < STAGES; ++st)
#pragma unroll
    for (int a = 0; a < ARRAYS; ++a) {
      const bool present = a == 0 ? p.dr != nullptr : a == 3 ? p.y != nullptr : a == 4 || p.pre;
      A::zero_rest(buf(st, a), present, left);
    }
  A::sync();
  const int seg = A::segment(warp0), seg_left = static_cast<int>(p.cols) - seg;
  const float* g1 = p.post && p.g1 ? p.g1 + j0 : nullptr;
  const float* g2p = p.pre && p.g2 ? p.g2 + j0 : nullptr;
  A::fill_factors(gbuf, left, [&](int o) { return g2p ? g2p[o] : 1.f; });
  if constexpr (MODE != GATE_SHARED) A::fill_factors(wbuf, left, [&](int o) { return p.b * (g1 ? g1[o] : 1.f); });

  const int64_t worker = TPR ? static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32 : blockIdx.x / ranks;
  const int64_t workers = TPR ? static_cast<int64_t>(gridDim.x) * (blockDim.x / 32) : gridDim.x / ranks;
  // the worker's units [u, last) are one run of rows; a unit's rows are taken RW at a time
  struct Walk {
    int u;
    int todo, left;  // rows of the worker, rows of the unit still to take
    __device__ __forceinline__ void enter(const JoinBwdParams& q) {
      const int cut = u % static_cast<int>(q.cuts);
      left = static_cast<int>(min(q.chunk, q.per - cut * q.chunk));
    }
    // takes the next rows; returns how many
    __device__ __forceinline__ int next(const JoinBwdParams& q) {
      const int n = RW == 1 ? 1 : min(RW, left);
      todo -= n;
      left -= n;
      if (left == 0 && todo > 0) { ++u; enter(q); }
      return n;
    }
  };
  const int64_t u0 = worker * p.units / workers, u1 = (worker + 1) * p.units / workers;
  auto first_row = [&](int64_t u) {
    const int64_t group = u / p.cuts;
    return group * p.per + (u - group * p.cuts) * p.chunk;
  };
  const int row0 = static_cast<int>(first_row(u0)) + rl;  // rows are fewer than 2^31
  Walk at;
  at.u = static_cast<int>(u0);
  at.left = 0;
  at.todo = u0 < u1 ? static_cast<int>(first_row(u1) - first_row(u0)) : 0;
  if (at.todo) at.enter(p);
  Walk ahead = at;
  // rows are addressed from their number: a running pointer per array is 20 registers of the 128
  int row = row0, row_ahead = row0;
  auto at_row = [&](const void* base, int64_t stride, int r) { return static_cast<const T*>(base) + r * stride + seg; };
  float i1_next[STAGES], i2_next[STAGES];
  const int row_end = row0 + at.todo;
  auto fetch = [&](int stage, float& i1, float& i2) {
    i1 = 1.f;
    i2 = 0.f;
    if (RW == 1 ? row_ahead < row_end : ahead.todo > 0) {
      if (RW == 1 || rl < ahead.left) {
        if (p.dr) A::copy(buf(stage, 0), at_row(p.dr, p.dr_stride, row_ahead), seg_left, p.dr);
        if (p.pre) {
          A::copy(buf(stage, 1), at_row(p.dn, p.dn_stride, row_ahead), seg_left, p.dn);
          A::copy(buf(stage, 2), at_row(p.r, p.r_stride, row_ahead), seg_left, p.r);
          i2 = p.inv2[row_ahead];
        }
        if (p.y) A::copy(buf(stage, 3), at_row(p.y, p.y_stride, row_ahead), seg_left, p.y);
        if constexpr (MODE == GATE_ROW) A::copy(buf(stage, 4), at_row(p.gate, p.gate_stride, row_ahead), seg_left, p.gate);
        if (p.post) i1 = p.inv1[row_ahead];
      }
      // the rows of a worker follow one another; several at once stop at a unit's end
      if constexpr (RW == 1) ++row_ahead;
      else row_ahead += ahead.next(p);
    }
    copy_commit();
  };
#pragma unroll
  for (int q = 0; q < STAGES; ++q) fetch(q, i1_next[q], i2_next[q]);

  float sum1[E], sum2[E];
#pragma unroll
  for (int i = 0; i < E; ++i) sum1[i] = sum2[i] = 0.f;
  // adds the values of a worker's RW rows; every lane gets the result
  auto over_rows = [&](float (&v)[E]) {
    if constexpr (RW > 1) {
#pragma unroll
      for (int i = 0; i < E; ++i)
#pragma unroll
        for (int d = TPR; d < 32; d <<= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], d);
    }
  };
  // the gate row of unit u, from this thread's first column on
  auto gate_of = [&](int u) { return static_cast<const T*>(p.gate) + u / static_cast<int>(p.cuts) * p.gate_stride + j0; };
  bool first_unit = true, enter = true;
  int phase = 0, stage = 0;
  while (at.todo > 0) {
    if constexpr (MODE == GATE_SHARED) {
      if (enter) {
        const T* gate = gate_of(at.u);
        A::fill_factors(wbuf, left, [&](int o) { return p.b * (g1 ? g1[o] : 1.f) * to_f(gate[o]); });
      }
    }
    copy_wait<STAGES - 1>();
    A::sync();
    const bool live = RW == 1 || rl < at.left;
    const float i2 = i2_next[0];
    float i1 = i1_next[0], ir = i2;  // of the rows as they lie in shared memory
    const bool far_y = far_row<T>(i1);
    if (far_y || far_row<T>(i2)) {
      if (live && far_y) A::scale(buf(stage, 3), A::shift(p.y, p.y_stride, row), left, power_of_two(i1));
      if (live && far_row<T>(i2)) A::scale(buf(stage, 2), A::shift(p.r, p.r_stride, row), left, power_of_two(i2));
      if (far_y) i1 /= power_of_two(i1);
      if (far_row<T>(i2)) ir /= power_of_two(i2);
    }
    float s[3] = {0.f, 0.f, 0.f};
    float up[E];  // dr + i2 dn g2, kept for the second pass
    if (live) {
#pragma unroll
      for (int c = 0; c < A::N; ++c) {
        float dr[C], dn[C], r[C], y[C], w[C], g2[C];
        A::read(buf(stage, 0), A::shift(p.dr, p.dr_stride, row), c, dr);
        A::read(buf(stage, 1), A::shift(p.dn, p.dn_stride, row), c, dn);
        A::read(buf(stage, 2), A::shift(p.r, p.r_stride, row), c, r);
        A::read(buf(stage, 3), A::shift(p.y, p.y_stride, row), c, y);
        A::read_factors(wbuf, c, w);
        A::read_factors(gbuf, c, g2);
        if constexpr (MODE == GATE_ROW) {
          float gt[C];
          A::read(buf(stage, 4), A::shift(p.gate, p.gate_stride, row), c, gt);
#pragma unroll
          for (int e = 0; e < C; ++e) w[e] *= gt[e];
        }
#pragma unroll
        for (int e = 0; e < C; ++e) {
          const int i = c * C + e;
          const float dnr = dn[e] * r[e], wy = w[e] * y[e];
          up[i] = fmaf(i2, dn[e] * g2[e], dr[e]);
          s[0] = fmaf(dnr, g2[e], s[0]);
          s[1] = fmaf(wy, up[i], s[1]);
          s[2] = fmaf(wy, r[e], s[2]);
          sum2[i] = fmaf(dnr, ir, sum2[i]);
        }
      }
    }
    sum_row<TPR, 3>(s, red, phase, p.ranks);
    const float c2 = (i2 * inv_cols) * ir * (ir * s[0]);
    const float c1 = p.post ? (i1 * inv_cols) * i1 * (i1 * (s[1] - c2 * s[2])) : 0.f;
    if (live) {
      const int64_t o = static_cast<int64_t>(row) * p.cols + j0;
#pragma unroll
      for (int c = 0; c < A::N; ++c) {
        float r[C], y[C], w[C], gt[C], ox[C], oy[C], og[C];
        A::read(buf(stage, 2), A::shift(p.r, p.r_stride, row), c, r);
        A::read(buf(stage, 3), A::shift(p.y, p.y_stride, row), c, y);
        A::read_factors(wbuf, c, w);
        if constexpr (MODE == GATE_ROW) A::read(buf(stage, 4), A::shift(p.gate, p.gate_stride, row), c, gt);
#pragma unroll
        for (int e = 0; e < C; ++e) {
          const int i = c * C + e;
          const float G = fmaf(-c2, r[e], up[i]), Gi = G * i1;
          ox[e] = p.a * G;
          if constexpr (MODE == GATE_ROW) {
            const float Gy = Gi * y[e];
            og[e] = Gy * w[e];
            sum1[i] = fmaf(Gy, gt[e], sum1[i]);
            w[e] *= gt[e];
          } else {
            sum1[i] = fmaf(Gi, y[e], sum1[i]);
          }
          // without the norm (c1 = 0, i1 = 1) dy does not depend on y, not even on a NaN in it
          oy[e] = p.post ? fmaf(Gi, w[e], -c1 * y[e]) : Gi * w[e];
        }
        A::write(static_cast<T*>(p.dx) + o, c, left, ox);
        A::write(static_cast<T*>(p.dy) + o, c, left, oy);
        if constexpr (MODE == GATE_ROW) {
          if (p.dgate) A::write(static_cast<T*>(p.dgate) + o, c, left, og);
        }
      }
      // dy = i (G w - ..) came out with i 2^-k
      if (far_y) A::scale_row(static_cast<T*>(p.dy) + o, left, power_of_two(p.inv1[row]));
    }
#pragma unroll
    for (int q = 0; q + 1 < STAGES; ++q) {
      i1_next[q] = i1_next[q + 1];
      i2_next[q] = i2_next[q + 1];
    }
    A::sync();
    fetch(stage, i1_next[STAGES - 1], i2_next[STAGES - 1]);
    stage = stage + 1 == STAGES ? 0 : stage + 1;
    const int unit = at.u;
    row += at.next(p);
    enter = at.todo == 0 || at.u != unit;
    if constexpr (MODE == GATE_SHARED) {
      if (!enter) continue;
      over_rows(sum1);
      const int64_t group = unit / static_cast<int>(p.cuts);
      const T* gate = gate_of(unit);
      if (rl == 0) {
#pragma unroll
        for (int c = 0; c < A::N; ++c) {
          float og[C];
#pragma unroll
          for (int e = 0; e < C; ++e) {
            const int o = A::off(c, e);
            const float P = p.b * sum1[c * C + e];
            const float Pg = o < left && g1 ? P * g1[o] : P;
            og[e] = Pg;
            if (o >= left) continue;
            if (p.ws_gate) p.ws_gate[unit * p.cols + j0 + o] = Pg;
            if (p.ws_g1) {  // the worker's running part, in its own row
              float* part = p.ws_g1 + worker * p.cols + j0 + o;
              *part = (first_unit ? 0.f : *part) + P * to_f(gate[o]);
            }
          }
          if (p.dgate && p.ws_gate == nullptr)
            A::write(static_cast<T*>(p.dgate) + group * p.cols + j0, c, left, og);
        }
      }
      first_unit = false;
#pragma unroll
      for (int i = 0; i < E; ++i) sum1[i] = 0.f;
    }
  }
  copy_wait<0>();
  if (ranks > 1) cluster_sync();  // no block leaves while another may still write to its shared memory
  if constexpr (MODE != GATE_SHARED) over_rows(sum1);
  over_rows(sum2);
  if (rl == 0) {
#pragma unroll
    for (int c = 0; c < A::N; ++c)
#pragma unroll
      for (int e = 0; e < C; ++e) {
        if (A::off(c, e) >= left) continue;
        const int64_t o = worker * p.cols + j0 + A::off(c, e);
        if (p.ws_g1) {
          if constexpr (MODE == GATE_SHARED) {
            if (first_unit) p.ws_g1[o] = 0.f;  // a worker without rows
          } else {
            p.ws_g1[o] = p.b * sum1[c * C + e];
          }
        }
        if (p.ws_g2) p.ws_g2[o] = sum2[c * C + e];
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
      const float c2 = (i2 * inv_cols) * (i2 * s[0]);
      const float c1 = p.post ? (i1 * inv_cols) * (i1 * (s[1] - c2 * (i2 * s[2]))) : 0.f;
      for (int64_t j = t; j < p.cols; j += THREADS) {
        const float d = dn ? to_f(dn[j]) : 0.f, rv = rr ? to_f(rr[j]) : 0.f, yv = y ? to_f(y[j]) : 0.f;
        const float g1 = p.post && p.g1 ? p.g1[j] : 1.f;
        const float G = fmaf(-c2, rv * i2, fmaf(i2 * d, p.pre && p.g2 ? p.g2[j] : 1.f, dr ? to_f(dr[j]) : 0.f));
        float bg = p.b * G;
        const float hat = yv * i1, full = bg * hat;
        const int64_t at = row * p.cols + j;
        static_cast<T*>(p.dx)[at] = from_f<T>(p.a * G);
        if (MODE == GATE_ROW && p.dgate) static_cast<T*>(p.dgate)[at] = from_f<T>(full * g1);
        if (gt) bg *= to_f(gt[j]);
        if (sg) sg[j] = fmaf(full, g1, sg[j]);
        if (s1) s1[j] = fmaf(bg, hat, s1[j]);
        static_cast<T*>(p.dy)[at] = from_f<T>(p.post ? fmaf(i1 * bg, g1, -c1 * hat) : bg);
      }
    }
    if (sg && p.cuts == 1)
      for (int64_t j = t; j < p.cols; j += THREADS) static_cast<T*>(p.dgate)[group * p.cols + j] = from_f<T>(sg[j]);
  }
}

// Column sums of partial rows in a fixed order.  blockIdx.y says which: dgamma_post and dgamma_pre over the
// workers' rows, the gradient of one gate row that serves all over its units.
struct JoinFoldParams {
  float* out[2];
  const float* ws[2];
  void* dgate;
  const float* ws_gate;
  int64_t cols, parts, cuts;
  int what[3];
};
template <class T>
__global__ void __launch_bounds__(kStripThreads) residual_norm_fold_kernel(const __grid_constant__ JoinFoldParams p) {
  __shared__ float sm[kStripThreads / 32][8];
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 8 + threadIdx.x;
  const int what = p.what[blockIdx.y];
  const float s = what < 2 ? strip_sum(p.ws[what], p.parts, p.cols, sm) : strip_sum(p.ws_gate, p.cuts, p.cols, sm);
  if (threadIdx.x < 8 && c < p.cols) {
    if (what < 2) p.out[what][c] = s;
    else static_cast<T*>(p.dgate)[c] = from_f<T>(s);
  }
}
// Several gate rows, few units each: 32 columns per block, eight warps take every eighth unit.
template <class T>
__global__ void __launch_bounds__(256) residual_norm_gate_fold_kernel(T* dgate, const float* ws, int64_t cuts, int64_t cols,
                                                                      int64_t gates) {
  __shared__ float sm[8][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  for (int64_t g = blockIdx.y; g < gates; g += gridDim.y) {
    const float* src = ws + g * cuts * cols + c;
    float acc = 0.f;
    if (c < cols) {
      for (int64_t r = w; r < cuts; r += 8 * 8) {
        float v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = r + 8 * q < cuts ? __ldcg(src + (r + 8 * q) * cols) : 0.f;
#pragma unroll
        for (int q = 0; q < 8; ++q) acc += v[q];
      }
    }
    sm[w][lane] = acc;
    __syncthreads();
    if (w == 0 && c < cols) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) s += sm[k][lane];
      dgate[g * cols + c] = from_f<T>(s);
    }
    __syncthreads();
  }
}

// How the backward runs: `tpr` lanes of a warp share a row, or (0) `ranks` blocks of `threads` do; what
// eight blocks cannot hold takes the stream kernel (threads == 0).
struct JoinShape {
  int tpr, threads, stages, smem, per_sm, ranks;
  int workers() const { return tpr ? threads / 32 : 1; }
  // workers on the card at once
  int64_t most(int sms) const {
    return ranks > 1 ? clusters_at_once(sms * per_sm, ranks) : int64_t{sms} * per_sm * (threads ? workers() : 1);
  }
};
inline JoinShape join_bwd_shape(int64_t cols, int elt, bool gate_row, bool vec) {
  JoinShape h{0, 0, 0, 0, 4, 1};
  const int elts = vec ? kVecElts : elt == 2 ? kSingleElts<__half> : kSingleElts<float>;
  const int64_t lanes = (cols + elts - 1) / elts;
  if (lanes > int64_t{kBwdMaxThreads} * kMaxRanks) return h;
  h.tpr = lanes <= 8 ? 8 : lanes <= 16 ? 16 : lanes <= 32 ? 32 : 0;
  const int factors = 2 * elts * 4, row = (gate_row ? 5 : 4) * row_bytes_per_thread(elts, elt, vec, h.tpr);
  auto smem = [&](int stages) { return h.threads * (factors + stages * row) + (h.tpr ? 0 : sum_bytes(h.ranks)); };
  for (h.ranks = 1; h.ranks <= kMaxRanks; h.ranks *= 2) {
    const int64_t part = (lanes + h.ranks - 1) / h.ranks;
    h.threads = h.tpr ? 256 : static_cast<int>((part + 31) / 32 * 32);
    // Few blocks of many threads: of [8192,16384] bf16 without a gate, two per row against four with 256 threads
    // each, 427 us and 486; fp32 [4096,16384] 316 and 431.  With a gate row per 1024 rows, whose units end
    // often, 605 and 527.
    if (h.threads > kBwdMaxThreads) continue;
    // two rows ahead where they fit; the warp forms are built for that alone
    h.stages = 2;
    if (!h.tpr && smem(2) > kSmemPerBlock) h.stages = 1;
    h.smem = smem(h.stages);
    if (h.smem > kSmemPerBlock) continue;
    // registers allow 512 threads per SM (128 each)
    h.per_sm = std::max(1, std::min(512 / h.threads, kSmemPerSm / (h.smem + 1024)));
    return h;
  }
  return JoinShape{0, 0, 0, 0, 4, 1};
}
// How the rows are cut: units of `chunk` rows, `cuts` of them per gate row, dealt out evenly to the
// workers that fit the card.  At least as many units as workers, and up to eight times that where it
// evens out what a worker gets (30 gate rows of 1000 rows of 4096 on 296 workers: 463 us with as many units
// as workers, 335 with more); the end of a unit is counted as eight steps.
struct JoinCut {
  int64_t chunk, cuts, units, blocks, workers;
};
inline JoinCut join_cut(int64_t rows, int64_t per, const JoinShape& h, int sms) {
  const int per_block = h.threads ? h.workers() : 1;
  const int64_t groups = rows / per, most = h.most(sms);
  const int64_t at_once = h.tpr ? 32 / h.tpr : 1;
  const int64_t least = (most + groups - 1) / groups, finest = (per + at_once - 1) / at_once;
  JoinCut c{};
  int64_t best = INT64_MAX;
  for (int k = 1; k <= 8; ++k) {
    const int64_t want = std::min(finest, least * k);
    const int64_t steps = (finest + want - 1) / want;  // of a unit
    const int64_t cuts = (finest + steps - 1) / steps, units = groups * cuts;
    const int64_t cost = (units + most - 1) / most * (steps + 8);
    if (cost < best) {
      best = cost;
      c.chunk = steps * at_once;
      c.cuts = cuts;
      c.units = units;
    }
  }
  c.blocks = (std::min<int64_t>(c.units, most) + per_block - 1) / per_block;
  c.workers = c.blocks * per_block;
  return c;
}
inline size_t join_bwd_floats(const JoinCut& c, const JoinShape& h) {
  // dgamma_post, dgamma_pre, and the gate's: a row per unit where a gate row is cut, else one per block of
  // the stream kernel
  return static_cast<size_t>(2 * c.workers + (c.cuts > 1 ? c.units : h.threads ? 0 : c.blocks));
}

template <class T, int V, int TPR, int MODE, int STAGES>
vbt_b200_status go_join_bwd(const JoinBwdParams& p, const JoinShape& h, unsigned grid, cudaStream_t s, int device) {
  static std::atomic<uint64_t> done{0};
  VB_CUDA(allow_shared(residual_norm_bwd_kernel<T, V, TPR, MODE, STAGES>, device, done));
  VB_CUDA(launch_ranks(residual_norm_bwd_kernel<T, V, TPR, MODE, STAGES>, p, grid, h.threads, h.smem, h.ranks, s));
  return VBT_B200_OK;
}

template <class T>
vbt_b200_status launch_join_bwd(JoinBwdParams p, int mode, float* dg1, float* dg2, float* ws, cudaStream_t s, int device) {
  constexpr int VW = 16 / sizeof(T);
  const bool vec = p.cols % VW == 0 && p.dr_stride % VW == 0 && p.dn_stride % VW == 0 && p.y_stride % VW == 0 &&
                   p.r_stride % VW == 0 && p.gate_stride % VW == 0 && a16(p.dr) && a16(p.dn) && a16(p.y) && a16(p.r) &&
                   a16(p.gate) && a16(p.dx) && a16(p.dy) && a16(p.dgate);
  const JoinShape h = join_bwd_shape(p.cols, sizeof(T), mode == GATE_ROW, vec);
  const JoinCut cut = join_cut(p.rows, p.per, h, sm_count(device));
  p.chunk = cut.chunk; p.cuts = cut.cuts; p.units = cut.units; p.ranks = h.ranks;
  const unsigned g = static_cast<unsigned>(cut.blocks * h.ranks);
  float* at = ws;
  if (dg1) { p.ws_g1 = at; at += cut.workers * p.cols; }
  if (dg2) { p.ws_g2 = at; at += cut.workers * p.cols; }
  const bool split_gate = mode == GATE_SHARED && p.dgate != nullptr && cut.cuts > 1;
  // the stream kernel sums a gate row in memory even where it has all its rows
  if (split_gate || (mode == GATE_SHARED && p.dgate != nullptr && h.threads == 0)) p.ws_gate = at;
#define VB_JB(V, MODE)                                                             \
  (h.tpr == 8      ? go_join_bwd<T, V, 8, MODE, 2>(p, h, g, s, device)             \
   : h.tpr == 16   ? go_join_bwd<T, V, 16, MODE, 2>(p, h, g, s, device)            \
   : h.tpr == 32   ? go_join_bwd<T, V, 32, MODE, 2>(p, h, g, s, device)            \
   : h.stages == 2 ? go_join_bwd<T, V, 0, MODE, 2>(p, h, g, s, device)             \
                   : go_join_bwd<T, V, 0, MODE, 1>(p, h, g, s, device))
#define VB_JB_MODE(MODE)                                                           \
  do {                                                                             \
    if (h.threads == 0) residual_norm_bwd_stream_kernel<T, MODE><<<g, 512, 0, s>>>(p); \
    else if (vec) VB_TRY(VB_JB(VW, MODE));                                         \
    else VB_TRY(VB_JB(1, MODE));                                                   \
  } while (0)
  if (mode == GATE_NONE) VB_JB_MODE(GATE_NONE);
  else if (mode == GATE_SHARED) VB_JB_MODE(GATE_SHARED);
  else VB_JB_MODE(GATE_ROW);
#undef VB_JB_MODE
#undef VB_JB
  VB_LAUNCH_CHECK();
  const int threads = h.threads ? h.threads : 512;
  int launches = 1;
  const int64_t gates = p.rows / p.per;
  JoinFoldParams f{};
  f.out[0] = dg1; f.out[1] = dg2; f.ws[0] = p.ws_g1; f.ws[1] = p.ws_g2;
  f.dgate = p.dgate; f.ws_gate = p.ws_gate;
  f.cols = p.cols; f.parts = cut.workers; f.cuts = cut.cuts;
  unsigned sums = 0;
  if (dg1) f.what[sums++] = 0;
  if (dg2) f.what[sums++] = 1;
  if (split_gate && gates == 1) f.what[sums++] = 2;
  if (sums) {
    residual_norm_fold_kernel<T><<<dim3(static_cast<unsigned>((p.cols + 7) / 8), sums), kStripThreads, 0, s>>>(f);
    VB_LAUNCH_CHECK();
    ++launches;
  }
  if (split_gate && gates > 1) {
    const dim3 grid(static_cast<unsigned>((p.cols + 31) / 32), static_cast<unsigned>(std::min<int64_t>(gates, 65535)));
    residual_norm_gate_fold_kernel<T><<<grid, 256, 0, s>>>(static_cast<T*>(p.dgate), p.ws_gate, cut.cuts, p.cols, gates);
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
  const int elt = itemsize(dtype);
  for (int form = 0; form < 4; ++form) {  // whichever the gate given and the pointers' alignment take
    const JoinShape h = join_bwd_shape(cols, elt, form & 1, form & 2);
    const JoinCut c = join_cut(rows, rows_per_gate == 1 ? rows : rows_per_gate, h, sm_count(device));
    *bytes = std::max(*bytes, join_bwd_floats(c, h) * static_cast<size_t>(cols) * 4);
  }
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
  VB_ARG(rows < (int64_t{1} << 31), std::string(name) + ": too many rows");
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

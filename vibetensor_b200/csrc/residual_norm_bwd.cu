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
// rounds nothing: r i = (r 2^k) (i 2^-k).  A factor per value instead, i (r i), took up to 8 % longer.
//
// Bound by memory and, close behind, by instructions: four rows read, two written, 14 fp32 operations
// and six conversions per value.  [32768,4096] bf16 with a gate row per 4096 rows takes, a call by
// itself, 300 us = 5.4 TB/s, 0.82 of the measured copy bandwidth (16 warps per SM at 128 registers, half
// of the issue slots busy).  What it came through: rows in registers 678 us; staged by asynchronous copies
// 370; one base per warp and compile-time offsets instead of an address per access (744 instructions per warp and row
// against 964) 314; runs of neighbouring rows rather than every n-th one 306 (379).  Arithmetic on
// float pairs was slower here (335: moves to pair the registers), and so were one block per SM with
// four rows in flight (759), eight values per thread (424), and one row in flight (333).
// Rows shared by two blocks: [8192,16384] bf16 440 us for a floor of 245, 415 without a gate.  Rows that no
// vector divides: [16384,4095] bf16 253 us for 123, 228 without a gate; their values are single 16-bit loads
// from shared memory and single stores.
#include <algorithm>

#include "row_tile.cuh"

namespace vb {
namespace {

enum { GATE_NONE = 0, GATE_SHARED = 1, GATE_ROW = 2 };

// How the rows (fewer than 2^31) are cut: units of `chunk` rows, `cuts` to a gate row of `per` rows (its last
// one may be shorter), dealt out to the workers in runs of `least` units, one more to each of the first `more`.
struct RowCut {
  uint32_t chunk, cuts, per, units, workers, least, more;

  __host__ __device__ uint32_t first_unit(uint32_t worker) const { return worker * least + min_of(worker, more); }
  __host__ __device__ uint32_t worker_of(uint32_t unit) const {
    const uint32_t head = more * (least + 1);
    return unit < head ? unit / (least + 1) : more + (unit - head) / least;
  }
  __host__ __device__ uint32_t first_row(uint32_t unit) const {
    if (chunk == 1 || cuts == 1) return unit * chunk;
    const uint32_t group = unit / cuts;
    return group * per + (unit - group * cuts) * chunk;
  }
  static __host__ __device__ uint32_t min_of(uint32_t a, uint32_t b) { return a < b ? a : b; }
};

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
  float* ws_gate;    // [workers + gate rows][cols] when gate rows' rows are cut: row worker + gate row is the
                     // worker's part of it; the stream kernel sums whole ones in [gridDim.x][cols]
  int64_t rows, cols;
  int64_t dr_stride, dn_stride, y_stride, r_stride, gate_stride;
  int64_t per;       // rows of one gate row (GATE_SHARED), else all rows
  RowCut cut;
  float a, b, inv_cols;
  int dense;         // the rows of dr, dn, r and y follow one another without gaps
  int post, pre;
  int ranks;         // blocks that share a row
};

// A worker (a warp when TPR lanes of it share a row, else the block) walks one run of neighbouring
// rows, gate row after gate row.  Rows arrive in shared memory by asynchronous
// copies, `stages` rows ahead; a thread reads back only what it copied itself, once for the three
// sums and once for the outputs, so a row needs no barrier but the one of its reduction, and no
// registers between the two passes.  w = b * gate * g1 and g2 lie beside them.
// The sum over a gate row's rows of G * y * i1 gives the gate's gradient (times b * g1) and their part of
// dgamma_post (times b * gate).  A gate row of its own per row (GATE_ROW) is a factor of the sum.
// Values of a row per thread: two sums per column and the gradient at r stay in registers for each.  Single
// values: 16-bit ones fare better with sixteen ([16384,4095] bf16, a gate row per 2048: 251 us, 364 with eight),
// 32-bit ones with eight where blocks are small ([6151,1365], a gate row for all: 69 us, 75 with sixteen; not
// [8192,4095] without a gate, 194 and 179).
constexpr int kVecElts = 16;
template <class T> constexpr int kSingleElts = sizeof(T) == 2 ? 16 : 8;
constexpr int kBwdMaxThreads = 512;   // of a block that shares a row
// Two rows ahead of 32-bit vectors leave shared memory for 352 threads: they may have 184 registers each, and
// spill with 128 ([16384,4096] fp32 304 us, 278 so).
constexpr int bwd_max_threads(int elt, bool vec, int stages) { return elt == 4 && vec && stages == 2 ? 352 : kBwdMaxThreads; }

// A row is far from one if its i is: beyond 2^25 or below 2^-25, and a normal number.  16-bit floats of five
// exponent bits never are.
__device__ __forceinline__ bool beyond(float i) { return (__float_as_uint(i) >> 23) - (127 - 25) > 50u; }
template <class T> __device__ __forceinline__ bool far_row(float i) {
  return !std::is_same_v<T, __half> && beyond(i) && (__float_as_uint(i) >> 23) - 1 < 254u;
}
// its i as a power of two and a number between one and two
__device__ __forceinline__ float power_of_two(float i) { return __uint_as_float(__float_as_uint(i) & 0x7f800000u); }
__device__ __forceinline__ float near_one(float i) { return __uint_as_float((__float_as_uint(i) & 0x007fffffu) | 0x3f800000u); }

template <class T, int V, int TPR, int MODE, int STAGES>
__global__ void __launch_bounds__(TPR ? 256 : bwd_max_threads(sizeof(T), V > 1, STAGES), TPR ? 2 : 1) residual_norm_bwd_kernel(const __grid_constant__ JoinBwdParams p) {
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
  // b g1 of a chunk's columns
  auto factors = [&](int c, float (&v)[C]) {
    const float* g1 = p.post ? p.g1 : nullptr;
#pragma unroll
    for (int e = 0; e < C; ++e) v[e] = p.b;
    if (g1) {
#pragma unroll
      for (int e = 0; e < C; ++e)
        if (A::off(c, e) < left) v[e] *= g1[j0 + A::off(c, e)];
    }
  };
  A::fill_factors(gbuf, left, [&](int o) { return p.pre && p.g2 ? p.g2[j0 + o] : 1.f; });
  if constexpr (MODE != GATE_SHARED) {
#pragma unroll
    for (int c = 0; c < A::N; ++c) {
      float w[C];
      factors(c, w);
      A::write_factors(wbuf, c, w);
    }
  }

  const int worker = TPR ? blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32 : blockIdx.x / ranks;
  // the worker's rows; fewer than 2^31 in all
  const int begin = static_cast<int>(p.cut.first_row(p.cut.first_unit(min(worker, static_cast<int>(p.cut.workers)))));
  const int end = static_cast<int>(p.cut.first_row(p.cut.first_unit(min(worker + 1, static_cast<int>(p.cut.workers)))));
  // Rows are taken RW at a time, up to the end of a gate row where it is shared.  `row` is the first of
  // them, `lane_row` this lane's; a lane whose row lies behind `stop` has none.
  // Rows are addressed from their number: a running pointer per array is 20 registers of the 128.  Dense
  // 16-bit arrays share one offset per row: [32768,4096] without a gate 287 -> 281 us, with a row for all 301
  // -> 291; not with a gate row per row, another array, which spills then (367 -> 386).
  constexpr bool DENSE = sizeof(T) == 2 && MODE != GATE_ROW;
  const int per = static_cast<int>(p.per);
  int group = MODE == GATE_SHARED ? begin / per : 0;
  auto group_end = [&](int g) { return MODE == GATE_SHARED && (g + 1) * int64_t{per} < end ? (g + 1) * per : end; };
  int row = begin, stop = group_end(group);
  int row_ahead = begin, group_ahead = group, stop_ahead = stop;  // RW > 1
  auto next = [&](int& r, int& g, int& st) {
    r += RW;
    if constexpr (MODE == GATE_SHARED) {
      if (r >= st) {
        r = st;
        st = group_end(++g);
      }
    }
  };
  auto at_row = [&](const void* base, int64_t stride, int r) { return static_cast<const T*>(base) + r * stride + seg; };
  auto at = [&](const void* base, int64_t offset) { return static_cast<const T*>(base) + offset; };
  float i1_next[STAGES], i2_next[STAGES];
  auto fetch = [&](int stage, int steps, float& i1, float& i2) {  // `steps` ahead of `row`
    i1 = 1.f;
    i2 = 0.f;
    const int r = RW == 1 ? row + steps : row_ahead + rl;
    if (r < (RW == 1 ? end : stop_ahead)) {
      if (DENSE && p.dense) {
        const int64_t o = r * p.cols + seg;
        if (p.dr) A::copy(buf(stage, 0), at(p.dr, o), seg_left, p.dr);
        if (p.pre) {
          A::copy(buf(stage, 1), at(p.dn, o), seg_left, p.dn);
          A::copy(buf(stage, 2), at(p.r, o), seg_left, p.r);
          i2 = p.inv2[r];
        }
        if (p.y) A::copy(buf(stage, 3), at(p.y, o), seg_left, p.y);
        if (p.post) i1 = p.inv1[r];
      } else {
        if (p.dr) A::copy(buf(stage, 0), at_row(p.dr, p.dr_stride, r), seg_left, p.dr);
        if (p.pre) {
          A::copy(buf(stage, 1), at_row(p.dn, p.dn_stride, r), seg_left, p.dn);
          A::copy(buf(stage, 2), at_row(p.r, p.r_stride, r), seg_left, p.r);
          i2 = p.inv2[r];
        }
        if (p.y) A::copy(buf(stage, 3), at_row(p.y, p.y_stride, r), seg_left, p.y);
        if constexpr (MODE == GATE_ROW) A::copy(buf(stage, 4), at_row(p.gate, p.gate_stride, r), seg_left, p.gate);
        if (p.post) i1 = p.inv1[r];
      }
    }
    if constexpr (RW > 1) next(row_ahead, group_ahead, stop_ahead);
    copy_commit();
  };
#pragma unroll
  for (int q = 0; q < STAGES; ++q) fetch(q, q, i1_next[q], i2_next[q]);

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
  // the gate row, from this thread's first column on
  auto gate_of = [&](int g) { return static_cast<const T*>(p.gate) + g * p.gate_stride + j0; };
  auto fill_gate = [&] {
    const T* gate = gate_of(group);
#pragma unroll
    for (int c = 0; c < A::N; ++c) {
      float w[C], gt[C];
      A::load(gate, c, left, gt);
      factors(c, w);
#pragma unroll
      for (int e = 0; e < C; ++e) w[e] *= gt[e];
      A::write_factors(wbuf, c, w);
    }
  };
  if constexpr (MODE == GATE_SHARED) {
    if (row < end) fill_gate();
  }
  int phase = 0, stage = 0;
  while (row < end) {
    copy_wait<STAGES - 1>();
    A::sync();
    const int lane_row = row + rl;
    const bool live = RW == 1 || lane_row < stop;
    const float i2 = i2_next[0];
    float i1 = i1_next[0], ir = i2;  // of the rows as they lie in shared memory
    const bool far = !std::is_same_v<T, __half> && (beyond(i1) || (p.pre && beyond(i2)));
    if (far) {
      if (far_row<T>(i1)) {
        if (live) A::scale(buf(stage, 3), A::shift(p.y, p.y_stride, lane_row), left, power_of_two(i1));
        i1 = near_one(i1);
      }
      if (far_row<T>(i2)) {
        if (live) A::scale(buf(stage, 2), A::shift(p.r, p.r_stride, lane_row), left, power_of_two(i2));
        ir = near_one(i2);
      }
    }
    float s[3] = {0.f, 0.f, 0.f};
    float up[E];  // dr + i2 dn g2, kept for the second pass
    if (live) {
#pragma unroll
      for (int c = 0; c < A::N; ++c) {
        float dr[C], dn[C], r[C], y[C], w[C], g2[C];
        A::read(buf(stage, 0), A::shift(p.dr, p.dr_stride, lane_row), c, dr);
        A::read(buf(stage, 1), A::shift(p.dn, p.dn_stride, lane_row), c, dn);
        A::read(buf(stage, 2), A::shift(p.r, p.r_stride, lane_row), c, r);
        A::read(buf(stage, 3), A::shift(p.y, p.y_stride, lane_row), c, y);
        A::read_factors(wbuf, c, w);
        A::read_factors(gbuf, c, g2);
        if constexpr (MODE == GATE_ROW) {
          float gt[C];
          A::read(buf(stage, 4), A::shift(p.gate, p.gate_stride, lane_row), c, gt);
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
    // keeps the second reads of the row behind the sums: in front of them they cost registers that spill
    if constexpr (TPR != 0) __syncwarp();
    const float c2 = (i2 * p.inv_cols) * ir * (ir * s[0]);
    const float c1 = p.post ? (i1 * p.inv_cols) * i1 * (i1 * (s[1] - c2 * s[2])) : 0.f;
    if (live) {
      const int64_t o = static_cast<int64_t>(lane_row) * p.cols + j0;
#pragma unroll
      for (int c = 0; c < A::N; ++c) {
        float r[C], y[C], w[C], gt[C], ox[C], oy[C], og[C];
        A::read(buf(stage, 2), A::shift(p.r, p.r_stride, lane_row), c, r);
        A::read(buf(stage, 3), A::shift(p.y, p.y_stride, lane_row), c, y);
        A::read_factors(wbuf, c, w);
        if constexpr (MODE == GATE_ROW) A::read(buf(stage, 4), A::shift(p.gate, p.gate_stride, lane_row), c, gt);
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
          oy[e] = Gi * w[e];
        }
        // without the norm (i1 = 1) dy does not depend on y, not even on a NaN in it
        if (p.post) {
#pragma unroll
          for (int e = 0; e < C; ++e) oy[e] = fmaf(-c1, y[e], oy[e]);
        }
        A::write(static_cast<T*>(p.dx) + o, c, left, ox);
        A::write(static_cast<T*>(p.dy) + o, c, left, oy);
        if constexpr (MODE == GATE_ROW) {
          if (p.dgate) A::write(static_cast<T*>(p.dgate) + o, c, left, og);
        }
      }
      // dy = i (G w - ..) came out with i 2^-k
      if (far && p.post && far_row<T>(p.inv1[lane_row]))
        A::scale_row(static_cast<T*>(p.dy) + o, left, power_of_two(p.inv1[lane_row]));
    }
#pragma unroll
    for (int q = 0; q + 1 < STAGES; ++q) {
      i1_next[q] = i1_next[q + 1];
      i2_next[q] = i2_next[q + 1];
    }
    A::sync();
    fetch(stage, STAGES, i1_next[STAGES - 1], i2_next[STAGES - 1]);
    stage = stage + 1 == STAGES ? 0 : stage + 1;
    const int done = group;
    next(row, group, stop);
    if constexpr (MODE == GATE_SHARED) {
      if (group == done && row < end) continue;
      over_rows(sum1);
      const T* gate = gate_of(done);
      // all of the gate row's rows, or a part for the fold
      const bool whole = p.ws_gate == nullptr || (int64_t{done} * per >= begin && (done + 1) * int64_t{per} <= end);
      const bool first = done == begin / per;
      if (rl == 0) {
#pragma unroll
        for (int c = 0; c < A::N; ++c) {
          float gt[C], og[C];
          A::load(gate, c, left, gt);
          factors(c, og);
          float* sums = p.ws_g1 + int64_t{worker} * p.cols + j0;  // the worker's running part of dgamma_post
          float* part = p.ws_gate + (worker + int64_t{done}) * p.cols + j0;
#pragma unroll
          for (int e = 0; e < C; ++e) {
            og[e] *= sum1[c * C + e];
            gt[e] *= p.b * sum1[c * C + e];
          }
          if (p.ws_g1 && !first) {
#pragma unroll
            for (int e = 0; e < C; ++e)
              if (A::off(c, e) < left) gt[e] += sums[A::off(c, e)];
          }
#pragma unroll
          for (int e = 0; e < C; ++e) {
            if (A::off(c, e) >= left) continue;
            if (p.ws_g1) sums[A::off(c, e)] = gt[e];
            if (!whole) part[A::off(c, e)] = og[e];
          }
          if (p.dgate && whole) A::write(static_cast<T*>(p.dgate) + int64_t{done} * p.cols + j0, c, left, og);
        }
      }
#pragma unroll
      for (int i = 0; i < E; ++i) sum1[i] = 0.f;
      if (row < end) fill_gate();
    }
  }
  copy_wait<0>();
  if (ranks > 1) cluster_sync();  // no block leaves while another may still write to its shared memory
  if constexpr (MODE != GATE_SHARED) over_rows(sum1);
  over_rows(sum2);
  if (rl == 0 && worker < static_cast<int>(p.cut.workers)) {
#pragma unroll
    for (int c = 0; c < A::N; ++c)
#pragma unroll
      for (int e = 0; e < C; ++e) {
        if (A::off(c, e) >= left) continue;
        const int64_t o = int64_t{worker} * p.cols + j0 + A::off(c, e);
        if constexpr (MODE != GATE_SHARED) {
          if (p.ws_g1) p.ws_g1[o] = p.b * sum1[c * C + e];
        }
        if (p.ws_g2) p.ws_g2[o] = sum2[c * C + e];
      }
  }
}

// any length and alignment: a block walks its rows, scalar accesses, each row read twice (again from L2);
// the column sums live in the block's own workspace rows (a column is always the same thread's)
template <class T, int MODE>
__global__ void __launch_bounds__(512) residual_norm_bwd_stream_kernel(const __grid_constant__ JoinBwdParams p) {
  constexpr int THREADS = 512;
  __shared__ float red[2][3][THREADS / 32];
  RowFold<THREADS, 3, THREADS> fold{red};
  const int t = threadIdx.x;
  const float inv_cols = p.inv_cols;
  float* s1 = p.ws_g1 ? p.ws_g1 + static_cast<int64_t>(blockIdx.x) * p.cols : nullptr;
  float* s2 = p.ws_g2 ? p.ws_g2 + static_cast<int64_t>(blockIdx.x) * p.cols : nullptr;
  for (int64_t j = t; j < p.cols; j += THREADS) {
    if (s1) s1[j] = 0.f;
    if (s2) s2[j] = 0.f;
  }
  const int64_t start = p.cut.first_row(p.cut.first_unit(blockIdx.x)), last = p.cut.first_row(p.cut.first_unit(blockIdx.x + 1));
  for (int64_t begin = start, end; begin < last; begin = end) {
    const int64_t group = begin / p.per;
    end = min(last, (group + 1) * p.per);
    float* sg = MODE == GATE_SHARED && p.ws_gate ? p.ws_gate + (p.cut.cuts > 1 ? blockIdx.x + group : blockIdx.x) * p.cols : nullptr;
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
    if (sg && group * p.per >= start && (group + 1) * p.per <= last)
      for (int64_t j = t; j < p.cols; j += THREADS) static_cast<T*>(p.dgate)[group * p.cols + j] = from_f<T>(sg[j]);
  }
}

// Column sums of partial rows in a fixed order.  blockIdx.y says which: dgamma_post and dgamma_pre over the
// workers' rows, the gradient of one gate row that serves all.
struct JoinFoldParams {
  float* out[2];
  const float* ws[2];
  void* dgate;
  const float* ws_gate;
  int64_t cols, parts;
  int what[3];
};
template <class T>
__global__ void __launch_bounds__(kStripThreads) residual_norm_fold_kernel(const __grid_constant__ JoinFoldParams p) {
  __shared__ float sm[kStripThreads / 32][8];
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 8 + threadIdx.x;
  const int what = p.what[blockIdx.y];
  const float s = strip_sum(what < 2 ? p.ws[what] : p.ws_gate, p.parts, p.cols, sm);
  if (threadIdx.x < 8 && c < p.cols) {
    if (what < 2) p.out[what][c] = s;
    else static_cast<T*>(p.dgate)[c] = from_f<T>(s);
  }
}
// Several gate rows, workers' parts of the ones that are cut: WARPS warps take 32 columns of one.  There are as
// many to look at as gate rows, or as workers that may begin in the middle of one if these are fewer.
// Eight warps where the gate rows are few and their parts many, else one (8 gate rows of 4096 rows: 305 us with
// eight, 316 with one; 1024 of 32 rows: 409 and 335).
template <class T, int WARPS>
__global__ void __launch_bounds__(256) residual_norm_gate_fold_kernel(T* dgate, const float* ws,
                                                                      const __grid_constant__ RowCut cut, int64_t cols) {
  __shared__ float sm[8][32];
  constexpr int AT_ONCE = 8 / WARPS;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  const uint32_t gates = cut.units / cut.cuts, n = RowCut::min_of(gates, cut.workers);
  for (uint32_t i = blockIdx.y * AT_ONCE + w / WARPS; i < n; i += gridDim.y * AT_ONCE) {
    const uint32_t g = gates <= cut.workers ? i : cut.first_unit(i) / cut.cuts;
    const uint32_t w0 = cut.worker_of(g * cut.cuts), parts = cut.worker_of(g * cut.cuts + cut.cuts - 1) - w0 + 1;
    // written by the one worker that has it; or for the next worker to look at, who begins in it second
    if (parts == 1 || (gates > cut.workers && w0 + 1 != i)) continue;
    const float* src = ws + static_cast<int64_t>(w0 + g) * cols + c;
    float acc = 0.f;
    if (c < cols) {
      for (uint32_t r = w % WARPS; r < parts; r += 8 * WARPS) {
        float v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = r + WARPS * q < parts ? __ldcg(src + static_cast<int64_t>(r + WARPS * q) * cols) : 0.f;
#pragma unroll
        for (int q = 0; q < 8; ++q) acc += v[q];
      }
    }
    if constexpr (WARPS > 1) {
      sm[w][lane] = acc;
      __syncthreads();
      if (w == 0) {
        acc = 0.f;
#pragma unroll
        for (int k = 0; k < WARPS; ++k) acc += sm[k][lane];
      }
      __syncthreads();
    }
    if (w % WARPS == 0 && c < cols) dgate[static_cast<int64_t>(g) * cols + c] = from_f<T>(acc);
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
    // Few blocks of many threads: of [8192,16384] bf16, two per row against four with 256 threads each, 427
    // us and 486 without a gate, 468 and 519 with a row per 1024; fp32 [4096,16384] 316 and 431.
    if (h.threads > kBwdMaxThreads) continue;
    // two rows ahead where they fit; the warp forms are built for that alone
    h.stages = 2;
    if (!h.tpr && smem(2) > kSmemPerBlock) h.stages = 1;
    h.smem = smem(h.stages);
    if (h.smem > kSmemPerBlock || h.threads > bwd_max_threads(elt, vec, h.stages)) continue;
    // registers allow 512 threads per SM (128 each)
    h.per_sm = std::max(1, std::min(512 / h.threads, kSmemPerSm / (h.smem + 1024)));
    return h;
  }
  return JoinShape{0, 0, 0, 0, 4, 1};
}
// How the rows are cut: into units of as many rows as a worker takes at once, dealt out evenly in runs to the
// workers that fit the card, which sum a gate row's part each; or into whole gate rows where that is
// cheaper.  Units of more rows, each with a sum of its own, took [8192,16384] bf16 with a gate row per 1024
// rows 592 us against 464, [16384,8192] with one per 2048 437 against 350.
inline RowCut join_cut(int64_t rows, int64_t per, const JoinShape& h, int sms) {
  const int64_t groups = rows / per, most = h.most(sms);
  const int64_t at_once = h.tpr ? 32 / h.tpr : 1;
  const int64_t steps = (per + at_once - 1) / at_once;  // of a gate row
  // in steps; the end of a gate row's run counts as eight, the fold of parts as one
  const int64_t whole = (groups + most - 1) / most * (steps + 8);
  const int64_t share = (groups * steps + most - 1) / most, even = share + 8 * (share / steps + 1) + 1;
  const bool cut = steps > 1 && whole > even;
  RowCut c{};
  c.chunk = static_cast<uint32_t>(cut ? at_once : per);
  c.cuts = static_cast<uint32_t>(cut ? steps : 1);
  c.per = static_cast<uint32_t>(per);
  c.units = static_cast<uint32_t>(groups * c.cuts);
  c.workers = static_cast<uint32_t>(std::min<int64_t>(c.units, most));
  c.least = c.units / c.workers;
  c.more = c.units % c.workers;
  return c;
}
inline size_t join_bwd_rows(const RowCut& c, const JoinShape& h) {
  // dgamma_post, dgamma_pre, and the gate's: a row per worker and gate row where these are cut, else one per
  // block of the stream kernel
  return size_t{2} * c.workers + (c.cuts > 1 ? size_t{c.workers} + c.units / c.cuts : h.threads ? 0 : c.workers);
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
  const RowCut cut = join_cut(p.rows, p.per, h, sm_count(device));
  const int per_block = h.threads ? h.workers() : 1;
  p.cut = cut;
  p.dense = (!p.dr || p.dr_stride == p.cols) && (!p.dn || p.dn_stride == p.cols) && (!p.r || p.r_stride == p.cols) &&
            (!p.y || p.y_stride == p.cols);
  p.ranks = h.ranks; p.inv_cols = 1.f / static_cast<float>(p.cols);
  const unsigned g = (cut.workers + per_block - 1) / per_block * h.ranks;
  float* at = ws;
  if (dg1) { p.ws_g1 = at; at += int64_t{cut.workers} * p.cols; }
  if (dg2) { p.ws_g2 = at; at += int64_t{cut.workers} * p.cols; }
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
  f.cols = p.cols; f.parts = cut.workers;
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
    const int64_t n = std::min<int64_t>(gates, cut.workers), at_once = n <= 64 ? 1 : 8;
    const dim3 grid(static_cast<unsigned>((p.cols + 31) / 32), static_cast<unsigned>((n + at_once - 1) / at_once));
    auto fold = n <= 64 ? residual_norm_gate_fold_kernel<T, 8> : residual_norm_gate_fold_kernel<T, 1>;
    fold<<<grid, 256, 0, s>>>(static_cast<T*>(p.dgate), p.ws_gate, cut, p.cols);
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
  VB_ARG(rows < (int64_t{1} << 31), std::string(name) + ": too many rows");
  VB_ARG(is_float_dtype(dtype), std::string(name) + ": expected a floating dtype");
  VB_ARG(rows == 0 || (rows_per_gate > 0 && rows % rows_per_gate == 0),
         std::string(name) + ": rows_per_gate does not divide rows");
  *bytes = 0;
  if (rows == 0) return VBT_B200_OK;
  // a gate row of its own per row is no sum over rows: the rows are cut as if one gate row served all
  const int elt = itemsize(dtype);
  for (int form = 0; form < 4; ++form) {  // whichever the gate given and the pointers' alignment take
    const JoinShape h = join_bwd_shape(cols, elt, form & 1, form & 2);
    const RowCut c = join_cut(rows, rows_per_gate == 1 ? rows : rows_per_gate, h, sm_count(device));
    *bytes = std::max(*bytes, join_bwd_rows(c, h) * static_cast<size_t>(cols) * 4);
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

// The join of a transformer branch with the residual stream between two RMS norms (sm_100a).
//
//   v = y * i1 * g1,  i1 = rsqrt(mean(y^2) + eps)          (the norm behind the branch; v = y without)
//   r = a * x + b * gate * v
//   n = r * i2 * g2,  i2 = rsqrt(mean(r^2) + eps)          (the norm in front of the next block)
//
// The two sums stay apart: sum(r^2) expanded in x and v would save a reduction and cancel where the
// branch nearly undoes the stream.
//
// Bound by memory: two rows read, two written.  [32768,4096] bf16 with a gate row per 4096 rows takes, a
// call by itself, 178 us = 6.0 TB/s, 0.92 of the measured copy bandwidth; rows in registers, read when they are
// needed, took 254 us (93 registers, two blocks per SM, nothing in flight during the reductions).
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
  int64_t chunk;                            // rows of a worker
  int ranks;                                // blocks that share a row
  float a, b, eps;
  int post, pre;
};

__device__ __forceinline__ int64_t gate_row(const JoinParams& p, int64_t row) {
  return row / p.per;
}

constexpr int kFwdElts = 16;         // values of a row per thread
constexpr int kFwdMaxThreads = 1024;  // of a block that shares a row

// A worker (a warp when TPR lanes of it share a row, else the block) walks neighbouring rows.  x, y
// (and a gate row per row) arrive in shared memory by asynchronous copies; a thread reads back only
// what it copied itself, so a row needs no barrier but those of its two reductions, and the next
// row's copies start as soon as r stands in registers.  w = b * g1 (times a shared gate row) and g2 lie
// beside them.  One row per block in flight and four blocks per SM; two rows and three blocks (what
// shared memory holds) ran [32768,4096] bf16 in 198 us against 178, three rows and two blocks in 184.
template <class T, int V, int TPR, bool GATE_ROW>
__global__ void __launch_bounds__(TPR ? 256 : kFwdMaxThreads, TPR ? 4 : 1) residual_norm_kernel(const __grid_constant__ JoinParams p) {
  using A = RowChunks<T, V, TPR, kFwdElts>;
  constexpr int C = A::C, E = kFwdElts;
  constexpr int RW = TPR ? 32 / TPR : 1;
  constexpr int ARRAYS = GATE_ROW ? 3 : 2;
  extern __shared__ __align__(16) unsigned char smem[];
  const int ranks = TPR ? 1 : p.ranks;
  const int warp0 = ranks > 1 ? cluster_rank() * static_cast<int>(blockDim.x >> 5) : 0;
  if (ranks > 1) cluster_sync();  // the other blocks' shared memory is there
  const int rl = TPR ? static_cast<int>(threadIdx.x & 31) / A::STEP : 0;
  const int j0 = A::base(warp0), left = static_cast<int>(p.cols) - j0;
  const float inv_cols = 1.f / static_cast<float>(p.cols);
  unsigned char* wbuf = smem + static_cast<size_t>(threadIdx.x >> 5) * (2 * A::WARP_FACTORS + ARRAYS * A::WARP_ARRAY);
  float4* red = reinterpret_cast<float4*>(smem + static_cast<size_t>(blockDim.x >> 5) * (2 * A::WARP_FACTORS + ARRAYS * A::WARP_ARRAY));
  unsigned char* gbuf = wbuf + A::WARP_FACTORS;
  unsigned char* ring = gbuf + A::WARP_FACTORS;
  auto buf = [&](int array) { return ring + array * A::WARP_ARRAY; };
#pragma unroll
  for (int a = 0; a < ARRAYS; ++a) A::zero_rest(buf(a), true, left);
  A::sync();
  const int seg = A::segment(warp0), seg_left = static_cast<int>(p.cols) - seg;
  const float* g1 = p.post && p.g1 ? p.g1 + j0 : nullptr;
  const float* g2 = p.pre && p.g2 ? p.g2 + j0 : nullptr;

  const int64_t worker = TPR ? static_cast<int64_t>(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32 : blockIdx.x / ranks;
  const int64_t begin = min(worker * p.chunk, p.rows);
  const int todo = static_cast<int>(min(p.chunk, p.rows - begin));
  const T* x_at = static_cast<const T*>(p.x) + (begin + rl) * p.x_stride + seg;
  const T* y_at = static_cast<const T*>(p.y) + (begin + rl) * p.y_stride + seg;
  const T* gate_at = static_cast<const T*>(p.gate) + (begin + rl) * p.gate_stride + seg;  // GATE_ROW
  int ahead = rl;
  auto fetch = [&] {
    if (ahead < todo) {
      A::copy(buf(0), y_at, seg_left, p.y);
      A::copy(buf(1), x_at, seg_left, p.x);
      if constexpr (GATE_ROW) A::copy(buf(2), gate_at, seg_left, p.gate);
    }
    x_at += RW * p.x_stride;
    y_at += RW * p.y_stride;
    if constexpr (GATE_ROW) gate_at += RW * p.gate_stride;
    ahead += RW;
    copy_commit();
  };
  fetch();
  A::fill_factors(gbuf, left, [&](int o) { return g2 ? g2[o] : 1.f; });
  if (GATE_ROW || p.gate == nullptr) A::fill_factors(wbuf, left, [&](int o) { return p.b * (g1 ? g1[o] : 1.f); });

  T* r_out = static_cast<T*>(p.r) + (begin + rl) * p.cols + j0;
  T* n_out = static_cast<T*>(p.n) + (begin + rl) * p.cols + j0;
  int64_t group = -1, group_end = -1;  // the shared gate row that w holds, first row behind its rows
  int phase = 0;
  for (int r0 = 0; r0 < todo; r0 += RW) {
    const bool live = RW == 1 || r0 + rl < todo;
    const int64_t row = begin + r0 + rl;
    if (!GATE_ROW && p.gate != nullptr && live && row >= group_end) {
      group = row / p.per;
      group_end = (group + 1) * p.per;
      const T* gate = static_cast<const T*>(p.gate) + group * p.gate_stride + j0;
      A::fill_factors(wbuf, left, [&](int o) { return p.b * (g1 ? g1[o] : 1.f) * to_f(gate[o]); });
    }
    copy_wait<0>();
    A::sync();
    float s[1] = {0.f};
    float i1 = 1.f, i2 = 0.f;
    if (p.post) {
      if (live) {
#pragma unroll
        for (int c = 0; c < A::N; ++c) {
          if (!A::reaches(c, seg_left)) break;
          float y[C];
          A::read(buf(0), A::shift(p.y, p.y_stride, row), c, y);
#pragma unroll
          for (int e = 0; e < C; ++e) s[0] = fmaf(y[e], y[e], s[0]);
        }
      }
      sum_row<TPR, 1>(s, red, phase, p.ranks);
      i1 = rsqrtf(s[0] * inv_cols + p.eps);
    }
    float r[E];
    if constexpr (V == 1)
#pragma unroll
      for (int i = 0; i < E; ++i) r[i] = 0.f;
    s[0] = 0.f;
    if (live) {
#pragma unroll
      for (int c = 0; c < A::N; ++c) {
        if (!A::reaches(c, seg_left)) break;
        float x[C], y[C], w[C];
        A::read(buf(0), A::shift(p.y, p.y_stride, row), c, y);
        A::read(buf(1), A::shift(p.x, p.x_stride, row), c, x);
        A::read_factors(wbuf, c, w);
        if constexpr (GATE_ROW) {
          float gt[C];
          A::read(buf(2), A::shift(p.gate, p.gate_stride, row), c, gt);
#pragma unroll
          for (int e = 0; e < C; ++e) w[e] *= gt[e];
        }
#pragma unroll
        for (int e = 0; e < C; ++e) {
          const int i = c * C + e;
          r[i] = fmaf(w[e] * i1, y[e], p.a * x[e]);
          s[0] = fmaf(r[i], r[i], s[0]);
        }
      }
    }
    A::sync();
    fetch();
    if (live) {
#pragma unroll
      for (int c = 0; c < A::N && A::reaches(c, seg_left); ++c) A::write(r_out, c, left, *reinterpret_cast<const float(*)[C]>(&r[c * C]));
    }
    if (p.pre) {
      sum_row<TPR, 1>(s, red, phase, p.ranks);
      i2 = rsqrtf(s[0] * inv_cols + p.eps);
      if (live) {
#pragma unroll
        for (int c = 0; c < A::N; ++c) {
          if (!A::reaches(c, seg_left)) break;
          float g[C];
          A::read_factors(gbuf, c, g);
#pragma unroll
          for (int e = 0; e < C; ++e) g[e] *= r[c * C + e] * i2;
          A::write(n_out, c, left, g);
        }
      }
    }
    r_out += RW * p.cols;
    n_out += RW * p.cols;
    if (live && j0 == 0) {
      if (p.post && p.inv1) p.inv1[row] = i1;
      if (p.pre && p.inv2) p.inv2[row] = i2;
    }
  }
  copy_wait<0>();
  if (ranks > 1) cluster_sync();  // no block leaves while another may still write to its shared memory
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

// shared memory per thread: two factors, x, y and a gate row
constexpr int join_bytes(bool gate_row, int elt, bool vec, int tpr) {
  return kFwdElts * 8 + (gate_row ? 3 : 2) * row_bytes_per_thread(kFwdElts, elt, vec, tpr);
}

template <class T, int V, int TPR, bool GATE_ROW>
vbt_b200_status go_join(JoinParams& p, int threads, int sms, unsigned& grid, cudaStream_t s, int device) {
  static std::atomic<uint64_t> done{0};
  VB_CUDA(allow_shared(residual_norm_kernel<T, V, TPR, GATE_ROW>, device, done));
  const int smem = threads * join_bytes(GATE_ROW, sizeof(T), V > 1, TPR) + (TPR ? 0 : sum_bytes(p.ranks));
  const int per_sm = std::max(1, std::min(1024 / threads, kSmemPerSm / (smem + 1024)));
  const int workers = TPR ? threads / 32 : 1;
  // as many workers as fit the card at once, each with a run of rows
  const int64_t most = p.ranks > 1 ? clusters_at_once(sms, p.ranks) : int64_t{sms} * per_sm * workers;
  p.chunk = (p.rows + most - 1) / most;
  const int64_t used = (p.rows + p.chunk - 1) / p.chunk;
  grid = static_cast<unsigned>((used + workers - 1) / workers * p.ranks);
  VB_CUDA(launch_ranks(residual_norm_kernel<T, V, TPR, GATE_ROW>, p, grid, threads, smem, p.ranks, s));
  return VBT_B200_OK;
}

template <class T>
vbt_b200_status launch_join(JoinParams p, cudaStream_t s, int device) {
  constexpr int VW = 16 / sizeof(T);
  const int sms = sm_count(device);
  const bool vec = p.cols % VW == 0 && p.x_stride % VW == 0 && p.y_stride % VW == 0 && p.gate_stride % VW == 0 &&
                   a16(p.x) && a16(p.y) && a16(p.gate) && a16(p.r) && a16(p.n);
  const bool gate_row = p.gate != nullptr && p.per == 1 && p.rows > 1;
  const int64_t lanes = (p.cols + kFwdElts - 1) / kFwdElts;
  const int tpr = lanes <= 8 ? 8 : lanes <= 16 ? 16 : lanes <= 32 ? 32 : 0;
  int threads = 0;
  for (p.ranks = 1; p.ranks <= kMaxRanks; p.ranks *= 2) {
    const int64_t part = (lanes + p.ranks - 1) / p.ranks;
    const int64_t n = tpr ? 256 : (part + 31) / 32 * 32;
    if (n <= (p.ranks > 1 ? 512 : kFwdMaxThreads) && n * join_bytes(gate_row, sizeof(T), vec, tpr) + sum_bytes(p.ranks) <= kSmemPerBlock) {
      threads = static_cast<int>(n);
      break;
    }
  }
  unsigned g = 0;
  if (threads == 0) {
    threads = 512;
    g = static_cast<unsigned>(std::min<int64_t>(p.rows, int64_t{sms} * 4));
    residual_norm_stream_kernel<T><<<g, threads, 0, s>>>(p);
  } else {
#define VB_JOIN(V, GR)                                                           \
  (tpr == 8    ? go_join<T, V, 8, GR>(p, threads, sms, g, s, device)             \
   : tpr == 16 ? go_join<T, V, 16, GR>(p, threads, sms, g, s, device)            \
   : tpr == 32 ? go_join<T, V, 32, GR>(p, threads, sms, g, s, device)            \
               : go_join<T, V, 0, GR>(p, threads, sms, g, s, device))
    if (vec) VB_TRY(gate_row ? VB_JOIN(VW, true) : VB_JOIN(VW, false));
    else VB_TRY(gate_row ? VB_JOIN(1, true) : VB_JOIN(1, false));
#undef VB_JOIN
  }
  VB_LAUNCH_CHECK();
  note_launch(VBT_B200_FAMILY_ROWOP, VBT_B200_WK_RESIDUAL_NORM, dim3(g), dim3(threads), vec ? VW : 1, 1, 0, 1,
              p.rows * p.cols, p.cols, 0, s);
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
  VB_ARG(rows < (int64_t{1} << 36), std::string(name) + ": too many rows");
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
  p.a = residual_scale; p.b = branch_scale; p.eps = eps; p.post = post; p.pre = pre;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case VBT_B200_F32: return launch_join<float>(p, s, scope.device());
    case VBT_B200_F16: return launch_join<__half>(p, s, scope.device());
    default: return launch_join<__nv_bfloat16>(p, s, scope.device());
  }
}

}  // extern "C"

// The join of a transformer branch with the residual stream between two RMS norms (sm_100a).
//
//   v = y * i1 * g1,  i1 = rsqrt(mean(y^2) + eps)          (the norm behind the branch; v = y without)
//   r = a * x + b * gate * v
//   n = r * i2 * g2,  i2 = rsqrt(mean(r^2) + eps)          (the norm in front of the next block)
//
// The two sums stay apart: sum(r^2) expanded in x and v would save a reduction and cancel where the
// branch nearly undoes the stream.
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

}  // extern "C"

// Pieces shared by the row kernels whose rows live in registers: TPR neighbouring threads own a
// row, thread t holds the V-element vectors t, t + TPR, t + 2 TPR, ...
#pragma once

#include "common.cuh"

namespace vb {

// folds N sums over the TPR neighbouring threads that share a row; `red` holds two phases so that
// one barrier per fold is enough
template <int TPR, int N, int THREADS>
struct RowFold {
  float (*red)[N][THREADS / 32];
  int phase = 0;
  __device__ __forceinline__ void operator()(float (&s)[N]) {
    constexpr int G = TPR < 32 ? TPR : 32;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int d = G / 2; d > 0; d >>= 1) s[i] += __shfl_xor_sync(0xffffffffu, s[i], d);
    if constexpr (TPR > 32) {
      constexpr int W = TPR / 32;
      const int w = threadIdx.x >> 5;
      if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) red[phase][i][w] = s[i];
      __syncthreads();
      const int first = w / W * W;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float t = red[phase][i][first];
#pragma unroll
        for (int k = 1; k < W; ++k) t += red[phase][i][first + k];
        s[i] = t;
      }
      phase ^= 1;
    }
  }
};

template <class T, int V, int VPL>
__device__ __forceinline__ void load_vecs(const T* row, int first, int step, int nvec, Vec<T, V> (&v)[VPL]) {
#pragma unroll
  for (int k = 0; k < VPL; ++k) {
    const int j = first + k * step;
    if (j < nvec) {
      v[k] = *reinterpret_cast<const Vec<T, V>*>(row + static_cast<int64_t>(j) * V);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) v[k].v[e] = from_f<T>(0.f);
    }
  }
}
template <int V>
__device__ __forceinline__ void load_floats(const float* src, int j, int nvec, float (&v)[V], float other) {
  if (src == nullptr || j >= nvec) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = other;
  } else if constexpr (V % 4 == 0) {
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(src + static_cast<int64_t>(j) * V) + q);
      v[4 * q] = f.x; v[4 * q + 1] = f.y; v[4 * q + 2] = f.z; v[4 * q + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = __ldg(src + static_cast<int64_t>(j) * V + e);
  }
}
inline bool a16(const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; }

// Sums the n rows of src[n][cols] for the 8 columns of a strip (one
// 32-byte sector per row) with 256 threads, in a fixed order; the sum of column `lane` is returned
// to the first 8 lanes of warp 0.  `sm` is free again at the next barrier behind the call.
__device__ __forceinline__ float strip_sum(const float* src, int64_t n, int64_t cols, float (*sm)[8]) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 8 + (lane & 7);
  float acc = 0.f;
  if (c < cols) {
    for (int64_t r = w * 4 + (lane >> 3); r < n; r += 8 * 32) {
      float v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = r + 32 * q < n ? __ldcg(src + (r + 32 * q) * cols + c) : 0.f;
#pragma unroll
      for (int q = 0; q < 8; ++q) acc += v[q];
    }
  }
  acc += __shfl_xor_sync(0xffffffffu, acc, 8);
  acc += __shfl_xor_sync(0xffffffffu, acc, 16);
  if (lane < 8) sm[w][lane] = acc;
  __syncthreads();
  float s = 0.f;
  if (w == 0 && lane < 8)
#pragma unroll
    for (int k = 0; k < 8; ++k) s += sm[k][lane];
  return s;
}

}  // namespace vb

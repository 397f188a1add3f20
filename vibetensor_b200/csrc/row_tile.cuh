// Pieces shared by the row kernels whose rows live in registers: TPR neighbouring threads own a
// row, thread t holds the V-element vectors t, t + TPR, t + 2 TPR, ...
#pragma once

#include <atomic>

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

// ---------------------------------------------------------------------------------------
// rows in shared memory: a thread copies the values it will itself read
// ---------------------------------------------------------------------------------------
// Asynchronous copy of 16, 8 or 4 bytes into shared memory.
template <int BYTES> __device__ __forceinline__ void copy_async(void* dst, const void* src) {
  const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(d), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void narrow2(float* p, float2 v) { p[0] = v.x; p[1] = v.y; }
__device__ __forceinline__ void narrow2(__nv_bfloat16* p, float2 v) {
  *reinterpret_cast<__nv_bfloat162*>(p) = __float22bfloat162_rn(v);
}
__device__ __forceinline__ void narrow2(__half* p, float2 v) { *reinterpret_cast<__half2*>(p) = __float22half2_rn(v); }

// A thread's E values of a row, worked on in chunks of C: V neighbours for V-value vectors, two
// single values for V = 1.  TPR lanes of a warp share a row, or (TPR = 0) every warp of the block owns
// 32 E neighbouring values of it; either way the columns of a thread's chunks and their places in
// shared memory are compile-time offsets from one base.  A thread has slots of its own in every
// buffer: what it copied it may read after its own wait, without a barrier.
template <class T, int V, int TPR, int E> struct RowChunks {
  static constexpr int C = V > 1 ? V : 2;
  static constexpr int N = E / C;
  static constexpr int STEP = TPR ? TPR : 32;
  static constexpr int WARP_ARRAY = 32 * E * static_cast<int>(sizeof(T));  // bytes of one array in a warp's part
  static constexpr int WARP_FACTORS = 32 * E * 4;
  static constexpr int FW = C >= 4 ? 4 : 2;  // fp32 factors per access
  // first column of this thread
  static __device__ __forceinline__ int base() {
    return TPR ? static_cast<int>(threadIdx.x % STEP) * V : static_cast<int>(threadIdx.x >> 5) * (32 * E) + static_cast<int>(threadIdx.x & 31) * V;
  }
  // offset of element e of chunk c from it
  static __device__ __forceinline__ constexpr int off(int c, int e) { return V > 1 ? c * STEP * V + e : (2 * c + e) * STEP; }
  // a warp's array in shared memory -> the thread's slot for chunk c (element e for V = 1)
  static __device__ __forceinline__ T* slot(unsigned char* array, int c, int e) {
    return reinterpret_cast<T*>(array) + (V > 1 ? c : 2 * c + e) * (32 * V) + static_cast<int>(threadIdx.x & 31) * V;
  }
  // starts the copies of the thread's part of a row; `row` points at the thread's first column, `left`
  // values of the row lie from there on (single values of less than four bytes are copied at once: they
  // are smaller than the smallest asynchronous copy)
  static __device__ __forceinline__ void copy(unsigned char* array, const T* row, int left) {
#pragma unroll
    for (int c = 0; c < N; ++c) {
      if constexpr (V > 1) {
        if (off(c, 0) < left) copy_async<V * static_cast<int>(sizeof(T))>(slot(array, c, 0), row + off(c, 0));
      } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (off(c, e) < left) copy_async<4>(slot(array, c, e), row + off(c, e));
      }
    }
    if constexpr (V == 1 && sizeof(T) < 4) {
      T v[E];
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (i * STEP < left) v[i] = row[i * STEP];
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (i * STEP < left) *slot(array, i / 2, i & 1) = v[i];
    }
  }
  // zeros where no copy ever lands: behind the row's end, or everywhere if the array is absent
  static __device__ __forceinline__ void zero_rest(unsigned char* array, bool present, int left) {
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
      for (int e = 0; e < C; ++e)
        if (!present || off(c, e) >= left) (V > 1 ? slot(array, c, 0)[e] : *slot(array, c, e)) = T{};
  }
  static __device__ __forceinline__ void read(unsigned char* array, int c, float (&v)[C]) {
    if constexpr (V > 1) {
      const Vec<T, V> raw = *reinterpret_cast<const Vec<T, V>*>(slot(array, c, 0));
#pragma unroll
      for (int e = 0; e < C; ++e) v[e] = to_f(raw.v[e]);
    } else {
      v[0] = to_f(*slot(array, c, 0));
      v[1] = to_f(*slot(array, c, 1));
    }
  }
  // the same without the conversion
  static __device__ __forceinline__ void read_raw(unsigned char* array, int c, Vec<T, C>& v) {
    if constexpr (V > 1) {
      v = *reinterpret_cast<const Vec<T, V>*>(slot(array, c, 0));
    } else {
      v.v[0] = *slot(array, c, 0);
      v.v[1] = *slot(array, c, 1);
    }
  }
  static __device__ __forceinline__ void write(T* row, int c, int left, const float (&v)[C]) {
    if constexpr (V > 1) {
      if (off(c, 0) >= left) return;
      Vec<T, V> raw;
#pragma unroll
      for (int e = 0; e < C; e += 2) narrow2(&raw.v[e], make_float2(v[e], v[e + 1]));
      *reinterpret_cast<Vec<T, V>*>(row + off(c, 0)) = raw;
    } else {
      if (off(c, 0) < left) row[off(c, 0)] = from_f<T>(v[0]);
      if (off(c, 1) < left) row[off(c, 1)] = from_f<T>(v[1]);
    }
  }
  // per-column fp32 factors in the thread's own slots
  static __device__ __forceinline__ float* fslot(unsigned char* array, int c, int e) {
    return reinterpret_cast<float*>(array) + ((c * (C / FW) + e / FW) * 32 + static_cast<int>(threadIdx.x & 31)) * FW;
  }
  static __device__ __forceinline__ void read_factors(unsigned char* array, int c, float (&v)[C]) {
#pragma unroll
    for (int e = 0; e < C; e += FW) {
      const Vec<float, FW> f = *reinterpret_cast<const Vec<float, FW>*>(fslot(array, c, e));
#pragma unroll
      for (int i = 0; i < FW; ++i) v[e + i] = f.v[i];
    }
  }
  // fills them: value(offset from the thread's first column), 0 behind the row's end
  template <class Fn> static __device__ __forceinline__ void fill_factors(unsigned char* array, int left, Fn value) {
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
      for (int e = 0; e < C; e += FW) {
        Vec<float, FW> f;
#pragma unroll
        for (int i = 0; i < FW; ++i) f.v[i] = off(c, e + i) < left ? value(off(c, e + i)) : 0.f;
        *reinterpret_cast<Vec<float, FW>*>(fslot(array, c, e)) = f;
      }
  }
};

// Sums over the threads that share a row: TPR lanes of a warp, or the whole block (TPR = 0; `red`
// holds two phases, so one barrier per call is enough).  N <= 4.
template <int TPR, int N>
__device__ __forceinline__ void sum_row(float (&s)[N], float4 (*red)[32], int& phase) {
  constexpr int G = TPR ? TPR : 32;
#pragma unroll
  for (int d = G / 2; d > 0; d >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] += __shfl_xor_sync(0xffffffffu, s[i], d);
  if constexpr (TPR == 0) {
    const int w = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0)
      red[phase][w] = make_float4(s[0], N > 1 ? s[N > 1 ? 1 : 0] : 0.f, N > 2 ? s[N > 2 ? 2 : 0] : 0.f, N > 3 ? s[N > 3 ? 3 : 0] : 0.f);
    __syncthreads();
    float4 t = red[phase][0];
    for (int k = 1; k < warps; ++k) {
      const float4 f = red[phase][k];
      t.x += f.x; t.y += f.y; t.z += f.z; t.w += f.w;
    }
    s[0] = t.x;
    if constexpr (N > 1) s[1] = t.y;
    if constexpr (N > 2) s[2] = t.z;
    if constexpr (N > 3) s[3] = t.w;
    phase ^= 1;
  }
}

constexpr int kSmemPerSm = 228 * 1024;     // of which every block takes 1 KB for the system
constexpr int kSmemPerBlock = 226 * 1024;  // beside sum_row's 1 KB

// Shared memory beyond the default limit has to be asked for once per kernel and device.
template <class Kernel> inline cudaError_t allow_shared(Kernel kernel, int device, std::atomic<uint64_t>& done) {
  const uint64_t bit = 1ull << (device & 63);
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemPerBlock);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

}  // namespace vb

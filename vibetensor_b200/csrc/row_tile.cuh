// Pieces shared by the row kernels whose rows live in registers: TPR neighbouring threads own a
// row, thread t holds the V-element vectors t, t + TPR, t + 2 TPR, ...
#pragma once

#include <algorithm>
#include <atomic>
#include <type_traits>

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
inline bool a16(const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; }

// Sums the n rows of src[n][cols] for the 8 columns of a strip (one 32-byte sector per row) with
// kStripThreads threads, in a fixed order; the sum of column `lane` is returned to the first 8 lanes of
// warp 0.  `sm` is free again at the next barrier behind the call.  128 rows per step keep the ~600
// partial rows of a launch to one step: with 256 threads the fold of [586,4096] took 10 us.
constexpr int kStripThreads = 1024;
__device__ __forceinline__ float strip_sum(const float* src, int64_t n, int64_t cols, float (*sm)[8]) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 8 + (lane & 7);
  float acc = 0.f;
  if (c < cols) {
    for (int64_t r = w * 4 + (lane >> 3); r < n; r += 8 * 128) {
      float v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = r + 128 * q < n ? __ldcg(src + (r + 128 * q) * cols + c) : 0.f;
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
    for (int k = 0; k < kStripThreads / 32; ++k) s += sm[k][lane];
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
// single values for V = 1.  TPR lanes of a warp share a row, or (TPR = 0) every warp of the block (of
// the cluster, counted from `warp0`) owns a segment of 32 E neighbouring values of it; either way the columns of a thread's chunks and their
// places in shared memory are compile-time offsets from one base.
//
// V > 1 (16-byte aligned rows): a thread has slots of its own in every buffer; what it copied it may
// read after its own wait, without a barrier.
// V = 1 (any alignment): the lanes of a segment copy the 16-byte granules that cover it, whole, and
// read single values behind the segment's shift against a 16-byte boundary; sync() stands between the
// wait and the reads, and between the reads and the next copy.  Nothing in front of the tensor's
// first value or behind the row's last is read; every copy writes zeros behind its row up to where another
// shift's may end, so that reads need no bounds.  (Copies of single 4-byte values ran [6151,1365] fp32 at half the rate, and
// 2-byte ones cannot be asynchronous.)
template <class T, int V, int TPR, int E> struct RowChunks {
  static constexpr int C = V > 1 ? V : 2;
  static constexpr int N = E / C;
  static constexpr int STEP = TPR ? TPR : 32;
  static constexpr int ELT = static_cast<int>(sizeof(T));
  static constexpr int REGION = STEP * E * ELT + (V > 1 ? 0 : 16);  // bytes of one row's segment
  static constexpr int WARP_ARRAY = 32 / STEP * REGION;             // of one array in a warp's part
  static constexpr int WARP_FACTORS = 32 * E * 4;
  static constexpr int FW = C >= 4 ? 4 : 2;  // fp32 factors per access
  static_assert(V == 1 || V * ELT <= 16, "one vector per slot");

  static __device__ __forceinline__ int lane() { return static_cast<int>(threadIdx.x & 31) % STEP; }
  // first column of this thread's segment, and of this thread
  static __device__ __forceinline__ int segment(int warp0 = 0) {
    return TPR ? 0 : (warp0 + static_cast<int>(threadIdx.x >> 5)) * (32 * E);
  }
  static __device__ __forceinline__ int base(int warp0 = 0) { return segment(warp0) + lane() * V; }
  // offset of element e of chunk c from it
  static __device__ __forceinline__ constexpr int off(int c, int e) { return V > 1 ? c * STEP * V + e : (2 * c + e) * STEP; }
  // whether a row with `len` values from the segment's first column on has any in chunk c of some lane (V = 1)
  static __device__ __forceinline__ bool reaches(int c, int len) { return V > 1 || 2 * c * STEP < len; }
  static __device__ __forceinline__ unsigned char* region(unsigned char* array) {
    return array + (V > 1 ? 0 : static_cast<int>(threadIdx.x & 31) / STEP * REGION);
  }
  // V > 1: the thread's slot for chunk c
  static __device__ __forceinline__ T* slot(unsigned char* array, int c) {
    return reinterpret_cast<T*>(array) + c * (32 * V) + static_cast<int>(threadIdx.x & 31) * V;
  }
  static __device__ __forceinline__ void sync() {
    if constexpr (V == 1) __syncwarp();
  }
  // the shift of a row's segment: rows of `stride` values from `first` on
  static __device__ __forceinline__ int shift(const void* first, int64_t stride, int64_t row) {
    if constexpr (V > 1) return 0;
    return static_cast<int>((static_cast<uint32_t>(reinterpret_cast<uintptr_t>(first)) +
                             static_cast<uint32_t>(row) * static_cast<uint32_t>(stride) * ELT) & 15u);
  }
  // starts the copies of a segment: `seg` points at its first column, `len` values of the row lie from
  // there on, `floor` is the tensor's first value
  static __device__ __forceinline__ void copy(unsigned char* array, const T* seg, int len, const void* floor) {
    if constexpr (V > 1) {
      const int left = len - lane() * V;
      const T* row = seg + lane() * V;
#pragma unroll
      for (int c = 0; c < N; ++c)
        if (off(c, 0) < left) copy_async<V * ELT>(slot(array, c), row + off(c, 0));
    } else {
      if (len <= 0) return;
      const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(seg) & 15);
      const unsigned char* from = reinterpret_cast<const unsigned char*>(seg) - shift;
      const int bytes = shift + min(len, STEP * E) * ELT;
      unsigned char* to = region(array);
      constexpr int GRANULES = STEP * E * ELT / 16 + 1;
#pragma unroll
      for (int i = 0; i < (GRANULES + STEP - 1) / STEP; ++i) {
        const int at = (lane() + i * STEP) * 16;
        if (at >= min(len, STEP * E) * ELT + 16) break;  // where no shift's end lies
        if (i == 0 && at == 0 && from < floor) {
          for (int e = shift; e < 16; e += ELT)
            *reinterpret_cast<T*>(to + e) = e < bytes ? *reinterpret_cast<const T*>(from + e) : T{};
        } else {
          // behind the row's end nothing is read, from an address that is the row's all the same
          const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(to + at));
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                       ::"r"(d), "l"(from + min(at, (bytes - 1) & ~15)), "r"(max(0, min(16, bytes - at))) : "memory");
        }
      }
    }
  }
  // zeros where no copy ever lands: behind the row's end (V > 1), or everywhere if the array is absent.
  // sync() stands between this and the first copy.
  static __device__ __forceinline__ void zero_rest(unsigned char* array, bool present, int left) {
    if constexpr (V > 1) {
#pragma unroll
      for (int c = 0; c < N; ++c)
        if (!present || off(c, 0) >= left) *reinterpret_cast<Vec<T, V>*>(slot(array, c)) = Vec<T, V>{};
    } else {
      for (int i = lane() * 16; i < REGION; i += STEP * 16) *reinterpret_cast<uint4*>(region(array) + i) = uint4{};
    }
  }
  static __device__ __forceinline__ void read_raw(unsigned char* array, int shift, int c, Vec<T, C>& v) {
    if constexpr (V > 1) {
      v = *reinterpret_cast<const Vec<T, V>*>(slot(array, c));
    } else {
      const T* row = reinterpret_cast<const T*>(region(array) + shift) + lane();
#pragma unroll
      for (int e = 0; e < 2; ++e) v.v[e] = row[off(c, e)];
    }
  }
  static __device__ __forceinline__ void read(unsigned char* array, int shift, int c, float (&v)[C]) {
    Vec<T, C> raw;
    read_raw(array, shift, c, raw);
#pragma unroll
    for (int e = 0; e < C; ++e) v[e] = to_f(raw.v[e]);
  }
  // chunk c of a row in global memory; `left`: values of the row from the thread's first column on
  static __device__ __forceinline__ void load(const T* row, int c, int left, float (&v)[C]) {
    if constexpr (V > 1) {
      Vec<T, V> raw{};
      if (off(c, 0) < left) raw = *reinterpret_cast<const Vec<T, V>*>(row + off(c, 0));
#pragma unroll
      for (int e = 0; e < C; ++e) v[e] = to_f(raw.v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < C; ++e) v[e] = off(c, e) < left ? to_f(row[off(c, e)]) : 0.f;
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
  // multiplies the thread's own values of a staged row, or of the row it wrote, by a power of two
  static __device__ __forceinline__ void scale(unsigned char* array, int shift, int left, float by) {
    if constexpr (V > 1) {
#pragma unroll 1
      for (int c = 0; c < N; ++c) {
        Vec<T, V>& v = *reinterpret_cast<Vec<T, V>*>(slot(array, c));
        for (int e = 0; e < V; ++e) v.v[e] = from_f<T>(to_f(v.v[e]) * by);
      }
    } else {
      scale_row(reinterpret_cast<T*>(region(array) + shift) + lane(), left, by);
    }
  }
  static __device__ __forceinline__ void scale_row(T* row, int left, float by) {
#pragma unroll 1
    for (int c = 0; c < N; ++c)
      for (int e = 0; e < C; ++e)
        if (off(c, e) < left) row[off(c, e)] = from_f<T>(to_f(row[off(c, e)]) * by);
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
  static __device__ __forceinline__ void write_factors(unsigned char* array, int c, const float (&v)[C]) {
#pragma unroll
    for (int e = 0; e < C; e += FW) {
      Vec<float, FW> f;
#pragma unroll
      for (int i = 0; i < FW; ++i) f.v[i] = v[e + i];
      *reinterpret_cast<Vec<float, FW>*>(fslot(array, c, e)) = f;
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
// A thread's share of RowChunks::WARP_ARRAY, rounded up.
constexpr int row_bytes_per_thread(int elts, int elt, bool vec, int tpr) {
  const int step = tpr ? tpr : 32;
  return elts * elt + (vec ? 0 : (16 + step - 1) / step);
}
static_assert(32 * row_bytes_per_thread(16, 2, false, 0) >= RowChunks<__half, 1, 0, 16>::WARP_ARRAY &&
              32 * row_bytes_per_thread(16, 4, false, 8) >= RowChunks<float, 1, 8, 16>::WARP_ARRAY &&
              32 * row_bytes_per_thread(16, 1, false, 16) >= RowChunks<uint8_t, 1, 16, 16>::WARP_ARRAY &&
              32 * row_bytes_per_thread(16, 2, true, 32) >= RowChunks<__half, 8, 32, 16>::WARP_ARRAY);

// ---- thread-block clusters: rows wider than a block holds are shared by up to kMaxRanks blocks ----
constexpr int kMaxRanks = 8;
__device__ __forceinline__ int cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return static_cast<int>(r);
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// writes v to the same place of block `rank`'s shared memory
__device__ __forceinline__ void store_at_rank(float4* mine, int rank, float4 v) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(at) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(mine))), "r"(rank));
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
}

// Sums over the threads that share a row: TPR lanes of a warp, or (TPR = 0) the block or the `ranks`
// blocks of its cluster.  `red` (sum_bytes of shared memory) holds two phases of a float4 per warp
// of the row, so one barrier per call is enough: a block that runs ahead writes the other phase, and
// waits there for the ones behind it.  N <= 4.
constexpr int kBlockWarps = 32, kRowWarps = 128;  // at most, of a block and of kMaxRanks blocks of 16
constexpr int sum_bytes(int ranks) { return 2 * 16 * (ranks == 1 ? kBlockWarps : kRowWarps); }
template <int TPR, int N>
__device__ __forceinline__ void sum_row(float (&s)[N], float4* red, int& phase, int ranks = 1) {
  constexpr int G = TPR ? TPR : 32;
#pragma unroll
  for (int d = G / 2; d > 0; d >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] += __shfl_xor_sync(0xffffffffu, s[i], d);
  if constexpr (TPR == 0) {
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const float4 mine = make_float4(s[0], N > 1 ? s[N > 1 ? 1 : 0] : 0.f, N > 2 ? s[N > 2 ? 2 : 0] : 0.f, N > 3 ? s[N > 3 ? 3 : 0] : 0.f);
    float4 t;
    if (ranks == 1 && N == 1) {
      float* row = reinterpret_cast<float*>(red) + phase * kBlockWarps;
      if (lane == 0) row[w] = s[0];
      __syncthreads();
      t.x = row[0];
      for (int k = 1; k < warps; ++k) t.x += row[k];
    } else if (ranks == 1) {
      if (lane == 0) red[phase * kBlockWarps + w] = mine;
      __syncthreads();
      t = red[phase * kBlockWarps];
      for (int k = 1; k < warps; ++k) {
        const float4 f = red[phase * kBlockWarps + k];
        t.x += f.x; t.y += f.y; t.z += f.z; t.w += f.w;
      }
    } else {
      float4* row = red + phase * kRowWarps;
      if (lane < ranks) store_at_rank(row + cluster_rank() * warps + w, lane, mine);
      __syncwarp();
      cluster_sync();
      // a lane adds every 32nd warp's part and the lanes fold; all parts one after the other in every thread took
      // the backward of [8192,16384] bf16 458 us, so 428
      t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
      for (int k = lane; k < warps * ranks; k += 32) {
        const float4 f = row[k];
        t.x += f.x; t.y += f.y; t.z += f.z; t.w += f.w;
      }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) {
        t.x += __shfl_xor_sync(0xffffffffu, t.x, d);
        if constexpr (N > 1) t.y += __shfl_xor_sync(0xffffffffu, t.y, d);
        if constexpr (N > 2) t.z += __shfl_xor_sync(0xffffffffu, t.z, d);
        if constexpr (N > 3) t.w += __shfl_xor_sync(0xffffffffu, t.w, d);
      }
    }
    s[0] = t.x;
    if constexpr (N > 1) s[1] = t.y;
    if constexpr (N > 2) s[2] = t.z;
    if constexpr (N > 3) s[3] = t.w;
    phase ^= 1;
  }
}

// Launches `kernel` with clusters of `ranks` blocks (1: none).
template <class Kernel, class Params>
inline cudaError_t launch_ranks(Kernel kernel, const Params& p, unsigned grid, int threads, int smem, int ranks, cudaStream_t s) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(ranks);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ranks > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}
// Clusters of this size that fit the card at once: pairs always do, larger ones leave out what a
// group of SMs has left over.
inline int64_t clusters_at_once(int sms, int ranks) { return std::max(1, ranks <= 2 ? sms / ranks : sms / ranks * 7 / 8); }

constexpr int kSmemPerSm = 228 * 1024;     // of which every block takes 1 KB for the system
constexpr int kSmemPerBlock = 227 * 1024;

// Shared memory beyond the default limit has to be asked for once per kernel and device.
template <class Kernel>
inline cudaError_t allow_shared(Kernel kernel, int device, std::atomic<uint64_t>& done, int most = kSmemPerBlock) {
  const uint64_t bit = 1ull << (device & 63);
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

}  // namespace vb

// A paged key/value cache in 8 bits: rows quantised as they are written, and read back through a
// page table (sm_100a).
//
// A row is one head of one token; its levels lie at cache[slot][head][0 .. dim) and its scale at
// scale[slot][head].  Both directions move every byte once and are bound by memory: 135,000 tokens of
// 8 heads x 128 bf16 are read and written in 140 us each, 6.0 TB/s.
//
// Several tokens of one write may name the same slot.  A row and its scale are written by several
// threads in several stores, so two writers could leave one's levels with the other's scale; only
// the last token of a slot may write it.  Few tokens look for a later equal slot themselves; many settle
// it in `owner` in a launch of their own: the largest token number claims the slot, and the winner
// puts the entry back to zero.
#include <algorithm>

#include "quant8.cuh"
#include "row_tile.cuh"

namespace vb {
namespace {

constexpr int kKvThreads = 128;

__device__ __forceinline__ int64_t load_index(const void* p, int dtype, int64_t i) {
  return dtype == VBT_B200_I64 ? static_cast<const int64_t*>(p)[i] : static_cast<int64_t>(static_cast<const int32_t*>(p)[i]);
}
__device__ __forceinline__ void count_bad(unsigned long long* status, int64_t v) {
  if (status && atomicAdd(&status[0], 1ull) == 0ull) status[1] = static_cast<unsigned long long>(v);
}

struct KvWriteParams {
  const void* src[2];        // k, v
  int64_t src_t[2], src_h[2];
  uint8_t* cache[2];
  float* scale[2];
  const void* slots;
  int32_t* owner;
  unsigned long long* status;
  int64_t num_slots, tokens;
  int slots_dtype;
  int heads, dim;
  int tb;                    // tokens of a block
  int scan;                  // look for a later equal slot here; else `owner` has been settled
  FastDiv div_heads;
};

__global__ void __launch_bounds__(kKvThreads) kv_claim_kernel(const __grid_constant__ KvWriteParams p) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kKvThreads + threadIdx.x;
  if (i >= p.tokens) return;
  const int64_t s = load_index(p.slots, p.slots_dtype, i);
  if (s >= 0 && s < p.num_slots) atomicMax(p.owner + s, static_cast<int32_t>(i) + 1);
}

constexpr int kKvMaxTokens = 32;  // tokens of a block

// L lanes own a row; VEC: 16-byte vectors, VPL of them per lane; else single values, the row read twice
template <class T, bool VEC, int L, int VPL, int F>
__global__ void __launch_bounds__(kKvThreads) kv_write_kernel(const __grid_constant__ KvWriteParams p) {
  constexpr int V = 16 / sizeof(T);
  __shared__ int64_t slot_of[kKvMaxTokens];
  __shared__ int later[kKvMaxTokens];
  const int64_t first = static_cast<int64_t>(blockIdx.x) * p.tb;
  const int tb = static_cast<int>(min(static_cast<int64_t>(p.tb), p.tokens - first));
  if (threadIdx.x < tb) {
    const int64_t i = first + threadIdx.x;
    int64_t s = load_index(p.slots, p.slots_dtype, i);
    if (s >= p.num_slots) count_bad(p.status, s);
    if (s < 0 || s >= p.num_slots) s = -1;
    if (s >= 0 && !p.scan) {
      if (p.owner[s] == static_cast<int32_t>(i) + 1) p.owner[s] = 0;
      else s = -1;
    }
    slot_of[threadIdx.x] = s;
    later[threadIdx.x] = 0;
  }
  __syncthreads();
  if (p.scan && p.tokens > 1) {
    for (int64_t j = first + 1 + threadIdx.x; j < p.tokens; j += kKvThreads) {
      const int64_t s = load_index(p.slots, p.slots_dtype, j);
      if (s < 0) continue;
      for (int k = 0; k < tb; ++k)
        if (slot_of[k] == s && j > first + k) later[k] = 1;
    }
    __syncthreads();
  }
  const int lane = threadIdx.x % L;
  const int rows = tb * 2 * p.heads;
  // every lane of a warp makes the same number of rounds (shuffles inside)
  for (int r0 = 0; r0 < rows; r0 += kKvThreads / L) {
    const int r = r0 + threadIdx.x / L;
    uint32_t tk = 0, h = 0;
    if (r < rows) p.div_heads.divmod(static_cast<uint32_t>(r), tk, h);
    const int kv = tk & 1, tok = tk >> 1;
    const int64_t slot = r < rows && !later[tok] ? slot_of[tok] : -1;
    const bool live = slot >= 0;
    const int64_t row = live ? slot * p.heads + h : 0;
    const T* src = static_cast<const T*>(p.src[kv]) + (first + tok) * p.src_t[kv] + static_cast<int64_t>(h) * p.src_h[kv];
    uint8_t* dst = p.cache[kv] + row * p.dim;
    Q8Scale s;
    if constexpr (VEC) {
      const int nv = live ? p.dim / V : 0;
      Vec<T, V> raw[VPL];
      load_vecs<T, V, VPL>(src, lane, L, nv, raw);
      s = q8_scale<F>(group_mag<T, V, VPL, L>(raw));
#pragma unroll
      for (int k = 0; k < VPL; ++k) {
        const int j = lane + k * L;
        if (j >= nv) continue;
        float v[V];
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = to_f(raw[k].v[e]);
        q8_store<F, V>(dst + j * V, v, s.up);
      }
    } else {
      const int n = live ? p.dim : 0;
      uint32_t m = 0;
      for (int j = lane; j < n; j += L) m = max(m, mag_bits(to_f(src[j])));
      s = q8_scale<F>(lanes_max<L>(m));
      for (int j = lane; j < n; j += L) dst[j] = q8_pack1<F>(to_f(src[j]), s.up);
    }
    if (live && lane == 0) p.scale[kv][row] = s.down;
  }
}

struct KvReadParams {
  const uint8_t* cache[2];
  const float* scale[2];
  void* out[2];
  const void* table;
  const int64_t* starts;
  unsigned long long* status;
  int64_t rows, seqs, num_pages, page_size, table_stride, pages_per_seq;
  int table_dtype, fill;
  int heads, dim;
  int tb;          // rows of a block
  int chunks;      // vectors of a row (one of k or v)
  FastDiv div_row;   // by 2 * chunks
  FastDiv div_head;  // by vectors per head
};

// V values per piece of work: one load of levels, one scale, one store
template <class T, int V, int F, int U>
__global__ void __launch_bounds__(kKvThreads) kv_read_kernel(const __grid_constant__ KvReadParams p) {
  __shared__ int64_t slot_of[kKvMaxTokens];  // >= 0 slot, -1 zeros, -2 leave alone
  const int64_t first = static_cast<int64_t>(blockIdx.x) * p.tb;
  const int tb = static_cast<int>(min(static_cast<int64_t>(p.tb), p.rows - first));
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    // the sequence of the block's first row, the last s with starts[s] <= first: 32 probes at a time
    int64_t lo = 0, n = p.seqs;  // it lies in [lo - 1, lo + n)
    while (n > 0) {
      const int64_t hop = (n + 31) / 32;
      const int64_t probe = min(lo + (lane + 1) * hop, lo + n) - 1;
      const int below = __popc(__ballot_sync(0xffffffffu, p.starts[probe] <= first));  // ascending
      if (hop == 1) {
        lo += min(static_cast<int64_t>(below), n);
        break;
      }
      const int64_t from = below * hop;
      lo += min(from, n);
      n = from >= n ? 0 : min(hop, n - from) - 1;  // the last of the piece is known to lie above
    }
    const int64_t i = first + lane;
    int64_t s = lo - 1;
    if (lane < tb && s + 1 < p.seqs && p.starts[s + 1] <= i) {  // a later row's own sequence
      int64_t a = s + 1, b = p.seqs;
      while (a < b) {
        const int64_t mid = (a + b) >> 1;
        if (p.starts[mid] <= i) a = mid + 1;
        else b = mid;
      }
      s = a - 1;
    }
    int64_t slot = p.fill ? -1 : -2;
    if (lane < tb && s >= 0 && i < p.starts[s + 1]) {
      const int64_t pos = i - p.starts[s], pg = pos / p.page_size;  // negative: starts that do not ascend
      int64_t page = -1;
      if (pos >= 0 && pg < p.pages_per_seq) page = load_index(p.table, p.table_dtype, s * p.table_stride + pg);
      if (page >= 0 && page < p.num_pages) {
        slot = page * p.page_size + (pos - pg * p.page_size);
      } else {
        slot = -1;
        count_bad(p.status, page);
      }
    }
    if (lane < tb) slot_of[lane] = slot;
  }
  __syncthreads();
  const int total = tb * 2 * p.chunks;
  for (int i0 = threadIdx.x; i0 < total; i0 += kKvThreads * U) {
    typename Q8Raw<V>::type q[U];
    float sc[U];
    int64_t at[U];
    int kv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kKvThreads;
      at[u] = -1;
      kv[u] = 0;
      q[u] = {};
      sc[u] = 0.f;
      if (i < total) {
        uint32_t tok, c, h, rest;
        p.div_row.divmod(static_cast<uint32_t>(i), tok, c);
        kv[u] = c >= static_cast<uint32_t>(p.chunks);
        if (kv[u]) c -= p.chunks;
        const int64_t slot = slot_of[tok];
        if (slot != -2) at[u] = (first + tok) * p.heads * p.dim + static_cast<int64_t>(c) * V;
        if (slot >= 0) {
          p.div_head.divmod(c, h, rest);
          q[u] = *reinterpret_cast<const typename Q8Raw<V>::type*>(p.cache[kv[u]] + slot * p.heads * p.dim +
                                                                   static_cast<int64_t>(c) * V);
          sc[u] = __ldg(p.scale[kv[u]] + slot * p.heads + h);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (at[u] < 0) continue;
      float v[V];
      q8_widen<F, V>(q[u], sc[u], v);
      constexpr int W = V * sizeof(T) > 16 ? 16 / sizeof(T) : V;
#pragma unroll
      for (int a = 0; a < V; a += W) {
        Vec<T, W> o;
#pragma unroll
        for (int e = 0; e < W; ++e) o.v[e] = from_f<T>(v[a + e]);
        *reinterpret_cast<Vec<T, W>*>(static_cast<T*>(p.out[kv[u]]) + at[u] + a) = o;
      }
    }
  }
}

#define VB_KV_FORMAT(format, F, ...)                                                  \
  do {                                                                                \
    if ((format) == VBT_B200_Q8_INT8) { constexpr int F = VBT_B200_Q8_INT8; __VA_ARGS__; } \
    else { constexpr int F = VBT_B200_Q8_E4M3; __VA_ARGS__; }                         \
  } while (0)

inline bool aligned(const void* q, int bytes) { return reinterpret_cast<uintptr_t>(q) % bytes == 0; }

template <class T>
int launch_write(KvWriteParams p, int format, cudaStream_t s, int sms) {
  constexpr int V = 16 / sizeof(T);
  bool vec = p.dim % V == 0 && p.dim / V <= 256;
  for (int i = 0; i < 2; ++i)
    vec = vec && aligned(p.src[i], 16) && aligned(p.cache[i], 8) && p.src_t[i] % V == 0 && p.src_h[i] % V == 0;
  const int nv = vec ? p.dim / V : 0;
  // four vectors per lane: what a lane works out per row (slot, addresses, the scale) is shared by 32 or
  // 64 bytes of it.  135,000 tokens of 8 heads x 128 bf16: one vector per lane 200 us, two 155, four 133
  const int lanes = !vec || nv > 64 ? 32 : nv > 32 ? 16 : nv > 16 ? 8 : nv > 8 ? 4 : 2;
  // about eight rounds of rows per thread, as long as the card is full of blocks
  const int64_t rows = 2 * int64_t{p.heads};
  int64_t tb = std::max<int64_t>(1, 8 * (kKvThreads / lanes) / rows);
  tb = std::min<int64_t>(tb, std::max<int64_t>(1, p.tokens / (4 * sms)));
  p.tb = static_cast<int>(std::min<int64_t>(tb, kKvMaxTokens));
  p.scan = p.tokens <= 512;
  int launches = 1;
  if (!p.scan) {
    kv_claim_kernel<<<static_cast<unsigned>((p.tokens + kKvThreads - 1) / kKvThreads), kKvThreads, 0, s>>>(p);
    ++launches;
  }
  const unsigned g = static_cast<unsigned>((p.tokens + p.tb - 1) / p.tb);
#define VB_KW(VEC, L, VPL) VB_KV_FORMAT(format, F, (kv_write_kernel<T, VEC, L, VPL, F><<<g, kKvThreads, 0, s>>>(p)))
  if (!vec) VB_KW(false, 32, 1);
  else if (nv <= 8) VB_KW(true, 2, 4);
  else if (nv <= 16) VB_KW(true, 4, 4);
  else if (nv <= 32) VB_KW(true, 8, 4);
  else if (nv <= 64) VB_KW(true, 16, 4);
  else VB_KW(true, 32, 8);
#undef VB_KW
  note_launch(VBT_B200_FAMILY_INDEX, VBT_B200_IK_KV_CACHE_WRITE, dim3(g), dim3(kKvThreads), vec ? V : 1, 1, 0, launches,
              2 * p.tokens * p.heads * p.dim, p.tokens, 0, s);
  return 0;
}

template <class T>
int launch_read(KvReadParams p, int format, cudaStream_t s, int sms) {
  int v = 16 / static_cast<int>(sizeof(T));
  for (; v > 1; v /= 2) {
    if (v == 2) continue;
    bool ok = p.dim % v == 0;
    for (int i = 0; i < 2; ++i)
      ok = ok && aligned(p.cache[i], v) && aligned(p.out[i], std::min<int>(16, v * static_cast<int>(sizeof(T))));
    if (ok) break;
  }
  if (v < 4) v = 1;
  p.chunks = p.heads * p.dim / v;
  p.div_row = FastDiv(static_cast<uint32_t>(2 * p.chunks));
  p.div_head = FastDiv(static_cast<uint32_t>(p.dim / v));
  constexpr int U = 2;
  int64_t tb = std::max<int64_t>(1, 8 * U * kKvThreads / (2 * int64_t{p.chunks}));
  tb = std::min<int64_t>(tb, std::max<int64_t>(1, p.rows / (4 * sms)));
  p.tb = static_cast<int>(std::min<int64_t>(tb, kKvMaxTokens));
  const unsigned g = static_cast<unsigned>((p.rows + p.tb - 1) / p.tb);
#define VB_KR(V) VB_KV_FORMAT(format, F, (kv_read_kernel<T, V, F, U><<<g, kKvThreads, 0, s>>>(p)))
  if (v == 4) VB_KR(4);
  else if (v == 1) VB_KR(1);
  else if constexpr (sizeof(T) == 2) VB_KR(8);
#undef VB_KR
  note_launch(VBT_B200_FAMILY_INDEX, VBT_B200_IK_KV_CACHE_READ, dim3(g), dim3(kKvThreads), v, 1, 0, 1,
              2 * p.rows * p.heads * p.dim, p.rows, 0, s);
  return 0;
}

vbt_b200_status check_cache(const char* name, int64_t num_slots, int64_t heads, int64_t dim, int32_t format, int32_t dtype) {
  VB_ARG(is_float_dtype(dtype), std::string(name) + ": expected a floating dtype");
  VB_ARG(format == VBT_B200_Q8_INT8 || format == VBT_B200_Q8_E4M3, std::string(name) + ": unknown 8-bit format");
  VB_ARG(num_slots >= 0 && heads >= 0 && dim >= 0, std::string(name) + ": negative size");
  VB_ARG(heads <= 65536 && dim <= 65536 && heads * dim <= (int64_t{1} << 24), std::string(name) + ": rows too wide");
  return VBT_B200_OK;
}

}  // namespace
}  // namespace vb

extern "C" {

vbt_b200_status vbt_b200_kv_cache_write(void* k_cache, float* k_scale, void* v_cache, float* v_scale, int64_t num_slots,
                                        int64_t heads, int64_t dim, int32_t format, const void* k,
                                        const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                        int32_t dtype, const void* slots, int32_t slots_dtype, int64_t tokens,
                                        int32_t* owner, void* index_status, void* stream) {
  using namespace vb;
  const char* name = "kv_cache_write";
  VB_TRY(check_cache(name, num_slots, heads, dim, format, dtype));
  VB_ARG(tokens >= 0 && tokens < INT32_MAX, std::string(name) + ": bad number of tokens");
  VB_ARG(slots_dtype == VBT_B200_I64 || slots_dtype == VBT_B200_I32, std::string(name) + ": slots must be int64 or int32");
  if (tokens == 0 || heads == 0 || dim == 0) return VBT_B200_OK;
  VB_ARG(num_slots == 0 || (k_cache && k_scale && v_cache && v_scale && owner), std::string(name) + ": null pointer");
  VB_ARG(k && v && k_strides && v_strides && slots, std::string(name) + ": null pointer");
  VB_ARG(k_strides[0] >= 0 && k_strides[1] >= 0 && v_strides[0] >= 0 && v_strides[1] >= 0,
         std::string(name) + ": negative stride");
  DeviceScope scope(num_slots ? static_cast<const void*>(k_cache) : k);
  KvWriteParams p{};
  p.src[0] = k; p.src[1] = v;
  p.src_t[0] = k_strides[0]; p.src_h[0] = k_strides[1]; p.src_t[1] = v_strides[0]; p.src_h[1] = v_strides[1];
  p.cache[0] = static_cast<uint8_t*>(k_cache); p.cache[1] = static_cast<uint8_t*>(v_cache);
  p.scale[0] = k_scale; p.scale[1] = v_scale;
  p.slots = slots; p.slots_dtype = slots_dtype; p.owner = owner;
  p.status = static_cast<unsigned long long*>(index_status);
  p.num_slots = num_slots; p.tokens = tokens;
  p.heads = static_cast<int>(heads); p.dim = static_cast<int>(dim);
  p.div_heads = FastDiv(static_cast<uint32_t>(heads));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int sms = sm_count(scope.device());
  switch (dtype) {
    case VBT_B200_F32: launch_write<float>(p, format, s, sms); break;
    case VBT_B200_F16: launch_write<__half>(p, format, s, sms); break;
    default: launch_write<__nv_bfloat16>(p, format, s, sms); break;
  }
  VB_LAUNCH_CHECK();
  return VBT_B200_OK;
}

vbt_b200_status vbt_b200_kv_cache_read(void* k_out, void* v_out, int32_t dtype, int64_t rows, const void* k_cache,
                                       const float* k_scale, const void* v_cache, const float* v_scale,
                                       int64_t num_slots, int64_t page_size, int64_t heads, int64_t dim, int32_t format,
                                       const void* page_table, int32_t page_table_dtype, int64_t page_table_stride,
                                       int64_t pages_per_seq, const int64_t* starts, int64_t seqs, int32_t fill,
                                       void* index_status, void* stream) {
  using namespace vb;
  const char* name = "kv_cache_read";
  VB_TRY(check_cache(name, num_slots, heads, dim, format, dtype));
  VB_ARG(rows >= 0 && seqs >= 0 && pages_per_seq >= 0 && page_table_stride >= 0, std::string(name) + ": negative size");
  VB_ARG(rows < (int64_t{1} << 31), std::string(name) + ": too many rows");
  VB_ARG(page_size > 0 && num_slots % page_size == 0, std::string(name) + ": page_size does not divide the slots");
  VB_ARG(page_table_dtype == VBT_B200_I64 || page_table_dtype == VBT_B200_I32,
         std::string(name) + ": page_table must be int64 or int32");
  if (rows == 0 || heads == 0 || dim == 0) return VBT_B200_OK;
  VB_ARG(k_out && v_out && starts, std::string(name) + ": null pointer");
  VB_ARG(num_slots == 0 || (k_cache && k_scale && v_cache && v_scale), std::string(name) + ": null pointer");
  VB_ARG(seqs == 0 || pages_per_seq == 0 || page_table, std::string(name) + ": null pointer");
  DeviceScope scope(k_out);
  KvReadParams p{};
  p.cache[0] = static_cast<const uint8_t*>(k_cache); p.cache[1] = static_cast<const uint8_t*>(v_cache);
  p.scale[0] = k_scale; p.scale[1] = v_scale;
  p.out[0] = k_out; p.out[1] = v_out;
  p.table = page_table; p.table_dtype = page_table_dtype; p.table_stride = page_table_stride;
  p.pages_per_seq = pages_per_seq; p.starts = starts; p.seqs = seqs;
  p.status = static_cast<unsigned long long*>(index_status);
  p.rows = rows; p.num_pages = num_slots / page_size; p.page_size = page_size;
  p.heads = static_cast<int>(heads); p.dim = static_cast<int>(dim); p.fill = fill;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int sms = sm_count(scope.device());
  switch (dtype) {
    case VBT_B200_F32: launch_read<float>(p, format, s, sms); break;
    case VBT_B200_F16: launch_read<__half>(p, format, s, sms); break;
    default: launch_read<__nv_bfloat16>(p, format, s, sms); break;
  }
  VB_LAUNCH_CHECK();
  return VBT_B200_OK;
}

}  // extern "C"

// Rotary positions with several axes, queries and keys in one launch (sm_100a).
//
//   pair i of a head turns by  angle = positions[axis(i), b, t] * inv_freq[i]
//   a' = a cos - b sin,  b' = b cos + a sin      (the backward pass turns by -angle)
//
// The angle is formed in 64 bits and reduced there to the part of a turn behind the nearest
// quarter, so a position of a million keeps every bit of its angle; sine and cosine of what is left
// are 32-bit.  A block computes the table of its tokens' cosines and sines once in shared memory
// and turns all the heads it owns with it: the operator moves every value once and is bound by
// memory.  18432 tokens of 40 heads of 128 bf16, among other calls: 72 us = 5.3 TB/s, 0.80 of the measured copy
// bandwidth (32 registers, full SMs).  With few heads the table is the larger part: 147,456 tokens of
// five heads take 100 us, 0.58.
#include <algorithm>

#include "common.cuh"

namespace vb {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotTokens = 32;  // most tokens of a block

struct RotSide {
  const void* in;
  void* out;
  int64_t in_b, in_t, in_h;     // strides in elements
  int64_t out_b, out_t, out_h;
};
struct RotParams {
  RotSide q, k;
  const void* pos;
  const float* freq;
  int64_t pos_a, pos_b, pos_t;
  int64_t count;        // batch * tokens
  int64_t tokens;
  int pos_dtype;
  int q_heads, heads;   // heads: q and k together
  int dim, half;
  int rot_items, items; // per head: vector pairs that turn, all pieces of work
  int tb, hb;           // tokens and heads of a block
  int end[VBT_B200_ROTARY_MAX_AXES];  // end[a]: first pair behind axis a's section
  FastDiv div_heads, div_half;  // by a block's heads, by half
  float sign;
};

// cos and sin of pi / 2 * quarters.  Adding 1.5 * 2^52 rounds to the nearest whole quarter and leaves it
// in the sum's low bits (|quarters| < 2^51); what is left of the turn goes to 32 bits.
__device__ __forceinline__ void turn(double quarters, float& c, float& s) {
  constexpr double kRound = 6755399441055744.0;
  const double whole = quarters + kRound;
  const float left = 0.5f * static_cast<float>(quarters - (whole - kRound));  // half turns, |left| <= 1/4
  const int qd = __double2loint(whole) & 3;
  float sl, cl;
  sincospif(left, &sl, &cl);
  c = (qd & 1) ? sl : cl;
  s = (qd & 1) ? cl : sl;
  if (qd == 1 || qd == 2) c = -c;
  if (qd >= 2) s = -s;
}

// P pairs per piece of work.  PAIRED: neighbours (2i, 2i + 1) in one vector of 2P values; else P
// values at i and P at half + i.  VEC: the vectors may be read whole.
template <class T, int P, bool PAIRED, bool VEC>
__global__ void __launch_bounds__(kRotThreads, 8) rotary_kernel(const __grid_constant__ RotParams p) {
  extern __shared__ float table[];  // cosines [tb][half], then sines
  const int64_t first = static_cast<int64_t>(blockIdx.x) * p.tb;
  const int tb = static_cast<int>(min(static_cast<int64_t>(p.tb), p.count - first));
  float* cosines = table;
  float* sines = table + p.tb * p.half;
  __shared__ int64_t place[kRotTokens][4];  // where a token's q and k begin: in, out, in, out
  if (threadIdx.x < tb) {
    const int64_t at = first + threadIdx.x, b = at / p.tokens, t = at - b * p.tokens;
    place[threadIdx.x][0] = b * p.q.in_b + t * p.q.in_t;
    place[threadIdx.x][1] = b * p.q.out_b + t * p.q.out_t;
    place[threadIdx.x][2] = b * p.k.in_b + t * p.k.in_t;
    place[threadIdx.x][3] = b * p.k.out_b + t * p.k.out_t;
  }
  for (int i = threadIdx.x; i < tb * p.half; i += kRotThreads) {
    uint32_t tok, f;
    p.div_half.divmod(static_cast<uint32_t>(i), tok, f);
    const int64_t at = first + tok, b = at / p.tokens, t = at - b * p.tokens;
    int axis = 0;
#pragma unroll
    for (int a = 0; a < VBT_B200_ROTARY_MAX_AXES - 1; ++a) axis += static_cast<int>(f) >= p.end[a];
    const int64_t src = axis * p.pos_a + b * p.pos_b + t * p.pos_t;
    const double pos = p.pos_dtype == VBT_B200_I64   ? static_cast<double>(static_cast<const int64_t*>(p.pos)[src])
                       : p.pos_dtype == VBT_B200_I32 ? static_cast<double>(static_cast<const int32_t*>(p.pos)[src])
                                                     : static_cast<double>(static_cast<const float*>(p.pos)[src]);
    float c, s;
    turn(pos * (static_cast<double>(p.freq[f]) * 0.63661977236758134308), c, s);  // 2 / pi
    cosines[i] = c;
    sines[i] = p.sign * s;
  }
  __syncthreads();
  const int h0 = blockIdx.y * p.hb;
  constexpr int W = PAIRED ? 2 * P : P;
  // A thread keeps its place in a head and walks the (token, head) pairs of the block, `slots` apart.
  // (Two or four of them in flight per thread cost registers, hence threads: 72 -> 84 -> 127 us for
  // 18432 tokens of 40 heads of 128 bf16, whatever the order of loads.)
  const int span = min(p.items, kRotThreads);
  const int slots = kRotThreads / span;
  const int mine = threadIdx.x / span;
  if (mine >= slots) return;
  const int pairs = tb * p.hb;
  for (int item = threadIdx.x - mine * span; item < p.items; item += span) {
    const bool turns = item < p.rot_items;
    const int i0 = turns ? item * P : 0;                                                            // first pair
    const int e0 = turns ? (PAIRED ? 2 * i0 : i0) : 2 * p.half + (item - p.rot_items) * W;  // first value
    for (int k = mine; k < pairs; k += slots) {
      uint32_t tok, hl;
      p.div_heads.divmod(static_cast<uint32_t>(k), tok, hl);
      const int h = h0 + static_cast<int>(hl);
      if (h >= p.heads) continue;
      const bool isq = h < p.q_heads;
      const int hh = isq ? h : h - p.q_heads;
      const T* in = static_cast<const T*>(isq ? p.q.in : p.k.in) + place[tok][isq ? 0 : 2] + hh * (isq ? p.q.in_h : p.k.in_h) + e0;
      T* out = static_cast<T*>(isq ? p.q.out : p.k.out) + place[tok][isq ? 1 : 3] + hh * (isq ? p.q.out_h : p.k.out_h) + e0;
      Vec<T, W> x, y;
      if constexpr (VEC) {
        x = *reinterpret_cast<const Vec<T, W>*>(in);
        if (!PAIRED && turns) y = *reinterpret_cast<const Vec<T, W>*>(in + p.half);
      } else {
#pragma unroll
        for (int e = 0; e < W; ++e)
          if (turns || e0 + e < p.dim) x.v[e] = in[e];
      }
      if (turns) {
        const float* ct = cosines + tok * p.half + i0;
        const float* st = sines + tok * p.half + i0;
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const float c = ct[e], s = st[e];
          T& a = PAIRED ? x.v[(2 * e) % W] : x.v[e % W];
          T& b = PAIRED ? x.v[(2 * e + 1) % W] : y.v[e % W];
          const float af = to_f(a), bf = to_f(b);
          a = from_f<T>(af * c - bf * s);
          b = from_f<T>(bf * c + af * s);
        }
      }
      if constexpr (VEC) {
        *reinterpret_cast<Vec<T, W>*>(out) = x;
        if (!PAIRED && turns) *reinterpret_cast<Vec<T, W>*>(out + p.half) = y;
      } else {
#pragma unroll
        for (int e = 0; e < W; ++e)
          if (turns || e0 + e < p.dim) out[e] = x.v[e];
      }
    }
  }
}

template <class T>
bool side_fits(const RotSide& s, int values) {
  const int bytes = values * static_cast<int>(sizeof(T));
  auto ok = [&](int64_t stride) { return stride % values == 0; };
  return reinterpret_cast<uintptr_t>(s.in) % bytes == 0 && reinterpret_cast<uintptr_t>(s.out) % bytes == 0 &&
         ok(s.in_b) && ok(s.in_t) && ok(s.in_h) && ok(s.out_b) && ok(s.out_t) && ok(s.out_h);
}

template <class T>
vbt_b200_status launch_rotary(RotParams p, int interleaved, cudaStream_t s, int sms) {
  constexpr int most = 16 / sizeof(T);
  const bool has_k = p.heads > p.q_heads, has_q = p.q_heads > 0;
  auto fits = [&](int values) {
    return (!has_q || side_fits<T>(p.q, values)) && (!has_k || side_fits<T>(p.k, values)) &&
           (p.dim - 2 * p.half) % values == 0;
  };
  // the widest vector that every address, the pairs and the rest of a head divide into
  int values = most, pairs = 1;
  bool vec = false;
  for (; values >= (interleaved ? 2 : 1); values /= 2) {
    pairs = interleaved ? values / 2 : values;
    if (p.half % pairs == 0 && fits(values)) { vec = true; break; }
  }
  if (!vec) { pairs = 1; values = interleaved ? 2 : 1; }
  p.rot_items = p.half / pairs;
  p.items = p.rot_items + (p.dim - 2 * p.half + values - 1) / values;
  p.div_half = FastDiv(static_cast<uint32_t>(std::max(p.half, 1)));
  // a block takes all heads of as many tokens as give each thread eight vectors (the table is worked out once
  // per token); with too few tokens to fill the card the heads are cut instead
  const int64_t per_token = int64_t{p.heads} * p.items * (interleaved ? 1 : 2);
  p.tb = static_cast<int>(std::min<int64_t>({int64_t{kRotTokens}, 8 * kRotThreads / std::max<int64_t>(per_token, 1), int64_t{4096 / std::max(p.half, 1)}}));
  // but no fewer than four blocks per SM
  p.tb = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(p.tb, p.count / (4 * sms))));
  p.hb = p.heads;
  if (p.count <= 2 * sms) {
    p.tb = 1;
    p.hb = std::max(1, std::min(p.heads, kRotThreads / std::max(p.items, 1)));
  }
  p.div_heads = FastDiv(static_cast<uint32_t>(p.hb));
  dim3 grid(static_cast<unsigned>((p.count + p.tb - 1) / p.tb), static_cast<unsigned>((p.heads + p.hb - 1) / p.hb));
  const size_t smem = static_cast<size_t>(p.tb) * p.half * 8;
#define VB_ROT(P, PAIRED, VEC) rotary_kernel<T, P, PAIRED, VEC><<<grid, kRotThreads, smem, s>>>(p)
  if (interleaved) {
    if (!vec) VB_ROT(1, true, false);
    else if (pairs == 1) VB_ROT(1, true, true);
    else if (pairs == 2) VB_ROT(2, true, true);
    else if constexpr (most == 8) VB_ROT(4, true, true);
  } else {
    if (pairs == 1) VB_ROT(1, false, true);
    else if (pairs == 2) VB_ROT(2, false, true);
    else if (pairs == 4) VB_ROT(4, false, true);
    else if constexpr (most == 8) VB_ROT(8, false, true);
  }
#undef VB_ROT
  VB_LAUNCH_CHECK();
  note_launch(VBT_B200_FAMILY_ROWOP, VBT_B200_WK_ROTARY, grid, dim3(kRotThreads), values, 1, 0, 1,
              p.count * p.heads * p.dim, p.dim, 0, s);
  return VBT_B200_OK;
}

}  // namespace
}  // namespace vb

extern "C" {

vbt_b200_status vbt_b200_rotary(void* q_out, const void* q, int64_t q_heads, void* k_out, const void* k,
                                int64_t k_heads, const int64_t* strides, int32_t dtype, int64_t batch, int64_t tokens,
                                int64_t dim, const void* positions, int32_t positions_dtype, const float* inv_freq,
                                int64_t half, const int64_t* sections, int32_t naxes, int32_t interleaved,
                                int32_t inverse, void* stream) {
  using namespace vb;
  VB_ARG(is_float_dtype(dtype), "rotary: expected a floating dtype");
  VB_ARG(batch >= 0 && tokens >= 0 && dim >= 0 && q_heads >= 0 && k_heads >= 0 && half >= 0, "rotary: negative size");
  VB_ARG(2 * half <= dim, "rotary: more pairs than the head has values for");
  VB_ARG(naxes >= 1 && naxes <= VBT_B200_ROTARY_MAX_AXES && sections, "rotary: expected 1 to 4 sections");
  int64_t sum = 0;
  for (int a = 0; a < naxes; ++a) {
    VB_ARG(sections[a] >= 0, "rotary: negative section");
    sum += sections[a];
  }
  VB_ARG(sum == half, "rotary: the sections do not sum to the number of pairs");
  VB_ARG(positions_dtype == VBT_B200_I64 || positions_dtype == VBT_B200_I32 || positions_dtype == VBT_B200_F32,
         "rotary: positions must be int64, int32 or float32");
  if (k == nullptr) k_heads = 0;
  if (batch == 0 || tokens == 0 || dim == 0 || q_heads + k_heads == 0) return VBT_B200_OK;
  VB_ARG(half <= 4096 && q_heads <= 16384 && k_heads <= 16384 && dim <= (int64_t{1} << 28) / (q_heads + k_heads),
         "rotary: head too wide or too many heads");
  VB_ARG(q_heads == 0 || (q && q_out), "rotary: null pointer");
  VB_ARG(k_heads == 0 || (k && k_out), "rotary: null pointer");
  VB_ARG(strides && (half == 0 || (positions && inv_freq)), "rotary: null pointer");
  VB_ARG(batch <= (int64_t{1} << 31) / tokens, "rotary: too many tokens");
  DeviceScope scope(q_heads ? q_out : k_out);
  RotParams p{};
  auto side = [](RotSide& s, const void* in, const int64_t* is, void* out, const int64_t* os) {
    s.in = in; s.in_b = is[0]; s.in_t = is[1]; s.in_h = is[2];
    s.out = out; s.out_b = os[0]; s.out_t = os[1]; s.out_h = os[2];
  };
  if (q_heads) side(p.q, q, strides + 3, q_out, strides);
  if (k_heads) side(p.k, k, strides + 9, k_out, strides + 6);
  p.pos = positions; p.pos_dtype = positions_dtype;
  p.pos_a = strides[12]; p.pos_b = strides[13]; p.pos_t = strides[14];
  p.freq = inv_freq;
  p.count = batch * tokens; p.tokens = tokens;
  p.q_heads = static_cast<int>(q_heads); p.heads = static_cast<int>(q_heads + k_heads);
  p.dim = static_cast<int>(dim); p.half = static_cast<int>(half);
  int64_t end = 0;
  for (int a = 0; a < VBT_B200_ROTARY_MAX_AXES; ++a) {
    end += a < naxes ? sections[a] : 0;
    // behind the last given section every pair stays on its axis
    p.end[a] = a < naxes - 1 ? static_cast<int>(end) : INT32_MAX;
  }
  p.sign = inverse ? -1.f : 1.f;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case VBT_B200_F32: return launch_rotary<float>(p, interleaved, s, sm_count(scope.device()));
    case VBT_B200_F16: return launch_rotary<__half>(p, interleaved, s, sm_count(scope.device()));
    default: return launch_rotary<__nv_bfloat16>(p, interleaved, s, sm_count(scope.device()));
  }
}

}  // extern "C"

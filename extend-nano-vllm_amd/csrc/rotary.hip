// Rotary position embedding of query and key heads, angles in 64 bits.
//
// Pair i of a head at position p turns by a = p * inv_freq[i]:
//   (x, y) -> factor * (x cos a - y sin a, y cos a + x sin a),
// the pair being elements (i, i + rot / 2) (half layout) or (2 i, 2 i + 1)
// (interleaved) of the head's first `rot` elements; what follows them passes
// through.  Frequencies scaled for long contexts come in through inv_freq, the
// scaling's amplitude through factor.
//
// Angles: p * inv_freq is formed and reduced to [-pi/4, pi/4] in float64 (in
// float32 an angle of 1e5 radians has an error of 4e-3), the sine and cosine of
// the rest are Taylor polynomials in float32 (truncated below 3e-8), and the
// rotation is float32 with one rounding to the tensor's type.
//
// What bounds it: memory (each element once in and once out) from some thousand
// tokens up, launch latency below: 16384 tokens of 40 bf16 heads, 336 MB, 67-68 us
// (5.0 TB/s; a copy reaches 5.07), 384 tokens 4.4 us, one token 2.3.  A workgroup
// takes a token: its threads first form one angle each, shared by all heads through
// LDS, then turn pairs 16 bytes at a time.  With few heads that leaves most threads
// idle: 16384 tokens of one head of 64 elements, 4.2 MB, take 11 us.
#include <type_traits>

#include "common.h"

namespace nva {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 256;       // rot <= 512
constexpr int kMaxHeadDim = 1024;

struct Heads {
  const void* in;
  void* out;
  int64_t in_row, in_head, out_row, out_head;   // element strides
};

struct RotaryParams {
  const int64_t* positions;
  const double* inv_freq;
  Heads q, k;
  float factor;
  int32_t num_tokens, hq, heads;       // heads: queries and keys
  int32_t head_dim;
  int32_t pairs, per_head;             // units of a head: pair chunks, then tail chunks
  int32_t pair_chunks;
};

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(uint16_t v) { return bf16_to_f32(v); }
template <>
__device__ __forceinline__ float to_f32(_Float16 v) { return static_cast<float>(v); }
template <>
__device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ uint16_t from_f32(float v) { return f32_to_bf16(v); }
template <>
__device__ __forceinline__ _Float16 from_f32(float v) { return static_cast<_Float16>(v); }
template <>
__device__ __forceinline__ float from_f32(float v) { return v; }

// (cos a, sin a) of a float64 angle: a = n pi/2 + r with |r| <= pi/4, pi/2 in
// two parts; the quadrant n mod 4 picks and signs the two polynomials.
__device__ __forceinline__ float2 cos_sin_of(double a) {
  const double n = __builtin_rint(a * 0.63661977236758134308);
  const double rd = __builtin_fma(-n, 6.123233995736766036e-17,
                                  __builtin_fma(-n, 1.5707963267948965580, a));
  const float r = static_cast<float>(rd), z = r * r;
  const float s =
      r + r * z * (-1.0f / 6 + z * (1.0f / 120 + z * (-1.0f / 5040 + z * (1.0f / 362880))));
  const float c = 1.0f + z * (-0.5f + z * (1.0f / 24 + z * (-1.0f / 720 + z * (1.0f / 40320))));
  const int quadrant = static_cast<int>(n - 4.0 * __builtin_floor(n * 0.25));
  const float cc = quadrant & 1 ? s : c, ss = quadrant & 1 ? c : s;
  return make_float2(quadrant == 1 || quadrant == 2 ? -cc : cc, quadrant >= 2 ? -ss : ss);
}

// N elements of type T as one access
template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack {
  T v[N];
};
// two of them, aligned as one
template <typename T>
struct Two {
  T v[2];
};

// P: pairs of a unit.  Half layout: P elements at i and P at i + pairs;
// interleaved: 2 P elements side by side.  A tail unit copies 2 P elements, at
// the pairs' alignment; units of one pair take any address, and the last of an
// odd tail copies one element.
template <typename T, int P, bool INTERLEAVED>
__global__ void __launch_bounds__(kThreads) rotary_kernel(RotaryParams p) {
  using Unit = std::conditional_t<P == 1, Two<T>, Pack<T, 2 * P>>;   // of the interleaved layout
  using Tail = std::conditional_t<INTERLEAVED, Unit, Two<Pack<T, P>>>;
  __shared__ float2 turn[kMaxPairs];
  const int64_t t = blockIdx.x;
  const double position = static_cast<double>(p.positions[t]);
  for (int e = threadIdx.x; e < p.pairs; e += kThreads) {
    const float2 cs = cos_sin_of(position * p.inv_freq[e]);
    turn[e] = make_float2(cs.x * p.factor, cs.y * p.factor);
  }
  __syncthreads();
  for (int u = threadIdx.x; u < p.heads * p.per_head; u += kThreads) {
    const int head = u / p.per_head, c = u - head * p.per_head;
    const bool is_q = head < p.hq;
    const Heads& hd = is_q ? p.q : p.k;
    const int h = is_q ? head : head - p.hq;
    const T* in = static_cast<const T*>(hd.in) + t * hd.in_row + h * hd.in_head;
    T* out = static_cast<T*>(hd.out) + t * hd.out_row + h * hd.out_head;
    if (c >= p.pair_chunks) {
      const int d = 2 * p.pairs + 2 * P * (c - p.pair_chunks);
      if constexpr (P > 1) {
        *reinterpret_cast<Tail*>(out + d) = *reinterpret_cast<const Tail*>(in + d);
      } else {
        out[d] = in[d];
        if (d + 1 < p.head_dim) out[d + 1] = in[d + 1];
      }
      continue;
    }
    const float2* cs = turn + P * c;
    if constexpr (INTERLEAVED) {
      Unit v = *reinterpret_cast<const Unit*>(in + 2 * P * c);
#pragma unroll
      for (int e = 0; e < P; ++e) {
        const float x = to_f32(v.v[2 * e]), y = to_f32(v.v[2 * e + 1]);
        v.v[2 * e] = from_f32<T>(x * cs[e].x - y * cs[e].y);
        v.v[2 * e + 1] = from_f32<T>(y * cs[e].x + x * cs[e].y);
      }
      *reinterpret_cast<Unit*>(out + 2 * P * c) = v;
    } else {
      Pack<T, P> a = *reinterpret_cast<const Pack<T, P>*>(in + P * c);
      Pack<T, P> b = *reinterpret_cast<const Pack<T, P>*>(in + p.pairs + P * c);
#pragma unroll
      for (int e = 0; e < P; ++e) {
        const float x = to_f32(a.v[e]), y = to_f32(b.v[e]);
        a.v[e] = from_f32<T>(x * cs[e].x - y * cs[e].y);
        b.v[e] = from_f32<T>(y * cs[e].x + x * cs[e].y);
      }
      *reinterpret_cast<Pack<T, P>*>(out + P * c) = a;
      *reinterpret_cast<Pack<T, P>*>(out + p.pairs + P * c) = b;
    }
  }
}

// Whether units of P pairs are whole accesses of at most 16 bytes everywhere.
bool fits(const RotaryParams& p, int size, int P, bool interleaved, int32_t tail) {
  const int bytes = size * P * (interleaved ? 2 : 1);
  auto aligned = [&](const Heads& h) {
    return ((reinterpret_cast<uintptr_t>(h.in) | reinterpret_cast<uintptr_t>(h.out)) % bytes == 0) &&
           (h.in_row * size) % bytes == 0 && (h.in_head * size) % bytes == 0 &&
           (h.out_row * size) % bytes == 0 && (h.out_head * size) % bytes == 0;
  };
  return bytes <= 16 && p.pairs % P == 0 && tail % (2 * P) == 0 && aligned(p.q) && aligned(p.k);
}

template <typename T, int P>
void launch(RotaryParams p, bool interleaved, int32_t tail, bool in_place, hipStream_t s) {
  if constexpr (P > 1) {
    if (!fits(p, sizeof(T), P, interleaved, tail)) {
      launch<T, P / 2>(p, interleaved, tail, in_place, s);
      return;
    }
  }
  p.pair_chunks = p.pairs / P;
  // in place the tail is where it belongs
  p.per_head = p.pair_chunks + (in_place ? 0 : (tail + 2 * P - 1) / (2 * P));
  const int32_t grid = p.num_tokens;
  if (interleaved) {
    if constexpr (2 * P * sizeof(T) <= 16) rotary_kernel<T, P, true><<<grid, kThreads, 0, s>>>(p);
  } else {
    rotary_kernel<T, P, false><<<grid, kThreads, 0, s>>>(p);
  }
}

}  // namespace
}  // namespace nva

using namespace nva;

extern "C" int nva_rotary_embedding(
    const int64_t* positions, const double* inv_freq, float factor, int interleaved, int dtype,
    const void* q, int64_t q_row_stride, int64_t q_head_stride, int32_t num_q_heads, const void* k,
    int64_t k_row_stride, int64_t k_head_stride, int32_t num_k_heads, int32_t num_tokens,
    int32_t head_dim, int32_t rotary_dim, void* q_out, int64_t q_out_row_stride,
    int64_t q_out_head_stride, void* k_out, int64_t k_out_row_stride, int64_t k_out_head_stride,
    void* stream) {
  if (num_tokens < 0 || num_q_heads < 0 || num_k_heads < 0 || head_dim <= 0 || rotary_dim <= 0 ||
      rotary_dim % 2 || rotary_dim > head_dim)
    return NVA_ERR_ARG;
  if (dtype != NVA_BF16 && dtype != NVA_F16 && dtype != NVA_F32) return NVA_ERR_ARG;
  if (head_dim > kMaxHeadDim || rotary_dim > 2 * kMaxPairs || num_q_heads > 4096 || num_k_heads > 4096)
    return NVA_ERR_UNSUPPORTED;
  if (num_tokens == 0 || num_q_heads + num_k_heads == 0) return NVA_OK;
  if (!positions || !inv_freq || (num_q_heads && (!q || !q_out)) || (num_k_heads && (!k || !k_out)))
    return NVA_ERR_ARG;
  RotaryParams p = {};
  p.positions = positions;
  p.inv_freq = inv_freq;
  p.factor = factor;
  if (num_q_heads) p.q = {q, q_out, q_row_stride, q_head_stride, q_out_row_stride, q_out_head_stride};
  if (num_k_heads) p.k = {k, k_out, k_row_stride, k_head_stride, k_out_row_stride, k_out_head_stride};
  p.num_tokens = num_tokens;
  p.hq = num_q_heads;
  p.heads = num_q_heads + num_k_heads;
  p.head_dim = head_dim;
  p.pairs = rotary_dim / 2;
  const int32_t tail = head_dim - rotary_dim;
  auto same = [](const Heads& h) { return h.in == h.out && h.in_row == h.out_row && h.in_head == h.out_head; };
  const bool in_place = same(p.q) && same(p.k);
  auto* s = static_cast<hipStream_t>(stream);
  const bool il = interleaved != 0;
  if (dtype == NVA_F32)
    launch<float, 4>(p, il, tail, in_place, s);
  else if (dtype == NVA_F16)
    launch<_Float16, 8>(p, il, tail, in_place, s);
  else
    launch<uint16_t, 8>(p, il, tail, in_place, s);
  return launch_status();
}

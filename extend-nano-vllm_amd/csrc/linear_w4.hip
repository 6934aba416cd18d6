// Projections of few rows over 4-bit weights:
//   out[m, n] = sum_k x[m, k] (code[n, k] - zero[k / G, n]) scale[k / G, n] + bias[n]
// with x in bf16, codes 0..15 two to a byte, group scales in bf16.
//
// A group's sum is formed from exact operands and scaled afterwards, so no
// weight is ever rounded: a code c becomes the bf16 value 16 + c by placing its
// four bits in the mantissa of 16 (one shift, one and-or for two codes), the
// MFMA sums (16 + c) x in fp32, a second MFMA with an operand of ones sums x
// itself, and  sum (c - z) x = sum (16 + c) x - (16 + z) sum x.  Scales and
// the sum over groups are fp32, the output is rounded once.
//
// What bounds it: the codes' stream from HBM for a few rows (a quarter of the
// bf16 weights'), then x's way from L2 into each CU.
//
// A workgroup of eight waves owns 16 NT weight rows; wave w takes the 128-wide
// chunks w, w + 8, ... of K.  A lane's 16 bytes are 32 codes of one row (lane l:
// row l % 16, codes 32 (l / 16) ..): a 128-wide chunk is four MFMAs deep.  Where
// groups are shorter than 128 the four lanes of a row exchange dwords (two
// permlane swaps each), so that an MFMA sums over 32 neighbouring codes.  x rows
// load as whole lines and become the B operand through LDS rows of the wave's
// own.  The waves' sums meet in LDS in wave order (deterministic).
#include "common.h"

namespace nva {
namespace {

constexpr int kWaves = 8;
constexpr int kChunkK = 128;
constexpr int kXPitch = 68;            // dwords per staged x row: 16-byte reads of 16 rows cover all banks

struct W4Params {
  const uint16_t* x;
  int64_t x_stride;
  const uint8_t* w;
  const uint16_t* scales;
  const uint8_t* zeros;
  const uint16_t* bias;
  uint16_t* out;
  int64_t out_stride;
  int32_t M, N, K, group;
};

// Two codes of a dword, nibbles S / 4 and S / 4 + 4, as the bf16 values 16 + c:
// 16 is 0x4180 and a code's lowest bit is bit 3 of the mantissa.
template <int S>
__device__ __forceinline__ uint32_t codes(uint32_t w) {
  const uint32_t at = S < 4 ? w << 3 : w >> (S - 3);
  return (at & 0x00780078u) | 0x41804180u;
}

// Eight codes as an MFMA operand, in the order 0, 4, 1, 5, 2, 6, 3, 7.
__device__ __forceinline__ bf16x8_t operand(uint32_t w) {
  return __builtin_bit_cast(bf16x8_t, make_uint4(codes<0>(w), codes<4>(w), codes<8>(w), codes<12>(w)));
}

// Eight neighbouring values of x in that order.
__device__ __forceinline__ uint4 as_operand(uint4 v) {
  return make_uint4(__builtin_amdgcn_perm(v.z, v.x, 0x05040100u), __builtin_amdgcn_perm(v.z, v.x, 0x07060302u),
                    __builtin_amdgcn_perm(v.w, v.y, 0x05040100u), __builtin_amdgcn_perm(v.w, v.y, 0x07060302u));
}

// Dword d of lane quarter r becomes dword r of quarter d.
__device__ __forceinline__ void transpose(uint32_t (&w)[4]) {
#pragma unroll
  for (int d = 0; d < 2; ++d) {
    const auto r = __builtin_amdgcn_permlane32_swap(w[d], w[d + 2], false, false);
    const uint32_t a = r[0], b = r[1];
    w[d] = a;
    w[d + 2] = b;
  }
#pragma unroll
  for (int d = 0; d < 4; d += 2) {
    const auto r = __builtin_amdgcn_permlane16_swap(w[d], w[d + 1], false, false);
    const uint32_t a = r[0], b = r[1];
    w[d] = a;
    w[d + 1] = b;
  }
}

// XL: x loads of a lane per chunk (4 rows each); NT: tiles of 16 weight rows;
// PER: MFMAs (of 32 codes) per group, 1, 2 or 4; D: chunks in flight.
template <int XL, int NT, int PER, int D>
__global__ void __launch_bounds__(kWave * kWaves, 2) linear_w4_kernel(W4Params p) {
  constexpr int MT = XL <= 4 ? 1 : XL / 4;             // tiles of 16 rows of x
  constexpr int kGroups = 4 / PER;                     // groups of a chunk
  constexpr int kStage = 4 * XL * kXPitch;
  constexpr int kSums = NT * MT * kWave * 4;
  constexpr int kOwn = kStage > kSums ? kStage : kSums;
  __shared__ __attribute__((aligned(16))) uint32_t lds[kWaves * kOwn];
  const int lane = threadIdx.x & (kWave - 1);
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int m16 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16 * NT;
  const int m0 = blockIdx.y * 64;
  const int M = p.M - m0 < 64 ? p.M - m0 : 64;
  uint32_t* const stage = lds + wv * kOwn;

  // rows past the end repeat the last one; what they give is not stored
  const uint8_t* wp[NT];
  int32_t sp[NT];                                      // first of this lane's four scales of a group
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = n0 + 16 * t + m16;
    wp[t] = p.w + static_cast<int64_t>(r < p.N ? r : p.N - 1) * (p.K / 2) + 16 * g;
    sp[t] = n0 + 16 * t + 4 * g;
  }
  const uint16_t* xp[XL];
#pragma unroll
  for (int t = 0; t < XL; ++t) {
    const int r = 4 * t + (lane >> 4);
    xp[t] = p.x + static_cast<int64_t>(m0 + (r < M ? r : M - 1)) * p.x_stride + 8 * m16;
  }
  const bool four = p.N % 4 == 0;                      // whole 8-byte reads of four scales
  const int groups = p.K / p.group;
  struct Chunk {
    uint4 w[NT], x[XL];
    uint2 s[NT][kGroups];
    uint32_t z[NT][kGroups];
  };
  auto load = [&](int c, Chunk& b) {
    const int k = c * kChunkK;
    // past the end of K x is zero and the codes are any (the row's first)
    const bool w_in = k + 32 * g < p.K, x_in = k + 8 * m16 < p.K;
#pragma unroll
    for (int t = 0; t < NT; ++t) b.w[t] = *reinterpret_cast<const uint4*>(wp[t] + (w_in ? k / 2 : -16 * g));
#pragma unroll
    for (int t = 0; t < XL; ++t)
      b.x[t] = x_in ? *reinterpret_cast<const uint4*>(xp[t] + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      int grp = (k + 32 * PER * i) / p.group;
      grp = grp < groups ? grp : groups - 1;
      const int64_t row = static_cast<int64_t>(grp) * p.N;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        b.z[t][i] = 0x08080808u;
        if (four) {
          const int n = sp[t] < p.N ? sp[t] : p.N - 4;
          b.s[t][i] = *reinterpret_cast<const uint2*>(p.scales + row + n);
          if (p.zeros) b.z[t][i] = *reinterpret_cast<const uint32_t*>(p.zeros + row + n);
        } else {
          uint32_t s[4], z = 0;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int n = sp[t] + e < p.N ? sp[t] + e : p.N - 1;
            s[e] = p.scales[row + n];
            if (p.zeros) z |= static_cast<uint32_t>(p.zeros[row + n]) << (8 * e);
          }
          b.s[t][i] = make_uint2(s[0] | (s[1] << 16), s[2] | (s[3] << 16));
          if (p.zeros) b.z[t][i] = z;
        }
      }
    }
  };
  f32x4_t acc[NT][MT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[t][m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const bf16x8_t ones = __builtin_bit_cast(bf16x8_t, make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u));
  const f32x4_t none = f32x4_t{0.f, 0.f, 0.f, 0.f};
  // an operand row that is not staged repeats one that is
  const int xrow = XL < 4 ? m16 & (4 * XL - 1) : m16;
  // the stage belongs to this wave: LDS runs its operations in order
  auto compute = [&](const Chunk& b) {
#pragma unroll
    for (int t = 0; t < XL; ++t)
      *reinterpret_cast<uint4*>(stage + (4 * t + (lane >> 4)) * kXPitch + 4 * m16) = as_operand(b.x[t]);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    uint32_t w[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      w[t][0] = b.w[t].x; w[t][1] = b.w[t].y; w[t][2] = b.w[t].z; w[t][3] = b.w[t].w;
      if constexpr (PER < 4) transpose(w[t]);
    }
    f32x4_t sum[NT][MT], xs[MT];
#pragma unroll
    for (int d = 0; d < 4; ++d) {
      if (d % PER == 0) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          xs[m] = none;
#pragma unroll
          for (int t = 0; t < NT; ++t) sum[t][m] = none;
        }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const bf16x8_t xo = *reinterpret_cast<const bf16x8_t*>(
            stage + (16 * m + xrow) * kXPitch + (PER < 4 ? 16 * d + 4 * g : 16 * g + 4 * d));
        xs[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, xo, xs[m], 0, 0, 0);
#pragma unroll
        for (int t = 0; t < NT; ++t)
          sum[t][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(w[t][d]), xo, sum[t][m], 0, 0, 0);
      }
      if (d % PER == PER - 1) {
        const int i = d / PER;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float s[4] = {bf16_to_f32(b.s[t][i].x & 0xFFFFu), bf16_to_f32(b.s[t][i].x >> 16),
                              bf16_to_f32(b.s[t][i].y & 0xFFFFu), bf16_to_f32(b.s[t][i].y >> 16)};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float z = 16.0f + static_cast<float>((b.z[t][i] >> (8 * e)) & 0xFFu);
#pragma unroll
            for (int m = 0; m < MT; ++m)
              acc[t][m][e] = __builtin_fmaf(s[e], __builtin_fmaf(-z, xs[m][e], sum[t][m][e]), acc[t][m][e]);
          }
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  };

  const int nchunks = (p.K + kChunkK - 1) / kChunkK;
  Chunk buf[D];
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (wv + d * kWaves < nchunks) load(wv + d * kWaves, buf[d]);
  for (int c0 = wv; c0 < nchunks; c0 += D * kWaves) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int c = c0 + d * kWaves;
      if (c < nchunks) compute(buf[d]);
      if (c + D * kWaves < nchunks) load(c + D * kWaves, buf[d]);
    }
  }

  // the sums of all waves, tile by tile
  __syncthreads();
  f32x4_t* const sums = reinterpret_cast<f32x4_t*>(lds);
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m) sums[(wv * NT * MT + t * MT + m) * kWave + lane] = acc[t][m];
  __syncthreads();
  for (int it = wv; it < NT * MT; it += kWaves) {
    f32x4_t s = sums[it * kWave + lane];
#pragma unroll
    for (int v = 1; v < kWaves; ++v) {
      const f32x4_t a = sums[(v * NT * MT + it) * kWave + lane];
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] += a[i];
    }
    // accumulator rows are weight rows: four consecutive columns of out
    const int m = 16 * (it % MT) + m16, n = n0 + 16 * (it / MT) + 4 * g;
    if (m >= M) continue;
    uint16_t* o = p.out + static_cast<int64_t>(m0 + m) * p.out_stride + n;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < p.N) o[e] = f32_to_bf16(p.bias ? s[e] + bf16_to_f32(p.bias[n + e]) : s[e]);
  }
}

template <int XL, int NT, int D>
void launch(const W4Params& p, hipStream_t s) {
  const dim3 grid((p.N + 16 * NT - 1) / (16 * NT), (p.M + 63) / 64);
  if (p.group % 128 == 0)
    linear_w4_kernel<XL, NT, 4, D><<<grid, kWave * kWaves, 0, s>>>(p);
  else if (p.group % 64 == 0)
    linear_w4_kernel<XL, NT, 2, D><<<grid, kWave * kWaves, 0, s>>>(p);
  else
    linear_w4_kernel<XL, NT, 1, D><<<grid, kWave * kWaves, 0, s>>>(p);
}

}  // namespace
}  // namespace nva

using namespace nva;

extern "C" int nva_linear_w4(const void* x, int64_t x_row_stride, const void* qweight,
                             const void* scales, const void* zeros, const void* bias, void* out,
                             int64_t out_row_stride, int32_t rows, int32_t n, int32_t k,
                             int32_t group, void* stream) {
  if (rows < 0 || n <= 0 || k <= 0 || group <= 0 || k % group) return NVA_ERR_ARG;
  if (rows == 0) return NVA_OK;
  if (!x || !qweight || !scales || !out || (rows > 1 && (x_row_stride < k || out_row_stride < n)))
    return NVA_ERR_ARG;
  // 64 rows a grid row, of which there are at most 65535
  if (group % 32 || x_row_stride % 8 || !aligned16(x) || !aligned16(qweight) || rows > 64 * 65535 ||
      reinterpret_cast<uintptr_t>(scales) % 8 || reinterpret_cast<uintptr_t>(zeros) % 4)
    return NVA_ERR_UNSUPPORTED;
  const W4Params p{static_cast<const uint16_t*>(x), x_row_stride, static_cast<const uint8_t*>(qweight),
                   static_cast<const uint16_t*>(scales), static_cast<const uint8_t*>(zeros),
                   static_cast<const uint16_t*>(bias), static_cast<uint16_t*>(out), out_row_stride,
                   rows, n, k, group};
  auto* s = static_cast<hipStream_t>(stream);
  if (rows <= 4)
    launch<1, 1, 3>(p, s);
  else if (rows <= 16)
    launch<4, 1, 3>(p, s);
  else if (rows <= 32)
    launch<8, 1, 2>(p, s);
  else
    launch<16, 1, 1>(p, s);
  return launch_status();
}

// Projections of few rows over 4-bit weights:
//   out[m, n] = sum_k x[m, k] (code[n, k] - zero[k / G, n]) scale[k / G, n] + bias[n]
// with x in bf16, codes 0..15 two to a byte, group scales in bf16.
//
// A group's sum is formed from exact operands and scaled afterwards, so no
// weight is ever rounded: a code c becomes the bf16 value 2^-12 (16 + c) by placing
// its four bits in the mantissa of 2^-8 (one shift, one and-or for two codes), the
// MFMA sums the products with x in fp32, and with the group's sum of 2^-8 x
//   2^-12 sum (c - z) x = sum 2^-12 (16 + c) x - (1 + z / 16) sum 2^-8 x.
// Scales, the sums of x and the sum over groups are fp32, brought back by 2^12 at the
// end, and the output is rounded once.  The power of two is what keeps the up to 128
// products of a sum finite for every finite x (128 * 31 < 2^12); sums below 2^-126
// lose bits, which takes x or outputs below 2^-114.
//
// What bounds it (times of the kernel alone, from a trace): for wide outputs the
// codes' stream from HBM, a quarter of the bf16 weights' (1 x 151936 x 4096: 65 us,
// 4.9 TB/s; a 1 GiB copy reaches 5.07).  Below that the launch and the start (1 x
// 4096 x 4096: 5.6 us, an empty kernel 2.2; a workgroup has its x staged 2.1 us after
// its first instruction and ends at 4.1).  From some dozen rows on a step's work,
// products, codes to operands, scales and x through LDS, each about a quarter of its
// time (64 x 24576 x 4096, 37 us: under counters matrix and vector units are busy 21%
// and 20% of the cycles, waves wait half of theirs).  Prompts take the slab of 64 rows
// again and again: 4096 x 24576 x 4096 1.46 ms, 564 TFLOP/s.
//
// Codes come to the waves in steps: 256 codes of each of 16 rows, 128 bytes of a
// row.  A lane's 16 bytes are 32 codes of one row (lane l: row l % 16, codes
// 32 (l / 16) .. of a 128-wide chunk), four MFMAs deep.  Where groups are shorter
// than 128 the four lanes of a row exchange dwords (four swaps), so that an MFMA
// sums over 32 neighbouring codes.  The accumulator's lanes hold one weight row
// each, so a group costs a lane one scale and one zero: the four lanes of a row
// load those of four groups and broadcast them by swaps.  WK of a workgroup's eight
// waves take a tile's steps in turn and meet in LDS.
//
// Up to 16 rows a workgroup stages its range of K of all x rows in LDS once, as
// MFMA operands, and then only streams codes: no barrier, no x traffic in the loop
// (a group's sum of x is a product with ones beside the others).  More rows would
// leave room for short ranges only, whose staging and joining took most of the time
// (61 x 6144 x 4096 21.5 us, 64 x 24576 x 4096 45); there x passes through LDS in
// chunks of 128 (17.1 and 37 us).  For up to 16 rows the chunks are the slower form
// where N is wide (16 x 24576 x 4096 18.8 us against 17.9, timed side by side).
//
// Ranges of K shared out over workgroups leave fp32 parts that a second kernel
// sums in order.
#include "common.h"

namespace nva {
namespace {

constexpr int kWaves = 8;
constexpr int kThreads = kWave * kWaves;
constexpr int kChunkK = 128;
constexpr int kStepK = 2 * kChunkK;    // a step: 128 bytes of a row's codes
constexpr int kXPitch = 68;            // dwords per staged x row: 16-byte reads of 16 rows cover all banks
constexpr int kMaxLds = 160 * 1024;

struct W4Params {
  const uint16_t* x;
  int64_t x_stride;
  const uint8_t* w;
  const uint16_t* scales;
  const uint8_t* zeros;
  const uint16_t* bias;
  uint16_t* out;
  int64_t out_stride;
  float* partial;                      // [range][M][N], or null
  int32_t M, N, K;
  // groups of K, 32-wide parts of a group, and ceil(2^32 / per_group): the part's
  // group is a product's high half while parts * per_group < 2^32
  uint32_t groups, per_group, group_magic;
};

constexpr float kCodeUnit = 4096.0f;   // what a code's steps are divided by

// Two codes of a dword, nibbles S / 4 and S / 4 + 4, as the bf16 values 2^-12 (16 + c):
// 2^-8 is 0x3B80 and a code's lowest bit is bit 3 of the mantissa.
// The two constants come in registers (one and-or; as literals they take two
// instructions).
struct CodeBits {
  uint32_t mask, base;
  __device__ __forceinline__ CodeBits() : mask(0x00780078u), base(0x3B803B80u) {
    asm volatile("" : "+s"(mask));
    asm volatile("" : "+v"(base));
  }
  template <int S>
  __device__ __forceinline__ uint32_t pair(uint32_t w) const {
    const uint32_t at = S < 4 ? w << 3 : w >> (S - 3);
    return (at & mask) | base;
  }
  // Eight codes as an MFMA operand, in the order 0, 4, 1, 5, 2, 6, 3, 7.
  __device__ __forceinline__ bf16x8_t operand(uint32_t w) const {
    return __builtin_bit_cast(bf16x8_t, make_uint4(pair<0>(w), pair<4>(w), pair<8>(w), pair<12>(w)));
  }
};

// Eight neighbouring values of x in that order.
__device__ __forceinline__ uint4 as_operand(uint4 v) {
  return make_uint4(__builtin_amdgcn_perm(v.z, v.x, 0x05040100u), __builtin_amdgcn_perm(v.z, v.x, 0x07060302u),
                    __builtin_amdgcn_perm(v.w, v.y, 0x05040100u), __builtin_amdgcn_perm(v.w, v.y, 0x07060302u));
}

// The swaps exchange the odd quarters (halves) of the first operand with the
// even ones of the second.
__device__ __forceinline__ void swap16(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
  const uint32_t lo = r[0], hi = r[1];
  a = lo;
  b = hi;
}
__device__ __forceinline__ void swap32(uint32_t& a, uint32_t& b) {
  const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  const uint32_t lo = r[0], hi = r[1];
  a = lo;
  b = hi;
}

// Dword d of lane quarter r becomes dword r of quarter d.
__device__ __forceinline__ void transpose(uint32_t (&w)[4]) {
  swap32(w[0], w[2]);
  swap32(w[1], w[3]);
  swap16(w[0], w[1]);
  swap16(w[2], w[3]);
}

// A row's value of each lane quarter, in all four: v[0] in, v[0..3] out.
__device__ __forceinline__ void broadcast(uint32_t (&v)[4]) {
  uint32_t hi = v[0];
  swap32(v[0], hi);
  v[1] = v[0];
  v[2] = v[3] = hi;
  swap16(v[0], v[1]);
  swap16(v[2], v[3]);
}

// What a wave streams: the steps of NT times 16 weight rows from row n0, groups of
// PER products (32 codes each; 4 also where a group is several).  Rows past the end
// repeat the last one; what they give is not stored.  Loads go through descriptors
// that end with their array (the whole offset in the lane's, which alone is
// checked): past the end of K the codes are any (the next row's, or zeros past the
// last), and past the last group scales are zero.
template <int PER, int NT>
struct CodeStream {
  static constexpr int kGroups = 8 / PER;              // of a step
  static constexpr int kLoads = (kGroups + 3) / 4;     // of a lane's scales per step
  struct Step {
    uint4 w[NT][2];
    uint32_t s[NT][kLoads], z[NT][kLoads];
  };
  __amdgpu_buffer_rsrc_t wr, sr, zr;
  int row[NT], woff[NT], n, g;
  uint32_t magic;
  bool straight, zeros;                                // a group is what an accumulator sums

  __device__ __forceinline__ CodeStream(const W4Params& p, int n0, int lane) {
    const int top = n0 < p.N ? n0 : p.N - 1;
    const int64_t base = static_cast<int64_t>(top) * (p.K / 2);
    const int64_t rest = static_cast<int64_t>(p.N) * (p.K / 2) - base;
    wr = make_rsrc(p.w + base, rest < 0x7FFFFFFF ? static_cast<int>(rest) : 0x7FFFFFFF);
    const int scales = static_cast<int>(p.groups * p.N);
    sr = make_rsrc(p.scales, 2 * scales);
    zr = make_rsrc(p.zeros, scales);
    n = p.N;
    g = lane >> 4;
#pragma unroll
    for (int q = 0; q < NT; ++q) {
      row[q] = n0 + 16 * q + (lane & 15) < n ? n0 + 16 * q + (lane & 15) : n - 1;
      woff[q] = (row[q] - top) * (p.K / 2) + 16 * g;
    }
    magic = p.group_magic;
    straight = p.per_group == PER;
    zeros = p.zeros != nullptr;
  }

  __device__ __forceinline__ void load(int c, Step& b) const {
#pragma unroll
    for (int q = 0; q < NT; ++q)
#pragma unroll
      for (int t = 0; t < 2; ++t)
        b.w[q][t] = __builtin_bit_cast(
            uint4, __builtin_amdgcn_raw_buffer_load_b128(wr, woff[q] + 128 * c + 64 * t, 0, 0));
    // quarter g holds group 4 i + g of the step (two groups: g % 2)
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int j = kGroups < 4 ? g % kGroups : 4 * i + g;
      int at = j * n + kGroups * c * n;
      if (!straight) at = static_cast<int>(__umulhi(8 * c + PER * j, magic)) * n;
#pragma unroll
      for (int q = 0; q < NT; ++q) {
        b.s[q][i] = __builtin_amdgcn_raw_buffer_load_b16(sr, 2 * (at + row[q]), 0, 0);
        b.z[q][i] = zeros ? __builtin_amdgcn_raw_buffer_load_b8(zr, at + row[q], 0, 0) : 8;
      }
    }
  }
};

// Adds up the WK waves of a tile in wave order, through LDS that holds nothing any
// wave still reads, and stores the rows m0 .. m0 + M: a lane has column n0 + 16 q +
// l % 16 of four rows.  The tiles of 16 x 16 are dealt to the waves that share them.
template <int NT, int MT, int WK>
__device__ __forceinline__ void store_tiles(const W4Params& p, const f32x4_t (&acc)[NT][MT], uint32_t* lds, int wv,
                                            int lane, int n0, int split, int m0, int M) {
  f32x4_t* const sums = reinterpret_cast<f32x4_t*>(lds);
  if constexpr (WK > 1) {
#pragma unroll
    for (int q = 0; q < NT; ++q)
#pragma unroll
      for (int m = 0; m < MT; ++m) sums[((wv * NT + q) * MT + m) * kWave + lane] = acc[q][m];
    __syncthreads();
  }
#pragma unroll
  for (int qm = 0; qm < NT * MT; ++qm) {
    const int q = qm / MT, m = qm % MT;
    f32x4_t sum = acc[q][m];
    if constexpr (WK > 1) {
      if (qm % WK != wv % WK) continue;
      const f32x4_t* at = sums + ((wv / WK * WK) * NT * MT + qm) * kWave + lane;
      sum = at[0];
#pragma unroll
      for (int v = 1; v < WK; ++v) {
        const f32x4_t a = at[v * NT * MT * kWave];
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += a[e];
      }
    }
    const int n = n0 + 16 * q + (lane & 15);
    if (n >= p.N) continue;
    const float bias = !p.partial && p.bias ? bf16_to_f32(p.bias[n]) : 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = 16 * m + 4 * (lane >> 4) + e;
      if (r >= M) continue;
      if (p.partial)
        p.partial[(static_cast<int64_t>(split) * p.M + m0 + r) * p.N + n] = sum[e] * kCodeUnit;
      else
        p.out[static_cast<int64_t>(m0 + r) * p.out_stride + n] =
            f32_to_bf16(__builtin_fmaf(sum[e], kCodeUnit, bias));
    }
  }
}

// Up to 16 rows of x, RT of them staged; WK waves share a tile of 16 weight rows.
template <int RT, int PER, int WK>
__global__ void __launch_bounds__(kThreads, 4) linear_w4_kernel(W4Params p) {
  using Stream = CodeStream<PER, 1>;
  constexpr int D = 3;                                 // steps in flight
  constexpr int kGroups = Stream::kGroups, kLoads = Stream::kLoads;
  extern __shared__ __attribute__((aligned(16))) uint32_t xs[];
  const int lane = threadIdx.x & (kWave - 1);
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int m16 = lane & 15, g = lane >> 4;
  const int n0 = 16 * (blockIdx.x * (kWaves / WK) + wv / WK);
  const int nsteps = (p.K + kStepK - 1) / kStepK;
  const int first = static_cast<int>(static_cast<int64_t>(nsteps) * blockIdx.y / gridDim.y);
  const int end = static_cast<int>(static_cast<int64_t>(nsteps) * (blockIdx.y + 1) / gridDim.y);
  const int mine = first + wv % WK;
  const Stream codes(p, n0, lane);

  // ---- x of this range, once: piece i is 16 bytes, sixteen lanes a chunk's row,
  // zeros past the end of K.  The first batch is asked for before the codes: loads
  // return in order, and x comes from L2 in half the time that the codes take from
  // HBM.
  constexpr int kBatch = 8;
  const int pieces = (end - first) * 2 * RT * 16;
  uint4 xv[kBatch];
  auto load_x = [&](int i0) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int i = i0 + u * kThreads;
      const int xr = (i / 16) % RT, k = first * kStepK + i / (16 * RT) * kChunkK + 8 * m16;
      xv[u] = make_uint4(0, 0, 0, 0);
      if (i < pieces && xr < p.M && k < p.K)
        xv[u] = *reinterpret_cast<const uint4*>(p.x + static_cast<int64_t>(xr) * p.x_stride + k);
    }
  };
  auto stage_x = [&](int i0) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int i = i0 + u * kThreads;
      const int xr = (i / 16) % RT, chunk = i / (16 * RT);
      if (i < pieces)
        *reinterpret_cast<uint4*>(xs + (chunk * RT + xr) * kXPitch + 4 * m16) = as_operand(xv[u]);
    }
  };
  load_x(threadIdx.x);
  __builtin_amdgcn_sched_barrier(0);
  typename Stream::Step buf[D];
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (mine + d * WK < end) codes.load(mine + d * WK, buf[d]);
  __builtin_amdgcn_sched_barrier(0);
  stage_x(threadIdx.x);
  for (int i0 = threadIdx.x + kBatch * kThreads; i0 < pieces; i0 += kBatch * kThreads) {
    load_x(i0);
    stage_x(i0);
  }
  __syncthreads();

  const int xrow = RT < 16 ? m16 & (RT - 1) : m16;     // an operand row that is not staged repeats one that is
  const bf16x8_t ones =                                // of 2^-8, as the codes'
      __builtin_bit_cast(bf16x8_t, make_uint4(0x3B803B80u, 0x3B803B80u, 0x3B803B80u, 0x3B803B80u));
  const CodeBits bits;
  const f32x4_t none = f32x4_t{0.f, 0.f, 0.f, 0.f};
  f32x4_t acc[1][1] = {{none}};
  auto compute = [&](int c, const typename Stream::Step& b) {
    const uint32_t* step = xs + (c - first) * 2 * RT * kXPitch;
    uint32_t sz[4 * kLoads];                           // scale (low half) and zero of each group
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      uint32_t v[4] = {b.s[0][i] | (b.z[0][i] << 16), 0, 0, 0};
      if constexpr (kGroups >= 4) {
        broadcast(v);
      } else {
        v[1] = v[0];
        swap16(v[0], v[1]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) sz[4 * i + j] = v[j];
    }
    // the step's two chunks side by side: their chains of products are independent
    uint32_t w[2][4];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint4 v = b.w[0][t];
      w[t][0] = v.x; w[t][1] = v.y; w[t][2] = v.z; w[t][3] = v.w;
      if constexpr (PER < 4) transpose(w[t]);
    }
    f32x4_t sum[2], xsum[2];                           // of a group: codes by x, and x
#pragma unroll
    for (int d = 0; d < 4; ++d) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const bf16x8_t xo = *reinterpret_cast<const bf16x8_t*>(
            step + (t * RT + xrow) * kXPitch + (PER < 4 ? 16 * d + 4 * g : 16 * g + 4 * d));
        xsum[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xo, ones, d % PER == 0 ? none : xsum[t], 0, 0, 0);
        sum[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xo, bits.operand(w[t][d]),
                                                         d % PER == 0 ? none : sum[t], 0, 0, 0);
      }
      if (d % PER == PER - 1) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int i = t * (4 / PER) + d / PER;
          const float s = __uint_as_float(sz[i] << 16), z = __builtin_fmaf(static_cast<float>(sz[i] >> 16), 0.0625f, 1.0f);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[0][0][e] = __builtin_fmaf(s, __builtin_fmaf(-z, xsum[t][e], sum[t][e]), acc[0][0][e]);
          // the sums so far are wanted here: put off to the end of the step, the
          // operands of all its groups stay in registers and spill
          asm("" : "+v"(acc[0][0]));
        }
      }
    }
  };
  for (int c0 = mine; c0 < end; c0 += D * WK) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int c = c0 + d * WK;
      if (c < end) compute(c, buf[d]);
      if (c + D * WK < end) codes.load(c + D * WK, buf[d]);
    }
  }
  if constexpr (WK > 1) __syncthreads();
  store_tiles<1, 1, WK>(p, acc, xs, wv, lane, n0, blockIdx.y, 0, p.M);
}

// A wave's LDS accesses happen in order; this keeps the compiler to it where lanes
// read what others of their wave have written.
__device__ __forceinline__ void in_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// More rows, in slabs of 64 (MT tiles of 16 staged).  A wave holds two tiles of 16
// weight rows; the 8 / WK waves of the same step share its x, a chunk at a time in
// LDS (with one wave a step its own), the next one or two chunks in registers.
// The zeros' part of a sum, -scale (1 + zero / 16) sum 2^-8 x, is a product of its own
// over four groups (fp32 operands; a scale times up to 31 sixteenths is exact).
template <int MT, int PER, int WK>
__global__ void __launch_bounds__(kThreads, 2) linear_w4_slab_kernel(W4Params p) {
  constexpr int NT = 2, D = 2;
  using Stream = CodeStream<PER, NT>;
  constexpr int kGroups = Stream::kGroups, kLoads = Stream::kLoads;
  constexpr int kShare = kWaves / WK, kBufs = kShare > 1 ? 2 : 1;
  constexpr int kPieces = 4 * MT / kShare;             // of a chunk, four rows each, that a wave stages
  constexpr int kAhead = kPieces >= 8 ? 1 : 2;         // chunks on their way in registers
  extern __shared__ __attribute__((aligned(16))) uint32_t xs[];
  const int lane = threadIdx.x & (kWave - 1);
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int m16 = lane & 15, g = lane >> 4;
  const int n0 = 16 * NT * (blockIdx.x * kShare + wv / WK);
  const int m0 = blockIdx.z * 64;
  const int M = p.M - m0 < 64 ? p.M - m0 : 64;
  const int nsteps = (p.K + kStepK - 1) / kStepK;
  const int first = static_cast<int>(static_cast<int64_t>(nsteps) * blockIdx.y / gridDim.y);
  const int end = static_cast<int>(static_cast<int64_t>(nsteps) * (blockIdx.y + 1) / gridDim.y);
  const int mine = first + wv % WK;
  const int kend = end * kStepK < p.K ? end * kStepK : p.K;
  const Stream codes(p, n0, lane);

  // x past its last row or the end of the range is zero: outside the descriptor,
  // which ends with row M - 1 (at most 2^31 bytes: the caller has checked)
  const uint32_t stride = static_cast<uint32_t>(p.x_stride);
  const __amdgpu_buffer_rsrc_t xr = make_rsrc(p.x + static_cast<int64_t>(m0) * p.x_stride,
                                              static_cast<int>(2 * (stride * (M - 1) + p.K)));
  uint32_t* const stage = xs + (wv % WK) * kBufs * (16 * MT * kXPitch);
  const int member = wv / WK * kPieces;                // this wave's first piece
  const uint32_t xlane = stride * 2 * (4 * member + g) + 16 * m16;
  uint4 xv[kAhead][kPieces];
  auto load_x = [&](int c, int t) {
    const int k = c * kStepK + kChunkK * t;
    const uint32_t at = k + 8 * m16 < kend ? xlane + 2 * k : 0x80000000u;
#pragma unroll
    for (int u = 0; u < kPieces; ++u)
      xv[t % kAhead][u] = __builtin_bit_cast(
          uint4, __builtin_amdgcn_raw_buffer_load_b128(xr, static_cast<int>(at + stride * (8 * u)), 0, 0));
  };
  auto stage_x = [&](int t) {
#pragma unroll
    for (int u = 0; u < kPieces; ++u)
      *reinterpret_cast<uint4*>(stage + (t % kBufs * 16 * MT + 4 * (member + u) + g) * kXPitch + 4 * m16) =
          as_operand(xv[t % kAhead][u]);
  };
#pragma unroll
  for (int t = 0; t < kAhead; ++t) load_x(mine, t);
  __builtin_amdgcn_sched_barrier(0);
  typename Stream::Step buf[D];
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (mine + d * WK < end) codes.load(mine + d * WK, buf[d]);
  __builtin_amdgcn_sched_barrier(0);

  // operand rows 4 d .. 4 d + 3 of ones (2^-8, as the codes'): the product with x leaves the sum of x's
  // row l % 16 in lane quarter d, as the fp32 product takes it
  bf16x8_t ones[4];
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const uint32_t v = m16 / 4 == d ? 0x3B803B80u : 0u;
    ones[d] = __builtin_bit_cast(bf16x8_t, make_uint4(v, v, v, v));
  }
  const CodeBits bits;
  const f32x4_t none = f32x4_t{0.f, 0.f, 0.f, 0.f};
  f32x4_t acc[NT][MT];
#pragma unroll
  for (int q = 0; q < NT; ++q)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[q][m] = none;
  auto compute = [&](int c, const typename Stream::Step& b) {
    uint32_t scale[NT][4];                             // of group d and, in the high half, 4 + d
    float below[NT][kLoads];                           // -scale (1 + zero / 16) of the lane quarter's groups
#pragma unroll
    for (int q = 0; q < NT; ++q) {
      scale[q][0] = kLoads == 2 ? b.s[q][0] | b.s[q][kLoads - 1] << 16 : b.s[q][0];
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        below[q][i] = -__uint_as_float(b.s[q][i] << 16) * __builtin_fmaf(static_cast<float>(b.z[q][i]), 0.0625f, 1.0f);
      if constexpr (kGroups >= 4) {
        broadcast(scale[q]);
      } else {
        scale[q][1] = scale[q][0];
        swap16(scale[q][0], scale[q][1]);
      }
    }
    f32x4_t sum[NT][MT], xsum[MT];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      uint32_t w[NT][4];
#pragma unroll
      for (int q = 0; q < NT; ++q) {
        const uint4 v = b.w[q][t];
        w[q][0] = v.x; w[q][1] = v.y; w[q][2] = v.z; w[q][3] = v.w;
        if constexpr (PER < 4) transpose(w[q]);
      }
      if constexpr (kShare == 1) in_order();
      stage_x(t);
      if constexpr (kShare == 1) in_order();
      if (kAhead == 2)
        load_x(c + WK, t);
      else if (t == 0)
        load_x(c, 1);
      else
        load_x(c + WK, 0);
      // two buffers: whoever writes one again has passed the barrier behind the
      // other's use of it
      if constexpr (kShare > 1) __syncthreads();
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        constexpr int kJoined = 4 * PER < 8 ? 4 * PER : 8;   // products whose sums of x are joined: four groups, or the step
        const int j = 4 * t + d, group = j / PER;
        bf16x8_t wo[NT];
#pragma unroll
        for (int q = 0; q < NT; ++q) wo[q] = bits.operand(w[q][d]);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          const bf16x8_t xo = *reinterpret_cast<const bf16x8_t*>(
              stage + (t % kBufs * 16 * MT + 16 * m + m16) * kXPitch + (PER < 4 ? 16 * d + 4 * g : 16 * g + 4 * d));
          xsum[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones[group % 4], xo,
                                                            j % kJoined == 0 ? none : xsum[m], 0, 0, 0);
#pragma unroll
          for (int q = 0; q < NT; ++q)
            sum[q][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xo, wo[q], j % PER == 0 ? none : sum[q][m], 0, 0, 0);
        }
        if (j % PER == PER - 1) {
#pragma unroll
          for (int q = 0; q < NT; ++q) {
            const uint32_t two = scale[q][group % 4];
            const float s = __uint_as_float(group / 4 ? two & 0xFFFF0000u : two << 16);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[q][m][e] = __builtin_fmaf(s, sum[q][m][e], acc[q][m][e]);
              asm("" : "+v"(acc[q][m]));               // not put off, as above
            }
          }
        }
        if (j % kJoined == kJoined - 1) {
#pragma unroll
          for (int q = 0; q < NT; ++q)
#pragma unroll
            for (int m = 0; m < MT; ++m)
              acc[q][m] = __builtin_amdgcn_mfma_f32_16x16x4f32(xsum[m][0], below[q][group / 4], acc[q][m], 0, 0, 0);
        }
      }
    }
  };
  // waves that share a barrier go as many rounds as the first of them
  for (int c0 = mine; c0 - mine + first < end; c0 += D * WK) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int c = c0 + d * WK;
      if (c < end) {
        compute(c, buf[d]);
      } else if (kShare > 1 && c - mine + first < end) {
        __syncthreads();
        __syncthreads();
      }
      if (c + D * WK < end) codes.load(c + D * WK, buf[d]);
    }
  }
  if constexpr (WK > 1) __syncthreads();
  store_tiles<NT, MT, WK>(p, acc, xs, wv, lane, n0, blockIdx.y, m0, M);
}

// The sum of the K ranges' parts, in order.  Bound by latency: a thread loads
// kSumBatch parts at a time and owns one column, which takes the most workgroups
// (twelve parts of 1 x 5120: with the main kernel 20.7 us; four columns a thread in
// batches of eight 21.9).
constexpr int kSumBatch = 16;
__global__ void __launch_bounds__(256) linear_w4_sum_kernel(W4Params p, int32_t splits) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t size = static_cast<int64_t>(p.M) * p.N;
  if (i >= size) return;
  const int64_t m = i / p.N;
  const int n = static_cast<int>(i - m * p.N);
  const float* part = p.partial + i;
  float s = 0.0f;
  for (int j0 = 0; j0 < splits; j0 += kSumBatch) {
    float a[kSumBatch];
#pragma unroll
    for (int u = 0; u < kSumBatch; ++u) a[u] = j0 + u < splits ? part[(j0 + u) * size] : 0.0f;
#pragma unroll
    for (int u = 0; u < kSumBatch; ++u) s += a[u];
  }
  p.out[m * p.out_stride + n] = f32_to_bf16(p.bias ? s + bf16_to_f32(p.bias[n]) : s);
}

// Rows of x a workgroup stages, ranges of K, and waves that share a tile of weight
// rows.
struct W4Plan {
  int32_t rows, splits, shared;
};

// LDS of a workgroup: its range's x (up to 16 rows; more: a chunk or two for every
// step under way), and room for the waves' tiles behind.
int lds_bytes(const W4Plan& plan, int32_t k) {
  const int steps = ((k + kStepK - 1) / kStepK + plan.splits - 1) / plan.splits;
  const bool slab = plan.rows > 16;
  const int staged = !slab ? 2 * steps : plan.shared == kWaves ? kWaves : 2 * plan.shared;
  const int x = staged * plan.rows * kXPitch * 4;
  const int tiles = plan.shared > 1 ? kThreads * (slab ? 2 * (plan.rows / 16) : 1) * 16 : 0;
  return x > tiles ? x : tiles;
}

// More than the default bound of dynamic LDS, once per device and kernel.
template <void (*Kernel)(W4Params)>
bool allow_lds() {
  static bool set[64] = {};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return false;
  const bool known = dev >= 0 && dev < 64;
  if (known && set[dev]) return true;
  if (hipFuncSetAttribute(reinterpret_cast<const void*>(Kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                          kMaxLds) != hipSuccess)
    return false;
  if (known) set[dev] = true;
  return true;
}

template <int RT, int PER, int WK>
int launch(const W4Params& p, const W4Plan& plan, hipStream_t s) {
  const int bytes = lds_bytes(plan, p.K);
  if constexpr (RT > 16) {
    constexpr auto kern = linear_w4_slab_kernel<RT / 16, PER, WK>;
    if (bytes > 64 * 1024 && !allow_lds<kern>()) return NVA_ERR_LAUNCH;
    const int tile = 32 * (kWaves / WK);
    kern<<<dim3((p.N + tile - 1) / tile, plan.splits, (p.M + 63) / 64), kThreads, bytes, s>>>(p);
  } else {
    constexpr auto kern = linear_w4_kernel<RT, PER, WK>;
    if (bytes > 64 * 1024 && !allow_lds<kern>()) return NVA_ERR_LAUNCH;
    const int tile = 16 * (kWaves / WK);
    kern<<<dim3((p.N + tile - 1) / tile, plan.splits), kThreads, bytes, s>>>(p);
  }
  return launch_status();
}

template <int RT, int WK>
int launch_rows(const W4Params& p, const W4Plan& plan, hipStream_t s) {
  if (p.per_group % 4 == 0) return launch<RT, 4, WK>(p, plan, s);
  if (p.per_group % 2 == 0) return launch<RT, 2, WK>(p, plan, s);
  return launch<RT, 1, WK>(p, plan, s);
}

template <int RT>
int launch_shared(const W4Params& p, const W4Plan& plan, hipStream_t s) {
  switch (plan.shared) {
    case 1: return launch_rows<RT, 1>(p, plan, s);
    case 2: return launch_rows<RT, 2>(p, plan, s);
    case 4: return launch_rows<RT, 4>(p, plan, s);
    default: return launch_rows<RT, 8>(p, plan, s);
  }
}

// Compute units of the current device (cached per device; 256 when the query fails).
int32_t device_cus() {
  static int32_t cus[64] = {0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) dev = 0;
  if (cus[dev] == 0) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
    cus[dev] = n;
  }
  return cus[dev];
}

// The ranges of K and the waves that share a tile, by the least modelled time
// (us): rounds of workgroups over the device, each a wave's steps and what comes
// before and behind them, and with several ranges the summing kernel.
//   * Up to 16 rows two workgroups share a CU and its time; a range's x is staged
//     first, and LDS bounds the range.  Fitted to 18 shapes (1-64 rows, N 800-151936,
//     K 640-25600, groups of 32-128) timed over all choices (the times here are that
//     sweep's), where its choice is 3% from the best: 1 x 4096 x 4096 one range with
//     eight waves a tile 5.5 us, with four 7.2, eight ranges with one 7.4; 16 x 5120 x
//     25600 twelve ranges 23.9, six 24.3, sixteen 25.3.
//   * More rows take a CU a workgroup; a step costs more where fewer waves share its
//     x.  Fitted to 17 shapes (17-256 rows, N 1024-151936, K 512-25600), 1% from the
//     best: 61 x 6144 x 4096 one range with eight waves a tile 17.7 us, two with four
//     19.8, eight with one 24.9; 64 x 24576 x 4096 one with two 37, with eight 43.
W4Plan make_plan(int32_t rows, int32_t n, int32_t k, int32_t group) {
  W4Plan best = {}, plan = {};
  plan.rows = rows <= 4 ? 4 : rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
  const bool slab = plan.rows > 16;
  const int rt = plan.rows;
  const int parts = group % 128 == 0 ? 1 : group % 64 == 0 ? 2 : 4;   // groups of a chunk, if they end in it
  const int32_t steps = (k + kStepK - 1) / kStepK, most = slab ? steps : kMaxLds / (2 * rt * kXPitch * 4);
  const int32_t fewest = (steps + most - 1) / most;
  const int64_t cus = device_cus(), slabs = (rows + 63) / 64;
  float least = 0.0f;
  for (int shared = 1; shared <= kWaves; shared *= 2) {
    const int tile = (slab ? 32 : 16) * (kWaves / shared);
    const int64_t tiles = (n + tile - 1) / tile * slabs;
    for (int fill = 0; fill <= 4; fill = fill ? 2 * fill : 1) {
      // as few ranges as LDS allows, or as many as make one, two, four rounds
      const int32_t splits = fill ? static_cast<int32_t>(fill * cus / tiles) : fewest;
      if (splits < fewest || (fill && splits == fewest) || splits > steps) continue;
      plan.splits = splits;
      plan.shared = shared;
      const int32_t of_range = (steps + splits - 1) / splits;
      const int32_t of_wave = (of_range + shared - 1) / shared;
      const int64_t per_cu = (tiles * splits + cus - 1) / cus;
      float t;
      if (slab) {
        const float step = (rt == 64 ? 2.15f : 1.53f) * (1.0f + 0.065f * (parts - 1)) * (1.0f + 0.04f * shared);
        t = (step * of_wave + 1.3f) * per_cu;
        if (splits > 1) t += 2.8f + 1.9e-6f * splits * rows * n;
      } else {
        const int64_t fit = 2 * lds_bytes(plan, k) <= kMaxLds && per_cu > 1 ? 2 : 1;
        t = 0.53f * (1.0f + 0.23f * (parts - 1)) * of_wave * fit + 0.014f * of_range * rt;
        if (shared > 1) t += 0.012f * shared;
        t *= static_cast<float>((per_cu + fit - 1) / fit);
        if (splits > 1) t += 2.3f + 2.8e-6f * splits * rows * n;
      }
      if (best.splits == 0 || t < least) {
        least = t;
        best = plan;
      }
    }
  }
  return best;
}

size_t plan_bytes(const W4Plan& w, int32_t rows, int32_t n) {
  return w.splits > 1 ? static_cast<size_t>(w.splits) * rows * n * sizeof(float) : 0;
}

}  // namespace
}  // namespace nva

using namespace nva;

extern "C" size_t nva_linear_w4_workspace_size(int32_t rows, int32_t n, int32_t k, int32_t group) {
  if (rows <= 0 || n <= 0 || k <= 0 || group <= 0 || k % group || group % 32) return 0;
  return plan_bytes(make_plan(rows, n, k, group), rows, n);
}

extern "C" int nva_linear_w4(const void* x, int64_t x_row_stride, const void* qweight,
                             const void* scales, const void* zeros, const void* bias, void* out,
                             int64_t out_row_stride, int32_t rows, int32_t n, int32_t k,
                             int32_t group, void* workspace, size_t workspace_bytes, void* stream) {
  if (rows < 0 || n <= 0 || k <= 0 || group <= 0 || k % group) return NVA_ERR_ARG;
  if (rows == 0) return NVA_OK;
  if (!x || !qweight || !scales || !out || (rows > 1 && (x_row_stride < k || out_row_stride < n)))
    return NVA_ERR_ARG;
  // 64 rows a grid row, of which there are at most 65535; scales are counted in
  // 32 bits, groups by a 32-bit reciprocal
  if (group % 32 || x_row_stride % 8 || !aligned16(x) || !aligned16(qweight) || rows > 64 * 65535 ||
      k > (1 << 20) || static_cast<int64_t>(k / group) * n >= 1 << 29)
    return NVA_ERR_UNSUPPORTED;
  // a slab of x is addressed in 31 bits, and what lies 2^31 bytes behind its rows
  // must not come round to it
  if (rows > 16 && x_row_stride >= 1 << 24) return NVA_ERR_UNSUPPORTED;
  const W4Plan plan = make_plan(rows, n, k, group);
  const size_t need = plan_bytes(plan, rows, n);
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace))) return NVA_ERR_WORKSPACE;
  const W4Params p{static_cast<const uint16_t*>(x), x_row_stride, static_cast<const uint8_t*>(qweight),
                   static_cast<const uint16_t*>(scales), static_cast<const uint8_t*>(zeros),
                   static_cast<const uint16_t*>(bias), static_cast<uint16_t*>(out), out_row_stride,
                   need ? static_cast<float*>(workspace) : nullptr, rows, n, k,
                   static_cast<uint32_t>(k / group), static_cast<uint32_t>(group / 32),
                   static_cast<uint32_t>(((int64_t{1} << 32) + group / 32 - 1) / (group / 32))};
  auto* s = static_cast<hipStream_t>(stream);
  int status;
  switch (plan.rows) {
    case 4: status = launch_shared<4>(p, plan, s); break;
    case 8: status = launch_shared<8>(p, plan, s); break;
    case 16: status = launch_shared<16>(p, plan, s); break;
    case 32: status = launch_shared<32>(p, plan, s); break;
    default: status = launch_shared<64>(p, plan, s); break;
  }
  if (status != NVA_OK || plan.splits == 1) return status;
  const int64_t blocks = (static_cast<int64_t>(rows) * n + 255) / 256;
  linear_w4_sum_kernel<<<static_cast<uint32_t>(blocks), 256, 0, s>>>(p, plan.splits);
  return launch_status();
}

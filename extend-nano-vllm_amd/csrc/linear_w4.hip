// Projections of few rows over 4-bit weights:
//   out[m, n] = sum_k x[m, k] (code[n, k] - zero[k / G, n]) scale[k / G, n] + bias[n]
// with x in bf16, codes 0..15 two to a byte, group scales in bf16.
//
// A group's sum is formed from exact operands and scaled afterwards, so no
// weight is ever rounded: a code c becomes the bf16 value 16 + c by placing its
// four bits in the mantissa of 16 (one shift, one and-or for two codes), the
// MFMA sums (16 + c) x in fp32, and with the group's sum of x
//   sum (c - z) x = sum (16 + c) x - (16 + z) sum x.
// Scales, the sums of x and the sum over groups are fp32, the output is rounded
// once.
//
// What bounds it: for wide outputs the codes' stream from HBM, a quarter of the
// bf16 weights' (1 x 151936 x 4096: 58-64 us, 5.0-5.4 TB/s; a 1 GiB copy reaches
// 5.07).  Below that the start (at 1 x 4096 x 4096, 5.1 us, x is staged 2.1 us
// into the kernel's 4.1), and from some dozen rows the staging of x and the joining
// of parts as well (61 x 6144 x 4096 in groups of 32, 21.5 us: staging 5, codes 6,
// joining waves 4, joining ranges 5).
//
// A workgroup of eight waves stages its range of K of all x rows in LDS once, as
// MFMA operands, and then only streams codes: no barrier, no x traffic in the
// loop (a group's sum of x is a product with ones beside the others).  WK waves
// take the steps (256 codes of a row, 128 bytes) of 16 weight rows in turn, 8 / WK
// times 16 rows a workgroup.  A lane's 16 bytes are 32 codes of one row (lane l:
// row l % 16, codes 32 (l / 16) .. of a 128-wide chunk), four MFMAs deep.  Where
// groups are shorter than 128 the four lanes of a row exchange dwords (four swaps),
// so that an MFMA sums over 32 neighbouring codes.  The accumulator's lanes hold
// one weight row each, so a group costs a lane one scale and one zero: the four
// lanes of a row load those of four groups and broadcast them by swaps.
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

// Two codes of a dword, nibbles S / 4 and S / 4 + 4, as the bf16 values 16 + c:
// 16 is 0x4180 and a code's lowest bit is bit 3 of the mantissa.
// The two constants come in registers (one and-or; as literals they take two
// instructions).
struct CodeBits {
  uint32_t mask, sixteen;
  __device__ __forceinline__ CodeBits() : mask(0x00780078u), sixteen(0x41804180u) {
    asm volatile("" : "+s"(mask));
    asm volatile("" : "+v"(sixteen));
  }
  template <int S>
  __device__ __forceinline__ uint32_t pair(uint32_t w) const {
    const uint32_t at = S < 4 ? w << 3 : w >> (S - 3);
    return (at & mask) | sixteen;
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

// RT: rows of x staged; PER: MFMAs (32 codes each) per group, 1, 2 or 4 (whole
// chunks); NT: tiles of 16 weight rows of a wave; D: steps in flight; WK: waves
// that share a tile.
template <int RT, int PER, int NT, int D, int WK>
__global__ void __launch_bounds__(kThreads, RT <= 16 ? 4 : 2) linear_w4_kernel(W4Params p) {
  constexpr int MT = RT <= 16 ? 1 : RT / 16;           // tiles of 16 rows of x
  constexpr int kGroups = 8 / PER;                     // of a step
  constexpr int kLoads = (kGroups + 3) / 4;            // of a lane's scales per step
  extern __shared__ __attribute__((aligned(16))) uint32_t xs[];
  const int lane = threadIdx.x & (kWave - 1);
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int m16 = lane & 15, g = lane >> 4;
  const int waves = blockDim.x / kWave;
  const int n0 = blockIdx.x * (16 * NT * (waves / WK)) + 16 * NT * (wv / WK);
  const int split = blockIdx.y;
  const int m0 = blockIdx.z * 64;
  const int M = p.M - m0 < 64 ? p.M - m0 : 64;
  const int nsteps = (p.K + kStepK - 1) / kStepK;
  const int first = static_cast<int>(static_cast<int64_t>(nsteps) * split / gridDim.y);
  const int end = static_cast<int>(static_cast<int64_t>(nsteps) * (split + 1) / gridDim.y);
  const int mine = first + wv % WK;

  // rows past the end repeat the last one; what they give is not stored.  Loads
  // go through descriptors that end with their array (the whole offset in the
  // lane's, which alone is checked): past the end of K x is zero and the codes
  // are any (the next row's, or zeros past the last), and past the last group
  // scales are zero.
  const int top = n0 < p.N ? n0 : p.N - 1;
  const int64_t base = static_cast<int64_t>(top) * (p.K / 2);
  const int64_t rest = static_cast<int64_t>(p.N) * (p.K / 2) - base;
  const __amdgpu_buffer_rsrc_t wr = make_rsrc(p.w + base, rest < 0x7FFFFFFF ? static_cast<int>(rest) : 0x7FFFFFFF);
  int row[NT], woff[NT];
#pragma unroll
  for (int q = 0; q < NT; ++q) {
    row[q] = n0 + 16 * q + m16 < p.N ? n0 + 16 * q + m16 : p.N - 1;
    woff[q] = (row[q] - top) * (p.K / 2) + 16 * g;
  }
  const int codes_of_zeros = static_cast<int>(p.groups * p.N);
  const __amdgpu_buffer_rsrc_t sr = make_rsrc(p.scales, 2 * codes_of_zeros);
  const __amdgpu_buffer_rsrc_t zr = make_rsrc(p.zeros, codes_of_zeros);
  const bool straight = p.per_group == PER;            // a group is what an accumulator sums
  struct Codes {
    uint4 w[NT][2];
    uint32_t s[NT][kLoads], z[NT][kLoads];
  };
  auto load = [&](int c, Codes& b) {
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
      int at = j * p.N + kGroups * c * p.N;
      if (!straight) at = static_cast<int>(__umulhi(8 * c + PER * j, p.group_magic)) * p.N;
#pragma unroll
      for (int q = 0; q < NT; ++q) {
        b.s[q][i] = __builtin_amdgcn_raw_buffer_load_b16(sr, 2 * (at + row[q]), 0, 0);
        b.z[q][i] = p.zeros ? __builtin_amdgcn_raw_buffer_load_b8(zr, at + row[q], 0, 0) : 8;
      }
    }
  };

  // ---- x of this range, once: piece i is 16 bytes, sixteen lanes a chunk's row.
  // The first batch is asked for before the codes: loads return in order, and x
  // comes from L2 in half the time that the codes take from HBM.
  constexpr int kBatch = RT <= 16 ? 8 : 16;
  const int pieces = (end - first) * 2 * RT * 16;
  uint4 xv[kBatch];
  auto load_x = [&](int i0) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int i = i0 + u * blockDim.x;
      const int xr = (i / 16) % RT, k = first * kStepK + i / (16 * RT) * kChunkK + 8 * m16;
      xv[u] = make_uint4(0, 0, 0, 0);
      if (i < pieces && xr < M && k < p.K)
        xv[u] = *reinterpret_cast<const uint4*>(p.x + static_cast<int64_t>(m0 + xr) * p.x_stride + k);
    }
  };
  auto stage_x = [&](int i0) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int i = i0 + u * blockDim.x;
      const int xr = (i / 16) % RT, chunk = i / (16 * RT);
      if (i < pieces)
        *reinterpret_cast<uint4*>(xs + (chunk * RT + xr) * kXPitch + 4 * m16) = as_operand(xv[u]);
    }
  };
  load_x(threadIdx.x);
  __builtin_amdgcn_sched_barrier(0);
  Codes buf[D];
#pragma unroll
  for (int d = 0; d < D; ++d)
    if (mine + d * WK < end) load(mine + d * WK, buf[d]);
  __builtin_amdgcn_sched_barrier(0);
  stage_x(threadIdx.x);
  for (int i0 = threadIdx.x + kBatch * blockDim.x; i0 < pieces; i0 += kBatch * blockDim.x) {
    load_x(i0);
    stage_x(i0);
  }
  __syncthreads();

  const int xrow = RT < 16 ? m16 & (RT - 1) : m16;     // an operand row that is not staged repeats one that is
  const bf16x8_t ones = __builtin_bit_cast(bf16x8_t, make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u));
  const CodeBits bits;
  f32x4_t acc[NT][MT];
#pragma unroll
  for (int q = 0; q < NT; ++q)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[q][m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const f32x4_t none = f32x4_t{0.f, 0.f, 0.f, 0.f};
  // TU chunks of a step side by side, where registers allow: their chains of
  // products are independent
  constexpr int TU = MT == 1 ? 2 : 1;
  auto compute = [&](int c, const Codes& b) {
    const uint32_t* step = xs + (c - first) * 2 * RT * kXPitch;
    uint32_t sz[NT][4 * kLoads];                       // scale (low half) and zero of each group
#pragma unroll
    for (int q = 0; q < NT; ++q)
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        uint32_t v[4] = {b.s[q][i] | (b.z[q][i] << 16), 0, 0, 0};
        if constexpr (kGroups >= 4) {
          broadcast(v);
        } else {
          v[1] = v[0];
          swap16(v[0], v[1]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) sz[q][4 * i + j] = v[j];
      }
#pragma unroll
    for (int t0 = 0; t0 < 2; t0 += TU) {
      uint32_t w[NT][TU][4];
#pragma unroll
      for (int q = 0; q < NT; ++q)
#pragma unroll
        for (int t = 0; t < TU; ++t) {
          const uint4 v = b.w[q][t0 + t];
          w[q][t][0] = v.x; w[q][t][1] = v.y; w[q][t][2] = v.z; w[q][t][3] = v.w;
          if constexpr (PER < 4) transpose(w[q][t]);
        }
      f32x4_t sum[TU][NT][MT], xsum[TU][MT];           // of a group: codes by x, and x
#pragma unroll
      for (int d = 0; d < 4; ++d) {
#pragma unroll
        for (int t = 0; t < TU; ++t) {
          bf16x8_t wo[NT];
#pragma unroll
          for (int q = 0; q < NT; ++q) wo[q] = bits.operand(w[q][t][d]);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            const bf16x8_t xo = *reinterpret_cast<const bf16x8_t*>(
                step + ((t0 + t) * RT + 16 * m + xrow) * kXPitch + (PER < 4 ? 16 * d + 4 * g : 16 * g + 4 * d));
            xsum[t][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xo, ones, d % PER == 0 ? none : xsum[t][m], 0, 0, 0);
#pragma unroll
            for (int q = 0; q < NT; ++q)
              sum[t][q][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                  xo, wo[q], d % PER == 0 ? none : sum[t][q][m], 0, 0, 0);
          }
        }
        if (d % PER == PER - 1) {
#pragma unroll
          for (int t = 0; t < TU; ++t) {
            const int i = (t0 + t) * (4 / PER) + d / PER;
#pragma unroll
            for (int q = 0; q < NT; ++q) {
              const float s = __uint_as_float(sz[q][i] << 16), z = 16.0f + static_cast<float>(sz[q][i] >> 16);
#pragma unroll
              for (int m = 0; m < MT; ++m) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  acc[q][m][e] =
                      __builtin_fmaf(s, __builtin_fmaf(-z, xsum[t][m][e], sum[t][q][m][e]), acc[q][m][e]);
                // the sums so far are wanted here: put off to the end of the
                // step, the operands of all its groups stay in registers and spill
                asm("" : "+v"(acc[q][m]));
              }
            }
          }
        }
      }
    }
  };
  for (int c0 = mine; c0 < end; c0 += D * WK) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int c = c0 + d * WK;
      if (c < end) compute(c, buf[d]);
      if (c + D * WK < end) load(c + D * WK, buf[d]);
    }
  }

  if constexpr (WK > 1) {
    // the waves of a tile meet in LDS and are summed in wave order (deterministic)
    __syncthreads();
    f32x4_t* const sums = reinterpret_cast<f32x4_t*>(xs);
#pragma unroll
    for (int q = 0; q < NT; ++q)
#pragma unroll
      for (int m = 0; m < MT; ++m) sums[((wv * NT + q) * MT + m) * kWave + lane] = acc[q][m];
    __syncthreads();
  }

  // a lane's column n of four rows; the tiles of 16 x 16 are dealt to the waves
  // that share them
#pragma unroll
  for (int qm = 0; qm < NT * MT; ++qm) {
    const int q = qm / MT, m = qm % MT;
    f32x4_t sum = acc[q][m];
    if constexpr (WK > 1) {
      if (qm % WK != wv % WK) continue;
      const f32x4_t* at = reinterpret_cast<const f32x4_t*>(xs) + ((wv / WK * WK) * NT * MT + qm) * kWave + lane;
      sum = at[0];
#pragma unroll
      for (int v = 1; v < WK; ++v) {
        const f32x4_t a = at[v * NT * MT * kWave];
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += a[e];
      }
    }
    const int n = n0 + 16 * q + m16;
    if (n >= p.N) continue;
    const float bias = !p.partial && p.bias ? bf16_to_f32(p.bias[n]) : 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = 16 * m + 4 * g + e;
      if (r >= M) continue;
      if (p.partial)
        p.partial[(static_cast<int64_t>(split) * p.M + m0 + r) * p.N + n] = sum[e];
      else
        p.out[static_cast<int64_t>(m0 + r) * p.out_stride + n] = f32_to_bf16(sum[e] + bias);
    }
  }
}

// The sum of the K ranges' parts, in order: a thread owns V columns of a row and
// loads kSumBatch parts at a time (one latency, not one a part).
constexpr int kSumBatch = 8;
template <int V>
__global__ void __launch_bounds__(256) linear_w4_sum_kernel(W4Params p, int32_t splits) {
  typedef __attribute__((ext_vector_type(V))) float vec;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t size = static_cast<int64_t>(p.M) * p.N / V;
  if (i >= size) return;
  const int64_t m = i / (p.N / V);
  const int n = static_cast<int>(i - m * (p.N / V)) * V;
  const vec* part = reinterpret_cast<const vec*>(p.partial) + i;
  vec s = 0.0f;
  for (int j0 = 0; j0 < splits; j0 += kSumBatch) {
    vec a[kSumBatch];
#pragma unroll
    for (int u = 0; u < kSumBatch; ++u) a[u] = j0 + u < splits ? part[(j0 + u) * size] : vec(0.0f);
#pragma unroll
    for (int u = 0; u < kSumBatch; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) s[e] += a[u][e];
  }
  uint16_t* o = p.out + m * p.out_stride + n;
#pragma unroll
  for (int e = 0; e < V; ++e) o[e] = f32_to_bf16(p.bias ? s[e] + bf16_to_f32(p.bias[n + e]) : s[e]);
}

// Rows of x a workgroup stages, ranges of K, waves of a workgroup, and how many of
// them share a tile of weight rows.
struct W4Plan {
  int32_t rows, splits, waves, shared;
};

// Tiles of 16 weight rows a wave holds with RT rows of x.
constexpr int tiles_of(int rt) { return rt <= 16 ? 1 : 2; }

template <int RT, int PER, int NT, int D, int WK>
int launch(const W4Params& p, const W4Plan& plan, hipStream_t s) {
  const int steps = ((p.K + kStepK - 1) / kStepK + plan.splits - 1) / plan.splits;
  int bytes = steps * 2 * RT * kXPitch * 4;
  const int sums = plan.waves * kWave * NT * (RT <= 16 ? 1 : RT / 16) * 16;
  if (WK > 1 && bytes < sums) bytes = sums;
  const int tile = 16 * NT * (plan.waves / WK);
  const dim3 grid((p.N + tile - 1) / tile, plan.splits, (p.M + 63) / 64);
  auto* kern = linear_w4_kernel<RT, PER, NT, D, WK>;
  if (bytes > 64 * 1024) {
    // more than the default bound of dynamic LDS, once per device
    static bool set[64] = {};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return NVA_ERR_LAUNCH;
    if (dev < 0 || dev >= 64 || !set[dev]) {
      if (hipFuncSetAttribute(reinterpret_cast<const void*>(kern),
                              hipFuncAttributeMaxDynamicSharedMemorySize, kMaxLds) != hipSuccess)
        return NVA_ERR_LAUNCH;
      if (dev >= 0 && dev < 64) set[dev] = true;
    }
  }
  kern<<<grid, plan.waves * kWave, bytes, s>>>(p);
  return launch_status();
}

template <int RT, int WK>
int launch_rows(const W4Params& p, const W4Plan& plan, hipStream_t s) {
  constexpr int NT = tiles_of(RT), D = 3;
  if (p.per_group % 4 == 0) return launch<RT, 4, NT, D, WK>(p, plan, s);
  if (p.per_group % 2 == 0) return launch<RT, 2, NT, D, WK>(p, plan, s);
  return launch<RT, 1, NT, D, WK>(p, plan, s);
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
// (us): rounds of workgroups over the device, each a wave's steps (longer with
// more waves a SIMD, shorter groups and more rows) and the staging of its x, and
// with several ranges the summing kernel.  The constants are a fit to 18 shapes
// (1-64 rows, N 800-151936, K 640-25600, groups of 32-128) timed over all
// choices: its choice is 3% from the best on the geometric mean.
W4Plan make_plan(int32_t rows, int32_t n, int32_t k, int32_t group) {
  W4Plan best = {};
  best.rows = rows <= 4 ? 4 : rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
  best.waves = kWaves;
  const int rt = best.rows, nt = tiles_of(rt), mt = rt <= 16 ? 1 : rt / 16;
  const int per = group % 128 == 0 ? 4 : group % 64 == 0 ? 2 : 1;
  const int step_bytes = 2 * rt * kXPitch * 4;
  const int32_t steps = (k + kStepK - 1) / kStepK, most = kMaxLds / step_bytes;
  const int64_t cus = device_cus(), slabs = (rows + 63) / 64;
  const float unit = 0.53f * nt * (1.0f + 0.22f * (mt - 1)) * (1.0f + 0.23f * (4 / per - 1));
  const int slots = rt <= 16 ? 2 : 1;                  // workgroups of a CU by registers
  float least = 0.0f;
  for (int shared = 1; shared <= kWaves; shared *= 2) {
    const int tile = 16 * nt * (kWaves / shared);
    const int64_t tiles = (n + tile - 1) / tile * slabs;
    const int32_t fewest = (steps + most - 1) / most;
    for (int fill = 0; fill <= 4; fill = fill ? 2 * fill : 1) {
      // as few ranges as LDS allows, or as many as make one, two, four rounds
      int32_t splits = fill ? static_cast<int32_t>(fill * cus / tiles) : fewest;
      if (splits < fewest || (fill && splits == fewest) || splits > steps) continue;
      const int32_t of_range = (steps + splits - 1) / splits;
      int bytes = of_range * step_bytes;
      const int parked = kThreads * nt * mt * 16;
      if (shared > 1 && bytes < parked) bytes = parked;
      const int fit = kMaxLds / bytes < slots ? kMaxLds / bytes : slots;
      const int64_t per_cu = (tiles * splits + cus - 1) / cus;
      const int64_t at_once = per_cu < fit ? per_cu : fit;
      float t = unit * ((of_range + shared - 1) / shared) * (at_once > 1 ? at_once : 1.0f) +
                0.014f * of_range * rt + (shared > 1 ? 0.012f * nt * mt * shared : 0.0f);
      t *= static_cast<float>((per_cu + at_once - 1) / at_once);
      if (splits > 1) t += 2.3f + 2.8e-6f * splits * rows * n;
      if (best.splits == 0 || t < least) {
        least = t;
        best.splits = splits;
        best.shared = shared;
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
  const int64_t threads = static_cast<int64_t>(rows) * n / (n % 4 == 0 ? 4 : 1);
  auto* sum = n % 4 == 0 ? linear_w4_sum_kernel<4> : linear_w4_sum_kernel<1>;
  sum<<<static_cast<uint32_t>((threads + 255) / 256), 256, 0, s>>>(p, plan.splits);
  return launch_status();
}

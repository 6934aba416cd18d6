// Paged attention of a batch whose sequences share a long prefix (gfx950).
//
// The softmax over a row's keys is joined from parts: for a part P of the keys
//   m_P = max s, l_P = sum exp(s - m_P), o_P = sum exp(s - m_P) v / l_P,
// the whole is  sum_P w_P o_P / sum_P w_P  with w_P = l_P exp(m_P - max m).
// The prefix's keys are the same for every sequence, so their parts are
// computed for tiles of query rows of all sequences together: each K and V byte
// of the prefix is read once per tile instead of once per sequence, and the
// products run on full matrix tiles.  Each sequence's own keys are parts of
// tiles of its own rows.  Parts, sums and states are fp32; a probability is
// rounded to bf16 for the product with V (relative 2^-8, as in the paged
// attention), the output once more.
//
// Two launches: the parts, then the join.  The parts of the prefix and of the own
// keys are units of one grid, two workgroups a CU, prefix units first: they
// are the longer ones, bound by the matrix cores, and the own keys' units, bound
// by the memory, run in the places beside and behind them.
//
//   * Prefix units and sequences of more than 32 rows: wide_unit below.
//   * Own keys of up to 32 rows: attend_segment, four waves sharing a part, each
//     streaming chunks of its own without a barrier.
#include <math.h>

#include "attention_tiles.h"

namespace nva {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWave * kWaves;
constexpr int kTileRows = 32 * kWaves;               // query rows of a wide tile
constexpr int32_t kMaxKeys = 1 << 30;                // ends of parts are rounded up in 32 bits
constexpr int kParkPitch = kD + 4;                   // floats per row of a part on its way out
constexpr int kSegDwords = 2 * kWaves * kVStage;     // attend_segment's stages, then its query operands
constexpr int kWideDwords = 2 * kWideBuf;
static_assert(kTileRows * kParkPitch <= kWideDwords, "a tile's part fits the buffers");

struct PrefixParams {
  AttnParams a;        // max_splits: the parts of a row; row_nsplit: its own keys' (-1: none, zeros)
  int32_t prefix;                                    // shared keys (a multiple of 32)
  int32_t prefix_split, prefix_parts;                // keys of a prefix part, parts
  int32_t own_split, own_parts;                      // the same of a sequence's own keys (parts: bound)
  int32_t prefix_tiles, own_tiles;                   // tiles of a.qtile query positions
  int32_t prefix_units, own_units;                   // per kv head
};

// Ones over the bf16 values of a dword that are finite.
__device__ __forceinline__ uint32_t finite_mask(uint32_t w) {
  return ((w & 0x7F80u) == 0x7F80u ? 0u : 0xFFFFu) | ((w & 0x7F800000u) == 0x7F800000u ? 0u : 0xFFFF0000u);
}

// A tile of query rows of one kv head (positions tok0 .. tok0 + jn - 1 of the
// batch, all heads of the group) against the keys [kv_begin, kv_end) of a block
// table, 64 keys a step; the part goes to the workspace.
//   * A wave holds 32 rows on the 32x32x16 MFMA; HALVES (tiles of up to 64 rows):
//     wave w has row group w % 2 and takes keys 32 (w / 2) .. + 31 of each
//     step, and the two halves' states meet in LDS.
//   * S^T = K . Q^T with keys as M: lane 32 h + c holds, for query column c, the
//     keys 8 b + 4 h + i (b, i = 0..3) of a 32-key tile in accumulator element
//     4 b + i.  Elements 8 t .. 8 t + 7 are the k-slots of lane half h in the B
//     operand of slice t of O^T += V^T . P^T, if slot j of half h stands for key
//     16 t + 8 (j / 4) + 4 h + j % 4, so P goes from accumulator to operand by
//     rounding alone, and V^T is read from LDS in that order by two transpose
//     loads (wide_v_operand).
//   * K/V go through registers two steps ahead and one of two LDS buffers one
//     step ahead, one barrier a step.  FP8 pages become bf16 on the way.
//   * The part leaves through LDS as whole rows of 512 bytes.
//   * A hidden key's weight of zero does not keep an infinity or NaN in its V out of
//     a product (0 * inf is NaN).  Tiles with keys that some row does not see are
//     staged with zeros in place of such elements; where there was one (a flag, which
//     the caller has cleared), they are added at the end, read again, to the rows
//     that see them.  Rows that see no key of the range have no part in the join.
//     Where every row sees every key that costs a comparison a tile: 96.2 for 95.7 us
//     for 100 x 5 rows over 16384 FP8 keys.
// last_key[j]: the last key that position tok0 + j sees (less than 0: none);
// last_key[kTileRows]: the flag.
template <bool HALVES, bool FP8>
__device__ __forceinline__ void wide_unit(const AttnParams& p, uint32_t* lds, int32_t* last_key,
                                          const int kvh, const int tok0, const int jn,
                                          const int kv_begin, const int kv_end, const int part,
                                          const int32_t* table) {
  constexpr int kEsz = FP8 ? 1 : 2;
  constexpr int kRowGran = kD * kEsz / 16;               // 16-byte granules per K or V row
  constexpr int kPer = kWideKeys * kRowGran / kThreads;  // a thread's granules of K (and of V)
  constexpr int kTiles = HALVES ? 1 : 2;                 // 32-key tiles of a wave's step
  static_assert(kPer >= 1, "every thread loads at least one granule");
  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int wv = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int rw = HALVES ? wv & 1 : wv;                   // row group
  const int half = HALVES ? wv >> 1 : 0;
  const int h = lane >> 5;
  const int col = lane & 31;
  const int rows = jn * p.group;
  float kscale = 1.0f, vscale = 1.0f;
  if (FP8) {
    kscale = p.k_scale ? *p.k_scale : 1.0f;
    vscale = p.v_scale ? *p.v_scale : 1.0f;
  }
  const float sl2 = p.scale_log2 * kscale;

  // ---- this lane's query column (a padding column repeats row 0 and is not
  // stored), its last visible key, and the wave's least and greatest
  const int n = 32 * rw + col;
  const int nn = n < rows ? n : 0;
  const int jc = nn / p.group, hc = kvh * p.group + nn % p.group;
  bf16x8_t qv[8];
  {
    const uint16_t* qp = p.q + static_cast<int64_t>(tok0 + jc) * p.q_row_stride +
                         static_cast<int64_t>(hc) * p.q_head_stride + 8 * h;
#pragma unroll
    for (int s = 0; s < 8; ++s) qv[s] = *reinterpret_cast<const bf16x8_t*>(qp + 16 * s);
  }
  const int lim = last_key[jc];
  int least = lim, most = lim;
#pragma unroll
  for (int m = 16; m >= 1; m >>= 1) {
    const int a = __shfl_xor(least, m, kWave), b = __shfl_xor(most, m, kWave);
    least = a < least ? a : least;
    most = b > most ? b : most;
  }
  const int wave_full = __builtin_amdgcn_readfirstlane(least) + 1;   // keys below it are seen by every row
  // of this lane's positions that see a key of the range, the one that sees the fewest
  int seen = 0x7FFFFFFF;
  for (int j = lane; j < jn; j += kWave) {
    const int k = last_key[j];
    if (k >= kv_begin && k < seen) seen = k;
  }
  // keys from it on by none
  const int wave_end = 32 * rw < rows ? __builtin_amdgcn_readfirstlane(most) + 1 : 0;

  // ---- loads: thread granule i is row (tid + i kThreads) / kRowGran of the
  // step; its 32-key half is the same for the whole wave.  The halves have
  // descriptors of their own (blocks hold a multiple of 32 tokens), which end at
  // the last key of the range.
  const uint32_t tokb = static_cast<uint32_t>(p.tok_stride * kEsz);
  constexpr int kStepRows = kThreads / kRowGran;         // rows between a thread's granules
  uint32_t goff[kPer], kdst[kPer], vdst[kPer];
  bool upper[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int gi = tid + i * kThreads;
    const int row = gi / kRowGran, c = gi % kRowGran;
    upper[i] = kStepRows <= 32 ? i * kStepRows >= 32 : __builtin_amdgcn_readfirstlane(row) >= 32;
    goff[i] = static_cast<uint32_t>(row & 31) * tokb + c * 16;
    kdst[i] = row * kWideKPitch + c * (FP8 ? 8 : 4);
    vdst[i] = kWideKeys * kWideKPitch + row * kWideVPitch + c * (FP8 ? 8 : 4);
  }
  // lane i of lane_blk holds the id of the i-th block from the one ld_blk counts from
  auto block_ids = [&](int key) {
    const int c = key / p.block_size + lane;
    return c < p.bt_cols ? table[c] : -1;
  };
  int lane_blk = block_ids(kv_begin);
  int ld_key = kv_begin;                                 // first key of the next half to load,
  int ld_blk = 0;                                        // its block
  int ld_tok = kv_begin % p.block_size;                  // and its token there
  auto next_half = [&](__amdgpu_buffer_rsrc_t& kr, __amdgpu_buffer_rsrc_t& vr) -> bool {
    const bool live = ld_key < kv_end;
    if (live && ld_blk >= kWave) {
      ld_blk = 0;
      lane_blk = block_ids(ld_key);
    }
    const int raw = __builtin_amdgcn_readlane(lane_blk, ld_blk & (kWave - 1));
    const bool valid = live && raw >= 0 && raw < p.num_blocks;
    const int seen = kv_end - ld_key < 32 ? kv_end - ld_key : 32;
    const int nrec = valid ? seen * static_cast<int>(tokb) : 0;
    const int64_t tile = (static_cast<int64_t>(valid ? raw : 0) * p.blk_stride +
                          static_cast<int64_t>(kvh) * p.head_stride +
                          static_cast<int64_t>(valid ? ld_tok : 0) * p.tok_stride) * kEsz;
    kr = make_rsrc(p.k_cache + tile, nrec);
    vr = make_rsrc(p.v_cache + tile, nrec);
    ld_key += 32;
    ld_tok += 32;
    if (ld_tok == p.block_size) {
      ld_tok = 0;
      ++ld_blk;
    }
    return valid;
  };
  struct Tile {
    uint4 k[kPer], v[kPer];
    int valid;                                           // bit 0, 1: the halves
  };
  auto load_tile = [&](Tile& t) {
    __amdgpu_buffer_rsrc_t k0, v0, k1, v1;
    const bool a = next_half(k0, v0);
    const bool b = next_half(k1, v1);
    t.valid = (a ? 1 : 0) | (b ? 2 : 0);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      t.k[i] = __builtin_bit_cast(
          uint4, __builtin_amdgcn_raw_buffer_load_b128(upper[i] ? k1 : k0, goff[i], 0, 0));
      t.v[i] = __builtin_bit_cast(
          uint4, __builtin_amdgcn_raw_buffer_load_b128(upper[i] ? v1 : v0, goff[i], 0, 0));
    }
  };
  auto stage = [&](const Tile& t, int b, int key0) {
    uint32_t* base = lds + b * kWideBuf;
    constexpr int kVecs = FP8 ? 2 : 1;                     // staged 16-byte pieces of a granule
    uint4 v[kPer * kVecs];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if constexpr (FP8) {
        *reinterpret_cast<bf16x8_t*>(base + kdst[i]) = fp8x8_to_bf16(make_uint2(t.k[i].x, t.k[i].y));
        *reinterpret_cast<bf16x8_t*>(base + kdst[i] + 4) = fp8x8_to_bf16(make_uint2(t.k[i].z, t.k[i].w));
        v[2 * i] = __builtin_bit_cast(uint4, fp8x8_to_bf16(make_uint2(t.v[i].x, t.v[i].y)));
        v[2 * i + 1] = __builtin_bit_cast(uint4, fp8x8_to_bf16(make_uint2(t.v[i].z, t.v[i].w)));
      } else {
        *reinterpret_cast<uint4*>(base + kdst[i]) = t.k[i];
        v[i] = t.v[i];
      }
    }
    const int top = key0 + kWideKeys < kv_end ? key0 + kWideKeys - 1 : kv_end - 1;
    if (__any(seen < top)) {
      uint32_t all = 0xFFFFFFFFu;
#pragma unroll
      for (int i = 0; i < kPer * kVecs; ++i) {
        const uint4 m = make_uint4(finite_mask(v[i].x), finite_mask(v[i].y), finite_mask(v[i].z),
                                   finite_mask(v[i].w));
        all &= m.x & m.y & m.z & m.w;
        v[i] = make_uint4(v[i].x & m.x, v[i].y & m.y, v[i].z & m.z, v[i].w & m.w);
      }
      if (all != 0xFFFFFFFFu) last_key[kTileRows] = 1;
    }
#pragma unroll
    for (int i = 0; i < kPer * kVecs; ++i)
      *reinterpret_cast<uint4*>(base + vdst[i / kVecs] + 4 * (i % kVecs)) = v[i];
  };

  float m_run = -INFINITY, l_run = 0.0f;
  f32x16_t acc[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[dt][i] = 0.0f;

  auto compute = [&](int key0, int ok, int b) {
    const int kb = key0 + 32 * half;                     // the wave's first key
    if (HALVES) ok = ok >> half & 1;
    if (kb >= wave_end || ok == 0) return;
    const uint32_t* kst = lds + b * kWideBuf + 32 * half * kWideKPitch;
    const uint32_t* vst = lds + b * kWideBuf + kWideKeys * kWideKPitch + 32 * half * kWideVPitch;
    f32x16_t sacc[kTiles];
#pragma unroll
    for (int kt = 0; kt < kTiles; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) sacc[kt][i] = 0.0f;
#pragma unroll
    for (int s = 0; s < 8; ++s)
#pragma unroll
      for (int kt = 0; kt < kTiles; ++kt) {
        const bf16x8_t ko =
            *reinterpret_cast<const bf16x8_t*>(kst + (32 * kt + col) * kWideKPitch + 8 * s + 4 * h);
        sacc[kt] = mfma32(ko, qv[s], sacc[kt]);
      }
    if (kb + 32 * kTiles > wave_full || ok != (1 << kTiles) - 1) {
#pragma unroll
      for (int kt = 0; kt < kTiles; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = kb + 32 * kt + 8 * (i >> 2) + 4 * h + (i & 3);
          if (key > lim || !((ok >> kt) & 1)) sacc[kt][i] = -INFINITY;
        }
    }
    float cmax = sacc[0][0];
#pragma unroll
    for (int kt = 0; kt < kTiles; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) cmax = fmaxf(cmax, sacc[kt][i]);
    cmax = max_xor32(cmax) * sl2;
    const bool need = cmax > m_run + kRescaleSlack;
    if (__any(need)) {
      const float m_new = need ? cmax : m_run;
      const float alpha = need ? exp2f_fast(m_run - m_new) : 1.0f;
      l_run *= alpha;
      m_run = m_new;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[dt][i] *= alpha;
    }
    const float msub = m_run == -INFINITY ? 0.0f : m_run;
    bf16x8_t pb[2 * kTiles];
    float psum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < 2 * kTiles; ++t) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f32x2_t pv;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          pv[e] = exp2f_fast(__builtin_fmaf(sacc[t >> 1][8 * (t & 1) + 2 * j + e], sl2, -msub));
          psum[e] += pv[e];
        }
        w[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(pv, bf16x2_t));
      }
      pb[t] = __builtin_bit_cast(bf16x8_t, make_uint4(w[0], w[1], w[2], w[3]));
    }
    l_run += psum[0] + psum[1];
#pragma unroll
    for (int t = 0; t < 2 * kTiles; ++t)
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) acc[dt] = mfma32(wide_v_operand(vst, lane, t, dt), pb[t], acc[dt]);
  };

  // step c computes tile c from buffer c & 1, stages tile c + 1 into the other
  // buffer and loads tile c + 2; the barrier publishes the staged tile and
  // frees the computed one
  const int ntiles = (kv_end - kv_begin + kWideKeys - 1) / kWideKeys;
  Tile t;
  load_tile(t);
  stage(t, 0, kv_begin);
  int valid = t.valid;
  load_tile(t);
  __syncthreads();
  for (int c = 0; c < ntiles; ++c) {
    compute(kv_begin + c * kWideKeys, valid, c & 1);
    if (c + 1 < ntiles) {
      stage(t, (c + 1) & 1, kv_begin + (c + 1) * kWideKeys);
      valid = t.valid;
      load_tile(t);
    }
    __syncthreads();
  }

  // ---- the part: elements 4 b + i of tile dt are d = 32 dt + 8 b + 4 h + i.
  // Every buffer is free behind the loop's last barrier.
  float* const park = reinterpret_cast<float*>(lds) + rw * 32 * kParkPitch;
  if constexpr (HALVES) {
    // the second half's waves park their states (behind the two row groups'
    // parts), the first's take them in
    float* const other = reinterpret_cast<float*>(lds) + 2 * 32 * kParkPitch + rw * kWave * 66;
    static_assert(2 * 32 * kParkPitch + 2 * kWave * 66 <= kWideDwords, "parked states fit");
    if (half == 1) {
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int b = 0; b < 4; ++b)
          reinterpret_cast<f32x4_t*>(other)[(4 * dt + b) * kWave + lane] =
              f32x4_t{acc[dt][4 * b], acc[dt][4 * b + 1], acc[dt][4 * b + 2], acc[dt][4 * b + 3]};
      other[64 * kWave + lane] = m_run;
      other[65 * kWave + lane] = l_run;
    }
    __syncthreads();
    if (half == 1) return;
    const float m1 = other[64 * kWave + lane], l1 = other[65 * kWave + lane];
    const float M = fmaxf(m_run, m1);
    const float f0 = m_run == -INFINITY ? 0.0f : exp2f_fast(m_run - M);
    const float f1 = m1 == -INFINITY ? 0.0f : exp2f_fast(m1 - M);
    m_run = M;
    l_run = f0 * l_run + f1 * l1;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const f32x4_t o = reinterpret_cast<const f32x4_t*>(other)[(4 * dt + b) * kWave + lane];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[dt][4 * b + i] = f0 * acc[dt][4 * b + i] + f1 * o[i];
      }
  }
  if (last_key[kTileRows]) {
#pragma unroll 1
    for (int key = kv_begin; key < kv_end; ++key) {
      const int c = key / p.block_size;
      const int raw = c < p.bt_cols ? table[c] : -1;
      if (raw < 0 || raw >= p.num_blocks || key > lim) continue;
      const uint8_t* row = p.v_cache + (static_cast<int64_t>(raw) * p.blk_stride +
                                        static_cast<int64_t>(kvh) * p.head_stride +
                                        static_cast<int64_t>(key % p.block_size) * p.tok_stride) * kEsz;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const uint8_t* at = row + (32 * dt + 8 * b + 4 * h) * kEsz;
          if constexpr (FP8) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(at);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if ((w >> (8 * i) & 0x7Fu) == 0x7Fu) acc[dt][4 * b + i] = __builtin_nanf("");
          } else {
            const uint2 v = *reinterpret_cast<const uint2*>(at);
            const uint32_t x = v.x & ~finite_mask(v.x), y = v.y & ~finite_mask(v.y);
            acc[dt][4 * b] += __uint_as_float(x << 16);
            acc[dt][4 * b + 1] += __uint_as_float(x & 0xFFFF0000u);
            acc[dt][4 * b + 2] += __uint_as_float(y << 16);
            acc[dt][4 * b + 3] += __uint_as_float(y & 0xFFFF0000u);
          }
        }
    }
  }
  const float lsum = sum_xor32(l_run);
  const float inv = lsum > 0.0f ? vscale / lsum : 0.0f;
  // through the wave's own rows of LDS, then out row by row
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int b = 0; b < 4; ++b)
      *reinterpret_cast<float4*>(park + col * kParkPitch + 32 * dt + 8 * b + 4 * h) =
          make_float4(acc[dt][4 * b] * inv, acc[dt][4 * b + 1] * inv, acc[dt][4 * b + 2] * inv,
                      acc[dt][4 * b + 3] * inv);
  lds_wave_sync();
  const auto slot_of = [&](int r) {
    return (static_cast<int64_t>(tok0 + r / p.group) * p.hq + kvh * p.group + r % p.group) * p.max_splits + part;
  };
#pragma unroll 4
  for (int i = 0; i < 16; ++i) {
    const int r = 32 * rw + 2 * i + h;
    const float4 o = *reinterpret_cast<const float4*>(park + (2 * i + h) * kParkPitch + 4 * col);
    if (r < rows) *reinterpret_cast<float4*>(p.ws_o + slot_of(r) * kD + 4 * col) = o;
  }
  if (n < rows && h == 0) p.ws_lse[slot_of(n)] = part_lse(m_run, lsum);
}

// OWN: how the own keys' units run: tiles of 16 (1) or 32 (2) rows on
// attend_segment, of 64 (3) on attend_tile (bf16) or wide_unit, of 128 (4) on
// wide_unit.  FEW: prefix tiles of up to 64 rows.
template <int OWN, bool FEW, bool FP8>
__global__ void __launch_bounds__(kThreads, 2) shared_prefix_kernel(PrefixParams pp) {
  constexpr int kDwords = OWN > 2 ? kWideDwords
                          : kSegDwords + OWN * 4 * kWave * 4 > kWideDwords ? kSegDwords + OWN * 4 * kWave * 4
                                                                           : kWideDwords;
  __shared__ __attribute__((aligned(16))) uint32_t lds[kDwords];
  __shared__ int32_t last_key[kTileRows + 1];            // of each query position of a wide tile, and its flag
  const AttnParams& p = pp.a;
  const int kvh = blockIdx.x % p.hkv;
  const int u = blockIdx.x / p.hkv;
  if (u < pp.prefix_units) {
    const int tile = u % pp.prefix_tiles, split = u / pp.prefix_tiles;
    const int tok0 = tile * p.qtile;
    const int jn = p.num_tokens - tok0 < p.qtile ? p.num_tokens - tok0 : p.qtile;
    const int kv_begin = split * pp.prefix_split;
    const int kv_end = kv_begin + pp.prefix_split < pp.prefix ? kv_begin + pp.prefix_split : pp.prefix;
    // every position's last visible key, from the sequence that holds it
    for (int i = threadIdx.x; i < jn; i += kThreads) last_key[i] = -1;
    if (threadIdx.x == 0) last_key[kTileRows] = 0;
    __syncthreads();
    for (int seq = p.cu_q ? static_cast<int>(threadIdx.x) : tok0 + static_cast<int>(threadIdx.x);
         seq < (p.cu_q ? p.num_seqs : tok0 + jn); seq += kThreads) {
      int q_start, q_len, L;
      seq_geometry(p, seq, q_start, q_len, L);
      const int lo = q_start > tok0 ? q_start : tok0;
      const int hi = q_start + q_len < tok0 + jn ? q_start + q_len : tok0 + jn;
      for (int t = lo; t < hi; ++t) last_key[t - tok0] = L - q_len + (t - q_start);
    }
    __syncthreads();
    wide_unit<FEW, FP8>(p, lds, last_key, kvh, tok0, jn, kv_begin, kv_end, split, p.block_tables);
    return;
  }
  int rest = u - pp.prefix_units;
  const int seq = rest % p.num_seqs;
  rest /= p.num_seqs;
  const int qt = pp.own_tiles - 1 - rest % pp.own_tiles, split = rest / pp.own_tiles;
  const int kv_begin = pp.prefix + split * pp.own_split;
  int lane_blk = 0;
  if constexpr (OWN <= 2 || !FP8) lane_blk = split_block_ids(p, seq, kv_begin);
  int q_start, q_len, L, q_raw;
  seq_geometry_uniform(p, seq, q_start, q_len, L, &q_raw);
  const int j0 = qt * p.qtile;
  const int jn = q_len - j0 < p.qtile ? q_len - j0 : p.qtile;
  const int limit = L - q_len + j0 + jn;                 // keys seen by the tile's last row
  const int kv_end = kv_begin + pp.own_split < limit ? kv_begin + pp.own_split : limit;
  if (kvh == 0 && split == 0) {
    // what the join reads of each row: the parts written for it
    const int parts = limit > pp.prefix ? (limit - pp.prefix + pp.own_split - 1) / pp.own_split : 0;
    for (int j = threadIdx.x; j < jn; j += kThreads) p.row_nsplit[q_start + j0 + j] = parts;
    if (qt == 0)
      for (int j = q_len + static_cast<int>(threadIdx.x); j < q_raw; j += kThreads) p.row_nsplit[q_start + j] = -1;
  }
  if (jn <= 0 || kv_begin >= kv_end) return;
  if constexpr (OWN <= 2) {
    // (a count of parts other than 1, which would mean an output)
    attend_segment<OWN, FP8, false, kWaves>(p, lds, reinterpret_cast<bf16x8_t*>(lds + kSegDwords), kvh, seq,
                                            q_start, q_len, L, kv_begin, kv_end, pp.prefix_parts + split, 2,
                                            lane_blk);
  } else if constexpr (OWN == 3 && !FP8) {
    attend_tile<kWaves, 4>(p, lds, kvh, q_start, q_len, L, 0, jn, limit, kv_begin, kv_end,
                           pp.prefix_parts + split, 2, lane_blk);
  } else {
    for (int j = threadIdx.x; j < jn; j += kThreads) last_key[j] = L - q_len + j0 + j;
    if (threadIdx.x == 0) last_key[kTileRows] = 0;
    __syncthreads();
    wide_unit<OWN == 3, FP8>(p, lds, last_key, kvh, q_start + j0, jn, kv_begin, kv_end,
                             pp.prefix_parts + split, p.block_tables + static_cast<int64_t>(seq) * p.bt_stride);
  }
}

// The join.  A thread owns four head_dim elements of one (token, head).
constexpr int kJoinThreads = 256;
__global__ void __launch_bounds__(kJoinThreads) join_kernel(PrefixParams pp) {
  const AttnParams& p = pp.a;
  const int t = blockIdx.x;
  // rows of no sequence are left alone
  const int lo = p.cu_q ? p.cu_q[0] : 0;
  const int hi = p.cu_q ? p.cu_q[p.num_seqs] : p.num_seqs;
  int own = p.row_nsplit[t];
  if (t < lo || t >= hi) return;
  const int idx = blockIdx.y * kJoinThreads + threadIdx.x;
  if (idx >= p.hq * (kD / 4)) return;
  const int h = idx / (kD / 4), d4 = idx % (kD / 4);
  own = own < pp.own_parts ? own : pp.own_parts;
  const int parts = own < 0 ? 0 : pp.prefix_parts + own;
  const int64_t base = (static_cast<int64_t>(t) * p.hq + h) * p.max_splits;
  const float4 o = join_parts(p, base, parts, d4);
  uint16_t* op = p.out + static_cast<int64_t>(t) * p.out_row_stride +
                 static_cast<int64_t>(h) * p.out_head_stride + 4 * d4;
  *reinterpret_cast<uint2*>(op) = make_uint2(pack_bf16(o.x, o.y), pack_bf16(o.z, o.w));
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

int32_t ceil_div(int64_t a, int64_t b) { return static_cast<int32_t>((a + b - 1) / b); }

// Whether the prefix is one tile of up to 64 rows (the kernel's FEW).
bool few_rows(const AttnParams& p) { return static_cast<int64_t>(p.num_tokens) * p.group <= 64; }

// How the own keys of tiles of so many rows run (the kernel's OWN).
int own_kind(int64_t rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : rows <= 64 ? 3 : 4; }

// Tiles and parts of a call.  Unknown lengths are bounded by max_k; block_size
// 0 (the workspace query does not name one) assumes the smallest, which bounds
// the parts from above.
//
// p parts of the prefix take about A / p + B p us: a unit's steps (1.6 us, 1.0 for
// tiles of up to 64 rows) against the parts written and read again (1032 bytes a
// row and head at 3.5 TB/s) and the units' start (5 us over 512 places), where a
// part costs three times that beside the own keys' units.  Past a unit a CU, as
// many as fill one or two a CU.  Own keys are cut into parts of about 512 keys, 320
// where there are few units; prompts (several tiles a sequence) no further than two
// rounds of units, since every part is a slot of every row: 8 x 2048 rows of 64/8
// heads over 4096 + 4096 keys take 1.1 GB of workspace and 4.53 ms (parts of 512: 4.9 GB,
// 5.88 ms), 1 x 4096 rows over 36864 own keys 0.27 GB and 5.6 ms (9.9 GB, 9.0 ms), 4 x
// 512 rows over 4096 + 512 at 32/8 182 us (179).
//
// Over 16 shapes (batches of 2-160, 1-64 rows, heads 5/1-64/8, prefixes of 512-16384
// keys, bf16 and FP8) timed with all counts of parts the choice is 3% from the best on
// the geometric mean; a part more or less around it costs little: 64 x 8192 shared keys
// at 32/8 heads 4 / 6 / 8 / 12 / 16 parts 64 / 52 / 45 / 46 / 53 us, 128 x 8 rows over
// 4111 at 64/8 heads 1 / 2 / 4 183 / 189 / 194 (that sweep's times).
void make_plan(PrefixParams& pp, int32_t prefix_len, int32_t block_size) {
  AttnParams& p = pp.a;
  pp.prefix = prefix_len < p.max_k ? prefix_len / 32 * 32 : p.max_k / 32 * 32;
  p.qtile = kTileRows / p.group;
  pp.prefix_tiles = ceil_div(p.num_tokens, p.qtile);
  pp.own_tiles = p.max_q > 0 ? ceil_div(p.max_q, p.qtile) : 1;   // one, which marks the rows past max_q
  const int64_t cus = device_cus();
  const float heads = static_cast<float>(p.num_tokens) * p.hq;
  const float units = static_cast<float>(pp.prefix_tiles) * p.hkv;   // of one part
  const float a = (few_rows(p) ? 1.0f : 1.6f) * pp.prefix / kWideKeys;
  const float b = 3.0f * (heads * 1032.0f / 3.5e6f + units * 5.0f / (2 * cus));
  float parts = sqrtf(a / b);
  if (parts * units > cus) {
    float fill = cus;
    while (parts * units > 1.41f * fill) fill *= 2.0f;
    parts = fill / units;
  }
  const int32_t most = pp.prefix / (2 * kWideKeys);
  int32_t count = parts + 0.5f < most ? static_cast<int32_t>(parts + 0.5f) : most;
  count = count < 1 ? 1 : count;
  pp.prefix_split = ceil_div(ceil_div(pp.prefix, count), kWideKeys) * kWideKeys;
  pp.prefix_parts = pp.prefix > 0 ? ceil_div(pp.prefix, pp.prefix_split) : 0;
  // own keys
  const int32_t own = p.max_k - pp.prefix;
  const int32_t length = static_cast<int64_t>(p.num_seqs) * pp.own_tiles * p.hkv < cus / 2 ? 320 : 512;
  int32_t own_count = own / length + (own % length >= length / 2 ? 1 : 0);
  if (pp.own_tiles > 1) {
    const int64_t rounds = 4 * cus / (static_cast<int64_t>(pp.prefix_tiles) * p.hkv);
    if (own_count > rounds) own_count = static_cast<int32_t>(rounds);
  }
  pp.own_split = own > 0 ? ceil_div(ceil_div(own, own_count < 1 ? 1 : own_count), kWideKeys) * kWideKeys : kWideKeys;
  // attend_segment and attend_tile hold a part's block ids one a lane
  const int32_t span = (kWave - 2) * (block_size > 0 ? block_size : kChunk) / kWideKeys * kWideKeys;
  if (own_kind(static_cast<int64_t>(p.max_q) * p.group) < 4 && pp.own_split > span) pp.own_split = span;
  pp.own_parts = own > 0 ? ceil_div(own, pp.own_split) : 1;
  p.max_splits = pp.prefix_parts + pp.own_parts;
  const int64_t prefix_units = static_cast<int64_t>(pp.prefix_parts) * pp.prefix_tiles;
  const int64_t own_units = static_cast<int64_t>(p.num_seqs) * pp.own_tiles * pp.own_parts;
  const bool fits = (prefix_units + own_units) * p.hkv <= 0x7FFFFFFF;
  pp.prefix_units = fits ? static_cast<int32_t>(prefix_units) : -1;
  pp.own_units = fits ? static_cast<int32_t>(own_units) : -1;
}

size_t plan_bytes(const PrefixParams& pp) {
  const size_t slots = static_cast<size_t>(pp.a.num_tokens) * pp.a.hq * pp.a.max_splits;
  return slots * (kD + 1) * sizeof(float) + static_cast<size_t>(pp.a.num_tokens) * sizeof(int32_t);
}

template <int OWN, bool FEW>
void launch(const PrefixParams& pp, bool fp8, int32_t grid, hipStream_t s) {
  if (fp8)
    shared_prefix_kernel<OWN, FEW, true><<<grid, kThreads, 0, s>>>(pp);
  else
    shared_prefix_kernel<OWN, FEW, false><<<grid, kThreads, 0, s>>>(pp);
}
template <int OWN>
void launch(const PrefixParams& pp, bool fp8, int32_t grid, hipStream_t s) {
  if (few_rows(pp.a))
    launch<OWN, true>(pp, fp8, grid, s);
  else
    launch<OWN, false>(pp, fp8, grid, s);
}

int run(PrefixParams& pp, int kv_dtype, int32_t prefix_len, void* workspace, size_t workspace_bytes,
        hipStream_t s) {
  AttnParams& p = pp.a;
  if (p.hq <= 0 || p.hkv <= 0 || p.hq % p.hkv != 0) return NVA_ERR_ARG;
  if (kv_dtype != NVA_KV_BF16 && kv_dtype != NVA_KV_FP8_E4M3) return NVA_ERR_ARG;
  if (p.num_seqs < 0 || p.num_tokens < 0 || p.max_q < 0 || p.max_k < 0 || prefix_len < 0) return NVA_ERR_ARG;
  if (!(p.scale_log2 > 0.0f)) return NVA_ERR_ARG;      // the running maximum is the scaled scores'
  if (p.num_seqs == 0 || p.num_tokens == 0) return NVA_OK;
  if (!p.q || !p.k_cache || !p.v_cache || !p.block_tables || !p.out) return NVA_ERR_ARG;
  if (p.block_size <= 0 || p.block_size % 32 != 0 || p.num_blocks <= 0) return NVA_ERR_UNSUPPORTED;
  if (p.bt_cols < 0 || p.bt_stride < p.bt_cols) return NVA_ERR_ARG;
  p.group = p.hq / p.hkv;
  if (p.group > 64 || p.max_k > kMaxKeys) return NVA_ERR_UNSUPPORTED;
  const int64_t vec = kv_dtype == NVA_KV_BF16 ? 8 : 16;        // elements of a 16-byte access
  if (!aligned16(p.q) || !aligned16(p.out) || !aligned16(p.k_cache) || !aligned16(p.v_cache) ||
      p.q_row_stride % 8 || p.q_head_stride % 8 || p.out_row_stride % 8 || p.out_head_stride % 8 ||
      p.blk_stride % vec || p.tok_stride % vec || p.head_stride % vec)
    return NVA_ERR_UNSUPPORTED;
  // the workspace is the query's, which knows no block size
  make_plan(pp, prefix_len, 0);
  const size_t need = plan_bytes(pp);
  make_plan(pp, prefix_len, p.block_size);
  if (pp.own_units < 0) return NVA_ERR_UNSUPPORTED;    // more workgroups than a grid holds
  if (!workspace || workspace_bytes < need || workspace_bytes < plan_bytes(pp) || !aligned16(workspace))
    return NVA_ERR_WORKSPACE;
  const size_t slots = static_cast<size_t>(p.num_tokens) * p.hq * p.max_splits;
  p.ws_o = static_cast<float*>(workspace);
  p.ws_lse = p.ws_o + slots * kD;
  p.row_nsplit = reinterpret_cast<int32_t*>(p.ws_lse + slots);
  const int32_t grid = p.hkv * (pp.prefix_units + pp.own_units);
  const bool fp8 = kv_dtype == NVA_KV_FP8_E4M3;
  switch (own_kind(static_cast<int64_t>(p.max_q) * p.group)) {
    case 1: launch<1>(pp, fp8, grid, s); break;
    case 2: launch<2>(pp, fp8, grid, s); break;
    case 3: launch<3>(pp, fp8, grid, s); break;
    default: launch<4>(pp, fp8, grid, s); break;
  }
  if (hipGetLastError() != hipSuccess) return NVA_ERR_LAUNCH;
  join_kernel<<<dim3(p.num_tokens, ceil_div(p.hq * (kD / 4), kJoinThreads)), kJoinThreads, 0, s>>>(pp);
  return launch_status();
}

}  // namespace
}  // namespace nva

using namespace nva;

extern "C" size_t nva_shared_prefix_workspace_size(int32_t num_seqs, int32_t num_tokens,
                                                   int32_t num_q_heads, int32_t num_kv_heads,
                                                   int32_t head_dim, int32_t max_seqlen_q,
                                                   int32_t max_seqlen_k, int32_t prefix_len) {
  if (num_seqs <= 0 || num_tokens <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim != kD ||
      max_seqlen_q < 0 || max_seqlen_k < 0 || max_seqlen_k > kMaxKeys || prefix_len < 0 || num_q_heads % num_kv_heads ||
      num_q_heads / num_kv_heads > 64)
    return 0;
  PrefixParams pp = {};
  AttnParams& p = pp.a;
  p.num_seqs = num_seqs;
  p.num_tokens = num_tokens;
  p.hq = num_q_heads;
  p.hkv = num_kv_heads;
  p.group = num_q_heads / num_kv_heads;
  p.max_q = max_seqlen_q;
  p.max_k = max_seqlen_k;
  make_plan(pp, prefix_len, 0);
  return plan_bytes(pp);
}

extern "C" int nva_shared_prefix_attention_varlen(
    const void* q, int64_t q_row_stride, int64_t q_head_stride, const void* k_cache,
    const void* v_cache, int kv_dtype, int64_t cache_block_stride, int64_t cache_token_stride,
    int64_t cache_head_stride, int32_t num_blocks, int32_t block_size, const int32_t* cu_seqlens_q,
    const int32_t* cu_seqlens_k, const int32_t* block_tables, int64_t block_table_stride,
    int32_t max_blocks_per_seq, int32_t num_seqs, int32_t num_tokens, int32_t max_seqlen_q,
    int32_t max_seqlen_k, int32_t prefix_len, int32_t num_q_heads, int32_t num_kv_heads,
    int32_t head_dim, float softmax_scale, const float* k_scale, const float* v_scale, void* out,
    int64_t out_row_stride, int64_t out_head_stride, void* workspace, size_t workspace_bytes,
    void* stream) {
  if (head_dim != kD) return NVA_ERR_UNSUPPORTED;
  if (!cu_seqlens_q || !cu_seqlens_k) return NVA_ERR_ARG;
  PrefixParams pp = {};
  AttnParams& p = pp.a;
  p.q = static_cast<const uint16_t*>(q);
  p.q_row_stride = q_row_stride;
  p.q_head_stride = q_head_stride;
  p.k_cache = static_cast<const uint8_t*>(k_cache);
  p.v_cache = static_cast<const uint8_t*>(v_cache);
  p.blk_stride = cache_block_stride;
  p.tok_stride = cache_token_stride;
  p.head_stride = cache_head_stride;
  p.num_blocks = num_blocks;
  p.block_size = block_size;
  p.cu_q = cu_seqlens_q;
  p.cu_k = cu_seqlens_k;
  p.block_tables = block_tables;
  p.bt_stride = block_table_stride;
  p.bt_cols = max_blocks_per_seq;
  p.num_seqs = num_seqs;
  p.num_tokens = num_tokens;
  p.max_q = max_seqlen_q;
  p.max_k = max_seqlen_k;
  p.hq = num_q_heads;
  p.hkv = num_kv_heads;
  p.scale_log2 = softmax_scale * kLog2e;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.out = static_cast<uint16_t*>(out);
  p.out_row_stride = out_row_stride;
  p.out_head_stride = out_head_stride;
  return run(pp, kv_dtype, prefix_len, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int nva_shared_prefix_attention_decode(
    const void* q, int64_t q_row_stride, int64_t q_head_stride, const void* k_cache,
    const void* v_cache, int kv_dtype, int64_t cache_block_stride, int64_t cache_token_stride,
    int64_t cache_head_stride, int32_t num_blocks, int32_t block_size, const int32_t* cache_seqlens,
    const int32_t* block_tables, int64_t block_table_stride, int32_t max_blocks_per_seq,
    int32_t num_seqs, int32_t max_seqlen_k, int32_t prefix_len, int32_t num_q_heads,
    int32_t num_kv_heads, int32_t head_dim, float softmax_scale, const float* k_scale,
    const float* v_scale, void* out, int64_t out_row_stride, int64_t out_head_stride,
    void* workspace, size_t workspace_bytes, void* stream) {
  if (head_dim != kD) return NVA_ERR_UNSUPPORTED;
  if (!cache_seqlens) return NVA_ERR_ARG;
  PrefixParams pp = {};
  AttnParams& p = pp.a;
  p.q = static_cast<const uint16_t*>(q);
  p.q_row_stride = q_row_stride;
  p.q_head_stride = q_head_stride;
  p.k_cache = static_cast<const uint8_t*>(k_cache);
  p.v_cache = static_cast<const uint8_t*>(v_cache);
  p.blk_stride = cache_block_stride;
  p.tok_stride = cache_token_stride;
  p.head_stride = cache_head_stride;
  p.num_blocks = num_blocks;
  p.block_size = block_size;
  p.seqlens = cache_seqlens;
  p.block_tables = block_tables;
  p.bt_stride = block_table_stride;
  p.bt_cols = max_blocks_per_seq;
  p.num_seqs = num_seqs;
  p.num_tokens = num_seqs;
  p.max_q = 1;
  p.max_k = max_seqlen_k;
  p.hq = num_q_heads;
  p.hkv = num_kv_heads;
  p.scale_log2 = softmax_scale * kLog2e;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.out = static_cast<uint16_t*>(out);
  p.out_row_stride = out_row_stride;
  p.out_head_stride = out_head_stride;
  return run(pp, kv_dtype, prefix_len, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

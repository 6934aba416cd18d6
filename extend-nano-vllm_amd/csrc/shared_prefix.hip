// Paged attention of a batch whose sequences share a long prefix (gfx950,
// MFMA 32x32x16 bf16).
//
// The softmax over a row's keys is joined from parts: for a part P of the keys
//   m_P = max s, l_P = sum exp(s - m_P), o_P = sum exp(s - m_P) v / l_P,
// the whole is  sum_P w_P o_P / sum_P w_P  with w_P = l_P exp(m_P - max m).
// The prefix's keys are the same for every sequence, so their parts are
// computed for tiles of query rows of all sequences together: each K and V byte
// of the prefix is read once per tile instead of once per sequence, and the
// products run on full matrix tiles.  Each sequence's own keys are parts of
// tiles of its own rows.
//
// Two launches: the parts (prefix and own keys side by side in one grid, so that
// the matrix work of the one runs beside the memory stream of the other), then
// the join.
//
// A unit of work is a tile of up to 32 NW query rows (NW waves of 32 columns)
// of one kv head against a range of keys, 64 keys a step:
//   * S^T = K . Q^T with keys as M: lane 32 h + c holds, for query column c, the
//     keys 8 b + 4 h + i (b, i = 0..3) of each 32-key tile in accumulator
//     element 4 b + i.  Elements 8 t .. 8 t + 7 are the k-slots of lane half h
//     in the B operand of slice t of O^T += V^T . P^T, if slot j of half h stands
//     for key 16 t + 8 (j / 4) + 4 h + j % 4, so P goes from accumulator to
//     operand by rounding to bf16 alone (relative 2^-9 per probability, as the
//     paged attention does), and V^T is read from LDS in that key order by two
//     transpose loads.  Sums and states are fp32.
//   * K/V tiles go through registers two steps ahead and one of two LDS buffers
//     one step ahead, one barrier a step.  FP8 pages become bf16 on the way.
#include "common.h"

namespace nva {
namespace {

constexpr int kD = 128;
constexpr int kKeys = 64;                            // keys of a step
constexpr int kKPitch = 68, kVPitch = 80;            // dwords per staged row
constexpr int kBuf = kKeys * (kKPitch + kVPitch);
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescaleSlack = 8.0f;                // log2 headroom before the running max moves

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
typedef __attribute__((ext_vector_type(2))) float f32x2_t;
typedef __attribute__((ext_vector_type(16))) float f32x16_t;
typedef __attribute__((ext_vector_type(4))) short s16x4_t;
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;

struct PrefixParams {
  const uint16_t* q;
  int64_t q_row_stride, q_head_stride;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  int64_t blk_stride, tok_stride, head_stride;       // elements
  int32_t num_blocks, block_size;
  const int32_t* cu_q;                               // null: row i is sequence i
  const int32_t* cu_k;                               // non-null: L_i = cu_k[i+1] - cu_k[i]
  const int32_t* seqlens;                            // otherwise L_i = seqlens[i]
  const int32_t* block_tables;
  int64_t bt_stride;
  int32_t bt_cols;
  int32_t num_seqs, num_tokens, max_q, max_k;
  int32_t hq, hkv, group;
  float scale_log2;
  const float* k_scale;
  const float* v_scale;
  uint16_t* out;
  int64_t out_row_stride, out_head_stride;
  float* ws_o;                                       // [token][head][part][kD], normalised
  float* ws_lse;                                     // [token][head][part], log2
  int32_t* row_parts;                                // [token] parts of its own keys, -1: no output but zeros
  // the plan
  int32_t prefix;                                    // shared keys (a multiple of 32)
  int32_t prefix_split, prefix_parts;                // keys of a prefix part, parts
  int32_t own_split, own_parts;                      // the same of a sequence's own keys (parts: bound)
  int32_t qtile, prefix_tiles, own_tiles;            // query positions of a tile, tiles
  int32_t prefix_units, own_units;                   // per kv head
};

__device__ __forceinline__ float exp2f_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// over the lane pair (l, l ^ 32), by the swap of the two halves; the results are
// read into integers first (a bit cast of the second element of the builtin's
// result vector compiles to the first, ROCm 7.2)
__device__ __forceinline__ float max_halves(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t lo = r[0], hi = r[1];
  return fmaxf(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
}
__device__ __forceinline__ float sum_halves(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t lo = r[0], hi = r[1];
  return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
}

__device__ __forceinline__ f32x16_t mfma32(bf16x8_t a, bf16x8_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// 8 e4m3 bytes as bf16, exact
__device__ __forceinline__ bf16x8_t fp8x8_to_bf16(uint2 w) {
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, 1.0f, false);
  const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, 1.0f, true);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, 1.0f, false);
  const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, 1.0f, true);
  return __builtin_bit_cast(bf16x8_t,
                            make_uint4(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b),
                                       __builtin_bit_cast(uint32_t, c), __builtin_bit_cast(uint32_t, d)));
}

// V^T operand of head_dim tile dt (d = 32 dt + lane % 32) and key slice t (16
// keys): transpose load r (0, 1) hands lane 32 h + c the keys 16 t + 8 r + 4 h ..
// + 3.  ds_read_b64_tr_b16 gives lane l element e of the 8-byte piece that lane
// 16 (l / 16) + 4 e + (l % 16) / 4 addressed, at position (l % 16) % 4.
__device__ __forceinline__ bf16x8_t v_operand(const uint32_t* rows, int lane, int t, int dt) {
  const int h = lane >> 5, dh = (lane >> 4) & 1, i = lane & 15;
  uint32_t* p0 = const_cast<uint32_t*>(rows) + (16 * t + 4 * h + (i >> 2)) * kVPitch + 16 * dt + 8 * dh +
                 2 * (i & 3);
  const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(p0));
  const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(p0 + 8 * kVPitch));
  return bf16x8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// Query rows and keys of a sequence.  A sequence clipped to its first max_q
// rows also drops the keys of the rows cut, so that each kept row j still sees
// keys [0, L - raw + j]; then at most max_k keys are seen.
struct Geometry {
  int q_start, q_len, raw, L;
};
__device__ __forceinline__ Geometry geometry(const PrefixParams& p, int seq) {
  int q0 = seq, q1 = seq + 1, k0 = 0;
  const int k1 = (p.cu_k ? p.cu_k + 1 : p.seqlens)[seq];
  if (p.cu_q) {
    q0 = p.cu_q[seq];
    q1 = p.cu_q[seq + 1];
  }
  if (p.cu_k) k0 = p.cu_k[seq];
  Geometry r;
  r.q_start = q0;
  r.raw = q1 - q0;
  if (q0 < 0 || q0 >= p.num_tokens) r.raw = 0;
  else if (r.raw > p.num_tokens - q0) r.raw = p.num_tokens - q0;
  if (r.raw < 0) r.raw = 0;
  r.q_len = r.raw > p.max_q ? p.max_q : r.raw;
  r.L = k1 - k0 - (r.raw - r.q_len);
  r.L = r.L > p.max_k ? p.max_k : r.L;
  return r;
}

// the id of the block that lane i's column is from `first` on, -1 past the table
__device__ __forceinline__ int block_ids(const PrefixParams& p, const int32_t* table, int key) {
  const int col = key / p.block_size + static_cast<int>(threadIdx.x & (kWave - 1));
  return col < p.bt_cols ? table[col] : -1;
}

template <int NW, bool FP8>
__global__ void __launch_bounds__(kWave * NW, 2) shared_prefix_kernel(PrefixParams p) {
  constexpr int kThreads = kWave * NW;
  constexpr int kEsz = FP8 ? 1 : 2;
  constexpr int kRowGran = kD * kEsz / 16;               // 16-byte granules per K or V row
  constexpr int kPer = kKeys * kRowGran / kThreads;      // a thread's granules of K (and of V)
  static_assert(kPer >= 1, "every thread loads at least one granule");
  __shared__ __attribute__((aligned(16))) uint32_t lds[2 * kBuf];
  __shared__ int32_t last_key[32 * NW];                  // of each query position of the tile, -1: none

  const int kvh = blockIdx.x % p.hkv;
  // prefix units are spread evenly among the others
  const int all = p.prefix_units + p.own_units;
  const int u = blockIdx.x / p.hkv;
  const int before = static_cast<int>(static_cast<int64_t>(u) * p.prefix_units / all);
  const bool is_prefix = static_cast<int>(static_cast<int64_t>(u + 1) * p.prefix_units / all) > before;

  int tok0, jn, kv_begin, kv_end, part;
  const int32_t* table;
  if (is_prefix) {
    const int tile = before % p.prefix_tiles, split = before / p.prefix_tiles;
    tok0 = tile * p.qtile;
    jn = p.num_tokens - tok0 < p.qtile ? p.num_tokens - tok0 : p.qtile;
    kv_begin = split * p.prefix_split;
    kv_end = kv_begin + p.prefix_split < p.prefix ? kv_begin + p.prefix_split : p.prefix;
    part = split;
    table = p.block_tables;
    // every position's last visible key, from the sequence that holds it
    for (int i = threadIdx.x; i < jn; i += kThreads) last_key[i] = -1;
    __syncthreads();
    for (int seq = p.cu_q ? static_cast<int>(threadIdx.x) : tok0 + static_cast<int>(threadIdx.x);
         seq < (p.cu_q ? p.num_seqs : tok0 + jn); seq += kThreads) {
      const Geometry g = geometry(p, seq);
      const int lo = g.q_start > tok0 ? g.q_start : tok0;
      const int hi = g.q_start + g.q_len < tok0 + jn ? g.q_start + g.q_len : tok0 + jn;
      for (int t = lo; t < hi; ++t) last_key[t - tok0] = g.L - g.q_len + (t - g.q_start);
    }
    __syncthreads();
  } else {
    int rest = u - before;
    const int seq = rest % p.num_seqs;
    rest /= p.num_seqs;
    const int qt = p.own_tiles - 1 - rest % p.own_tiles, split = rest / p.own_tiles;
    Geometry g = geometry(p, seq);
    const int j0 = qt * p.qtile;
    jn = g.q_len - j0 < p.qtile ? g.q_len - j0 : p.qtile;
    jn = __builtin_amdgcn_readfirstlane(jn);
    const int limit = __builtin_amdgcn_readfirstlane(g.L - g.q_len + j0 + jn);   // keys seen by the last row
    tok0 = __builtin_amdgcn_readfirstlane(g.q_start + j0);
    kv_begin = p.prefix + split * p.own_split;
    kv_end = kv_begin + p.own_split < limit ? kv_begin + p.own_split : limit;
    part = p.prefix_parts + split;
    table = p.block_tables + static_cast<int64_t>(seq) * p.bt_stride;
    if (kvh == 0 && split == 0) {
      // what the join reads of each row: the parts written for it
      const int parts = limit > p.prefix ? (limit - p.prefix + p.own_split - 1) / p.own_split : 0;
      for (int j = threadIdx.x; j < jn; j += kThreads) p.row_parts[tok0 + j] = parts;
      if (qt == 0)
        for (int j = g.q_len + threadIdx.x; j < g.raw; j += kThreads) p.row_parts[g.q_start + j] = -1;
    }
    if (jn <= 0 || kv_begin >= kv_end) return;
    for (int j = threadIdx.x; j < jn; j += kThreads) last_key[j] = g.L - g.q_len + j0 + j;
    __syncthreads();
  }

  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int wv = __builtin_amdgcn_readfirstlane(tid / kWave);
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
  const int n = 32 * wv + col;
  const int nn = n < rows ? n : 0;
  const int jc = nn / p.group, hc = kvh * p.group + nn % p.group;
  const int64_t tok = tok0 + jc;
  bf16x8_t qv[8];
  {
    const uint16_t* qp = p.q + tok * p.q_row_stride + static_cast<int64_t>(hc) * p.q_head_stride + 8 * h;
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
  // keys from it on by none
  const int wave_end = 32 * wv < rows ? __builtin_amdgcn_readfirstlane(most) + 1 : 0;

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
    kdst[i] = row * kKPitch + c * (FP8 ? 8 : 4);
    vdst[i] = kKeys * kKPitch + row * kVPitch + c * (FP8 ? 8 : 4);
  }
  // lane i of lane_blk holds the id of the i-th block from the one ld_blk counts from
  int lane_blk = block_ids(p, table, kv_begin);
  int ld_key = kv_begin;                                 // first key of the next half to load,
  int ld_blk = 0;                                        // its block
  int ld_tok = kv_begin % p.block_size;                  // and its token there
  auto next_half = [&](__amdgpu_buffer_rsrc_t& kr, __amdgpu_buffer_rsrc_t& vr) -> bool {
    const bool live = ld_key < kv_end;
    if (live && ld_blk >= kWave) {
      ld_blk = 0;
      lane_blk = block_ids(p, table, ld_key);
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
  auto stage = [&](const Tile& t, int b) {
    uint32_t* base = lds + b * kBuf;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if constexpr (FP8) {
        *reinterpret_cast<bf16x8_t*>(base + kdst[i]) = fp8x8_to_bf16(make_uint2(t.k[i].x, t.k[i].y));
        *reinterpret_cast<bf16x8_t*>(base + kdst[i] + 4) = fp8x8_to_bf16(make_uint2(t.k[i].z, t.k[i].w));
        *reinterpret_cast<bf16x8_t*>(base + vdst[i]) = fp8x8_to_bf16(make_uint2(t.v[i].x, t.v[i].y));
        *reinterpret_cast<bf16x8_t*>(base + vdst[i] + 4) = fp8x8_to_bf16(make_uint2(t.v[i].z, t.v[i].w));
      } else {
        *reinterpret_cast<uint4*>(base + kdst[i]) = t.k[i];
        *reinterpret_cast<uint4*>(base + vdst[i]) = t.v[i];
      }
    }
  };

  float m_run = -INFINITY, l_run = 0.0f;
  f32x16_t acc[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[dt][i] = 0.0f;

  auto compute = [&](int kb, int valid, int b) {
    if (kb >= wave_end || valid == 0) return;
    const uint32_t* kst = lds + b * kBuf;
    const uint32_t* vst = kst + kKeys * kKPitch;
    f32x16_t sacc[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) sacc[kt][i] = 0.0f;
#pragma unroll
    for (int s = 0; s < 8; ++s)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const bf16x8_t ko =
            *reinterpret_cast<const bf16x8_t*>(kst + (32 * kt + col) * kKPitch + 8 * s + 4 * h);
        sacc[kt] = mfma32(ko, qv[s], sacc[kt]);
      }
    if (kb + kKeys > wave_full || valid != 3) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = kb + 32 * kt + 8 * (i >> 2) + 4 * h + (i & 3);
          if (key > lim || !((valid >> kt) & 1)) sacc[kt][i] = -INFINITY;
        }
    }
    float cmax = sacc[0][0];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) cmax = fmaxf(cmax, sacc[kt][i]);
    cmax = max_halves(cmax) * sl2;
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
    bf16x8_t pb[4];
    float psum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int t = 0; t < 4; ++t) {
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
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) acc[dt] = mfma32(v_operand(vst, lane, t, dt), pb[t], acc[dt]);
  };

  // step c computes tile c from buffer c & 1, stages tile c + 1 into the other
  // buffer and loads tile c + 2; the barrier publishes the staged tile and
  // frees the computed one
  const int ntiles = (kv_end - kv_begin + kKeys - 1) / kKeys;
  Tile t;
  load_tile(t);
  stage(t, 0);
  int valid = t.valid;
  load_tile(t);
  __syncthreads();
  for (int c = 0; c < ntiles; ++c) {
    compute(kv_begin + c * kKeys, valid, c & 1);
    if (c + 1 < ntiles) {
      stage(t, (c + 1) & 1);
      valid = t.valid;
      load_tile(t);
    }
    __syncthreads();
  }

  // ---- the part: elements 4 b + i of tile dt are d = 32 dt + 8 b + 4 h + i
  const float lsum = sum_halves(l_run);
  const float inv = lsum > 0.0f ? vscale / lsum : 0.0f;
  if (n < rows) {
    const int64_t slot = (tok * p.hq + hc) * (p.prefix_parts + p.own_parts) + part;
    float* wo = p.ws_o + slot * kD;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        *reinterpret_cast<float4*>(wo + 32 * dt + 8 * b + 4 * h) =
            make_float4(acc[dt][4 * b] * inv, acc[dt][4 * b + 1] * inv, acc[dt][4 * b + 2] * inv,
                        acc[dt][4 * b + 3] * inv);
    if (h == 0) p.ws_lse[slot] = lsum > 0.0f ? m_run + __log2f(lsum) : -INFINITY;
  }
}

// The join.  A thread owns four head_dim elements of one (token, head) and folds
// its parts, kBatch loads at a time, into a running maximum, weight and sum.
constexpr int kJoinThreads = 256;
constexpr int kBatch = 8;
__global__ void __launch_bounds__(kJoinThreads) join_kernel(PrefixParams p) {
  const int t = blockIdx.x;
  // rows of no sequence are left alone
  const int lo = p.cu_q ? p.cu_q[0] : 0;
  const int hi = p.cu_q ? p.cu_q[p.num_seqs] : p.num_seqs;
  int own = p.row_parts[t];
  if (t < lo || t >= hi) return;
  const int idx = blockIdx.y * kJoinThreads + threadIdx.x;
  if (idx >= p.hq * (kD / 4)) return;
  const int h = idx / (kD / 4), d4 = idx % (kD / 4);
  own = own < p.own_parts ? own : p.own_parts;
  const int parts = own < 0 ? 0 : p.prefix_parts + own;
  const int64_t base = (static_cast<int64_t>(t) * p.hq + h) * (p.prefix_parts + p.own_parts);
  float M = -INFINITY, wsum = 0.0f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < parts; s0 += kBatch) {
    float lse[kBatch];
    float4 v[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const bool in = s0 + u < parts;
      lse[u] = in ? p.ws_lse[base + s0 + u] : -INFINITY;
      v[u] = in ? *reinterpret_cast<const float4*>(p.ws_o + (base + s0 + u) * kD + 4 * d4)
                : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float mb = M;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) mb = fmaxf(mb, lse[u]);
    if (mb == -INFINITY) continue;
    const float r = M == -INFINITY ? 0.0f : exp2f_fast(M - mb);
    wsum *= r;
    o.x *= r; o.y *= r; o.z *= r; o.w *= r;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const float w = lse[u] == -INFINITY ? 0.0f : exp2f_fast(lse[u] - mb);
      wsum += w;
      o.x += w * v[u].x; o.y += w * v[u].y; o.z += w * v[u].z; o.w += w * v[u].w;
    }
    M = mb;
  }
  const float inv = wsum > 0.0f ? 1.0f / wsum : 0.0f;
  auto pack = [&](float a, float b) {
    return static_cast<uint32_t>(f32_to_bf16(a * inv)) | (static_cast<uint32_t>(f32_to_bf16(b * inv)) << 16);
  };
  uint16_t* op = p.out + static_cast<int64_t>(t) * p.out_row_stride +
                 static_cast<int64_t>(h) * p.out_head_stride + 4 * d4;
  *reinterpret_cast<uint2*>(op) = make_uint2(pack(o.x, o.y), pack(o.z, o.w));
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

constexpr int kWaves = 4;
constexpr int kMinPart = 256;          // keys a part has at least

// Tiles and parts of a call.  Unknown lengths are bounded by max_k.
void make_plan(PrefixParams& p, int32_t prefix_len) {
  p.prefix = prefix_len < p.max_k ? prefix_len / 32 * 32 : p.max_k / 32 * 32;
  p.qtile = 32 * kWaves / p.group;
  p.prefix_tiles = ceil_div(p.num_tokens, p.qtile);
  p.own_tiles = ceil_div(p.max_q, p.qtile);
  const int64_t places = 2 * static_cast<int64_t>(device_cus());
  // prefix: parts enough to give every place of the device a unit
  int32_t parts = static_cast<int32_t>(places / (static_cast<int64_t>(p.prefix_tiles) * p.hkv));
  const int32_t most = p.prefix / kMinPart;
  parts = parts < 1 ? 1 : parts;
  parts = parts > most ? (most < 1 ? 1 : most) : parts;
  p.prefix_split = ceil_div(ceil_div(p.prefix, parts), kKeys) * kKeys;
  p.prefix_parts = p.prefix > 0 ? ceil_div(p.prefix, p.prefix_split) : 0;
  // own keys
  const int32_t own = p.max_k - p.prefix;
  int64_t own_parts = places / (static_cast<int64_t>(p.num_seqs) * p.own_tiles * p.hkv);
  const int32_t own_most = own / kMinPart;
  own_parts = own_parts < 1 ? 1 : own_parts;
  own_parts = own_parts > own_most ? (own_most < 1 ? 1 : own_most) : own_parts;
  p.own_split = own > 0 ? ceil_div(ceil_div(own, own_parts), kKeys) * kKeys : kKeys;
  p.own_parts = own > 0 ? ceil_div(own, p.own_split) : 1;
  const int64_t prefix_units = static_cast<int64_t>(p.prefix_parts) * p.prefix_tiles;
  const int64_t own_units = static_cast<int64_t>(p.num_seqs) * p.own_tiles * p.own_parts;
  const bool fits = (prefix_units + own_units) * p.hkv <= 0x7FFFFFFF;
  p.prefix_units = fits ? static_cast<int32_t>(prefix_units) : -1;
  p.own_units = fits ? static_cast<int32_t>(own_units) : -1;
}

size_t plan_bytes(const PrefixParams& p) {
  const size_t slots = static_cast<size_t>(p.num_tokens) * p.hq * (p.prefix_parts + p.own_parts);
  return slots * (kD + 1) * sizeof(float) + static_cast<size_t>(p.num_tokens) * sizeof(int32_t);
}

int run(PrefixParams& p, int kv_dtype, int32_t prefix_len, void* workspace, size_t workspace_bytes,
        hipStream_t s) {
  if (p.hq <= 0 || p.hkv <= 0 || p.hq % p.hkv != 0) return NVA_ERR_ARG;
  if (kv_dtype != NVA_KV_BF16 && kv_dtype != NVA_KV_FP8_E4M3) return NVA_ERR_ARG;
  if (p.num_seqs < 0 || p.num_tokens < 0 || p.max_q < 0 || p.max_k < 0 || prefix_len < 0) return NVA_ERR_ARG;
  if (!(p.scale_log2 > 0.0f)) return NVA_ERR_ARG;      // the running maximum is the scaled scores'
  if (p.num_seqs == 0 || p.num_tokens == 0 || p.max_q == 0) return NVA_OK;
  if (!p.q || !p.k_cache || !p.v_cache || !p.block_tables || !p.out) return NVA_ERR_ARG;
  if (p.block_size <= 0 || p.block_size % 32 != 0 || p.num_blocks <= 0) return NVA_ERR_UNSUPPORTED;
  if (p.bt_cols < 0 || p.bt_stride < p.bt_cols) return NVA_ERR_ARG;
  p.group = p.hq / p.hkv;
  if (p.group > 64) return NVA_ERR_UNSUPPORTED;
  const int64_t vec = kv_dtype == NVA_KV_BF16 ? 8 : 16;        // elements of a 16-byte access
  if (!aligned16(p.q) || !aligned16(p.out) || !aligned16(p.k_cache) || !aligned16(p.v_cache) ||
      p.q_row_stride % 8 || p.q_head_stride % 8 || p.out_row_stride % 8 || p.out_head_stride % 8 ||
      p.blk_stride % vec || p.tok_stride % vec || p.head_stride % vec)
    return NVA_ERR_UNSUPPORTED;
  make_plan(p, prefix_len);
  if (p.own_units < 0) return NVA_ERR_UNSUPPORTED;     // more workgroups than a grid holds
  if (!workspace || workspace_bytes < plan_bytes(p) || !aligned16(workspace)) return NVA_ERR_WORKSPACE;
  const size_t slots = static_cast<size_t>(p.num_tokens) * p.hq * (p.prefix_parts + p.own_parts);
  p.ws_o = static_cast<float*>(workspace);
  p.ws_lse = p.ws_o + slots * kD;
  p.row_parts = reinterpret_cast<int32_t*>(p.ws_lse + slots);
  const int32_t grid = p.hkv * (p.prefix_units + p.own_units);
  if (kv_dtype == NVA_KV_FP8_E4M3)
    shared_prefix_kernel<kWaves, true><<<grid, kWave * kWaves, 0, s>>>(p);
  else
    shared_prefix_kernel<kWaves, false><<<grid, kWave * kWaves, 0, s>>>(p);
  if (hipGetLastError() != hipSuccess) return NVA_ERR_LAUNCH;
  join_kernel<<<dim3(p.num_tokens, ceil_div(p.hq * (kD / 4), kJoinThreads)), kJoinThreads, 0, s>>>(p);
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
      max_seqlen_q <= 0 || max_seqlen_k < 0 || prefix_len < 0 || num_q_heads % num_kv_heads ||
      num_q_heads / num_kv_heads > 64)
    return 0;
  PrefixParams p = {};
  p.num_seqs = num_seqs;
  p.num_tokens = num_tokens;
  p.hq = num_q_heads;
  p.hkv = num_kv_heads;
  p.group = num_q_heads / num_kv_heads;
  p.max_q = max_seqlen_q;
  p.max_k = max_seqlen_k;
  make_plan(p, prefix_len);
  return plan_bytes(p);
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
  PrefixParams p = {};
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
  return run(p, kv_dtype, prefix_len, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
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
  PrefixParams p = {};
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
  return run(p, kv_dtype, prefix_len, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

// Device code that the attention kernels share (gfx950): parameters and sequence
// geometry, lane exchanges, operand reads, and attend_segment, one query tile
// against a range of a sequence's keys (paged_attention.hip describes it).
#pragma once

#include "common.h"

namespace nva {
namespace {

constexpr int kD = 128;
constexpr int kChunk = 32;
constexpr int kVPitch = 68;                          // dwords per staged V row
constexpr int kVStage = kChunk * kVPitch;            // dwords of the wave's V stage
// a split of attend_segment spans at most kWave - 2 blocks; blocks hold at least
// kChunk tokens
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescaleSlack = 8.0f;   // log2 headroom before the running max moves

typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;
typedef __attribute__((ext_vector_type(2))) float f32x2_t;

struct AttnParams {
  const uint16_t* q;
  int64_t q_row_stride, q_head_stride;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  int64_t blk_stride, tok_stride, head_stride;       // elements
  int32_t num_blocks, block_size;
  const int32_t* cu_q;                                // null: row i is sequence i
  const int32_t* cu_k;                                // non-null: L_i = cu_k[i+1]-cu_k[i]
  const int32_t* seqlens;                             // otherwise L_i = seqlens[i]
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
  float* ws_o;
  float* ws_lse;
  int32_t split_len, max_splits;
  int32_t qtile, n_qtiles;                            // query positions per tile (wide-tile kernel: several)
  // stream decomposition (one query tile per sequence)
  int32_t min_range_chunks, max_range_chunks;
  int32_t* row_nsplit;                                // [num_tokens] split count per query row
  // paired mode: grid rows y >= pair_rows take the sequences from the last
  // one backwards (0: row y is sequence y)
  int32_t pair_rows;
};

__device__ __forceinline__ float exp2f_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// Log-sum-exp (log2 domain) of a part of a row's keys, from its running maximum
// and sum: -inf where the row sees no key of it (the sum is 0; the largest score
// of those it sees leaves at least 1), NaN where a score was NaN or +inf.
__device__ __forceinline__ float part_lse(float m, float sum) {
  return sum == 0.0f ? -INFINITY : m + __log2f(sum);
}

// Reductions over the lane pairs (l, l ^ 16) and (l, l ^ 32), every lane
// receiving the pair's result.  gfx950's v_permlane16_swap /
// v_permlane32_swap with both operands x leave the pair's two values, the
// lower lane's first, in the two results of every lane of the pair: a
// VALU exchange.  __shfl_xor compiles to ds_bpermute, which goes through
// the LDS unit and makes the next use wait for every outstanding LDS
// operation of the wave (in the key loop: the V rows just staged).  Both
// lanes combine the same two values in the same order, and max and + are
// commutative, so the results equal the shuffle forms' bit for bit.  The
// two results are read into integers before the bit cast: a bit cast of
// the second element of the builtin's result vector compiles to the first
// element (ROCm 7.2 clang).
__device__ __forceinline__ float max_xor16(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t lo = r[0], hi = r[1];
  return fmaxf(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
}
__device__ __forceinline__ float max_xor32(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t lo = r[0], hi = r[1];
  return fmaxf(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
}
__device__ __forceinline__ float sum_xor16(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t lo = r[0], hi = r[1];
  return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
}
__device__ __forceinline__ float sum_xor32(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t lo = r[0], hi = r[1];
  return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
}

// Orders a wave's own LDS writes and reads: LDS executes one wave's
// operations in issue order, so the compiler must only keep program order
// and wait for outstanding LDS operations.
__device__ __forceinline__ void lds_wave_sync() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

typedef __attribute__((ext_vector_type(4))) short s16x4_t;
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;

// The V^T operand of the O^T += V^T . P^T product for head_dim tile (pp, hf),
// read from a staged chunk (32 key rows of `pitch` dwords, bf16) with gfx950's
// LDS transpose load.  ds_read_b64_tr_b16 hands lane l element e of the
// 8-byte piece that lane 16 (l / 16) + 4 e + (l % 16) / 4 addressed, at that
// piece's position (l % 16) % 4.  Lane l addresses key row
// 4 (l / 16) + (l % 16) / 4 (+ 16 for the second load), head_dim
// 32 pp + 8 (l % 4) + 4 hf, so lane (g, m16) receives
//   A row m16 <-> d = 32 pp + 8 (m16 / 4) + 4 hf + m16 % 4,
//   k-slot 8 g + 4 r + e <-> key 16 r + 4 g + e   (the P^T operand's order),
// and the accumulator tile (pp, hf) holds d = 32 pp + 8 g + 4 hf + i in
// element i of lane (g, m16): the two tiles of pair pp give the lane eight
// consecutive head_dim values.  With a row pitch of 72 dwords the 16 lanes
// one LDS cycle serves fall on at most two addresses per bank (at 68 dwords,
// four).
__device__ __forceinline__ bf16x8_t v_operand_tr(const uint32_t* rows, int pitch, int lane, int pp,
                                                 int hf) {
  const int row = 4 * (lane >> 4) + ((lane & 15) >> 2);
  uint32_t* p0 = const_cast<uint32_t*>(rows) + row * pitch + 16 * pp + 4 * (lane & 3) + 2 * hf;
  const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(p0));
  const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(p0 + 16 * pitch));
  return bf16x8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

__device__ __forceinline__ f32x4_t mfma(bf16x8_t a, bf16x8_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  return static_cast<uint32_t>(f32_to_bf16(lo)) | (static_cast<uint32_t>(f32_to_bf16(hi)) << 16);
}

// 8 fp8 (OCP e4m3fn) bytes -> 8 bf16, exact: v_cvt_scalef32_pk_bf16_fp8 with
// scale 1.0 converts two bytes of the selected 16-bit half (every e4m3 value,
// subnormals included, is a bf16 value; 0x7F / 0xFF give NaN).  The kernel
// applies k_scale / v_scale in fp32 elsewhere.
__device__ __forceinline__ bf16x8_t fp8x8_to_bf16(uint2 w) {
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, 1.0f, false);
  const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.x, 1.0f, true);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, 1.0f, false);
  const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w.y, 1.0f, true);
  const uint4 r = make_uint4(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b),
                            __builtin_bit_cast(uint32_t, c), __builtin_bit_cast(uint32_t, d));
  return __builtin_bit_cast(bf16x8_t, r);
}

// Query rows and keys of sequence seq (any lane's own sequence).  The end
// of the key range is one load from a selected pointer (cu_k + 1 or
// seqlens), issued with the others before any value is used, so the
// geometry costs one memory latency.
// q_rows_raw (optional) receives the sequence's row count before the
// max_seqlen_q clip (bounded by num_tokens the same way).  A sequence
// clipped to its first max_q rows also drops the keys of its clipped rows
// (L shrinks by the rows cut), so each kept row j still sees keys
// [0, L - q_raw + j], its unclipped causal window.
__device__ __forceinline__ void seq_geometry(const AttnParams& p, int seq, int& q_start, int& q_len,
                                             int& L, int* q_rows_raw = nullptr) {
  int q0 = seq, q1 = seq + 1, k0 = 0;
  const int k1 = (p.cu_k ? p.cu_k + 1 : p.seqlens)[seq];
  if (p.cu_q) {
    q0 = p.cu_q[seq];
    q1 = p.cu_q[seq + 1];
  }
  if (p.cu_k) k0 = p.cu_k[seq];
  q_start = q0;
  int raw = q1 - q0;
  if (q_start < 0 || q_start >= p.num_tokens) raw = 0;
  else if (raw > p.num_tokens - q_start) raw = p.num_tokens - q_start;
  q_len = raw > p.max_q ? p.max_q : raw;
  if (q_rows_raw) *q_rows_raw = raw;
  L = k1 - k0 - (raw - q_len);
  L = L > p.max_k ? p.max_k : L;
}

// seq_geometry for a wave-uniform seq: readfirstlane states the values'
// uniformity, which the compiler cannot see through the pointer select, so
// that they stay in scalar registers (a buffer descriptor built from them
// would otherwise need a waterfall loop per load).
__device__ __forceinline__ void seq_geometry_uniform(const AttnParams& p, int seq, int& q_start,
                                                     int& q_len, int& L,
                                                     int* q_rows_raw = nullptr) {
  seq_geometry(p, seq, q_start, q_len, L, q_rows_raw);
  q_start = __builtin_amdgcn_readfirstlane(q_start);
  q_len = __builtin_amdgcn_readfirstlane(q_len);
  L = __builtin_amdgcn_readfirstlane(L);
  if (q_rows_raw) *q_rows_raw = __builtin_amdgcn_readfirstlane(*q_rows_raw);
}

// Block ids of the split that starts at key kv_begin, one per lane: lane i
// holds logical block kv_begin / block_size + i (the host keeps a split
// within kWave - 2 blocks; lanes past the split hold ids nobody reads).
// Needs no sequence geometry, so the fixed kernel issues it together with
// the geometry loads instead of after them.
__device__ __forceinline__ int split_block_ids(const AttnParams& p, int seq, int kv_begin) {
  const int col = kv_begin / p.block_size + static_cast<int>(threadIdx.x & (kWave - 1));
  return col < p.bt_cols ? p.block_tables[static_cast<int64_t>(seq) * p.bt_stride + col] : -1;
}

// Segments over an FP8 cache, and shared segments over a bf16 cache
// (several waves, one chunk buffer), also stage K through a wave-private
// LDS tile: the K rows then load like the V rows, whole 128-byte lines per
// instruction with the non-temporal hint (FP8 rows dequantised to bf16 on
// the way in, as V's), and the MFMA operands are read back in the order
// the registers held them.
// NVA_K_STAGE=0 at build time keeps K in registers (half lines, default
// policy) for comparison.
#ifndef NVA_K_STAGE
#define NVA_K_STAGE 1
#endif
// Dword offset of 16-byte column c (0..15) of K row r in a K stage: rows of
// 64 dwords, the column XORed with the row's low four bits, so that the
// 16 rows of an operand read (one column) and the 16 columns of a staging
// write (one row) each fall on 16 different 16-byte bank groups.  With the
// V stage's 68-dword pitch instead, the operand reads conflicted (626 k
// conflict cycles per config-3 call, 10.5 M per FP8 config-4 call; 0 with
// the swizzle, the call times unchanged).
__device__ __forceinline__ int kst_slot(int r, int c) { return r * 64 + ((c ^ (r & 15)) << 2); }
constexpr bool k_staged(bool fp8, bool pipe, int wps) {
  return NVA_K_STAGE && (fp8 || (!pipe && wps > 1));
}

// One segment of work: the query tile of sequence seq (all its rows
// for kv head kvh; the sequence's rows start at q_start, it has q_len query
// rows and L keys) against keys [kv_begin, kv_end), which is split `split`
// of the `nsplit` splits covering its keys.  lane_blk is
// split_block_ids(p, seq, kv_begin).  A single split
// writes the bf16 output; otherwise a normalised fp32 partial and its
// log-sum-exp go to the workspace for combine_kernel.
//
// WPS > 1 waves (one workgroup) share a segment: wave w takes chunks w,
// w + WPS, ...; their softmax states are merged through LDS at the end and
// wave 0 writes the result.  `vst` then holds WPS stages.
template <int NT, bool FP8, bool PIPE, int WPS>
__device__ __forceinline__ void attend_segment(const AttnParams& p, uint32_t* vst, bf16x8_t* qst,
                                               const int kvh, const int seq, const int q_start,
                                               const int q_len, const int L, const int kv_begin,
                                               const int kv_end, const int split,
                                               const int nsplit, const int lane_blk) {
  static_assert(WPS == 1 || !PIPE, "shared segments use the single-buffer loop");
  static_assert(WPS == 1 || (NT <= 2 && (8 * kWave * 4 + 2 * kWave) <= kVStage),
                "a wave's parked state must fit one V stage per column tile");
  constexpr bool KST = k_staged(FP8, PIPE, WPS);
  const int lane = threadIdx.x & (kWave - 1);
  const int wv = WPS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) : 0;
  const int g = lane >> 4;
  const int m16 = lane & 15;
  uint32_t* const stage = vst + wv * kVStage;           // this wave's V stage
  uint32_t* const kstage = KST ? vst + (WPS + wv) * kVStage : stage;  // its K stage

  const int rows = q_len * p.group;

  float kscale = 1.0f, vscale = 1.0f;
  if (FP8) {
    kscale = p.k_scale ? *p.k_scale : 1.0f;
    vscale = p.v_scale ? *p.v_scale : 1.0f;
  }
  const float sl2 = p.scale_log2 * kscale;

  // ---- query operands, loaded here and parked in LDS (in operand order:
  // entry (nt, s) is one 16-byte vector per lane, read back conflict-free
  // for every chunk so that they hold no registers across the loop) once
  // the first chunk's K/V loads are in flight; and the causal limits
  // Padding columns (n >= rows) load row 0 and are zeroed when parked, so
  // the loads are unconditional and nothing waits for them before the K/V
  // loads go out.
  int lim[NT];
  bf16x8_t qv[NT][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int n = nt * 16 + m16;
    const int nn = n < rows ? n : 0;
    const int j = nn / p.group, hh = nn % p.group;
    const uint16_t* qp = p.q + static_cast<int64_t>(q_start + j) * p.q_row_stride +
                         static_cast<int64_t>(kvh * p.group + hh) * p.q_head_stride;
#pragma unroll
    for (int s = 0; s < 4; ++s) qv[nt][s] = *reinterpret_cast<const bf16x8_t*>(qp + 32 * s + 8 * g);
    const int c = L - q_len + j;
    lim[nt] = n < rows ? (c < L - 1 ? c : L - 1) : -1;
  }

  float m_run[NT], l_run[NT];
  f32x4_t acc[NT][8];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m_run[nt] = -INFINITY;
    l_run[nt] = 0.0f;
#pragma unroll
    for (int t = 0; t < 8; ++t) acc[nt][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  const int nchunks = (kv_end - kv_begin + kChunk - 1) / kChunk;
  constexpr int64_t esz = FP8 ? 1 : 2;

  // lane i of lane_blk holds the id of logical block first_blk + i: one
  // load for the split instead of a dependent load per chunk
  const int first_blk = kv_begin / p.block_size;

  // Raw K/V registers of one 32-key chunk (bf16: K 2x4 and V 8 16-byte
  // vectors per lane; FP8: K 2x4 8-byte and V 4 16-byte vectors).
  struct Chunk {
    uint4 k[2][4];
    uint4 v[8];
    int kb;        // first key of the chunk
    bool valid;    // block id in range; otherwise the chunk's keys are masked
  };

  // Loop-invariant byte offsets of this lane's loads inside one (block, kv
  // head) tile of 32 tokens; a chunk only builds two buffer descriptors
  // (uniform), so no per-chunk address arithmetic runs on the vector ALUs.
  //   K: key (16*kt + m16), d 32*s + 8*g .. +7   (s through the immediate offset)
  //   V: bf16 row (4*i + g), d 8*m16 .. +7; FP8 row (8*i + lane/8), bytes 16*(lane%8)
  const uint32_t tokb = static_cast<uint32_t>(p.tok_stride * esz);
  uint32_t koff[2], voff[8];
#pragma unroll
  for (int kt = 0; kt < 2; ++kt) koff[kt] = (kt * 16 + m16) * tokb + 8 * g * esz;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    voff[i] = FP8 ? (8 * i + (lane >> 3)) * tokb + (lane & 7) * 16 : (4 * i + g) * tokb + m16 * 16;

  // Issue the loads of chunk c (no waits: the data is consumed by
  // compute_chunk one chunk later, so each load's latency overlaps the
  // previous chunk's math).  The descriptors' record count ends at the last
  // visible key, so rows past the sequence end (and every row of an invalid
  // block) read as zeros instead of stale cache contents.  V loads (whole
  // 128-byte lines per instruction) carry the non-temporal hint.  K loaded
  // straight into operand order reads half lines per instruction (the
  // other half one instruction later), where the hint costs time: measured
  // on the Qwen3-8B bench shapes, no hint 63.5 us per call, both 61.3, K
  // only 63.7, V only 59.3; FP8 config 4: 486 -> 442 us.  Staged K (KST)
  // loads as V does, whole lines with the hint: config 3 56.4 -> 55.2 us,
  // FP8 config 4 430.6 -> 414 us.  Issuing the next chunk's loads as soon
  // as the staging frees the registers (before this chunk's math) ran
  // slower, 55.2 -> 56.1 us: more requests in flight per CU, less DRAM
  // efficiency.
  auto load_chunk = [&](int c, Chunk& ch) {
    const int kb = kv_begin + c * kChunk;
    ch.kb = kb;
    // the host keeps a split within kWave blocks, so the id is always in a lane
    const int raw = __builtin_amdgcn_readlane(lane_blk, kb / p.block_size - first_blk);
    ch.valid = raw >= 0 && raw < p.num_blocks;
    const int pblk = ch.valid ? raw : 0;
    const int visible = L - kb < kChunk ? L - kb : kChunk;
    const int nrec = ch.valid ? visible * static_cast<int>(tokb) : 0;
    const int64_t tile = (static_cast<int64_t>(pblk) * p.blk_stride +
                          static_cast<int64_t>(kvh) * p.head_stride +
                          static_cast<int64_t>(kb % p.block_size) * p.tok_stride) * esz;
    const __amdgpu_buffer_rsrc_t kr = make_rsrc(p.k_cache + tile, nrec);
    const __amdgpu_buffer_rsrc_t vr = make_rsrc(p.v_cache + tile, nrec);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        if (KST && FP8) {
          // whole lines, as V: FP8 row 8 s + lane / 8, bytes 16 (lane % 8) .. +15
          if (kt == 0)
            ch.k[0][s] = __builtin_bit_cast(
                uint4, __builtin_amdgcn_raw_buffer_load_b128(kr, voff[s], 0, kLoadStreamed));
        } else if (FP8) {
          const uint2 w = __builtin_bit_cast(
              uint2,
              __builtin_amdgcn_raw_buffer_load_b64(kr, koff[kt] + 32 * s, 0, 0));
          ch.k[kt][s] = make_uint4(w.x, w.y, 0, 0);
        } else if (KST) {
          // whole lines, as V: row 4 (4 kt + s) + g, bytes 16 m16 .. +15
          ch.k[kt][s] = __builtin_bit_cast(
              uint4,
              __builtin_amdgcn_raw_buffer_load_b128(kr, voff[4 * kt + s], 0, kLoadStreamed));
        } else {
          ch.k[kt][s] = __builtin_bit_cast(
              uint4,
              __builtin_amdgcn_raw_buffer_load_b128(kr, koff[kt] + 64 * s, 0, 0));
        }
      }
    }
#pragma unroll
    for (int i = 0; i < (FP8 ? 4 : 8); ++i)
      ch.v[i] = __builtin_bit_cast(
          uint4, __builtin_amdgcn_raw_buffer_load_b128(vr, voff[i], 0, kLoadStreamed));
  };

  auto compute_chunk = [&](const Chunk& ch) {
    if (!ch.valid) return;
    const int kb = ch.kb;
    // ---- V rows into the wave's LDS stage.  The stage belongs to this wave
    // alone and LDS executes a wave's operations in order, so a compiler
    // barrier plus an LDS wait (before the first read) orders them.
    if (FP8) {
      // Lane l stages 16 values of row 8 i + l / 8 as two 16-byte halves
      // at dwords 8 (l % 8) and + 4.  A 16-byte LDS store serves eight
      // lanes per cycle over 32 four-byte banks, so if every lane stored
      // its first half first, lanes l and l + 4 would share a bank group
      // (2-way conflicts on every store).  Lanes 4-7 of each eight store
      // their second half first: each store's eight lanes then cover all
      // 32 banks.
      const bool swap = (lane >> 2) & 1;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = 8 * i + (lane >> 3);
        uint32_t* dst = stage + row * kVPitch + (lane & 7) * 8;
        const uint2 lo = make_uint2(ch.v[i].x, ch.v[i].y), hi = make_uint2(ch.v[i].z, ch.v[i].w);
        *reinterpret_cast<bf16x8_t*>(dst + (swap ? 4 : 0)) = fp8x8_to_bf16(swap ? hi : lo);
        *reinterpret_cast<bf16x8_t*>(dst + (swap ? 0 : 4)) = fp8x8_to_bf16(swap ? lo : hi);
      }
      if (KST) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = 8 * i + (lane >> 3);
          const int c0 = 2 * (lane & 7);
          const uint4 k = ch.k[0][i];
          const uint2 lo = make_uint2(k.x, k.y), hi = make_uint2(k.z, k.w);
          *reinterpret_cast<bf16x8_t*>(kstage + kst_slot(row, c0 + (swap ? 1 : 0))) =
              fp8x8_to_bf16(swap ? hi : lo);
          *reinterpret_cast<bf16x8_t*>(kstage + kst_slot(row, c0 + (swap ? 0 : 1))) =
              fp8x8_to_bf16(swap ? lo : hi);
        }
        lds_wave_sync();
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        *reinterpret_cast<uint4*>(stage + (4 * i + g) * kVPitch + m16 * 4) = ch.v[i];
      if (KST) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          *reinterpret_cast<uint4*>(kstage + kst_slot(4 * i + g, m16)) = ch.k[i / 4][i % 4];
        lds_wave_sync();
      }
    }

    // ---- S^T = K . Q^T: per head_dim slice s, every (key tile, query
    // tile) pair; the query operands come from LDS one slice at a time
    f32x4_t sacc[2][NT];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) sacc[kt][nt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      bf16x8_t kop[2];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        if (KST)  // key 16 kt + m16, head_dim 32 s + 8 g .. +7 (the Q operands' order)
          kop[kt] = *reinterpret_cast<const bf16x8_t*>(kstage + kst_slot(16 * kt + m16, 4 * s + g));
        else
          kop[kt] = FP8 ? fp8x8_to_bf16(make_uint2(ch.k[kt][s].x, ch.k[kt][s].y))
                        : __builtin_bit_cast(bf16x8_t, ch.k[kt][s]);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const bf16x8_t qo = qst[(nt * 4 + s) * kWave + lane];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) sacc[kt][nt] = mfma(kop[kt], qo, sacc[kt][nt]);
      }
    }

    // ---- online softmax (per query column; lanes l, l^16, l^32, l^48 share one).
    // Scores stay raw (the scale is folded into the exp2 argument); the
    // running max m_run (scaled, log2 domain) is only raised when a column's
    // new max exceeds it by more than kRescaleSlack, so the accumulator
    // rescale is skipped for most chunks: probabilities stay <= 2^kRescaleSlack.
    // Only a chunk that reaches past some column's causal limit (or the
    // sequence end) is masked, behind a uniform branch: written as a select
    // per score, the compare and select ran on every chunk (40 VALU
    // instructions of ~170 per chunk).
    const bool full = kb + kChunk - 1 <= L - q_len && kb + kChunk <= L;
    if (!full) {
      const int rel = kb + 4 * g;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (rel + kt * 16 + i > lim[nt]) sacc[kt][nt][i] = -INFINITY;
    }
    bf16x8_t pb[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float sv[8];
      float cmax = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = sacc[kt][nt][i];
          sv[kt * 4 + i] = v;
          cmax = fmaxf(cmax, v);
        }
      }
      cmax = max_xor16(cmax);
      cmax = max_xor32(cmax);
      cmax *= sl2;
      const bool need = cmax > m_run[nt] + kRescaleSlack;
      if (__any(need)) {
        const float m_new = need ? cmax : m_run[nt];
        const float alpha = need ? exp2f_fast(m_run[nt] - m_new) : 1.0f;
        l_run[nt] *= alpha;
        m_run[nt] = m_new;
#pragma unroll
        for (int t = 0; t < 8; ++t) {
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[nt][t][i] *= alpha;
        }
      }
      const float msub = m_run[nt] == -INFINITY ? 0.0f : m_run[nt];
      float psum = 0.0f;
      f32x2_t pv[4];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float e = exp2f_fast(__builtin_fmaf(sv[k], sl2, -msub));
        pv[k >> 1][k & 1] = e;
        psum += e;
      }
      l_run[nt] += psum;
      uint4 pk;
      pk.x = __builtin_bit_cast(uint32_t, __builtin_convertvector(pv[0], bf16x2_t));
      pk.y = __builtin_bit_cast(uint32_t, __builtin_convertvector(pv[1], bf16x2_t));
      pk.z = __builtin_bit_cast(uint32_t, __builtin_convertvector(pv[2], bf16x2_t));
      pk.w = __builtin_bit_cast(uint32_t, __builtin_convertvector(pv[3], bf16x2_t));
      pb[nt] = __builtin_bit_cast(bf16x8_t, pk);
    }

    lds_wave_sync();

    // ---- O^T += V^T . P^T ; pair pp covers d = 32*pp + 2*m + {0 (even tile), 1 (odd tile)}
#pragma unroll
    for (int pp = 0; pp < 4; ++pp) {
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = (j < 4) ? (4 * g + j) : (16 + 4 * g + (j - 4));
        w[j] = stage[key * kVPitch + 16 * pp + m16];
      }
      uint4 ev, od;
      ev.x = __builtin_amdgcn_perm(w[1], w[0], 0x05040100u);
      ev.y = __builtin_amdgcn_perm(w[3], w[2], 0x05040100u);
      ev.z = __builtin_amdgcn_perm(w[5], w[4], 0x05040100u);
      ev.w = __builtin_amdgcn_perm(w[7], w[6], 0x05040100u);
      od.x = __builtin_amdgcn_perm(w[1], w[0], 0x07060302u);
      od.y = __builtin_amdgcn_perm(w[3], w[2], 0x07060302u);
      od.z = __builtin_amdgcn_perm(w[5], w[4], 0x07060302u);
      od.w = __builtin_amdgcn_perm(w[7], w[6], 0x07060302u);
      const bf16x8_t ea = __builtin_bit_cast(bf16x8_t, ev);
      const bf16x8_t oa = __builtin_bit_cast(bf16x8_t, od);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        acc[nt][2 * pp] = mfma(ea, pb[nt], acc[nt][2 * pp]);
        acc[nt][2 * pp + 1] = mfma(oa, pb[nt], acc[nt][2 * pp + 1]);
      }
    }
    // the next chunk overwrites the stage: its reads must be done first
    lds_wave_sync();
  };

  // The wave's first chunk is requested before the query operands are
  // parked, so its latency overlaps the parking and the barrier (a barrier
  // waits for LDS operations only, not for outstanding loads).
  Chunk ca;
  if (PIPE || wv < nchunks) load_chunk(PIPE ? 0 : wv, ca);
  __builtin_amdgcn_sched_barrier(0);
  if (wv == 0) {
    const bf16x8_t zero = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int s = 0; s < 4; ++s) qst[(nt * 4 + s) * kWave + lane] = nt * 16 + m16 < rows ? qv[nt][s] : zero;
  }
  if constexpr (WPS > 1) __syncthreads(); else lds_wave_sync();

  // Two register buffers, unrolled by two so that no buffer is copied: the
  // loads of chunk c+1 are issued before chunk c is computed.  The
  // scheduling barriers keep the compiler from sinking them to their use.
  // Every load is unconditional (past the end the last chunk is loaded
  // again, from L2) so the compiler's wait counts only ever wait for the
  // older buffer.
  if constexpr (PIPE) {
    Chunk cb;
    const int last = nchunks - 1;
    int c = 0;
    for (; c < last; c += 2) {
      load_chunk(c + 1, cb);
      __builtin_amdgcn_sched_barrier(0);
      compute_chunk(ca);
      load_chunk(c + 2 < last ? c + 2 : last, ca);
      __builtin_amdgcn_sched_barrier(0);
      compute_chunk(cb);
    }
    if (c == last) compute_chunk(ca);
  } else {
    // one buffer: other resident waves on the SIMD hide the latency
    for (int c = wv; c < nchunks; c += WPS) {
      compute_chunk(ca);
      if (c + WPS < nchunks) load_chunk(c + WPS, ca);
    }
  }

  if constexpr (WPS > 1) {
    // ---- shared segment: every wave parks its (max, sum, accumulator)
    // state, half per column tile: tile 0 in its own V stage (free once its
    // loop is done), tile 1 in a second bank of WPS stages that no loop
    // touches, so no barrier is needed before parking.  After one barrier
    // the NT * 4 items (column tile nt, head_dim columns 32 pp .. 32 pp + 31)
    // are dealt to the waves in turn; each folds the WPS states of its item
    // in wave order (deterministic) and writes them straight from registers:
    // lane (g, m16) holds 8 consecutive values of query column m16.
    constexpr int kAccWords = 8 * kWave * 4;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float* mine = reinterpret_cast<float*>(vst + (nt * WPS + wv) * kVStage);
#pragma unroll
      for (int t = 0; t < 8; ++t) reinterpret_cast<f32x4_t*>(mine)[t * kWave + lane] = acc[nt][t];
      mine[kAccWords + lane] = m_run[nt];
      mine[kAccWords + kWave + lane] = l_run[nt];
    }
    __syncthreads();
    // NT * 4 (column tile, 32-wide head_dim group) items, one per wave
    // where there are enough waves
    for (int it = wv; it < NT * 4; it += WPS) {
      const int nt = it / 4, pp = it % 4;
      const float* st[WPS];
      float fw[WPS];
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < WPS; ++w) {
        st[w] = reinterpret_cast<const float*>(vst + (nt * WPS + w) * kVStage);
        fw[w] = st[w][kAccWords + lane];
        M = fmaxf(M, fw[w]);
      }
      float lsum = 0.0f;
#pragma unroll
      for (int w = 0; w < WPS; ++w) {
        fw[w] = fw[w] == -INFINITY ? 0.0f : exp2f_fast(fw[w] - M);
        lsum += fw[w] * st[w][kAccWords + kWave + lane];
      }
      lsum = sum_xor16(lsum);
      lsum = sum_xor32(lsum);
      const float inv = lsum > 0.0f ? vscale / lsum : 0.0f;
      const int n = nt * 16 + m16;
      if (n < rows) {
        const int j = n / p.group, hh = n % p.group;
        const int tok = q_start + j;
        const int h = kvh * p.group + hh;
        const int64_t slot = (static_cast<int64_t>(tok) * p.hq + h) * p.max_splits + split;
        // tiles 2 pp (even d) and 2 pp + 1 (odd d): d = 32 pp + 8 g + 2 i + e
        float o[8];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          f32x4_t sum = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int w = 0; w < WPS; ++w) {
            const f32x4_t a = reinterpret_cast<const f32x4_t*>(st[w])[(2 * pp + e) * kWave + lane];
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] += fw[w] * a[i];
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) o[2 * i + e] = sum[i] * inv;
        }
        const int d0 = 32 * pp + 8 * g;
        if (nsplit == 1) {
          uint16_t* op = p.out + static_cast<int64_t>(tok) * p.out_row_stride +
                         static_cast<int64_t>(h) * p.out_head_stride + d0;
          *reinterpret_cast<uint4*>(op) = make_uint4(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]),
                                                     pack_bf16(o[4], o[5]), pack_bf16(o[6], o[7]));
        } else {
          float* wo = p.ws_o + slot * kD + d0;
          *reinterpret_cast<float4*>(wo) = make_float4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<float4*>(wo + 4) = make_float4(o[4], o[5], o[6], o[7]);
          // log-sum-exp (log2 domain) of the column for combine_kernel
          if (pp == 0 && g == 0) p.ws_lse[slot] = part_lse(M, lsum);
        }
      }
    }
    return;
  }

  // ---- finish (one wave): per column sum, then straight from registers:
  // lane (g, m16) holds d = 32 pp + 8 g + 0..7 of query column m16 in the
  // tiles 2 pp (even d) and 2 pp + 1 (odd d)
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float lsum = l_run[nt];
    lsum = sum_xor16(lsum);
    lsum = sum_xor32(lsum);
    const float inv = lsum > 0.0f ? vscale / lsum : 0.0f;
    const int n = nt * 16 + m16;
    if (n < rows) {
      const int j = n / p.group, hh = n % p.group;
      const int tok = q_start + j;
      const int h = kvh * p.group + hh;
      const int64_t slot = (static_cast<int64_t>(tok) * p.hq + h) * p.max_splits + split;
#pragma unroll
      for (int pp = 0; pp < 4; ++pp) {
        float o[8];
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[2 * i + e] = acc[nt][2 * pp + e][i] * inv;
        const int d0 = 32 * pp + 8 * g;
        if (nsplit == 1) {
          uint16_t* op = p.out + static_cast<int64_t>(tok) * p.out_row_stride +
                         static_cast<int64_t>(h) * p.out_head_stride + d0;
          *reinterpret_cast<uint4*>(op) = make_uint4(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]),
                                                     pack_bf16(o[4], o[5]), pack_bf16(o[6], o[7]));
        } else {
          float* wo = p.ws_o + slot * kD + d0;
          *reinterpret_cast<float4*>(wo) = make_float4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<float4*>(wo + 4) = make_float4(o[4], o[5], o[6], o[7]);
        }
      }
      // log-sum-exp (log2 domain) of the column for combine_kernel
      if (nsplit > 1 && g == 0) p.ws_lse[slot] = part_lse(m_run[nt], lsum);
    }
  }
}

// ---------------------------------------------------------------- shared tiles

constexpr int kTileVPitch = 72;                          // dwords per staged V row (transpose loads)
constexpr int kTileSlot = kChunk * (kVPitch + kTileVPitch);  // dwords: K rows, then V rows

// One query tile of up to 64 rows (positions j0 .. j0 + jn - 1 of the sequence)
// against keys [kv_begin, kv_end), of which its last row sees those below
// kv_limit, on WPT waves that share each chunk through the two `slots`, D chunks
// in flight (bf16 caches; paged_attention.hip describes it).  The other
// arguments as for attend_segment.
template <int WPT, int D>
__device__ __forceinline__ void attend_tile(const AttnParams& p, uint32_t* slots, const int kvh,
                                            const int q_start, const int q_len, const int L,
                                            const int j0, const int jn, const int kv_limit,
                                            const int kv_begin, const int kv_end, const int split,
                                            const int nsplit, const int lane_blk) {
  constexpr int NTW = 4 / WPT;
  constexpr int kThreads = kWave * WPT;
  constexpr int kRowGran = kD * 2 / 16;                  // 16-byte granules per K or V row
  constexpr int kHalf = kChunk * kRowGran / kThreads;    // per thread per chunk, of K (and of V)
  constexpr int kSlot = kTileSlot;
  static_assert(WPT == 2 || WPT == 4, "two or four waves per 64-row tile");

  const int tid = threadIdx.x;
  const int lane = tid & (kWave - 1);
  const int wv = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int g = lane >> 4;
  const int m16 = lane & 15;
  const int rows = jn * p.group;
  const float sl2 = p.scale_log2;

  // ---- this wave's query operands (padding columns zero) and causal limits
  int lim[NTW];
  bf16x8_t qv[NTW][4];
#pragma unroll
  for (int nt = 0; nt < NTW; ++nt) {
    const int n = (wv * NTW + nt) * 16 + m16;
    const int nn = n < rows ? n : 0;
    const int j = j0 + nn / p.group, hh = nn % p.group;
    const uint16_t* qp = p.q + static_cast<int64_t>(q_start + j) * p.q_row_stride +
                         static_cast<int64_t>(kvh * p.group + hh) * p.q_head_stride;
#pragma unroll
    for (int s = 0; s < 4; ++s) qv[nt][s] = *reinterpret_cast<const bf16x8_t*>(qp + 32 * s + 8 * g);
    const int c = L - q_len + j;
    lim[nt] = n < rows ? (c < L - 1 ? c : L - 1) : -1;
  }

  const int nchunks = (kv_end - kv_begin + kChunk - 1) / kChunk;
  const int first_blk = kv_begin / p.block_size;
  const uint32_t tokb = static_cast<uint32_t>(p.tok_stride * 2);
  // granule i of this thread: row (tid + i * kThreads) / 16, column % 16
  uint32_t goff[kHalf], loff[kHalf], vloff[kHalf];
#pragma unroll
  for (int i = 0; i < kHalf; ++i) {
    const int gi = tid + i * kThreads;
    goff[i] = static_cast<uint32_t>(gi / kRowGran) * tokb + (gi % kRowGran) * 16;
    loff[i] = static_cast<uint32_t>(gi / kRowGran) * kVPitch + (gi % kRowGran) * 4;
    vloff[i] = static_cast<uint32_t>(gi / kRowGran) * kTileVPitch + (gi % kRowGran) * 4;
  }

  // chunk c's block id (uniform), in range or not
  auto chunk_block = [&](int c) {
    const int kb = kv_begin + c * kChunk;
    return __builtin_amdgcn_readlane(lane_blk, kb / p.block_size - first_blk);
  };
  auto load_chunk = [&](int c, uint4 (&r)[2 * kHalf]) {
    const bool live = c < nchunks;
    const int cc = live ? c : nchunks - 1;
    const int kb = kv_begin + cc * kChunk;
    const int raw = chunk_block(cc);
    const bool valid = live && raw >= 0 && raw < p.num_blocks;
    const int visible = kv_limit - kb < kChunk ? kv_limit - kb : kChunk;
    const int nrec = valid ? visible * static_cast<int>(tokb) : 0;
    const int64_t tile = (static_cast<int64_t>(valid ? raw : 0) * p.blk_stride +
                          static_cast<int64_t>(kvh) * p.head_stride +
                          static_cast<int64_t>(kb % p.block_size) * p.tok_stride) * 2;
    const __amdgpu_buffer_rsrc_t kr = make_rsrc(p.k_cache + tile, nrec);
    const __amdgpu_buffer_rsrc_t vr = make_rsrc(p.v_cache + tile, nrec);
#pragma unroll
    for (int i = 0; i < kHalf; ++i)
      r[i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(kr, goff[i], 0,
                                                                             kLoadStreamed));
#pragma unroll
    for (int i = 0; i < kHalf; ++i)
      r[kHalf + i] = __builtin_bit_cast(
          uint4, __builtin_amdgcn_raw_buffer_load_b128(vr, goff[i], 0, kLoadStreamed));
  };
  auto stage = [&](const uint4 (&r)[2 * kHalf], int slot) {
    uint32_t* kst = slots + slot * kSlot;
#pragma unroll
    for (int i = 0; i < kHalf; ++i) *reinterpret_cast<uint4*>(kst + loff[i]) = r[i];
#pragma unroll
    for (int i = 0; i < kHalf; ++i)
      *reinterpret_cast<uint4*>(kst + kChunk * kVPitch + vloff[i]) = r[kHalf + i];
  };

  float m_run[NTW], l_run[NTW];
  f32x4_t acc[NTW][8];
#pragma unroll
  for (int nt = 0; nt < NTW; ++nt) {
    m_run[nt] = -INFINITY;
    l_run[nt] = 0.0f;
#pragma unroll
    for (int t = 0; t < 8; ++t) acc[nt][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

  auto compute = [&](int c, int slot) {
    const int raw = chunk_block(c);
    if (raw < 0 || raw >= p.num_blocks) return;       // invalid block: its keys are masked
    const int kb = kv_begin + c * kChunk;
    const uint32_t* kst = slots + slot * kSlot;
    const uint32_t* vst = kst + kChunk * kVPitch;
    f32x4_t sacc[2][NTW];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int nt = 0; nt < NTW; ++nt) sacc[kt][nt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      bf16x8_t kop[2];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
        kop[kt] = *reinterpret_cast<const bf16x8_t*>(kst + (16 * kt + m16) * kVPitch + 16 * s + 4 * g);
#pragma unroll
      for (int nt = 0; nt < NTW; ++nt)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) sacc[kt][nt] = mfma(kop[kt], qv[nt][s], sacc[kt][nt]);
    }
    // masked only past a causal limit, behind a uniform branch (as above)
    const bool full = kb + kChunk - 1 <= L - q_len + j0 && kb + kChunk <= kv_limit;
    if (!full) {
      const int rel = kb + 4 * g;
#pragma unroll
      for (int nt = 0; nt < NTW; ++nt)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (rel + kt * 16 + i > lim[nt]) sacc[kt][nt][i] = -INFINITY;
    }
    bf16x8_t pb[NTW];
#pragma unroll
    for (int nt = 0; nt < NTW; ++nt) {
      float sv[8];
      float cmax = -INFINITY;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = sacc[kt][nt][i];
          sv[kt * 4 + i] = v;
          cmax = fmaxf(cmax, v);
        }
      }
      cmax = max_xor16(cmax);
      cmax = max_xor32(cmax);
      cmax *= sl2;
      const bool need = cmax > m_run[nt] + kRescaleSlack;
      if (__any(need)) {
        const float m_new = need ? cmax : m_run[nt];
        const float alpha = need ? exp2f_fast(m_run[nt] - m_new) : 1.0f;
        l_run[nt] *= alpha;
        m_run[nt] = m_new;
#pragma unroll
        for (int t = 0; t < 8; ++t) {
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[nt][t][i] *= alpha;
        }
      }
      const float msub = m_run[nt] == -INFINITY ? 0.0f : m_run[nt];
      float psum = 0.0f;
      f32x2_t pv[4];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float e = exp2f_fast(__builtin_fmaf(sv[k], sl2, -msub));
        pv[k >> 1][k & 1] = e;
        psum += e;
      }
      l_run[nt] += psum;
      uint4 pk;
      pk.x = __builtin_bit_cast(uint32_t, __builtin_convertvector(pv[0], bf16x2_t));
      pk.y = __builtin_bit_cast(uint32_t, __builtin_convertvector(pv[1], bf16x2_t));
      pk.z = __builtin_bit_cast(uint32_t, __builtin_convertvector(pv[2], bf16x2_t));
      pk.w = __builtin_bit_cast(uint32_t, __builtin_convertvector(pv[3], bf16x2_t));
      pb[nt] = __builtin_bit_cast(bf16x8_t, pk);
    }
    // O^T += V^T . P^T through the LDS transpose load (v_operand_tr): tile
    // (pp, hf) covers d = 32 pp + 8 (m / 4) + 4 hf + m % 4.  Against four
    // 4-byte reads and eight byte permutes per tile pair (the one-wave
    // segments' form), this removes 32 of the chunk's ~87 VALU instructions
    // per wave: config 5 417 -> 407 us per call, output bits unchanged.
#pragma unroll
    for (int pp = 0; pp < 4; ++pp) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const bf16x8_t va = v_operand_tr(vst, kTileVPitch, lane, pp, hf);
#pragma unroll
        for (int nt = 0; nt < NTW; ++nt) acc[nt][2 * pp + hf] = mfma(va, pb[nt], acc[nt][2 * pp + hf]);
      }
    }
  };

  // ---- D chunks in flight in registers, two LDS slots: step c computes
  // chunk c from slot c & 1, stages chunk c + 1 (loaded D steps ago) into
  // the other slot, refills its registers with chunk c + 1 + D, and one
  // barrier publishes the staged chunk and frees slot c & 1.
  uint4 buf[D][2 * kHalf];
#pragma unroll
  for (int d = 0; d < D; ++d) load_chunk(d, buf[d]);
  stage(buf[0], 0);
  load_chunk(D, buf[0]);
  __syncthreads();
  for (int cb = 0; cb < nchunks; cb += D) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int c = cb + d;
      if (c < nchunks) compute(c, c & 1);
      const int nb = (d + 1) % D;          // a constant once the loop is unrolled
      stage(buf[nb], (c + 1) & 1);
      load_chunk(c + 1 + D, buf[nb]);
      __syncthreads();
    }
  }

  // ---- finish: this wave's columns, straight from registers (lane (g, m16)
  // holds d = 32 pp + 8 g + 0..7 of query column m16: d .. d + 3 in tile
  // 2 pp, d + 4 .. d + 7 in tile 2 pp + 1)
#pragma unroll
  for (int nt = 0; nt < NTW; ++nt) {
    float lsum = l_run[nt];
    lsum = sum_xor16(lsum);
    lsum = sum_xor32(lsum);
    const float inv = lsum > 0.0f ? 1.0f / lsum : 0.0f;
    const int n = (wv * NTW + nt) * 16 + m16;
    if (n < rows) {
      const int j = j0 + n / p.group, hh = n % p.group;
      const int tok = q_start + j;
      const int h = kvh * p.group + hh;
      const int64_t slot = (static_cast<int64_t>(tok) * p.hq + h) * p.max_splits + split;
#pragma unroll
      for (int pp = 0; pp < 4; ++pp) {
        float o[8];
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[4 * e + i] = acc[nt][2 * pp + e][i] * inv;
        const int d0 = 32 * pp + 8 * g;
        if (nsplit == 1) {
          uint16_t* op = p.out + static_cast<int64_t>(tok) * p.out_row_stride +
                         static_cast<int64_t>(h) * p.out_head_stride + d0;
          *reinterpret_cast<uint4*>(op) = make_uint4(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]),
                                                     pack_bf16(o[4], o[5]), pack_bf16(o[6], o[7]));
        } else {
          float* wo = p.ws_o + slot * kD + d0;
          *reinterpret_cast<float4*>(wo) = make_float4(o[0], o[1], o[2], o[3]);
          *reinterpret_cast<float4*>(wo + 4) = make_float4(o[4], o[5], o[6], o[7]);
        }
      }
      if (nsplit > 1 && g == 0) p.ws_lse[slot] = part_lse(m_run[nt], lsum);
    }
  }
}

// ---------------------------------------------------------------- joining parts

// Elements 4 d4 .. 4 d4 + 3 of a row and head's output from its `parts` parts (the
// first at slot `base`): sum w o / sum w with w = exp2(lse - max lse), kJoinBatch
// loads at a time folded into a running maximum, weight and sum.  Parts without a
// visible key have no weight; without any the row is zero.  A NaN part makes the
// row NaN, whatever the others hold: the maximum passes over it, its weight is NaN.
constexpr int kJoinBatch = 8;
__device__ __forceinline__ float4 join_parts(const AttnParams& p, int64_t base, int parts, int d4) {
  float M = -INFINITY, wsum = 0.0f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < parts; s0 += kJoinBatch) {
    float lse[kJoinBatch];
    float4 v[kJoinBatch];
#pragma unroll
    for (int u = 0; u < kJoinBatch; ++u) {
      const bool in = s0 + u < parts;
      lse[u] = in ? p.ws_lse[base + s0 + u] : -INFINITY;
      v[u] = in ? *reinterpret_cast<const float4*>(p.ws_o + (base + s0 + u) * kD + 4 * d4)
                : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float mb = M;
#pragma unroll
    for (int u = 0; u < kJoinBatch; ++u) mb = fmaxf(mb, lse[u]);
    const float msub = mb == -INFINITY ? 0.0f : mb;
    const float r = M == -INFINITY ? 0.0f : exp2f_fast(M - msub);
    wsum *= r;
    o.x *= r; o.y *= r; o.z *= r; o.w *= r;
#pragma unroll
    for (int u = 0; u < kJoinBatch; ++u) {
      if (lse[u] == -INFINITY) v[u] = make_float4(0.f, 0.f, 0.f, 0.f);   // whatever is there
      const float w = lse[u] == -INFINITY ? 0.0f : exp2f_fast(lse[u] - msub);
      wsum += w;
      o.x += w * v[u].x; o.y += w * v[u].y; o.z += w * v[u].z; o.w += w * v[u].w;
    }
    M = mb;
  }
  const float inv = wsum == 0.0f ? 0.0f : 1.0f / wsum;
  return make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

// ---------------------------------------------------------------- 32-row waves

typedef __attribute__((ext_vector_type(16))) float f32x16_t;
constexpr int kWideKeys = 64;
constexpr int kWideKPitch = 68, kWideVPitch = 80;   // dwords per staged row
constexpr int kWideBuf = kWideKeys * (kWideKPitch + kWideVPitch);

__device__ __forceinline__ f32x16_t mfma32(bf16x8_t a, bf16x8_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// V^T operand of head_dim tile dt (d = 32 dt + lane % 32) and key slice t
// (16 keys) from staged rows: transpose load r (0, 1) hands lane 32 h + c the
// keys 16 t + 8 r + 4 h .. + 3 (see v_operand_tr for the instruction).
__device__ __forceinline__ bf16x8_t wide_v_operand(const uint32_t* rows, int lane, int t, int dt) {
  const int h = lane >> 5, dh = (lane >> 4) & 1, i = lane & 15;
  uint32_t* p0 = const_cast<uint32_t*>(rows) + (16 * t + 4 * h + (i >> 2)) * kWideVPitch + 16 * dt +
                 8 * dh + 2 * (i & 3);
  const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(p0));
  const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(p0 + 8 * kWideVPitch));
  return bf16x8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

}  // namespace
}  // namespace nva

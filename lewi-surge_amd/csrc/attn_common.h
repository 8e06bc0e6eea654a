// Device helpers of the softmax attention kernels (attn.hip, attn_decode.hip): 16-bit matrix-core products, the LDS tile
// layout and its copies, and the lookup of a packed sequence's tiles.
#pragma once
#include "gemm_kernels.h"

namespace lsattn {

using lsgemm::copy16;
using lsgemm::lds_addr;
using lsgemm::make_rsrc;
using lsgemm::stage_barrier;
using lsgemm::u32x2;

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// Products of the 16-bit type DT (LSURGE_BF16 or LSURGE_F16) with f32 sums.  mma32: D[32 x 32] += P[32 x 16] Q[16 x 32];
// lane l supplies row l % 32 of P and column l % 32 of Q at k = 8 (l / 32) .. + 7 and holds
// D[8 (r / 4) + 4 (l / 32) + r % 4][l % 32] in register r.  mma16: D[16 x 16] += P[16 x 32] Q[32 x 16]; lane l supplies
// row / column l % 16 at k = 8 (l / 16) .. + 7 and holds D[4 (l / 16) + r][l % 16].
template <int DT>
__device__ __forceinline__ f32x16 mma32(u32x4 p, u32x4 q, f32x16 c) {
  if constexpr (DT == LSURGE_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, p), __builtin_bit_cast(f16x8, q), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, p), __builtin_bit_cast(bf16x8, q), c, 0, 0, 0);
}
template <int DT>
__device__ __forceinline__ f32x4 mma16(u32x4 p, u32x4 q, f32x4 c) {
  if constexpr (DT == LSURGE_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, p), __builtin_bit_cast(f16x8, q), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, p), __builtin_bit_cast(bf16x8, q), c, 0, 0, 0);
}
// two f32 -> two values of DT in one register, rounded to nearest even
template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (DT == LSURGE_F16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){lo, hi}, f16x2_t));
  else
    return pack_bf16x2(lo, hi);
}
template <int DT>
__device__ __forceinline__ void unpack2(uint32_t v, float& lo, float& hi) {
  if constexpr (DT == LSURGE_F16) {
    lo = f16_to_f32((uint16_t)v);
    hi = f16_to_f32((uint16_t)(v >> 16));
  } else {
    lo = __uint_as_float(v << 16);
    hi = __uint_as_float(v & 0xffff0000u);
  }
}

// the sum of a register's two values, added to c
template <int DT>
__device__ __forceinline__ float add2(uint32_t v, float c) {
  if constexpr (DT == LSURGE_F16)
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, v), f16x2_t{(_Float16)1, (_Float16)1}, c, false);
  else
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, v), __builtin_bit_cast(bf16x2_t, 0x3f803f80u), c,
                                           false);
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// a value's partner in the other half of the wave (lane ^ 32), combined with op; both halves get the result
template <class Op>
__device__ __forceinline__ float halves(float x, Op&& op) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return op(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// ------------------------------------------------------------------------------------ LDS tiles
// A tile holds rows of D 16-bit values, row-major, its 16-byte chunks permuted within a row: logical chunk c of row r
// lies at chunk c ^ swz(r).  Both kinds of read are then free of bank conflicts.  A row read (ds_read_b128: 16 rows at
// one chunk) needs 16 different places among the 16 chunks that fill the banks once: swz is one-to-one on 16 rows (for
// D = 64, whose row fills half of the banks, on 8 row pairs).  A transpose read (ds_read_b64_tr_b16: 4 consecutive rows,
// 4 aligned chunks of each) needs the rows in different groups of 4 chunks: the low row bits go to the upper bits.
template <int D>
__device__ __forceinline__ int swz(int r) {
  if constexpr (D == 64) return ((r >> 1 & 1) << 2) | (r >> 2 & 3);
  else return ((r & 3) << 2) | (r >> 2 & 3);
}

// Copies of a ROWS x D tile by NW waves straight into LDS, 1 KiB each: copy c fills chunks 64 c .. + 63.
template <int D, int ROWS, int NW>
struct TileCopy {
  static constexpr int CPR = D / 8;                       // chunks per row
  static constexpr int N = ROWS * CPR / 64 / NW;          // copies per wave
  static_assert(N * 64 * NW == ROWS * CPR, "whole copies");
  uint32_t off[N];  // this lane's byte offset in the source for each copy
  __device__ __forceinline__ void init(int64_t row_stride, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = (wave * N + i) * 64 + lane, row = id / CPR, pc = id % CPR;
      off[i] = (uint32_t)(row * (int)row_stride * 2 + ((pc ^ swz<D>(row)) * 16));
    }
  }
  // rows [0, rows) of the tile that starts at `base`; the others are filled with zeros
  __device__ __forceinline__ void issue(const uint16_t* base, int64_t row_stride, int rows, uint32_t lds, int wave) const {
    const int n = min(rows, ROWS);
    const u32x4 rs = make_rsrc(base, n > 0 ? (int64_t)(n - 1) * row_stride * 2 + D * 2 : 0);
#pragma unroll
    for (int i = 0; i < N; ++i) copy16(rs, off[i], lds + (wave * N + i) * 1024);
  }
};

// 64 consecutive 4-byte values, lane p's at LDS byte address m0 + 4 p
__device__ __forceinline__ void copy4(u32x4 rsrc, uint32_t byte_off, uint32_t m0) {
  const uint32_t m0s = (uint32_t)__builtin_amdgcn_readfirstlane(m0);
  asm volatile("s_mov_b32 m0, %2\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(byte_off), "s"(rsrc), "s"(m0s)
               : "memory");
}

// Fragment addresses of a tile at LDS byte address `base` (a multiple of 1024).
// rows: lane l holds row r0 + l % 32 at k = 16 s + 8 (l / 32) .. + 7, read from row_step(row_addr, s), r0 a multiple of 32
// (the swizzle reaches the low 4 bits of a chunk's number, so at D = 256 the upper half of a row is a constant away)
template <int D>
__device__ __forceinline__ uint32_t row_addr(int lane) {
  const int r = lane & 31;
  return (uint32_t)(r * D * 2 + (((lane >> 5) ^ swz<D>(r)) << 4));
}
template <int D>
__device__ __forceinline__ uint32_t row_step(uint32_t a, int s) { return (a ^ ((s & 7) * 32)) + (s >> 3) * 256; }
typedef const __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
__device__ __forceinline__ u32x4 lds_read16(uint32_t a) { return *(lds_u32x4*)(uintptr_t)a; }
// columns: lane l holds column m0 + l % 32 (m0 = 32 dt) at the 8 rows k0 + 4 (l / 32) + {0..3, 8..11}, k0 a multiple of
// 16: the rows whose scores lane l holds in 8 consecutive registers of a 32 x 32 product, so a product's result is
// the next product's operand without leaving its lane
template <int D>
__device__ __forceinline__ uint32_t col_addr(int lane, int dt) {
  const int g = lane >> 4, s = lane & 15;
  const int r = 4 * (g >> 1) + (s >> 2), c = 32 * dt + 16 * (g & 1) + 4 * (s & 3);
  return (uint32_t)(r * D * 2 + (((c >> 3) ^ swz<D>(r)) << 4) + (c & 7) * 2);
}
template <int D> constexpr int COLS = D / 32 < 4 ? D / 32 : 4;
// col_addr of all dt from those of dt < min(D / 32, 4)
template <int D>
__device__ __forceinline__ uint32_t col_step(const uint32_t* a, int dt) { return a[dt & 3] + (dt >> 2) * 256; }
// r + 8 has another swizzle than r: bit 1 of row / 4 flips, so chunk bit 1 does
template <int D>
__device__ __forceinline__ u32x4 lds_read_col(uint32_t a) {
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)a);
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)((a ^ 32u) + 8 * D * 2));
  typedef short s16x8 __attribute__((ext_vector_type(8)));
  const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  return __builtin_bit_cast(u32x4, v);
}

// ------------------------------------------------------------------------------------ packed sequences
// Sequence s holds rows [cu[s], cu[s + 1]) (cu ascending from 0), or, without cu, total / nseq rows each.  Entries are
// held to [0, total], so that no table makes a kernel read or write outside its rows.
__device__ __forceinline__ int cu_at(const int32_t* cu, int i, int total) { return min(max(cu[i], 0), total); }

// Tile t of the rows.  Up to 63 sequences: the tiles in a row, the largest of a sequence first, and what a launch has more
// of slots comes last; all ends are read at once, one trip to memory.  From 64 on sequence s owns the tiles from
// cu[s] / B + s, which leaves it at least ceil(rows / B), and is found by a 64-way search (with few sequences too: 24 prompts
// 182 us against 176 so, 3 prompts after 20000 keys 225 and 209, 24 prompts of 1024 146 and 149).  Tiles of all sequences by
// size, in phases of an octave of keys or half one, were no faster: 179 to 188, 204, 151 to 159.  Dense: tile t of sequence
// `seq`.
constexpr int IN_A_ROW = 64;  // fewer sequences than this
struct Place {
  int seq, tile;          // sequence (-1: none) and its tile
  int q0, nq, k0, nk;     // its rows
  int64_t end;            // the first row behind the last sequence
};
// sums over the lanes up to each
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // the lane 1, 2, 4, 8 before it in a row of 16
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // the last lane of row 0 to 1, of 2 to 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // of row 1 to 2 and 3
  return v;
}
template <int B, bool KEYS>  // tiles of the keys, or of the queries
__device__ __forceinline__ Place find_tile(const int32_t* cu_q, const int32_t* cu_k, int nseq, int total_q, int total_k,
                                           int seq, int t, int lane) {
  Place p;
  p.seq = -1;
  p.tile = p.q0 = p.nq = p.k0 = p.nk = 0;
  if (!cu_q) {
    p.nq = total_q / nseq, p.nk = total_k / nseq;
    p.end = KEYS ? total_k : total_q;
    p.seq = seq, p.tile = t;
    p.q0 = seq * p.nq, p.k0 = seq * p.nk;
    return p;
  }
  const int32_t* cu = KEYS ? cu_k : cu_q;
  const int total = KEYS ? total_k : total_q;
  int q1, k1;
  if (nseq < IN_A_ROW) {
    const int i = min(lane, nseq), j = min(lane + 1, nseq);
    const int eq = cu_at(cu_q, i, total_q), fq = cu_at(cu_q, j, total_q);
    const int ek = cu_at(cu_k, i, total_k), fk = cu_at(cu_k, j, total_k);
    p.end = __builtin_amdgcn_readlane(KEYS ? ek : eq, nseq);
    const int nt = (max(0, KEYS ? fk - ek : fq - eq) + B - 1) / B;  // 0 from lane nseq on
    const int upto = wave_scan(nt);
    const int s = __popcll(__ballot(upto <= t));
    if (s >= nseq) return p;
    p.seq = s;
    const int rest = __builtin_amdgcn_readlane(upto, s) - t;  // tiles from this one on
    p.tile = KEYS ? __builtin_amdgcn_readlane(nt, s) - rest : rest - 1;
    p.q0 = __builtin_amdgcn_readlane(eq, s), q1 = __builtin_amdgcn_readlane(fq, s);
    p.k0 = __builtin_amdgcn_readlane(ek, s), k1 = __builtin_amdgcn_readlane(fk, s);
  } else {
    p.end = cu_at(cu, nseq, total);
    int lo = 0, n = nseq;
    while (true) {
      const int step = (n + 63) / 64, i = lo + lane * step;
      const int c = __popcll(__ballot(lane * step < n && cu_at(cu, i, total) / B + i <= t));
      if (c == 0) return p;
      n = min(step, n - (c - 1) * step);
      lo += (c - 1) * step;
      if (step == 1) break;
    }
    p.seq = lo = __builtin_amdgcn_readfirstlane(lo);
    p.tile = t - (cu_at(cu, lo, total) / B + lo);
    p.q0 = cu_at(cu_q, lo, total_q), q1 = cu_at(cu_q, lo + 1, total_q);
    p.k0 = cu_at(cu_k, lo, total_k), k1 = cu_at(cu_k, lo + 1, total_k);
    p.tile = __builtin_amdgcn_readfirstlane(p.tile);
    p.q0 = __builtin_amdgcn_readfirstlane(p.q0), p.k0 = __builtin_amdgcn_readfirstlane(p.k0);
    q1 = __builtin_amdgcn_readfirstlane(q1), k1 = __builtin_amdgcn_readfirstlane(k1);
  }
  p.nq = max(0, q1 - p.q0), p.nk = max(0, k1 - p.k0);
  if (p.tile < 0) p.seq = -1;  // ends out of order
  return p;
}

}  // namespace lsattn

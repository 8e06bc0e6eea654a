// Device helpers of the kernels that walk packed rows of 16-bit values: eight values to and from f32, and the sequence that
// holds a row.
#pragma once
#include "common.h"

namespace lsrows {

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

template <int DT>
__device__ __forceinline__ void unpack8(u32x4 v, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == LSURGE_F16) {
      f[2 * i] = f16_to_f32((uint16_t)v[i]);
      f[2 * i + 1] = f16_to_f32((uint16_t)(v[i] >> 16));
    } else {
      f[2 * i] = __uint_as_float(v[i] << 16);
      f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    }
  }
}
template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (DT == LSURGE_F16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){lo, hi}, f16x2_t));
  else
    return pack_bf16x2(lo, hi);
}
template <int DT>
__device__ __forceinline__ u32x4 pack8(const float* f) {
  return u32x4{pack2<DT>(f[0], f[1]), pack2<DT>(f[2], f[3]), pack2<DT>(f[4], f[5]), pack2<DT>(f[6], f[7])};
}

// The sequence of a packed row: s holds the rows [cu[s], cu[s + 1]), cu ascending from 0; without cu one row each.  Entries
// are held to [0, rows], so that no table leads out of the rows.  seq < 0: the row belongs to none.
struct Seq {
  int seq, begin, end;
};
__device__ __forceinline__ int end_at(const int32_t* cu, int i, int rows) { return min(max(cu[i], 0), rows); }
// The last sequence that starts at or before a row that all 64 lanes of the wave ask for: one trip to memory for up to 64
// sequences, two for up to 4096.  0 where none does.
__device__ __forceinline__ int find_seq(const int32_t* cu, int nseq, int row, int lane) {
  int lo = 0, n = nseq;
  while (n > 1) {
    const int step = (n + 63) / 64;
    const int c = __popcll(__ballot(lane * step < n && cu[lo + min(lane * step, n - 1)] <= row));
    if (c == 0) return 0;
    n = min(step, n - (c - 1) * step);
    lo += (c - 1) * step;
  }
  return lo;
}
// The sequence of a row, looked for from sequence `s` on, which starts no later.
__device__ __forceinline__ Seq seq_from(const int32_t* cu, int nseq, int rows, int row, int s) {
  if (!cu) return {row, row, row + 1};
  if (nseq < 1) return {-1, row, row + 1};
  int begin = end_at(cu, s, rows), end = end_at(cu, s + 1, rows);
  while (end <= row && s + 1 < nseq) {
    ++s;
    begin = end;
    end = end_at(cu, s + 1, rows);
  }
  return begin <= row && row < end ? Seq{s, begin, end} : Seq{-1, row, row + 1};
}

}  // namespace lsrows

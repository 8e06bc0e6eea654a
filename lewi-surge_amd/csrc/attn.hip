// Causal softmax attention of packed or dense sequences with grouped heads, forward and backward, on the matrix cores.
//
// Query i of a sequence with nq queries and nk keys attends to the keys j <= i + nk - nq (the queries are the last ones):
//   s_ij = scale q_i . k_j,  o_i = sum_j e^(s_ij - lse_i) v_j,  lse_i = log sum_j e^(s_ij)
// and o_i = 0, lse_i = -inf for a query with no key.  Scores and sums are f32, in base 2 (the scale carries log2 e); the
// weights are rounded to the operands' type for the second product, as its operands have to be (half a step of the type,
// relative to each weight, so that errors average out over the keys).
//
// Every product is formed transposed: S^T = K Q^T has a query per lane (column l % 32), so a row's maximum and sum are
// sums over a lane's own registers and one exchange with lane ^ 32, the accumulators O^T = V^T P^T have the same query in
// the same lane, and P^T is in place as the second product's operand (the keys of 8 consecutive registers are the ones
// its fragment takes, in an order that V^T's fragment is read in as well).  No value crosses lanes on the way.
#include <algorithm>

#include "attn_common.h"
#include "launchers.h"

namespace lsattn {
namespace {

struct AttnArgs {
  const uint16_t *q, *k, *v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;  // strides in elements
  const int32_t *cu_q, *cu_k;
  int nseq, total_q, total_k, hq, hk;
  float scale2;  // scale log2(e)
  // the launch (see head_tile): heads of a sequence, their pairs with the sequences, pairs of an XCD (0: not cut into
  // runs), heads that go together, tiles of a sequence
  int heads, pairs, run, together, tiles;
};

// Workgroup -> (sequence, head, tile).  Workgroups are dealt to the 8 XCDs round-robin and each XCD has an L2 of its own, so
// the (sequence, head) pairs are cut into 8 runs where their number allows, and within a run `together` heads that read the
// same rows go tile by tile: the workgroups that run on an XCD at a time then walk the same keys.  8 x 4096 tokens, 8 heads
// over 2: 1530 us a training step with heads dealt to XCDs, 1441 so; 8 x 2048 prompts, 16 heads: 172 and 161.  Where an XCD
// has few workgroups (two rounds) all its heads go together, so that the longest start first (one sequence of 4096: 356 and
// 328 us).  Packed sequences have their borders on the device: their tile slots are one sequence here.  Tiles go from the
// last to the first (the long ones of a causal sequence first) or, with `up`, the other way.
__device__ __forceinline__ void head_tile(const AttnArgs& a, bool up, int& seq, int& head, int& tile) {
  const int id = (int)blockIdx.x;
  int pair;
  if (a.run) {
    const int i = id / 8, set = i / (a.together * a.tiles), r = i - set * a.together * a.tiles;
    tile = r / a.together;
    pair = id % 8 * a.run + set * a.together + r - tile * a.together;
  } else {
    tile = id / a.pairs;
    pair = id - tile * a.pairs;
  }
  seq = pair / a.heads;
  head = pair - seq * a.heads;
  if (!up) tile = a.tiles - 1 - tile;
}

// rows [first, first + n) of [rows, heads, D] at one head, zeroed (rows behind the last sequence)
template <int D>
__device__ __forceinline__ void zero_rows(uint16_t* p, int64_t first, int n, int heads, int head, int tid, int nthr) {
  for (int i = tid; i < n * (D / 8); i += nthr)
    *reinterpret_cast<u32x4*>(p + ((first + i / (D / 8)) * heads + head) * D + i % (D / 8) * 8) = u32x4{0, 0, 0, 0};
}

// Issue orders for the compiler's scheduler.  feed: MFMAS products that take READS LDS reads each, AHEAD reads issued
// before the first, the others spread between the products.
enum { SG_VALU = 0x2, SG_MFMA = 0x8, SG_DS_R = 0x100, SG_TRANS = 0x400 };
template <int MFMAS, int READS, int AHEAD>
__device__ __forceinline__ void feed() {
  __builtin_amdgcn_sched_group_barrier(SG_DS_R, AHEAD, 0);
#pragma unroll
  for (int i = 0; i < MFMAS; ++i) {
    __builtin_amdgcn_sched_group_barrier(SG_MFMA, 1, 0);
    if (i < MFMAS - AHEAD / READS) __builtin_amdgcn_sched_group_barrier(SG_DS_R, READS, 0);
  }
}
// interleave: MFMAS products of one LDS read each (AHEAD reads first) with a softmax's arithmetic between them
template <int MFMAS, int AHEAD>
__device__ __forceinline__ void interleave() {
  __builtin_amdgcn_sched_group_barrier(SG_DS_R, AHEAD, 0);
#pragma unroll
  for (int i = 0; i < MFMAS; ++i) {
    __builtin_amdgcn_sched_group_barrier(SG_MFMA, 1, 0);
    if (i < MFMAS - AHEAD) __builtin_amdgcn_sched_group_barrier(SG_DS_R, 1, 0);
    __builtin_amdgcn_sched_group_barrier(SG_VALU, (64 + MFMAS - 1) / MFMAS, 0);
    if (i >= MFMAS / 4) __builtin_amdgcn_sched_group_barrier(SG_TRANS, (24 + MFMAS - 1) / MFMAS, 0);
  }
}

// ------------------------------------------------------------------------------------ forward
constexpr int FN = 32;  // keys per stage of the forward
// its stages in LDS; at D = 256 a fourth made prompts of 16384 slower (2385 -> 2779 us: the unrolled loop's code grows)
template <int D> constexpr int STAGES = D == 256 ? 3 : 4;
constexpr int BN = 64;  // keys per stage of the pass over queries

constexpr float LAZY = 8.f;  // log2 of the growth of a row's largest weight that the base lets pass
// log2 of the f16 weights' room above that: one below 2^-25 of the largest would be none, though thousands of them may hold a
// share of the row that counts, so the base is taken lower, and the sums have the factor too.  4 is a constant that the fma
// takes, so it costs nothing (7: an instruction and 1%, or a register, which undoes the loop's schedule, and 7%).  Weights are
// off by 2^-29 of the largest at most, 2^18 of them by half of f16's step, and stay in its range up to scores of 2^26 (base 2,
// with an f32 step of 4).
constexpr float LIFT = 4.f;

// acc *= f.  At D = 256 the accumulators fill half of the registers and have to stay in the accumulation file, which the
// vector unit cannot work on: written as plain products, the compiler moves all of them to the other file and back in
// every stage (256 moves for 32 matrix instructions).  They go through a temporary here, in the rare branch only; the
// no-ops cover the distance that a matrix instruction's result needs before it is read, and a move's before the next.
template <int D>
__device__ __forceinline__ void rescale(f32x16& acc, float f) {
  if constexpr (D == 256) {
    asm volatile("s_nop 15\n\ts_nop 7" ::: );
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float x = acc[r], t;
      asm volatile("v_accvgpr_read_b32 %1, %0\n\ts_nop 1\n\tv_mul_f32 %1, %1, %2\n\ts_nop 1\n\tv_accvgpr_write_b32 %0, %1"
                   : "+a"(x), "=&v"(t) : "v"(f));
      acc[r] = x;
    }
    asm volatile("s_nop 7" ::: );
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] *= f;
  }
}

// f acc (a product's transposed result: lane l holds column l % 32) as 16-bit rows p[row][d], n of them, through the wave's
// piece of LDS: stores straight from the lanes would be 8 bytes in each of 32 rows.
template <int D, int DT>
__device__ __forceinline__ void store_rows(char* lds, const f32x16* acc, float f, uint16_t* p, int64_t row_stride, int n,
                                           int lane) {
  constexpr int PITCH = D * 2 + 16, CPR = D / 8;  // bytes of a row in LDS; 16-byte chunks of a row
  char* w = lds + (lane & 31) * PITCH + 8 * (lane >> 5);
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4)
      *reinterpret_cast<u32x2*>(w + 64 * d + 4 * r) = u32x2{pack2<DT>(acc[d][r] * f, acc[d][r + 1] * f),
                                                            pack2<DT>(acc[d][r + 2] * f, acc[d][r + 3] * f)};
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // a wave reads its own piece only
#pragma unroll
  for (int i = 0; i < CPR / 2; ++i) {
    const int id = i * 64 + lane, row = id / CPR, c = id % CPR;
    const u32x4 x = *reinterpret_cast<const u32x4*>(lds + row * PITCH + c * 16);
    if (row < n) *reinterpret_cast<u32x4*>(p + row * row_stride + c * 8) = x;
  }
}

// a part's f32 sums f acc, the lane's row from p on
template <int D>
__device__ __forceinline__ void store_sums(float* p, const f32x16* acc, float f) {
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4)
      *reinterpret_cast<f32x4*>(p + 32 * d + 2 * r) =
          f32x4{acc[d][r] * f, acc[d][r + 1] * f, acc[d][r + 2] * f, acc[d][r + 3] * f};
}

// What a 16-bit output leaves of f32 values, kept for the backward (delta = do . o would otherwise carry the output's
// rounding into every score gradient: dq and dk 0.0027 off in bf16 at 2000 keys instead of 0.0024, where their own
// rounding alone makes 0.0017): the difference times 2^12 as E5M2, an eighth of it left over at most.
constexpr float LO_SCALE = 4096.f;
template <int DT>
__device__ __forceinline__ uint32_t left_over(float a, float b, float c, float d) {
  float x[4];
  unpack2<DT>(pack2<DT>(a, b), x[0], x[1]);
  unpack2<DT>(pack2<DT>(c, d), x[2], x[3]);
  return e5m2x4((a - x[0]) * LO_SCALE, (b - x[1]) * LO_SCALE, (c - x[2]) * LO_SCALE, (d - x[3]) * LO_SCALE);
}
// the left-overs of f acc as rows p[row][d] of bytes, as store_rows
template <int D, int DT>
__device__ __forceinline__ void store_left_over(char* lds, const f32x16* acc, float f, uint8_t* p, int64_t row_stride, int n,
                                                int lane) {
  constexpr int PITCH = D + 16, CPR = D / 16;
  char* w = lds + (lane & 31) * PITCH + 4 * (lane >> 5);
#pragma unroll
  for (int d = 0; d < D / 32; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4)
      *reinterpret_cast<uint32_t*>(w + 32 * d + 2 * r) =
          left_over<DT>(acc[d][r] * f, acc[d][r + 1] * f, acc[d][r + 2] * f, acc[d][r + 3] * f);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
  for (int i = 0; i < CPR / 2; ++i) {
    const int id = i * 64 + lane, row = id / CPR, c = id % CPR;
    const u32x4 x = *reinterpret_cast<const u32x4*>(lds + row * PITCH + c * 16);
    if (row < n) *reinterpret_cast<u32x4*>(p + row * row_stride + c * 16) = x;
  }
}

// A workgroup takes NW x 32 queries of one head, 32 a wave, and walks the keys in stages of 32 through a ring in LDS.  The
// scores of stage j + 1 are formed beside the softmax of stage j, so that the matrix cores and the vector unit work at the
// same time; one barrier a stage.
// 32 queries a wave, not 64: the accumulators, Q's fragments and two stages of scores leave two waves a SIMD at D = 128.  K
// and V then cost 1 KiB of LDS reads a matrix instruction, which its 128 bytes a clock just carry.
// Measured, one sequence of 16384, 16 heads over 4 (2): 1.02 ms, 1080 TFLOP/s at D = 128 (a library product of 8192^3
// reaches 1190 to 1240 on these cards); D = 64 0.60 ms, 910 (as many exponentials for half the products); D = 256 2.30 ms,
// 955 (one wave a SIMD).  24 prompts of 1024: 136 us, 755; start and end are 9000 of a workgroup's 45000 cycles there.
template <int D> constexpr int FWD_EU = D == 256 ? 1 : D == 128 ? 2 : 3;  // waves per SIMD that the registers allow
// TRAIN: for a backward, with what o's rounding leaves over, and o divided by the sum of the weights as they were rounded:
// a rounding then moves o by (v - o) of it and not by v, and a weight that makes up most of a row by nothing (o 0.0022 off
// in bf16 without, 0.0020 with; dq, which takes delta from it, 0.0025 and 0.0024).  8% of the forward's time, 1% of a step.
template <int D, int DT, int NW, bool TRAIN>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(FWD_EU<D>)))
void attn_fwd_kernel(AttnArgs a, int parts, float* __restrict__ po, f32x4* __restrict__ pm, uint16_t* __restrict__ o,
                     uint8_t* __restrict__ olo, float* __restrict__ lse) {
  constexpr int BM = NW * 32, FR = STAGES<D>, TILE = FN * D * 2;  // bytes of one operand of one stage
  __shared__ __attribute__((aligned(1024))) char smem[2 * FR * TILE];  // FR stages of K, then FR of V
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ln = lane & 31, hf = lane >> 5;
  const int group = a.hq / a.hk;
  int sq, unit, slot;  // unit: key head, part, head of the group, so that the heads that share keys stay together
  head_tile(a, a.cu_q && a.nseq < IN_A_ROW, sq, unit, slot);
  const int kvh = unit / (parts * group), part = parts == 1 ? 0 : unit / group % parts, head = kvh * group + unit % group;
  const Place pl = find_tile<BM, false>(a.cu_q, a.cu_k, a.nseq, a.total_q, a.total_k, sq, slot, lane);
  if (pl.end + (int64_t)slot * BM < a.total_q && part == 0) {  // the slots cover the rows behind the last sequence too
    const int64_t first = pl.end + (int64_t)slot * BM;
    const int n = (int)min((int64_t)BM, a.total_q - first);
    zero_rows<D>(o, first, n, a.hq, head, threadIdx.x, NW * 64);
    if (lse && (int)threadIdx.x < n) lse[(int64_t)head * a.total_q + first + threadIdx.x] = -INFINITY;
  }
  const int tile = pl.tile, q0 = pl.q0, nq = pl.nq, k0 = pl.k0, nk = pl.nk;
  if (pl.seq < 0 || tile * BM >= nq) return;
  const int off = nk - nq, w0 = tile * BM + wave * 32, row = w0 + ln;

  const uint32_t lds = lds_addr((const bf16_t*)smem);
  TileCopy<D, FN, NW> ck, cv;
  ck.init(a.k_row, wave, lane);
  cv.init(a.v_row, wave, lane);
  const int kend = min(nq, (tile + 1) * BM) + off;  // keys the workgroup's last row sees
  const int all = (max(kend, 0) + FN - 1) / FN;
  const int begin = (int)((int64_t)all * part / parts), nst = (int)((int64_t)all * (part + 1) / parts) - begin;
  // stages that the wave's rows see
  const int nsw = w0 < nq ? (max(w0 + 32 + off, 0) + FN - 1) / FN - begin : 0;
  const int kfirst = begin * FN, left = nk - kfirst;  // the part's first key, and the keys from there on
  const uint16_t* kb = a.k + (int64_t)(k0 + kfirst) * a.k_row + kvh * a.k_head;
  const uint16_t* vb = a.v + (int64_t)(k0 + kfirst) * a.v_row + kvh * a.v_head;
  auto issue_k = [&](int st, int slot) {  // stages past the end fill with zeros
    ck.issue(kb + (int64_t)st * FN * a.k_row, a.k_row, left - st * FN, lds + slot * TILE, wave);
  };
  auto issue_v = [&](int st, int slot) {
    cv.issue(vb + (int64_t)st * FN * a.v_row, a.v_row, left - st * FN, lds + (FR + slot) * TILE, wave);
  };
  constexpr int CP = 2 * TileCopy<D, FN, NW>::N;  // copies of a stage
  if (nst) {
    issue_k(0, 0);
#pragma unroll
    for (int s = 1; s < FR; ++s) {
      issue_v(s - 1, s - 1);
      issue_k(s, s);
    }
  }
  u32x4 qf[D / 16];
  {
    const uint16_t* qp = a.q + (int64_t)(q0 + min(row, nq - 1)) * a.q_row + head * a.q_head + 8 * hf;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) qf[s] = *reinterpret_cast<const u32x4*>(qp + 16 * s);
  }
  f32x16 acc[D / 32];
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[t][r] = 0.f;
  // m: base of the weights, in base 2 (mc: 0 before the first); this half's share of the row's sum of the weights (l: lse
  // is from it) and of the weights as rounded (lr)
  float m = -INFINITY, mc = 0.f, l = 0.f, lr = 0.f;
  const uint32_t ka = lds + row_addr<D>(lane);
  uint32_t va[COLS<D>];
#pragma unroll
  for (int t = 0; t < COLS<D>; ++t) va[t] = lds + FR * TILE + col_addr<D>(lane, t);

  auto scores = [&](int slot, f32x16& s) {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int x = 0; x < D / 16; ++x) s = mma32<DT>(lds_read16(row_step<D>(ka, x) + slot * TILE), qf[x], s);
  };
  // Stage st in slot u: the next stage's scores on the matrix cores beside this one's softmax, then the weights times V.
  auto step = [&](int st, auto uc, f32x16& s, f32x16& next) {
    constexpr int u = decltype(uc)::value;
    if constexpr (D == 256) {
#pragma unroll
      for (int d = 0; d < D / 32; ++d) asm volatile("" : "+a"(acc[d]));
    }
    stage_barrier<(FR - 2) * CP>();  // K of st + 1 and V of st have landed; nobody reads K of st and V of st - 1 any more
    issue_v(st + FR - 1, (u + FR - 1) % FR);
    issue_k(st + FR, u);
    if (st >= nsw) return;  // nothing of this stage is visible to the wave's rows
    if (st * FN + FN - 1 > w0 + off - kfirst) {  // the diagonal or the end of the keys
      const int lim = row + off - kfirst - st * FN;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (8 * (r / 4) + 4 * hf + r % 4 > lim) s[r] = -INFINITY;
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);  // of the two waves of a SIMD the one with a softmax to do goes first (up to 4%)
    scores((u + 1) % FR, next);
    float mx = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
    mx = fmaf(halves(mx, [](float x, float y) { return fmaxf(x, y); }), a.scale2, DT == LSURGE_F16 ? -LIFT : 0.f);
    // the weights' base follows the maximum only when it has grown by 2^8: any base does, and f32 sums and 16-bit weights
    // have room for it, so that the accumulators are rescaled in few stages
    mx = mx > m + LAZY ? mx : m;
    mc = mx == -INFINITY ? 0.f : mx;
    const float alpha = exp2_hw(m - mc);
    float sum[2] = {0.f, 0.f};
    u32x4 p[2];
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
      const float e0 = exp2_hw(fmaf(s[r], a.scale2, -mc)), e1 = exp2_hw(fmaf(s[r + 1], a.scale2, -mc));
      sum[0] += e0;
      sum[1] += e1;
      p[r / 8][r % 8 / 2] = pack2<DT>(e0, e1);
    }
    float rsum = 0.f;
    if constexpr (TRAIN) {
#pragma unroll
      for (int i = 0; i < 8; ++i) rsum = add2<DT>(p[i / 4][i % 4], rsum);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) asm volatile("" : "+v"(p[i]));  // formed here, not after the branch below
    interleave<D / 16, 4>();
    __builtin_amdgcn_sched_barrier(0);
    if (__any(mx != m)) {
      l *= alpha;
      if (TRAIN) lr *= alpha;
#pragma unroll
      for (int d = 0; d < D / 32; ++d) rescale<D>(acc[d], alpha);
    }
    if constexpr (D == 256) {
#pragma unroll
      for (int d = 0; d < D / 32; ++d) asm volatile("" : "+a"(acc[d]));
    }
    m = mx;
    l += sum[0] + sum[1];
    if (TRAIN) lr += rsum;
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int d = 0; d < D / 32; ++d)
        acc[d] = mma32<DT>(lds_read_col<D>(col_step<D>(va, d) + 16 * i * D * 2 + u * TILE), p[i], acc[d]);
    feed<D / 16, 2, 8>();
    __builtin_amdgcn_sched_barrier(0);
  };
  if (nst) {
    stage_barrier<(FR - 1) * CP>();  // K of stage 0
    f32x16 s0, s1, s2;
    scores(0, s0);
    for (int st = 0; st < nst; st += FR) {
      step(st, std::integral_constant<int, 0>(), s0, s1);
      if constexpr (FR == 4) {
        if (st + 1 < nst) step(st + 1, std::integral_constant<int, 1>(), s1, s0);
        if (st + 2 < nst) step(st + 2, std::integral_constant<int, 2>(), s0, s1);
        if (st + 3 < nst) step(st + 3, std::integral_constant<int, FR - 1>(), s1, s0);
      } else {
        if (st + 1 < nst) step(st + 1, std::integral_constant<int, 1>(), s1, s2);
        if (st + 2 < nst) step(st + 2, std::integral_constant<int, 2>(), s2, s0);
      }
    }
    __builtin_amdgcn_s_waitcnt(0);  // the copies past the end land before LDS is used again, or the wave ends
  }
  l = halves(l, [](float x, float y) { return x + y; });
  lr = TRAIN ? halves(lr, [](float x, float y) { return x + y; }) : l;
  if (parts > 1) {
    if (row >= nq) return;  // the sums as they are, and what they are relative to
    const int64_t at = (int64_t)part * a.total_q + q0 + row;
    float* pp = po + (at * a.hq + head) * D + 4 * hf;
    store_sums<D>(pp, acc, 1.f);
    if (hf == 0) pm[at * a.hq + head] = f32x4{mc, l, lr, 0.f};
    return;
  }
  const float inv = lr == 0.f ? 0.f : 1.f / lr;
  __syncthreads();
  store_rows<D, DT>(smem + wave * 32 * (D * 2 + 16), acc, inv, o + ((int64_t)(q0 + w0) * a.hq + head) * D, (int64_t)a.hq * D,
                    min(32, nq - w0), lane);
  if (TRAIN)
    store_left_over<D, DT>(smem + wave * 32 * (D * 2 + 16), acc, inv, olo + ((int64_t)(q0 + w0) * a.hq + head) * D,
                           (int64_t)a.hq * D, min(32, nq - w0), lane);
  if (lse && hf == 0 && row < nq)
    lse[(int64_t)head * a.total_q + q0 + row] = l == 0.f ? -INFINITY : (mc + __log2f(l)) * LN2;
}

// o and lse from the parts' sums, added in order: D / 4 threads a row and head
template <int D, int DT>
__global__ __launch_bounds__(256) void attn_fwd_join_kernel(AttnArgs a, int parts, const float* __restrict__ po,
                                                            const f32x4* __restrict__ pm, uint16_t* __restrict__ o,
                                                            uint8_t* __restrict__ olo, float* __restrict__ lse) {
  constexpr int LPR = D / 4;
  const int64_t n = (int64_t)(a.cu_q ? cu_at(a.cu_q, a.nseq, a.total_q) : a.total_q) * a.hq;
  const int64_t step = (int64_t)a.total_q * a.hq;
  const int d = threadIdx.x % LPR * 4;
  for (int64_t i = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR; i < n; i += (int64_t)gridDim.x * (256 / LPR)) {
    float m = -INFINITY, l = 0.f, lr = 0.f;
    for (int p = 0; p < parts; ++p)
      if (pm[p * step + i][1] != 0.f) m = fmaxf(m, pm[p * step + i][0]);
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
    for (int p = 0; p < parts; ++p) {
      const f32x4 s = pm[p * step + i];
      const float f = s[1] == 0.f ? 0.f : exp2_hw(s[0] - m);
      l += f * s[1];
      lr += f * s[2];
      if (f != 0.f) x += f * *reinterpret_cast<const f32x4*>(po + (p * step + i) * D + d);
    }
    const float inv = lr == 0.f ? 0.f : 1.f / lr;
    x *= inv;
    *reinterpret_cast<u32x2*>(o + i * D + d) = u32x2{pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3])};
    if (olo) *reinterpret_cast<uint32_t*>(olo + i * D + d) = left_over<DT>(x[0], x[1], x[2], x[3]);
    if (lse && d == 0) lse[i % a.hq * a.total_q + i / a.hq] = l == 0.f ? -INFINITY : (m + __log2f(l)) * LN2;
  }
}

// ------------------------------------------------------------------------------------ backward
// What the passes need of each query, laid out [hq][total_q]: lse2 = lse log2(e) (+inf for a row with no key, whose weights
// 2^(s - lse2) are then 0) and delta = do . o - dlse, found by the pass over queries, whose lanes hold do already, and kept
// for the pass over keys.
//
// f16 values have few exponent bits: weights of long rows (2^-15 and less) and their products with small gradients would be
// subnormal, so the f16 passes work on weights 2^SHIFT times too large (lse2 smaller by SHIFT) and on score gradients scaled
// by a power of two, undone in f32 at the end.  The scale is a query's own in the pass over queries and a key's own in the
// pass over keys: a lane's, both times.  It starts from the largest upstream gradient, the query's or that of all the
// queries which see the workgroup's keys (amax: a tile's largest; other sequences have no part in it, nor do infinities),
// which becomes 1 to 2, and is lowered whenever a score gradient would pass f16's largest (fit_f16).  What is lost is half of
// f16's least subnormal, 2^-25, at that scale: 2^-35 of the largest upstream gradient, or 2^-25 of the largest score gradient
// where the scale was lowered.  The check costs half an instruction a score gradient, 2% of a step (31 packed documents of
// 64-wide heads: 776 -> 791 us).
template <int DT> constexpr float SHIFT = DT == LSURGE_F16 ? 10.f : 0.f;
struct RowPrep {
  f32x2_t* rows;  // lse2, delta
  float* amax;    // f16: [hq][nblk], tile t of sequence s at entry (its first row) / rows of a tile + s + t
  int nblk;
};
// 2^e with 2^e amax in [1, 2); 1 for 0
__device__ __forceinline__ float grad_scale(float amax) {
  if (!(amax > 0.f)) return 1.f;
  int e;
  (void)frexpf(amax, &e);
  return ldexpf(1.f, min(max(1 - e, -60), 60));
}
__device__ __forceinline__ float finite_abs(float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.f; }
// Score gradients x of the lane's query or key, as scaled by gs, brought into f16's range, with what is summed up already.
// A lane's partner in the other half of the wave has the same query or key.
constexpr float F16_MAX = 65504.f;
template <int D>
__device__ __forceinline__ void fit_f16(f32x16& x, float& gs, f32x16* acc) {
  float big = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) big = fmaxf(big, fabsf(x[r]));
  if (__any(big > F16_MAX)) {
    big = halves(big, [](float p, float q) { return fmaxf(p, q); });
    // a power of two that makes it 1 to 2; an infinite one is beyond help, and nobody else's business
    const float c =
        big > F16_MAX && big < INFINITY ? __uint_as_float(max(254 - (int)(__float_as_uint(big) >> 23), 1) << 23) : 1.f;
    gs *= c;
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] *= c;
#pragma unroll
    for (int d = 0; d < D / 32; ++d) rescale<D>(acc[d], c);
  }
}

// dq_i = scale sum_j ds_ij k_j with ds_ij = p_ij (do_i . v_j - delta_i): the forward's walk, a query per lane, dS^T in
// place as the operand of dQ^T = K^T dS^T.  The scores are formed again rather than handed over by the pass over keys:
// two products more, but no sum over workgroups, whose order would change the results.  Bound by the matrix cores: 6.0 ms
// for one sequence of 32768, 16 heads over 4, 1110 TFLOP/s of its three products.
template <int D, int DT, int NW>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : 2)))
void attn_dq_kernel(AttnArgs a, const uint16_t* __restrict__ o, const uint8_t* __restrict__ olo,
                    const uint16_t* __restrict__ dout, const float* __restrict__ lse, const float* __restrict__ dlse,
                    RowPrep w, float scale, int parts, float* __restrict__ psum, uint16_t* __restrict__ dq) {
  constexpr int BM = NW * 32, TILE = BN * D * 2;
  __shared__ __attribute__((aligned(1024))) char smem[4 * TILE];
  __shared__ float red[NW];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ln = lane & 31, hf = lane >> 5;
  const int group = a.hq / a.hk;
  int sq, unit, slot;
  head_tile(a, a.cu_q && a.nseq < IN_A_ROW, sq, unit, slot);
  const int kvh = unit / (parts * group), part = parts == 1 ? 0 : unit / group % parts, head = kvh * group + unit % group;
  const Place pl = find_tile<BM, false>(a.cu_q, a.cu_k, a.nseq, a.total_q, a.total_k, sq, slot, lane);
  if (pl.end + (int64_t)slot * BM < a.total_q && part == 0) {
    const int64_t first = pl.end + (int64_t)slot * BM;
    zero_rows<D>(dq, first, (int)min((int64_t)BM, a.total_q - first), a.hq, head, threadIdx.x, NW * 64);
  }
  const int tile = pl.tile, q0 = pl.q0, nq = pl.nq, k0 = pl.k0, nk = pl.nk;
  if (pl.seq < 0 || tile * BM >= nq) return;
  const int off = nk - nq, w0 = tile * BM + wave * 32, row = w0 + ln;

  const uint32_t lds = lds_addr((const bf16_t*)smem);
  TileCopy<D, BN, NW> ck, cv;
  ck.init(a.k_row, wave, lane);
  cv.init(a.v_row, wave, lane);
  const int kend = min(nq, (tile + 1) * BM) + off;
  const int all = (max(kend, 0) + BN - 1) / BN;
  const int begin = (int)((int64_t)all * part / parts), nst = (int)((int64_t)all * (part + 1) / parts) - begin;
  const int kfirst = begin * BN;  // the part's first key
  const uint16_t* kb = a.k + (int64_t)(k0 + kfirst) * a.k_row + kvh * a.k_head;
  const uint16_t* vb = a.v + (int64_t)(k0 + kfirst) * a.v_row + kvh * a.v_head;
  auto issue = [&](int st) {
    const uint32_t at = lds + (st & 1) * 2 * TILE;
    ck.issue(kb + (int64_t)st * BN * a.k_row, a.k_row, nk - kfirst - st * BN, at, wave);
    cv.issue(vb + (int64_t)st * BN * a.v_row, a.v_row, nk - kfirst - st * BN, at + TILE, wave);
  };
  if (nst) issue(0);
  // delta and the row's scale from the fragments of do (the two halves of the wave hold the two halves of a row)
  u32x4 qf[D / 16], df[D / 16];
  const int crow = q0 + min(row, nq - 1);
  const int64_t pi = (int64_t)head * a.total_q + crow;
  const float row_lse = lse[pi];
  float delta = 0.f, big = 0.f;
  {
    const uint16_t* qp = a.q + (int64_t)crow * a.q_row + head * a.q_head + 8 * hf;
    const int64_t at = ((int64_t)crow * a.hq + head) * D + 8 * hf;
    u32x4 of[D / 16];
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      df[s] = *reinterpret_cast<const u32x4*>(dout + at + 16 * s);
      of[s] = *reinterpret_cast<const u32x4*>(o + at + 16 * s);
    }
#pragma unroll
    for (int s = 0; s < D / 16; ++s) qf[s] = *reinterpret_cast<const u32x4*>(qp + 16 * s);
    u32x2 lo[D / 16];
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
      lo[s] = olo ? *reinterpret_cast<const u32x2*>(olo + at + 16 * s) : u32x2{0, 0};
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x0, x1, y0, y1;
        unpack2<DT>(of[s][i], x0, x1);
        const f32x2_t e = i % 2 ? __builtin_amdgcn_cvt_pk_f32_bf8(lo[s][i / 2], true)
                                : __builtin_amdgcn_cvt_pk_f32_bf8(lo[s][i / 2], false);
        x0 = fmaf(e[0], 1.f / LO_SCALE, x0);
        x1 = fmaf(e[1], 1.f / LO_SCALE, x1);
        unpack2<DT>(df[s][i], y0, y1);
        delta = fmaf(x0, y0, fmaf(x1, y1, delta));
        if (DT == LSURGE_F16) big = fmaxf(big, fmaxf(finite_abs(y0), finite_abs(y1)));
      }
  }
  // a row without a key: o and lse are constants there, whatever their upstream gradients (0 x NaN would reach dk)
  const bool none = row_lse == -INFINITY;
  const float row_dlse = dlse && !none ? dlse[pi] : 0.f;
  delta = halves(delta, [](float x, float y) { return x + y; });
  delta = none ? 0.f : delta - row_dlse;
  const float lse2 = none ? INFINITY : row_lse * LOG2E - SHIFT<DT>;
  if (hf == 0 && row < nq && part == 0) w.rows[pi] = f32x2_t{lse2, delta};
  float gs = 1.f;
  if constexpr (DT == LSURGE_F16) {
    big = halves(big, [](float x, float y) { return fmaxf(x, y); });
    big = none ? 0.f : fmaxf(big, finite_abs(row_dlse));
    gs = grad_scale(big);
    big = wave_max(big);  // rows past the end repeat the last one
    if (lane == 0) red[wave] = big;
    __syncthreads();
    if (threadIdx.x == 0 && part == 0) {
#pragma unroll
      for (int i = 1; i < NW; ++i) big = fmaxf(big, red[i]);
      w.amax[(int64_t)head * w.nblk + q0 / BM + pl.seq + tile] = big;
    }
  }
  f32x16 acc[D / 32];
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[t][r] = 0.f;

  const uint32_t ra = row_addr<D>(lane);
  uint32_t ca[COLS<D>];
#pragma unroll
  for (int t = 0; t < COLS<D>; ++t) ca[t] = col_addr<D>(lane, t);

  if constexpr (D == 256 && DT == LSURGE_F16) {
#pragma unroll
    for (int d = 0; d < D / 32; ++d) asm volatile("" : "+a"(acc[d]));
  }
  for (int st = 0; st < nst; ++st) {
    if constexpr (D == 256) {  // as in the forward
#pragma unroll
      for (int d = 0; d < D / 32; ++d) asm volatile("" : "+a"(acc[d]));
    }
    stage_barrier<0>();
    if (st + 1 < nst) issue(st + 1);
    if (kfirst + st * BN > w0 + 31 + off || w0 >= nq) continue;
    const uint32_t kt = lds + (st & 1) * 2 * TILE, vt = kt + TILE;
    const int lim = row + off - kfirst - st * BN;
    const bool edge = kfirst + st * BN + BN - 1 > w0 + off;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      f32x16 s, g;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = g[r] = 0.f;
#pragma unroll
      for (int x = 0; x < D / 16; ++x) {
        s = mma32<DT>(lds_read16(row_step<D>(ra, x) + kt + t * 32 * D * 2), qf[x], s);
        g = mma32<DT>(lds_read16(row_step<D>(ra, x) + vt + t * 32 * D * 2), df[x], g);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = exp2_hw(fmaf(s[r], a.scale2, -lse2));
        s[r] = p * ((g[r] - delta) * gs);
      }
      if (edge)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (32 * t + 8 * (r / 4) + 4 * hf + r % 4 > lim) s[r] = 0.f;
      if constexpr (DT == LSURGE_F16) fit_f16<D>(s, gs, acc);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4 p;
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = pack2<DT>(s[8 * h + 2 * i], s[8 * h + 2 * i + 1]);
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
          acc[d] = mma32<DT>(lds_read_col<D>(kt + (32 * t + 16 * h) * D * 2 + col_step<D>(ca, d)), p, acc[d]);
      }
    }
  }
  const float f = scale / gs * exp2_hw(-SHIFT<DT>);
  if (parts > 1) {
    if (row >= nq) return;
    float* pp = psum + (((int64_t)part * a.total_q + q0 + row) * a.hq + head) * D + 4 * hf;
    store_sums<D>(pp, acc, f);
    return;
  }
  __syncthreads();
  store_rows<D, DT>(smem + wave * 32 * (D * 2 + 16), acc, f, dq + ((int64_t)(q0 + w0) * a.hq + head) * D, (int64_t)a.hq * D,
                    min(32, nq - w0), lane);
}

// dv_j = sum_i p_ij do_i, dk_j = scale sum_i ds_ij q_i over the queries of every head of the group.  A workgroup takes
// NW x 32 keys of one key head, 32 a wave, a key per lane (S = Q K^T), and walks the group's queries in stages of 32 rows
// of q and do through a three-deep LDS ring; dV^T = dO^T P and dK^T = Q^T dS take P and dS from the lanes they were formed
// in.  Both accumulators and the fragments of K and V would fill all 256 registers that two waves a SIMD leave at
// D = 128, so V waits in LDS there.  The stages of a tile are cut into `parts` equal runs, a workgroup each, where there
// are too few tiles (the first keys of a causal sequence have many more queries than the last); the parts' sums are then
// f32 in `psum` and added up in order by attn_sum_kernel.  Bound by the matrix cores: 8.5 ms for one sequence of 32768, 16
// heads over 4, 1030 TFLOP/s of its four products (10.5 with both fragments in registers, 75 of them spilled; 11 to 13.5
// with one wave a SIMD, whose instructions alone outlast its products).
constexpr int QN = 32;  // query rows per stage
template <int D> constexpr bool V_IN_LDS = D >= 128;
template <int D> constexpr int DKV_EU = D == 256 ? 1 : 2;  // waves per SIMD that the registers allow
template <int D, int DT, int NW>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(DKV_EU<D>)))
void attn_dkv_kernel(AttnArgs a, const uint16_t* __restrict__ dout, RowPrep w, float scale, int parts,
                     float* __restrict__ psum, uint16_t* __restrict__ dk, uint16_t* __restrict__ dv) {
  constexpr int BK = NW * 32, R = V_IN_LDS<D> ? 2 : 3, TILE = QN * D * 2, VBYTES = V_IN_LDS<D> ? BK * D * 2 : 0;
  // R stages of q, R of do, R of the rows' lse2 and delta, then V
  __shared__ __attribute__((aligned(1024))) char smem[2 * R * TILE + 1024 + VBYTES];
  __shared__ float red[NW];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ln = lane & 31, hf = lane >> 5;
  int sq, unit, slot;
  head_tile(a, true, sq, unit, slot);  // the first keys are seen by the most queries
  const int kvh = unit / parts, part = unit % parts;
  const Place pl = find_tile<BK, true>(a.cu_q, a.cu_k, a.nseq, a.total_q, a.total_k, sq, slot, lane);
  if (pl.end + (int64_t)slot * BK < a.total_k && part == 0) {
    const int64_t first = pl.end + (int64_t)slot * BK;
    const int n = (int)min((int64_t)BK, a.total_k - first);
    zero_rows<D>(dk, first, n, a.hk, kvh, threadIdx.x, NW * 64);
    zero_rows<D>(dv, first, n, a.hk, kvh, threadIdx.x, NW * 64);
  }
  const int tile = pl.tile, q0 = pl.q0, nq = pl.nq, k0 = pl.k0, nk = pl.nk;
  if (pl.seq < 0 || tile * BK >= nk) return;
  const int off = nk - nq, w0 = tile * BK + wave * 32, col = w0 + ln, group = a.hq / a.hk;

  const uint32_t lds = lds_addr((const bf16_t*)smem), lds_rows = lds + 2 * R * TILE, lds_v = lds_rows + 1024;
  TileCopy<D, QN, NW> cq, cd;
  const int64_t d_row = (int64_t)a.hq * D;
  cq.init(a.q_row, wave, lane);
  cd.init(d_row, wave, lane);
  const int first = max(0, tile * BK - off) / QN;  // the stage of the first query that sees the tile's first key
  const int per = max(0, (nq + QN - 1) / QN - first), all = per * group;
  const int begin = (int)((int64_t)all * part / parts), nst = (int)((int64_t)all * (part + 1) / parts) - begin;
  // the stage to issue next: its head and first row
  int ih = per ? kvh * group + begin / per : 0, ir = per ? (first + begin % per) * QN : 0;
  auto issue = [&](int slot) {  // stages past the end fill with other rows of the group, or zeros
    const int n = ih < (kvh + 1) * group ? nq - ir : 0;
    cq.issue(a.q + (int64_t)(q0 + ir) * a.q_row + ih * a.q_head, a.q_row, n, lds + slot * TILE, wave);
    cd.issue(dout + (int64_t)(q0 + ir) * d_row + ih * D, d_row, n, lds + (R + slot) * TILE, wave);
    // rows past the end get zeros: q and do are zeros there, so any finite values do
    copy4(make_rsrc(w.rows + (int64_t)ih * a.total_q + q0 + ir, 8 * (int64_t)max(0, min(n, QN))),
          lane % 32 * 8 + lane / 32 * 4, lds_rows + slot * 256);
    ir += QN;
    if (ir >= nq) {
      ir = first * QN;
      ++ih;
    }
  };
  constexpr int CP = 2 * TileCopy<D, QN, NW>::N + 1;
  const uint16_t* kp = a.k + (int64_t)(k0 + min(col, nk - 1)) * a.k_row + kvh * a.k_head + 8 * hf;
  u32x4 kf[D / 16], vf[V_IN_LDS<D> ? 1 : D / 16];
  if (nst) {
    if constexpr (V_IN_LDS<D>) {
      TileCopy<D, BK, NW> cv;
      cv.init(a.v_row, wave, lane);
      cv.issue(a.v + (int64_t)(k0 + tile * BK) * a.v_row + kvh * a.v_head, a.v_row, nk - tile * BK, lds_v, wave);
    } else {
      const uint16_t* vp = a.v + (int64_t)(k0 + min(col, nk - 1)) * a.v_row + kvh * a.v_head + 8 * hf;
#pragma unroll
      for (int s = 0; s < D / 16; ++s) vf[s] = *reinterpret_cast<const u32x4*>(vp + 16 * s);
    }
#pragma unroll
    for (int s = 0; s < D / 16; ++s) kf[s] = *reinterpret_cast<const u32x4*>(kp + 16 * s);
    issue(0);
    if (R > 2) issue(1);
  }
  float gs = 1.f;
  if constexpr (DT == LSURGE_F16) {  // the largest upstream gradient of the rows that see the tile's keys, all heads
    float mx = 0.f;
    const int t0 = first * QN / BK, nt = (nq + BK - 1) / BK - t0;  // tiles of the pass over queries, as large as these
    const float* am = w.amax + (int64_t)kvh * group * w.nblk + q0 / BK + pl.seq + t0;
    for (int i = threadIdx.x; i < group * nt; i += NW * 64) mx = fmaxf(mx, am[(int64_t)(i / nt) * w.nblk + i % nt]);
    mx = wave_max(mx);
    if (lane == 0) red[wave] = mx;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NW; ++i) mx = fmaxf(mx, red[i]);
    gs = grad_scale(mx);
  }
  f32x16 ak[D / 32], av[D / 32];
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) ak[t][r] = av[t][r] = 0.f;
  const uint32_t ra = lds + row_addr<D>(lane), rv = lds_v + wave * 32 * D * 2 + row_addr<D>(lane);
  uint32_t ca[COLS<D>];
#pragma unroll
  for (int t = 0; t < COLS<D>; ++t) ca[t] = lds + col_addr<D>(lane, t);

  int cr = per ? (first + begin % per) * QN : 0;  // first row of the stage being computed
  // weights and score gradients of the stage in `slot`, packed as the products' operands
  auto weigh = [&](int slot, const f32x16& s, f32x16& g, u32x4* p, u32x4* x) {
    const uint32_t rw = lds_rows + slot * 256 + 16 * hf;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const u32x4 ls = lds_read16(rw + 32 * b), de = lds_read16(rw + 128 + 32 * b);
      float e[4], f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 4 * b + i;
        e[i] = exp2_hw(fmaf(s[r], a.scale2, -__uint_as_float(ls[i])));
        f[i] = g[r] - __uint_as_float(de[i]);
        if (DT == LSURGE_F16) f[i] *= gs;
        f[i] *= e[i];
        if (DT == LSURGE_F16) g[r] = f[i];
      }
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        p[b / 2][b % 2 * 2 + i / 2] = pack2<DT>(e[i], e[i + 1]);
        if (DT != LSURGE_F16) x[b / 2][b % 2 * 2 + i / 2] = pack2<DT>(f[i], f[i + 1]);
      }
    }
    if constexpr (DT == LSURGE_F16) {
      fit_f16<D>(g, gs, ak);
#pragma unroll
      for (int r = 0; r < 16; r += 2) x[r / 8][r % 8 / 2] = pack2<DT>(g[r], g[r + 1]);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) asm volatile("" : "+v"(p[h]), "+v"(x[h]));
  };
  auto products = [&](int slot, const u32x4* p, const u32x4* x) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int d = 0; d < D / 32; ++d) {
        av[d] = mma32<DT>(lds_read_col<D>(col_step<D>(ca, d) + 16 * h * D * 2 + (R + slot) * TILE), p[h], av[d]);
        ak[d] = mma32<DT>(lds_read_col<D>(col_step<D>(ca, d) + 16 * h * D * 2 + slot * TILE), x[h], ak[d]);
      }
  };
  auto step = [&](auto uc) {
    constexpr int u = decltype(uc)::value;
    if constexpr (DKV_EU<D> == 1) {
#pragma unroll
      for (int d = 0; d < D / 32; ++d) asm volatile("" : "+a"(ak[d]), "+a"(av[d]));
    }
    stage_barrier<(R - 2) * CP>();  // this stage has landed, and nobody reads the one before it any more
    issue((u + R - 1) % R);
    const int r0 = cr;
    cr = cr + QN >= nq ? first * QN : cr + QN;
    if (r0 + QN - 1 + off < w0 || w0 >= nk) return;  // no row of this stage sees the wave's keys
    f32x16 s, g;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = g[r] = 0.f;
#pragma unroll
    for (int x = 0; x < D / 16; ++x) s = mma32<DT>(lds_read16(row_step<D>(ra, x) + u * TILE), kf[x], s);
    if (r0 + off < w0 + 31) {  // the diagonal: a key's lane sees the rows from lim on
      const int lim = col - off - r0;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (8 * (r / 4) + 4 * hf + r % 4 < lim) s[r] = -INFINITY;
    }
    u32x4 p[2], x[2];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int x = 0; x < D / 16; ++x)
      g = mma32<DT>(lds_read16(row_step<D>(ra, x) + (R + u) * TILE),
                    V_IN_LDS<D> ? lds_read16(row_step<D>(rv, x)) : vf[V_IN_LDS<D> ? 0 : x], g);
    weigh(u, s, g, p, x);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);  // the wave with products to issue goes first (1 to 2%)
    products(u, p, x);
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
  };
  for (int st = 0; st < nst; st += R) {
    step(std::integral_constant<int, 0>());
    if (st + 1 < nst) step(std::integral_constant<int, 1>());
    if constexpr (R > 2)
      if (st + 2 < nst) step(std::integral_constant<int, R - 1>());
  }
  __builtin_amdgcn_s_waitcnt(0);  // the copies past the end land before the wave ends
  const float fv = exp2_hw(-SHIFT<DT>), fk = scale / gs * fv;
  const int64_t at = ((int64_t)(k0 + col) * a.hk + kvh) * D + 4 * hf;
  if (parts > 1) {
    if (col >= nk) return;
    const int64_t size = (int64_t)a.total_k * a.hk * D;
    float* pk = psum + 2 * part * size + at;
    store_sums<D>(pk, ak, fk);
    store_sums<D>(pk + size, av, fv);
    return;
  }
  __syncthreads();
  char* piece = smem + wave * 32 * (D * 2 + 16);
  const int64_t first_at = ((int64_t)(k0 + w0) * a.hk + kvh) * D;
  const int n = min(32, nk - w0);
  store_rows<D, DT>(piece, ak, fk, dk + first_at, (int64_t)a.hk * D, n, lane);
  store_rows<D, DT>(piece, av, fv, dv + first_at, (int64_t)a.hk * D, n, lane);
}

// `tensors` gradients (x, then y) of `size` values each = the parts' sums, added in order, 4 values a thread; psum
// [parts][tensors][size].  The rows (`row` values each) from cu[nseq] on were zeroed already.
template <int DT>
__global__ __launch_bounds__(256) void attn_sum_kernel(const float* __restrict__ psum, int parts, int tensors, int64_t size,
                                                       int64_t row, const int32_t* __restrict__ cu, int nseq, int total,
                                                       uint16_t* __restrict__ x, uint16_t* __restrict__ y) {
  const int64_t n = cu ? cu_at(cu, nseq, total) * row : size, step = tensors * size;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < tensors * n; i += (int64_t)gridDim.x * 1024) {
    const bool second = i >= n;
    const int64_t at = second ? i - n : i;
    const float* p = psum + (second ? size : 0) + at;
    f32x4 s = *reinterpret_cast<const f32x4*>(p);
    for (int j = 1; j < parts; ++j) s += *reinterpret_cast<const f32x4*>(p + j * step);
    *reinterpret_cast<u32x2*>((second ? y : x) + at) = u32x2{pack2<DT>(s[0], s[1]), pack2<DT>(s[2], s[3])};
  }
}

// ------------------------------------------------------------------------------------ host
int check_rows(const char* what, const lsurge_attn_rows& r, int64_t d) {
  LSURGE_REQUIRE(r.data, "%s: null pointer", what);
  LSURGE_REQUIRE((uintptr_t)r.data % 16 == 0 && r.row_stride % 8 == 0 && r.head_stride % 8 == 0,
                 "%s: rows must be 16-byte aligned (strides %lld, %lld in elements)", what, (long long)r.row_stride,
                 (long long)r.head_stride);
  LSURGE_REQUIRE(r.row_stride >= d && r.row_stride < (1 << 22) && r.head_stride >= 0 && r.head_stride < (1ll << 40),
                 "%s: row stride %lld outside [head_dim, 2^22), or head stride %lld outside [0, 2^40)", what,
                 (long long)r.row_stride, (long long)r.head_stride);
  return LSURGE_OK;
}

int check_shape(const char* what, const lsurge_attn_shape* s, const int32_t* cu_q, const int32_t* cu_k, float scale) {
  LSURGE_REQUIRE(s, "%s: null shape", what);
  LSURGE_REQUIRE(s->d == 64 || s->d == 128 || s->d == 256, "%s: head_dim %lld (64, 128 or 256)", what, (long long)s->d);
  LSURGE_REQUIRE(s->hk >= 1 && s->hq >= s->hk && s->hq % s->hk == 0 && s->hq <= 65535,
                 "%s: %lld query heads over %lld key heads", what, (long long)s->hq, (long long)s->hk);
  LSURGE_REQUIRE(s->nseq >= 0 && s->nseq < (1 << 24) && s->total_q >= 0 && s->total_q < (1ll << 30) && s->total_k >= 0 &&
                     s->total_k < (1ll << 30),
                 "%s: nseq=%lld total_q=%lld total_k=%lld", what, (long long)s->nseq, (long long)s->total_q,
                 (long long)s->total_k);
  LSURGE_REQUIRE((cu_q != nullptr) == (cu_k != nullptr), "%s: cu_q and cu_k go together", what);
  if (!cu_q)
    LSURGE_REQUIRE(s->nseq == 0 ? s->total_q == 0 && s->total_k == 0
                                : s->total_q % s->nseq == 0 && s->total_k % s->nseq == 0,
                   "%s: %lld and %lld rows are no whole number for each of %lld sequences", what, (long long)s->total_q,
                   (long long)s->total_k, (long long)s->nseq);
  LSURGE_REQUIRE(scale > 0.f && scale < INFINITY, "%s: scale must be positive and finite", what);
  if (s->dtype != LSURGE_BF16 && s->dtype != LSURGE_F16) return lsurge::set_error(LSURGE_ERR_DTYPE, "%s: bf16 or f16", what);
  return LSURGE_OK;
}

// tile slots of the rows: of one dense sequence, or of all packed ones (at least 1: rows behind the last sequence)
int64_t tile_slots(const lsurge_attn_shape& s, bool packed, int64_t total, int64_t rows) {
  return packed ? total / rows + std::max<int64_t>(s.nseq, 1) : (total / s.nseq + rows - 1) / rows;
}
// the launch of `tiles` tile slots for each of `heads` heads, `share` of which read the same rows; 0 workgroups: none
int plan_grid(const char* what, const lsurge_attn_shape& s, bool packed, int64_t heads, int64_t share, int64_t tiles,
              AttnArgs* a, unsigned* grid) {
  const int64_t pairs = (packed ? 1 : s.nseq) * heads;
  // a launch holds less than 2^32 threads, 256 a workgroup
  LSURGE_REQUIRE(pairs * tiles < (1ll << 24), "%s: %lld tiles of %lld heads", what, (long long)tiles, (long long)pairs);
  const int64_t run = pairs % 8 == 0 ? pairs / 8 : 0;
  a->heads = (int)heads, a->pairs = (int)pairs, a->tiles = (int)tiles, a->run = (int)run;
  a->together = (int)(run * tiles <= 128 ? std::max<int64_t>(run, 1)
                                         : run % share == 0 ? share : share % run == 0 ? run : 1);
  *grid = (unsigned)(pairs * tiles);
  return LSURGE_OK;
}

AttnArgs make_args(const lsurge_attn_shape& s, const lsurge_attn_rows& q, const lsurge_attn_rows& k,
                   const lsurge_attn_rows& v, const int32_t* cu_q, const int32_t* cu_k, float scale) {
  AttnArgs a;
  a.q = (const uint16_t*)q.data, a.k = (const uint16_t*)k.data, a.v = (const uint16_t*)v.data;
  a.q_row = q.row_stride, a.k_row = k.row_stride, a.v_row = v.row_stride;
  a.q_head = q.head_stride, a.k_head = k.head_stride, a.v_head = v.head_stride;
  a.cu_q = cu_q, a.cu_k = cu_k;
  a.nseq = (int)s.nseq, a.total_q = (int)s.total_q, a.total_k = (int)s.total_k, a.hq = (int)s.hq, a.hk = (int)s.hk;
  a.heads = a.pairs = a.run = a.together = a.tiles = 0;
  a.scale2 = scale * LOG2E;
  return a;
}

constexpr int WAVES = 4;  // of a workgroup, 32 rows each (8 were as fast or slower at every head dim)

// Parts that the stages of a tile of keys are cut into in attn_dkv_kernel, by the sizes that the host knows (the
// sequences' own lengths are on the device): as many as give every place for a workgroup two of them, so that the ones
// with few queries fill up behind the ones with many, but no part under 4 stages; one part for every 1024 stages where
// they are that many, but no more than 2 of these where the sums would pass 512 MiB (two parts' are 4 times dk and dv).  A
// part costs a write and a read of the tile's f32 sums.  Measured, us a training step at 1, 2, 4 and 8 parts: 8 x 4096 tokens,
// 8 heads over 2 (512 tiles, 256 stages): 1568, 1346, 1435, 1485; one of 32768, 16 heads over 4 (1024, 2048): 19532, 19021,
// 18961, 18864; one of 4096, 8 heads of their own keys (256, 64): 433, 351, 330, 391; one of 512, 8 over 2 (8, 32): 154, 106,
// 82, 72; 2 x 4096, 16 over 2, 256-wide (128, 512): 3552, 2357, 1721, 1756.  What the limit costs: 65536 tokens, 16 heads over
// 4, 2 parts instead of 4: 75.3 -> 75.9 ms; 131072, 8 over 2, instead of 8: 149.9 -> 152.9 ms.
int64_t dkv_parts(const lsurge_attn_shape& s) {
  if (s.total_q == 0 || s.total_k == 0 || s.nseq == 0) return 1;
  const int64_t tiles = s.nseq * ((s.total_k / s.nseq + 127) / 128) * s.hk, places = s.d == 256 ? 256 : 512;
  const int64_t stages = s.hq / s.hk * (s.total_q / s.nseq) / QN / 2;  // half of the queries, on average, see a key
  const int64_t bytes = 2 * sizeof(float) * s.total_k * s.hk * s.d;  // of a part's sums
  const int64_t most = std::max<int64_t>((int64_t(512) << 20) / bytes, 2);
  const int64_t parts =
      std::min(std::max(2 * places / std::max<int64_t>(tiles, 1), std::min(stages / 1024, most)), stages / 4);
  return parts >= 8 ? 8 : parts >= 4 ? 4 : parts >= 2 ? 2 : 1;
}

// Parts that the keys of a tile of queries are cut into in attn_fwd_kernel: as many as fill the places for a workgroup,
// where there are few tiles, and none under 16 stages (a part costs a write and a read of the tile's f32 sums).  Measured,
// us at 1, 2, 3, 4, 8 parts: 3 chunks of 350 rows over 10000 keys, 32 heads (288 tiles, 300 stages): 369, 247, 260, 254,
// 259; 64 rows over 6000 keys, 16 heads (16, 190): 118, 68, 51, 42, 33; one prompt of 2048 (256, 32): 48, 47, 52, 57, 83;
// of 4096, 8 heads, 64-wide (256, 64): 71, 51, 44, 45, 57; of 512 (64, 8): 20, 23, 24, 26, 33.
int64_t key_parts(const lsurge_attn_shape& s, int64_t places) {
  if (s.total_q == 0 || s.total_k == 0 || s.nseq == 0) return 1;
  const int64_t rows = s.total_q / s.nseq, keys = s.total_k / s.nseq;
  const int64_t tiles = std::max<int64_t>(s.nseq * ((rows + 127) / 128) * s.hq, 1);
  const int64_t stages = std::max<int64_t>(keys - rows / 2, 0) / FN;  // of an average tile
  return std::max<int64_t>(1, std::min((places + tiles / 2) / tiles, stages / 16));
}
int64_t fwd_parts(const lsurge_attn_shape& s) { return key_parts(s, s.d == 256 ? 256 : s.d == 128 ? 512 : 768); }
// The same for attn_dq_kernel, us a training step at 1, 2, 3, 4, 8 parts of it: one sequence of 4096, 8 heads of their own
// keys (256 tiles, 64 stages): 314, 269, 257, 261, 288; 8 x 4096, 8 heads over 2 (2048, 64): 1361, 1477, 1546, 1613, 1889.
int64_t dq_parts(const lsurge_attn_shape& s) { return key_parts(s, s.d == 256 ? 256 : s.d == 128 ? 512 : 1024); }

#define ATTN_DISPATCH(CALL)                             \
  do {                                                  \
    if (s->dtype == LSURGE_BF16) {                      \
      if (s->d == 64) { CALL(64, LSURGE_BF16); }        \
      else if (s->d == 128) { CALL(128, LSURGE_BF16); } \
      else { CALL(256, LSURGE_BF16); }                  \
    } else {                                            \
      if (s->d == 64) { CALL(64, LSURGE_F16); }         \
      else if (s->d == 128) { CALL(128, LSURGE_F16); }  \
      else { CALL(256, LSURGE_F16); }                   \
    }                                                   \
  } while (0)

}  // namespace
}  // namespace lsattn

using namespace lsattn;

extern "C" {

size_t lsurge_attn_fwd_workspace_bytes(const lsurge_attn_shape* s) {
  if (!s || s->hq < 1 || s->hk < 1 || s->d < 1 || s->nseq < 0 || s->total_q < 0 || s->total_k < 0) return 0;
  const int64_t parts = fwd_parts(*s);
  return parts > 1 ? sizeof(float) * (size_t)(parts * s->total_q * s->hq * (s->d + 4)) : 0;
}

int lsurge_attn_fwd(const lsurge_attn_shape* s, const lsurge_attn_rows* q, const lsurge_attn_rows* k,
                    const lsurge_attn_rows* v, const int32_t* cu_q, const int32_t* cu_k, float scale, void* o, void* o_lo,
                    float* lse, void* workspace, size_t workspace_bytes, lsurge_stream_t stream) {
  if (int rc = check_shape("attn_fwd", s, cu_q, cu_k, scale)) return rc;
  if (s->total_q == 0) return LSURGE_OK;
  LSURGE_REQUIRE(q && k && v && o && ((uintptr_t)o | (uintptr_t)o_lo) % 16 == 0, "attn_fwd: null or misaligned pointer");
  if (int rc = check_rows("attn_fwd q", *q, s->d)) return rc;
  if (s->total_k) {
    if (int rc = check_rows("attn_fwd k", *k, s->d)) return rc;
    if (int rc = check_rows("attn_fwd v", *v, s->d)) return rc;
  }
  const size_t need = lsurge_attn_fwd_workspace_bytes(s);
  if (workspace_bytes < need)
    return lsurge::set_error(LSURGE_ERR_WORKSPACE, "attn_fwd: workspace %zu < %zu bytes", workspace_bytes, need);
  LSURGE_REQUIRE(need == 0 || (workspace && (uintptr_t)workspace % 16 == 0), "attn_fwd: null or misaligned workspace");
  hipStream_t st = (hipStream_t)stream;
  AttnArgs a = make_args(*s, *q, *k, *v, cu_q, cu_k, scale);
  const int parts = (int)fwd_parts(*s);
  float* po = (float*)workspace;
  f32x4* pm = (f32x4*)(po + (size_t)parts * s->total_q * s->hq * s->d);
#define ATTN_FWD(D, DT)                                                                                                 \
  constexpr int NW = WAVES;                                                                                             \
  unsigned grid;                                                                                                        \
  if (int rc = plan_grid("attn_fwd", *s, cu_q, s->hq * parts, s->hq / s->hk, tile_slots(*s, cu_q, s->total_q, NW * 32), \
                         &a, &grid))                                                                                    \
    return rc;                                                                                                          \
  if (o_lo)                                                                                                             \
    LSURGE_LAUNCH(KID_ATTN, st, hipLaunchKernelGGL((attn_fwd_kernel<D, DT, NW, true>), dim3(grid), dim3(NW * 64), 0,    \
                                                   st, a, parts, po, pm, (uint16_t*)o, (uint8_t*)o_lo, lse));           \
  else                                                                                                                  \
    LSURGE_LAUNCH(KID_ATTN, st, hipLaunchKernelGGL((attn_fwd_kernel<D, DT, NW, false>), dim3(grid), dim3(NW * 64), 0,   \
                                                   st, a, parts, po, pm, (uint16_t*)o, (uint8_t*)nullptr, lse));        \
  const int64_t rows = (s->total_q * s->hq + 1024 / D - 1) / (1024 / D);                                                \
  if (parts > 1)                                                                                                        \
    LSURGE_LAUNCH(KID_ATTN, st, hipLaunchKernelGGL((attn_fwd_join_kernel<D, DT>),                                       \
                                                   dim3((unsigned)std::min<int64_t>(rows, 8192)), dim3(256), 0, st, a,  \
                                                   parts, po, pm, (uint16_t*)o, (uint8_t*)o_lo, lse))
  ATTN_DISPATCH(ATTN_FWD);
#undef ATTN_FWD
  return LSURGE_OK;
}

// entries for the tiles of the queries of a head (see RowPrep): sequence s has at least as many as tiles between its first
// and the next sequence's, packed or not
static int64_t most_query_tiles(const lsurge_attn_shape* s) { return s->total_q / 128 + std::max<int64_t>(s->nseq, 1); }
static size_t prep_bytes(const lsurge_attn_shape* s) {
  const int64_t rows = s->hq * s->total_q;
  const int64_t floats = 2 * rows + (s->dtype == LSURGE_F16 ? s->hq * most_query_tiles(s) : 0);
  return (sizeof(float) * (size_t)floats + 255) / 256 * 256;
}
size_t lsurge_attn_bwd_workspace_bytes(const lsurge_attn_shape* s) {
  if (!s || s->hq < 1 || s->hk < 1 || s->d < 1 || s->nseq < 0 || s->total_q < 0 || s->total_k < 0) return 0;
  const int64_t kp = dkv_parts(*s), qp = dq_parts(*s);  // the passes run one after the other: one room for both
  const int64_t sums = std::max(kp > 1 ? 2 * kp * s->total_k * s->hk : 0, qp > 1 ? qp * s->total_q * s->hq : 0) * s->d;
  return prep_bytes(s) + sizeof(float) * (size_t)sums + 256;
}

int lsurge_attn_bwd(const lsurge_attn_shape* s, const lsurge_attn_rows* q, const lsurge_attn_rows* k,
                    const lsurge_attn_rows* v, const int32_t* cu_q, const int32_t* cu_k, float scale, const void* o,
                    const void* o_lo, const float* lse, const void* dout, const float* dlse, void* dq, void* dk, void* dv,
                    void* workspace, size_t workspace_bytes, lsurge_stream_t stream) {
  if (int rc = check_shape("attn_bwd", s, cu_q, cu_k, scale)) return rc;
  LSURGE_REQUIRE(q && k && v && workspace, "attn_bwd: null pointer");
  const size_t need = lsurge_attn_bwd_workspace_bytes(s);
  if (workspace_bytes < need)
    return lsurge::set_error(LSURGE_ERR_WORKSPACE, "attn_bwd: workspace %zu < %zu bytes", workspace_bytes, need);
  LSURGE_REQUIRE(((uintptr_t)o | (uintptr_t)o_lo | (uintptr_t)dout | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv |
                  (uintptr_t)workspace) % 16 == 0,
                 "attn_bwd: buffers must be 16-byte aligned");
  if (s->total_q) {
    LSURGE_REQUIRE(o && lse && dout && dq, "attn_bwd: null pointer");
    if (int rc = check_rows("attn_bwd q", *q, s->d)) return rc;
  }
  if (s->total_k) {
    LSURGE_REQUIRE(dk && dv, "attn_bwd: null pointer");
    if (int rc = check_rows("attn_bwd k", *k, s->d)) return rc;
    if (int rc = check_rows("attn_bwd v", *v, s->d)) return rc;
  }
  hipStream_t st = (hipStream_t)stream;
  AttnArgs a = make_args(*s, *q, *k, *v, cu_q, cu_k, scale);
  const int64_t nrow = s->hq * s->total_q;
  RowPrep w;
  w.rows = (f32x2_t*)workspace, w.amax = (float*)(w.rows + nrow);
  w.nblk = (int)most_query_tiles(s);
  float* psum = (float*)((char*)workspace + prep_bytes(s));
  const int parts = (int)dkv_parts(*s), qparts = (int)dq_parts(*s);
  const uint16_t* g = (const uint16_t*)dout;
#define ATTN_BWD(D, DT)                                                                                                    \
  constexpr int NW = WAVES;                                                                                                \
  AttnArgs ak = a;                                                                                                         \
  unsigned gq = 0, gk = 0;                                                                                                 \
  if (s->total_q)                                                                                                          \
    if (int rc = plan_grid("attn_bwd", *s, cu_q, s->hq * qparts, s->hq / s->hk, tile_slots(*s, cu_q, s->total_q, NW * 32), \
                           &a, &gq))                                                                                       \
      return rc;                                                                                                           \
  if (s->total_k)                                                                                                          \
    if (int rc = plan_grid("attn_bwd", *s, cu_q, s->hk * parts, 1, tile_slots(*s, cu_q, s->total_k, NW * 32), &ak, &gk))   \
      return rc;                                                                                                           \
  const auto sum_grid = [](int64_t n) { return dim3((unsigned)std::min<int64_t>((n + 1023) / 1024, 4096)); };              \
  if (gq) {                                                                                                                \
    LSURGE_LAUNCH(KID_ATTN, st, hipLaunchKernelGGL((attn_dq_kernel<D, DT, NW>), dim3(gq), dim3(NW * 64), 0, st, a,         \
                                                   (const uint16_t*)o, (const uint8_t*)o_lo, g, lse, dlse, w, scale,       \
                                                   qparts, psum,                                                           \
                                                   (uint16_t*)dq));                                                        \
    const int64_t size = s->total_q * s->hq * D;                                                                           \
    if (qparts > 1)                                                                                                        \
      LSURGE_LAUNCH(KID_ATTN, st, hipLaunchKernelGGL((attn_sum_kernel<DT>), sum_grid(size), dim3(256), 0, st, psum,        \
                                                     qparts, 1, size, s->hq * D, cu_q, a.nseq, a.total_q,                  \
                                                     (uint16_t*)dq, (uint16_t*)dq));                                       \
  }                                                                                                                        \
  if (gk) {                                                                                                                \
    LSURGE_LAUNCH(KID_ATTN, st, hipLaunchKernelGGL((attn_dkv_kernel<D, DT, NW>), dim3(gk), dim3(NW * 64), 0, st, ak, g,    \
                                                   w, scale, parts, psum, (uint16_t*)dk, (uint16_t*)dv));                  \
    const int64_t size = s->total_k * s->hk * D;                                                                           \
    if (parts > 1)                                                                                                         \
      LSURGE_LAUNCH(KID_ATTN, st, hipLaunchKernelGGL((attn_sum_kernel<DT>), sum_grid(2 * size), dim3(256), 0, st, psum,    \
                                                     parts, 2, size, s->hk * D, cu_k, a.nseq, a.total_k,                   \
                                                     (uint16_t*)dk, (uint16_t*)dv));                                       \
  }
  ATTN_DISPATCH(ATTN_BWD);
#undef ATTN_BWD
  return LSURGE_OK;
}

}  // extern "C"

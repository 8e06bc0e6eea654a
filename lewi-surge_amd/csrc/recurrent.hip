// The gated delta rule over new tokens, from and to the states that serving keeps: one token for each of many sequences, a few
// drafted ones, or prompts.
//
// Per sequence and value head, S [128, 128] f32:  S <- e^g S,  d = beta (v - S^T k),  S <- S + k d^T,  o = S^T q / sqrt(128).
// The columns of S evolve independently of each other, so a wave takes a block of them through all tokens of its sequence:
// its part of S stays in registers, is read once and written once, and no wave waits for another.  A token's two products run
// on the decayed S before it, S^T k and S^T q in one walk over the registers, with
//   o = (S^T q + (k . q) d) / sqrt(128),
// so that one exchange between lanes serves both; the l2 norms of q and k are factors of these sums and cost no pass of their
// own.  Everything is f32 but the inputs and o.
//
// Bound by memory for a token or a few (64 KiB of state a sequence and head, read and written): one token for 64 sequences of
// 32 heads takes 42.5 us, 6.0 TB/s, with a part of the states in the caches, 54 us, 5.0 TB/s, with none (a copy reaches 5.1);
// 100 runs of 1 to 8 tokens of 8 heads 28.5 us, 3.8 TB/s.  Longer runs go in chunks on the matrix cores and are a chain: 2000
// tokens take 107 us, 1.7 us for 32 of them.  A chunk's products follow each other in one wave: its 90 matrix instructions are
// 1440 of the 3800 cycles, its 440 vector instructions 1750, the rest waits for the one before.
#include <algorithm>
#include <type_traits>
#include <utility>

#include "launchers.h"
#include "rows16.h"

namespace lsgdn {
namespace {

constexpr int D = 128;
constexpr int WAVES = 4;

struct TokenArgs {
  const uint16_t *q, *k, *v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  const float* g;
  const void* beta;
  int64_t g_row, beta_row;
  float* state;
  int64_t slot_stride;
  uint16_t* o;
  const int32_t *slots, *cu;
  int rows, nseq, hk, hv, num_slots;
  float l2_eps;
  int units;  // workgroups of the sequences; those behind them clear the rows of none
};

// the sum over the RG lanes of a group (RG consecutive lanes), in all of them
template <int RG>
__device__ __forceinline__ float group_sum(float x) {
  auto add = [](float v, auto ctrl) {
    const int r = __builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, true);
    return v + __int_as_float(r);
  };
  x = add(x, std::integral_constant<int, 0xb1>());   // the lane's neighbour (quad_perm 1, 0, 3, 2)
  x = add(x, std::integral_constant<int, 0x4e>());   // two lanes on (2, 3, 0, 1)
  x = add(x, std::integral_constant<int, 0x141>());  // the other quad of 8 lanes (half row mirrored)
  if constexpr (RG >= 16) x = add(x, std::integral_constant<int, 0x140>());  // the other 8 of 16 (row mirrored)
  if constexpr (RG >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return x;
}

// what the l2 norm multiplies a head by; without an eps zeros stay zeros (a chunk's rows behind the end are such)
__device__ __forceinline__ float norm_factor(float square, float eps) {
  const float x = square + eps;
  return eps < 0.f || x == 0.f ? 1.f : rsqrtf(x);
}

template <int DT>
__device__ __forceinline__ float scalar_at(const void* p, int64_t i, int f32) {
  if (f32) return ((const float*)p)[i];
  const uint16_t x = ((const uint16_t*)p)[i];
  return DT == LSURGE_F16 ? f16_to_f32(x) : bf16_to_f32(x);
}

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <int DT>
__device__ __forceinline__ void unpack2(uint32_t x, float& lo, float& hi) {
  if constexpr (DT == LSURGE_F16) {
    lo = f16_to_f32((uint16_t)x);
    hi = f16_to_f32((uint16_t)(x >> 16));
  } else {
    lo = __uint_as_float(x << 16);
    hi = __uint_as_float(x & 0xffff0000u);
  }
}

// One (sequence, value head), its rows [begin, end) and slot.
struct Unit {
  int b, h, begin, end, slot;
};
__device__ __forceinline__ Unit unit_of(const TokenArgs& a, int sh) {
  Unit u;
  u.h = sh % a.hv, u.b = sh / a.hv;
  u.begin = a.cu ? lsrows::end_at(a.cu, u.b, a.rows) : u.b;
  u.end = a.cu ? lsrows::end_at(a.cu, u.b + 1, a.rows) : u.b + 1;
  u.slot = a.slots ? a.slots[u.b] : u.b;
  return u;
}
// workgroup i of n: the rows before the first sequence and behind the last give zeros
__device__ __forceinline__ void clear_others(const TokenArgs& a, int i, int n) {
  const int64_t row = (int64_t)a.hv * (D / 8);  // 16-byte pieces
  const int64_t before = a.nseq ? lsrows::end_at(a.cu, 0, a.rows) * row : 0;
  const int64_t behind = a.nseq ? lsrows::end_at(a.cu, a.nseq, a.rows) * row : 0;
  u32x4* o = reinterpret_cast<u32x4*>(a.o);
  const int64_t j0 = (int64_t)i * blockDim.x + threadIdx.x, step = (int64_t)n * blockDim.x;
  for (int64_t j = j0; j < before; j += step) o[j] = u32x4{0u, 0u, 0u, 0u};
  for (int64_t j = behind + j0; j < a.rows * row; j += step) o[j] = u32x4{0u, 0u, 0u, 0u};
}

// Columns `col0` .. + CB - 1 through a unit's tokens by one wave, token by token: lane l holds the rows R (l % RG) .. + R - 1 of
// the columns 4 (l / RG) .. + 3, RG = 256 / CB lanes a column.
template <int DT, int CB, bool BETA32>
__device__ __forceinline__ void walk_tokens(const TokenArgs& a, const Unit& u, int col0, int lane) {
  constexpr int RG = 256 / CB, R = D / RG, V = R / 8 > 0 ? R / 8 : 1;  // V: 16-byte loads of a lane's rows of q or k
  const int rg = lane % RG, col = col0 + lane / RG * 4, h = u.h;
  uint16_t* o = a.o + (int64_t)h * D + col;
  const int64_t o_row = (int64_t)a.hv * D;
  if ((unsigned)u.slot >= (unsigned)a.num_slots) {
    if (rg == 0)
      for (int t = u.begin; t < u.end; ++t) *reinterpret_cast<u32x2*>(o + t * o_row) = u32x2{0u, 0u};
    return;
  }
  float* sp = a.state + u.slot * a.slot_stride + (int64_t)h * D * D + (int64_t)rg * R * D + col;
  f32x4 S[R];
#pragma unroll
  for (int i = 0; i < R; ++i) S[i] = *reinterpret_cast<const f32x4*>(sp + i * D);

  const int kh = h / (a.hv / a.hk);
  const uint16_t* qp = a.q + kh * a.q_head + rg * R;
  const uint16_t* kp = a.k + kh * a.k_head + rg * R;
  const uint16_t* vp = a.v + h * a.v_head + col;
  struct Token {
    u32x4 q[V], k[V];
    u32x2 v;
    float g, beta;
  };
  auto load = [&](int t, Token& x) {
    if constexpr (R >= 8) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        x.q[i] = reinterpret_cast<const u32x4*>(qp + t * a.q_row)[i];
        x.k[i] = reinterpret_cast<const u32x4*>(kp + t * a.k_row)[i];
      }
    } else {
      const u32x2 q2 = *reinterpret_cast<const u32x2*>(qp + t * a.q_row), k2 = *reinterpret_cast<const u32x2*>(kp + t * a.k_row);
      x.q[0] = u32x4{q2[0], q2[1], 0u, 0u};
      x.k[0] = u32x4{k2[0], k2[1], 0u, 0u};
    }
    x.v = *reinterpret_cast<const u32x2*>(vp + t * a.v_row);
    x.g = a.g[t * a.g_row + h];
    x.beta = scalar_at<DT>(a.beta, t * a.beta_row + h, BETA32);
  };
  Token cur, next;
  load(u.begin, next);
  for (int t = u.begin; t < u.end; ++t) {
    cur = next;
    load(min(t + 1, u.end - 1), next);
    float q[8 * V], k[8 * V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      lsrows::unpack8<DT>(cur.q[i], q + 8 * i);
      lsrows::unpack8<DT>(cur.k[i], k + 8 * i);
    }
    const float decay = expf(cur.g);
    float kk = 0.f, qq = 0.f, kq = 0.f;
    f32x4 kS{0.f, 0.f, 0.f, 0.f}, qS{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < R; ++i) {
      kk = fmaf(k[i], k[i], kk);
      qq = fmaf(q[i], q[i], qq);
      kq = fmaf(k[i], q[i], kq);
      S[i] *= decay;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        kS[j] = fmaf(k[i], S[i][j], kS[j]);
        qS[j] = fmaf(q[i], S[i][j], qS[j]);
      }
    }
    kq = group_sum<RG>(kq);
    float rk = 1.f, rq = 0.08838834764831845f;  // 1 / sqrt(128)
    if (a.l2_eps >= 0.f) {
      rk = norm_factor(group_sum<RG>(kk), a.l2_eps);
      rq *= norm_factor(group_sum<RG>(qq), a.l2_eps);
    }
    float v[4], out[4], kd[4];
    unpack2<DT>(cur.v[0], v[0], v[1]);
    unpack2<DT>(cur.v[1], v[2], v[3]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      kd[j] = rk * (cur.beta * fmaf(-rk, group_sum<RG>(kS[j]), v[j]));  // rk d
      out[j] = rq * fmaf(kq, kd[j], group_sum<RG>(qS[j]));
    }
    if (rg == 0)
      *reinterpret_cast<u32x2*>(o + t * o_row) = u32x2{lsrows::pack2<DT>(out[0], out[1]), lsrows::pack2<DT>(out[2], out[3])};
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) S[i][j] = fmaf(k[i], kd[j], S[i][j]);
  }
#pragma unroll
  for (int i = 0; i < R; ++i) *reinterpret_cast<f32x4*>(sp + i * D) = S[i];
}

// One token for each sequence.
template <int DT, int CB, bool BETA32>
__global__ __launch_bounds__(64 * WAVES) void gdn_token_kernel(TokenArgs a) {
  constexpr int BLOCKS = D / CB / WAVES;  // workgroups a (sequence, head)
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Unit u = unit_of(a, blockIdx.x / BLOCKS);
  if (u.begin < u.end) walk_tokens<DT, CB, BETA32>(a, u, (blockIdx.x % BLOCKS * WAVES + wave) * CB, lane);
}

// ------------------------------------------------------------------------------------ runs of tokens
// Sequences of any length, packed.  From CHUNKED tokens on a sequence goes in chunks of C = 32.  With G_i the sum of the log
// decays up to token i of a chunk, S0 the state before it, and k and q normalised,
//   (I + A) X = R,  R_i = beta_i (v_i - e^{G_i} S0^T k_i),  A_ij = beta_i e^{G_i - G_j} k_i.k_j (j < i),
//   o_i = (e^{G_i} S0^T q_i + sum_{j <= i} e^{G_i - G_j} (q_i.k_j) x_j) / sqrt(128),
//   S = e^{G_C} S0 + sum_j e^{G_C - G_j} k_j x_j^T
// (row i of X is the token's d).  A and the weights of o do not depend on the state: a pair of waves forms them a chunk
// ahead, or two pairs in turn two chunks ahead, while two or four waves of 16 columns each take this one; one barrier a chunk.
//
// Every product runs on the matrix cores of 16-bit operands with f32 sums.  The inputs are exact operands; f32 ones are sums of
// terms of 16 bits.  Against inputs, three bf16 terms hold all 24 bits; two f16 ones leave up to 2^-23 of a value over, two
// roundings of f32 (the first leaves 12 bits and a sign, the second holds 11), since a third would take a prompt of 2000 tokens
// from 109 to 128 us.  f16's range is short, so a column of the state is kept times a power of two there, its largest value
// between 2^8 and 2^15: what is lost of small values is below 2^-33 of it; the power ends at 2^60, so a column below 2^-52,
// nothing beside f16 inputs, loses 2^-85.
// The 16 x 16 matrices R, X, A, the inverse of A's diagonal blocks and the weights of o are three bf16 terms: o is held to f32
// before its own rounding too, since a token that reads what it erases is a small difference of large parts (with two terms for
// o's parts 12 prompts took 103 us instead of 112).  A wave's 16 columns of every matrix lie in its lanes (lane l: column
// l % 16), so that each product's result is in place as the next one's operand: the state, R and X never leave their lane.
// (I + A) is solved by blocks of 16: X0 = B0 R0, X1 = B1 (R1 - A10 X0), B the inverses of the diagonal blocks.  Log decays are
// summed in 64 bits, since differences of sums go into exponents.
constexpr int C = 32;
// us token by token and in a chunk: 100 sequences of 8 heads with 2 tokens each 27 and 30 (f16: 27 and 28), 3 30 and 30 (30 and
// 28), 4 33 and 30 (33 and 28), 5 37 and 30, 7 43 and 31; 4 sequences with 3 5.4 and 6.2, 4 6.2 and 6.3, 5 7.0 and 6.2.
constexpr int CHUNKED = 4;
constexpr int64_t MOST_ROW = 1ll << 22;  // elements between rows: a chunk's are within 32 bits of bytes
constexpr float QSCALE = 0.08838834764831845f;  // 1 / sqrt(128)

// a barrier behind this wave's writes to LDS; loads from memory go on across it
__device__ __forceinline__ void stage_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// A row's 16 bytes 4 b + g hold the values 32 b + 4 g .. + 3 and 32 b + 16 + 4 g .. + 3, as the products with the state take them.
// Rows 32 bytes apart in the banks: reads of a row's 16 bytes by 16 rows, which is most of them, meet no bank twice.
constexpr int PITCH = D + 16;
struct ChunkTiles {
  uint16_t k[C][PITCH], q[C][PITCH];
};
struct ChunkTerms {
  // operands of products over 16 tokens, lane l's four values (row l % 16, columns 4 (l / 16) .. + 3) at [l]
  u32x2 inv[2][3][64];  // the inverses of the diagonal blocks of I + A, by terms as `left` takes them
  u32x2 a10[3][64];     // -A, rows 16.., columns ..15
  u32x2 m00[3][64];     // the weights of o
  u32x2 m1[2][3][64];   // their rows 16.., columns by halves
  // by token: R = beta v - c1 (S0^T k), o = c2 (S0^T q) + .., the factor of k in the state's update
  float beta[C], c1[C], c2[C], w[C];
  float decay;
};

template <int DT>
__device__ __forceinline__ f32x4 mma_32(u32x4 p, u32x4 q, f32x4 c) {  // D[16 x 16] += P[16 x 32] Q[32 x 16]
  typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
  if constexpr (DT == LSURGE_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, p), __builtin_bit_cast(f16x8_t, q), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, p), __builtin_bit_cast(bf16x8, q), c, 0, 0, 0);
}
// c minus the lower (HIGH: the upper) value of a register of two
template <int DT, bool HIGH>
__device__ __forceinline__ float minus(uint32_t x, float c) {
  if constexpr (DT == LSURGE_F16) {
    const lsrows::f16x2_t one{(_Float16)(HIGH ? 0.f : -1.f), (_Float16)(HIGH ? -1.f : 0.f)};
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(lsrows::f16x2_t, x), one, c, false);
  } else {
    uint32_t one = HIGH ? 0xbf800000u : 0xbf80u;
    asm("" : "+s"(one));  // as a literal the compiler encodes (-1, 0) as (-1, -1)
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, x), __builtin_bit_cast(bf16x2_t, one), c, false);
  }
}
// x as a sum of N terms of DT, four values each.  What a term leaves over is exact.  The dot product overwrites its c, and a
// copy of x and it are no fewer instructions than a shift and a difference: bf16's first term takes these (2% of a long run).
template <int DT, int N>
__device__ __forceinline__ void split(f32x4 x, u32x2* t) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    t[n] = u32x2{lsrows::pack2<DT>(x[0], x[1]), lsrows::pack2<DT>(x[2], x[3])};
    if (n + 1 < N) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (DT == LSURGE_BF16 && n == 0) {
          x[2 * i] -= __uint_as_float(t[n][i] << 16);
          x[2 * i + 1] -= __uint_as_float(t[n][i] & 0xffff0000u);
        } else {
          x[2 * i] = minus<DT, false>(t[n][i], x[2 * i]);
          x[2 * i + 1] = minus<DT, true>(t[n][i], x[2 * i + 1]);
        }
      }
    }
  }
}
template <int N>
__device__ __forceinline__ void split(f32x4 x, u32x2* t) { split<LSURGE_BF16, N>(x, t); }
// orders a wave's accesses to LDS between its lanes
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
__device__ __forceinline__ u32x4 join(u32x2 a, u32x2 b) { return u32x4{a[0], a[1], b[0], b[1]}; }
// 16 x 16 operands (lane l: row / column l % 16 at 4 (l / 16) .. + 3), whose terms are taken two at a time.  They lie so that
// every pair is a range of registers: 1, 0, 2 of a left one, 2, 0, 1, 0 of a right one.
typedef uint32_t u32x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ u32x8 left(const u32x2 (*t)[64], int lane) {
  const u32x2 a = t[0][lane], b = t[1][lane], c = t[2][lane];
  return u32x8{a[0], a[1], b[0], b[1], c[0], c[1], 0u, 0u};
}
__device__ __forceinline__ u32x8 right(f32x4 x) {
  u32x2 t[3];
  split<3>(x, t);
  return u32x8{t[2][0], t[2][1], t[0][0], t[0][1], t[1][0], t[1][1], t[0][0], t[0][1]};
}
template <int AT>
__device__ __forceinline__ u32x4 pair(u32x8 x) { return __builtin_shufflevector(x, x, AT, AT + 1, AT + 2, AT + 3); }
// c + P Q: the six products of 2^-24 and more
__device__ __forceinline__ f32x4 mma_f32(u32x8 p, u32x8 q, f32x4 c) {
  f32x4 less = mma_32<LSURGE_BF16>(pair<2>(p), pair<0>(q), f32x4{0.f, 0.f, 0.f, 0.f});
  c = mma_32<LSURGE_BF16>(pair<0>(p), pair<4>(q), c);
  less = mma_32<LSURGE_BF16>(pair<0>(p), pair<2>(q), less);
  return c + less;
}
// the same six, one after the other
__device__ __forceinline__ f32x4 mma_f32_on(u32x8 p, u32x8 q, f32x4 c) {
  c = mma_32<LSURGE_BF16>(pair<2>(p), pair<0>(q), c);
  c = mma_32<LSURGE_BF16>(pair<0>(p), pair<2>(q), c);
  return mma_32<LSURGE_BF16>(pair<0>(p), pair<4>(q), c);
}

// A pair of waves forms a chunk's terms from its tiles.
struct Scratch {
  double G[C];  // sums of the log2 decays
  float rk[C], rq[C], beta[C];
};
// operand of a tile's tokens 16 i .. + 15, values 32 s .. + 31
__device__ __forceinline__ u32x4 token_frag(const uint16_t (*rows)[PITCH], int i, int s, int lane) {
  return *reinterpret_cast<const u32x4*>(&rows[16 * i + (lane & 15)][32 * s + 8 * (lane >> 4)]);
}
// The sum of the log2 decays up to token lane % 32, and of all.  A decay below e^-104 is 0 in f32 whatever it is.
__device__ __forceinline__ double decay_sums(float decay, double& last) {
  const double x = (double)(decay < -104.f ? -104.f : decay) * 1.4426950408889634;
  auto add = [](double v, auto ctrl, auto rows) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    constexpr int CT = decltype(ctrl)::value, RM = decltype(rows)::value;
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CT, RM, 0xf, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CT, RM, 0xf, true);
    return v + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
  };
  typedef std::integral_constant<int, 0xf> All;
  double G = x;
  G = add(G, std::integral_constant<int, 0x111>(), All());  // the lane 1, 2, 4, 8 before it in a row of 16
  G = add(G, std::integral_constant<int, 0x112>(), All());
  G = add(G, std::integral_constant<int, 0x114>(), All());
  G = add(G, std::integral_constant<int, 0x118>(), All());
  G = add(G, std::integral_constant<int, 0x142>(), std::integral_constant<int, 0xa>());  // the last lane of the row before
  const uint64_t u = __builtin_bit_cast(uint64_t, G);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, C - 1), hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), C - 1);
  last = __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
  return G;
}
// the element of a diagonal block's product that lies on its diagonal, in the lanes that hold one (on_diagonal)
__device__ __forceinline__ bool on_diagonal(int lane) { return lane >> 4 == (lane & 15) >> 2; }
__device__ __forceinline__ float diagonal(f32x4 x, int lane) {
  float d = x[0];
#pragma unroll
  for (int r = 1; r < 4; ++r)
    if ((lane & 3) == r) d = x[r];
  return d;
}

// e^{G_i - G_j} times k's factor, j = j0 .. + 3; without branches, whose loads would wait one after the other
__device__ __forceinline__ f32x4 decays(const Scratch& s, int i, int j0) {
  typedef double f64x2 __attribute__((ext_vector_type(2)));
  const double Gi = s.G[i];
  const f64x2 a = *reinterpret_cast<const f64x2*>(&s.G[j0]), b = *reinterpret_cast<const f64x2*>(&s.G[j0 + 2]);
  const f32x4 rk = *reinterpret_cast<const f32x4*>(&s.rk[j0]);
  return f32x4{rk[0] * __builtin_amdgcn_exp2f((float)(Gi - a[0])), rk[1] * __builtin_amdgcn_exp2f((float)(Gi - a[1])),
               rk[2] * __builtin_amdgcn_exp2f((float)(Gi - b[0])), rk[3] * __builtin_amdgcn_exp2f((float)(Gi - b[1]))};
}
// y[j] += y[k] A_kj for four j from J on (those below k), A_kj from lane k of the row of 16.  In assembly, since the compiler
// takes a move and a multiply-add for each; the nop is what a register needs between its last write and a read across lanes.
template <int K, int J>
__device__ __forceinline__ void subtract_4(float* y, const float* A) {
  if constexpr (J + 4 <= K)
    asm("s_nop 1\n\t"
        "v_fmac_f32_dpp %0, %4, %8 row_newbcast:%c9 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %1, %5, %8 row_newbcast:%c9 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %2, %6, %8 row_newbcast:%c9 row_mask:0xf bank_mask:0xf\n\t"
        "v_fmac_f32_dpp %3, %7, %8 row_newbcast:%c9 row_mask:0xf bank_mask:0xf"
        : "+&v"(y[J]), "+&v"(y[J + 1]), "+&v"(y[J + 2]), "+&v"(y[J + 3])
        : "v"(A[J]), "v"(A[J + 1]), "v"(A[J + 2]), "v"(A[J + 3]), "v"(y[K]), "n"(K));
  else
#pragma unroll
    for (int j = J; j < K; ++j)
      asm("s_nop 1\n\tv_fmac_f32_dpp %0, %1, %2 row_newbcast:%c3 row_mask:0xf bank_mask:0xf"
          : "+v"(y[j]) : "v"(A[j]), "v"(y[K]), "n"(K));
}
template <int... STEP>
__device__ __forceinline__ void subtract_rows(float* y, const float* A, std::integer_sequence<int, STEP...>) {
  ((subtract_4<15 - STEP, 0>(y, A), subtract_4<15 - STEP, 4>(y, A), subtract_4<15 - STEP, 8>(y, A),
    subtract_4<15 - STEP, 12>(y, A)), ...);
}

// The inverses of A's diagonal blocks; the log decay and beta are those of token lane % 32 (0 behind the end).
// half: called half way.
template <int DT, class F>
__device__ __forceinline__ void prepare_inverse(const ChunkTiles& x, float decay, float beta, float l2_eps, int lane, Scratch& s,
                                                float (*blocks)[16][20], ChunkTerms& out, F half) {
  asm volatile("" : "+v"(lane));  // LDS addresses are formed again in every chunk, not kept in registers that spill
  const int c = lane & 15, g = lane >> 4, t = lane & 31;
  u32x4 k[2][4];
#pragma unroll
  for (int st = 0; st < 4; ++st) k[0][st] = token_frag(x.k, 0, st, lane), k[1][st] = token_frag(x.k, 1, st, lane);
  double last;
  const double G = decay_sums(decay, last);
  if (lane < C) s.G[t] = G, s.beta[t] = beta;
  f32x4 kk[2];  // blocks (0, 0), (1, 1) of products [token j][token i], lane: i = c, j = 4 g + r
#pragma unroll
  for (int i = 0; i < 2; ++i) kk[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int st = 0; st < 4; ++st)
#pragma unroll
    for (int i = 0; i < 2; ++i) kk[i] = mma_32<DT>(k[i][st], k[i][st], kk[i]);
  if (on_diagonal(lane)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) s.rk[16 * i + c] = norm_factor(diagonal(kk[i], lane), l2_eps);
  }
  wave_sync();
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const int i = 16 * b + c, j0 = 16 * b + 4 * g;
    const f32x4 e = decays(s, i, j0);
    const float f = -s.beta[i] * s.rk[i];
    f32x4 A;
#pragma unroll
    for (int r = 0; r < 4; ++r) A[r] = j0 + r < i ? f * (e[r] * kk[b][r]) : 0.f;
    *reinterpret_cast<f32x4*>(&blocks[b][c][4 * g]) = A;
  }
  wave_sync();
  half();
  // Row c of a block's inverse, y (I + A) = e_c, from its last value on; lanes below 32 the first block, the others the second.
  // Lane k of a row of 16 holds row k of -A, which the others read from its register as they go: 120 multiply-adds, no LDS.
  const int blk = lane >> 5;
  float y[16], A[16];
#pragma unroll
  for (int j = 0; j < 16; j += 4) {
    const f32x4 x4 = *reinterpret_cast<const f32x4*>(&blocks[blk][c][j]);
#pragma unroll
    for (int r = 0; r < 4; ++r) A[j + r] = x4[r], y[j + r] = j + r == c ? 1.f : 0.f;
  }
  subtract_rows(y, A, std::make_integer_sequence<int, 15>());
  // its columns 8 (g % 2) .. + 7 as operands
  u32x2 terms[3];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    f32x4 z;
#pragma unroll
    for (int r = 0; r < 4; ++r) z[r] = g & 1 ? y[8 + 4 * h + r] : y[4 * h + r];
    split<3>(z, terms);
#pragma unroll
    for (int n = 0; n < 3; ++n) out.inv[blk][n < 2 ? 1 - n : 2][c + 16 * (2 * (g & 1) + h)] = terms[n];
  }
}

// Everything else: A's block (1, 0), the weights of o, the factors by token.
template <int DT, class F>
__device__ __forceinline__ void prepare_rest(const ChunkTiles& x, float decay, float beta, float l2_eps, int lane, Scratch& s,
                                             ChunkTerms& out, F half) {
  asm volatile("" : "+v"(lane));
  const int c = lane & 15, g = lane >> 4, t = lane & 31;
  double last;
  const double G = decay_sums(decay, last);
  if (lane < C) s.G[t] = G, s.beta[t] = beta;
  const f32x4 zero{0.f, 0.f, 0.f, 0.f};
  // blocks (0, 0), (1, 1), (0, 1) of products [token j][token i], lane: i = c, j = 4 g + r
  f32x4 kk[3] = {zero, zero, zero}, kq[3] = {zero, zero, zero}, qq[2] = {zero, zero};
#pragma unroll
  for (int st = 0; st < 4; ++st) {
    u32x4 k[2], q[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) k[i] = token_frag(x.k, i, st, lane), q[i] = token_frag(x.q, i, st, lane);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      kk[i] = mma_32<DT>(k[i], k[i], kk[i]);
      kq[i] = mma_32<DT>(k[i], q[i], kq[i]);
      qq[i] = mma_32<DT>(q[i], q[i], qq[i]);
    }
    kk[2] = mma_32<DT>(k[0], k[1], kk[2]);
    kq[2] = mma_32<DT>(k[0], q[1], kq[2]);
  }
  if (on_diagonal(lane)) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s.rk[16 * i + c] = norm_factor(diagonal(kk[i], lane), l2_eps);
      s.rq[16 * i + c] = QSCALE * norm_factor(diagonal(qq[i], lane), l2_eps);
    }
  }
  wave_sync();
  half();
  if (lane < C) {
    const float rk = s.rk[t], e = __builtin_amdgcn_exp2f((float)G);
    out.beta[t] = beta;
    out.c1[t] = beta * e * rk;
    out.c2[t] = e * s.rq[t];
    out.w[t] = rk * __builtin_amdgcn_exp2f((float)(last - G));
    if (t == 0) out.decay = __builtin_amdgcn_exp2f((float)last);
  }
#pragma unroll
  for (int b = 0; b < 3; ++b) {
    const int i = (b == 0 ? 0 : 16) + c, j0 = (b == 1 ? 16 : 0) + 4 * g;
    const f32x4 e = decays(s, i, j0);
    const float f = s.rq[i];
    f32x4 m;
#pragma unroll
    for (int r = 0; r < 4; ++r) m[r] = j0 + r <= i ? f * (e[r] * kq[b][r]) : 0.f;
    u32x2 terms[3];
    split<3>(m, terms);
#pragma unroll
    for (int n = 0; n < 3; ++n) (b == 0 ? out.m00 : out.m1[b == 1])[n < 2 ? 1 - n : 2][lane] = terms[n];
    if (b == 2) {
      split<3>(-s.beta[i] * s.rk[i] * (e * kk[2]), terms);
#pragma unroll
      for (int n = 0; n < 3; ++n) out.a10[n < 2 ? 1 - n : 2][lane] = terms[n];
    }
  }
}

// A unit's rows chunk by chunk, `width` values of `size` bytes each and `row` values apart, as buffers that end with the
// sequence: behind it reads give 0 and writes are dropped.
struct ChunkRows {
  const char* at;
  int64_t step;        // bytes a chunk
  int left, row, tail;  // rows left; bytes a row, and of the last one short of that
  __device__ __forceinline__ ChunkRows(const Unit& u, const void* head, int64_t row_, int width, int size)
      : at((const char*)head + u.begin * row_ * size), step(C * row_ * size), left(u.end - u.begin), row((int)row_ * size),
        tail((int)row_ * size - width * size) {}
  __device__ __forceinline__ auto next() {
    const int bytes = max(min(left, C) * row - tail, 0);
    const auto b = __builtin_amdgcn_make_buffer_rsrc((void*)at, (short)0, left > 0 ? bytes : 0, 0x00027000);
    at += step, left -= C;
    return b;
  }
};

// the largest of a column's values, from each of the four lanes that hold it
__device__ __forceinline__ float column_max(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// S, its scale and a column's `most` changed by a power of two that brings `most` to 2^12 .. 2^13, where it is outside
// [2^8, 2^15)
__device__ __forceinline__ void rescale(float& most, f32x4* S, float& scale, float& unscale) {
  const bool out = most < 0x1p8f || most >= 0x1p15f;
  if (__ballot(out) == 0) return;
  const int e = out && most > 0.f ? (int)(__float_as_uint(most) >> 23) - 127 : 12;  // 2^e <= most < 2^(e + 1)
  const int now = (int)(__float_as_uint(scale) >> 23) - 127;
  const int n = min(max(12 - e, -60 - now), 60 - now);  // the scale within 2^-60 .. 2^60
  const float up = __uint_as_float((uint32_t)(127 + n) << 23), down = __uint_as_float((uint32_t)(127 - n) << 23);
#pragma unroll
  for (int m = 0; m < 8; ++m) S[m] *= up;
  most *= up, scale *= up, unscale *= down;
}

// NW waves take columns, PAIRS pairs of waves prepare: one pair during the chunk before, two in turn during two.
template <int DT, bool BETA32, int NW, int PAIRS>
__global__ __launch_bounds__(64 * (NW + 2 * PAIRS), NW == 4 && PAIRS == 1 ? 3 : 2) void gdn_run_kernel(TokenArgs a) {
  constexpr int PARTS = D / (16 * NW);  // workgroups a (sequence, head)
  constexpr int RING = PAIRS + 2;
  constexpr int NT = DT == LSURGE_F16 ? 2 : 3;  // terms of f32 operands against k and q
  __shared__ ChunkTiles tiles[RING];
  __shared__ ChunkTerms terms[2];
  __shared__ Scratch scratch[2 * PAIRS];
  __shared__ float blocks[PAIRS][2][16][20];  // the diagonal blocks of -A, rows 16 bytes apart
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if ((int)blockIdx.x >= a.units) return clear_others(a, blockIdx.x - a.units, gridDim.x - a.units);
  const Unit u = unit_of(a, blockIdx.x / PARTS);
  const int col0 = (blockIdx.x % PARTS * NW + wave) * 16;
  const int total = u.end - u.begin;
  if (total <= 0) return;
  if (total < CHUNKED || (unsigned)u.slot >= (unsigned)a.num_slots) {
    if (wave < NW) walk_tokens<DT, 16, BETA32>(a, u, col0, lane);
    return;
  }
  const int chunks = (total + C - 1) / C;
  const int c = lane & 15, g = lane >> 4;

  // The first four waves stage: a thread's part of the tiles is two pieces of 8 values of k and of q.
  const int kh = u.h / (a.hv / a.hk), srow = threadIdx.x >> 4, scol = (threadIdx.x & 15) * 8;
  const int place = scol / 32 * 32 + scol % 16 * 2 + scol % 32 / 16 * 4;  // its first four values' place, its others' 8 further
  int k_off = (srow * (int)a.k_row + scol) * 2, q_off = (srow * (int)a.q_row + scol) * 2;
  u32x4 kr[2], qr[2];
  ChunkRows ks(u, a.k + kh * a.k_head, a.k_row, D, 2), qs(u, a.q + kh * a.q_head, a.q_row, D, 2);
  auto load_tiles = [&]() {
    const auto kb = ks.next(), qb = qs.next();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      kr[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(kb, k_off + 32 * i * (int)a.k_row, 0, 0));
      qr[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(qb, q_off + 32 * i * (int)a.q_row, 0, 0));
    }
  };
  auto store_tiles = [&](ChunkTiles& x) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      *reinterpret_cast<u32x2*>(&x.k[srow + 16 * i][place]) = u32x2{kr[i][0], kr[i][1]};
      *reinterpret_cast<u32x2*>(&x.k[srow + 16 * i][place + 8]) = u32x2{kr[i][2], kr[i][3]};
      *reinterpret_cast<u32x2*>(&x.q[srow + 16 * i][place]) = u32x2{qr[i][0], qr[i][1]};
      *reinterpret_cast<u32x2*>(&x.q[srow + 16 * i][place + 8]) = u32x2{qr[i][2], qr[i][3]};
    }
  };

  // Between barriers n and n + 1 the takers take chunk n - PAIRS, the pair of chunk n begins to prepare it, and chunk n + 1 is
  // staged; a chunk is prepared PAIRS barriers after its begin.
  if (wave >= NW) {
    constexpr bool stages = NW == 2;  // two of the first four waves
    const int mine = __builtin_amdgcn_readfirstlane(wave) - NW, pair = mine >> 1;  // scalar: barriers depend on them
    const int g_off = (lane & 31) * (int)a.g_row * 4, b_size = BETA32 ? 4 : 2, b_off = (lane & 31) * (int)a.beta_row * b_size;
    ChunkRows gs(u, a.g + u.h, a.g_row, 1, 4), bs(u, (const char*)a.beta + u.h * b_size, a.beta_row, 1, b_size);
    auto load = [&](float& decay, float& beta) {
      const auto gb = gs.next(), bb = bs.next();
      decay = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(gb, g_off, 0, 0));
      if constexpr (BETA32) {
        beta = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(bb, b_off, 0, 0));
      } else {
        const uint16_t x = __builtin_amdgcn_raw_buffer_load_b16(bb, b_off, 0, 0);
        beta = DT == LSURGE_F16 ? f16_to_f32(x) : bf16_to_f32(x);
      }
    };
    auto skip = [&]() {
      gs.next();
      bs.next();
    };
    float decay, beta, decay1, beta1;
    if (stages) load_tiles();
    if (pair) skip();
    load(decay, beta);
    if (stages) store_tiles(tiles[0]), load_tiles();
    stage_barrier();  // the first chunk is staged
    if (pair) stage_barrier();
    int barriers = 1 + pair;
    for (int n = pair, ring = pair; n < chunks; n += PAIRS) {
      const ChunkTiles& tile = tiles[ring];
      ring = ring + PAIRS < RING ? ring + PAIRS : ring + PAIRS - RING;  // n % RING
      if (stages) {
        asm volatile("" : "+v"(k_off), "+v"(q_off));
        store_tiles(tiles[ring]);
        load_tiles();
      }
      if (PAIRS == 2) skip();
      load(decay1, beta1);
      auto half = [&]() {
        if (PAIRS == 2) stage_barrier();
      };
      if (mine & 1) prepare_rest<DT>(tile, decay, beta, a.l2_eps, lane, scratch[mine], terms[n & 1], half);
      else prepare_inverse<DT>(tile, decay, beta, a.l2_eps, lane, scratch[mine], blocks[pair], terms[n & 1], half);
      decay = decay1, beta = beta1;
      stage_barrier();  // chunk n is prepared
      barriers += PAIRS;
    }
    for (; barriers < chunks + PAIRS; ++barriers) stage_barrier();  // as many as the takers'
    return;
  }
  static_assert(NW == 4 || PAIRS == 1, "a preparing wave that stages does so once a barrier");

  // the columns col0 .. + 15 of the state: tile m, register r: row 16 m + 4 g + r, column c
  float* sp = a.state + u.slot * a.slot_stride + (int64_t)u.h * D * D + 4 * g * D + col0 + c;
  f32x4 S[8];
  float scale = 1.f, unscale = 1.f;  // f16: S holds the state times `scale`, a power of two of the column's own
#pragma unroll
  for (int m = 0; m < 8; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) S[m][r] = sp[(16 * m + r) * D];

  const int o_row = a.hv * D;
  int v_off = (4 * g * (int)a.v_row + col0 + c) * 2, o_off = (4 * g * o_row + col0 + c) * 2;
  uint16_t vr[8];
  ChunkRows vs(u, a.v + u.h * a.v_head, a.v_row, D, 2), os(u, a.o + (int64_t)u.h * D, o_row, D, 2);
  auto load_v = [&]() {
    const auto vb = vs.next();
#pragma unroll
    for (int i = 0; i < 8; ++i)
      vr[i] = __builtin_amdgcn_raw_buffer_load_b16(vb, v_off + (32 * (i >> 2) + 2 * (i & 3)) * (int)a.v_row, 0, 0);
  };
  load_tiles();
  store_tiles(tiles[0]);
  load_tiles();
  stage_barrier();  // the first chunk is staged
  store_tiles(tiles[1]);
  load_tiles();
  if (PAIRS == 2) {
    stage_barrier();
    store_tiles(tiles[2]);
    load_tiles();
  }
  __builtin_amdgcn_sched_barrier(0);  // in the loop's order, or its first wait is for all of them in every turn
  load_v();
  u32x2 s[2][2][NT];  // two tiles of the state by terms, and the next two
  if constexpr (DT == LSURGE_BF16) split<DT, NT>(S[0], s[0][0]), split<DT, NT>(S[1], s[0][1]);

  int ring = 0;  // n % RING
  for (int n = 0; n < chunks; ++n) {
    stage_barrier();  // chunk n is prepared, chunk n + PAIRS staged, chunk n - 1 no longer read
    const ChunkTiles& tile = tiles[ring];
    const ChunkTerms& x = terms[n & 1];
    // the addresses' multiples of the rows are added again in every chunk: kept, they spill, and a spill's reload waits for
    // all loads before it
    asm volatile("" : "+v"(k_off), "+v"(q_off), "+v"(v_off), "+v"(o_off));
    // Operands are read from LDS a step before their products: k and q of the tokens 16 i + c, at the state's rows
    // 32 st + {4 g .. + 3, 16 + 4 g .. + 3}, in that order.
    u32x4 kf[2][2], qf[2][2];
    auto frags = [&](int st) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        kf[st & 1][i] = token_frag(tile.k, i, st, lane);
        qf[st & 1][i] = token_frag(tile.q, i, st, lane);
      }
    };
    frags(0);
    store_tiles(tiles[ring == 0 ? RING - 1 : ring - 1]);  // of chunk n + RING - 1, zeros behind the last
    load_tiles();
    ring = ring == RING - 1 ? 0 : ring + 1;
    float most = 0.f;  // f16: the largest of the column's values
    if constexpr (DT == LSURGE_F16) {
#pragma unroll
      for (int m = 0; m < 8; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) most = fmaxf(most, fabsf(S[m][r]));
      most = column_max(most);
      rescale(most, S, scale, unscale);
      split<DT, NT>(S[0], s[0][0]);
      split<DT, NT>(S[1], s[0][1]);
    }
    // P = K S0, O = Q S0 by halves of the tokens; the next step's state is split between this one's products
    f32x4 P[2], O[2];
    const f32x4 zero{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2; ++i) P[i] = O[i] = zero;
    u32x8 inv0, inv1, a10, m00, m1[2];
    f32x4 beta[2], c1[2], c2[2], w[2];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int st = 0; st < 4; ++st) {
      if (st < 3) {
        frags(st + 1);
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int t = 16 * i + 4 * g;
          beta[i] = *reinterpret_cast<const f32x4*>(&x.beta[t]), c1[i] = *reinterpret_cast<const f32x4*>(&x.c1[t]);
        }
        inv0 = left(x.inv[0], lane), a10 = left(x.a10, lane), inv1 = left(x.inv[1], lane);
        m00 = left(x.m00, lane), m1[0] = left(x.m1[0], lane), m1[1] = left(x.m1[1], lane);
      }
      const u32x2(*now)[NT] = s[st & 1];
#pragma unroll
      for (int j = NT - 1; j >= 0; --j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          P[i] = mma_32<DT>(kf[st & 1][i], join(now[0][j], now[1][j]), P[i]);
          O[i] = mma_32<DT>(qf[st & 1][i], join(now[0][j], now[1][j]), O[i]);
        }
      if (st < 3) {
        split<DT, NT>(S[2 * st + 2], s[(st + 1) & 1][0]);
        split<DT, NT>(S[2 * st + 3], s[(st + 1) & 1][1]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    // R, and X by blocks of 16 tokens
    f32x4 R[2], X[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float v = DT == LSURGE_F16 ? f16_to_f32(vr[4 * i + r]) : bf16_to_f32(vr[4 * i + r]);
        R[i][r] = fmaf(-c1[i][r] * unscale, P[i][r], beta[i][r] * v);  // 0 behind the end, as beta is
      }
      c2[i] = *reinterpret_cast<const f32x4*>(&x.c2[16 * i + 4 * g]), w[i] = *reinterpret_cast<const f32x4*>(&x.w[16 * i + 4 * g]);
    }
    const float decay = x.decay;
    load_v();
    X[0] = mma_f32(inv0, right(R[0]), zero);
#pragma unroll
    for (int m = 0; m < 4; ++m) S[m] *= decay;  // beside the chain of products
    const u32x8 x0 = right(X[0]);
    X[1] = mma_f32(inv1, right(mma_f32(a10, x0, R[1])), zero);
#pragma unroll
    for (int m = 4; m < 8; ++m) S[m] *= decay;
#pragma unroll
    for (int i = 0; i < 2; ++i) O[i] *= c2[i] * unscale;
    O[0] = mma_f32_on(m00, x0, O[0]);
    O[1] = mma_f32_on(m1[0], x0, O[1]);
    // the state's update
    f32x4 E[2] = {X[0] * w[0], X[1] * w[1]};
    if constexpr (DT == LSURGE_F16) {  // the decayed state's size, or what is added to it
      float added = 0.f;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) added = fmaxf(added, fabsf(E[i][r]));
      most = fmaxf(most * decay, column_max(added) * scale);
      rescale(most, S, scale, unscale);
#pragma unroll
      for (int i = 0; i < 2; ++i) E[i] *= scale;
    }
    u32x4 kt[8];  // k's values 16 m + c of the tokens 4 g .. + 3 and 16 + 4 g .. + 3
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      const uint16_t* p = &tile.k[4 * g + (c >> 2)][32 * (m >> 1) + 8 * (c & 3) + 4 * (m & 1)];
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(s16x4, p));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(LDS_PTR(s16x4, p + 16 * PITCH));
      kt[m] = join(__builtin_bit_cast(u32x2, lo), __builtin_bit_cast(u32x2, hi));
    }
    u32x2 e0[NT], e1[NT];
    split<DT, NT>(E[0], e0);
    split<DT, NT>(E[1], e1);
#pragma unroll
    for (int m = 0; m < 8; m += 2)  // two tiles in turn: a product waits for the one before it
#pragma unroll
      for (int j = NT - 1; j >= 0; --j) {
        S[m] = mma_32<DT>(kt[m], join(e0[j], e1[j]), S[m]);
        S[m + 1] = mma_32<DT>(kt[m + 1], join(e0[j], e1[j]), S[m + 1]);
      }
    if constexpr (DT == LSURGE_BF16) split<DT, NT>(S[0], s[0][0]), split<DT, NT>(S[1], s[0][1]);
    O[1] = mma_f32_on(m1[1], right(X[1]), O[1]);
    const auto ob = os.next();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float o = O[i >> 2][i & 3];
      __builtin_amdgcn_raw_buffer_store_b16(DT == LSURGE_F16 ? f32_to_f16(o) : f32_to_bf16(o), ob,
                                            o_off + (32 * (i >> 2) + 2 * (i & 3)) * o_row, 0, 0);
    }
  }
  asm volatile("" : "+v"(sp));  // its 32 addresses are formed again, not kept in 64 registers through the loop
  auto* to = (__attribute__((address_space(1))) float*)sp;
#pragma unroll
  for (int m = 0; m < 8; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) to[(16 * m + r) * D] = S[m][r] * unscale;
}

int check_tokens(const lsurge_gdn_tokens* t) {
  const char* what = "gdn_recurrent";
  LSURGE_REQUIRE(t, "%s: null arguments", what);
  LSURGE_REQUIRE(t->rows >= 0 && t->rows < (1ll << 30) && t->nseq >= 0 && t->nseq < (1ll << 24) && (t->cu || t->rows == t->nseq),
                 "%s: %lld rows of %lld sequences", what, (long long)t->rows, (long long)t->nseq);
  LSURGE_REQUIRE(t->hk >= 1 && t->hv >= t->hk && t->hv % t->hk == 0 && t->hv <= 65535, "%s: %lld value heads over %lld key heads",
                 what, (long long)t->hv, (long long)t->hk);
  if ((t->dtype != LSURGE_BF16 && t->dtype != LSURGE_F16) || (t->beta_dtype != t->dtype && t->beta_dtype != LSURGE_F32))
    return lsurge::set_error(LSURGE_ERR_DTYPE, "%s: bf16 or f16, beta alike or f32", what);
  if (t->rows == 0) return LSURGE_OK;
  for (const lsurge_attn_rows* r : {&t->q, &t->k, &t->v}) {
    LSURGE_REQUIRE(r->data && (uintptr_t)r->data % 16 == 0, "%s: null or misaligned rows", what);
    LSURGE_REQUIRE(r->row_stride >= D && r->row_stride < MOST_ROW && r->head_stride >= 0 && r->head_stride < (1ll << 32) &&
                       r->row_stride % 8 == 0 && r->head_stride % 8 == 0,
                   "%s: row and head strides (%lld, %lld elements) must be multiples of 8 in [128, 2^22) and [0, 2^32)", what,
                   (long long)r->row_stride, (long long)r->head_stride);
  }
  LSURGE_REQUIRE(t->g && t->beta && t->o && (t->state || t->num_slots == 0), "%s: null pointer", what);
  LSURGE_REQUIRE(((uintptr_t)t->state | (uintptr_t)t->o) % 16 == 0 && (uintptr_t)t->g % 4 == 0, "%s: misaligned pointer", what);
  LSURGE_REQUIRE(t->g_stride >= t->hv && t->g_stride < MOST_ROW && t->beta_stride >= t->hv && t->beta_stride < MOST_ROW &&
                     t->num_slots >= 0 && t->num_slots < (1ll << 31) && t->slot_stride >= 0 && t->slot_stride < (1ll << 40) &&
                     t->slot_stride % 4 == 0 && (t->num_slots < 2 || t->slot_stride >= t->hv * D * D),
                 "%s: strides of g, beta and a slot (%lld, %lld, %lld), %lld slots", what, (long long)t->g_stride,
                 (long long)t->beta_stride, (long long)t->slot_stride, (long long)t->num_slots);
  return LSURGE_OK;
}

TokenArgs token_args(const lsurge_gdn_tokens* t) {
  TokenArgs a;
  a.q = (const uint16_t*)t->q.data, a.q_row = t->q.row_stride, a.q_head = t->q.head_stride;
  a.k = (const uint16_t*)t->k.data, a.k_row = t->k.row_stride, a.k_head = t->k.head_stride;
  a.v = (const uint16_t*)t->v.data, a.v_row = t->v.row_stride, a.v_head = t->v.head_stride;
  a.g = t->g, a.beta = t->beta, a.g_row = t->g_stride, a.beta_row = t->beta_stride;
  a.state = t->state, a.slot_stride = t->slot_stride, a.o = (uint16_t*)t->o;
  a.slots = t->slots, a.cu = t->cu;
  a.rows = (int)t->rows, a.nseq = (int)t->nseq, a.hk = (int)t->hk, a.hv = (int)t->hv, a.num_slots = (int)t->num_slots;
  a.l2_eps = t->l2_eps;
  return a;
}

// Columns a wave takes: 8 where there are few (sequence, head) pairs, whose one walk over a state is then shorter, else 32,
// which reads whole lines.  us for 8 and 32, states in the caches: 64 pairs 4.3 and 6.1, 128 5.5 and 6.7, 256 8.7 and 7.6; from
// memory: 128 7.5 and 7.7, 256 12.0 and 9.6, 2048 70 and 54, where a copy of the states takes 52.3.
int columns(int64_t seq_heads) { return seq_heads < 256 ? 8 : 32; }
// Waves of a workgroup that take columns of runs: 2 as long as each of the 256 CUs then holds one workgroup at most, whose four
// waves have a SIMD each; else 4, which prepare half as often.  us for 2 and 4: one sequence of 2000 tokens and 8 heads 107 and
// 119, 8 of up to 2000 105 and 117, 8 of 60 9.5 and 9.2, 16 of up to 2000 159 and 118, of 40 to 80 15.5 and 13.3.
int takers(int64_t seq_heads) { return seq_heads <= 64 ? 2 : 4; }
// Pairs of waves that prepare beside four takers: two share the work of a chunk out to all SIMDs, for a longer start, and leave
// one workgroup a CU where else there may be two.  So it takes long sequences, on average, which is all the host knows.  us for
// one pair and two: 12 sequences of 8 heads of 32 tokens 7.6 and 7.6, of 128 16.0 and 15.8, of 1000 75 and 66; 32 of 32 14.0 and
// 15.8, of 256 48 and 49, of 512 83 and 81, of 1000 154 and 147, of up to 2000 259 and 229.
int preparing_pairs(int64_t seq_heads, int64_t rows, int64_t nseq) {
  return rows >= nseq * (seq_heads <= 128 ? 64 : 300) ? 2 : 1;
}

}  // namespace
}  // namespace lsgdn

using namespace lsgdn;

extern "C" {

int lsurge_gdn_recurrent(const lsurge_gdn_tokens* t, lsurge_stream_t stream) {
  if (int rc = check_tokens(t)) return rc;
  if (t->rows == 0) return LSURGE_OK;
  TokenArgs a = token_args(t);
  const int64_t sh = t->nseq * t->hv;
  hipStream_t s = (hipStream_t)stream;
  // a launch holds less than 2^32 threads: two workgroups of up to 512 a pair, and 256 for the rows of none
  LSURGE_REQUIRE(sh <= (1ll << 22) - 256, "gdn_recurrent: %lld sequences of %lld heads", (long long)t->nseq, (long long)t->hv);
  const bool b32 = t->beta_dtype == LSURGE_F32;
  if (t->cu) {  // runs of any length
    const int64_t tail = std::min<int64_t>(256, 1 + t->rows * t->hv * D * 2 / (1 << 17));
    const int nw = takers(sh), pairs = preparing_pairs(sh, t->rows, t->nseq);
    a.units = (int)(sh * (D / 16 / nw));
#define RUNS_AS(DT, B32, NW, PAIRS)                                                                      \
  LSURGE_LAUNCH(KID_GDN_SCAN, s,                                                                         \
                hipLaunchKernelGGL((gdn_run_kernel<DT, B32, NW, PAIRS>), dim3((unsigned)(a.units + tail)), \
                                   dim3(64 * (NW + 2 * PAIRS)), 0, s, a))
#define RUNS(DT, B32)                             \
  if (nw == 2) { RUNS_AS(DT, B32, 2, 1); }        \
  else if (pairs == 2) { RUNS_AS(DT, B32, 4, 2); } \
  else { RUNS_AS(DT, B32, 4, 1); }
    if (t->dtype == LSURGE_BF16) {
      if (b32) { RUNS(LSURGE_BF16, true) }
      else { RUNS(LSURGE_BF16, false) }
    } else {
      if (b32) { RUNS(LSURGE_F16, true) }
      else { RUNS(LSURGE_F16, false) }
    }
#undef RUNS
#undef RUNS_AS
    return LSURGE_OK;
  }
  const int cb = columns(sh);
  a.units = (int)(sh * (D / cb / WAVES));
#define TOKENS(DT, CB, B32)                                                                                   \
  LSURGE_LAUNCH(KID_GDN_SCAN, s,                                                                              \
                hipLaunchKernelGGL((gdn_token_kernel<DT, CB, B32>), dim3((unsigned)a.units), dim3(64 * WAVES), 0, s, a))
#define TOKENS_CB(DT, B32)                        \
  if (cb == 32) { TOKENS(DT, 32, B32); }          \
  else { TOKENS(DT, 8, B32); }
  if (t->dtype == LSURGE_BF16) {
    if (b32) { TOKENS_CB(LSURGE_BF16, true) }
    else { TOKENS_CB(LSURGE_BF16, false) }
  } else {
    if (b32) { TOKENS_CB(LSURGE_F16, true) }
    else { TOKENS_CB(LSURGE_F16, false) }
  }
#undef TOKENS_CB
#undef TOKENS
  return LSURGE_OK;
}

}  // extern "C"

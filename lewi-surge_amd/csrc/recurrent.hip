// The gated delta rule over new tokens, from and to the states that serving keeps: one token for each of many sequences, a few
// drafted ones, or prompts.
//
// Per sequence and value head, S [128, 128] f32:  S <- e^g S,  d = beta (v - S^T k),  S <- S + k d^T,  o = S^T q / sqrt(128).
// The columns of S evolve independently of each other, so a wave takes a block of them through all tokens of its sequence:
// its part of S stays in registers, is read once and written once, and no wave waits for another.  A token's two products run
// on the S before it, S^T k and S^T q in one walk over the registers, with
//   o = (e^g S^T q + (k . q) d) / sqrt(128),
// so that one exchange between lanes serves both; the l2 norms of q and k are factors of these sums and cost no pass of their
// own.  Everything is f32 but the inputs and o.
//
// Bound by memory for a token or a few (the state's 128 KiB a sequence and head), by the vector unit from about ten tokens on:
// 4 x 128 x 128 multiply-adds a token and head, which have to follow each other.
#include <algorithm>

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
  int units;  // workgroups of the sequences; those behind them clear the rows behind the last sequence
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

template <int DT>
__device__ __forceinline__ float scalar_at(const void* p, int64_t i, int f32) {
  if (f32) return ((const float*)p)[i];
  const uint16_t x = ((const uint16_t*)p)[i];
  return DT == LSURGE_F16 ? f16_to_f32(x) : bf16_to_f32(x);
}

// CB columns a wave: lane l holds the rows R (l % RG) .. + R - 1 of the columns 4 (l / RG) .. + 3, RG = 256 / CB lanes a column
template <int DT, int CB, bool BETA32>
__global__ __launch_bounds__(64 * WAVES) void gdn_token_kernel(TokenArgs a) {
  constexpr int RG = 256 / CB, R = D / RG, V = R / 8 > 0 ? R / 8 : 1;  // V: 16-byte loads of a lane's rows of q or k
  constexpr int BLOCKS = D / CB / WAVES;  // workgroups a (sequence, head)
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if ((int)blockIdx.x >= a.units) {  // rows behind the last sequence
    const int64_t first = a.nseq ? lsrows::end_at(a.cu, a.nseq, a.rows) : 0;
    const int64_t n = (a.rows - first) * a.hv * (D / 8), step = (int64_t)(gridDim.x - a.units) * 64 * WAVES;
    u32x4* o = reinterpret_cast<u32x4*>(a.o + first * a.hv * D);
    for (int64_t i = (int64_t)(blockIdx.x - a.units) * 64 * WAVES + threadIdx.x; i < n; i += step) o[i] = u32x4{0u, 0u, 0u, 0u};
    return;
  }
  const int block = blockIdx.x % BLOCKS, sh = blockIdx.x / BLOCKS, h = sh % a.hv, b = sh / a.hv;
  const int rg = lane % RG, col = (block * WAVES + wave) * CB + lane / RG * 4;
  const int begin = a.cu ? lsrows::end_at(a.cu, b, a.rows) : b;
  const int end = a.cu ? lsrows::end_at(a.cu, b + 1, a.rows) : b + 1;
  const int slot = a.slots ? a.slots[b] : b;
  if (begin >= end) return;
  uint16_t* o = a.o + (int64_t)h * D + col;
  const int64_t o_row = (int64_t)a.hv * D;
  if ((unsigned)slot >= (unsigned)a.num_slots) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    if (rg == 0)
      for (int t = begin; t < end; ++t) *reinterpret_cast<u32x2*>(o + t * o_row) = u32x2{0u, 0u};
    return;
  }
  float* sp = a.state + slot * a.slot_stride + (int64_t)h * D * D + (int64_t)rg * R * D + col;
  f32x4 S[R];
#pragma unroll
  for (int i = 0; i < R; ++i) S[i] = *reinterpret_cast<const f32x4*>(sp + i * D);

  const int kh = h / (a.hv / a.hk);
  const uint16_t* qp = a.q + kh * a.q_head + rg * R;
  const uint16_t* kp = a.k + kh * a.k_head + rg * R;
  const uint16_t* vp = a.v + h * a.v_head + col;
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
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
  load(begin, next);
  for (int t = begin; t < end; ++t) {
    cur = next;
    load(min(t + 1, end - 1), next);
    float q[8 * V], k[8 * V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      lsrows::unpack8<DT>(cur.q[i], q + 8 * i);
      lsrows::unpack8<DT>(cur.k[i], k + 8 * i);
    }
    float kk = 0.f, qq = 0.f, kq = 0.f;
    f32x4 kS{0.f, 0.f, 0.f, 0.f}, qS{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < R; ++i) {
      kk = fmaf(k[i], k[i], kk);
      qq = fmaf(q[i], q[i], qq);
      kq = fmaf(k[i], q[i], kq);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        kS[c] = fmaf(k[i], S[i][c], kS[c]);
        qS[c] = fmaf(q[i], S[i][c], qS[c]);
      }
    }
    kq = group_sum<RG>(kq);
    float rk = 1.f, rq = 0.08838834764831845f;  // 1 / sqrt(128)
    if (a.l2_eps >= 0.f) {
      rk = rsqrtf(group_sum<RG>(kk) + a.l2_eps);
      rq *= rsqrtf(group_sum<RG>(qq) + a.l2_eps);
    }
    const float decay = expf(cur.g);
    float v[4], out[4], kd[4];
    v[0] = DT == LSURGE_F16 ? f16_to_f32((uint16_t)cur.v[0]) : bf16_to_f32((uint16_t)cur.v[0]);
    v[1] = DT == LSURGE_F16 ? f16_to_f32((uint16_t)(cur.v[0] >> 16)) : bf16_to_f32((uint16_t)(cur.v[0] >> 16));
    v[2] = DT == LSURGE_F16 ? f16_to_f32((uint16_t)cur.v[1]) : bf16_to_f32((uint16_t)cur.v[1]);
    v[3] = DT == LSURGE_F16 ? f16_to_f32((uint16_t)(cur.v[1] >> 16)) : bf16_to_f32((uint16_t)(cur.v[1] >> 16));
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      kd[c] = rk * (cur.beta * fmaf(-decay * rk, group_sum<RG>(kS[c]), v[c]));  // rk d
      out[c] = rq * fmaf(decay, group_sum<RG>(qS[c]), kq * kd[c]);
    }
    if (rg == 0)
      *reinterpret_cast<u32x2*>(o + t * o_row) = u32x2{lsrows::pack2<DT>(out[0], out[1]), lsrows::pack2<DT>(out[2], out[3])};
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) S[i][c] = fmaf(k[i], kd[c], decay * S[i][c]);
  }
#pragma unroll
  for (int i = 0; i < R; ++i) *reinterpret_cast<f32x4*>(sp + i * D) = S[i];
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
    LSURGE_REQUIRE(r->row_stride >= 0 && r->row_stride < (1ll << 32) && r->head_stride >= 0 && r->head_stride < (1ll << 32) &&
                       r->row_stride % 8 == 0 && r->head_stride % 8 == 0,
                   "%s: row and head strides (%lld, %lld elements) must be multiples of 8 in [0, 2^32)", what,
                   (long long)r->row_stride, (long long)r->head_stride);
  }
  LSURGE_REQUIRE(t->g && t->beta && t->o && (t->state || t->num_slots == 0), "%s: null pointer", what);
  LSURGE_REQUIRE(((uintptr_t)t->state | (uintptr_t)t->o) % 16 == 0 && (uintptr_t)t->g % 4 == 0, "%s: misaligned pointer", what);
  LSURGE_REQUIRE(t->g_stride >= 0 && t->g_stride < (1ll << 32) && t->beta_stride >= 0 && t->beta_stride < (1ll << 32) &&
                     t->num_slots >= 0 && t->num_slots < (1ll << 31) && t->slot_stride >= 0 && t->slot_stride < (1ll << 40) &&
                     t->slot_stride % 4 == 0,
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

// Columns a wave takes: 32 while that leaves four waves for every SIMD, then 16, then 8, whose shorter walks end sooner.
int columns(int64_t seq_heads) { return seq_heads * 4 >= 4096 ? 32 : seq_heads * 8 >= 2048 ? 16 : 8; }

}  // namespace
}  // namespace lsgdn

using namespace lsgdn;

extern "C" {

size_t lsurge_gdn_recurrent_workspace_bytes(const lsurge_gdn_tokens* t) {
  (void)t;
  return 0;
}

int lsurge_gdn_recurrent(const lsurge_gdn_tokens* t, void* workspace, size_t workspace_bytes, lsurge_stream_t stream) {
  if (int rc = check_tokens(t)) return rc;
  (void)workspace, (void)workspace_bytes;
  if (t->rows == 0) return LSURGE_OK;
  TokenArgs a = token_args(t);
  const int64_t sh = t->nseq * t->hv;
  const int cb = columns(sh);
  const int64_t units = sh * (D / cb / WAVES);
  const int64_t tail = t->cu ? std::min<int64_t>(256, 1 + t->rows * t->hv * D * 2 / (1 << 17)) : 0;
  LSURGE_REQUIRE(units < (1ll << 24) - 256, "gdn_recurrent: %lld sequences of %lld heads", (long long)t->nseq, (long long)t->hv);
  a.units = (int)units;
  const unsigned grid = (unsigned)(units + tail);
  hipStream_t s = (hipStream_t)stream;
#define TOKENS(DT, CB, B32)                                                                                   \
  LSURGE_LAUNCH(KID_GDN_SCAN, s,                                                                              \
                hipLaunchKernelGGL((gdn_token_kernel<DT, CB, B32>), dim3(grid), dim3(64 * WAVES), 0, s, a))
#define TOKENS_CB(DT, B32)                        \
  if (cb == 32) { TOKENS(DT, 32, B32); }          \
  else if (cb == 16) { TOKENS(DT, 16, B32); }     \
  else { TOKENS(DT, 8, B32); }
  if (t->dtype == LSURGE_BF16) {
    if (t->beta_dtype == LSURGE_F32) { TOKENS_CB(LSURGE_BF16, true) }
    else { TOKENS_CB(LSURGE_BF16, false) }
  } else {
    if (t->beta_dtype == LSURGE_F32) { TOKENS_CB(LSURGE_F16, true) }
    else { TOKENS_CB(LSURGE_F16, false) }
  }
#undef TOKENS_CB
#undef TOKENS
  return LSURGE_OK;
}

}  // extern "C"

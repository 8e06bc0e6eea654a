// Rotation of query and key heads by their tokens' positions, by itself (forward, and backward as the rotation by the negative
// angle) and on the way into the paged key-value cache.
//
// Pair i of a head's first `rot` values turns by the angle p f_i of the token's position p:
//   (a, b) -> (a cos - b sin, b cos + a sin),   a, b = values i and i + rot / 2, or (interleaved) 2 i and 2 i + 1;
// the values behind them pass through.  p f_i / 2 pi is formed in 64 bits and only its fraction goes on in f32: a position of
// 10^6 is 1.6 10^5 turns, of whose fraction f32 would keep 6 bits.  Sine and cosine are the Taylor series of the angle within
// an eighth of a turn (the rest is below 2^-24), the rotation is f32, each output rounded once.
//
// Bound by memory: every value read and written once.  A thread turns 16 values (two 16-byte loads and stores) of up to
// HEADS heads of one row, so that angles, frequencies and the row's sequence are found once for all of them; a wave's lanes
// cover whole heads in a row.  20652 tokens, 16 query and 2 key heads of 256, into their pages: 89 us, 5.0 TB/s (a copy reaches
// 5.1); 32768 tokens of 10 heads of 128 by themselves: 34 us, 4.9 TB/s; 64 tokens: 4 us, a launch and three trips to memory.
#include <algorithm>

#include "kv_cache.h"
#include "launchers.h"
#include "rows16.h"

namespace lsattn {
namespace {

constexpr int RT = 256;  // threads of a workgroup

struct RotaryArgs {
  const uint16_t *q, *k, *v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  uint16_t *q_out, *k_out;  // contiguous, or null
  const double* freq;
  const int32_t *cu, *pos, *lens;  // lens: of the cache (null: rotation alone)
  CacheArgs c;
  int rows, nseq, hq, hk, hv;      // hv: value heads to write (hk, or 0 for the rotation alone)
  int log2_units;                  // D / 16 = 2^log2_units units of 16 values a head
  int turned;                      // units of a head that are turned, rot / 16
  int groups;                      // ceil(heads / HEADS)
  int steps;                       // without cu and cache: rows of a sequence
  float sign;
};

// cos and sin of 2 pi times the fraction of a turn u in [-0.5, 0.5]
__device__ __forceinline__ void cos_sin_turn(float u, float& c, float& s) {
  const float n = rintf(4.f * u);
  const float x = (u - 0.25f * n) * 6.283185307179586f;  // exact difference; |x| <= pi / 4
  const float z = x * x;
  const float sn = fmaf(x * z, fmaf(z, fmaf(z, fmaf(z, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), x);
  const float cs = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24), -0.5f), 1.f);
  const int m = (int)n;  // quarter turns, -2 .. 2
  const float a = m & 1 ? sn : cs, b = m & 1 ? cs : sn;
  c = (m + 1) & 2 ? -a : a;
  s = m & 2 ? -b : b;
}

// 6 waves a SIMD: the compiler's own choice leaves 3 to 5 and takes 10% longer, for 8 it spills.
template <int DT, bool INTER, int HEADS>
__global__ __launch_bounds__(RT, 6) void rotary_kernel(RotaryArgs a, int row0) {
  using lsrows::pack8;
  using lsrows::unpack8;
  const uint32_t id = blockIdx.x * RT + threadIdx.x;
  const uint32_t per_row = (uint32_t)a.groups << a.log2_units;
  const int64_t row64 = (int64_t)row0 + id / per_row;
  const int row = (int)min(row64, (int64_t)a.rows - 1);
  // the sequence of the wave's first row, by all of its lanes
  const int near = a.cu ? lsrows::find_seq(a.cu, a.nseq, __builtin_amdgcn_readfirstlane(row), threadIdx.x & 63) : 0;
  if (row64 >= a.rows) return;
  const uint32_t in_row = id % per_row;
  const int unit = in_row & ((1 << a.log2_units) - 1), group = in_row >> a.log2_units;
  const int D = 16 << a.log2_units, heads = a.hq + a.hk + a.hv;

  const bool turns = unit < a.turned;
  // a unit's 16 values: two runs of 8, half of the turned values apart, or consecutive
  const int at0 = turns && !INTER ? 8 * unit : 16 * unit;
  const int at1 = at0 + (turns && !INTER ? 8 * a.turned : 8);

  const int pos = a.pos ? a.pos[row] : 0;
  // The row is read whatever it holds, while its token is looked up.
  u32x4 x[HEADS][2];
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    const int h = i * a.groups + group;
    if (h >= heads) continue;
    const uint16_t* p = h < a.hq          ? a.q + row * a.q_row + h * a.q_head
                        : h < a.hq + a.hk ? a.k + row * a.k_row + (h - a.hq) * a.k_head
                                          : a.v + row * a.v_row + (h - a.hq - a.hk) * a.v_head;
    const bool moved = turns && h < a.hq + a.hk;
    x[i][0] = *reinterpret_cast<const u32x4*>(p + (moved ? at0 : 16 * unit));
    x[i][1] = *reinterpret_cast<const u32x4*>(p + (moved ? at1 : 16 * unit + 8));
  }
  // the row's token: its position, and its place in the cache
  int seq = -1, tok = -1;
  if (a.lens || a.cu) {
    const lsrows::Seq s = lsrows::seq_from(a.cu, a.nseq, a.rows, row, near);
    seq = s.seq;
    if (seq >= 0) tok = a.lens ? max(a.lens[seq], 0) - (s.end - row) : row - s.begin;
  } else {
    tok = row % a.steps;
  }
  const bool live = tok >= 0;
  int page = -1, slot = 0;
  if (a.lens && live && (tok >> a.c.page_log2) < a.c.max_pages) {
    page = a.c.table[seq * a.c.table_stride + (tok >> a.c.page_log2)];
    slot = tok & ((1 << a.c.page_log2) - 1);
  }
  const bool paged = (unsigned)page < (unsigned)a.c.num_pages;
  float c[8], s[8];
  if (turns && live) {
    const double p = (double)(a.pos ? pos : tok) * 0.15915494309189533577;  // 1 / 2 pi
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double t = p * a.freq[8 * unit + i];
      cos_sin_turn((float)(t - rint(t)), c[i], s[i]);
      s[i] *= a.sign;
    }
  }
#pragma unroll
  for (int i = 0; i < HEADS; ++i) {
    const int h = i * a.groups + group;
    if (h >= heads) continue;
    const bool value = h >= a.hq + a.hk;
    if (!live) {
      x[i][0] = x[i][1] = u32x4{0u, 0u, 0u, 0u};
    } else if (turns && !value) {
      float f[16], g[16];
      unpack8<DT>(x[i][0], f);
      unpack8<DT>(x[i][1], f + 8);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int ia = INTER ? 2 * j : j, ib = INTER ? 2 * j + 1 : j + 8;
        g[ia] = fmaf(f[ia], c[j], -f[ib] * s[j]);
        g[ib] = fmaf(f[ib], c[j], f[ia] * s[j]);
      }
      x[i][0] = pack8<DT>(g);
      x[i][1] = pack8<DT>(g + 8);
    }
    const int o0 = value ? 16 * unit : at0, o1 = value ? 16 * unit + 8 : at1;
    if (h < a.hq) {
      uint16_t* o = a.q_out + ((int64_t)row * a.hq + h) * D;
      *reinterpret_cast<u32x4*>(o + o0) = x[i][0];
      *reinterpret_cast<u32x4*>(o + o1) = x[i][1];
      continue;
    }
    const int kh = value ? h - a.hq - a.hk : h - a.hq;
    if (!value && a.k_out) {
      uint16_t* o = a.k_out + ((int64_t)row * a.hk + kh) * D;
      *reinterpret_cast<u32x4*>(o + o0) = x[i][0];
      *reinterpret_cast<u32x4*>(o + o1) = x[i][1];
    }
    if (a.lens && paged) {
      uint16_t* o = value ? const_cast<uint16_t*>(a.c.v) + page * a.c.v_page + slot * a.c.v_slot + kh * a.c.v_head
                          : const_cast<uint16_t*>(a.c.k) + page * a.c.k_page + slot * a.c.k_slot + kh * a.c.k_head;
      *reinterpret_cast<u32x4*>(o + o0) = x[i][0];
      *reinterpret_cast<u32x4*>(o + o1) = x[i][1];
    }
  }
}

// Heads a thread turns, at most 4: as many as leave two waves for every SIMD.  us for 1, 2 and 4: 64 tokens of 48 heads of 128
// 3.8, 4.3, 5.1; 2210 of 12 8.3, 7.8, 8.7; 20652 of 20 of 256 112, 91, 89.
int heads_per_thread(int64_t rows, int64_t heads, int units) {
  int n = 1;
  while (n < 4 && 2 * n <= heads && rows * heads * units / (2 * n) >= (1 << 17)) n *= 2;
  return n;
}

int launch_rotary(const char* what, RotaryArgs& a, int64_t d, const lsurge_rotary* r, hipStream_t st) {
  a.freq = r->inv_freq, a.pos = r->positions, a.sign = r->inverse ? -1.f : 1.f;
  a.log2_units = d == 64 ? 2 : d == 128 ? 3 : 4;
  a.turned = (int)(r->rotary_dim / 16);
  const int heads = a.hq + a.hk + a.hv;
  if (a.rows == 0 || heads == 0) return LSURGE_OK;
  const int per = heads_per_thread(a.rows, heads, 1 << a.log2_units);
  a.groups = (heads + per - 1) / per;
  // a launch holds less than 2^31 threads
  const int64_t per_row = (int64_t)a.groups << a.log2_units, most = std::max<int64_t>(1, ((1ll << 31) - RT) / per_row);
  LSURGE_REQUIRE(per_row < (1ll << 30), "%s: %d heads", what, heads);
  for (int64_t row0 = 0; row0 < a.rows; row0 += most) {
    const unsigned grid = (unsigned)((std::min<int64_t>(most, a.rows - row0) * per_row + RT - 1) / RT);
#define ROTARY(DT, INTER, HEADS)                                                                                       \
  LSURGE_LAUNCH(KID_ATTN, st,                                                                                          \
                hipLaunchKernelGGL((rotary_kernel<DT, INTER, HEADS>), dim3(grid), dim3(RT), 0, st, a, (int)row0))
#define ROTARY_HEADS(DT, INTER)                \
  if (per == 1) { ROTARY(DT, INTER, 1); }      \
  else if (per == 2) { ROTARY(DT, INTER, 2); } \
  else { ROTARY(DT, INTER, 4); }
    if (r->dtype == LSURGE_BF16) {
      if (r->interleaved) { ROTARY_HEADS(LSURGE_BF16, true) }
      else { ROTARY_HEADS(LSURGE_BF16, false) }
    } else {
      if (r->interleaved) { ROTARY_HEADS(LSURGE_F16, true) }
      else { ROTARY_HEADS(LSURGE_F16, false) }
    }
#undef ROTARY_HEADS
#undef ROTARY
  }
  return LSURGE_OK;
}

int check_rotary(const char* what, const lsurge_rotary* r, int64_t rows, int64_t nseq, int64_t hq, int64_t hk,
                 int64_t d) {
  LSURGE_REQUIRE(r, "%s: null arguments", what);
  LSURGE_REQUIRE(d == 64 || d == 128 || d == 256, "%s: head_dim %lld (64, 128 or 256)", what, (long long)d);
  LSURGE_REQUIRE(r->rotary_dim >= 16 && r->rotary_dim <= d && r->rotary_dim % 16 == 0,
                 "%s: rotary_dim %lld of %lld (a multiple of 16)", what, (long long)r->rotary_dim, (long long)d);
  LSURGE_REQUIRE(r->inv_freq && (uintptr_t)r->inv_freq % 8 == 0, "%s: null or misaligned frequencies", what);
  if (r->dtype != LSURGE_BF16 && r->dtype != LSURGE_F16) return lsurge::set_error(LSURGE_ERR_DTYPE, "%s: bf16 or f16", what);
  LSURGE_REQUIRE(hq >= 0 && hq <= 65535 && hk >= 0 && hk <= 65535, "%s: %lld and %lld heads", what, (long long)hq,
                 (long long)hk);
  LSURGE_REQUIRE(rows >= 0 && rows < (1ll << 30) && nseq >= 0 && nseq < (1ll << 24), "%s: %lld rows of %lld sequences", what,
                 (long long)rows, (long long)nseq);
  return LSURGE_OK;
}

}  // namespace
}  // namespace lsattn

using namespace lsattn;

extern "C" {

int lsurge_rotary_rows(const lsurge_rotary* r, const lsurge_attn_rows* q, int64_t hq, const lsurge_attn_rows* k, int64_t hk,
                       int64_t d, int64_t rows, int64_t nseq, const int32_t* cu, void* q_out, void* k_out,
                       lsurge_stream_t stream) {
  if (int rc = check_rotary("rotary", r, rows, nseq, hq, hk, d)) return rc;
  LSURGE_REQUIRE(cu || nseq == 0 || rows % nseq == 0, "rotary: %lld rows of %lld dense sequences", (long long)rows,
                 (long long)nseq);
  if (rows == 0) return LSURGE_OK;
  RotaryArgs a{};
  a.rows = (int)rows, a.nseq = (int)nseq;
  a.steps = cu || nseq == 0 ? (int)rows : (int)(rows / nseq);
  if (hq) {
    if (int rc = check_new_rows("rotary q", q)) return rc;
    LSURGE_REQUIRE(q_out && (uintptr_t)q_out % 16 == 0, "rotary: null or misaligned q_out");
    a.q = (const uint16_t*)q->data, a.q_row = q->row_stride, a.q_head = q->head_stride, a.q_out = (uint16_t*)q_out;
    a.hq = (int)hq;
  }
  if (hk) {
    if (int rc = check_new_rows("rotary k", k)) return rc;
    LSURGE_REQUIRE(k_out && (uintptr_t)k_out % 16 == 0, "rotary: null or misaligned k_out");
    a.k = (const uint16_t*)k->data, a.k_row = k->row_stride, a.k_head = k->head_stride, a.k_out = (uint16_t*)k_out;
    a.hk = (int)hk;
  }
  a.cu = cu;
  return launch_rotary("rotary", a, d, r, (hipStream_t)stream);
}

int lsurge_rotary_append(const lsurge_kv_cache* c, const lsurge_rotary* r, const lsurge_attn_rows* q, int64_t hq,
                         const lsurge_attn_rows* k, const lsurge_attn_rows* v, int64_t rows, int64_t nseq, const int32_t* cu,
                         void* q_out, void* k_out, lsurge_stream_t stream) {
  const char* what = "rotary_append";
  RotaryArgs a{};
  if (int rc = check_cache(what, c, &a.c)) return rc;
  if (int rc = check_rotary(what, r, rows, nseq, hq, c->heads, c->d)) return rc;
  LSURGE_REQUIRE(cu || rows == nseq, "rotary_append: %lld rows for %lld sequences", (long long)rows, (long long)nseq);
  LSURGE_REQUIRE(r->dtype == c->dtype, "rotary_append: the caches' dtype %d, the rows' %d", c->dtype, r->dtype);
  if (rows == 0) return LSURGE_OK;
  if (hq) {
    if (int rc = check_new_rows("rotary_append q", q)) return rc;
    a.q = (const uint16_t*)q->data, a.q_row = q->row_stride, a.q_head = q->head_stride;
    LSURGE_REQUIRE(q_out && (uintptr_t)q_out % 16 == 0, "rotary_append: null or misaligned q_out");
  }
  if (int rc = check_new_rows("rotary_append k", k)) return rc;
  if (int rc = check_new_rows("rotary_append v", v)) return rc;
  LSURGE_REQUIRE((uintptr_t)k_out % 16 == 0, "rotary_append: misaligned k_out");
  a.k = (const uint16_t*)k->data, a.k_row = k->row_stride, a.k_head = k->head_stride;
  a.v = (const uint16_t*)v->data, a.v_row = v->row_stride, a.v_head = v->head_stride;
  a.q_out = (uint16_t*)q_out, a.k_out = (uint16_t*)k_out;
  a.rows = (int)rows, a.nseq = (int)nseq, a.hq = (int)hq, a.hk = (int)c->heads, a.hv = (int)c->heads;
  a.cu = cu, a.lens = c->seq_lens, a.steps = 1;
  return launch_rotary(what, a, c->d, r, (hipStream_t)stream);
}

}  // extern "C"

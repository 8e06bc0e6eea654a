// Attention of one new token per sequence over a paged key-value cache, and the write of new tokens into its pages.
//
// Cache: pages of `page_size` tokens; page p's key of head h at slot t starts at k + p page_stride + h head_stride + t
// slot_stride (elements; v alike).  page_table[b][i] is the page of sequence b's tokens [i page_size, (i + 1) page_size).
// An entry outside [0, num_pages) names no page: its tokens are left out (read) or not written.
//
// Bound by the cache's bytes: 4 D bytes a token and key head are read once for all query heads that share it, and the
// 4 D flops a query head needs for them are a few percent of the matrix cores' rate even with one head a group.  The keys'
// fragments come straight from memory; the values are read in whole rows (256 bytes at D = 128, in the order in which the
// weights lie in their lanes) and turned by byte permutes, 4 for each 4 registers: no LDS on the way, so that every wave
// keeps one or two tiles of loads in flight.  Measured: 64 sequences of 4150 tokens on average, 8 key heads of 128: 193 us,
// 5.6 TB/s (a copy reaches 5.0 reading and writing); 2 of them of 256: 107 us and 5 for the join, 5.1 TB/s; 2 of 120000, 4
// heads of 128: 89 us and 6, 5.1 TB/s; 96 of 900, 16 heads of 64: 71 us and 5, 4.6 TB/s; one of 777 tokens: 10 us and 4, a
// chain of trips to memory.
#include <algorithm>

#include "attn_common.h"
#include "kv_cache.h"
#include "launchers.h"

namespace lsattn {
namespace {

// ------------------------------------------------------------------------------------ one token per sequence
// Work is dealt by the keys that are there, not by sequence: the units of UK keys of every (sequence, key head) in a row
// are cut into equal shares, one a workgroup, so a batch of uneven lengths keeps every CU equally busy and the host needs
// no lengths.  A workgroup's share is a run of pieces, each of one (sequence, head); a piece that is the whole of it is
// written out, another goes to the workspace (slot 0: the share began inside it; slot 1: it ends past the share) and the
// join kernel adds the pieces of a (sequence, head) up in order.
constexpr int DW = 4;             // waves of a workgroup; each takes 32 keys at a time
constexpr int UK = DW * 32;       // keys of a unit
constexpr int DT_THREADS = DW * 64;
constexpr int64_t decode_eu(int64_t d) { return d == 64 ? 3 : d == 128 ? 2 : 1; }  // waves per SIMD that the registers leave
constexpr int64_t CUS = 256;
constexpr int64_t DECODE_GRID = CUS * decode_eu(64);  // workgroups at most: 4 waves each, one a SIMD

struct DecodeArgs {
  CacheArgs c;
  const uint16_t* q;
  int64_t q_row, q_head;
  const int32_t* lens;
  int nseq, hq, hk, group, hblocks;  // hblocks: blocks of 16 query heads a group
  float scale2;
  uint16_t* o;
  float* lse;  // [nseq, hq] or null
  float *po, *pm;  // [grid][2][16][D], [grid][2][2][16] (maximum in base 2, sum)
  int32_t* shares;  // [nseq heads] first and last share of a (sequence, head block)
  int grid;
};

__device__ __forceinline__ int seq_len(const DecodeArgs& a, int b) {
  const int64_t cap = (int64_t)a.c.max_pages << a.c.page_log2;
  return (int)min((int64_t)max(a.lens[b], 0), cap);
}
__device__ __forceinline__ int units_of(int len) { return (len + UK - 1) / UK; }
__device__ __forceinline__ int64_t uni64(int64_t v) {
  return (int64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)v) |
         (int64_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32;
}
// n / d, in 32 bits where that will do (a 64-bit division is hundreds of instructions)
__device__ __forceinline__ int64_t div64(int64_t n, int64_t d) {
  return (uint64_t)(n | d) >> 32 ? n / d : (int64_t)((uint32_t)n / (uint32_t)d);
}

// log2 of the room that a row's weights are given above 1, as operands of their product with V: f16 has few exponent bits,
// and a weight below 2^-25 of the largest would be none, though thousands of them may hold a share of the row that counts.
// The base is taken that much below the largest scaled score `top`, and the sums of the weights have the same factor.  2^15,
// less where the roundings of the base (2^-24 of top each, two of them) leave the largest score above it.  Not needed in bf16.
template <int DT>
__device__ __forceinline__ float room(float top) {
  return DT == LSURGE_F16 ? fmaxf(fmaf(fabsf(top), -0x1p-23f, 15.f), 0.f) : 0.f;
}

template <int D, int DT>
__global__ __launch_bounds__(DT_THREADS) __attribute__((amdgpu_waves_per_eu(decode_eu(D))))
void attn_decode_kernel(DecodeArgs a) {
  constexpr int KC = D / 32, VE = D / 16, VW = VE / 2;  // a lane's 16-byte chunks of a key, columns and registers of a value
  __shared__ int64_t wsum[DW], found;
  __shared__ int found_b, found_len;
  __shared__ __attribute__((aligned(16))) float so[DW][16][D];
  __shared__ float sm[DW][16], sl[DW][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ln = lane & 15, g = lane >> 4;
  const int heads = a.hk * a.hblocks;
  // units of all sequences: each thread sums a slab of them, then a scan over the threads
  const int slab = (a.nseq + DT_THREADS - 1) / DT_THREADS;
  int64_t mine = 0;
  int first_len = 0;
  for (int i = 0; i < slab; ++i) {
    const int b = tid * slab + i, n = b < a.nseq ? seq_len(a, b) : 0;
    if (i == 0) first_len = n;
    mine += units_of(n);
  }
  // below 2^39 (2^16 sequences a slab, 2^23 units each): scanned in two halves that cannot overflow
  int64_t pre = ((int64_t)wave_scan((int)(mine >> 20)) << 20) + wave_scan((int)mine & 0xfffff);
  if (lane == 63) wsum[wave] = pre;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < DW; ++w) {
    if (w < wave) pre += wsum[w];
    total += wsum[w];
  }
  total = uni64(total * heads);
  const int64_t per = max(div64(total + a.grid - 1, a.grid), (int64_t)1);
  int64_t u = blockIdx.x * per;
  const int64_t uend = min(total, u + per);
  if (u >= uend) return;
  // the sequence of the share's first unit: in the slab that holds it, then one by one
  if (mine && (pre - mine) * heads <= u && u < pre * heads) {
    int b = tid * slab, len = first_len;
    int64_t base = (pre - mine) * heads;
    while (true) {
      const int64_t n = (int64_t)units_of(len) * heads;
      if (u < base + n) break;
      base += n;
      len = seq_len(a, ++b);
    }
    found = base;
    found_b = b;
    found_len = len;
  }
  __syncthreads();
  int64_t base = uni64(found);  // units before sequence b (all heads)
  int b = __builtin_amdgcn_readfirstlane(found_b);
  int len = __builtin_amdgcn_readfirstlane(found_len), nu = units_of(len);
  int hb = (int)div64(u - base, nu);
  const int pmask = (1 << a.c.page_log2) - 1;

  while (u < uend) {
    const int64_t item = base + (int64_t)hb * nu;  // first unit of this (sequence, head block)
    const int u0 = (int)(u - item), u1 = (int)min((int64_t)nu, uend - item);
    const int kvh = hb / a.hblocks, h0 = kvh * a.group + hb % a.hblocks * 16;
    const int nh = min(16, (kvh + 1) * a.group - h0);
    const int32_t* tab = a.c.table + b * a.c.table_stride;
    const uint16_t* kb = a.c.k + kvh * a.c.k_head + 8 * g;
    const uint16_t* vb = a.c.v + kvh * a.c.v_head + VE * ln;
    // this wave's tiles of 32 keys: from key first on, UK apart
    const int first = u0 * UK + wave * 32, end = min(len, u1 * UK);
    const int n = first < end ? (end - first + UK - 1) / UK : 0;

    struct Pages {
      int k[2], v[2];
    };
    struct Tile {
      u32x4 k[2][KC];
      uint32_t v[8][VW];
      bool ok[2];
    };
    // pages of the lane's keys (rows 16 t + l % 16) and of its values (rows 16 t + 4 (l / 16) .. + 3)
    auto pages = [&](int key0, Pages& p) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int kk = key0 + 16 * t + ln, kv = key0 + 16 * t + 4 * g;
        p.k[t] = kk < len ? tab[kk >> a.c.page_log2] : -1;
        p.v[t] = kv < len ? tab[kv >> a.c.page_log2] : -1;
      }
    };
    // a key or value without a page is read from token 0 of page 0 and gets weight 0
    auto load_k = [&](int key0, const Pages& p, Tile& x) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const bool ok = (unsigned)p.k[t] < (unsigned)a.c.num_pages;
        const uint16_t* kp = kb + (ok ? p.k[t] * a.c.k_page + ((key0 + 16 * t + ln) & pmask) * a.c.k_slot : 0);
#pragma unroll
        for (int j = 0; j < KC; ++j) x.k[t][j] = *reinterpret_cast<const u32x4*>(kp + 32 * j);
      }
    };
    auto load_v = [&](int key0, const Pages& p, Tile& x) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        x.ok[t] = (unsigned)p.v[t] < (unsigned)a.c.num_pages;
        const uint16_t* vp = vb + (x.ok[t] ? p.v[t] * a.c.v_page + ((key0 + 16 * t + 4 * g) & pmask) * a.c.v_slot : 0);
        const int64_t step = x.ok[t] ? a.c.v_slot : 0;  // pages hold multiples of 4 tokens: the next 3 are in this one
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (VW == 2) {
            const u32x2 y = *reinterpret_cast<const u32x2*>(vp + i * step);
            x.v[4 * t + i][0] = y[0], x.v[4 * t + i][1] = y[1];
          } else {
#pragma unroll
            for (int c = 0; c < VW / 4; ++c) {
              const u32x4 y = *reinterpret_cast<const u32x4*>(vp + i * step + 8 * c);
#pragma unroll
              for (int e = 0; e < 4; ++e) x.v[4 * t + i][4 * c + e] = y[e];
            }
          }
        }
      }
    };
    Pages pg;
    Tile x0;
    if (n) {
      pages(first, pg);
      load_k(first, pg, x0);
      load_v(first, pg, x0);
      if (n > 1) pages(first + UK, pg);
    }
    u32x4 qf[KC];
#pragma unroll
    for (int j = 0; j < KC; ++j)
      qf[j] = ln < nh ? *reinterpret_cast<const u32x4*>(a.q + b * a.q_row + (h0 + ln) * a.q_head + 32 * j + 8 * g)
                      : u32x4{0, 0, 0, 0};
    f32x4 acc[VE];
#pragma unroll
    for (int t = 0; t < VE; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    // m: the largest score so far times the scale, less its room, as rounded.  Weights, sums and the join all take this one value
    // as their base: the product formed anew inside an fma would be the unrounded one, a factor of 2^(its rounding) for every
    // tile.
    float m = -INFINITY, l = 0.f;

    auto compute = [&](int key0, Tile& x, auto&& after_scores) {
      f32x4 s[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < KC; ++j) s[t] = mma16<DT>(x.k[t][j], qf[j], s[t]);
      }
      after_scores();
      if (!__all(x.ok[0] && x.ok[1] && key0 + 32 <= len)) {  // keys past the end or without a page: weight 0, value 0
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (!x.ok[i / 4] || key0 + 16 * (i / 4) + 4 * g + i % 4 >= len) {
            s[i / 4][i % 4] = -INFINITY;
#pragma unroll
            for (int c = 0; c < VW; ++c) x.v[i][c] = 0;
          }
      }
      float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                       fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = halves(mx, [](float p, float q) { return fmaxf(p, q); }) * a.scale2;
      mx = fmaxf(m, mx - room<DT>(mx));
      const float mc = mx == -INFINITY ? 0.f : mx;
      const float alpha = exp2_hw(m - mc);  // 1 where the largest score stays
      m = mx;
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[t][r] = exp2_hw(fmaf(s[t][r], a.scale2, -mc));
          sum += s[t][r];
        }
      l = l * alpha + sum;
      const u32x4 p = {pack2<DT>(s[0][0], s[0][1]), pack2<DT>(s[0][2], s[0][3]), pack2<DT>(s[1][0], s[1][1]),
                       pack2<DT>(s[1][2], s[1][3])};
#pragma unroll
      for (int t = 0; t < VE; ++t) {
        const uint32_t sel = t & 1 ? 0x07060302u : 0x05040100u;  // the pair's high or low halves
        u32x4 f;
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = __builtin_amdgcn_perm(x.v[2 * e + 1][t / 2], x.v[2 * e][t / 2], sel);
        f32x4 c = acc[t];
#pragma unroll
        for (int r = 0; r < 4; ++r) c[r] *= alpha;
        acc[t] = mma16<DT>(f, p, c);
      }
    };
    if constexpr (D == 256) {  // no registers for a second tile: the next keys and values as soon as these are used
      for (int i = 0; i < n; ++i) {
        const int next = first + (i + 1) * UK;
        compute(first + i * UK, x0, [&] {
          if (i + 1 < n) load_k(next, pg, x0);
        });
        if (i + 1 < n) load_v(next, pg, x0);
        if (i + 2 < n) pages(next + UK, pg);
      }
    } else {
      Tile x1;
      auto turn = [&](int i, Tile& now, Tile& then) {  // the next tile's loads and the one after's pages before the products
        const int next = first + (i + 1) * UK;
        if (i + 1 < n) {
          load_k(next, pg, then);
          load_v(next, pg, then);
        }
        if (i + 2 < n) pages(next + UK, pg);
        compute(first + i * UK, now, [] {});
      };
      for (int i = 0; i < n; i += 2) {
        turn(i, x0, x1);
        if (i + 1 < n) turn(i + 1, x1, x0);
      }
    }
    l += __shfl_xor(l, 16, 64);
    l = halves(l, [](float p, float q) { return p + q; });

    // the waves' pieces, joined in wave order
    if (g == 0) {
      sm[wave][ln] = m;
      sl[wave][ln] = l;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int t = 0; t < VE; t += 4)
        *reinterpret_cast<f32x4*>(&so[wave][ln][VE * (4 * g + r) + t]) =
            f32x4{acc[t][r], acc[t + 1][r], acc[t + 2][r], acc[t + 3][r]};
    __syncthreads();
    const bool whole = u0 == 0 && u1 == nu;
    const int64_t slot = blockIdx.x * 2 + (u0 == 0);
    if (u0 == 0 && tid == 0) {
      const int64_t at = ((int64_t)b * heads + hb) * 2;
      a.shares[at] = blockIdx.x;
      a.shares[at + 1] = (int)div64(item + nu - 1, per);
    }
    for (int i = tid; i < nh * (D / 4); i += DT_THREADS) {
      const int h = i / (D / 4), d = i % (D / 4) * 4;
      float mm = sm[0][h];
#pragma unroll
      for (int w = 1; w < DW; ++w) mm = fmaxf(mm, sm[w][h]);
      const float mc = mm == -INFINITY ? 0.f : mm;
      float ll = 0.f;
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < DW; ++w) {
        const float f = exp2_hw(sm[w][h] - mc);
        ll += f * sl[w][h];
        x += f * *reinterpret_cast<const f32x4*>(&so[w][h][d]);
      }
      if (whole) {
        const float inv = ll == 0.f ? 0.f : 1.f / ll;
        *reinterpret_cast<u32x2*>(a.o + ((int64_t)b * a.hq + h0 + h) * D + d) =
            u32x2{pack2<DT>(x[0] * inv, x[1] * inv), pack2<DT>(x[2] * inv, x[3] * inv)};
        if (a.lse && d == 0) a.lse[(int64_t)b * a.hq + h0 + h] = ll == 0.f ? -INFINITY : (mc + __log2f(ll)) * LN2;
      } else {
        *reinterpret_cast<f32x4*>(a.po + (slot * 16 + h) * D + d) = x;
        if (d == 0) {
          a.pm[slot * 32 + h] = ll == 0.f ? -INFINITY : mc;
          a.pm[slot * 32 + 16 + h] = ll;
        }
      }
    }
    __syncthreads();
    u = item + u1;
    if (++hb == heads && u < uend) {  // the next sequence that has keys
      base += (int64_t)nu * heads;
      hb = 0;
      do len = __builtin_amdgcn_readfirstlane(seq_len(a, ++b));
      while (len == 0);
      nu = units_of(len);
    }
  }
}

// One workgroup per (sequence, query head): adds up the pieces that the shares cut the head's keys into, in order; zeros
// for a sequence without keys.  Groups of D / 4 threads take every so many-th piece, then their sums are added.
template <int D, int DT>
__global__ __launch_bounds__(256) void attn_join_kernel(DecodeArgs a) {
  constexpr int LPR = D / 4, G = 256 / LPR;
  __shared__ float red[4], wt[DECODE_GRID + 1];
  __shared__ __attribute__((aligned(16))) f32x4 part[G][LPR];
  __shared__ float psum[G];
  const int b = blockIdx.x / a.hq, hq = blockIdx.x % a.hq, tid = threadIdx.x;
  const int kvh = hq / a.group, h = hq % a.group % 16, hb = kvh * a.hblocks + hq % a.group / 16;
  const int grp = tid / LPR, d = tid % LPR * 4;
  const int64_t at = ((int64_t)b * a.hk * a.hblocks + hb) * 2;
  const bool empty = seq_len(a, b) == 0;
  // held to the grid, so that lengths changed between the two kernels make no read outside the workspace
  const int w0 = empty ? 0 : min(max(a.shares[at], 0), a.grid - 1);
  const int n = empty ? 0 : min(max(a.shares[at + 1] - w0 + 1, 1), a.grid - w0);
  if (n == 1) return;
  auto slot = [&](int i) { return (int64_t)(w0 + i) * 2 + (i == 0); };
  float m = -INFINITY;
  for (int i = tid; i < n; i += 256) m = fmaxf(m, wt[i] = a.pm[slot(i) * 32 + h]);
  m = wave_max(m);
  if (tid % 64 == 0) red[tid / 64] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  float l = 0.f;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  for (int i = grp; i < n; i += G) {
    const float f = wt[i] == -INFINITY ? 0.f : exp2_hw(wt[i] - m);
    l += f * a.pm[slot(i) * 32 + 16 + h];
    x += f * *reinterpret_cast<const f32x4*>(a.po + (slot(i) * 16 + h) * D + d);
  }
  part[grp][tid % LPR] = x;
  if (d == 0) psum[grp] = l;
  __syncthreads();
  if (grp) return;
  l = 0.f;
  x = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < G; ++i) {
    l += psum[i];
    x += part[i][tid];
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<u32x2*>(a.o + ((int64_t)b * a.hq + hq) * D + d) =
      u32x2{pack2<DT>(x[0] * inv, x[1] * inv), pack2<DT>(x[2] * inv, x[3] * inv)};
  if (a.lse && d == 0) a.lse[(int64_t)b * a.hq + hq] = l == 0.f ? -INFINITY : (m + __log2f(l)) * LN2;
}

// ------------------------------------------------------------------------------------ writing to the cache
// The new tokens of sequence b, rows [cu[b], cu[b + 1]) of k and v (without cu: row b), are the last ones of its
// seq_lens[b].  One 16-byte chunk a thread: 13 us for 14900 tokens of 2 heads of 256 (61 MB, 4.7 TB/s), 3.3 us for 64 tokens.
struct AppendArgs {
  CacheArgs c;
  const uint16_t *k, *v;
  int64_t k_row, k_head, v_row, v_head;
  const int32_t *cu, *lens;
  int nseq, rows, hk, dchunks;
};
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a) {
  const int64_t n = (int64_t)a.rows * a.hk * a.dchunks;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int row = (int)(i / (a.hk * a.dchunks)), rest = (int)(i % (a.hk * a.dchunks));
    const int h = rest / a.dchunks, c = rest % a.dchunks * 8;
    int b = row, after = 1;  // tokens from this one to the sequence's end
    if (a.cu) {
      int lo = 0, hi = a.nseq;  // the last sequence that starts at or before the row
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.cu[mid] <= row) lo = mid;
        else hi = mid;
      }
      b = lo;
      if (a.nseq == 0 || a.cu[b] > row) continue;
      after = a.cu[b + 1] - row;
      if (after <= 0) continue;  // behind the last sequence
    }
    const int pos = max(a.lens[b], 0) - after;
    if (pos < 0 || (pos >> a.c.page_log2) >= a.c.max_pages) continue;
    const int page = a.c.table[b * a.c.table_stride + (pos >> a.c.page_log2)];
    if ((unsigned)page >= (unsigned)a.c.num_pages) continue;
    const int slot = pos & ((1 << a.c.page_log2) - 1);
    const u32x4 x = *reinterpret_cast<const u32x4*>(a.k + row * a.k_row + h * a.k_head + c);
    const u32x4 y = *reinterpret_cast<const u32x4*>(a.v + row * a.v_row + h * a.v_head + c);
    *reinterpret_cast<u32x4*>(const_cast<uint16_t*>(a.c.k) + page * a.c.k_page + slot * a.c.k_slot + h * a.c.k_head + c) = x;
    *reinterpret_cast<u32x4*>(const_cast<uint16_t*>(a.c.v) + page * a.c.v_page + slot * a.c.v_slot + h * a.c.v_head + c) = y;
  }
}

// ------------------------------------------------------------------------------------ host
// Workgroups that the units are dealt to: as many as the registers let the GPU's CUs hold at a time, or one for every unit
// that the page table's width allows where that is less.  Twice as many at 256 wide, us for 512 and 256 workgroups: 32
// sequences of 4000, 16 heads over 2: 52.2 and 47.4; 64 of 100 to 8192: 106.6 and 100.5; 2 of 120000: 97.4 and 88.5; 200 of up
// to 2000: 97.9 and 96.1.
int64_t decode_grid(int64_t nseq, int64_t heads, int64_t d, int64_t max_pages, int64_t page_size) {
  const double most = (double)nseq * heads * (((double)max_pages * page_size + UK - 1) / UK);
  const int64_t full = CUS * decode_eu(d);
  return most < full ? std::max<int64_t>(1, (int64_t)most) : full;
}
size_t decode_parts_bytes(int64_t d) { return sizeof(float) * (size_t)DECODE_GRID * 2 * 16 * (size_t)(d + 2); }

}  // namespace
}  // namespace lsattn

using namespace lsattn;

extern "C" {

size_t lsurge_paged_attn_workspace_bytes(int64_t nseq, int64_t hq, int64_t d) {
  if (nseq < 0 || nseq >= (1 << 24) || hq < 1 || hq > 65535 || d < 1 || d > 256) return 0;
  return decode_parts_bytes(d) + sizeof(int32_t) * 2 * (size_t)(nseq * hq);
}

int lsurge_paged_attn(const lsurge_kv_cache* c, const lsurge_attn_rows* q, int64_t nseq, int64_t hq, float scale, void* o,
                      float* lse, void* workspace, size_t workspace_bytes, lsurge_stream_t stream) {
  DecodeArgs a;
  if (int rc = check_cache("paged_attn", c, &a.c)) return rc;
  LSURGE_REQUIRE(nseq >= 0 && nseq < (1 << 24) && hq >= c->heads && hq % c->heads == 0 && hq <= 65535,
                 "paged_attn: nseq=%lld, %lld query heads over %lld key heads", (long long)nseq, (long long)hq,
                 (long long)c->heads);
  LSURGE_REQUIRE(scale > 0.f && scale < INFINITY, "paged_attn: scale must be positive and finite");
  if (nseq == 0) return LSURGE_OK;
  if (int rc = check_new_rows("paged_attn q", q)) return rc;
  LSURGE_REQUIRE(o && workspace && ((uintptr_t)o | (uintptr_t)workspace) % 16 == 0,
                 "paged_attn: null or misaligned pointer");
  const size_t need = lsurge_paged_attn_workspace_bytes(nseq, hq, c->d);
  if (workspace_bytes < need)
    return lsurge::set_error(LSURGE_ERR_WORKSPACE, "paged_attn: workspace %zu < %zu bytes", workspace_bytes, need);
  LSURGE_REQUIRE((int64_t)c->max_pages * c->page_size <= (1ll << 30), "paged_attn: %lld pages of %lld tokens a sequence",
                 (long long)c->max_pages, (long long)c->page_size);
  a.q = (const uint16_t*)q->data, a.q_row = q->row_stride, a.q_head = q->head_stride;
  a.lens = c->seq_lens;
  a.nseq = (int)nseq, a.hq = (int)hq, a.hk = (int)c->heads, a.group = (int)(hq / c->heads);
  a.hblocks = (a.group + 15) / 16;
  a.scale2 = scale * LOG2E;
  a.o = (uint16_t*)o, a.lse = lse;
  a.grid = (int)decode_grid(nseq, (int64_t)a.hk * a.hblocks, c->d, c->max_pages, c->page_size);
  a.po = (float*)workspace;
  a.pm = a.po + (size_t)DECODE_GRID * 2 * 16 * c->d;
  a.shares = (int32_t*)((char*)workspace + decode_parts_bytes(c->d));
  const int64_t rows = nseq * hq;
  // the join's launch holds less than 2^32 threads, 256 a row
  LSURGE_REQUIRE(rows < (1ll << 24), "paged_attn: %lld sequences of %lld heads", (long long)nseq, (long long)hq);
  hipStream_t st = (hipStream_t)stream;
#define DECODE(D, DT)                                                                                              \
  LSURGE_LAUNCH(KID_ATTN, st, hipLaunchKernelGGL((attn_decode_kernel<D, DT>), dim3(a.grid), dim3(DT_THREADS), 0, st, a)); \
  LSURGE_LAUNCH(KID_ATTN, st, hipLaunchKernelGGL((attn_join_kernel<D, DT>), dim3((unsigned)rows), dim3(256), 0, st, a))
  if (c->dtype == LSURGE_BF16) {
    if (c->d == 64) { DECODE(64, LSURGE_BF16); }
    else if (c->d == 128) { DECODE(128, LSURGE_BF16); }
    else { DECODE(256, LSURGE_BF16); }
  } else {
    if (c->d == 64) { DECODE(64, LSURGE_F16); }
    else if (c->d == 128) { DECODE(128, LSURGE_F16); }
    else { DECODE(256, LSURGE_F16); }
  }
#undef DECODE
  return LSURGE_OK;
}

int lsurge_kv_append(const lsurge_kv_cache* c, const lsurge_attn_rows* k, const lsurge_attn_rows* v, int64_t rows,
                     int64_t nseq, const int32_t* cu, lsurge_stream_t stream) {
  AppendArgs a;
  if (int rc = check_cache("kv_append", c, &a.c)) return rc;
  LSURGE_REQUIRE(rows >= 0 && rows < (1ll << 31) && nseq >= 0 && nseq < (1 << 24) && (cu || rows == nseq),
                 "kv_append: %lld rows for %lld sequences", (long long)rows, (long long)nseq);
  if (rows == 0 || nseq == 0) return LSURGE_OK;
  if (int rc = check_new_rows("kv_append k", k)) return rc;
  if (int rc = check_new_rows("kv_append v", v)) return rc;
  a.k = (const uint16_t*)k->data, a.k_row = k->row_stride, a.k_head = k->head_stride;
  a.v = (const uint16_t*)v->data, a.v_row = v->row_stride, a.v_head = v->head_stride;
  a.cu = cu, a.lens = c->seq_lens;
  a.nseq = (int)nseq, a.rows = (int)rows, a.hk = (int)c->heads, a.dchunks = (int)c->d / 8;
  const int64_t chunks = rows * a.hk * a.dchunks;
  const unsigned grid = (unsigned)std::min<int64_t>((chunks + 255) / 256, 16384);
  hipStream_t st = (hipStream_t)stream;
  LSURGE_LAUNCH(KID_ATTN, st, hipLaunchKernelGGL(kv_append_kernel, dim3(grid), dim3(256), 0, st, a));
  return LSURGE_OK;
}

}  // extern "C"

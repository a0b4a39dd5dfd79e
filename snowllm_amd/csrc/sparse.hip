// Attention over selected pages of the paged KV cache, in four operators:
//
//   append   the cache write of new rows: optional per-head RMSNorm, rotate-half RoPE, K/V into
//            the pages, and the bounds of every page written (element-wise minimum and maximum of
//            the page's live keys)
//   bounds   the same bounds from pages that another writer filled
//   select   per row and kv head, the pages with the largest upper bound of their scores
//   attend   softmax attention of each row over its listed pages only
//
// Pools are the paged attention's: K [blocks, Hkv, d/16, 16, 16], V [blocks, Hkv, 4, d, 4], page =
// 16, bf16. Bounds are [blocks, Hkv, 2, d] bf16 (minima, then maxima), 1/16 of the K and V bytes.
// Rows are padded [batch, tokens]; request b's page p is block table[b, p].
#include "common.h"
#include "pages.h"

#include <algorithm>
#include <atomic>

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef short short2v __attribute__((ext_vector_type(2)));

// bf16 pairs as signed 16-bit keys in the order of their values (and back: it is an involution),
// so that minima and maxima are one packed integer operation for two elements. NaNs lie outside
// the infinities: above +inf or below -inf, by their sign.
__device__ __forceinline__ short2v order_keys(uint32_t w) {
  const short2v x = __builtin_bit_cast(short2v, w);
  return x ^ ((x >> (short)15) & (short)0x7fff);
}
__device__ __forceinline__ short2v min2(short2v a, short2v b) { return __builtin_elementwise_min(a, b); }
__device__ __forceinline__ short2v max2(short2v a, short2v b) { return __builtin_elementwise_max(a, b); }
constexpr short KEY_INF = 0x7f80, KEY_NEG_INF = (short)0x807f;   // keys of +inf and -inf

// Keys back to bf16 words; a NaN among a page's elements makes both its bounds NaN.
__device__ __forceinline__ void bounds_words(short2v lo, short2v hi, uint32_t& wlo, uint32_t& whi) {
  const uint32_t a = __builtin_bit_cast(uint32_t, order_keys(__builtin_bit_cast(uint32_t, lo)));
  const uint32_t b = __builtin_bit_cast(uint32_t, order_keys(__builtin_bit_cast(uint32_t, hi)));
  const uint32_t nan = (lo.x < KEY_NEG_INF || hi.x > KEY_INF ? 0x7fc0u : 0u) |
                       (lo.y < KEY_NEG_INF || hi.y > KEY_INF ? 0x7fc00000u : 0u);
  wlo = a | nan;
  whi = b | nan;
}

// ---------------------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------------------
struct AppendArgs {
  const uint16_t* k;       // row m, head h at k + m * k_stride + h * D
  const uint16_t* v;
  QueryRows rows;          // the queries, rotated alongside
  int64_t k_stride, v_stride;
  const float* cosv;       // [rows, half], rows cs_stride apart
  const float* sinv;
  int64_t cs_stride;
  const uint16_t* k_gamma; // null: no norm
  float eps;
  uint16_t* k_pool;
  uint16_t* v_pool;
  uint16_t* bounds;        // null: none kept
  const int32_t* table;
  const int32_t* starts;   // [batch] position of a request's first row
  const int32_t* counts;   // [batch] its rows
  int64_t table_stride, blocks;
  int batch, T, Hkv, half, pages;   // pages: most pages that T rows touch
  int64_t page_wgs;        // workgroups over (request, page, kv head); the rest rotate queries
};

// Bound by its bytes: four prompts of about 2048 rows (q and k normalised, 150 MB) take 31 us (4.8 TB/s); one
// row of a 128-wide model 4 us, a dependent load of start, table entry and rows each. A thread has four heads
// of queries (41 us against 47 with one, when gammas and angles were loaded for each head and the queries went
// through the caches).
// 2 D threads: sixteen heads of D / 8 threads each. A page workgroup owns one (request, page, kv
// head): its threads take a token's row each, normalise and rotate it, and pass it through LDS into
// the page's layout, so that global reads and writes are both contiguous. The page's bounds are
// taken from the same LDS image, to which the page's older keys are loaded first: they come out the
// same whatever was in the page behind the last row (rejected drafts) and need no atomics.
template <int D, bool PASS_BY>
__global__ void __launch_bounds__(2 * D) append_kernel(AppendArgs a) {
  constexpr int W = D / 8, LD = D + 8;   // row pitch of the LDS tiles: 16 bytes more than a row
  __shared__ __attribute__((aligned(16))) uint16_t ks[PAGE * LD];
  __shared__ __attribute__((aligned(16))) uint16_t vs[PAGE * LD];
  const int tid = threadIdx.x, r = tid / W, c = tid % W;
  int64_t wg = blockIdx.x;
  if (wg >= a.page_wgs) {   // queries: sixteen units of a row and Q_HEADS heads
    rotate_queries<D, PASS_BY>((uint32_t)(wg - a.page_wgs) * 16 + r, c, a.rows);
    return;
  }
  const int h = (int)(wg % a.Hkv);
  wg /= a.Hkv;
  const int j = (int)(wg % a.pages), b = (int)(wg / a.pages);
  const int64_t start = a.starts[b];
  int64_t count = a.counts[b];
  count = count < a.T ? count : a.T;
  if (start < 0 || count <= 0) return;
  const int64_t page = start / PAGE + j, first = page * PAGE;
  const int64_t end = start + count;   // one past the last position
  if (first >= end) return;
  const int blk = page_block(a.table, a.table_stride, b, page, a.blocks);
  if (blk < 0) return;
  const int lo = start > first ? (int)(start - first) : 0;             // new tokens lo .. hi - 1
  const int hi = end - first < PAGE ? (int)(end - first) : PAGE;
  const int64_t base = ((int64_t)blk * a.Hkv + h) * PAGE * D;
  uint16_t* kp = a.k_pool + base;
  uint16_t* vp = a.v_pool + base;
  // unit u of the K page: 16 bytes of token (u / 2) % 16, elements 16 (u / 32) + 8 (u % 2) ..
  const int ku = (tid >> 5) * 16 + (tid & 1) * 8, ktok = (tid >> 1) & 15;
  if (ktok < lo) *(u32x4*)(ks + ktok * LD + ku) = *(const u32x4*)(kp + tid * 8);
  {
    const bool live = r >= lo && r < hi;
    const int64_t m = (int64_t)b * a.T + (live ? first + r - start : 0);
    u32x4 kraw = {0u, 0u, 0u, 0u}, vraw = {0u, 0u, 0u, 0u};
    if (live) {
      kraw = *(const u32x4*)(a.k + m * a.k_stride + (int64_t)h * D + 8 * c);
      vraw = *(const u32x4*)(a.v + m * a.v_stride + (int64_t)h * D + 8 * c);
    }
    const u32x4 o = rotate_norm<D>(kraw, load_rotation(c, a.k_gamma, a.eps, a.cosv + m * a.cs_stride,
                                                       a.sinv + m * a.cs_stride, a.half));
    if (live) {
      *(u32x4*)(ks + r * LD + 8 * c) = o;
      *(u32x4*)(vs + r * LD + 8 * c) = vraw;
    }
  }
  __syncthreads();
  if (ktok >= lo && ktok < hi) *(u32x4*)(kp + tid * 8) = *(const u32x4*)(ks + ktok * LD + ku);
  // unit of the V page: tokens 4 tg .. 4 tg + 3 of elements d, d + 1
  const int tg = tid / (D / 2), d = tid % (D / 2) * 2;
  if (4 * tg >= lo && 4 * tg + 4 <= hi) {
    uint32_t w[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) w[t] = *(const uint32_t*)(vs + (4 * tg + t) * LD + d);
    u32x4 o;
    o[0] = (w[0] & 0xffffu) | w[1] << 16;
    o[1] = (w[2] & 0xffffu) | w[3] << 16;
    o[2] = w[0] >> 16 | (w[1] & 0xffff0000u);
    o[3] = w[2] >> 16 | (w[3] & 0xffff0000u);
    *(u32x4*)(vp + (tg * D + d) * 4) = o;
  } else {
    for (int t = 4 * tg; t < 4 * tg + 4; ++t)
      if (t >= lo && t < hi) {
        vp[(tg * D + d) * 4 + (t & 3)] = vs[t * LD + d];
        vp[(tg * D + d + 1) * 4 + (t & 3)] = vs[t * LD + d + 1];
      }
  }
  if (a.bounds && tid < D / 2) {   // two elements a thread
    short2v l = order_keys(*(const uint32_t*)(ks + 2 * tid)), u = l;
    for (int t = 1; t < hi; ++t) {
      const short2v x = order_keys(*(const uint32_t*)(ks + t * LD + 2 * tid));
      l = min2(l, x);
      u = max2(u, x);
    }
    uint32_t wl, wu;
    bounds_words(l, u, wl, wu);
    uint16_t* bp = a.bounds + ((int64_t)blk * a.Hkv + h) * 2 * D;
    *(uint32_t*)(bp + 2 * tid) = wl;
    *(uint32_t*)(bp + D + 2 * tid) = wu;
  }
}

// ---------------------------------------------------------------------------------------
// bounds
// ---------------------------------------------------------------------------------------
// Lane swaps for the bounds: with the lane 2 away, and with one 4 or 6 away (the values of those two
// are equal by then).
__device__ __forceinline__ short2v lanes_xor2(short2v v) {
  return __builtin_bit_cast(short2v, dpp_u32<DPP_QUAD_XOR2>(__builtin_bit_cast(uint32_t, v)));
}
__device__ __forceinline__ short2v lanes_xor4(short2v v) {
  return __builtin_bit_cast(short2v, dpp_u32<DPP_QUAD_XOR1>(dpp_u32<DPP_HALF_MIRROR>(__builtin_bit_cast(uint32_t, v))));
}

// A half wave takes 64 elements of a (page, kv head), that is four chunks of [16 tokens][16], in four
// loads that are whole 128-byte lines: lane (chunk, token % 4, half chunk). A lane's four tokens meet in
// its registers, the four lanes of an element by lane swaps. A page's dead tokens are read as its last
// live one. Bound by the read of K: 220K
// tokens of two 256-wide heads 52 us (4.9 TB/s) from HBM, 36 from the last-level cache.
template <int D>
__global__ void __launch_bounds__(256) page_bounds_kernel(
    const uint16_t* __restrict__ k_pool, uint16_t* __restrict__ bounds,
    const int32_t* __restrict__ table, const int32_t* __restrict__ starts,
    const int32_t* __restrict__ counts, int64_t table_stride, int64_t blocks, int batch, int Hkv,
    int tokens, int64_t pages) {
  constexpr int SLABS = D / 64;
  int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) / 32;
  const int lane = threadIdx.x & 31, half = lane & 1, quarter = lane >> 1 & 3, chunk = lane >> 3;
  const int slab = (int)(unit % SLABS);
  unit /= SLABS;
  const int h = (int)(unit % Hkv);
  const int64_t j = unit / Hkv % pages, b = unit / Hkv / pages;
  if (b >= batch) return;
  const int64_t start = starts[b];
  int64_t count = counts[b];
  count = count < tokens ? count : tokens;
  if (start < 0 || count <= 0) return;
  const int64_t page = start / PAGE + j, left = start + count - page * PAGE;
  if (left <= 0) return;
  const int blk = page_block(table, table_stride, (int)b, page, blocks);
  if (blk < 0) return;
  const int last = left < PAGE ? (int)left - 1 : PAGE - 1;
  const uint16_t* kp = k_pool + ((int64_t)blk * Hkv + h) * PAGE * D + (slab * 4 + chunk) * 256 + half * 8;
  u32x4 x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = 4 * i + quarter;
    x[i] = *(const u32x4*)(kp + (t < last ? t : last) * 16);
  }
  u32x4 wl, wu;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    short2v l = order_keys(x[0][i]), u = l;
#pragma unroll
    for (int t = 1; t < 4; ++t) {
      const short2v k = order_keys(x[t][i]);
      l = min2(l, k);
      u = max2(u, k);
    }
    l = min2(l, lanes_xor2(l));
    u = max2(u, lanes_xor2(u));
    l = min2(l, lanes_xor4(l));
    u = max2(u, lanes_xor4(u));
    uint32_t a0, b0;
    bounds_words(l, u, a0, b0);
    wl[i] = a0;
    wu[i] = b0;
  }
  uint16_t* bp = bounds + ((int64_t)blk * Hkv + h) * 2 * D + slab * 64 + chunk * 16 + half * 8;
  if (quarter == 0) *(u32x4*)bp = wl;
  if (quarter == 1) *(u32x4*)(bp + D) = wu;
}

// ---------------------------------------------------------------------------------------
// select
// ---------------------------------------------------------------------------------------
// A page's score for a row and kv head is the sum over the group's heads of the largest q . k that
// keys within the page's bounds could have:
//   s = sum_g sum_d max(q_gd low_d, q_gd high_d) = sum_d P_d high_d + N_d low_d,
//   P_d = sum_g max(q_gd, 0), N_d = sum_g min(q_gd, 0),
// one product of 2 D terms per (row, kv head, page), as long as all is finite. The choice turns on
// differences between nearly equal scores, so it is made on 64-bit sums; but only few pages are near
// the border. The matrix cores give every page a 32-bit s~ and a bound E on its error; with t the
// need-th largest s~, a page above t + 2 E is chosen and one below t - 2 E is not whatever the exact
// sums are, and only the pages between are summed in 64 bits.
//
// E: with A = sum_d |P_d high_d| + |N_d low_d|,
//   P and N are 32-bit sums of G values                               <= G 2^-24 A
//   each is multiplied as two bf16 pieces, what is left is            <= 2^-16 A
//   2 . 2 D / 32 matrix instructions add to one accumulator, each taken to make at most 16 roundings
//   of 2^-24 of what has been summed                                  <= 2 D 2^-24 A
// (over normal, positive, rising and heavy-tailed operands of 64- to 256-wide heads the whole error came
// to 2^-17.7 A at most, nearly all of it the second), A from a third product of the larger pieces with
// |bounds| (2^-8 too small at most: 1.01 A). What the matrix cores could flush (below 2^-126) adds at
// most 2^-74: a row has E = infinity, and all its pages summed in 64 bits, where a P or |N| is below
// 2^-90 (and not 0) or above 2^40, or anything is not finite.
struct SelectArgs {
  const uint16_t* q;        // [rows, Hq, D]
  const uint16_t* bounds;
  const int32_t* table;
  const int32_t* positions; // [rows] the last position a row sees, negative: none
  int32_t* pages;           // [rows, Hkv, budget]
  float* scores;            // [requests, Hkv, rows, width] s~
  float* errors;            // [requests, Hkv, rows, width / 16] E of 16 pages
  uint64_t* exact;          // [requests, Hkv, rows, width] keys, where a row needs them all
  u32x4* operands;          // [requests, Hkv, row tiles] of more than sixteen rows
  int32_t* tile_last;       // [requests, row tiles] pages seen
  int64_t table_stride, blocks, width, T, row0;   // row0: first row of every request in this launch
  int rows, Hq, Hkv, G, budget, sink, recent;     // rows: of a request in this launch
};

// Pages a row sees.
__device__ __forceinline__ int64_t pages_seen(int pos, int64_t stride) {
  const int64_t n = pos < 0 ? 0 : pos / PAGE + 1;
  return n < stride ? n : stride;
}

__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ float pos_part(float f) { return !(f <= 0.f) ? f : 0.f; }   // NaN stays
__device__ __forceinline__ float neg_part(float f) { return !(f >= 0.f) ? f : 0.f; }

constexpr int SCORE_WAVES = 4;

// The sums P and N of sixteen rows, of which `live` are rows, both pieces, as operands of
// v_mfma_f32_16x16x32_bf16 in LDS: [D / 16 steps of 32 terms][piece][64 lanes], D terms of N (for the
// minima), then D of P. By 256 threads, four elements d .. of a row at a time (D / 4 threads a row), all
// heads of them; a row's slots are rotated by (d / 8) % 16, so that its threads write to different banks.
template <int D>
__device__ __forceinline__ void rows_operand(const SelectArgs& a, int64_t m0, int h, int live, uint16_t* ops) {
  constexpr int NS = D / 16, UNITS = 16 * (D / 4) / (64 * SCORE_WAVES), PER = 64 * SCORE_WAVES / (D / 4);
  const int tid = threadIdx.x;
  float pp[UNITS][4], nn[UNITS][4];
#pragma unroll
  for (int k = 0; k < UNITS; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) pp[k][i] = nn[k][i] = 0.f;
  const int r0 = tid / (D / 4), d = tid % (D / 4) * 4;
  const uint16_t* qp = a.q + ((m0 + r0) * a.Hq + (int64_t)h * a.G) * D + d;
  const int64_t row_step = (int64_t)PER * a.Hq * D;
#pragma unroll 4
  for (int e = 0; e < a.G; ++e) {
    uint2 w[UNITS];
#pragma unroll
    for (int k = 0; k < UNITS; ++k) {
      w[k] = uint2{0u, 0u};
      if (r0 + k * PER < live) w[k] = *(const uint2*)(qp + k * row_step + (int64_t)e * D);
    }
#pragma unroll
    for (int k = 0; k < UNITS; ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t x2 = i ? w[k].y : w[k].x;
        const short2v sign = __builtin_bit_cast(short2v, x2) >> (short)15;   // -1 where negative
        const uint32_t ng = x2 & __builtin_bit_cast(uint32_t, sign), ps = x2 & ~__builtin_bit_cast(uint32_t, sign);
        pp[k][2 * i] += bf_lo(ps);
        pp[k][2 * i + 1] += bf_hi(ps);
        nn[k][2 * i] += bf_lo(ng);
        nn[k][2 * i + 1] += bf_hi(ng);
      }
  }
#pragma unroll
  for (int k = 0; k < UNITS; ++k) {
    const int r = r0 + k * PER;
    uint2 ph, pl, nh, nl;
#pragma unroll
    for (int i = 0; i < 4; ++i) {   // NaN: the row's scores are not to be trusted
      const float most = fmaxf(pp[k][i], -nn[k][i]);
      const bool small = (pp[k][i] > 0.f && pp[k][i] < 0x1p-90f) || (nn[k][i] < 0.f && nn[k][i] > -0x1p-90f);
      if (small || most > 0x1p40f) pp[k][i] = __builtin_nanf("");
    }
    ph.x = pack_bf16x2(pp[k][0], pp[k][1]);
    ph.y = pack_bf16x2(pp[k][2], pp[k][3]);
    nh.x = pack_bf16x2(nn[k][0], nn[k][1]);
    nh.y = pack_bf16x2(nn[k][2], nn[k][3]);
    pl.x = pack_bf16x2(pp[k][0] - bf_lo(ph.x), pp[k][1] - bf_hi(ph.x));
    pl.y = pack_bf16x2(pp[k][2] - bf_lo(ph.y), pp[k][3] - bf_hi(ph.y));
    nl.x = pack_bf16x2(nn[k][0] - bf_lo(nh.x), nn[k][1] - bf_hi(nh.x));
    nl.y = pack_bf16x2(nn[k][2] - bf_lo(nh.y), nn[k][3] - bf_hi(nh.y));
    const int st = d / 32, slot = (d / 8 % 4) * 16 + ((r + d / 8) & 15);
    uint16_t* to = ops + (st * 2 * 64 + slot) * 8 + d % 8;
    *(uint2*)to = nh;
    *(uint2*)(to + 64 * 8) = nl;
    *(uint2*)(to + NS * 64 * 8) = ph;           // NS / 2 steps of two pieces on
    *(uint2*)(to + NS * 64 * 8 + 64 * 8) = pl;
  }
}

// Lane (col, g)'s slot in step s of such an operand.
template <int D>
__device__ __forceinline__ int operand_slot(int s, int col, int g) {
  return g * 16 + ((col + s % (D / 32) * 4 + g) & 15);
}

// One step of 32 terms for PT times sixteen pages: s~ and the sum of the terms' magnitudes.
template <int PT>
__device__ __forceinline__ void score_step(bool minima, const u32x4* x, u32x4 hi, u32x4 lo, floatx4 (&acc)[PT],
                                           floatx4 (&mag)[PT], int pitch) {
  const bf16x8 wh = __builtin_bit_cast(bf16x8, hi), wl = __builtin_bit_cast(bf16x8, lo);
  u32x4 ab[PT];   // |bounds|, with the sign of the larger piece: N is negative
#pragma unroll
  for (int i = 0; i < PT; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) ab[i][k] = minima ? x[i * pitch][k] | 0x80008000u : x[i * pitch][k] & 0x7fff7fffu;
#pragma unroll
  for (int i = 0; i < PT; ++i)
    acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x[i * pitch]), wh, acc[i], 0, 0, 0);
#pragma unroll
  for (int i = 0; i < PT; ++i)
    mag[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, ab[i]), wh, mag[i], 0, 0, 0);
#pragma unroll
  for (int i = 0; i < PT; ++i)
    acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x[i * pitch]), wl, acc[i], 0, 0, 0);
}

// E of a tile of sixteen pages from page pt (lane (row col, g): pages pt + 4 g + k), whose first
// `sink`, always chosen, and those from `last` on do not count; what is no page (bits of none) scores
// -inf.
template <int D>
__device__ __forceinline__ float tile_error(const SelectArgs& a, int64_t pt, int64_t last, uint32_t none, int g,
                                            floatx4& acc, floatx4 mag) {
  const float rel = 1.01f * (0x1p-16f + (float)(2 * D + a.G) * 0x1p-24f), inf = __builtin_huge_valf();
  float e = 0.f;
  if (none == 0 && pt >= a.sink && pt + 16 <= last) {
    const float sum = (mag[0] + mag[1]) + (mag[2] + mag[3]);   // infinite or NaN where one of them is
    e = sum < 0x1p120f ? __builtin_fmaf(rel, fmaxf(fmaxf(mag[0], mag[1]), fmaxf(mag[2], mag[3])), 0x1p-74f) : inf;
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool no = none >> (4 * g + k) & 1;
      if (no) acc[k] = -inf;
      const int64_t pg = pt + 4 * g + k;
      if (!no && pg >= a.sink && pg < last) {
        const float e1 = __builtin_fmaf(rel, mag[k], 0x1p-74f);
        e = e1 < 0x1p120f ? fmaxf(e, e1) : inf;   // NaN too
      }
    }
  }
  return column_max(e);
}

// This lane's bounds of PT times sixteen pages from page p: blocks (-1: no page; past the table's end
// its last page's), then 16-byte loads of each step.
template <int D, int PT>
struct PageTiles {
  int blk[PT];
  u32x4 x[PT][D / 16];
  __device__ __forceinline__ void entries(const SelectArgs& a, int b, int64_t p, int col) {
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      const int64_t pg = p + 16 * i + col;
      blk[i] = page_block(a.table, a.table_stride, b, pg < a.table_stride ? pg : a.table_stride - 1, a.blocks);
    }
  }
  __device__ __forceinline__ void fetch(const SelectArgs& a, int h, int g) {
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      const uint16_t* bp = a.bounds + ((int64_t)(blk[i] < 0 ? 0 : blk[i]) * a.Hkv + h) * 2 * D + 8 * g;
#pragma unroll
      for (int s = 0; s < D / 16; ++s) x[i][s] = *(const u32x4*)(bp + 32 * s);
    }
  }
};

// Bound by the bytes of the bounds where the cache is long: 32 requests of 16K to 32K tokens and eight
// 128-wide kv heads, 205 MB read in 48 us (4.3 TB/s); eleven rows at 220K and two 256-wide heads 12 us
// (28 MB from the last-level cache); 8 us for one row at 8K, a chain of loads (position, table, bounds) and
// of the rows' sums. Up to sixteen rows of a request and kv head a workgroup, which sums them for itself. A wave takes
// PT times sixteen pages at a time, whose bounds are an operand as they lie in memory: they are read
// ahead of the rows' sums, and each step's pages while the last one's scores are stored. Two page
// tiles to each read of the rows' operand keep LDS (85 bytes a clock) behind the matrix cores.
template <int D, int PT>
__global__ void __launch_bounds__(64 * SCORE_WAVES, 2) score_kernel(SelectArgs a, uint32_t pages_per_wg) {
  constexpr int NS = D / 16;
  __shared__ u32x4 op[NS][2][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), col = lane & 15, g = lane >> 4;
  uint32_t y = blockIdx.x;
  const int h = (int)(y % (uint32_t)a.Hkv), b = (int)(y / (uint32_t)a.Hkv);
  const int64_t m0 = (int64_t)b * a.T + a.row0;
  const int live = a.rows;
  const int64_t p0 = (int64_t)blockIdx.y * pages_per_wg;
  PageTiles<D, PT> t;
  int64_t p = p0 + 16 * PT * wave;
  t.entries(a, b, p, col);
  const int pos = lane < live ? a.positions[m0 + lane] : -1;
  t.fetch(a, h, g);
  const int64_t last = (int64_t)wave_max<int>((int)pages_seen(pos, a.table_stride));
  if (p0 >= last) return;
  const int64_t p1 = p0 + pages_per_wg < last ? p0 + pages_per_wg : last;
  rows_operand<D>(a, m0, h, live, (uint16_t*)op);
  __syncthreads();
  const int64_t item = ((int64_t)b * a.Hkv + h) * a.rows + col;
  for (; p < p1; p += 16 * PT * SCORE_WAVES) {
    uint32_t none[PT];
#pragma unroll
    for (int i = 0; i < PT; ++i) none[i] = (uint32_t)__ballot(t.blk[i] < 0);
    const bool more = p + 16 * PT * SCORE_WAVES < p1;
    if (more) t.entries(a, b, p + 16 * PT * SCORE_WAVES, col);
    floatx4 acc[PT], mag[PT];
#pragma unroll
    for (int i = 0; i < PT; ++i) acc[i] = mag[i] = floatx4{0.f, 0.f, 0.f, 0.f};
    u32x4 w[3][2];
    auto operand = [&](int s) {
      const int slot = operand_slot<D>(s, col, g);
      w[s % 3][0] = op[s][0][slot], w[s % 3][1] = op[s][1][slot];
    };
    operand(0);
    operand(1);
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      // two steps ahead and no more: held over the loop they would not fit the registers
      asm volatile("" ::: "memory");
      if (s + 2 < NS) operand(s + 2);
      __builtin_amdgcn_sched_barrier(0);
      score_step<PT>(s < NS / 2, &t.x[0][s], w[s % 3][0], w[s % 3][1], acc, mag, NS);
    }
    if (more) t.fetch(a, h, g);
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      const int64_t pt = p + 16 * i;
      const float e = tile_error<D>(a, pt, last, none[i], g, acc[i], mag[i]);
      if (col < live && pt < p1) {
        *(floatx4*)(a.scores + item * a.width + pt + 4 * g) = acc[i];
        if (g == 0) a.errors[item * (a.width / 16) + pt / 16] = e;
      }
    }
  }
}

// More rows: their operands once, into the workspace, in tiles of sixteen; with each the most pages
// that one of its rows sees.
template <int D>
__global__ void __launch_bounds__(64 * SCORE_WAVES) operand_kernel(SelectArgs a) {
  constexpr int NS = D / 16;
  __shared__ u32x4 op[NS * 2 * 64];
  const int tiles = (a.rows + 15) / 16, lane = threadIdx.x & 63;
  uint32_t y = blockIdx.x;
  const int tile = (int)(y % (uint32_t)tiles);
  y /= (uint32_t)tiles;
  const int h = (int)(y % (uint32_t)a.Hkv), b = (int)(y / (uint32_t)a.Hkv);
  const int64_t m0 = (int64_t)b * a.T + a.row0 + tile * 16;
  const int live = a.rows - tile * 16 < 16 ? a.rows - tile * 16 : 16;
  rows_operand<D>(a, m0, h, live, (uint16_t*)op);
  const int last = wave_max<int>((int)pages_seen(lane < live ? a.positions[m0 + lane] : -1, a.table_stride));
  if (h == 0 && threadIdx.x == 0) a.tile_last[b * tiles + tile] = last;
  __syncthreads();
  u32x4* out = a.operands + (int64_t)blockIdx.x * (NS * 2 * 64);
#pragma unroll
  for (int i = 0; i < NS * 2 / SCORE_WAVES; ++i) out[i * 256 + threadIdx.x] = op[i * 256 + threadIdx.x];
}

// Many rows are bound by the products, three of 16 x 16 x 2 D per page tile and row tile: 1024 rows over
// 4064 pages, two 256-wide kv heads, 34 us (8.5 GFLOP that are needed, 13 with the products for E; matrix
// cores 38 % busy, the rest LDS reads of the operands and the stores of the scores); the whole choice 62 us,
// 82 with workgroups of the other form, one for each sixteen rows, which read and sum everything again.
// A wave keeps the bounds of 32 pages in registers and goes over the row tiles of its part of the
// rows, whose operands come through LDS for all four waves (global_load_lds), the next tile's while
// one is used. A tile's scores are stored a step later, so that the one wait of a step is for loads
// and stores that have had a step's time.
template <int D>
__global__ void __launch_bounds__(64 * SCORE_WAVES, 2) score_rows_kernel(SelectArgs a, uint32_t tiles_per_wg,
                                                                       uint32_t columns) {
  typedef __attribute__((address_space(3))) void lds_void;
  constexpr int NS = D / 16, PT = 2, TILE = NS * 2 * 64;   // 16-byte words of a row tile's operands
  __shared__ u32x4 op[2][TILE];
  const int lane = threadIdx.x & 63, wave = wave_id(), col = lane & 15, g = lane >> 4;
  const int tiles = (a.rows + 15) / 16;
  const uint32_t parts = ((uint32_t)tiles + tiles_per_wg - 1) / tiles_per_wg;
  uint32_t y = blockIdx.x / columns;
  const int t0 = (int)(y % parts * tiles_per_wg);
  y /= parts;
  const int h = (int)(y % (uint32_t)a.Hkv), b = (int)(y / (uint32_t)a.Hkv);
  const int t1 = t0 + (int)tiles_per_wg < tiles ? t0 + (int)tiles_per_wg : tiles;
  const int64_t p = (int64_t)(blockIdx.x % columns) * (16 * PT * SCORE_WAVES) + 16 * PT * wave;
  const u32x4* src = a.operands + ((int64_t)b * a.Hkv + h) * tiles * TILE + lane;
  auto load = [&](int t) {
#pragma unroll
    for (int i = 0; i < TILE / 64 / SCORE_WAVES; ++i) {
      const int c = i * SCORE_WAVES + wave;
      __builtin_amdgcn_global_load_lds((const void*)(src + (int64_t)t * TILE + c * 64), (lds_void*)&op[t & 1][c * 64], 16, 0, 0);
    }
  };
  PageTiles<D, PT> t;
  t.entries(a, b, p, col);
  load(t0);
  t.fetch(a, h, g);
  uint32_t none[PT];
#pragma unroll
  for (int i = 0; i < PT; ++i) none[i] = (uint32_t)__ballot(t.blk[i] < 0);
  floatx4 acc[PT], mag[PT];
  float err[PT] = {};
  const int lasts = t0 + lane < t1 ? a.tile_last[b * tiles + t0 + lane] : 0;   // at most 64 tiles
  int64_t done_last = 0;   // pages that the last tile's rows see: what of it is stored
  auto store = [&](int r) {
    const int64_t item = ((int64_t)b * a.Hkv + h) * a.rows + r * 16 + col;
#pragma unroll
    for (int i = 0; i < PT; ++i)
      if (p + 16 * i < done_last && r * 16 + col < a.rows) {
        *(floatx4*)(a.scores + item * a.width + p + 16 * i + 4 * g) = acc[i];
        if (g == 0) a.errors[item * (a.width / 16) + p / 16 + i] = err[i];
      }
  };
  for (int r = t0; r < t1; ++r) {
    wait_vmcnt<0>();
    wait_lgkmcnt0();
    block_barrier();
    store(r - 1);
    if (r + 1 < t1) load(r + 1);
    done_last = __builtin_amdgcn_readlane(lasts, r - t0);
    if (p >= done_last) continue;
#pragma unroll
    for (int i = 0; i < PT; ++i) acc[i] = mag[i] = floatx4{0.f, 0.f, 0.f, 0.f};
    u32x4 w[3][2];
    auto operand = [&](int s) {
      const u32x4* o = op[r & 1] + s * 128 + operand_slot<D>(s, col, g);
      w[s % 3][0] = o[0], w[s % 3][1] = o[64];
    };
    operand(0);
    operand(1);
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      asm volatile("" ::: "memory");
      // or the loop would hold |bounds| too
#pragma unroll
      for (int i = 0; i < PT; ++i) asm volatile("" : "+v"(t.x[i][s]));
      if (s + 2 < NS) operand(s + 2);
      __builtin_amdgcn_sched_barrier(0);
      score_step<PT>(s < NS / 2, &t.x[0][s], w[s % 3][0], w[s % 3][1], acc, mag, NS);
    }
#pragma unroll
    for (int i = 0; i < PT; ++i) err[i] = tile_error<D>(a, p + 16 * i, done_last, none[i], g, acc[i], mag[i]);
  }
  store(t1 - 1);
}

// 64-bit keys in the order of the scores; NaN is -inf, -0 is +0 (the rule of ord_key).
__device__ __forceinline__ uint64_t score_key(double s) {
  if (s != s) s = -__builtin_huge_val();
  if (s == 0.0) s = 0.0;
  const uint64_t u = (uint64_t)__double_as_longlong(s);
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

// Inclusive sum over a wave.
__device__ __forceinline__ uint32_t wave_incl_sum_u32(uint32_t v) {
  v = row_scan_u32_dpp(v);
  const int lane = threadIdx.x & 63;
  const uint32_t a = (uint32_t)__builtin_amdgcn_readlane((int)v, 15);
  const uint32_t b = (uint32_t)__builtin_amdgcn_readlane((int)v, 31);
  const uint32_t c = (uint32_t)__builtin_amdgcn_readlane((int)v, 47);
  return v + (lane >= 16 ? a : 0u) + (lane >= 32 ? b : 0u) + (lane >= 48 ? c : 0u);
}

constexpr int PICK_NEAR = 512;    // pages near the border that are ranked in LDS
constexpr int PICK_KEYS = 16;     // scores a thread keeps in registers

// The 64-bit score's key of one page for row m, by a wave: lane l sums terms l, l + 64, .. in order, then
// a fixed tree, so that equal pages have equal sums. pn [2 D]: N, then P. N low + P high is not the sum
// over g of max(q_gd low, q_gd high) where one of them is not finite (N = 0 and low = -inf: NaN for
// q_gd high); its sum is not finite then, and the page is summed head by head, NaN where a product is.
// FINITE: there is no such page, as everywhere where E is finite.
template <int D, bool FINITE>
__device__ __forceinline__ uint64_t exact_key(const SelectArgs& a, const double* pn, int64_t m, int b, int h,
                                              int64_t page) {
  const int lane = threadIdx.x & 63;
  const int blk = page_block(a.table, a.table_stride, b, page, a.blocks);
  if (blk < 0) return score_key(-__builtin_huge_val());
  const uint16_t* bp = a.bounds + ((int64_t)blk * a.Hkv + h) * 2 * D;
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < 2 * D / 64; ++i) s += pn[64 * i + lane] * (double)bf16_to_f32(bp[64 * i + lane]);
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) s += __shfl_xor(s, k, 64);
  if (!FINITE && !__builtin_isfinite(s)) {   // the same in all lanes
    const uint16_t* qp = a.q + (m * a.Hq + (int64_t)h * a.G) * D;
    s = 0.0;
    int i = lane;
    asm volatile("" : "+v"(i));   // no address of it is held before
#pragma unroll 1
    for (; i < a.G * D; i += 64) {   // head i / D, element i % D
      const double q = bf16_to_f32(qp[i]), x = q * bf16_to_f32(bp[i % D]), y = q * bf16_to_f32(bp[D + i % D]);
      s += x > y ? x : y >= x ? y : __builtin_nan("");
    }
#pragma unroll
    for (int k = 32; k > 0; k >>= 1) s += __shfl_xor(s, k, 64);
  }
  return score_key(s);
}

// One workgroup per (row, kv head). CACHED: its scores fit the threads' registers. One row is bound by the
// chain of its barriers and reductions (8 us over 512 pages, 14 over 13751), many rows by the number of
// instructions per score (1024 rows over 4064 pages and two kv heads 26 us), so the scores are looked at twice only: for each thread's
// largest, of which the need-th largest is a lower bound of the row's (`low`), and for those not
// clearly below it, which go to a list in LDS (a few more than are needed); t, the choice and the
// near pages come from the list. Where more pass than the list holds (budgets of over about half
// its length, many equal pages) the same steps go over all scores.
template <int D, int NT, bool CACHED>
__global__ void __launch_bounds__(NT, NT == 256 ? 8 : 2) pick_kernel(SelectArgs a) {
  constexpr int BINS = 4 * NT, WAVES = NT / 64, LIST = NT == 256 ? 512 : 1024;   // scores the choice is made from
  extern __shared__ uint64_t masks[];   // [words] chosen pages, [words] equal ones
  // a histogram, then the near pages' keys and numbers
  __shared__ uint64_t lists[BINS / 2 > PICK_NEAR * 3 / 2 ? BINS / 2 : PICK_NEAR * 3 / 2];
  uint32_t* hist = (uint32_t*)lists;
  uint64_t* near_key = lists;
  uint32_t* near_page = (uint32_t*)(lists + PICK_NEAR);
  __shared__ __attribute__((aligned(16))) float top_score[LIST];
  __shared__ uint32_t top_page[LIST];
  __shared__ double pn[2 * D];
  __shared__ uint32_t red[4][WAVES];
  __shared__ float member[64];
  __shared__ uint32_t sh[8];            // 0: members, 1: bin, 2: above the bin, 3: in the bin, 4: near, 5: chosen, 6: listed
  __shared__ uint64_t sh_prefix;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id();
  const uint32_t item = blockIdx.x;     // (request, kv head, row)
  const int row = (int)(item % (uint32_t)a.rows);
  const int h = (int)(item / (uint32_t)a.rows % (uint32_t)a.Hkv);
  const int b = (int)(item / (uint32_t)a.rows / (uint32_t)a.Hkv);
  const int64_t m = (int64_t)b * a.T + a.row0 + row;
  int32_t* out = a.pages + (m * a.Hkv + h) * a.budget;
  const int n = (int)pages_seen(a.positions[m], a.table_stride);
  if (n <= a.budget) {
    for (int i = tid; i < a.budget; i += NT) out[i] = i < n ? i : -1;
    return;
  }
  const int first = a.sink, end = n - a.recent;   // candidates; n > budget >= sink + recent
  const uint32_t need0 = (uint32_t)(a.budget - a.sink - a.recent);
  const float* sc = a.scores + (int64_t)item * a.width;
  const int words = (n + 63) / 64;
  uint64_t* equal = masks + words;
  uint32_t* rank = hist;                // pages chosen before a word's, at the end
  const float inf = __builtin_huge_valf();

  float key[CACHED ? PICK_KEYS : 1];
  float e = 0.f;
  if (need0 > 0) {
    if constexpr (CACHED) {
#pragma unroll
      for (int j = 0; j < PICK_KEYS; ++j) key[j] = sc[j * NT + tid < end ? j * NT + tid : end - 1];
    }
    const float* er = a.errors + (int64_t)item * (a.width / 16);
    for (int i = tid; i < (n + 15) / 16; i += NT) e = fmaxf(e, er[i]);
  }
  // P and N in 64 bits, for the pages that are summed again
  for (int d = tid; d < D; d += NT) {
    double p = 0.0, q = 0.0;
    const uint16_t* qp = a.q + (m * a.Hq + (int64_t)h * a.G) * D + d;
#pragma unroll 8
    for (int g = 0; g < a.G; ++g) {
      const float f = bf16_to_f32(qp[(int64_t)g * D]);
      p += (double)pos_part(f);
      q += (double)neg_part(f);
    }
    pn[d] = q;
    pn[D + d] = p;
  }
  // the chosen pages as a bit each, first the ones that always are
  for (int w = tid; w < words; w += NT) {
    const int p0 = w * 64;
    auto below = [&](int x) { return x <= p0 ? 0ull : x - p0 >= 64 ? ~0ull : (1ull << (x - p0)) - 1; };
    masks[w] = below(first) | (below(n) & ~below(end));
  }
  for (int i = tid; i < BINS; i += NT) hist[i] = 0;
  if (tid < 8) sh[tid] = 0;
  if constexpr (CACHED) {
    if (need0 > 0) {
#pragma unroll
      for (int j = 0; j < PICK_KEYS; ++j)
        if (j * NT + tid < first || j * NT + tid >= end) key[j] = -inf;
    }
  }
  // f(page, score) over the row's candidates, from memory or (others then come as -inf) registers
  auto over_row = [&](auto f) {
    for (int i = first + tid; i < end; i += NT) f(i, sc[i]);
  };
  auto over_all = [&](auto f) {
    if constexpr (CACHED) {
#pragma unroll
      for (int j = 0; j < PICK_KEYS; ++j) f(j * NT + tid, key[j]);
    } else {
      over_row(f);
    }
  };
  // largest and smallest of the threads' hi and lo, and the sum of their counts
  auto reduce = [&](float& hi, float& lo, uint32_t& count) {
    const uint32_t wh = wave_max_u32_all(ord_key(hi)), wl = wave_max_u32_all(~ord_key(lo)),
                   wc = wave_sum_u32_dpp(count);
    __syncthreads();
    if (lane == 0) red[1][wave] = wh, red[2][wave] = wl, red[3][wave] = wc;
    __syncthreads();
    const int w = lane % WAVES;
    hi = ord_key_to_float(wave_max_u32_all(red[1][w]));
    lo = ord_key_to_float(~wave_max_u32_all(red[2][w]));
    count = wave_sum_u32_dpp(lane < WAVES ? red[3][w] : 0u);
  };
  auto bin_of = [&](float s, float lo, float inv) {
    const float x = (s - lo) * inv;
    return x >= (float)(BINS - 1) ? BINS - 1 : x > 0.f ? (int)x : 0;
  };
  // histogram (cleared before) -> the bin of the k-th largest: sh[1]; scores above it, of all that
  // were counted and `above` more: sh[2]; in it: sh[3]. A barrier after it.
  auto find_bin = [&](uint32_t k, uint32_t above) {
    __syncthreads();
    const int top = BINS - 1 - 4 * tid;   // thread: four bins, from the top
    uint32_t c[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += c[i] = hist[top - i];
    uint32_t before = wave_incl_sum_u32(sum);
    if (lane == 63) red[0][wave] = before;
    before -= sum;
    __syncthreads();
    before += above + wave_sum_u32_dpp(lane < wave ? red[0][lane % WAVES] : 0u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (before < k && before + c[i] >= k) sh[1] = (uint32_t)(top - i), sh[2] = before, sh[3] = c[i];
      before += c[i];
    }
    __syncthreads();
  };
  // the k-th largest score that `scan` passes over, all of it in [lo, hi]: histograms, ever narrower,
  // until 64 scores are left. False: not found in 32 of them.
  auto kth = [&](auto scan, float hi, float lo, uint32_t k, float& t) {
    uint32_t above = 0;                 // scores > hi
    for (int round = 0; round < 32; ++round) {
      t = lo;
      if (lo == hi) return true;
      const float inv = (float)(BINS - 1) / (hi - lo);
      __syncthreads();
      for (int i = tid; i < BINS; i += NT) hist[i] = 0;
      if (tid == 0) sh[0] = 0;
      __syncthreads();
      scan([&](int i, float s) {
        if (s >= lo && s <= hi) atomicAdd(&hist[bin_of(s, lo, inv)], 1u);
      });
      find_bin(k, above);
      const int at = (int)sh[1];
      const uint32_t count = sh[3];
      above = sh[2];
      if (count <= 64) {
        scan([&](int i, float s) {
          if (s >= lo && s <= hi && bin_of(s, lo, inv) == at) member[atomicAdd(&sh[0], 1u)] = s;
        });
        __syncthreads();
        const float mine = lane < (int)count ? member[lane] : -inf;
        uint32_t over = 0, same = 0;
        for (int i = 0; i < (int)count; ++i) {
          over += member[i] > mine;
          same += member[i] == mine;
        }
        const uint32_t r = k - above;   // 1 .. count
        const uint64_t is = __ballot(lane < (int)count && over < r && over + same >= r);
        t = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(mine), __builtin_ctzll(is)));
        return true;
      }
      float nh = -inf, nl = inf;
      uint32_t none = 0;
      scan([&](int i, float s) {
        if (s >= lo && s <= hi && bin_of(s, lo, inv) == at) nh = fmaxf(nh, s), nl = fminf(nl, s);
      });
      reduce(nh, nl, none);
      hi = nh;
      lo = nl;
    }
    return false;
  };
  // marks the pages above t + 2 E, lists those within 2 E of t
  auto classify = [&](auto scan, float t) {
    const float over = t + 2.f * e, under = t - 2.f * e;
    scan([&](int i, float s) {
      if (s >= under) {
        if (s > over) {
          atomicOr((unsigned long long*)&masks[i / 64], 1ull << (i & 63));
          atomicAdd(&sh[5], 1u);
        } else {
          const uint32_t to = atomicAdd(&sh[4], 1u);
          if (to < PICK_NEAR) near_page[to] = (uint32_t)i;
        }
      }
    });
    __syncthreads();
  };

  bool all = false;                     // all candidates summed in 64 bits
  if (need0 > 0) {
    float most = -inf;                  // of this thread
    over_all([&](int i, float s) { most = fmaxf(most, s); });
    uint32_t pages = 0;                 // candidates that are pages, where that may be too few
    e = __uint_as_float(wave_max_u32_all(__float_as_uint(e)));
    if (lane == 0) red[0][wave] = __float_as_uint(e);
    float hi = most, lo = most > -inf ? most : inf;
    uint32_t maxima = most > -inf;
    reduce(hi, lo, maxima);
    e = __uint_as_float(wave_max_u32_all(red[0][lane % WAVES]));
    all = !(e < inf && hi < inf && maxima > 0);
    if (!all) {
      float low = -inf;                 // at least need0 scores are not below it
      if (maxima >= need0) {
        const float inv = hi > lo ? (float)(BINS - 1) / (hi - lo) : 0.f;
        const int bin = bin_of(most, lo, inv);
        if (most > -inf) atomicAdd(&hist[bin], 1u);
        find_bin(need0, 0);
        float ignore = -inf;
        uint32_t none = 0;
        low = most > -inf && bin >= (int)sh[1] ? most : inf;
        reduce(ignore, low, none);
      }
      const float from = low - 2.f * e;
      over_all([&](int i, float s) {
        if (s >= from && s > -inf) {
          const uint32_t to = atomicAdd(&sh[6], 1u);
          if (to < LIST) top_score[to] = s, top_page[to] = (uint32_t)i;
        }
      });
      __syncthreads();
      const uint32_t listed = sh[6];
      float t;
      if (listed < need0) {             // fewer pages than are needed
        all = true;
      } else if (listed <= LIST) {
        if (listed <= 256) {            // few: each against all
          for (uint32_t i = listed + tid; i < (listed + 3) / 4 * 4; i += NT) top_score[i] = -inf;
          __syncthreads();
          if (tid < (int)listed) {
            const float mine = top_score[tid];
            uint32_t over = 0, same = 0;
            for (uint32_t i = 0; i < listed; i += 4) {
              const floatx4 x = *(const floatx4*)(top_score + i);
#pragma unroll
              for (int k = 0; k < 4; ++k) over += x[k] > mine, same += x[k] == mine;
            }
            if (over < need0 && over + same >= need0) red[1][0] = __float_as_uint(mine);   // equal ones write the same
          }
          __syncthreads();
          t = __uint_as_float(red[1][0]);
        }
        auto over_list = [&](auto f) {
          for (uint32_t i = tid; i < listed; i += NT) f((int)top_page[i], top_score[i]);
        };
        if (listed > 256) {
          float l2 = inf, h2 = -inf;
          over_list([&](int i, float s) { l2 = fminf(l2, s), h2 = fmaxf(h2, s); });
          reduce(h2, l2, pages);
          all = !kth(over_list, h2, l2, need0, t);
          __syncthreads();
        }
        if (!all) classify(over_list, t);
      } else {
        float l2 = inf;
        over_row([&](int i, float s) {
          if (s > -inf) l2 = fminf(l2, s);
        });
        reduce(hi, l2, pages);
        all = !kth(over_row, hi, l2, need0, t);
        __syncthreads();
        if (!all) classify(over_row, t);
      }
    }
  }
  __syncthreads();
  uint32_t need = 0;                    // of the pages in `equal`, the lowest that many
  if (need0 > 0 && !all) {
    const uint32_t near = sh[4], left = need0 - sh[5];   // of the near ones, `left` are chosen
    if (near > PICK_NEAR) {
      all = true;
    } else {
      if (near > left) {
        for (uint32_t i = wave; i < near; i += WAVES) {
          const uint64_t k = exact_key<D, true>(a, pn, m, b, h, near_page[i]);
          if (lane == 0) near_key[i] = k;
        }
        __syncthreads();
      }
      for (uint32_t i = tid; i < near; i += NT) {
        const uint32_t pg = near_page[i];
        uint32_t ahead = 0;
        if (near > left) {
          const uint64_t k = near_key[i];
          for (uint32_t j = 0; j < near; ++j) ahead += near_key[j] > k || (near_key[j] == k && near_page[j] < pg);
        }
        if (ahead < left) atomicOr((unsigned long long*)&masks[pg / 64], 1ull << (pg & 63));
      }
    }
    __syncthreads();
  }
  if (all) {
    // every candidate in 64 bits, the need-th largest key by radix selection, eight bits a pass
    uint64_t* ex = a.exact + (int64_t)item * a.width;
    for (int i = first + wave; i < end; i += WAVES) {
      const uint64_t k = exact_key<D, false>(a, pn, m, b, h, i);
      if (lane == 0) ex[i] = k;
    }
    __threadfence_block();
    __syncthreads();
    uint64_t prefix = 0;
    need = need0;
    for (int shift = 56; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += NT) hist[i] = 0;
      __syncthreads();
      for (int i = first + tid; i < end; i += NT) {
        const uint64_t k = ex[i];
        if (shift == 56 || (k >> (shift + 8)) == (prefix >> (shift + 8)))
          atomicAdd(&hist[(k >> shift) & 255], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        uint32_t seen = 0;
        int d = 255;
        while (d > 0 && seen + hist[d] < need) seen += hist[d--];
        sh_prefix = prefix | (uint64_t)d << shift;
        sh[2] = need - seen;
      }
      __syncthreads();
      prefix = sh_prefix;
      need = sh[2];
      __syncthreads();
    }
    for (int i = tid; i < words * 64; i += NT) {
      const bool mid = i >= first && i < end;
      const uint64_t k = mid ? ex[i] : 0;
      const uint64_t mo = __ballot(i < n && (!mid || k > prefix)), me = __ballot(mid && k == prefix);
      if (lane == 0) masks[i / 64] = mo, equal[i / 64] = me;
    }
    __syncthreads();
    // of equal pages the lowest `need`
    if (wave == 0) {
      uint32_t before = 0;
      for (int w0 = 0; w0 < words; w0 += 64) {
        const int w = w0 + lane;
        uint64_t mo = w < words ? masks[w] : 0, me = w < words ? equal[w] : 0;
        const uint32_t ec = (uint32_t)__popcll(me);
        const uint32_t ei = wave_incl_sum_u32(ec);
        const uint32_t eb = before + ei - ec;
        uint32_t take = eb >= need ? 0u : need - eb < ec ? need - eb : ec;
        while (take > 0) {   // the lowest `take` set bits
          const uint64_t bit = me & (~me + 1);
          mo |= bit;
          me ^= bit;
          --take;
        }
        before += (uint32_t)__builtin_amdgcn_readlane((int)ei, 63);
        if (w < words) masks[w] = mo;
      }
    }
    __syncthreads();
  }
  // ranks of the words' first pages
  uint32_t before = 0;
  for (int w0 = 0; w0 < words; w0 += NT) {
    const int w = w0 + tid;
    const uint32_t cnt = w < words ? (uint32_t)__popcll(masks[w]) : 0u;
    const uint32_t ci = wave_incl_sum_u32(cnt);
    __syncthreads();
    if (lane == 63) red[0][wave] = ci;
    __syncthreads();
    // every lane takes part in the sums, also those past the last word
    const uint32_t t0 = lane < WAVES ? red[0][lane] : 0u;
    const uint32_t earlier = wave_sum_u32_dpp(lane < wave ? t0 : 0u);
    if (w < words) rank[w] = before + earlier + ci - cnt;
    before += wave_sum_u32_dpp(t0);
  }
  __syncthreads();
  for (int w = wave; w < words; w += WAVES) {
    const uint64_t mo = masks[w];
    if (mo >> lane & 1) {
      const uint32_t at = rank[w] + (uint32_t)__popcll(mo & ((1ull << lane) - 1));
      if (at < (uint32_t)a.budget) out[at] = w * 64 + lane;
    }
  }
}

// ---------------------------------------------------------------------------------------
// attend
// ---------------------------------------------------------------------------------------
struct AttendArgs {
  const uint16_t* q;        // [rows, Hq, D]
  const uint16_t* k_pool;
  const uint16_t* v_pool;
  uint16_t* out;            // [rows, Hq, D]
  const int32_t* table;
  const int32_t* positions;
  const int32_t* pages;     // [rows, Hkv, budget]
  float* part_o;            // [rows * Hq, splits, D]
  float* part_ml;           // [rows * Hq, splits, 2]
  int64_t table_stride, blocks, items;
  int T, Hq, Hkv, G, GT, budget, splits;
  int rpt, ring_bytes, union_most;   // attend_rows_kernel: rows of a wave, LDS in front of the union, its entries
  float qk_scale;           // softmax scale * log2(e)
};

constexpr int ATT_WAVES = 4;

// Keys of a page that a row at `pos` sees, PAGE of a whole one; the page is not past the row's position.
// pos may be 2^31 - 1, so the one is added last.
__device__ __forceinline__ int keys_seen(int pos, int page) {
  const int before = pos - page * PAGE;
  return (before < PAGE - 1 ? before : PAGE - 1) + 1;
}

// The V^T operands of elements d and d + 1 over two pages' keys, from a 16-byte load of each page
// (d's four keys, then d + 1's): the middle pairs change places.
__device__ __forceinline__ void v_operands(u32x4 a, u32x4 b, bf16x8& f0, bf16x8& f1) {
  uint32_t a2 = a[2], a3 = a[3], b0 = b[0], b1 = b[1];
  asm("v_swap_b32 %0, %1" : "+v"(a2), "+v"(b0));
  asm("v_swap_b32 %0, %1" : "+v"(a3), "+v"(b1));
  f0 = __builtin_bit_cast(bf16x8, u32x4{a[0], a[1], a2, a3});
  f1 = __builtin_bit_cast(bf16x8, u32x4{b0, b1, b[2], b[3]});
}

// One step of the running softmax over a wave's 32 keys: exponents e (lane (head col, g): keys 4 g ..
// of two pages, masked ones -inf) to weights 2^(e - m), as a bf16 pair hi + lo (16 bits of
// mantissa: hi is the upper half of the word below the weight's, lo what is left, rounded; single bf16
// weights would add about two thirds of the output's own rounding to its error). That word is one
// less so that lo is not 0 where the weight is a bf16 itself, as the largest key's 1 is: an infinite V
// times 0 would be NaN. m moves, and O and l are scaled, only where a score passes it by 2^8, for all
// of a wave's columns at once; all in 32 bits.
constexpr float RESCALE = 8.f;

template <int D>
__device__ __forceinline__ void softmax_step(const float (&e)[8], float& m, float& l,
                                             floatx4 (&acc)[D / 16], uint32_t (&hi)[4], uint32_t (&lo)[4]) {
  const float inf = __builtin_huge_valf();
  float top = fmaxf(fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])), fmaxf(fmaxf(e[4], e[5]), fmaxf(e[6], e[7])));
  if (__ballot(top > m + RESCALE)) {
    const float nm = fmaxf(m, column_max(top));
    const float c = m == nm ? 1.f : __builtin_amdgcn_exp2f(m - nm);   // 0 at the first keys
    m = nm;
    l *= c;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) acc[i] *= c;
  }
  const float ref = m == -inf ? 0.f : m;
  float p[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    p[i] = __builtin_amdgcn_exp2f(e[i] - ref);
    l += p[i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = __builtin_elementwise_sub_sat(__float_as_uint(p[2 * i]), 1u);   // 0 stays 0
    const uint32_t v = __builtin_elementwise_sub_sat(__float_as_uint(p[2 * i + 1]), 1u);
    hi[i] = __builtin_amdgcn_perm(v, u, 0x07060302u);
    lo[i] = pack_bf16x2(p[2 * i] - __uint_as_float(u & 0xffff0000u), p[2 * i + 1] - __uint_as_float(v & 0xffff0000u));
  }
}

// The waves' sums meet in LDS: in rounds of D / 2 elements where they would pass 64 KiB; floats.
__host__ __device__ __forceinline__ int attend_rounds(int D, int heads) { return D == 256 && heads > 8 ? 2 : 1; }
__host__ __device__ __forceinline__ int attend_lds(int D, int heads) {
  return ATT_WAVES * heads * (D / attend_rounds(D, heads) + 4);
}

// One workgroup per (row, kv head, 16 heads of its group, split of the list), one page pair per wave
// and step. Per pair (32 keys):
//   S^T[key, head] = K . q^T       v_mfma_f32_16x16x32_bf16 over d, A = K straight from the page
//                                  (its layout is the operand's: 1 KiB per wave load)
//   O^T[d, head]  += V^T . P^T     over the 32 keys, A = V^T (a 16-byte load holds a lane's keys of
//                                  elements d and d + 1: two operands), B = P^T from S^T's registers
// so neither K, V nor P passes through LDS. Bound by the bytes of the pages where rows have their own (64
// requests of 64 pages and eight 128-wide kv heads, 270 MB in 50 us, 5.3 TB/s; their reads from HBM 263
// MB), by L2 where neighbouring rows share them (1024 rows of 64 pages and two 256-wide kv heads, 2.1 GB in
// 77 to 90 us, 25 TB/s), by a chain of loads (position, list, table, pages) where there are few (one row of 64
// pages 6.3 us).
// By four waves, whose threads are tid; `write`: or the result is dropped.
template <int D>
__device__ __forceinline__ void attend_row(const AttendArgs& a, int b, int h, int gt, int t, int split,
                                           int tid, int wave, bool write, float* so, float (*sml)[16][2]) {
  constexpr int KS = D / 32, NW = ATT_WAVES;
  const int lane = tid & 63, col = lane & 15, g = lane >> 4;
  const int64_t m = (int64_t)b * a.T + t;
  const int heads = a.G - gt * 16 < 16 ? a.G - gt * 16 : 16;
  const int64_t head0 = (int64_t)h * a.G + gt * 16;
  const int pos = a.positions[m];
  const int32_t* list = a.pages + (m * a.Hkv + h) * a.budget;

  bf16x8 qf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    u32x4 x = {0u, 0u, 0u, 0u};
    if (col < heads) x = *(const u32x4*)(a.q + (m * a.Hq + head0 + col) * D + 32 * s + 8 * g);
    qf[s] = __builtin_bit_cast(bf16x8, x);
  }
  floatx4 acc[D / 16];
#pragma unroll
  for (int i = 0; i < D / 16; ++i) acc[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  float mx = -__builtin_huge_valf(), l = 0.f;

  const int parts = a.splits * NW, part = split * NW + wave;
  const int64_t page_elems = (int64_t)PAGE * D;
  for (int e0 = part; e0 < a.budget; e0 += 64 * parts) {
    const int64_t e = e0 + (int64_t)lane * parts;
    int pg = e < a.budget ? list[e] : -1;
    int blk = pg >= 0 && pg <= pos / PAGE && pos >= 0
                  ? page_block(a.table, a.table_stride, b, pg, a.blocks) : -1;
    uint64_t todo = __ballot(blk >= 0);
    while (todo) {
      const int ia = __builtin_ctzll(todo);
      todo &= todo - 1;
      const bool two = todo != 0;
      const int ib = two ? __builtin_ctzll(todo) : ia;
      if (two) todo &= todo - 1;
      const int ba = __builtin_amdgcn_readlane(blk, ia), bb = __builtin_amdgcn_readlane(blk, ib);
      const int left_a = keys_seen(pos, __builtin_amdgcn_readlane(pg, ia));
      const int left_b = two ? keys_seen(pos, __builtin_amdgcn_readlane(pg, ib)) : 0;
      const int64_t offa = ((int64_t)ba * a.Hkv + h) * page_elems, offb = ((int64_t)bb * a.Hkv + h) * page_elems;
      // K: lane (key col, g) holds d = 32 s + 8 g .. of its key
      const uint16_t* ka = a.k_pool + offa + (g >> 1) * 256 + col * 16 + (g & 1) * 8;
      const uint16_t* kb = a.k_pool + offb + (g >> 1) * 256 + col * 16 + (g & 1) * 8;
      floatx4 sa = {0.f, 0.f, 0.f, 0.f}, sb = {0.f, 0.f, 0.f, 0.f};
      u32x4 xa[KS], xb[KS];
#pragma unroll
      for (int s = 0; s < KS; ++s) xa[s] = *(const u32x4*)(ka + 512 * s);
#pragma unroll
      for (int s = 0; s < KS; ++s) xb[s] = *(const u32x4*)(kb + 512 * s);
      // V: lane (col, g) holds keys 4 g .. 4 g + 3 of d = 32 j + 2 col and of the next
      const uint16_t* va = a.v_pool + offa + (g * D + 2 * col) * 4;
      const uint16_t* vb = a.v_pool + offb + (g * D + 2 * col) * 4;
      u32x4 ya[KS], yb[KS];
#pragma unroll
      for (int j = 0; j < KS; ++j) ya[j] = *(const u32x4*)(va + 128 * j);
#pragma unroll
      for (int j = 0; j < KS; ++j) yb[j] = *(const u32x4*)(vb + 128 * j);
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        sa = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, xa[s]), qf[s], sa, 0, 0, 0);
        sb = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, xb[s]), qf[s], sb, 0, 0, 0);
      }
      // lane (head col, g): keys 4 g + r of both pages
      float x[8];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[r] = 4 * g + r < left_a ? sa[r] * a.qk_scale : -__builtin_huge_valf();
        x[4 + r] = 4 * g + r < left_b ? sb[r] * a.qk_scale : -__builtin_huge_valf();
      }
      uint32_t ph[4], pl[4];
      softmax_step<D>(x, mx, l, acc, ph, pl);
      const bf16x8 hi = __builtin_bit_cast(bf16x8, u32x4{ph[0], ph[1], ph[2], ph[3]});
      const bf16x8 lo = __builtin_bit_cast(bf16x8, u32x4{pl[0], pl[1], pl[2], pl[3]});
      // what lies behind the row's last position never enters: 0 . NaN would
      if (left_a < PAGE || left_b < PAGE) {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const int t0 = 4 * g + 2 * w;
          const uint32_t ma = t0 + 1 < left_a ? 0xffffffffu : t0 < left_a ? 0xffffu : 0u;
          const uint32_t mb = t0 + 1 < left_b ? 0xffffffffu : t0 < left_b ? 0xffffu : 0u;
#pragma unroll
          for (int j = 0; j < KS; ++j) {
            ya[j][w] &= ma;
            ya[j][2 + w] &= ma;
            yb[j][w] &= mb;
            yb[j][2 + w] &= mb;
          }
        }
      }
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        bf16x8 f0, f1;
        v_operands(ya[j], yb[j], f0, f1);
        acc[2 * j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f0, hi, acc[2 * j], 0, 0, 0);
        acc[2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f1, hi, acc[2 * j + 1], 0, 0, 0);
        acc[2 * j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f0, lo, acc[2 * j], 0, 0, 0);
        acc[2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f1, lo, acc[2 * j + 1], 0, 0, 0);
      }
    }
  }
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  // join the waves: each scales its sums to the common maximum
  if (g == 0) sml[wave][col][0] = mx, sml[wave][col][1] = l;
  __syncthreads();
  float top = sml[0][col][0];
#pragma unroll
  for (int w = 1; w < NW; ++w) top = fmaxf(top, sml[w][col][0]);
  const float c = mx == top ? 1.f : __builtin_amdgcn_exp2f(mx - top);
  const int rounds = attend_rounds(D, heads), DR = D / rounds, ld = DR + 4;
  for (int rd = 0; rd < rounds; ++rd) {
    if (rd) __syncthreads();
    if (col < heads) {
      float* o = so + (wave * heads + col) * ld + 8 * g - rd * DR;
#pragma unroll
      for (int j = 0; j < KS; ++j) {   // register r of tiles 2 j, 2 j + 1: d = 32 j + 8 g + 2 r, + 1
        if (32 * j / DR != rd) continue;
        const floatx4 e = acc[2 * j], f = acc[2 * j + 1];
        *(floatx4*)(o + 32 * j) = floatx4{e[0] * c, f[0] * c, e[1] * c, f[1] * c};
        *(floatx4*)(o + 32 * j + 4) = floatx4{e[2] * c, f[2] * c, e[3] * c, f[3] * c};
      }
    }
    __syncthreads();
    for (int u = write ? tid : heads * (DR / 4); u < heads * (DR / 4); u += 64 * NW) {
      const int hd = u / (DR / 4), dr = u % (DR / 4) * 4, d = rd * DR + dr;
      float hm = sml[0][hd][0];
#pragma unroll
      for (int w = 1; w < NW; ++w) hm = fmaxf(hm, sml[w][hd][0]);
      float sum = 0.f;
      floatx4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float wm = sml[w][hd][0];
        sum += sml[w][hd][1] * (wm == hm ? 1.f : __builtin_amdgcn_exp2f(wm - hm));
        o += *(const floatx4*)(so + (w * heads + hd) * ld + dr);
      }
      const int64_t row = m * a.Hq + head0 + hd;
      if (a.splits == 1) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;   // nothing seen: zeros
        uint2 y;
        y.x = pack_bf16x2(o[0] * inv, o[1] * inv);
        y.y = pack_bf16x2(o[2] * inv, o[3] * inv);
        *(uint2*)(a.out + row * D + d) = y;
      } else {
        *(floatx4*)(a.part_o + (row * a.splits + split) * D + d) = o;
        if (d == 0) {
          a.part_ml[(row * a.splits + split) * 2] = hm;
          a.part_ml[(row * a.splits + split) * 2 + 1] = sum;
        }
      }
    }
  }
}

template <int D>
__global__ void __launch_bounds__(64 * ATT_WAVES, 2) attend_kernel(AttendArgs a) {
  extern __shared__ float so[];   // [waves][heads][elements of a round + 4]
  __shared__ float sml[ATT_WAVES][16][2];
  // neighbouring rows, which list many of the same pages, run on one XCD
  const uint32_t per_xcd = gridDim.x / 8;
  uint32_t item = blockIdx.x % 8 * per_xcd + blockIdx.x / 8;
  if (item >= (uint64_t)a.items) return;
  const int split = (int)(item % (uint32_t)a.splits);
  item /= (uint32_t)a.splits;
  const int t = (int)(item % (uint32_t)a.T);
  item /= (uint32_t)a.T;
  const int gt = (int)(item % (uint32_t)a.GT);
  item /= (uint32_t)a.GT;
  attend_row<D>(a, (int)(item / (uint32_t)a.Hkv), (int)(item % (uint32_t)a.Hkv), gt, t, split, threadIdx.x,
                wave_id(), true, so, sml);
}

// Many rows: neighbouring rows of a request list many of the same pages. A workgroup takes R = 4 rpt
// rows of one kv head (rpt rows fill the 16 columns of a matrix instruction) and goes once over the
// union of their lists, each page with the set of rows that list it: the pages stream through LDS
// (global_load_lds, 1 KiB per wave instruction), two pairs in use and the next two on their way. Four
// waves, one for each rpt rows, multiply the first pair of a step and four the second, with the columns
// of rows that do not list a page masked; the two halves are joined at the end. A page that not all
// rows see whole is entered once for each row. Two waves a SIMD, so that one's softmax and LDS reads
// run beside the other's products: with one (the same step with four waves) 81 us for 1024 rows of 64
// pages and two 256-wide kv heads instead of 62. Of these, a step's products, softmax and LDS reads alone
// take 37 us and its loads alone 29 (13 TB/s from L2).
// Time grows with the union where the per-row form's does not: those 1024 rows take 44 us where all
// lists are one, 64 with 1.8 lists' pages in a union of eight rows, 86 with 2.6, 121 with 3.9, and row
// by row 77 to 90. A workgroup whose union is past union_most therefore computes its rows alone, two
// at a time (92 to 97 us). Lists that the choice gives have little in common where the queries have: of
// independent ones 5.7 lists' pages in eight rows (136 us, 140 in two calls that go row by row), of
// queries correlated 0.5 4.1 (133 and 117), 0.9 2.1 (104 and 101), 0.97 1.6 (73 and 97).
// What is masked in a row's column is multiplied by a weight of zero, so a V that is not finite in a
// page of another row would reach it as NaN: rows whose result is not finite are computed again alone,
// as are those of a workgroup with a list in which a page stands twice.
constexpr int ROWS_MAX = 16, ROWS_GROUPS = 4, ROWS_WAVES = 8;
constexpr int ROWS_ENTRIES = 4;               // of the rows' lists, that a thread holds
constexpr int ROWS_LDS = 160 * 1024 - 2048;   // dynamic LDS at most

// LDS image of one (page, kv head): K, then V, as they are in memory (a lane's 16 bytes of either
// operand are next to its neighbours': no two lanes that are served together share a bank).
template <int D>
struct PageImage {
  static constexpr int HALF = PAGE * D * 2, GROUP = D * 8, BYTES = 2 * HALF, CHUNKS = BYTES / 1024;
};

template <int D>
__global__ void __launch_bounds__(64 * ROWS_WAVES, 2) attend_rows_kernel(AttendArgs a) {
  typedef __attribute__((address_space(3))) void lds_void;
  using Image = PageImage<D>;
  static_assert(Image::CHUNKS % ROWS_WAVES == 0, "a load of all waves is of one page");
  constexpr int KS = D / 32, NT = 64 * ROWS_WAVES, CPW = 4 * Image::CHUNKS / ROWS_WAVES;   // loads of a wave per step
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];   // two steps' pages (first the rows of every page), union
  __shared__ float sml[ROWS_WAVES][16][2];
  __shared__ int spos[ROWS_MAX];
  __shared__ uint32_t counts[ROWS_WAVES];
  __shared__ uint32_t again, twice;   // rows to compute alone; a list names a page twice
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_id(), col = lane & 15, g = lane >> 4;
  const uint32_t per_xcd = gridDim.x / 8;
  uint32_t item = blockIdx.x % 8 * per_xcd + blockIdx.x / 8;
  if (item >= (uint64_t)a.items) return;
  const int rpt = a.rpt, R = ROWS_GROUPS * rpt, K = a.budget;
  const uint32_t groups = (uint32_t)(a.T + R - 1) / R;
  const int t0 = (int)(item % groups) * R;
  item /= groups;
  const int h = (int)(item % (uint32_t)a.Hkv), b = (int)(item / (uint32_t)a.Hkv);
  const int64_t m0 = (int64_t)b * a.T + t0;
  const int live = a.T - t0 < R ? a.T - t0 : R;
  uint32_t* page_rows = (uint32_t*)lds;         // 16 bits a page
  uint2* merged = (uint2*)(lds + a.ring_bytes); // the union: block, page << 16 | rows
  if (tid < ROWS_MAX) spos[tid] = tid < live ? a.positions[m0 + tid] : -1;
  if (tid == 0) again = twice = 0;
  // this wave's queries: column col is head col % G of row wave * rpt + col / G
  const int rg = wave % ROWS_GROUPS, half = wave / ROWS_GROUPS;
  const int row = col < rpt * a.G ? rg * rpt + col / a.G : ROWS_MAX;
  bf16x8 qf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    u32x4 x = {0u, 0u, 0u, 0u};
    if (row < live) x = *(const u32x4*)(a.q + ((m0 + row) * a.Hq + (int64_t)h * a.G + col % a.G) * D + 32 * s + 8 * g);
    qf[s] = __builtin_bit_cast(bf16x8, x);
  }
  const int32_t* lists = a.pages + (m0 * a.Hkv + h) * K;
  const int64_t list_step = (int64_t)a.Hkv * K;
  const int entries = live * K;
  __syncthreads();
  int low = 0x7fffffff;
  for (int r = 0; r < live; ++r) low = spos[r] >= 0 && spos[r] < low ? spos[r] : low;
  auto whole = [&](int p) { return p * PAGE + PAGE - 1 <= low; };
  // this thread's entries of the lists: pages, or -1
  int page[ROWS_ENTRIES], from[ROWS_ENTRIES];
#pragma unroll
  for (int i = 0; i < ROWS_ENTRIES; ++i) {
    const int e = i * NT + tid, r = e < entries ? e / K : 0;
    from[i] = r;
    page[i] = e < entries ? lists[r * list_step + e % K] : -1;
  }
#pragma unroll
  for (int i = 0; i < ROWS_ENTRIES; ++i) {
    const int p = page[i], seen = spos[from[i]];
    if (!(p >= 0 && seen >= 0 && p <= seen / PAGE && p < a.table_stride)) page[i] = -1;
    if (page[i] >= 0) page_rows[p >> 1] = 0;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < ROWS_ENTRIES; ++i)
    if (page[i] >= 0) {
      const uint32_t bit = 1u << (from[i] + (page[i] & 1) * 16);
      if (atomicOr(&page_rows[page[i] >> 1], bit) & bit) twice = 1;
    }
  __syncthreads();
  bool merge = twice == 0;
  uint32_t total = 0;
  if (merge) {
#pragma unroll
    for (int i = 0; i < ROWS_ENTRIES; ++i) {
      if (i * NT >= entries) break;
      int blk = -1;
      uint32_t rows = 0;
      if (page[i] >= 0) {
        rows = whole(page[i]) ? page_rows[page[i] >> 1] >> (page[i] & 1) * 16 & 0xffffu : 1u << from[i];
        if (__builtin_ctz(rows) == from[i]) blk = page_block(a.table, a.table_stride, b, page[i], a.blocks);
      }
      const uint64_t have = __ballot(blk >= 0);
      if (lane == 0) counts[wave] = (uint32_t)__popcll(have);
      __syncthreads();
      uint32_t at = total + (uint32_t)__popcll(have & ((1ull << lane) - 1));
      for (int w = 0; w < ROWS_WAVES; ++w) {
        if (w < wave) at += counts[w];
        total += counts[w];
      }
      if (blk >= 0) merged[at] = uint2{(uint32_t)blk, (uint32_t)page[i] << 16 | rows};
      __syncthreads();
    }
    if (total > (uint32_t)a.union_most) merge = false, total = 0;
  }

  floatx4 acc[D / 16];
#pragma unroll
  for (int i = 0; i < D / 16; ++i) acc[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  float mx = -__builtin_huge_valf(), l = 0.f;
  const int pos = row < live ? spos[row] : -1;
  const uint32_t mine = ((1u << rpt) - 1) << (rg * rpt);   // the wave's rows
  const uint32_t pairs = (total + 1) / 2;
  const uint32_t steps = (pairs + 1) / 2;
  // The four pages of step j into its half of the ring, the last pair again past the end.
  auto fetch = [&](uint32_t j) {
    uint8_t* to = lds + (j & 1) * (4 * Image::BYTES);
    int64_t base[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t e = 4 * j + i;
      e = e < total ? e : total - 1;
      base[i] = ((int64_t)__builtin_amdgcn_readfirstlane((int)merged[e].x) * a.Hkv + h) * Image::HALF;
    }
#pragma unroll
    for (int i = 0; i < CPW; ++i) {
      const int c = i * ROWS_WAVES + wave, cc = c % Image::CHUNKS;
      const int64_t from = base[i * ROWS_WAVES / Image::CHUNKS];
      const bool is_v = cc >= Image::CHUNKS / 2;
      const int off = (is_v ? cc - Image::CHUNKS / 2 : cc) * 1024;
      const uint8_t* src = (const uint8_t*)(is_v ? a.v_pool : a.k_pool) + from + off + lane * 16;
      __builtin_amdgcn_global_load_lds((const void*)src, (lds_void*)(to + c * 1024), 16, 0, 0);
    }
  };
  const uint32_t k_at = (g >> 1) * 512 + col * 32 + (g & 1) * 16, v_at = Image::HALF + g * Image::GROUP + col * 16;
  if (pairs) fetch(0);
  for (uint32_t j = 0; j < steps; ++j) {
    // this step's pages have landed, for every wave, and every wave is done with the last step's
    wait_vmcnt<0>();
    wait_lgkmcnt0();
    block_barrier();
    if (j + 1 < steps) fetch(j + 1);
    const uint32_t e = 4 * j + 2 * half;
    if (e >= total) continue;
    const bool two = e + 1 < total;
    const uint32_t info_a = (uint32_t)__builtin_amdgcn_readfirstlane((int)merged[e].y);
    const uint32_t info_b = two ? (uint32_t)__builtin_amdgcn_readfirstlane((int)merged[e + 1].y) : 0u;
    const uint32_t rows_a = info_a & 0xffffu, rows_b = info_b & 0xffffu;
    if (!((rows_a | rows_b) & mine)) continue;   // by none of the wave's rows
    const int page_a = (int)(info_a >> 16), page_b = (int)(info_b >> 16);
    // a page that one row sees in part: what lies behind its last position never enters
    int end_a = PAGE, end_b = two ? PAGE : 0;
    if (!whole(page_a)) end_a = keys_seen(__builtin_amdgcn_readfirstlane(spos[__builtin_ctz(rows_a)]), page_a);
    if (two && !whole(page_b)) end_b = keys_seen(__builtin_amdgcn_readfirstlane(spos[__builtin_ctz(rows_b)]), page_b);
    const uint8_t* slot = lds + (j & 1) * (4 * Image::BYTES) + half * (2 * Image::BYTES);
    // all of K is asked for before the first is used, all of V before the softmax
    u32x4 ka[KS], kb[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      ka[s] = *(const u32x4*)(slot + k_at + 1024 * s);
      kb[s] = *(const u32x4*)(slot + Image::BYTES + k_at + 1024 * s);
    }
    __builtin_amdgcn_sched_barrier(0);
    floatx4 s0 = {0.f, 0.f, 0.f, 0.f}, s1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      s0 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, ka[s]), qf[s], s0, 0, 0, 0);
      s1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kb[s]), qf[s], s1, 0, 0, 0);
    }
    u32x4 va[KS], vb[KS];   // keys 4 g .. 4 g + 3 of d = 32 s + 2 col and of the next
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      va[s] = *(const u32x4*)(slot + v_at + 256 * s);
      vb[s] = *(const u32x4*)(slot + Image::BYTES + v_at + 256 * s);
    }
    __builtin_amdgcn_sched_barrier(0);
    const int left_a = rows_a >> row & 1 ? keys_seen(pos, page_a) : 0;
    const int left_b = rows_b >> row & 1 ? keys_seen(pos, page_b) : 0;
    float x[8];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      x[r] = 4 * g + r < left_a ? s0[r] * a.qk_scale : -__builtin_huge_valf();
      x[4 + r] = 4 * g + r < left_b ? s1[r] * a.qk_scale : -__builtin_huge_valf();
    }
    uint32_t hi[4], lo[4];
    softmax_step<D>(x, mx, l, acc, hi, lo);
    const bf16x8 ph = __builtin_bit_cast(bf16x8, u32x4{hi[0], hi[1], hi[2], hi[3]});
    const bf16x8 pl = __builtin_bit_cast(bf16x8, u32x4{lo[0], lo[1], lo[2], lo[3]});
    if (end_a < PAGE || end_b < PAGE) {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const int k0 = 4 * g + 2 * w;
        const uint32_t ma = k0 + 1 < end_a ? 0xffffffffu : k0 < end_a ? 0xffffu : 0u;
        const uint32_t mb = k0 + 1 < end_b ? 0xffffffffu : k0 < end_b ? 0xffffu : 0u;
#pragma unroll
        for (int s = 0; s < KS; ++s) va[s][w] &= ma, va[s][2 + w] &= ma, vb[s][w] &= mb, vb[s][2 + w] &= mb;
      }
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      bf16x8 f0, f1;
      v_operands(va[s], vb[s], f0, f1);
      acc[2 * s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f0, ph, acc[2 * s], 0, 0, 0);
      acc[2 * s + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f1, ph, acc[2 * s + 1], 0, 0, 0);
      acc[2 * s] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f0, pl, acc[2 * s], 0, 0, 0);
      acc[2 * s + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f1, pl, acc[2 * s + 1], 0, 0, 0);
    }
  }
  // join the halves: the second leaves its sums in LDS
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  __syncthreads();
  floatx4* other = (floatx4*)lds + rg * (D / 16) * 64 + lane;
  if (half) {
#pragma unroll
    for (int i = 0; i < D / 16; ++i) other[i * 64] = acc[i];
    if (g == 0) sml[rg][col][0] = mx, sml[rg][col][1] = l;
  }
  __syncthreads();
  if (!half && merge && row < live) {
    const float m2 = sml[rg][col][0], top = fmaxf(mx, m2);
    const float c1 = mx == top ? 1.f : __builtin_amdgcn_exp2f(mx - top);
    const float c2 = m2 == top ? 1.f : __builtin_amdgcn_exp2f(m2 - top);
    l = l * c1 + sml[rg][col][1] * c2;
    const float inv = l == 0.f ? 0.f : 1.f / l;   // nothing seen: zeros
    uint16_t* o = a.out + ((m0 + row) * a.Hq + (int64_t)h * a.G + col % a.G) * D + 8 * g;
    float sum = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {   // register r of tiles 2 s, 2 s + 1: d = 32 s + 8 g + 2 r, + 1
      const floatx4 y = (acc[2 * s] * c1 + other[2 * s * 64] * c2) * inv;
      const floatx4 z = (acc[2 * s + 1] * c1 + other[(2 * s + 1) * 64] * c2) * inv;
      u32x4 w;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        sum += __builtin_fabsf(y[r]) + __builtin_fabsf(z[r]);
        w[r] = pack_bf16x2(y[r], z[r]);
      }
      *(u32x4*)(o + 32 * s) = w;
    }
    if (!(sum < __builtin_huge_valf())) atomicOr(&again, 1u << row);
  }
  __syncthreads();
  uint32_t alone = merge ? again : (1u << live) - 1;
  while (alone) {   // two at a time, each by four waves
    const int r0 = __builtin_ctz(alone);
    alone &= alone - 1;
    const bool two = alone != 0;
    const int r1 = two ? __builtin_ctz(alone) : r0;
    alone &= alone - 1;
    __syncthreads();
    attend_row<D>(a, b, h, 0, t0 + (half ? r1 : r0), 0, tid & 255, rg, !half || two,
                  (float*)lds + half * attend_lds(D, a.G), sml + half * ATT_WAVES);
  }
}

// The splits of one (row, head) joined: D / 4 threads a head. A round trip to memory bounds it, so all
// loads of eight splits are in flight at once (2.4 us; both kernels for two lists of 48 pages of 256-wide
// heads, six splits each, 8.7 us from HBM, 9.9 with the loads as the compiler places them).
constexpr int JOIN = 8;

template <int D>
__global__ void __launch_bounds__(256, 4) attend_join_kernel(const float* __restrict__ part_o,
                                                             const float* __restrict__ part_ml,
                                                             uint16_t* __restrict__ out, int64_t rows,
                                                             int splits) {
  const int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) / (D / 4);
  const int d = threadIdx.x % (D / 4) * 4;
  if (row >= rows) return;
  const float* ml = part_ml + row * splits * 2;
  const float* po = part_o + row * splits * D + d;
  float top = -__builtin_huge_valf(), sum = 0.f;
  floatx4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < splits; s0 += JOIN) {
    // the last split again past the end, without weight
    float2 w[JOIN];
    floatx4 x[JOIN];
#pragma unroll
    for (int i = 0; i < JOIN; ++i) {
      const int s = s0 + i < splits ? s0 + i : splits - 1;
      w[i] = *(const float2*)(ml + 2 * s);
      x[i] = *(const floatx4*)(po + s * D);
    }
    __builtin_amdgcn_sched_barrier(0);   // all in flight, or the compiler takes them one by one
    float nt = top;
#pragma unroll
    for (int i = 0; i < JOIN; ++i) nt = fmaxf(nt, w[i].x);
    const float k = top == nt ? 1.f : __builtin_amdgcn_exp2f(top - nt);   // 0 at first
    top = nt;
    sum *= k;
    o *= k;
#pragma unroll
    for (int i = 0; i < JOIN; ++i) {
      const bool in = s0 + i < splits;
      const float c = w[i].x == top ? 1.f : __builtin_amdgcn_exp2f(w[i].x - top);
      sum = in ? __builtin_fmaf(w[i].y, c, sum) : sum;
      o = in ? o + x[i] * c : o;
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint2 y;
  y.x = pack_bf16x2(o[0] * inv, o[1] * inv);
  y.y = pack_bf16x2(o[2] * inv, o[3] * inv);
  *(uint2*)(out + row * D + d) = y;
}

// ---------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------
constexpr int64_t MAX_WIDTH = 1 << 17;        // pages of a request that the choice covers (2M tokens)

// More than 64 KiB of dynamic LDS has to be allowed, once per kernel and device.
hipError_t raise_lds_limit(const void* kernel, std::atomic<uint64_t>& devices, int bytes) {
  int dev = 0;
  hipError_t err = hipGetDevice(&dev);
  if (err != hipSuccess) return err;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (devices.load() & bit) return hipSuccess;
  err = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (err == hipSuccess) devices |= bit;
  return err;
}

// Splits of a list: for 256 workgroups, a page pair or more per wave, and whole rounds of the join
// (whose second starts when the first is added up). With lists from HBM: eighteen of 128 pages and
// 256-wide heads take 32 us whole, 12.9 in sixteen splits; 128 of 64 pages and 128-wide heads 19.6 whole,
// 19.0 in two, of 256 pages 60 and 53. Short lists are done before a second launch would start (of 16
// pages of 256-wide heads, from L2: 6.8 us whole, 7.7 split; of 32, from HBM: 10.3 and 9.2).
int attend_splits(int64_t items, int64_t budget) {
  if (items <= 0 || budget <= 24) return 1;
  const int64_t most = (budget + 2 * ATT_WAVES - 1) / (2 * ATT_WAVES);
  int64_t s = (256 + items - 1) / items;
  if (s > JOIN) s = (s + JOIN - 1) / JOIN * JOIN;
  return (int)(s < most ? s : most);
}

// LDS of attend_rows_kernel in front of the union: the ring, and before it two bytes a page.
int64_t rows_ring_bytes(int64_t D, int64_t pages) {
  const int64_t image = D == 128 ? PageImage<128>::BYTES : PageImage<256>::BYTES;
  return std::max(8 * image, (pages + 1) / 2 * 4);
}

// Rows of a wave where rows go over the union of their lists (attend_rows_kernel), or 0: two rows or
// more for the columns of a matrix instruction, heads that are wide enough (1024 rows of 64 pages and
// two 64-wide kv heads take 26 us row by row, 40 at best over the union; sixteen 256-wide heads a group 46
// and 41 to 93), a table (16 bits a page) and lists that fit LDS, and rows that fill the rounds of 256
// workgroups to three quarters, as a round takes as long when it is not full (1024 rows of two 256-wide
// kv heads, one round: 77 us row by row, 64 over the union; 512 rows 42 and 57).
int attend_rows_per_wave(int64_t batch, int64_t tokens, int64_t Hkv, int64_t G, int64_t D, int64_t pages,
                         int64_t budget) {
  if (D < 128 || G > 8) return 0;
  const int64_t most = ROWS_MAX / ROWS_GROUPS;
  int64_t rpt = 16 / G < most ? 16 / G : most;
  const int64_t room = ROWS_LDS - rows_ring_bytes(D, pages);
  while (rpt > 0 && (ROWS_GROUPS * rpt * budget * 8 > room ||
                     ROWS_GROUPS * rpt * budget > 64 * ROWS_WAVES * ROWS_ENTRIES))
    --rpt;
  if (rpt < 2 || pages > 65536) return 0;
  const int64_t R = ROWS_GROUPS * rpt, wgs = batch * Hkv * ((tokens + R - 1) / R);
  return 4 * batch * Hkv * tokens >= 3 * R * ((wgs + 255) / 256 * 256) ? (int)rpt : 0;
}

// The choice's workspace for some rows of every request: keys for where a row needs them all, scores,
// their errors, and, of more than sixteen rows, the operands.
struct SelectSpace {
  int64_t width, scores, errors, operands, lasts, bytes;   // pages, rounded up; offsets
};
SelectSpace select_space(int64_t batch, int64_t rows, int64_t Hkv, int64_t D, int64_t pages) {
  SelectSpace s;
  s.width = (pages + 15) / 16 * 16;
  const int64_t cells = batch * Hkv * rows * s.width, tiles = rows > 16 ? (rows + 15) / 16 : 0;
  s.scores = cells * 8;
  s.errors = s.scores + cells * 4;
  s.operands = (s.errors + cells / 4 + 255) / 256 * 256;
  s.lasts = s.operands + batch * Hkv * tiles * D * 128;
  s.bytes = s.lasts + batch * tiles * 4;
  return s;
}

// The choice's workspace holds the scores of all rows, or of a part of them: what 256 MiB hold, sixteen
// at least. It never falls where the shape grows, so that one for the largest shape serves them all.
int64_t select_bytes(int64_t batch, int64_t tokens, int64_t Hkv, int64_t D, int64_t pages) {
  const int64_t part = std::max((int64_t)256 << 20, select_space(batch, 16, Hkv, D, pages).bytes);
  return std::min(part, select_space(batch, tokens, Hkv, D, pages).bytes);
}

// Rows of a request in a part: a multiple of sixteen, or all.
int64_t select_rows(int64_t batch, int64_t tokens, int64_t Hkv, int64_t D, int64_t pages) {
  const int64_t bytes = select_bytes(batch, tokens, Hkv, D, pages);
  if (select_space(batch, tokens, Hkv, D, pages).bytes <= bytes) return tokens;
  int64_t lo = 1, hi = (tokens + 15) / 16;   // row tiles: lo fit (sixteen rows always do), hi do not
  while (hi - lo > 1) {
    const int64_t mid = lo + (hi - lo) / 2;
    (select_space(batch, mid * 16, Hkv, D, pages).bytes <= bytes ? lo : hi) = mid;
  }
  return lo * 16;
}

auto score_form(int64_t D, bool two) {
  return D == 64    ? two ? score_kernel<64, 2> : score_kernel<64, 1>
         : D == 128 ? two ? score_kernel<128, 2> : score_kernel<128, 1>
                    : two ? score_kernel<256, 2> : score_kernel<256, 1>;
}
template <int D>
auto pick_of(int64_t width) {
  return width <= 256 * PICK_KEYS    ? pick_kernel<D, 256, true>
         : width <= 1024 * PICK_KEYS ? pick_kernel<D, 1024, true>
                                     : pick_kernel<D, 1024, false>;
}
// A thread holds up to sixteen scores: four waves up to 4096 pages, sixteen above, and past 16384
// pages the scores are read again by every pass. The whole choice: 256 rows over 4096 pages and two kv
// heads 39 us with four waves, 46 with sixteen (one row the same with both); eleven rows over 13751 pages
// 25 us with the scores in registers, 29 read again.
auto pick_form(int64_t D, int64_t width) {
  return D == 64 ? pick_of<64>(width) : D == 128 ? pick_of<128>(width) : pick_of<256>(width);
}

}  // namespace

// =======================================================================================
// entry points
// =======================================================================================

SV_API int snowverify_kv_append(const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                                const void* q, int64_t q_stride, const float* cos_in,
                                const float* sin_in, int64_t cs_stride, int64_t half,
                                const void* q_gamma, const void* k_gamma, float eps, void* k_pool,
                                void* v_pool, void* bounds, void* q_out, const int32_t* table,
                                const int32_t* starts, const int32_t* counts, int64_t batch,
                                int64_t tokens, int64_t num_heads, int64_t num_kv_heads,
                                int64_t head_size, int64_t table_stride, int64_t blocks,
                                void* stream) {
  if (!head_shape_ok(batch, tokens, num_heads, num_kv_heads, head_size) || half < 0 || half % 8 ||
      2 * half > head_size || table_stride < 0 || blocks < 0 || k_stride % 8 || v_stride % 8 ||
      q_stride % 8 || (q && !q_out))
    return SV_EINVAL;
  if (batch * tokens == 0) return SV_OK;
  if (!k || !v || (blocks && (!k_pool || !v_pool)) || (table_stride && !table) || !starts ||
      !counts || (half && (!cos_in || !sin_in)))
    return SV_EINVAL;
  AppendArgs a{};
  a.k = (const uint16_t*)k;
  a.v = (const uint16_t*)v;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.cosv = cos_in;
  a.sinv = sin_in;
  a.cs_stride = cs_stride;
  a.k_gamma = (const uint16_t*)k_gamma;
  a.eps = eps;
  a.k_pool = (uint16_t*)k_pool;
  a.v_pool = (uint16_t*)v_pool;
  a.bounds = (uint16_t*)bounds;
  a.table = table;
  a.starts = starts;
  a.counts = counts;
  a.table_stride = table_stride;
  a.blocks = blocks;
  a.batch = (int)batch;
  a.T = (int)tokens;
  a.Hkv = (int)num_kv_heads;
  a.half = (int)half;
  a.rows = {(const uint16_t*)q, q_stride, (const uint16_t*)q_gamma, cos_in, sin_in, cs_stride, eps,
            (uint16_t*)q_out, starts, counts, (int)batch, (int)tokens, (int)num_heads, (int)half};
  a.pages = (int)((tokens + PAGE - 2) / PAGE + 1);
  a.page_wgs = batch * a.pages * num_kv_heads;
  const int64_t groups = (num_heads + Q_HEADS - 1) / Q_HEADS;
  const int64_t grid = a.page_wgs + (q ? (batch * tokens * groups + 15) / 16 : 0);
  if (!grid_ok(grid, 2 * head_size)) return SV_EINVAL;
  const bool by = q && queries_pass_by(batch * tokens, num_heads, head_size);
  auto kern = head_size == 64    ? by ? append_kernel<64, true> : append_kernel<64, false>
              : head_size == 128 ? by ? append_kernel<128, true> : append_kernel<128, false>
              : by               ? append_kernel<256, true> : append_kernel<256, false>;
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3((unsigned)(2 * head_size)), 0, S(stream), a);
  SV_CHECK_LAUNCH();
  return SV_OK;
}

SV_API int snowverify_page_bounds(const void* k_pool, void* bounds, const int32_t* table,
                                  const int32_t* starts, const int32_t* counts, int64_t batch,
                                  int64_t tokens, int64_t num_kv_heads, int64_t head_size,
                                  int64_t table_stride, int64_t blocks, void* stream) {
  if (batch < 0 || batch > MAX_BATCH_ROWS || tokens < 0 || tokens > 0x7fffffff || num_kv_heads <= 0 ||
      num_kv_heads > 4096 || (head_size != 64 && head_size != 128 && head_size != 256) ||
      table_stride < 0 || blocks < 0)
    return SV_EINVAL;
  if (batch == 0 || tokens == 0) return SV_OK;
  if ((blocks && (!k_pool || !bounds)) || (table_stride && !table) || !starts || !counts)
    return SV_EINVAL;
  const int64_t pages = (tokens + PAGE - 2) / PAGE + 1;
  const int64_t per_wg = 8;   // 64 elements of a page and head each
  if (pages > ((int64_t)1 << 40) / num_kv_heads / batch) return SV_EINVAL;
  const int64_t grid = (batch * pages * num_kv_heads * (head_size / 64) + per_wg - 1) / per_wg;
  if (!grid_ok(grid, 256)) return SV_EINVAL;
  auto kern = head_size == 64 ? page_bounds_kernel<64> : head_size == 128 ? page_bounds_kernel<128> : page_bounds_kernel<256>;
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(256), 0, S(stream), (const uint16_t*)k_pool,
                     (uint16_t*)bounds, table, starts, counts, table_stride, blocks, (int)batch,
                     (int)num_kv_heads, (int)tokens, pages);
  SV_CHECK_LAUNCH();
  return SV_OK;
}

SV_API int64_t snowverify_page_select_scratch_bytes(int64_t batch, int64_t tokens, int64_t num_heads,
                                                    int64_t num_kv_heads, int64_t head_size,
                                                    int64_t table_stride) {
  if (!head_shape_ok(batch, tokens, num_heads, num_kv_heads, head_size) || table_stride < 0 ||
      table_stride > MAX_WIDTH || batch * tokens == 0)
    return 0;
  return select_bytes(batch, tokens, num_kv_heads, head_size, table_stride);
}

SV_API int snowverify_page_select(const void* q, const void* bounds, const int32_t* table,
                                  const int32_t* positions, int32_t* pages, int64_t batch,
                                  int64_t tokens, int64_t num_heads, int64_t num_kv_heads,
                                  int64_t head_size, int64_t table_stride, int64_t blocks,
                                  int64_t budget, int64_t sink, int64_t recent, void* scratch,
                                  int64_t scratch_bytes, void* stream) {
  if (!head_shape_ok(batch, tokens, num_heads, num_kv_heads, head_size) || table_stride < 0 ||
      table_stride > MAX_WIDTH || blocks <= 0 || budget <= 0 || budget > MAX_WIDTH || sink < 0 ||
      recent < 1 || sink > budget || recent > budget - sink)
    return SV_EINVAL;
  if (batch * tokens == 0) return SV_OK;
  if (!q || !bounds || (table_stride && !table) || !positions || !pages ||
      scratch_bytes < snowverify_page_select_scratch_bytes(batch, tokens, num_heads, num_kv_heads,
                                                           head_size, table_stride) ||
      (table_stride > 0 && !scratch))
    return SV_EINVAL;
  const int64_t chunk = select_rows(batch, tokens, num_kv_heads, head_size, table_stride);
  const SelectSpace space = select_space(batch, chunk, num_kv_heads, head_size, table_stride);
  const int64_t width = space.width;
  const int threads = width <= 256 * PICK_KEYS ? 256 : 1024;
  if (!grid_ok(batch * num_kv_heads * chunk, threads)) return SV_EINVAL;
  SelectArgs a{};
  a.q = (const uint16_t*)q;
  a.bounds = (const uint16_t*)bounds;
  a.table = table;
  a.positions = positions;
  a.pages = pages;
  uint8_t* base = (uint8_t*)scratch;
  a.exact = (uint64_t*)base;
  a.scores = (float*)(base + space.scores);
  a.errors = (float*)(base + space.errors);
  a.operands = (u32x4*)(base + space.operands);
  a.tile_last = (int32_t*)(base + space.lasts);
  a.table_stride = table_stride;
  a.blocks = blocks;
  a.width = width;
  a.T = tokens;
  a.Hq = (int)num_heads;
  a.Hkv = (int)num_kv_heads;
  a.G = (int)(num_heads / num_kv_heads);
  a.budget = (int)budget;
  a.sink = (int)sink;
  a.recent = (int)recent;
  const size_t lds = (size_t)((table_stride + 63) / 64) * 16;
  auto pick = pick_form(head_size, width);
  for (int64_t r0 = 0; r0 < tokens; r0 += chunk) {
    a.row0 = r0;
    a.rows = (int)(tokens - r0 < chunk ? tokens - r0 : chunk);
    if (table_stride > budget) {   // otherwise every page of every row is taken
      const int64_t groups = batch * num_kv_heads, tiles = (a.rows + 15) / 16;
      if (tiles > 1) {
        auto prepare = head_size == 64 ? operand_kernel<64> : head_size == 128 ? operand_kernel<128> : operand_kernel<256>;
        hipLaunchKernelGGL(prepare, dim3((unsigned)(groups * tiles)), dim3(64 * SCORE_WAVES), 0, S(stream), a);
        SV_CHECK_LAUNCH();
        // two workgroups a CU (what LDS holds of a 256-wide head), at most 64 row tiles each: choice of
        // 1024 rows over 4064 pages 65.5 us, 70.9 for one a CU, 67.9 for four
        const int64_t columns = (table_stride + 32 * SCORE_WAVES - 1) / (32 * SCORE_WAVES);
        int64_t per = tiles * groups * columns / 512;
        per = per < 1 ? 1 : per > 64 ? 64 : per;
        const int64_t parts = (tiles + per - 1) / per;
        auto score = head_size == 64 ? score_rows_kernel<64> : head_size == 128 ? score_rows_kernel<128> : score_rows_kernel<256>;
        hipLaunchKernelGGL(score, dim3((unsigned)(groups * parts * columns)), dim3(64 * SCORE_WAVES),
                           0, S(stream), a, (uint32_t)per, (uint32_t)columns);
      } else {
        // two workgroups a CU; two page tiles a step where there are pages for about all waves then
        // (eleven rows of 13751 pages and two kv heads 25.1 us, 25.9 with one; of 2048 pages 20.4 with
        // one, 22.7 with two)
        const int64_t wgs = 512;
        const int pt = table_stride * groups >= 48 * wgs ? 2 : 1;
        const int64_t step = 16 * pt * SCORE_WAVES;
        int64_t per = (table_stride * groups + wgs * step - 1) / (wgs * step) * step;
        per = per > 4096 ? 4096 : per;
        hipLaunchKernelGGL(score_form(head_size, pt == 2), dim3((unsigned)groups, (unsigned)((table_stride + per - 1) / per)),
                           dim3(64 * SCORE_WAVES), 0, S(stream), a, (uint32_t)per);
      }
      SV_CHECK_LAUNCH();
    }
    hipLaunchKernelGGL(pick, dim3((unsigned)(batch * num_kv_heads * a.rows)), dim3(threads), lds,
                       S(stream), a);
    SV_CHECK_LAUNCH();
  }
  return SV_OK;
}

SV_API int64_t snowverify_sparse_attention_scratch_bytes(int64_t batch, int64_t tokens,
                                                         int64_t num_heads, int64_t num_kv_heads,
                                                         int64_t head_size, int64_t budget) {
  if (!head_shape_ok(batch, tokens, num_heads, num_kv_heads, head_size) || budget < 0) return 0;
  const int64_t GT = (num_heads / num_kv_heads + 15) / 16;
  const int64_t s = attend_splits(batch * tokens * num_kv_heads * GT, budget);
  return s == 1 ? 0 : batch * tokens * num_heads * s * (head_size + 2) * 4;
}

SV_API int snowverify_sparse_attention(const void* q, const void* k_pool, const void* v_pool,
                                       void* out, const int32_t* table, const int32_t* positions,
                                       const int32_t* pages, int64_t batch, int64_t tokens,
                                       int64_t num_heads, int64_t num_kv_heads, int64_t head_size,
                                       int64_t table_stride, int64_t blocks, int64_t budget,
                                       float scale, void* scratch, int64_t scratch_bytes,
                                       void* stream) {
  if (!head_shape_ok(batch, tokens, num_heads, num_kv_heads, head_size) || table_stride < 0 ||
      blocks < 0 || budget < 0 || budget > 0x7fffff)
    return SV_EINVAL;
  if (batch * tokens == 0) return SV_OK;
  const int64_t need = snowverify_sparse_attention_scratch_bytes(batch, tokens, num_heads,
                                                                 num_kv_heads, head_size, budget);
  if (!q || (blocks && (!k_pool || !v_pool)) || !out || out == q || (table_stride && !table) || !positions ||
      (budget && !pages) ||
      scratch_bytes < need || (need && !scratch))
    return SV_EINVAL;
  AttendArgs a{};
  a.q = (const uint16_t*)q;
  a.k_pool = (const uint16_t*)k_pool;
  a.v_pool = (const uint16_t*)v_pool;
  a.out = (uint16_t*)out;
  a.table = table;
  a.positions = positions;
  a.pages = pages;
  a.table_stride = table_stride;
  a.blocks = blocks;
  a.T = (int)tokens;
  a.Hq = (int)num_heads;
  a.Hkv = (int)num_kv_heads;
  a.G = (int)(num_heads / num_kv_heads);
  a.GT = (a.G + 15) / 16;
  a.budget = (int)budget;
  const int64_t items = batch * tokens * num_kv_heads * a.GT;
  a.splits = attend_splits(items, budget);
  a.items = items * a.splits;
  if (!grid_ok(a.items + 8, 64 * ATT_WAVES)) return SV_EINVAL;
  a.qk_scale = scale * kLog2e;
  a.part_o = (float*)scratch;
  a.part_ml = a.splits > 1 ? a.part_o + batch * tokens * num_heads * a.splits * head_size : nullptr;
  const int hm = a.G < 16 ? a.G : 16;
  size_t lds = (size_t)attend_lds((int)head_size, hm) * 4;
  const int rpt = attend_rows_per_wave(batch, tokens, num_kv_heads, a.G, head_size, table_stride, budget);
  if (rpt) {
    a.rpt = rpt;
    a.splits = 1;
    const int64_t R = ROWS_GROUPS * rpt, ring = rows_ring_bytes(head_size, table_stride);
    a.items = batch * num_kv_heads * ((tokens + R - 1) / R);
    a.ring_bytes = (int)ring;
    // where a workgroup's rows alone take as long (eight rows of 256-wide heads: 2.7 lists' pages; sixteen
    // rows of 128-wide ones: 4 lists', 92 us for 512 rows of 64 pages and eight kv heads, 45 at 1.5 lists')
    a.union_most = (int)(R * budget / (head_size == 256 ? 3 : 4));
    lds = std::max(2 * lds, (size_t)(ring + R * budget * 8));
    auto kern = head_size == 128 ? attend_rows_kernel<128> : attend_rows_kernel<256>;
    static std::atomic<uint64_t> raised[2];
    const hipError_t err = raise_lds_limit((const void*)kern, raised[head_size / 256], ROWS_LDS);
    if (err != hipSuccess) return (int)err;
    hipLaunchKernelGGL(kern, dim3((unsigned)((a.items + 7) / 8 * 8)), dim3(64 * ROWS_WAVES), lds,
                       S(stream), a);
    SV_CHECK_LAUNCH();
    return SV_OK;
  }
  auto kern = head_size == 64 ? attend_kernel<64> : head_size == 128 ? attend_kernel<128> : attend_kernel<256>;
  hipLaunchKernelGGL(kern, dim3((unsigned)((a.items + 7) / 8 * 8)), dim3(64 * ATT_WAVES), lds,
                     S(stream), a);
  SV_CHECK_LAUNCH();
  if (a.splits > 1) {
    const int64_t rows = batch * tokens * num_heads;
    auto join = head_size == 64 ? attend_join_kernel<64> : head_size == 128 ? attend_join_kernel<128> : attend_join_kernel<256>;
    hipLaunchKernelGGL(join, dim3((unsigned)((rows * (head_size / 4) + 255) / 256)), dim3(256), 0,
                       S(stream), a.part_o, a.part_ml, a.out, rows, a.splits);
    SV_CHECK_LAUNCH();
  }
  return SV_OK;
}

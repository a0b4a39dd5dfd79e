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

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef double doublex4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef short short2v __attribute__((ext_vector_type(2)));

constexpr int PAGE = 16;
constexpr float kLog2e = 1.4426950408889634f;

inline hipStream_t S(void* s) { return (hipStream_t)s; }

// The block of request b's page, or -1 past the table's width or where the entry is no block.
__device__ __forceinline__ int page_block(const int32_t* __restrict__ table, int64_t stride, int b,
                                          int64_t page, int64_t blocks) {
  if (page < 0 || page >= stride) return -1;
  const int e = table[(int64_t)b * stride + page];
  return e >= 0 && e < blocks ? e : -1;
}

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
  const uint16_t* q;       // null: no queries
  int64_t k_stride, v_stride, q_stride;
  const float* cosv;       // [rows, half], rows cs_stride apart
  const float* sinv;
  int64_t cs_stride;
  const uint16_t* q_gamma; // null: no norm
  const uint16_t* k_gamma;
  float eps;
  uint16_t* k_pool;
  uint16_t* v_pool;
  uint16_t* bounds;        // null: none kept
  uint16_t* q_out;         // [rows, Hq, D]
  const int32_t* table;
  const int32_t* starts;   // [batch] position of a request's first row
  const int32_t* counts;   // [batch] its rows
  int64_t table_stride, blocks;
  int batch, T, Hq, Hkv, half, pages;   // pages: most pages that T rows touch
  int64_t page_wgs;        // workgroups over (request, page, kv head); the rest rotate queries
};

// Eight elements d = 8 c .. 8 c + 7 of a head, normalised and rotated; the D / 8 threads of a head
// are neighbours in one wave. The rotation partner's raw words come from its thread.
template <int D>
__device__ __forceinline__ u32x4 rotate_norm(u32x4 raw, int c, const uint16_t* gamma, float eps,
                                             const float* cr, const float* sr, int half) {
  constexpr int W = D / 8;
  float inv = 1.f;
  if (gamma) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = __uint_as_float(raw[i] << 16), b = __uint_as_float(raw[i] & 0xffff0000u);
      ss = __builtin_fmaf(a, a, ss);
      ss = __builtin_fmaf(b, b, ss);
    }
#pragma unroll
    for (int s = W / 2; s > 0; s >>= 1) ss += __shfl_xor(ss, s, W);
    inv = __frsqrt_rn(ss / (float)D + eps);
  }
  const int h8 = half / 8;
  const int pc = c < h8 ? c + h8 : c < 2 * h8 ? c - h8 : c;
  u32x4 other;
#pragma unroll
  for (int i = 0; i < 4; ++i) other[i] = (uint32_t)__shfl((int)raw[i], pc, W);
  float y[8], z[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y[2 * i] = __uint_as_float(raw[i] << 16) * inv;
    y[2 * i + 1] = __uint_as_float(raw[i] & 0xffff0000u) * inv;
    z[2 * i] = __uint_as_float(other[i] << 16) * inv;
    z[2 * i + 1] = __uint_as_float(other[i] & 0xffff0000u) * inv;
  }
  if (gamma) {
    const u32x4 g = *(const u32x4*)(gamma + 8 * c), go = *(const u32x4*)(gamma + 8 * pc);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      y[2 * i] *= __uint_as_float(g[i] << 16);
      y[2 * i + 1] *= __uint_as_float(g[i] & 0xffff0000u);
      z[2 * i] *= __uint_as_float(go[i] << 16);
      z[2 * i + 1] *= __uint_as_float(go[i] & 0xffff0000u);
    }
  }
  if (c < 2 * h8) {
    const int i0 = c < h8 ? 8 * c : 8 * (c - h8);
    const float sign = c < h8 ? -1.f : 1.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = __builtin_fmaf(y[e], cr[i0 + e], sign * (z[e] * sr[i0 + e]));
  }
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = pack_bf16x2(y[2 * i], y[2 * i + 1]);
  return o;
}

// 2 D threads: sixteen heads of D / 8 threads each. A page workgroup owns one (request, page, kv
// head): its threads take a token's row each, normalise and rotate it, and pass it through LDS into
// the page's layout, so that global reads and writes are both contiguous. The page's bounds are
// taken from the same LDS image, to which the page's older keys are loaded first: they come out the
// same whatever was in the page behind the last row (rejected drafts) and need no atomics.
template <int D>
__global__ void __launch_bounds__(2 * D) append_kernel(AppendArgs a) {
  constexpr int W = D / 8, LD = D + 8;   // row pitch of the LDS tiles: 16 bytes more than a row
  __shared__ __attribute__((aligned(16))) uint16_t ks[PAGE * LD];
  __shared__ __attribute__((aligned(16))) uint16_t vs[PAGE * LD];
  const int tid = threadIdx.x, r = tid / W, c = tid % W;
  int64_t wg = blockIdx.x;
  if (wg >= a.page_wgs) {   // queries: sixteen (row, head) units
    const int64_t u = (wg - a.page_wgs) * 16 + r;
    const int64_t m = u / a.Hq;
    const int head = (int)(u % a.Hq);
    const int64_t b = m / a.T;
    const bool live = b < a.batch && m % a.T < a.counts[b] && a.starts[b] >= 0;
    const int64_t mr = live ? m : 0;
    u32x4 raw = {0u, 0u, 0u, 0u};
    if (live) raw = *(const u32x4*)(a.q + mr * a.q_stride + (int64_t)head * D + 8 * c);
    const u32x4 o = rotate_norm<D>(raw, c, a.q_gamma, a.eps, a.cosv + mr * a.cs_stride,
                                   a.sinv + mr * a.cs_stride, a.half);
    if (live) *(u32x4*)(a.q_out + (m * a.Hq + head) * D + 8 * c) = o;
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
    const u32x4 o = rotate_norm<D>(kraw, c, a.k_gamma, a.eps, a.cosv + m * a.cs_stride,
                                   a.sinv + m * a.cs_stride, a.half);
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
// D / 8 threads per (page, kv head), eight elements each, all sixteen tokens in flight at once; a
// page's dead tokens are read as its last live one.
template <int D>
__global__ void __launch_bounds__(256) page_bounds_kernel(
    const uint16_t* __restrict__ k_pool, uint16_t* __restrict__ bounds,
    const int32_t* __restrict__ table, const int32_t* __restrict__ starts,
    const int32_t* __restrict__ counts, int64_t table_stride, int64_t blocks, int batch, int Hkv,
    int tokens, int64_t pages) {
  constexpr int W = D / 8;
  const int64_t unit = ((int64_t)blockIdx.x * 256 + threadIdx.x) / W;
  const int c = threadIdx.x % W;
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
  const uint16_t* kp = k_pool + ((int64_t)blk * Hkv + h) * PAGE * D + (c / 2) * 256 + (c % 2) * 8;
  u32x4 x[PAGE];
#pragma unroll
  for (int t = 0; t < PAGE; ++t) x[t] = *(const u32x4*)(kp + (t < last ? t : last) * 16);
  u32x4 wl, wu;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    short2v l = order_keys(x[0][i]), u = l;
#pragma unroll
    for (int t = 1; t < PAGE; ++t) {
      const short2v k = order_keys(x[t][i]);
      l = min2(l, k);
      u = max2(u, k);
    }
    uint32_t a0, b0;
    bounds_words(l, u, a0, b0);
    wl[i] = a0;
    wu[i] = b0;
  }
  uint16_t* bp = bounds + ((int64_t)blk * Hkv + h) * 2 * D + 8 * c;
  *(u32x4*)bp = wl;
  *(u32x4*)(bp + D) = wu;
}

// ---------------------------------------------------------------------------------------
// select
// ---------------------------------------------------------------------------------------
// A page's score for a row and kv head is the sum over the group's heads of the largest q . k that
// keys within the page's bounds could have:
//   sum_g sum_d max(q_gd low_d, q_gd high_d) = sum_d P_d high_d - N_d low_d,
//   P_d = sum_g max(q_gd, 0), N_d = sum_g max(-q_gd, 0),
// one product of 2 D terms per (row, kv head, page). It is taken in 64 bits: the choice turns on
// differences between nearly equal scores, and P and each product are then exact.
struct SelectArgs {
  const uint16_t* q;        // [rows, Hq, D]
  const uint16_t* bounds;
  const int32_t* table;
  const int32_t* positions; // [rows] the last position a row sees, negative: none
  int32_t* pages;           // [rows, Hkv, budget]
  double* scores;           // [requests, Hkv, T, width]
  int64_t table_stride, blocks, width, T, row0;   // row0: first row of every request in this launch
  int rows, Hq, Hkv, G, budget, sink, recent;     // rows: of a request in this launch
};

// Pages a row sees.
__device__ __forceinline__ int64_t pages_seen(int pos, int64_t stride) {
  const int64_t n = pos < 0 ? 0 : pos / PAGE + 1;
  return n < stride ? n : stride;
}

constexpr int SCORE_TILES = 4;   // 16-page tiles per step of a score workgroup

// Four waves, each a quarter of the 2 D terms (waves 0, 1: -N and the minima; 2, 3: P and the
// maxima), sixteen rows and sixteen pages a matrix instruction (v_mfma_f64_16x16x4_f64). The rows'
// operand stays in registers; a lane's 16-byte load of a page's bounds feeds eight instructions.
// The quarters are added in LDS.
template <int D>
__global__ void __launch_bounds__(256) score_kernel(SelectArgs a, int64_t pages_per_wg) {
  constexpr int NS = D / 64;   // 16-byte loads of a lane per page: D / 2 terms of a wave
  __shared__ double part[4][SCORE_TILES][256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  const int tiles = (a.rows + 15) / 16;
  int64_t y = blockIdx.x;
  const int tile = (int)(y % tiles);
  y /= tiles;
  const int h = (int)(y % a.Hkv), b = (int)(y / a.Hkv);
  const int64_t t0 = a.row0 + tile * 16;
  const bool live = tile * 16 + col < a.rows;
  const int64_t m = (int64_t)b * a.T + t0 + (live ? col : 0);
  const int64_t n = live ? pages_seen(a.positions[m], a.table_stride) : 0;
  const int64_t last = (int64_t)wave_max<int>((int)n);
  const int64_t p0 = (int64_t)blockIdx.y * pages_per_wg;
  if (p0 >= last) return;
  const int64_t p1 = p0 + pages_per_wg < last ? p0 + pages_per_wg : last;
  const int side = wave >> 1, d0 = (wave & 1) * (D / 2);
  double w[NS * 8];
#pragma unroll
  for (int i = 0; i < NS * 8; ++i) w[i] = 0.0;
  if (live)
    for (int e = 0; e < a.G; ++e) {
      const uint16_t* qp = a.q + (m * a.Hq + h * a.G + e) * D + d0 + 8 * g;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        const u32x4 x = *(const u32x4*)(qp + 32 * s);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float f = __uint_as_float(i & 1 ? x[i / 2] & 0xffff0000u : x[i / 2] << 16);
          // max(q, 0) with the maxima, min(q, 0) = -N with the minima; NaN stays
          if (side ? !(f <= 0.f) : !(f >= 0.f)) w[s * 8 + i] += (double)f;
        }
      }
    }
  for (int64_t p = p0; p < p1; p += 16 * SCORE_TILES) {
    u32x4 x[SCORE_TILES][NS];
#pragma unroll
    for (int i = 0; i < SCORE_TILES; ++i) {
      const int64_t pg = p + 16 * i + col;
      const int blk = page_block(a.table, a.table_stride, b, pg < last ? pg : last - 1, a.blocks);
      const uint16_t* bp = a.bounds + (((int64_t)(blk < 0 ? 0 : blk) * a.Hkv + h) * 2 + side) * D + d0 + 8 * g;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        x[i][s] = *(const u32x4*)(bp + 32 * s);
        if (blk < 0) x[i][s] = u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};   // NaN
      }
    }
#pragma unroll
    for (int i = 0; i < SCORE_TILES; ++i) {
      doublex4 acc = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float f = __uint_as_float(e & 1 ? x[i][s][e / 2] & 0xffff0000u : x[i][s][e / 2] << 16);
          acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)f, w[s * 8 + e], acc, 0, 0, 0);
        }
      // lane (row col, g): pages g + 4 r
#pragma unroll
      for (int r = 0; r < 4; ++r) part[wave][i][col * 16 + g + 4 * r] = acc[r];
    }
    __syncthreads();
    // thread: a row and pages of one tile
#pragma unroll
    for (int i = 0; i < SCORE_TILES; ++i) {
      const int row = threadIdx.x >> 4, pg = threadIdx.x & 15;
      const double s = (part[0][i][threadIdx.x] + part[1][i][threadIdx.x]) +
                       (part[2][i][threadIdx.x] + part[3][i][threadIdx.x]);
      if (tile * 16 + row < a.rows && p + 16 * i + pg < p1)
        a.scores[(((int64_t)b * a.Hkv + h) * a.rows + tile * 16 + row) * a.width + p + 16 * i + pg] = s;
    }
    __syncthreads();
  }
}

// 64-bit keys in the order of the scores; NaN is -inf, -0 is +0 (the rule of ord_key).
__device__ __forceinline__ uint64_t score_key(double s) {
  if (s != s) s = -__builtin_huge_val();
  if (s == 0.0) s = 0.0;
  const uint64_t u = (uint64_t)__double_as_longlong(s);
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

constexpr int PICK_THREADS = 256;

// One workgroup per (row, kv head): the need-th largest key by radix selection, eight bits a pass,
// then the pages above it and the lowest-numbered of those equal to it, in ascending order, from
// ballots kept in LDS.
__global__ void __launch_bounds__(PICK_THREADS) pick_kernel(SelectArgs a) {
  extern __shared__ uint64_t masks[];   // [words] chosen pages, then u32 [words] ranks before
  __shared__ uint32_t hist[256];
  __shared__ uint64_t sh_prefix;
  __shared__ uint32_t sh_need;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t item = blockIdx.x;      // (request, kv head, row)
  const int row = (int)(item % a.rows);
  const int h = (int)(item / a.rows % a.Hkv);
  const int64_t b = item / a.rows / a.Hkv;
  const int64_t m = b * a.T + a.row0 + row;
  int32_t* out = a.pages + (m * a.Hkv + h) * a.budget;
  const int n = (int)pages_seen(a.positions[m], a.table_stride);
  if (n <= a.budget) {
    for (int i = tid; i < a.budget; i += PICK_THREADS) out[i] = i < n ? i : -1;
    return;
  }
  const int first = a.sink, end = n - a.recent;   // candidates; n > budget >= sink + recent
  const double* sc = a.scores + item * a.width;
  uint32_t need = (uint32_t)(a.budget - a.sink - a.recent);
  uint64_t prefix = 0;
  if (need > 0)
    for (int shift = 56; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += PICK_THREADS) hist[i] = 0;
      __syncthreads();
      for (int i = first + tid; i < end; i += PICK_THREADS) {
        const uint64_t k = score_key(sc[i]);
        if (shift == 56 || (k >> (shift + 8)) == (prefix >> (shift + 8)))
          atomicAdd(&hist[(k >> shift) & 255], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        uint32_t seen = 0;
        int d = 255;
        while (d > 0 && seen + hist[d] < need) seen += hist[d--];
        sh_prefix = prefix | (uint64_t)d << shift;
        sh_need = need - seen;
      }
      __syncthreads();
      prefix = sh_prefix;
      need = sh_need;
      __syncthreads();
    }
  // `need` of the pages equal to the threshold, lowest first; all above it
  const int words = (n + 63) / 64;
  uint32_t* rank = (uint32_t*)(masks + words);
  uint64_t* equal = masks + words + (words + 1) / 2;
  for (int w = wave; w < words; w += PICK_THREADS / 64) {
    const int i = w * 64 + lane;
    const bool mid = i >= first && i < end;
    const uint64_t k = mid && a.budget > a.sink + a.recent ? score_key(sc[i]) : 0;
    const bool over = i < n && (!mid || (a.budget > a.sink + a.recent && k > prefix));
    const bool eq = mid && a.budget > a.sink + a.recent && k == prefix;
    const uint64_t mo = __ballot(over), me = __ballot(eq);
    if (lane == 0) masks[w] = mo, equal[w] = me;
  }
  __syncthreads();
  if (wave == 0) {
    uint32_t eq_before = 0, before = 0;
    for (int w0 = 0; w0 < words; w0 += 64) {
      const int w = w0 + lane;
      uint64_t mo = w < words ? masks[w] : 0, me = w < words ? equal[w] : 0;
      const uint32_t ec = (uint32_t)__popcll(me);
      const uint32_t ei = (uint32_t)wave_incl_sum_u64(ec);
      const uint32_t eb = eq_before + ei - ec;
      uint32_t take = eb >= need ? 0u : need - eb < ec ? need - eb : ec;
      while (take > 0) {   // the lowest `take` set bits
        const uint64_t bit = me & (~me + 1);
        mo |= bit;
        me ^= bit;
        --take;
      }
      const uint32_t cnt = (uint32_t)__popcll(mo);
      const uint32_t ci = (uint32_t)wave_incl_sum_u64(cnt);
      if (w < words) masks[w] = mo, rank[w] = before + ci - cnt;
      eq_before += (uint32_t)__shfl((int)ei, 63, 64);
      before += (uint32_t)__shfl((int)ci, 63, 64);
    }
  }
  __syncthreads();
  for (int w = wave; w < words; w += PICK_THREADS / 64) {
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
  float qk_scale;           // softmax scale * log2(e)
};

constexpr int ATT_WAVES = 4;

// One workgroup per (row, kv head, 16 heads of its group, split of the list), one page pair per wave
// and step. Per pair (32 keys):
//   S^T[key, head] = K . q^T       v_mfma_f32_16x16x32_bf16 over d, A = K straight from the page
//                                  (its layout is the operand's: 1 KiB per wave load)
//   O^T[d, head]  += V^T . P^T     over the 32 keys, A = V^T (a 16-byte load holds a lane's keys of
//                                  elements d and d + 1: two operands), B = P^T from S^T's registers
// so neither K, V nor P passes through LDS. P is a bf16 hi + lo pair (16 bits of mantissa): single
// bf16 weights would add about two thirds of the output's own rounding to its error.
// The running maximum and sum, and O, are 32-bit.
template <int D>
__global__ void __launch_bounds__(64 * ATT_WAVES, 2) attend_kernel(AttendArgs a) {
  constexpr int KS = D / 32;
  extern __shared__ float so[];   // [waves][heads][elements of a round + 4]
  __shared__ float sml[ATT_WAVES][16][2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
  // neighbouring rows, which list many of the same pages, run on one XCD
  const int64_t per_xcd = (int64_t)gridDim.x / 8;
  int64_t item = (int64_t)(blockIdx.x % 8) * per_xcd + blockIdx.x / 8;
  if (item >= a.items) return;
  const int split = (int)(item % a.splits);
  item /= a.splits;
  const int t = (int)(item % a.T);
  item /= a.T;
  const int gt = (int)(item % a.GT);
  item /= a.GT;
  const int h = (int)(item % a.Hkv);
  const int b = (int)(item / a.Hkv);
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

  const int parts = a.splits * ATT_WAVES, part = split * ATT_WAVES + wave;
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
      const int left_a = pos - __builtin_amdgcn_readlane(pg, ia) * PAGE + 1;
      const int left_b = two ? pos - __builtin_amdgcn_readlane(pg, ib) * PAGE + 1 : 0;
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
      float p[8];
      float top = -__builtin_huge_valf();
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[r] = 4 * g + r < left_a ? sa[r] * a.qk_scale : -__builtin_huge_valf();
        p[4 + r] = 4 * g + r < left_b ? sb[r] * a.qk_scale : -__builtin_huge_valf();
      }
#pragma unroll
      for (int r = 0; r < 8; ++r) top = fmaxf(top, p[r]);
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      if (__ballot(top > mx)) {
        const float nm = fmaxf(mx, top);
        const float c = mx == nm ? 1.f : __builtin_amdgcn_exp2f(mx - nm);   // 0 at the first pair
        mx = nm;
        l *= c;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) acc[i] *= c;
      }
      const float ref = mx == -__builtin_huge_valf() ? 0.f : mx;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        p[r] = __builtin_amdgcn_exp2f(p[r] - ref);
        l += p[r];
      }
      bf16x8 hi, lo;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        hi[r] = (__bf16)p[r];
        lo[r] = (__bf16)(p[r] - (float)hi[r]);
      }
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
        const u32x4 v0 = {ya[j][0], ya[j][1], yb[j][0], yb[j][1]};
        const u32x4 v1 = {ya[j][2], ya[j][3], yb[j][2], yb[j][3]};
        const bf16x8 f0 = __builtin_bit_cast(bf16x8, v0), f1 = __builtin_bit_cast(bf16x8, v1);
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
  for (int w = 1; w < ATT_WAVES; ++w) top = fmaxf(top, sml[w][col][0]);
  const float c = mx == top ? 1.f : __builtin_amdgcn_exp2f(mx - top);
  // in two rounds of D / 2 elements where the waves' sums would pass 64 KiB of LDS
  const int rounds = D == 256 && heads > 8 ? 2 : 1, DR = D / rounds, ld = DR + 4;
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
    for (int u = threadIdx.x; u < heads * (DR / 4); u += 64 * ATT_WAVES) {
      const int hd = u / (DR / 4), dr = u % (DR / 4) * 4, d = rd * DR + dr;
      float hm = sml[0][hd][0];
#pragma unroll
      for (int w = 1; w < ATT_WAVES; ++w) hm = fmaxf(hm, sml[w][hd][0]);
      float sum = 0.f;
      floatx4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < ATT_WAVES; ++w) {
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

// The splits of one (row, head) joined: D / 4 threads a head.
template <int D>
__global__ void __launch_bounds__(256) attend_join_kernel(const float* __restrict__ part_o,
                                                          const float* __restrict__ part_ml,
                                                          uint16_t* __restrict__ out, int64_t rows,
                                                          int splits) {
  const int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) / (D / 4);
  const int d = threadIdx.x % (D / 4) * 4;
  if (row >= rows) return;
  const float* ml = part_ml + row * splits * 2;
  const float* po = part_o + row * splits * D + d;
  float top = -__builtin_huge_valf();
  for (int s = 0; s < splits; ++s) top = fmaxf(top, ml[2 * s]);
  float sum = 0.f;
  floatx4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < splits; ++s) {
    const float c = ml[2 * s] == top ? 1.f : __builtin_amdgcn_exp2f(ml[2 * s] - top);
    sum = __builtin_fmaf(ml[2 * s + 1], c, sum);
    o += *(const floatx4*)(po + (int64_t)s * D) * c;
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
constexpr int64_t MAX_BATCH_ROWS = 1 << 24;   // batch * tokens
constexpr int64_t MAX_WIDTH = 1 << 17;        // pages of a request that the choice covers (2M tokens)

// A launch holds fewer than 2^32 threads.
bool grid_ok(int64_t wgs, int64_t threads) { return wgs <= 0xffffffffll / threads; }

bool head_shape_ok(int64_t batch, int64_t tokens, int64_t Hq, int64_t Hkv, int64_t D) {
  return batch >= 0 && tokens >= 0 && Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && Hq <= 4096 &&
         (D == 64 || D == 128 || D == 256) &&
         (tokens == 0 || batch <= MAX_BATCH_ROWS / tokens);
}

// Splits of a list: enough workgroups for two on each of 256 CUs, a page pair or more per wave.
int attend_splits(int64_t items, int64_t budget) {
  const int64_t most = (budget + 2 * ATT_WAVES - 1) / (2 * ATT_WAVES);
  int64_t s = items > 0 ? (512 + items - 1) / items : 1;
  s = s < most ? s : most;
  return (int)(s < 1 ? 1 : s);
}

// Rows of a request whose scores are in the workspace at a time (256 MiB).
int64_t select_rows(int64_t batch, int64_t tokens, int64_t Hkv, int64_t width) {
  const int64_t per_row = batch * Hkv * width * 8;
  int64_t r = per_row > 0 ? ((int64_t)256 << 20) / per_row : tokens;
  r = r / 16 * 16;
  if (r < 16) r = 16;
  return r < tokens ? r : tokens;
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
  a.q = (const uint16_t*)q;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.q_stride = q_stride;
  a.cosv = cos_in;
  a.sinv = sin_in;
  a.cs_stride = cs_stride;
  a.q_gamma = (const uint16_t*)q_gamma;
  a.k_gamma = (const uint16_t*)k_gamma;
  a.eps = eps;
  a.k_pool = (uint16_t*)k_pool;
  a.v_pool = (uint16_t*)v_pool;
  a.bounds = (uint16_t*)bounds;
  a.q_out = (uint16_t*)q_out;
  a.table = table;
  a.starts = starts;
  a.counts = counts;
  a.table_stride = table_stride;
  a.blocks = blocks;
  a.batch = (int)batch;
  a.T = (int)tokens;
  a.Hq = (int)num_heads;
  a.Hkv = (int)num_kv_heads;
  a.half = (int)half;
  a.pages = (int)((tokens + PAGE - 2) / PAGE + 1);
  a.page_wgs = batch * a.pages * num_kv_heads;
  const int64_t grid = a.page_wgs + (q ? (batch * tokens * num_heads + 15) / 16 : 0);
  if (!grid_ok(grid, 2 * head_size)) return SV_EINVAL;
  auto kern = head_size == 64 ? append_kernel<64> : head_size == 128 ? append_kernel<128> : append_kernel<256>;
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
  const int64_t per_wg = 256 / (head_size / 8);
  if (pages > ((int64_t)1 << 40) / num_kv_heads / batch) return SV_EINVAL;
  const int64_t grid = (batch * pages * num_kv_heads + per_wg - 1) / per_wg;
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
      table_stride > MAX_WIDTH)
    return 0;
  return batch * select_rows(batch, tokens, num_kv_heads, table_stride) * num_kv_heads * table_stride * 8;
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
  const int64_t chunk = select_rows(batch, tokens, num_kv_heads, table_stride);
  if (!grid_ok(batch * num_kv_heads * chunk, PICK_THREADS)) return SV_EINVAL;
  SelectArgs a{};
  a.q = (const uint16_t*)q;
  a.bounds = (const uint16_t*)bounds;
  a.table = table;
  a.positions = positions;
  a.pages = pages;
  a.scores = (double*)scratch;
  a.table_stride = table_stride;
  a.blocks = blocks;
  a.width = table_stride;
  a.T = tokens;
  a.Hq = (int)num_heads;
  a.Hkv = (int)num_kv_heads;
  a.G = (int)(num_heads / num_kv_heads);
  a.budget = (int)budget;
  a.sink = (int)sink;
  a.recent = (int)recent;
  const int64_t words = (table_stride + 63) / 64;
  const size_t lds = (size_t)(2 * words + (words + 1) / 2) * 8;
  for (int64_t r0 = 0; r0 < tokens; r0 += chunk) {
    a.row0 = r0;
    a.rows = (int)(tokens - r0 < chunk ? tokens - r0 : chunk);
    const int64_t tiles = batch * num_kv_heads * ((a.rows + 15) / 16);
    if (table_stride > budget) {   // otherwise every page of every row is taken
      int64_t per = 16 * SCORE_TILES;
      while (per < 1024 && tiles * ((table_stride + per - 1) / per) > 4096) per *= 2;
      auto kern = head_size == 64 ? score_kernel<64> : head_size == 128 ? score_kernel<128> : score_kernel<256>;
      hipLaunchKernelGGL(kern, dim3((unsigned)tiles, (unsigned)((table_stride + per - 1) / per)),
                         dim3(256), 0, S(stream), a, per);
      SV_CHECK_LAUNCH();
    }
    hipLaunchKernelGGL(pick_kernel, dim3((unsigned)(batch * num_kv_heads * a.rows)),
                       dim3(PICK_THREADS), lds, S(stream), a);
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
  if (!q || (blocks && (!k_pool || !v_pool)) || !out || (table_stride && !table) || !positions ||
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
  const int64_t dr = head_size == 256 && hm > 8 ? 128 : head_size;
  const size_t lds = (size_t)ATT_WAVES * hm * (dr + 4) * 4;
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
